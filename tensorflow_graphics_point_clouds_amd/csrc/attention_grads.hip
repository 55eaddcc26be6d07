// Gradients of the attention inside the clouds of a packed batch (attention.h has the formulas).
//
//   D_i   = do_i . o_i
//   ds    = p (do_i . v_j - D_i)                  the gradient of the logits, and of the bias
//   dq_i  = scale sum_j ds k_j      dk_j = scale sum_i ds q_i      dv_j = sum_i p do_i
//
// Two passes over the pairs, one that owns queries and one that owns keys: each sums in registers
// and writes its rows once, in an order that does not change from run to run.  (One pass would
// save two of the seven products, and would have to add to the other side's rows with float
// atomics, from every block of the cloud, in any order.)
#include "attention.h"

namespace mccnn {
namespace {

__device__ __forceinline__ v16f zero16() {
  v16f z;
#pragma unroll
  for (int r = 0; r < 16; ++r) z[r] = 0.0f;
  return z;
}

// The wavefronts of a SIMD take turns at its matrix pipe: the one in the middle of its products goes
// first (s_setprio), the other one's exponentials fill the gaps.  1 to 6 % in both passes, 7 % in the
// float32 forward pass; the bfloat16 one is between 2 % faster and 1 % slower with it and goes without.

// Query gradients: three products per pair, 16 x 1024 points of 4 x 64 float32 in 158 us (163 TFLOP/s),
// 4 x 3250 tokens causal of 16 x 128 bfloat16 in 419 (638; their logit gradients are multiplied in two
// parts, a third more on the pipe).  A block as in the forward pass (128 rows, one part of the keys).
// D is formed here and left in `delta` for the other pass.  Where the bias has a gradient every wavefront adds its logit gradients up per offset in an LDS table of its own (one
// wavefront's additions to one address are served in lane order), and the block writes the sum of its
// four.  The table is in 64 bits for the speed of it: an LDS addition of 64 floats takes 192 cycles of
// the compute unit, whatever the addresses, one of 64 doubles 8 without conflicts and 33 into 32 random
// bins.
template <typename T, int DP, int BIAS, bool VEC>
__global__ __launch_bounds__(kAttnThreads, (attn_blocks_per_cu<T, DP>())) void attn_query_grads_kernel(
    AttnBatch b, int parts, const T *__restrict__ out, const float *__restrict__ out_low,
    const T *__restrict__ dout, const float *__restrict__ row_max, const float *__restrict__ row_sum,
    float *__restrict__ delta, T *__restrict__ dq, float *__restrict__ part_dq,
    float *__restrict__ offset_grads, int grad_blocks, int copies_log2) {
  constexpr int NP = sizeof(T) == 4 ? 3 : 1;
  constexpr int KT = attn_tile_rows<T, DP>();
  constexpr int SUB = KT / 32;
  using KTile = Tile<NP, DP, KT>;
  extern __shared__ __align__(16) char smem[];
  __bf16 *ktile = reinterpret_cast<__bf16 *>(smem);
  int *kpos = reinterpret_cast<int *>(ktile + 4 * KTile::kElems);
  float *table = reinterpret_cast<float *>(kpos + (BIAS == 2 ? 6 * KT : 0));
  const int width = 2 * b.max_offset + 1, per_head = b.axes * width, copies = 1 << copies_log2;
  // [4][pack][axes][width][copies]
  double *sums = reinterpret_cast<double *>(table + ((b.pack * per_head + 1) & ~1));

  const unsigned block = attn_block(), columns = b.heads / b.pack;
  const int column = block % columns, grad_block = block / columns;
  if (grad_block >= grad_blocks) return;               // (behind the last place)
  const int place = grad_block / parts, part = grad_block % parts;
  const int head0 = column * b.pack, kv_head = head0 / (b.heads / b.kv_heads);
  CloudWork work;
  if (!find_work<false>(b, place, b.causal, work)) {
    if (BIAS && offset_grads)
      for (int i = threadIdx.x; i < b.pack * per_head; i += kAttnThreads)
        offset_grads[((int64_t)(head0 + i / per_head) * grad_blocks + grad_block) * per_head + i % per_head] = 0.0f;
    return;
  }
  const int num_q = work.num_q, shift = work.used - num_q;
  const int lane = lane_id(), wave = uniform((int)(threadIdx.x / kWave)), half = lane >> 5;

  // keys that any row of the block may look at
  int end = work.used;
  if (b.causal) {
    int64_t last = (work.first + kAttnRows - 1) / b.pack;
    if (last > num_q - 1) last = num_q - 1;
    if (last + shift + 1 < end) end = (int)(last + shift + 1);
    if (end < 0) end = 0;
  }
  // ... and any row of the wavefront
  int wave_end = 0;
  if (work.first + wave * 32 < (int64_t)num_q * b.pack) {
    wave_end = end;
    const int64_t last = (work.first + wave * 32 + 31) / b.pack;
    if (b.causal && last + shift + 1 < wave_end) wave_end = (int)(last + shift + 1);
  }
  const int tiles = (end + KT - 1) / KT;
  const int tile0 = (int)((int64_t)tiles * part / parts), tile1 = (int)((int64_t)tiles * (part + 1) / parts);

  KeyStage<T, DP, KT, BIAS, VEC> stage(b, work.k_start, end, kv_head);
  if (tile0 < tile1) stage.fetch(tile0);

  const int64_t row = work.first + wave * 32 + (lane & 31);
  const bool row_ok = row < (int64_t)num_q * b.pack;
  const int query = row_ok ? (int)(row / b.pack) : 0, g = (int)(row % b.pack);
  const int64_t q_row = work.q_start + query;
  const int head = head0 + g;
  const int64_t at = (q_row * b.heads + head) * b.dim, stat = (int64_t)head * b.num_q + q_row;

  Frag<NP> qf[DP / 16], df[DP / 16];
  float dot = 0.0f;
  {
    const T *qp = static_cast<const T *>(b.q) + q_row * b.q_row + head * b.q_head;
#pragma unroll
    for (int s = 0; s < DP / 16; ++s) {
      const int col = 16 * s + 8 * half;
      qf[s] = to_frag(row8<VEC>(qp, col, b.dim, row_ok));
      const Row8<T> d = row8<VEC>(dout + at, col, b.dim, row_ok);
      dot += dot8(d, row8<VEC>(out + at, col, b.dim, row_ok));
      if (out_low) dot += dot8(d, row8<VEC>(out_low + at, col, b.dim, row_ok));
      df[s] = to_frag(d);
    }
  }
  dot += other_half(dot);
  if (row_ok && half == 0 && part == 0) delta[stat] = dot;
  // (a row without anything to look at: its exponentials are 0 beside a base of +inf)
  const float total = row_ok ? row_sum[stat] : 0.0f;
  const float base = total == 0.0f ? INFINITY : row_max[stat], inv = total == 0.0f ? 0.0f : 1.0f / total;

  int qpos[3] = {query + shift, 0, 0};
  int wave_first = 0, wave_last = 0;                   // places of the wavefront's queries
  if constexpr (BIAS == 1) {
    const int64_t last = (work.first + wave * 32 + 31) / b.pack;
    wave_first = (int)((work.first + wave * 32) / b.pack) + shift;
    wave_last = (int)(last < num_q - 1 ? last : num_q - 1) + shift;
    if (wave_first > wave_last) wave_first = wave_last;
    if (!row_ok) qpos[0] = wave_last;
  }
  float below = 0.0f, above = 0.0f;                    // sums of a lane's blocks outside the band
  const float *lane_table = table;
  double *lane_sums = sums;
  if constexpr (BIAS != 0) {
    load_bias_table(b, head0, b.pack, table);
    lane_table = table + g * per_head;
    lane_sums = sums + (wave * b.pack + g) * per_head * copies + (lane & (copies - 1));
    if (offset_grads)
      for (int i = threadIdx.x; i < 4 * b.pack * per_head * copies; i += kAttnThreads) sums[i] = 0.0;
  }
  if constexpr (BIAS == 2) {
    for (int a = 0; a < b.axes; ++a) qpos[a] = b.q_pos[q_row * b.axes + a];
  }

  v16f acc[DP / 32];
#pragma unroll
  for (int d = 0; d < DP / 32; ++d) acc[d] = zero16();
  const float factor = b.scale * kLog2e;

  if (tile0 < tile1) stage.park(tile0, ktile, ktile + KTile::kElems, kpos);
  for (int tile = tile0; tile < tile1; ++tile) {
    const int buf = (tile - tile0) & 1;
    const uint64_t allowed = stage.allowed();
    block_lds_sync();
    if (tile + 1 < tile1) stage.fetch(tile + 1);
    const __bf16 *kt = ktile + buf * 2 * KTile::kElems, *vt = kt + KTile::kElems;
    if (tile * KT < wave_end) {
      const int key0 = tile * KT;
      const bool cut = allowed != (KT == 64 ? ~0ull : (1ull << KT) - 1) ||
                       (b.causal && key0 + KT - 1 > (int)(work.first / b.pack) + shift);
      const int limit = b.causal ? query + shift - key0 - 4 * half : KT;
#pragma unroll
      for (int u = 0; u < SUB; ++u) {
        v16f s = zero16(), dp = zero16(), rest = zero16();
        __builtin_amdgcn_s_setprio(1);
#pragma unroll
        for (int step = 0; step < DP / 16; ++step) s = mma<NP>(KTile::operand(kt, 32 * u, step), qf[step], s);
#pragma unroll
        for (int step = 0; step < DP / 16; ++step) {
          const Frag<NP> v = KTile::operand(vt, 32 * u, step);
          if constexpr (NP == 3) {
            rest = mma_split_small(Split8{v.p[0], v.p[1], v.p[2]},
                                   Split8{df[step].p[0], df[step].p[1], df[step].p[2]}, rest);
            dp = mma_large(v.p[0], df[step].p[0], dp);
          } else {
            dp = mma<NP>(v, df[step], dp);
          }
        }
        // The matrix instructions round their sums down more often than up, and D does not: with six
        // roundings per step at the size of the sum, a bias gradient over 24 M pairs was off by 2.9e-5,
        // all of it of one sign.
        __builtin_amdgcn_s_setprio(0);
        if constexpr (NP == 3) dp += rest;
        float bias[16];
        Band band = kAcross;
        if constexpr (BIAS == 1) {
          const int first = key0 + 32 * u;
          band = token_band(first, first + 31, wave_first, wave_last, b.max_offset);
          token_biases<1>(lane_table, b.max_offset, band, first + 4 * half - qpos[0], bias);
        }
        if constexpr (BIAS == 2)
          position_biases<1>(lane_table, b.axes, b.max_offset, kpos + buf * 3 * KT + 32 * u + 4 * half, KT, qpos, bias);
#pragma unroll
        for (int r = 0; r < 16; ++r) {
          float x = s[r] * factor;
          if constexpr (BIAS != 0) x += bias[r];
          s[r] = exp2_fast(x - base) * inv * (dp[r] - dot);
        }
        if (cut) {
          const unsigned bits = (unsigned)(allowed >> (32 * u)) >> (4 * half);
#pragma unroll
          for (int r = 0; r < 16; ++r)
            if (!((bits >> result_row(r)) & 1) || 32 * u + result_row(r) > limit) s[r] = 0.0f;
        }
        float outside = 0.0f;
        if constexpr (BIAS == 1) {
#pragma unroll
          for (int r = 0; r < 16; ++r) outside += s[r];
        }
        if constexpr (BIAS == 2) {
          if (offset_grads && row_ok) {
#pragma unroll
            for (int a = 0; a < 3; ++a)
              if (a < b.axes) {
                int offset[16];
                position_offsets<1>(kpos + (buf * 3 + a) * KT + 32 * u + 4 * half, qpos[a], b.max_offset, offset);
                double *middle = lane_sums + ((a * width + b.max_offset) << copies_log2);
#pragma unroll
                for (int r = 0; r < 16; ++r) atomicAdd(middle + (offset[r] << copies_log2), (double)s[r]);
              }
          }
        }
        if constexpr (BIAS == 1) {
          if (band == kBelow) {
            below += outside;
          } else if (band == kAbove) {
            above += outside;
          } else if (offset_grads && row_ok) {
#pragma unroll
            for (int r = 0; r < 16; ++r)
              atomicAdd(lane_sums + b.max_offset + clamped_offset(key0 + 32 * u + result_row(r) + 4 * half, qpos[0],
                                                                  b.max_offset),
                        (double)s[r]);
          }
        }
        __builtin_amdgcn_s_setprio(1);
#pragma unroll
        for (int t = 0; t < 2; ++t) {
          const Frag<NP> grads = result_frag<NP>(s, t);
#pragma unroll
          for (int d = 0; d < DP / 32; ++d)
            acc[d] = mma<NP>(KTile::operand_t(kt, 32 * u + 16 * t, d), grads, acc[d]);
          if constexpr (NP == 1) {             // (in two parts, known to 2^-16, as the weights)
            const Frag<NP> rest = rest_frag(s, t, grads);
#pragma unroll
            for (int d = 0; d < DP / 32; ++d)
              acc[d] = mma<NP>(KTile::operand_t(kt, 32 * u + 16 * t, d), rest, acc[d]);
          }
        }
        __builtin_amdgcn_s_setprio(0);
      }
    }
    if (tile + 1 < tile1)
      stage.park(tile + 1, ktile + (buf ^ 1) * 2 * KTile::kElems, ktile + ((buf ^ 1) * 2 + 1) * KTile::kElems,
                 kpos + (buf ^ 1) * 3 * KT);
  }
  if (row_ok) {
    const bool whole = b.dim % 4 == 0;
#pragma unroll
    for (int d = 0; d < DP / 32; ++d)
#pragma unroll
      for (int r = 0; r < 16; r += 4) {
        const int col = 32 * d + result_row(r) + 4 * half;
        float o[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) o[i] = acc[d][r + i] * b.scale;
        if (parts > 1)
          store4<float>(part_dq + (int64_t)part * b.num_q * b.heads * b.dim + at, col, b.dim, whole, o);
        else
          store4<T>(dq + at, col, b.dim, whole, o);
      }
  }
  if constexpr (BIAS != 0) {
    if (offset_grads) {
      if constexpr (BIAS == 1) {
        atomicAdd(lane_sums, (double)below);
        atomicAdd(lane_sums + 2 * b.max_offset, (double)above);
      }
      __syncthreads();
      const int n = b.pack * per_head;
      for (int i = threadIdx.x; i < n; i += kAttnThreads) {
        double total = 0.0;
        for (int w = 0; w < 4; ++w)
          for (int c = 0; c < copies; ++c) total += sums[(w * n + i) * copies + c];
        offset_grads[((int64_t)(head0 + i / per_head) * grad_blocks + grad_block) * per_head + i % per_head] = (float)total;
      }
    }
  }
}

template <typename T, int DP>
constexpr int attn_query_tile() {
  return DP == 128 ? 32 : attn_tile_rows<T, DP>();
}

// With 128 channels the values of a lane's key, beside its key, two accumulators of 64 registers and
// the products, are more than half a SIMD's registers hold (354 spilled); in LDS two blocks fit.
template <typename T, int DP>
constexpr bool attn_values_in_lds() {
  return sizeof(T) == 2 && DP == 128;
}

// Key and value gradients: four products per pair, the same batches in 198 us (174 TFLOP/s) and 634
// (565, half as much again on the pipe): the matrix pipe, and with 128 channels LDS reads of as many
// cycles.  A block owns 128 keys (32 per wavefront, one per lane) of one cloud and key head and walks
// over the queries of all heads that share them, or over one part of that walk.
template <typename T, int DP, int BIAS, bool VEC>
__global__ __launch_bounds__(kAttnThreads, (attn_blocks_per_cu<T, DP>())) void attn_key_grads_kernel(
    AttnBatch b, int parts, const T *__restrict__ dout, const float *__restrict__ row_max,
    const float *__restrict__ row_sum, const float *__restrict__ delta, T *__restrict__ dk,
    T *__restrict__ dv, float *__restrict__ part_dk, float *__restrict__ part_dv) {
  constexpr int NP = sizeof(T) == 4 ? 3 : 1;
  constexpr int QT = attn_query_tile<T, DP>();
  constexpr int SUB = QT / 32;
  using QTile = Tile<NP, DP, QT>;
  using VTile = Tile<NP, DP, kAttnRows>;
  constexpr bool kShared = attn_values_in_lds<T, DP>();
  constexpr int kChunks = QT * (DP / 8);
  constexpr int CH = (kChunks + kAttnThreads - 1) / kAttnThreads;
  extern __shared__ __align__(16) char smem[];
  __bf16 *qtile = reinterpret_cast<__bf16 *>(smem);                     // [2][Q tile, dO tile]
  __bf16 *vtile = qtile + 4 * QTile::kElems;                            // the block's values, if they are kept there
  float *stats = reinterpret_cast<float *>(vtile + (kShared ? VTile::kElems : 0));   // [2][max, 1 / sum, D][QT]
  int *qposs = reinterpret_cast<int *>(stats + 6 * QT);                 // [2][3][QT]
  float *table = reinterpret_cast<float *>(qposs + (BIAS == 2 ? 6 * QT : 0));

  const unsigned block = attn_block();
  const int column = block % b.kv_heads, place = block / b.kv_heads / parts, part = block / b.kv_heads % parts;
  CloudWork work;
  if (!find_work<true>(b, place, false, work)) return;
  const int num_q = work.num_q, shift = work.used - num_q;
  const int64_t q_start = work.q_start;
  const int lane = lane_id(), wave = uniform((int)(threadIdx.x / kWave)), half = lane >> 5;
  const int kv_head = column, group = b.heads / b.kv_heads;

  const int key = (int)work.first + wave * 32 + (lane & 31);             // in its cloud
  const int64_t k_row = work.k_start + key;
  const bool stored = key < work.capacity;
  const bool key_ok = key < work.used && (!b.key_mask || b.key_mask[k_row]);
  // (a cloud's queries and keys that no cloud holds: nothing to add, zeros are written)
  const int first_q = b.causal ? ((int)work.first > shift ? (int)work.first - shift : 0) : 0;
  const int tiles = (int)work.first < work.used && num_q > first_q ? (num_q - first_q + QT - 1) / QT : 0;
  const int64_t walk = (int64_t)tiles * group;
  const int64_t at0 = walk * part / parts, at1 = walk * (part + 1) / parts;

  v16f acc_k[DP / 32], acc_v[DP / 32];
#pragma unroll
  for (int d = 0; d < DP / 32; ++d) {
    acc_k[d] = zero16();
    acc_v[d] = zero16();
  }
  const float factor = b.scale * kLog2e;
  Frag<NP> kf[DP / 16], vf[kShared ? 1 : DP / 16];
  int kpos[3] = {key, 0, 0};
  if (at0 < at1) {
    const int64_t r = key_ok ? k_row : work.k_start;
    const T *kp = static_cast<const T *>(b.k) + r * b.k_row + kv_head * b.k_head;
    const T *vp = static_cast<const T *>(b.v) + r * b.v_row + kv_head * b.v_head;
#pragma unroll
    for (int s = 0; s < DP / 16; ++s) {
      const int col = 16 * s + 8 * half;
      kf[s] = to_frag(row8<VEC>(kp, col, b.dim, key_ok));
      const Frag<NP> v = to_frag(row8<VEC>(vp, col, b.dim, key_ok));
      if constexpr (kShared) VTile::store(vtile, wave * 32 + (lane & 31), col, v);   // (read by this wavefront alone)
      else vf[s] = v;
    }
    if constexpr (BIAS == 2) {
      for (int a = 0; a < b.axes; ++a) kpos[a] = key_ok ? b.k_pos[k_row * b.axes + a] : 0;
    }
  }

  // The walk: tile after tile of the queries, head after head of the group.
  struct Step {
    int head, query0;
  };
  const int tile_end = first_q + tiles * QT;
  auto next_step = [&](Step &at) {
    at.query0 += QT;
    if (at.query0 >= tile_end) {
      at.query0 = first_q;
      ++at.head;
    }
  };
  Row8<T> qr[CH], dr[CH];
  float top_next, sum_next, dot_next;
  int pos_next[3];
  auto fetch = [&](const Step &at) {
    const T *qp = static_cast<const T *>(b.q) + q_start * b.q_row + at.head * b.q_head;
    const T *dp = dout + (q_start * b.heads + at.head) * b.dim;
#pragma unroll
    for (int c = 0; c < CH; ++c) {
      const int chunk = c * kAttnThreads + threadIdx.x;
      const int query = at.query0 + chunk / (DP / 8), col = 8 * (chunk % (DP / 8));
      const int64_t r = query < num_q ? query : 0;
      qr[c] = load8<VEC>(qp + r * b.q_row, col, b.dim);
      dr[c] = load8<VEC>(dp + r * b.heads * b.dim, col, b.dim);
    }
    // (by every thread, as the loads above: a branch would wait for what it has loaded)
    const int query = at.query0 + (threadIdx.x & (QT - 1));
    const int64_t r = q_start + (query < num_q ? query : 0), stat = (int64_t)at.head * b.num_q + r;
    top_next = row_max[stat];
    sum_next = row_sum[stat];
    dot_next = delta[stat];
    if constexpr (BIAS == 2) {
#pragma unroll
      for (int a = 0; a < 3; ++a) pos_next[a] = b.q_pos[r * b.axes + (a < b.axes ? a : 0)];
    }
  };
  auto park = [&](const Step &at, int buf) {
    __bf16 *qt = qtile + buf * 2 * QTile::kElems, *dt = qt + QTile::kElems;
#pragma unroll
    for (int c = 0; c < CH; ++c) {
      const int chunk = c * kAttnThreads + threadIdx.x;
      if (kChunks % kAttnThreads != 0 && chunk >= kChunks) break;
      const int query = chunk / (DP / 8), col = 8 * (chunk % (DP / 8));
      const bool in = at.query0 + query < num_q;
      QTile::store(qt, query, col, to_frag(clip8<VEC>(qr[c], col, b.dim, in)));
      QTile::store(dt, query, col, to_frag(clip8<VEC>(dr[c], col, b.dim, in)));
    }
    if (threadIdx.x < QT) {
      // (a row without anything to look at: its exponentials are 0 beside a base of +inf)
      const bool some = at.query0 + (int)threadIdx.x < num_q && sum_next != 0.0f;
      float *st = stats + buf * 3 * QT + threadIdx.x;
      st[0] = some ? top_next : INFINITY;
      st[QT] = some ? 1.0f / sum_next : 0.0f;
      st[2 * QT] = some ? dot_next : 0.0f;
      if constexpr (BIAS == 2) {
#pragma unroll
        for (int a = 0; a < 3; ++a)
          if (a < b.axes) qposs[(buf * 3 + a) * QT + threadIdx.x] = pos_next[a];
      }
    }
  };

  const bool missing = __any(!key_ok);
  const int wave_key = (int)work.first + wave * 32;
  int head_of_table = -1;
  Step now{0, 0}, next;
  if (at0 < at1) {
    now = Step{kv_head * group + (int)(at0 / tiles), first_q + (int)(at0 % tiles) * QT};
    fetch(now);
    park(now, 0);
  }
  int buf = 0;
  for (int64_t left = at1 - at0; left > 0; --left, now = next, buf ^= 1) {
    const int query0 = now.query0;
    next = now;
    next_step(next);
    if constexpr (BIAS != 0) {
      if (now.head != head_of_table) {               // (a table in use is not overwritten)
        block_lds_sync();
        load_bias_table(b, now.head, 1, table);
        head_of_table = now.head;
      }
    }
    block_lds_sync();
    if (left > 1) fetch(next);
    const __bf16 *qt = qtile + buf * 2 * QTile::kElems, *dt = qt + QTile::kElems;
    const float *st = stats + buf * 3 * QT;
    const bool cut = missing || (b.causal && query0 + shift < (int)work.first + kAttnRows - 1);
    const int limit = b.causal ? key - shift - query0 - 4 * half : 0;  // first query of the tile for this key
#pragma unroll
    for (int u = 0; u < SUB; ++u) {
      // (a wavefront without keys, or with queries that all stand before its keys)
      if (wave_key >= work.used || (b.causal && query0 + 32 * u + 31 + shift < wave_key)) continue;
      v16f s = zero16(), dp = zero16();
      __builtin_amdgcn_s_setprio(1);
#pragma unroll
      for (int step = 0; step < DP / 16; ++step) s = mma<NP>(QTile::operand(qt, 32 * u, step), kf[step], s);
#pragma unroll
      for (int step = 0; step < DP / 16; ++step) {
        if constexpr (kShared)
          dp = mma<NP>(QTile::operand(dt, 32 * u, step), VTile::operand(vtile, wave * 32, step), dp);
        else
          dp = mma<NP>(QTile::operand(dt, 32 * u, step), vf[step], dp);
      }
      __builtin_amdgcn_s_setprio(0);
      float bias[16];
      if constexpr (BIAS == 1) {
        const int first = query0 + 32 * u + shift;
        token_biases<-1>(table, b.max_offset,
                         token_band(wave_key, wave_key + 31, first, first + 31, b.max_offset),
                         key - first - 4 * half, bias);
      }
      if constexpr (BIAS == 2)
        position_biases<-1>(table, b.axes, b.max_offset, qposs + buf * 3 * QT + 32 * u + 4 * half, QT, kpos, bias);
#pragma unroll
      for (int r = 0; r < 16; ++r) {
        const int query = 32 * u + result_row(r) + 4 * half;
        float x = s[r] * factor;
        if constexpr (BIAS != 0) x += bias[r];
        const float p = exp2_fast(x - st[query]) * st[QT + query];
        s[r] = p;
        dp[r] = p * (dp[r] - st[2 * QT + query]);
      }
      if (cut) {
#pragma unroll
        for (int r = 0; r < 16; ++r)
          if (!key_ok || 32 * u + result_row(r) < limit) s[r] = dp[r] = 0.0f;
      }
      __builtin_amdgcn_s_setprio(1);
      if constexpr (NP == 1) {
        // weights and logit gradients in two parts, known to 2^-16; one sum after the other, which leaves
        // the weights' registers free for the second (both at once: 34 registers spilled with 128 channels)
        auto add = [&](const v16f &x, const __bf16 *tile, v16f *acc) {
#pragma unroll
          for (int t = 0; t < 2; ++t) {
            const Frag<NP> part = result_frag<NP>(x, t);
#pragma unroll
            for (int d = 0; d < DP / 32; ++d)
              acc[d] = mma<NP>(QTile::operand_t(tile, 32 * u + 16 * t, d), part, acc[d]);
            const Frag<NP> rest = rest_frag(x, t, part);
#pragma unroll
            for (int d = 0; d < DP / 32; ++d)
              acc[d] = mma<NP>(QTile::operand_t(tile, 32 * u + 16 * t, d), rest, acc[d]);
          }
        };
        add(s, dt, acc_v);
        add(dp, qt, acc_k);
      } else {
#pragma unroll
        for (int t = 0; t < 2; ++t) {
          const Frag<NP> weights = result_frag<NP>(s, t), grads = result_frag<NP>(dp, t);
#pragma unroll
          for (int d = 0; d < DP / 32; ++d) {
            acc_v[d] = mma<NP>(QTile::operand_t(dt, 32 * u + 16 * t, d), weights, acc_v[d]);
            acc_k[d] = mma<NP>(QTile::operand_t(qt, 32 * u + 16 * t, d), grads, acc_k[d]);
          }
        }
      }
      __builtin_amdgcn_s_setprio(0);
    }
    if (left > 1) park(next, buf ^ 1);
  }
  if (!stored) return;
  const int64_t to = (k_row * b.kv_heads + kv_head) * b.dim;
  const int64_t to_part = (int64_t)part * b.num_k * b.kv_heads * b.dim;
  const bool whole = b.dim % 4 == 0;
#pragma unroll
  for (int d = 0; d < DP / 32; ++d)
#pragma unroll
    for (int r = 0; r < 16; r += 4) {
      const int col = 32 * d + result_row(r) + 4 * half;
      float gk[4], gv[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        gk[i] = acc_k[d][r + i] * b.scale;
        gv[i] = acc_v[d][r + i];
      }
      if (parts > 1) {
        store4<float>(part_dk + to_part + to, col, b.dim, whole, gk);
        store4<float>(part_dv + to_part + to, col, b.dim, whole, gv);
      } else {
        store4<T>(dk + to, col, b.dim, whole, gk);
        store4<T>(dv + to, col, b.dim, whole, gv);
      }
    }
}

// out[i] = sum over the parts, W wavefronts for 64 values, each with every W-th part.
template <typename T, int W>
__global__ __launch_bounds__(kAttnThreads) void attn_add_parts_kernel(int64_t n, int parts,
                                                                      const float *__restrict__ in,
                                                                      T *__restrict__ out) {
  __shared__ float sums[kAttnThreads];
  const int wave = threadIdx.x / kWave, turn = wave % W;
  const int64_t i = ((int64_t)blockIdx.x * (4 / W) + wave / W) * kWave + lane_id();
  float s = 0.0f;
  if (i < n) {
#pragma unroll 8
    for (int p = turn; p < parts; p += W) s += in[p * n + i];
  }
  if constexpr (W > 1) {
    sums[threadIdx.x] = s;
    __syncthreads();
#pragma unroll
    for (int j = 1; j < W; ++j) s += turn == 0 ? sums[threadIdx.x + j * kWave] : 0.0f;
  }
  if (turn == 0 && i < n) out[i] = (T)s;
}
template <typename T>
int add_parts(hipStream_t s, int64_t n, int parts, const float *in, void *out) {
  auto kernel = parts > 8 ? attn_add_parts_kernel<T, 4> : attn_add_parts_kernel<T, 1>;
  kernel<<<blocks_for(n, parts > 8 ? kWave : kAttnThreads), kAttnThreads, 0, s>>>(n, parts, in, static_cast<T *>(out));
  MCCNN_LAUNCH_CHECK();
  return MCCNN_OK;
}

// Sums per offset over the blocks, sixteen offsets of a head per block and sixteen lanes over the blocks
// for each.  The sums run over millions of terms of either sign: in 64 bits from here on.
__global__ __launch_bounds__(kAttnThreads) void attn_offset_sums_kernel(int64_t blocks, int per_head,
                                                                        const float *__restrict__ in,
                                                                        double *__restrict__ out) {
  __shared__ double lds[16][17];
  const int lane = threadIdx.x & 15, group = threadIdx.x >> 4, o = blockIdx.x * 16 + lane;
  const int64_t head = blockIdx.y;
  double s = 0.0;
  if (o < per_head) {
#pragma unroll 8
    for (int64_t k = group; k < blocks; k += 16) s += (double)in[(head * blocks + k) * per_head + o];
  }
  lds[group][lane] = s;
  __syncthreads();
  if (group == 0 && o < per_head) {
    double total = 0.0;
#pragma unroll
    for (int i = 0; i < 16; ++i) total += lds[i][lane];
    out[head * per_head + o] = total;
  }
}

// Sums per bucket: a wavefront per (axis, bucket, head) over the offsets of the axis.  (64-bit indices:
// nothing bounds the buckets of a table.)
constexpr int64_t kBucketBlocks = 1 << 20;
__global__ __launch_bounds__(kAttnThreads) void attn_bucket_sums_kernel(int axes, int num_buckets, int heads,
                                                                        int width, const int *__restrict__ buckets,
                                                                        const double *__restrict__ in,
                                                                        float *__restrict__ dtable) {
  constexpr int kWaves = kAttnThreads / kWave;
  const int64_t n = (int64_t)axes * num_buckets * heads;
  for (int64_t i = (int64_t)blockIdx.x * kWaves + threadIdx.x / kWave; i < n; i += (int64_t)gridDim.x * kWaves) {
    const int head = (int)(i % heads), bucket = (int)(i / heads % num_buckets), axis = (int)(i / heads / num_buckets);
    double s = 0.0;
    for (int o = lane_id(); o < width; o += kWave)
      if (buckets[o] == bucket) s += in[((int64_t)head * axes + axis) * width + o];
#pragma unroll
    for (int off = kWave / 2; off > 0; off >>= 1) s += __shfl_xor(s, off, kWave);
    if (lane_id() == 0) dtable[i] = (float)s;
  }
}


struct GradPlan {
  int q_pack, q_parts, k_parts;
  int64_t grad_blocks;                     // blocks that write sums per offset, per head
  size_t delta, part_q, part_k, part_v, offsets, sums, bytes;
};
GradPlan grad_plan(const AttnBatch &b, bool table) {
  GradPlan p{};
  p.q_pack = attn_pack(b, kAttnMaxOffsets);
  p.q_parts = attn_parts(b.num_q * p.q_pack, b.clouds, b.heads / p.q_pack, b.num_k, b.causal);
  p.k_parts = attn_parts(b.num_k, b.clouds, b.kv_heads, b.num_q * (b.heads / b.kv_heads), b.causal);
  const int per_head = b.axes * (2 * b.max_offset + 1);
  size_t at = 0;
  auto take = [&](size_t bytes) {
    const size_t here = at;
    at += align256(bytes);
    return here;
  };
  p.delta = take((size_t)b.num_q * b.heads * sizeof(float));
  const size_t q = (size_t)b.num_q * b.heads * b.dim, k = (size_t)b.num_k * b.kv_heads * b.dim;
  p.part_q = take(p.q_parts > 1 ? p.q_parts * q * sizeof(float) : 0);
  p.part_k = take(p.k_parts > 1 ? p.k_parts * k * sizeof(float) : 0);
  p.part_v = take(p.k_parts > 1 ? p.k_parts * k * sizeof(float) : 0);
  p.grad_blocks = attn_places(b.num_q * p.q_pack, b.clouds) * p.q_parts;
  if (table) {
    p.offsets = take((size_t)b.heads * p.grad_blocks * per_head * sizeof(float));
    p.sums = take((size_t)b.heads * per_head * sizeof(double));
  }
  p.bytes = at;
  return p;
}

template <typename T, int DP, int BIAS, bool VEC>
int launch_grads(hipStream_t s, AttnBatch b, const GradPlan &p, const void *out, const float *out_low,
                 const float *row_max, const float *row_sum, const void *dout, char *ws, void *dq, void *dk,
                 void *dv, float *dtable) {
  constexpr int NP = sizeof(T) == 4 ? 3 : 1, KT = attn_tile_rows<T, DP>();
  const size_t tiles = 4 * Tile<NP, DP, KT>::kElems * sizeof(__bf16);
  const int per_head = b.axes * (2 * b.max_offset + 1);
  auto at = [&](size_t offset) { return reinterpret_cast<float *>(ws + offset); };
  float *delta = at(p.delta), *offsets = dtable ? at(p.offsets) : nullptr;
  if (b.num_q > 0) {
    b.pack = p.q_pack;
    // Lanes of other queries and keys meet in few bins where positions are cells: neighbouring lanes add
    // to copies of the table, side by side, as far as two blocks fit a compute unit's LDS.  (Places of
    // tokens are other bins for every lane.)
    const size_t offsets_of_block = (size_t)b.pack * per_head, sums = dtable ? 4 * offsets_of_block * sizeof(double) : 0;
    const size_t others = tiles + (BIAS == 2 ? 6 * KT * sizeof(int) : 0) + ((offsets_of_block + 1) & ~1) * sizeof(float);
    int copies_log2 = 0;
    while (BIAS == 2 && copies_log2 < 3 && others + (sums << (copies_log2 + 1)) <= 80 * 1024) ++copies_log2;
    const size_t lds = others + (sums << copies_log2);
    auto kernel = attn_query_grads_kernel<T, DP, BIAS, VEC>;
    if (const int rc = allow_lds(reinterpret_cast<const void *>(kernel), lds)) return rc;
    const int64_t grid = p.grad_blocks * (b.heads / b.pack);
    MCCNN_REQUIRE(grid <= kAttnMaxBlocks, "attention gradients of %lld queries and %d heads take too many blocks",
                  (long long)b.num_q, b.heads);
    kernel<<<attn_grid(grid), kAttnThreads, lds, s>>>(b, p.q_parts, static_cast<const T *>(out), out_low,
                                           static_cast<const T *>(dout), row_max, row_sum, delta, static_cast<T *>(dq),
                                           at(p.part_q), offsets, (int)p.grad_blocks, copies_log2);
    MCCNN_LAUNCH_CHECK();
    if (p.q_parts > 1) {
      const int64_t n = b.num_q * b.heads * b.dim;
      if (const int rc = add_parts<T>(s, n, p.q_parts, at(p.part_q), dq)) return rc;
    }
  }
  if (b.num_k > 0 && dk) {
    b.pack = 1;
    constexpr int QT = attn_query_tile<T, DP>();
    const size_t lds = 4 * Tile<NP, DP, QT>::kElems * sizeof(__bf16) + 6 * QT * sizeof(float) +
                       (attn_values_in_lds<T, DP>() ? Tile<NP, DP, kAttnRows>::kElems * sizeof(__bf16) : 0) +
                       (BIAS == 2 ? 6 * QT * sizeof(int) : 0) + per_head * sizeof(float);
    auto kernel = attn_key_grads_kernel<T, DP, BIAS, VEC>;
    if (const int rc = allow_lds(reinterpret_cast<const void *>(kernel), lds)) return rc;
    const int64_t grid = attn_places(b.num_k, b.clouds) * b.kv_heads * p.k_parts;
    MCCNN_REQUIRE(grid <= kAttnMaxBlocks, "attention gradients of %lld keys and %d heads take too many blocks",
                  (long long)b.num_k, b.kv_heads);
    kernel<<<attn_grid(grid), kAttnThreads, lds, s>>>(b, p.k_parts, static_cast<const T *>(dout), row_max, row_sum, delta,
                                           static_cast<T *>(dk), static_cast<T *>(dv), at(p.part_k), at(p.part_v));
    MCCNN_LAUNCH_CHECK();
    if (p.k_parts > 1) {
      const int64_t n = b.num_k * b.kv_heads * b.dim;
      if (const int rc = add_parts<T>(s, n, p.k_parts, at(p.part_k), dk)) return rc;
      if (const int rc = add_parts<T>(s, n, p.k_parts, at(p.part_v), dv)) return rc;
    }
  }
  if (dtable) {
    double *sums = reinterpret_cast<double *>(ws + p.sums);
    const dim3 grid(blocks_for(per_head, 16), (unsigned)b.heads);
    attn_offset_sums_kernel<<<grid, kAttnThreads, 0, s>>>(b.num_q > 0 ? p.grad_blocks : 0, per_head, offsets, sums);
    MCCNN_LAUNCH_CHECK();
    const int64_t blocks = ((int64_t)b.axes * b.num_buckets * b.heads + kAttnThreads / kWave - 1) / (kAttnThreads / kWave);
    attn_bucket_sums_kernel<<<(unsigned)(blocks < kBucketBlocks ? blocks : kBucketBlocks), kAttnThreads, 0, s>>>(
        b.axes, b.num_buckets, b.heads, 2 * b.max_offset + 1, b.buckets, sums, dtable);
    MCCNN_LAUNCH_CHECK();
  }
  return MCCNN_OK;
}

bool aligned16(const void *p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }

}  // namespace
}  // namespace mccnn

using namespace mccnn;

extern "C" size_t mccnn_attention_grads_workspace_bytes(const mccnn_attention *attention_host, int with_table) {
  AttnBatch b;
  if (attn_batch(attention_host, b) != MCCNN_OK) return 0;
  return grad_plan(b, with_table && b.axes).bytes;
}

extern "C" int mccnn_attention_grads(mccnn_stream_t stream, const mccnn_attention *attention_host, const void *out,
                                     const float *out_low, const float *row_max, const float *row_sum,
                                     const void *dout, void *workspace, size_t workspace_bytes, void *dq, void *dk,
                                     void *dv, float *dtable) {
  AttnBatch b;
  if (const int rc = attn_batch(attention_host, b)) return rc;
  MCCNN_REQUIRE(!dtable || b.axes, "attention without a relative bias has no gradient of its table");
  MCCNN_REQUIRE((out && row_max && row_sum && dout && dq) || b.num_q == 0, "attention gradients got a null tensor");
  MCCNN_REQUIRE((dk == nullptr) == (dv == nullptr), "attention writes the gradients of keys and values or neither");
  const GradPlan p = grad_plan(b, dtable != nullptr);
  MCCNN_REQUIRE(workspace_bytes >= p.bytes && (workspace || p.bytes == 0),
                "attention gradients workspace too small: %zu < %zu", workspace_bytes, p.bytes);
  b.vec = b.vec && aligned16(out) && aligned16(out_low) && aligned16(dout);
  hipStream_t s = as_stream(stream);
  auto launch = [&](auto type, auto dp, auto bias, auto vec) {
    return launch_grads<decltype(type), decltype(dp)::value, decltype(bias)::value, decltype(vec)::value != 0>(
        s, b, p, out, out_low, row_max, row_sum, dout, static_cast<char *>(workspace), dq, dk, dv, dtable);
  };
  return attention_host->dtype == MCCNN_FLOAT32 ? attn_dispatch_bias<float>(b, launch)
                                                : attn_dispatch_bias<__bf16>(b, launch);
}
