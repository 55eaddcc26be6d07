// Forward pass of the attention inside the clouds of a packed batch (attention.h has the formulas).
#include "attention.h"

namespace mccnn {
namespace {

// How far above the reference point of a row's exponentials (in units of log 2) a logit may lie before
// the point moves.
constexpr float kSlack = 8.0f;

// One block: 128 rows (32 per wavefront) of one cloud and head, and one part of the cloud's keys,
// which pass through LDS in tiles that the four wavefronts share, two tiles deep (the next one is
// in flight to registers while the current one is multiplied).  A lane owns one row: its reference
// point, its share of the running sum (the other half of the row's keys belongs to the lane 32
// further) and a column of the transposed result.
//
// Bound, with full rows, by the matrix pipe and the exponentials beside it (per wavefront and 32 x 32
// logits 32 cycles for each of the 48 float32 / 12 bfloat16 matrix instructions of 64 channels, some
// 300 / 200 vector instructions of 4 and 16 exponentials of 16): 8 x 4096 tokens of 4 x 64 float32 in
// 684 us are 201 TFLOP/s, six times that on the bf16 pipe; of 4 x 128 bfloat16 in 407 us 675, half as
// much again on the pipe.  With a query per cloud by memory: 4 x 200 k keys, 655 MB in 132 us.  Small
// batches by a block's walk: 5 us for an empty one, 1.5 us per tile.
template <typename T, int DP, int BIAS, bool VEC>
__global__ __launch_bounds__(kAttnThreads, (attn_forward_blocks_per_cu<T, DP, BIAS>())) void attn_forward_kernel(
    AttnBatch b, int parts, T *__restrict__ out, float *__restrict__ out_low,
    float *__restrict__ part_out, float *__restrict__ row_max, float *__restrict__ row_sum) {
  constexpr int NP = sizeof(T) == 4 ? 3 : 1;
  constexpr int KT = attn_tile_rows<T, DP>();
  constexpr int SUB = KT / 32;
  using KTile = Tile<NP, DP, KT>;
  extern __shared__ __align__(16) char smem[];
  __bf16 *ktile = reinterpret_cast<__bf16 *>(smem);                    // [2][K tile, V tile]
  int *kpos = reinterpret_cast<int *>(ktile + 4 * KTile::kElems);      // [2][3][KT]
  float *table = reinterpret_cast<float *>(kpos + (BIAS == 2 ? 6 * KT : 0));

  const unsigned block = attn_block(), columns = b.heads / b.pack;
  const int column = block % columns, place = block / columns / parts, part = block / columns % parts;
  CloudWork work;
  if (!find_work<false>(b, place, b.causal, work)) return;
  const int num_q = work.num_q, shift = work.used - num_q;
  const int lane = lane_id(), wave = uniform((int)(threadIdx.x / kWave)), half = lane >> 5;
  const int head0 = column * b.pack, kv_head = head0 / (b.heads / b.kv_heads);

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

  Frag<NP> qf[DP / 16];
  {
    const T *qp = static_cast<const T *>(b.q) + q_row * b.q_row + (head0 + g) * b.q_head;
#pragma unroll
    for (int s = 0; s < DP / 16; ++s) {
      const int col = 16 * s + 8 * half;
      qf[s] = to_frag(row8<VEC>(qp, col, b.dim, row_ok));
    }
  }
  int qpos[3] = {query + shift, 0, 0};
  int wave_first = 0, wave_last = 0;                   // places of the wavefront's queries
  if constexpr (BIAS == 1) {
    const int64_t last = (work.first + wave * 32 + 31) / b.pack;
    wave_first = (int)((work.first + wave * 32) / b.pack) + shift;
    wave_last = (int)(last < num_q - 1 ? last : num_q - 1) + shift;
    if (wave_first > wave_last) wave_first = wave_last;
    if (!row_ok) qpos[0] = wave_last;
  }
  const float *lane_table = table;
  if constexpr (BIAS != 0) {
    load_bias_table(b, head0, b.pack, table);
    lane_table = table + g * b.axes * (2 * b.max_offset + 1);
  }
  if constexpr (BIAS == 2) {
    for (int a = 0; a < b.axes; ++a) qpos[a] = b.q_pos[q_row * b.axes + a];
  }

  v16f acc[DP / 32];
#pragma unroll
  for (int d = 0; d < DP / 32; ++d)
#pragma unroll
    for (int r = 0; r < 16; ++r) acc[d][r] = 0.0f;
  float top = -INFINITY, base = 0.0f, sum = 0.0f;
  const float factor = b.scale * kLog2e;

  if (tile0 < tile1) stage.park(tile0, ktile, ktile + KTile::kElems, kpos);
  for (int tile = tile0; tile < tile1; ++tile) {
    const int buf = (tile - tile0) & 1;
    const uint64_t allowed = stage.allowed();
    block_lds_sync();
    if (tile + 1 < tile1) stage.fetch(tile + 1);
    const __bf16 *kt = ktile + buf * 2 * KTile::kElems, *vt = kt + KTile::kElems;
    if (tile * KT < wave_end) {
      v16f s[SUB];
      if constexpr (NP == 3) __builtin_amdgcn_s_setprio(1);       // (as in attention_grads.hip)
#pragma unroll
      for (int u = 0; u < SUB; ++u) {
#pragma unroll
        for (int r = 0; r < 16; ++r) s[u][r] = 0.0f;
#pragma unroll
        for (int step = 0; step < DP / 16; ++step)
          s[u] = mma<NP>(KTile::operand(kt, 32 * u, step), qf[step], s[u]);
      }
      if constexpr (NP == 3) __builtin_amdgcn_s_setprio(0);
      // With a bias: the logits.  Without one the products themselves, factor and base come with the
      // exponential.  What may not be looked at at -inf.
      const int key0 = tile * KT;
#pragma unroll
      for (int u = 0; u < SUB; ++u) {
        if constexpr (BIAS != 0) {
          float bias[16];
          if constexpr (BIAS == 1) {
            const int first = key0 + 32 * u;
            token_biases<1>(lane_table, b.max_offset, token_band(first, first + 31, wave_first, wave_last, b.max_offset),
                            first + 4 * half - qpos[0], bias);
          } else {
            position_biases<1>(lane_table, b.axes, b.max_offset, kpos + buf * 3 * KT + 32 * u + 4 * half, KT, qpos, bias);
          }
#pragma unroll
          for (int r = 0; r < 16; ++r) s[u][r] = s[u][r] * factor + bias[r];
        }
      }
      if (allowed != (KT == 64 ? ~0ull : (1ull << KT) - 1) ||
          (b.causal && key0 + KT - 1 > (int)(work.first / b.pack) + shift)) {
        const int limit = b.causal ? query + shift - key0 - 4 * half : KT;   // last key of the tile for this row
#pragma unroll
        for (int u = 0; u < SUB; ++u) {
          const unsigned bits = (unsigned)(allowed >> (32 * u)) >> (4 * half);
#pragma unroll
          for (int r = 0; r < 16; ++r)
            if (!((bits >> result_row(r)) & 1) || 32 * u + result_row(r) > limit) s[u][r] = -INFINITY;
        }
      }
      float most = s[0][0];
#pragma unroll
      for (int u = 0; u < SUB; ++u)
#pragma unroll
        for (int r = 0; r < 16; ++r) most = fmaxf(most, s[u][r]);
      most = fmaxf(most, other_half(most));
      if constexpr (BIAS == 0) most *= factor;
      // The reference point of the exponentials moves only when a logit is more than 2^8 times above
      // it (sums and results in float32 have room for that, and roundings are relative): most
      // tiles then leave the accumulators alone.
      if (__any(most > top + kSlack)) {
        const float next = fmaxf(most, top);
        base = next == -INFINITY ? 0.0f : next;
        const float keep = exp2_fast(top - base);
        top = next;
        sum *= keep;
#pragma unroll
        for (int d = 0; d < DP / 32; ++d)
#pragma unroll
          for (int r = 0; r < 16; ++r) acc[d][r] *= keep;
      }
#pragma unroll
      for (int u = 0; u < SUB; ++u)
#pragma unroll
        for (int r = 0; r < 16; ++r) {
          const float p = exp2_fast(BIAS ? s[u][r] - base : s[u][r] * factor - base);
          s[u][r] = p;
          sum += p;
        }
      if constexpr (NP == 3) __builtin_amdgcn_s_setprio(1);
      // bfloat16 weights in two parts, known to 2^-15 (one part alone, 2^-8, left outputs 2.4e-3 off instead
      // of the 1.66e-3 of their own rounding, and D = do . o of the gradients with them).  Behind a relative
      // bias in three: gradients of its table are in float32, and they add up differences between o and
      // the weights over a bucket's pairs to 2 to 8e-6 of their size (with three 2e-7).  16 k causal
      // tokens of 8 x 64 without a bias take 74 us with one part and 90 with two, with a bias 86 with one
      // and 122 with three; one query over 4 x 200 k keys 133 and 136.  A call that a gradient will
      // follow gives the same bits as one that none will.  (Operands of the values held for all parts:
      // as fast or slower, 127 -> 145 us where they cost the third block of a compute unit.)
#pragma unroll
      for (int u = 0; u < SUB; ++u)
#pragma unroll
        for (int t = 0; t < 2; ++t) {
          constexpr int P = NP == 3 ? 1 : BIAS ? 3 : 2;
          Frag<NP> p[P];
          if constexpr (NP == 3) p[0] = result_frag<NP>(s[u], t);
          else weight_parts<P>(s[u], t, p);
#pragma unroll
          for (int q = 0; q < P; ++q)
#pragma unroll
            for (int d = 0; d < DP / 32; ++d)
              acc[d] = mma<NP>(KTile::operand_t(vt, 32 * u + 16 * t, d), p[q], acc[d]);
        }
      if constexpr (NP == 3) __builtin_amdgcn_s_setprio(0);
    }
    if (tile + 1 < tile1)
      stage.park(tile + 1, ktile + (buf ^ 1) * 2 * KTile::kElems, ktile + ((buf ^ 1) * 2 + 1) * KTile::kElems,
                 kpos + (buf ^ 1) * 3 * KT);
  }
  sum += other_half(sum);
  if (!row_ok) return;

  const int head = head0 + g;
  const int64_t stat = (int64_t)(part * b.heads + head) * b.num_q + q_row;
  if (half == 0 && row_max) {
    row_max[stat] = top;
    row_sum[stat] = sum;
  }
  const float inv = parts > 1 ? 1.0f : sum == 0.0f ? 0.0f : 1.0f / sum;
  const int64_t at = (q_row * b.heads + head) * b.dim;
  const bool whole = b.dim % 4 == 0;
#pragma unroll
  for (int d = 0; d < DP / 32; ++d)
#pragma unroll
    for (int r = 0; r < 16; r += 4) {
      const int col = 32 * d + result_row(r) + 4 * half;
      float o[4], low[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        o[i] = acc[d][r + i] * inv;
        low[i] = o[i] - (float)(T)o[i];
      }
      if (parts > 1) {
        store4<float>(part_out + (int64_t)part * b.num_q * b.heads * b.dim + at, col, b.dim, whole, o);
      } else {
        store4<T>(out + at, col, b.dim, whole, o);
        if (out_low) store4<float>(out_low + at, col, b.dim, whole, low);
      }
    }
}

// Parts of a row's keys put together: the parts' sums at the common maximum.  W wavefronts per row: each
// takes the weights of all parts (a lane four of them) and every W-th part, its lanes run over the
// channels.
constexpr int kMostParts = 256;
template <typename T, int W>
__global__ __launch_bounds__(kAttnThreads) void attn_join_kernel(
    int64_t num_q, int heads, int dim, int parts, const float *__restrict__ part_out,
    const float *__restrict__ part_max, const float *__restrict__ part_sum, T *__restrict__ out,
    float *__restrict__ out_low, float *__restrict__ row_max, float *__restrict__ row_sum) {
  constexpr int kRows = 4 / W;
  __shared__ float weight[kRows][kMostParts], sums[4][kAttnMaxDim];
  const int lane = lane_id(), wave = threadIdx.x / kWave, mine = wave / W, turn = wave % W;
  const int64_t rows = num_q * heads, row = (int64_t)blockIdx.x * kRows + mine, q = row / heads;
  const int head = (int)(row % heads);
  const bool in = row < rows;
  float m[4], l[4], top = -INFINITY, sum = 0.0f;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int p = lane + i * kWave;
    const int64_t at = ((int64_t)p * heads + head) * num_q + q;
    m[i] = in && p < parts ? part_max[at] : -INFINITY;
    l[i] = in && p < parts ? part_sum[at] : 0.0f;
    top = fmaxf(top, m[i]);
  }
#pragma unroll
  for (int off = kWave / 2; off > 0; off >>= 1) top = fmaxf(top, __shfl_xor(top, off, kWave));
  const float base = top == -INFINITY ? 0.0f : top;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float w = exp2_fast(m[i] - base);
    if (turn == 0) weight[mine][lane + i * kWave] = w;
    sum += l[i] * w;
  }
  sum = wave_sum(sum);
  __syncthreads();
#pragma unroll
  for (int c = 0; c < 2; ++c) {
    const int col = lane + c * kWave;
    float o = 0.0f;
    if (in && col < dim) {
#pragma unroll 8
      for (int p = turn; p < parts; p += W) o += part_out[((int64_t)p * rows + row) * dim + col] * weight[mine][p];
    }
    sums[wave][col] = o;
  }
  __syncthreads();
  if (!in || turn != 0) return;
#pragma unroll
  for (int c = 0; c < 2; ++c) {
    const int col = lane + c * kWave;
    if (col >= dim) break;
    float total = sums[wave][col];
#pragma unroll
    for (int i = 1; i < W; ++i) total += sums[wave + i][col];
    const float v = sum == 0.0f ? 0.0f : total / sum;
    const T rounded = (T)v;
    out[row * dim + col] = rounded;
    if (out_low) out_low[row * dim + col] = v - (float)rounded;
  }
  if (lane == 0 && row_max) {
    row_max[(int64_t)head * num_q + q] = top;
    row_sum[(int64_t)head * num_q + q] = sum;
  }
}

struct ForwardPlan {
  int parts;
  size_t part_out, part_max, part_sum, bytes;      // offsets in the workspace
};
ForwardPlan forward_plan(AttnBatch &b) {
  ForwardPlan p{};
  b.pack = attn_pack(b, 8192);
  // 768 and 1024 blocks of few rows, 32 channels: 4 x 200 k keys of two heads in float32 107 and 96 us, in
  // bfloat16 60.8 and 60.4; 5 x 12 k keys of eight heads 45.7 and 44.8, 29.1 and 29.5.
  const int few = b.dim <= 32 && !b.axes ? 1024 : 768;
  p.parts = attn_parts(b.num_q * b.pack, b.clouds, b.heads / b.pack, b.num_k, b.causal, few);
  if (p.parts > 1) {
    const size_t rows = (size_t)p.parts * b.num_q * b.heads;
    p.part_max = align256(rows * b.dim * sizeof(float));
    p.part_sum = p.part_max + align256(rows * sizeof(float));
    p.bytes = p.part_sum + align256(rows * sizeof(float));
  }
  return p;
}

template <typename T, int DP, int BIAS, bool VEC>
int launch_forward(hipStream_t s, const AttnBatch &b, const ForwardPlan &p, void *out, float *out_low,
                   float *row_max, float *row_sum, char *ws) {
  constexpr int NP = sizeof(T) == 4 ? 3 : 1, KT = attn_tile_rows<T, DP>();
  const size_t lds = 4 * Tile<NP, DP, KT>::kElems * sizeof(__bf16) + (BIAS == 2 ? 6 * KT * sizeof(int) : 0) +
                     (size_t)b.pack * b.axes * (2 * b.max_offset + 1) * sizeof(float);
  auto kernel = attn_forward_kernel<T, DP, BIAS, VEC>;
  if (const int rc = allow_lds(reinterpret_cast<const void *>(kernel), lds)) return rc;
  const int64_t grid = attn_places(b.num_q * b.pack, b.clouds) * (b.heads / b.pack) * p.parts;
  MCCNN_REQUIRE(grid <= kAttnMaxBlocks, "attention of %lld queries and %d heads takes too many blocks",
                (long long)b.num_q, b.heads);
  float *part_out = reinterpret_cast<float *>(ws + p.part_out);
  float *part_max = reinterpret_cast<float *>(ws + p.part_max), *part_sum = reinterpret_cast<float *>(ws + p.part_sum);
  kernel<<<attn_grid(grid), kAttnThreads, lds, s>>>(b, p.parts, static_cast<T *>(out), out_low, part_out,
                                          p.parts > 1 ? part_max : row_max, p.parts > 1 ? part_sum : row_sum);
  MCCNN_LAUNCH_CHECK();
  if (p.parts > 1) {
    const int64_t rows = b.num_q * b.heads;
    auto join = rows < 2048 ? attn_join_kernel<T, 4> : attn_join_kernel<T, 1>;
    join<<<blocks_for(rows, rows < 2048 ? 1 : 4), kAttnThreads, 0, s>>>(
        b.num_q, b.heads, b.dim, p.parts, part_out, part_max, part_sum, static_cast<T *>(out),
        out_low, row_max, row_sum);
    MCCNN_LAUNCH_CHECK();
  }
  return MCCNN_OK;
}

bool aligned16(const void *p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }

}  // namespace

int attn_batch(const mccnn_attention *a, AttnBatch &b) {
  MCCNN_REQUIRE(a, "attention expects a description of the batch");
  MCCNN_REQUIRE(a->dtype == MCCNN_FLOAT32 || a->dtype == MCCNN_BFLOAT16,
                "attention expects float32 or bfloat16 features, got type %d", a->dtype);
  MCCNN_REQUIRE(a->dim >= 1 && a->dim <= kAttnMaxDim, "attention expects 1 to %d channels per head, got %d",
                kAttnMaxDim, a->dim);
  MCCNN_REQUIRE(a->kv_heads >= 1 && a->heads >= a->kv_heads && a->heads % a->kv_heads == 0 && a->heads <= 65535,
                "attention expects the query heads (%d) to be a multiple of the key heads (%d)", a->heads, a->kv_heads);
  const int64_t most = ((int64_t)1 << 31) - 1024;
  MCCNN_REQUIRE(a->num_q >= 0 && a->num_k >= 0 && a->num_q <= most && a->num_k <= most,
                "attention expects 0 to 2^31 - 1024 queries and keys");
  MCCNN_REQUIRE(a->clouds >= 0 && a->clouds <= (1 << 24), "attention expects 0 to 2^24 clouds, got %d", a->clouds);
  MCCNN_REQUIRE((a->q_splits && a->k_splits) || a->clouds == 1, "attention of %d clouds expects their row splits", a->clouds);
  MCCNN_REQUIRE(a->q || a->num_q == 0, "attention got a null tensor of queries");
  MCCNN_REQUIRE((a->k && a->v) || a->num_k == 0, "attention got a null tensor of keys or values");
  const int64_t strides[6] = {a->q_row, a->q_head, a->k_row, a->k_head, a->v_row, a->v_head};
  for (int64_t s : strides) MCCNN_REQUIRE(s >= 0, "attention expects strides of at least 0");
  MCCNN_REQUIRE(a->scale > 0.0f && a->scale < INFINITY, "attention expects a finite scale above 0");
  MCCNN_REQUIRE(a->axes >= 0 && a->axes <= 3, "a relative bias has 1 to 3 axes, got %d", a->axes);
  if (a->axes > 0) {
    MCCNN_REQUIRE(a->table && a->buckets && a->num_buckets >= 1, "a relative bias expects its table and its buckets");
    MCCNN_REQUIRE(a->max_offset >= 0 && a->max_offset <= kAttnMaxOffsets &&
                      a->axes * (2 * a->max_offset + 1) <= kAttnMaxOffsets,
                  "a relative bias expects at most %d offsets over all axes", kAttnMaxOffsets);
    MCCNN_REQUIRE((a->q_pos == nullptr) == (a->k_pos == nullptr) || a->num_q == 0 || a->num_k == 0,
                  "a relative bias expects positions of the queries and the keys, or neither");
    MCCNN_REQUIRE((a->q_pos && a->k_pos) || a->axes == 1 || a->num_q == 0 || a->num_k == 0,
                  "a relative bias of %d axes expects positions", a->axes);
  }
  b = AttnBatch{a->num_q, a->num_k, a->clouds, a->heads, a->kv_heads, a->dim,
                a->q_splits, a->k_splits, a->k_sizes, a->key_mask, a->q, a->k, a->v,
                a->q_row, a->q_head, a->k_row, a->k_head, a->v_row, a->v_head,
                0, a->causal != 0, a->scale,
                a->axes ? a->table : nullptr, a->axes ? a->buckets : nullptr, a->axes ? a->q_pos : nullptr,
                a->axes ? a->k_pos : nullptr, a->axes, a->axes ? a->num_buckets : 0, a->axes ? a->max_offset : 0, 1};
  const int per16 = a->dtype == MCCNN_FLOAT32 ? 4 : 8;
  bool vec = a->dim % per16 == 0 && aligned16(a->q) && aligned16(a->k) && aligned16(a->v);
  for (int64_t s : strides) vec = vec && s % per16 == 0;
  b.vec = vec;
  return MCCNN_OK;
}

}  // namespace mccnn

using namespace mccnn;

extern "C" size_t mccnn_attention_workspace_bytes(const mccnn_attention *attention_host) {
  AttnBatch b;
  if (attn_batch(attention_host, b) != MCCNN_OK) return 0;
  return forward_plan(b).bytes;
}

extern "C" int mccnn_attention_forward(mccnn_stream_t stream, const mccnn_attention *attention_host, void *workspace,
                                       size_t workspace_bytes, void *out, float *out_low, float *row_max,
                                       float *row_sum) {
  AttnBatch b;
  if (const int rc = attn_batch(attention_host, b)) return rc;
  MCCNN_REQUIRE((row_max == nullptr) == (row_sum == nullptr), "attention writes both row statistics or neither");
  if (b.num_q == 0) return MCCNN_OK;
  MCCNN_REQUIRE(out, "attention got a null output");
  const ForwardPlan p = forward_plan(b);
  MCCNN_REQUIRE(workspace_bytes >= p.bytes && (workspace || p.bytes == 0), "attention workspace too small: %zu < %zu",
                workspace_bytes, p.bytes);
  hipStream_t s = as_stream(stream);
  char *ws = static_cast<char *>(workspace);
  auto launch = [&](auto type, auto dp, auto bias, auto vec) {
    return launch_forward<decltype(type), decltype(dp)::value, decltype(bias)::value, decltype(vec)::value != 0>(
        s, b, p, out, out_low, row_max, row_sum, ws);
  };
  return attention_host->dtype == MCCNN_FLOAT32 ? attn_dispatch_bias<float>(b, launch)
                                                : attn_dispatch_bias<__bf16>(b, launch);
}
