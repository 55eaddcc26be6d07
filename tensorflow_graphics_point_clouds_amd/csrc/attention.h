// Attention inside the clouds of a packed batch: what the forward and the gradient kernels share.
//
//   s[i, j]  = scale q_i . k_j + bias[i, j]          over the keys j that query i may look at
//   p[i, j]  = exp(s[i, j] - m_i) / l_i,   m_i = max_j s[i, j],  l_i = sum_j exp(s[i, j] - m_i)
//   o_i      = sum_j p[i, j] v_j                      (0 for a query that nothing is left for)
//   bias     = sum over the axes a of table[a, bucket(clamp(pos_j[a] - pos_i[a], -R, R)), head]
//
// Logits are kept in units of log 2 (scale and biases times 1 / log 2), exponentials are powers of 2.
//
// All products are 32 x 32 x 16 steps of the bf16 matrix pipe with float32 accumulation.  bfloat16
// operands are taken as they are (one part), softmax weights and logit gradients beside them in two or
// three; float32 operands as three bfloat16 parts each, six part products per step (split.h), which
// is as exact as float32 products.
//
// Layout of a 32 x 32 result in registers: lane l holds column l & 31, and its register r row
// 8 (r / 4) + 4 (l >> 5) + r % 4.  Scores are formed with the reduction's other side in the rows
// (forward and query gradients: rows = keys, column = query; key gradients: rows = queries, column
// = key), so that a lane owns one query (key) and the 16 weights in its registers are, eight at a
// time, an operand of the next product without leaving the lane: the order of a product's 16
// summands is free as long as both operands agree on it, and the transposing LDS reads of the
// other operand (operand_t below) are made in that order.
#pragma once
#include "common.h"
#include "mfma.h"
#include "split.h"

namespace mccnn {

constexpr float kLog2e = 1.4426950408889634f;
constexpr int kAttnThreads = 256;
constexpr int kAttnRows = 128;            // query rows (or keys) of a block, 32 per wavefront
constexpr int kAttnMaxDim = 128;
constexpr int kAttnMaxOffsets = MCCNN_ATTENTION_MAX_OFFSETS;   // axes * (2 R + 1): what the LDS has room for

// A packed batch as the kernels see it.  Strides are in elements; the innermost one is 1.
struct AttnBatch {
  int64_t num_q, num_k;
  int clouds, heads, kv_heads, dim;
  const int *q_splits, *k_splits, *k_sizes;   // splits [clouds + 1] (NULL: one cloud), sizes [clouds] or NULL
  const uint8_t *key_mask;                    // [num_k] or NULL
  const void *q, *k, *v;
  int64_t q_row, q_head, k_row, k_head, v_row, v_head;
  int vec;                                    // all rows start at 16 bytes and end at whole vectors
  int causal;
  float scale;
  const float *table;                         // [axes, num_buckets, heads]
  const int *buckets;                         // [2 R + 1]
  const int *q_pos, *k_pos;                   // [num, axes]; NULL: the token's index in its cloud
  int axes, num_buckets, max_offset;
  int pack;                                   // heads that share a block's rows: row = query * pack + head
};

// What a launch with more than the 64 KB of LDS that every kernel may take asks for first.
inline int allow_lds(const void *kernel, size_t bytes) {
  if (bytes > 64 * 1024)
    MCCNN_HIP_CHECK(hipFuncSetAttribute(kernel, hipFuncAttributeMaxDynamicSharedMemorySize, (int)bytes));
  return MCCNN_OK;
}
// The public description, checked and turned into the above (defined in attention.hip).
int attn_batch(const mccnn_attention *a, AttnBatch &b);

// Heads of a group that share a block's rows: with few queries per cloud (a token each, or a pooling
// query) one head alone would fill a fraction of the 128 rows and every head would read the keys
// again; with many, one head per block wants the smallest bias table.  `room`: floats of LDS that
// the tables of the packed heads may take.
inline int attn_pack(const AttnBatch &b, int room) {
  if (b.num_q > 32 * (int64_t)b.clouds) return 1;
  const int group = b.heads / b.kv_heads, per_head = b.axes * (2 * b.max_offset + 1);
  int best = 1;
  for (int p = 2; p <= group && p <= kAttnRows; ++p)
    if (group % p == 0 && p * per_head <= room) best = p;
  return best;
}
// Places for the 128-row pieces of all clouds, and of the rows outside them.
inline int64_t attn_places(int64_t rows, int clouds) { return rows / kAttnRows + clouds + 2; }
// Block id = (place * parts + part) * columns + column: the columns (heads) of a piece go to
// neighbouring XCDs, so that each of the eight L2 sees few heads' keys.
// A grid counts the threads of a dimension in 32 bits: blocks behind the first 2^24 - 1 of 256 take a
// second row of it, whose last ones may lie behind the last place.
constexpr int64_t kAttnRowBlocks = (1 << 24) - 1, kAttnMaxBlocks = ((int64_t)1 << 31) - 1;
inline dim3 attn_grid(int64_t blocks) {
  const int64_t row = blocks < kAttnRowBlocks ? blocks : kAttnRowBlocks;
  return dim3((unsigned)row, (unsigned)((blocks + row - 1) / row));
}
// Parts that a long axis is cut into, none with less than about 256 of its elements.  Blocks of full
// rows are bound by their arithmetic: as many as are at work at a time, two per compute unit, twice as
// many under a causal mask, whose walks differ (13 001 tokens, whose key gradients are 404 blocks: a
// training pass of 1761 us with those in one part, 1391 in two).  Blocks of few rows wait for memory:
// `few`, three per compute unit (one query per cloud over 4 x 200 k keys of 64 bfloat16 channels 256, 145,
// 134, 149 us with 256, 512, 768, 1024 blocks), in a forward pass of up to 32 channels four.
inline int attn_parts(int64_t rows, int clouds, int64_t columns, int64_t axis, bool causal, int few = 768) {
  const int64_t full = rows / kAttnRows, blocks = (full > clouds ? full : clouds) * columns;
  const int64_t want = (full <= clouds ? few : causal ? 1024 : 512) / (blocks > 0 ? blocks : 1);
  const int64_t most = axis / (clouds > 0 ? clouds : 1) / 256, parts = want < most ? want : most;
  return (int)(parts < 1 ? 1 : parts > 256 ? 256 : parts);
}
// The dtype, head size, bias and alignment of a call as template arguments: fn(T(), DP, BIAS, VEC) with
// the last three as integral constants.
template <int N>
struct AttnInt {
  static constexpr int value = N;
};
template <typename T, typename F>
int attn_dispatch_bias(const AttnBatch &b, F &&fn) {
  auto widths = [&](auto bias, auto vec) {
    if (b.dim <= 32) return fn(T(), AttnInt<32>(), bias, vec);
    if (b.dim <= 64) return fn(T(), AttnInt<64>(), bias, vec);
    if (b.dim <= 96) return fn(T(), AttnInt<96>(), bias, vec);
    return fn(T(), AttnInt<128>(), bias, vec);
  };
  auto dims = [&](auto bias) { return b.vec ? widths(bias, AttnInt<1>()) : widths(bias, AttnInt<0>()); };
  if (b.axes == 0) return dims(AttnInt<0>());
  return b.q_pos ? dims(AttnInt<2>()) : dims(AttnInt<1>());
}

// Blocks of a compute unit that the register budget of a kernel is cut for.
template <typename T, int DP>
constexpr int attn_blocks_per_cu() {
  return sizeof(T) == 4 && DP > 64 ? 1 : 2;
}
// The same of the forward pass: with up to 64 bfloat16 channels three blocks fit, all but a few
// registers of a lane with a bias of token offsets (8 x 2000 tokens forward: 130 us with three blocks and
// 3 registers spilled, 138 with two; with positions 28 to 38 of them would spill, and of the query
// gradients' 19, for a training pass of 466 us instead of 447).
template <typename T, int DP, int BIAS>
constexpr int attn_forward_blocks_per_cu() {
  return sizeof(T) == 2 && DP <= 64 && BIAS != 2 ? 3 : attn_blocks_per_cu<T, DP>();
}
// Rows of the tiles that pass through LDS.  (64 rows of 32 float32 channels: 5 x 12 k keys for one
// query each 36 us instead of 28, query gradients with three axes of bias 367 instead of 302.)
template <typename T, int DP>
constexpr int attn_tile_rows() {
  return sizeof(T) == 4 ? 32 : 64;
}

#ifdef __HIPCC__

__device__ __forceinline__ unsigned attn_block() { return blockIdx.y * gridDim.x + blockIdx.x; }

typedef short v4s __attribute__((ext_vector_type(4)));
typedef short v8s __attribute__((ext_vector_type(8)));
typedef unsigned v4u __attribute__((ext_vector_type(4)));

template <int NP>
struct Frag {
  v8bf p[NP];
};

template <int NP>
__device__ __forceinline__ v16f mma(const Frag<NP> &a, const Frag<NP> &b, v16f acc) {
  if constexpr (NP == 1) {
    return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a.p[0], b.p[0], acc, 0, 0, 0);
  } else {
    return mma_split(Split8{a.p[0], a.p[1], a.p[2]}, Split8{b.p[0], b.p[1], b.p[2]}, acc);
  }
}

__device__ __forceinline__ float exp2_fast(float x) { return __builtin_amdgcn_exp2f(x); }

// Eight consecutive values of a row as they come from memory.
template <typename T>
struct Row8;
template <>
struct Row8<__bf16> {
  v4u w;
};
template <>
struct Row8<float> {
  v4f lo, hi;
};

// Values col .. col + 7 of a row of `dim` values.  VEC (rows start at 16 bytes and end at whole
// vectors): loads without a branch, from the row's begin where it has no such values, which
// clip8 makes zeros once they have arrived.  Otherwise value by value, zeros behind the last.
template <bool VEC, typename T>
__device__ __forceinline__ Row8<T> load8(const T *__restrict__ row, int col, int dim) {
  Row8<T> r;
  if constexpr (VEC && sizeof(T) == 2) {
    r.w = *reinterpret_cast<const v4u *>(row + (col < dim ? col : 0));
  } else if constexpr (VEC) {
    r.lo = *reinterpret_cast<const v4f *>(row + (col < dim ? col : 0));
    r.hi = *reinterpret_cast<const v4f *>(row + (col + 4 < dim ? col + 4 : 0));
  } else if constexpr (sizeof(T) == 2) {
    const unsigned short *u = reinterpret_cast<const unsigned short *>(row);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      unsigned w = 0;
      if (col + 2 * i < dim) w = u[col + 2 * i];
      if (col + 2 * i + 1 < dim) w |= (unsigned)u[col + 2 * i + 1] << 16;
      r.w[i] = w;
    }
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      r.lo[i] = col + i < dim ? row[col + i] : 0.0f;
      r.hi[i] = col + 4 + i < dim ? row[col + 4 + i] : 0.0f;
    }
  }
  return r;
}
template <bool VEC>
__device__ __forceinline__ Row8<__bf16> clip8(const Row8<__bf16> &r, int col, int dim, bool in) {
  const bool keep = in && (!VEC || col < dim);
  return Row8<__bf16>{v4u{keep ? r.w[0] : 0, keep ? r.w[1] : 0, keep ? r.w[2] : 0, keep ? r.w[3] : 0}};
}
template <bool VEC>
__device__ __forceinline__ Row8<float> clip8(const Row8<float> &r, int col, int dim, bool in) {
  const bool a = in && (!VEC || col < dim), b = in && (!VEC || col + 4 < dim);
  return Row8<float>{v4f{a ? r.lo[0] : 0.0f, a ? r.lo[1] : 0.0f, a ? r.lo[2] : 0.0f, a ? r.lo[3] : 0.0f},
                     v4f{b ? r.hi[0] : 0.0f, b ? r.hi[1] : 0.0f, b ? r.hi[2] : 0.0f, b ? r.hi[3] : 0.0f}};
}
// Both at once, for what is loaded once.
template <bool VEC, typename T>
__device__ __forceinline__ Row8<T> row8(const T *__restrict__ row, int col, int dim, bool in) {
  return clip8<VEC>(load8<VEC>(row, col, dim), col, dim, in);
}

__device__ __forceinline__ Frag<1> to_frag(const Row8<__bf16> &r) {
  return Frag<1>{{__builtin_bit_cast(v8bf, r.w)}};
}
__device__ __forceinline__ Frag<3> to_frag(const Row8<float> &r) {
  const Split8 s = split8(r.lo, r.hi);
  return Frag<3>{{s.p[0], s.p[1], s.p[2]}};
}

__device__ __forceinline__ v2f widen_pair(const Frag<1> &f, int e) {
  const v4u u = __builtin_bit_cast(v4u, f.p[0]);
  const unsigned pair = u[e];             // (a bit cast of u[e] itself takes element 0 every time)
  return widen2(__builtin_bit_cast(v2bf, pair));
}
// What the rounding to one part has left of registers 8 t .. 8 t + 7, as an operand.
__device__ __forceinline__ Frag<1> rest_frag(const v16f &s, int t, const Frag<1> &rounded) {
  unsigned w[4];
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    const v2f x = v2f{s[8 * t + 2 * e], s[8 * t + 2 * e + 1]} - widen_pair(rounded, e);
    w[e] = __builtin_bit_cast(unsigned, __builtin_convertvector(x, v2bf));
  }
  return Frag<1>{{__builtin_bit_cast(v8bf, v4u{w[0], w[1], w[2], w[3]})}};
}

// Registers 8 t .. 8 t + 7 of a result as an operand.  One part: weights and logit gradients are
// rounded to bfloat16 here, 2^-8 of each, and rest_frag has what that took from them for a
// product of its own; their sums and everything that the statistics are made of stay in float32.
template <int NP>
__device__ __forceinline__ Frag<NP> result_frag(const v16f &s, int t) {
  const v4f lo = {s[8 * t], s[8 * t + 1], s[8 * t + 2], s[8 * t + 3]};
  const v4f hi = {s[8 * t + 4], s[8 * t + 5], s[8 * t + 6], s[8 * t + 7]};
  if constexpr (NP == 3) {
    return to_frag(Row8<float>{lo, hi});
  } else {
    unsigned w[4];
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const v2f x = e < 2 ? v2f{lo[2 * e], lo[2 * e + 1]} : v2f{hi[2 * e - 4], hi[2 * e - 3]};
      w[e] = __builtin_bit_cast(unsigned, __builtin_convertvector(x, v2bf));
    }
    return Frag<1>{{__builtin_bit_cast(v8bf, v4u{w[0], w[1], w[2], w[3]})}};
  }
}

// Registers 8 t .. 8 t + 7 of softmax weights as P operands, the leading bits, the following ones and at
// last the rounded rest: 2^-15 of a weight is left out of two, nothing of three.  All parts are above 0
// (2^-126 at least where nothing is left; cut off, not rounded, so that no rest is negative): a value of
// infinity, which each of them multiplies, then stays one.
template <int P>
__device__ __forceinline__ void weight_parts(const v16f &s, int t, Frag<1> *parts) {
  typedef unsigned short v2us __attribute__((ext_vector_type(2)));
  constexpr unsigned kTop = 0xffff0000u;
  unsigned w[P][4];
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    float a = s[8 * t + 2 * e], b = s[8 * t + 2 * e + 1];
#pragma unroll
    for (int q = 0; q < P; ++q) {
      unsigned u;
      if (q + 1 < P) {
        u = __builtin_amdgcn_perm(__float_as_uint(b), __float_as_uint(a), 0x07060302u);   // both upper halves
        a -= __uint_as_float(__float_as_uint(a) & kTop);
        b -= __uint_as_float(__float_as_uint(b) & kTop);
      } else {
        u = __builtin_bit_cast(unsigned, __builtin_convertvector(v2f{a, b}, v2bf));
      }
      if (q > 0) u = __builtin_bit_cast(unsigned, __builtin_elementwise_max(__builtin_bit_cast(v2us, u), v2us{0x80, 0x80}));
      w[q][e] = u;
    }
  }
#pragma unroll
  for (int q = 0; q < P; ++q) parts[q] = Frag<1>{{__builtin_bit_cast(v8bf, v4u{w[q][0], w[q][1], w[q][2], w[q][3]})}};
}

// The sum of the products of eight values with eight others, in float32.
__device__ __forceinline__ float dot8(const Row8<float> &a, const Row8<float> &b) {
  float s = 0.0f;
#pragma unroll
  for (int i = 0; i < 4; ++i) s += a.lo[i] * b.lo[i];
#pragma unroll
  for (int i = 0; i < 4; ++i) s += a.hi[i] * b.hi[i];
  return s;
}
__device__ __forceinline__ float dot8(const Row8<__bf16> &a, const Row8<__bf16> &b) {
  float s = 0.0f;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    s += __uint_as_float(a.w[i] << 16) * __uint_as_float(b.w[i] << 16);
    s += __uint_as_float(a.w[i] & 0xffff0000u) * __uint_as_float(b.w[i] & 0xffff0000u);
  }
  return s;
}

__device__ __forceinline__ float dot8(const Row8<__bf16> &a, const Row8<float> &b) {
  float s = 0.0f;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    s += __uint_as_float(a.w[i] << 16) * (i < 2 ? b.lo[2 * i] : b.hi[2 * i - 4]);
    s += __uint_as_float(a.w[i] & 0xffff0000u) * (i < 2 ? b.lo[2 * i + 1] : b.hi[2 * i - 3]);
  }
  return s;
}

// A tile of rows in LDS: [part][row][DP + 16] bfloat16.  The rows of eight lanes then begin at the
// eight multiples of eight banks, for all widths, and neither the reads of 16 bytes per row nor
// the transposing ones of eight rows by 64 bytes meet in a bank (with DP + 8 the latter did, twice over).
template <int NP, int DP, int ROWS>
struct Tile {
  static constexpr int kStride = DP + 16;
  static constexpr int kPlane = ROWS * kStride;
  static constexpr int kElems = NP * kPlane;

  static __device__ __forceinline__ void store(__bf16 *base, int row, int col, const Frag<NP> &f) {
#pragma unroll
    for (int q = 0; q < NP; ++q)
      *reinterpret_cast<v8bf *>(base + q * kPlane + row * kStride + col) = f.p[q];
  }
  // Operand with a tile row per lane: values 16 step + 8 (lane >> 5) .. + 7 of row row0 + (lane & 31).
  static __device__ __forceinline__ Frag<NP> operand(const __bf16 *base, int row0, int step) {
    const int lane = lane_id();
    const __bf16 *p = base + (row0 + (lane & 31)) * kStride + 16 * step + 8 * (lane >> 5);
    Frag<NP> f;
#pragma unroll
    for (int q = 0; q < NP; ++q) f.p[q] = *reinterpret_cast<const v8bf *>(p + q * kPlane);
    return f;
  }
  // Operand with a tile column per lane (column 32 dt + (lane & 31)) over the rows row0 .. row0 + 15,
  // in the order of a result's registers: rows 4 h .. 4 h + 3, then 8 + 4 h .. 11 + 4 h, h = lane >> 5.
  // Each read hands a lane four rows of its column out of a 4 x 16 block that sixteen lanes point at.
  static __device__ __forceinline__ Frag<NP> operand_t(const __bf16 *base, int row0, int dt) {
    const int lane = lane_id();
    const __bf16 *p = base + (row0 + 4 * (lane >> 5) + ((lane & 15) >> 2)) * kStride + 32 * dt +
                      16 * ((lane >> 4) & 1) + 4 * (lane & 3);
    Frag<NP> f;
#pragma unroll
    for (int q = 0; q < NP; ++q) {
      typedef __attribute__((address_space(3))) v4s *lds;
      const v4s a = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds)(p + q * kPlane));
      const v4s b = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds)(p + q * kPlane + 8 * kStride));
      f.p[q] = __builtin_bit_cast(v8bf, __builtin_shufflevector(a, b, 0, 1, 2, 3, 4, 5, 6, 7));
    }
    return f;
  }
};

// Row of a result's register r in lane half h.
__device__ __forceinline__ constexpr int result_row(int r) { return 8 * (r / 4) + r % 4; }

__device__ __forceinline__ float other_half(float v) { return __shfl_xor(v, 32, kWave); }

// First row of cloud c - 1 of a table of n rows; c = 0 and c = clouds + 1 are what lies before the
// first and behind the last cloud.  Whatever the splits hold, the answer is in [0, n].
__device__ __forceinline__ int64_t cloud_start(const int *__restrict__ splits, int clouds, int64_t n, int c) {
  if (c <= 0) return 0;
  if (c > clouds + 1) return n;
  const int64_t s = splits ? (int64_t)splits[c - 1] : (c == 1 ? 0 : n);
  return s < 0 ? 0 : s > n ? n : s;
}

// What a block works on: 128 rows (of its own side) of cloud c - 1 and what they meet.
struct CloudWork {
  int64_t q_start, k_start;        // first query and key of the cloud
  int num_q, used, capacity;       // its queries, the rows that hold a key, the rows of its key table
  int64_t first;                   // first of the block's rows, among the cloud's
};
__device__ __forceinline__ int uniform(int v) { return __builtin_amdgcn_readfirstlane(v); }
__device__ __forceinline__ int64_t uniform(int64_t v) {
  return ((int64_t)uniform((int)(v >> 32)) << 32) | (unsigned)uniform((int)v);
}
__device__ __forceinline__ int from_lane(int v, int lane) { return __builtin_amdgcn_readlane(v, lane); }

// Queries and keys of cloud c - 1; rows outside every cloud (c = 0, clouds + 1) meet nothing.
__device__ __forceinline__ void cloud_rows(const AttnBatch &b, int c, CloudWork &w) {
  w.q_start = cloud_start(b.q_splits, b.clouds, b.num_q, c);
  w.k_start = cloud_start(b.k_splits, b.clouds, b.num_k, c);
  const int64_t q_end = cloud_start(b.q_splits, b.clouds, b.num_q, c + 1);
  const int64_t k_end = cloud_start(b.k_splits, b.clouds, b.num_k, c + 1);
  w.num_q = (int)(q_end > w.q_start ? q_end - w.q_start : 0);
  w.capacity = (int)(k_end > w.k_start ? k_end - w.k_start : 0);
  w.used = w.capacity;
  const bool cloud = c >= 1 && c <= b.clouds;
  if (b.k_sizes && cloud) {
    const int size = b.k_sizes[c - 1];
    w.used = size < 0 ? 0 : size < w.capacity ? size : w.capacity;
  }
  if (!cloud) w.used = 0;
}

// The work of place t of a grid that has at least one place per 128 rows of every cloud, queries (times
// the heads that share a block) or, BY_KEYS, keys.  False: a place behind the last one.
//
// Up to 62 clouds are looked at by a lane each: the clouds whose blocks have the longest walks take the
// first places, no place between two clouds is empty, and with `reverse` a cloud's last rows come
// first (under a causal mask they have most to do).  (512 blocks of 16 x 1024 points with an empty
// place after every cloud left some compute units a third block: 156 us instead of 100.)  More clouds
// take places start / 128 + c, some of them empty, by a search over 64 of them at a time.
template <bool BY_KEYS>
__device__ __forceinline__ bool find_work(const AttnBatch &b, int t, bool reverse, CloudWork &w) {
  const int lane = lane_id(), n = b.clouds + 2;
  if (n <= kWave) {
    CloudWork mine{};
    if (lane < n) cloud_rows(b, lane, mine);
    const int64_t rows = BY_KEYS ? mine.capacity : (int64_t)mine.num_q * b.pack;
    const int tiles = (int)((rows + kAttnRows - 1) / kAttnRows), weight = BY_KEYS ? mine.num_q : mine.used;
    int before = 0;
    for (int c = 0; c < n; ++c) {
      const int other = from_lane(weight, c), theirs = from_lane(tiles, c);
      before += other > weight || (other == weight && c < lane) ? theirs : 0;
    }
    const uint64_t hit = __ballot(lane < n && t >= before && t < before + tiles);
    if (!hit) return false;
    const int src = __ffsll((unsigned long long)hit) - 1;
    auto wide = [&](int64_t v) {
      return ((int64_t)from_lane((int)(v >> 32), src) << 32) | (unsigned)from_lane((int)v, src);
    };
    w.q_start = wide(mine.q_start);
    w.k_start = wide(mine.k_start);
    w.num_q = from_lane(mine.num_q, src);
    w.used = from_lane(mine.used, src);
    w.capacity = from_lane(mine.capacity, src);
    const int local = t - from_lane(before, src);
    w.first = (int64_t)(reverse ? from_lane(tiles, src) - 1 - local : local) * kAttnRows;
    return true;
  }
  const int *splits = BY_KEYS ? b.k_splits : b.q_splits;
  const int64_t num = BY_KEYS ? b.num_k : b.num_q, pack = BY_KEYS ? 1 : b.pack;
  int lo = 0, count = n;
  while (count > 1) {
    const int step = (count + kWave - 1) / kWave, c = lo + lane * step;
    const bool below = lane * step < count && cloud_start(splits, b.clouds, num, c) * pack / kAttnRows + c <= t;
    const int k = __popcll(__ballot(below)), skip = (k > 1 ? k - 1 : 0) * step;
    lo += skip;
    count = count - skip < step ? count - skip : step;
  }
  const int c = uniform(lo);
  cloud_rows(b, c, w);
  w.q_start = uniform(w.q_start);
  w.k_start = uniform(w.k_start);
  w.num_q = uniform(w.num_q);
  w.used = uniform(w.used);
  w.capacity = uniform(w.capacity);
  const int64_t start = BY_KEYS ? w.k_start : w.q_start, rows = BY_KEYS ? w.capacity : (int64_t)w.num_q * pack;
  w.first = (t - (start * pack / kAttnRows + c)) * kAttnRows;
  return w.first >= 0 && w.first < rows;
}

// A bias in units of log 2.  Masks are written as the type's lowest value, which has none: everything
// below -6.9e37 becomes -1e38, three of which still add up to a finite logit, so that a row with
// nothing but such entries is the mean of its values, as it is in natural units; the largest values
// likewise.  Infinities and NaN stay.
__device__ __forceinline__ float log2_units(float bias) {
  const float x = bias * kLog2e;
  if (bias == INFINITY || bias == -INFINITY) return bias;
  return x > 1.0e38f ? 1.0e38f : x < -1.0e38f ? -1.0e38f : x;
}

// table[a, bucket(o - R), head0 + g] in units of log 2 for all offsets o, as [g][a][2 R + 1] in LDS.
__device__ __forceinline__ void load_bias_table(const AttnBatch &b, int head0, int pack, float *lds) {
  const int width = 2 * b.max_offset + 1, per_head = b.axes * width;
  for (int i = threadIdx.x; i < pack * per_head; i += kAttnThreads) {
    const int g = i / per_head, a = (i / width) % b.axes, o = i % width;
    const int bucket = b.buckets[o];
    const bool known = bucket >= 0 && bucket < b.num_buckets;   // (others: no bias)
    lds[i] = known ? log2_units(b.table[((int64_t)a * b.num_buckets + bucket) * b.heads + head0 + g]) : 0.0f;
  }
}

// An offset as a row of that table has it, counted from the row's middle (offset 0).
__device__ __forceinline__ int clamped_offset(int key_pos, int query_pos, int max_offset) {
  const int d = __builtin_elementwise_sub_sat(key_pos, query_pos);
  int clamped;                            // (one instruction; a minimum and a maximum are two)
  asm("v_med3_i32 %0, %1, %2, %3" : "=v"(clamped) : "v"(d), "v"(-max_offset), "v"(max_offset));
  return clamped;
}

// What passes a tile of KT keys and values from memory through registers to LDS: the rows of one cloud
// and key head from `start` on, up to `end`.  Masked rows are fetched along with the others (the
// mask arrives at the same time, not before) and zeroed on their way, whatever they hold.
template <typename T, int DP, int KT, int BIAS, bool VEC>
struct KeyStage {
  static constexpr int NP = sizeof(T) == 4 ? 3 : 1;
  using KTile = Tile<NP, DP, KT>;
  static constexpr int kChunks = KT * (DP / 8);
  static constexpr int CH = (kChunks + kAttnThreads - 1) / kAttnThreads;
  static constexpr int kElems = KTile::kElems;

  const T *k, *v;
  const uint8_t *mask;                    // without one: any byte that there is, `bare` set
  const int *pos;
  int64_t k_row, v_row;
  int end, dim, axes, mask_step;
  bool bare;
  Row8<T> kr[CH], vr[CH];
  uint8_t seen[CH], seen_key;             // mask values of the chunks' rows, of key `lane` of the tile
  int p[3];
  bool in_key;                            // whether the tile has a key `lane`

  __device__ __forceinline__ KeyStage(const AttnBatch &b, int64_t start, int end_, int kv_head)
      : k(static_cast<const T *>(b.k) + start * b.k_row + kv_head * b.k_head),
        v(static_cast<const T *>(b.v) + start * b.v_row + kv_head * b.v_head),
        mask(b.key_mask ? b.key_mask + start : reinterpret_cast<const uint8_t *>(k)), pos(BIAS == 2 ? b.k_pos + start * b.axes : nullptr),
        k_row(b.k_row), v_row(b.v_row), end(end_), dim(b.dim), axes(b.axes),
        mask_step(b.key_mask ? 1 : 0), bare(!b.key_mask) {}

  __device__ __forceinline__ void fetch(int tile) {
#pragma unroll
    for (int c = 0; c < CH; ++c) {
      const int chunk = c * kAttnThreads + threadIdx.x;
      const int key = tile * KT + chunk / (DP / 8), col = 8 * (chunk % (DP / 8));
      const int64_t r = key < end ? key : 0;
      kr[c] = load8<VEC>(k + r * k_row, col, dim);
      vr[c] = load8<VEC>(v + r * v_row, col, dim);
      seen[c] = mask[r * mask_step];
    }
    const int lane = lane_id(), key = tile * KT + lane;
    const bool in = lane < KT && key < end;
    in_key = in;
    seen_key = mask[in ? (int64_t)key * mask_step : 0];
    if constexpr (BIAS == 2) {
#pragma unroll
      for (int a = 0; a < 3; ++a) p[a] = in && a < axes && threadIdx.x < KT ? pos[(int64_t)key * axes + a] : 0;
    }
  }
  __device__ __forceinline__ uint64_t allowed() const { return __ballot(in_key && (bare || seen_key)); }
  __device__ __forceinline__ void park(int tile, __bf16 *kt, __bf16 *vt, int *kpos) {
#pragma unroll
    for (int c = 0; c < CH; ++c) {
      const int chunk = c * kAttnThreads + threadIdx.x;
      if (kChunks % kAttnThreads != 0 && chunk >= kChunks) break;
      const int key = chunk / (DP / 8), col = 8 * (chunk % (DP / 8));
      const bool in = tile * KT + key < end && (bare || seen[c]);
      KTile::store(kt, key, col, to_frag(clip8<VEC>(kr[c], col, dim, in)));
      KTile::store(vt, key, col, to_frag(clip8<VEC>(vr[c], col, dim, in)));
    }
    if constexpr (BIAS == 2) {
      if (threadIdx.x < KT)
#pragma unroll
        for (int a = 0; a < 3; ++a)
          if (a < axes) kpos[a * KT + threadIdx.x] = p[a];
    }
  }
};

// Four consecutive values of a row to memory: `whole` rows have lengths of whole fours.
template <typename T>
__device__ __forceinline__ void store4(T *__restrict__ row, int col, int dim, bool whole, const float *v) {
  if (whole) {
    if (col >= dim) return;
    if constexpr (sizeof(T) == 4) {
      *reinterpret_cast<v4f *>(row + col) = v4f{v[0], v[1], v[2], v[3]};
    } else {
      const unsigned a = __builtin_bit_cast(unsigned, __builtin_convertvector(v2f{v[0], v[1]}, v2bf));
      const unsigned c = __builtin_bit_cast(unsigned, __builtin_convertvector(v2f{v[2], v[3]}, v2bf));
      *reinterpret_cast<uint2 *>(row + col) = uint2{a, c};
    }
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i)
      if (col + i < dim) row[col + i] = (T)v[i];
  }
}

// Offsets between the 32 keys and the 32 rows of a wavefront where positions are the tokens' places:
// a 32 x 32 block mostly lies on one side of the band -R .. R as a whole.
enum Band { kBelow, kAbove, kInside, kAcross };
__device__ __forceinline__ Band token_band(int key_first, int key_last, int query_first, int query_last,
                                           int max_offset) {
  if (key_last - query_first <= -max_offset) return kBelow;
  if (key_first - query_last >= max_offset) return kAbove;
  return key_first - query_last >= -max_offset && key_last - query_first <= max_offset ? kInside : kAcross;
}
// Biases of a lane's 16 registers, offset + SIGN * result_row(r) each, from a row of the table in LDS.
template <int SIGN>
__device__ __forceinline__ void token_biases(const float *table, int max_offset, Band band, int offset, float *bias) {
  if (band == kBelow || band == kAbove) {
    const float v = table[band == kBelow ? 0 : 2 * max_offset];
#pragma unroll
    for (int r = 0; r < 16; ++r) bias[r] = v;
  } else if (band == kInside) {
    const float *t = table + max_offset + offset;
#pragma unroll
    for (int r = 0; r < 16; ++r) bias[r] = t[SIGN * result_row(r)];
  } else {
#pragma unroll
    for (int r = 0; r < 16; ++r) bias[r] = table[max_offset + clamped_offset(offset + SIGN * result_row(r), 0, max_offset)];
  }
}

// Clamped offsets of an axis for a lane's 16 registers: `rows` points at the positions (in LDS)
// of register 0's row, `own` is the lane's; SIGN is 1 where the rows are keys.
template <int SIGN>
__device__ __forceinline__ void position_offsets(const int *rows, int own, int max_offset, int *offset) {
#pragma unroll
  for (int r = 0; r < 16; ++r) {
    const int other = rows[result_row(r)];
    offset[r] = SIGN > 0 ? clamped_offset(other, own, max_offset) : clamped_offset(own, other, max_offset);
  }
}
// bias[r] = sum over the axes; the axes' positions lie `pitch` apart.
template <int SIGN>
__device__ __forceinline__ void position_biases(const float *table, int axes, int max_offset, const int *rows,
                                                int pitch, const int *own, float *bias) {
#pragma unroll
  for (int a = 0; a < 3; ++a)
    if (a < axes) {
      int offset[16];
      position_offsets<SIGN>(rows + a * pitch, own[a], max_offset, offset);
      const float *t = table + a * (2 * max_offset + 1) + max_offset;
#pragma unroll
      for (int r = 0; r < 16; ++r) bias[r] = a == 0 ? t[offset[r]] : bias[r] + t[offset[r]];
    }
}

#endif  // __HIPCC__
}  // namespace mccnn
