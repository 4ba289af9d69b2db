// tp_tiles.h -- attention over 64-token tiles of keys and values in LDS.
//
// Shared by the prompt kernel (tp_prompt.hip, dense keys) and the drafted-tree
// kernel (tp_tree.hip, decoded pages).  A wave owns 32 query rows; both products
// run on v_mfma_f32_32x32x16 with the rows as columns:
//   S^T[t][r] = sum_d K[t][d] Q[r][d]      (A = keys, B = queries)
//   O^T[d][r] += sum_t V[t][d] P[r][t]     (A = values, B = weights)
// so a lane's column is one query row from end to end: its maximum, sum and
// rescaling are plain registers, and one swap of the wave's halves per tile joins
// the two lanes of a row.  The accumulator of S^T holds tokens
//   32 nb + 8 (i / 4) + 4 h + i % 4   (register i of block nb, half h = lane / 32),
// and the second product takes its sum over tokens in that very order, so the
// weights go from one product to the other without leaving their lane: values are
// read from LDS by the transposing read (4 tokens of one dimension a lane) at the
// same tokens.
//
// Tiles lie in LDS as rows of 256 bytes, 16-byte chunk c of row t at chunk c ^
// tile_swizzle(t), which is another one for each 16 rows in turn (16 lanes read one chunk
// of 16 key rows together) and moves 4 rows in turn by 4 chunks (32 lanes read 4 chunks of
// 4 value rows together), so that both reads hit every bank once.  With 8 chunks in turn
// both took twice the cycles (42 % of the prompt kernel's LDS time was conflicts).
#pragma once

#include "tp_common.h"

namespace tp {

typedef float float16v __attribute__((ext_vector_type(16)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
typedef float float2v __attribute__((ext_vector_type(2)));
typedef short short4v __attribute__((ext_vector_type(4)));
typedef uint32_t uint4v __attribute__((ext_vector_type(4)));
typedef uint32_t uint2v __attribute__((ext_vector_type(2)));

constexpr int kTileTokens = 64;
constexpr int kTileBytes = kTileTokens * kHeadDim * 2;
constexpr int kWaveRows = 32;
constexpr float kLog2e = 1.4426950408889634f;

__host__ __device__ inline int tile_swizzle(int t) { return ((t & 3) << 2) | ((t >> 2) & 3); }
// Byte offset of 16-byte chunk c of token t.
__host__ __device__ inline int tile_at(int t, int c) { return t * (kHeadDim * 2) + ((c ^ tile_swizzle(t)) << 4); }

// Element types: the product and the rounding of a pair of weights (to nearest: each
// is off by at most half a step of itself, so an output's rounding error stays below
// half a step of the type relative to the largest value).
struct F16 {
  static __device__ __forceinline__ float16v mfma(uint4v a, uint4v b, float16v c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(half8v, a), __builtin_bit_cast(half8v, b), c, 0,
                                                  0, 0);
  }
  static __device__ __forceinline__ uint32_t pack(float x, float y) {
    return __builtin_bit_cast(uint32_t, __builtin_convertvector(float2v{x, y}, half2v));
  }
  static constexpr uint32_t kExponent = 0x7c00u;
  // Weights lie 2^kHeadroom higher than the largest being 1 (2^kSlack more at most, 2^15 in all): the smallest
  // that keeps all of its bits is then 2^-21 of the row's largest instead of 2^-14, and what vanishes 2^-32
  // instead of 2^-25 (32,767 keys of weight 2^-26 beside one of 1 are 5e-4 of the result, and were lost).
  static constexpr float kHeadroom = 7.0f;
};
struct BF16 {
  static __device__ __forceinline__ float16v mfma(uint4v a, uint4v b, float16v c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0,
                                                   0, 0);
  }
  static __device__ __forceinline__ uint32_t pack(float x, float y) {
    return __builtin_bit_cast(uint32_t, __builtin_convertvector(float2v{x, y}, bf16x2));
  }
  static constexpr uint32_t kExponent = 0x7f80u;
  static constexpr float kHeadroom = 0.0f;  // fp32's exponents
};

// Whether any of the pair's two 16-bit values is infinite or NaN.
template <class T>
__device__ __forceinline__ bool pair_nonfinite(uint32_t w) {
  return (w & T::kExponent) == T::kExponent || (w & (T::kExponent << 16)) == (T::kExponent << 16);
}
template <class T>
__device__ __forceinline__ uint32_t pair_finite(uint32_t w) {  // those set to 0
  if ((w & T::kExponent) == T::kExponent) w &= 0xffff0000u;
  if ((w & (T::kExponent << 16)) == (T::kExponent << 16)) w &= 0xffffu;
  return w;
}
template <class T>
__device__ __forceinline__ float from_bits(uint16_t b);
template <>
__device__ __forceinline__ float from_bits<F16>(uint16_t b) {
  return h2f(b);
}
template <>
__device__ __forceinline__ float from_bits<BF16>(uint16_t b) {
  return __uint_as_float((uint32_t)b << 16);
}

__device__ __forceinline__ uint4v lds_read16(const char* p) { return *reinterpret_cast<const uint4v*>(p); }

// 4 tokens of one dimension: lane l gets, of the four rows that lanes 4 j + (l % 16) / 4
// of its 16 address, element l % 4.
__device__ __forceinline__ uint2v lds_read_tr(const char* p) {
  typedef __attribute__((address_space(3))) short4v* lds_ptr;
  const short4v r = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_ptr)p);
  return __builtin_bit_cast(uint2v, r);
}

// The two lanes of a row, combined in both.
template <class Op>
__device__ __forceinline__ float across_halves(float x, Op op) {
  const auto p = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  return op(__uint_as_float(p[0]), __uint_as_float(p[1]));
}

struct RowState {
  float16v o[4];  // O^T, dimensions 32 db + 8 (i / 4) + 4 h + i % 4
  float m;        // running maximum of scale * score, in log2 units
  float l;        // this lane's part of the sum of the weights (2^kHeadroom times it, as o)

  __device__ __forceinline__ void clear() {
#pragma unroll
    for (int db = 0; db < 4; ++db)
#pragma unroll
      for (int i = 0; i < 16; ++i) o[db][i] = 0.0f;
    m = -INFINITY;
    l = 0.0f;
  }
};

// A wave's lane offsets into a tile.
struct TileLane {
  int k;  // key row lane % 32, chunk h
  int v;  // value rows of the transposing read, dimension block 0
  __device__ __forceinline__ explicit TileLane(int lane) {
    const int h = lane >> 5;
    k = tile_at(lane & 31, h);
    const int row = 4 * h + ((lane >> 2) & 3);
    v = tile_at(row, 2 * ((lane >> 4) & 1) + ((lane & 3) >> 1)) + 8 * (lane & 1);
  }
};

// The queries of a row as the B operand: q[ks] holds dimensions 16 ks + 8 h .. + 7.  Where the row is not
// a query's, `row` is some other one: the loads are not under a branch, whose join would wait for each of
// them in turn.
__device__ __forceinline__ void load_query(const uint16_t* row, int lane, uint4v* q) {
#pragma unroll
  for (int ks = 0; ks < 8; ++ks) q[ks] = *reinterpret_cast<const uint4v*>(row + 16 * ks + 8 * (lane >> 5));
}
// Negative scales: the queries' signs turned.
__device__ __forceinline__ void flip_query(uint32_t flip, uint4v* q) {
  if (flip)
#pragma unroll
    for (int ks = 0; ks < 8; ++ks) q[ks] ^= flip;
}

// Product reads: 16 bytes of a key row (run i / NB of the dimensions of block i % NB of the tokens), and 16
// tokens of the values (run i / 4 of the tokens of block i % 4 of the dimensions; 8 rows on, the swizzle
// differs by 2 chunks).
template <int NB>
__device__ __forceinline__ uint4v read_key(const char* kt, int t0, const TileLane& at, int i) {
  return lds_read16(kt + (at.k ^ (32 * (i / NB))) + (t0 + 32 * (i % NB)) * (kHeadDim * 2));
}
__device__ __forceinline__ uint4v read_value(const char* vt, int t0, const TileLane& at, int i) {
  const char* row = vt + (t0 + 16 * (i >> 2)) * (kHeadDim * 2);
  const uint2v lo = lds_read_tr(row + (at.v ^ (64 * (i & 3))));
  const uint2v hi = lds_read_tr(row + (at.v ^ (64 * (i & 3) + 32)) + 8 * kHeadDim * 2);
  return uint4v{lo.x, lo.y, hi.x, hi.y};
}

// Products take what was read from LDS kReadAhead products before; the order is held by scheduling barriers
// (left to itself the compiler puts each read right before its product, which then waits for the LDS every
// time).
constexpr int kReadAhead = 4;

// Scores of NB blocks of 32 tokens from token t0 of a tile of keys.  beside(i): what is issued under product i.
template <class T, int NB, class Beside>
__device__ __forceinline__ void score_tile(const char* kt, int t0, const TileLane& at, const uint4v* q, float16v* s,
                                           Beside beside) {
  uint4v k[kReadAhead];
#pragma unroll
  for (int i = 0; i < kReadAhead; ++i) k[i] = read_key<NB>(kt, t0, at, i);
  __builtin_amdgcn_sched_barrier(0);
#pragma unroll
  for (int i = 0; i < 8 * NB; ++i) {
    float16v& sum = s[i % NB];
    if (i < NB)
#pragma unroll
      for (int j = 0; j < 16; ++j) sum[j] = 0.0f;
    sum = T::mfma(k[i % kReadAhead], q[i / NB], sum);
    if (i + kReadAhead < 8 * NB) k[i % kReadAhead] = read_key<NB>(kt, t0, at, i + kReadAhead);
    beside(i);
    __builtin_amdgcn_sched_barrier(0);
  }
}

// Scores of tokens from `limit` on masked; limit counts from the lane's first token of the tile (4 (lane /
// 32)), so that the tokens it is compared with are constants.
template <int NB>
__device__ __forceinline__ void mask_scores(float16v* s, int limit) {
#pragma unroll
  for (int nb = 0; nb < NB; ++nb)
#pragma unroll
    for (int i = 0; i < 16; ++i) s[nb][i] = 32 * nb + 8 * (i >> 2) + (i & 3) < limit ? s[nb][i] : -INFINITY;
}

// The running maximum (of c times the scores, c > 0) moved to hold a tile's scores.  It moves only
// where some row of the wave grew by more than kSlack, so that most tiles need no rescaling: a weight
// is then at most 2^(kHeadroom + kSlack), which neither its 16 bits nor the sums in fp32 mind (their roundings
// are relative).
constexpr float kSlack = 8.0f;
template <int NB>
__device__ __forceinline__ void rescale(const float16v* s, float c, RowState& st) {
  float x = s[0][0];
#pragma unroll
  for (int nb = 0; nb < NB; ++nb)
#pragma unroll
    for (int i = 0; i < 16; ++i) x = fmaxf(x, s[nb][i]);
  const float top = across_halves(x, [](float u, float w) { return fmaxf(u, w); }) * c;
  if (__any(top > st.m + kSlack)) {  // -inf: a row that has seen nothing yet
    const float m = fmaxf(st.m, top);
    const float alpha = __builtin_amdgcn_exp2f(st.m - (m == -INFINITY ? 0.0f : m));
    st.m = m;
    st.l *= alpha;
#pragma unroll
    for (int db = 0; db < 4; ++db)
#pragma unroll
      for (int i = 0; i < 16; ++i) st.o[db][i] *= alpha;
  }
}

// The product of packed weights with NK runs of 16 values from token t0; v holds the first reads.
template <class T, int NK>
__device__ __forceinline__ void add_values(const char* vt, int t0, const TileLane& at, const uint4v* p, uint4v* v,
                                           RowState& st) {
#pragma unroll
  for (int i = 0; i < 4 * NK; ++i) {
    st.o[i & 3] = T::mfma(v[i % kReadAhead], p[i >> 2], st.o[i & 3]);
    if (i + kReadAhead < 4 * NK) v[i % kReadAhead] = read_value(vt, t0, at, i + kReadAhead);
    __builtin_amdgcn_sched_barrier(0);
  }
}

// Weights of a tile's scores, packed as the second product takes them, and their sum.
template <class T, int NB>
__device__ __forceinline__ void weigh(const float16v* s, float c, uint4v* p, RowState& st) {
  const float base = st.m == -INFINITY ? 0.0f : st.m - T::kHeadroom;
#pragma unroll
  for (int i = 0; i < 8 * NB; ++i) {
    const float x = __builtin_amdgcn_exp2f(__builtin_fmaf(s[i >> 3][2 * (i & 7)], c, -base));
    const float y = __builtin_amdgcn_exp2f(__builtin_fmaf(s[i >> 3][2 * (i & 7) + 1], c, -base));
    st.l += x;
    st.l += y;
    p[i >> 2][i & 3] = T::pack(x, y);
    if ((i & 3) == 3) __builtin_amdgcn_sched_barrier(0);  // scores give way to weights four pairs at a time
  }
}

// The rest of a pass over NB blocks of 32 tokens from token t0 of a tile, from its scores on.
template <class T, int NB>
__device__ __forceinline__ void finish_tile(const char* vt, int t0, const TileLane& at, float c, const float16v* s,
                                            RowState& st) {
  rescale<NB>(s, c, st);
  uint4v p[2 * NB], v[kReadAhead];
  // The first values are read under the softmax; of two blocks, whose scores leave no registers, after it.
  if (NB == 1)
#pragma unroll
    for (int i = 0; i < kReadAhead; ++i) v[i] = read_value(vt, t0, at, i);
  weigh<T, NB>(s, c, p, st);
  if (NB != 1)
#pragma unroll
    for (int i = 0; i < kReadAhead; ++i) v[i] = read_value(vt, t0, at, i);
  add_values<T, 2 * NB>(vt, t0, at, p, v, st);
}

// Infinities and NaN among the values of a tile that some rows do not see: a product
// with a weight of 0 would carry them into those rows, so the tile holds 0 in their
// place, and the rows that do see the token take the value itself (a positive weight
// leaves an infinity or NaN what it is).  row(t): the token's values.
template <class T, class Seen, class Row>
__device__ __forceinline__ void add_nonfinite(RowState& st, int lane, int tokens, Seen seen, Row row) {
  for (int t = 0; t < tokens; ++t) {
    if (!seen(t)) continue;
    const uint16_t* v = row(t) + 4 * (lane >> 5);
#pragma unroll
    for (int db = 0; db < 4; ++db)
#pragma unroll
      for (int i = 0; i < 16; ++i) {
        const uint16_t x = v[32 * db + 8 * (i >> 2) + (i & 3)];
        if ((x & T::kExponent) == T::kExponent) st.o[db][i] += from_bits<T>(x);
      }
  }
}

// The row's result, divided by its sum: 16 bytes a store (the halves of a row hold
// every other four dimensions; one swap gives each lane 8 in a row).
template <class T>
__device__ __forceinline__ void store_row(const RowState& st, float inv, uint16_t* row, bool live, int lane) {
#pragma unroll
  for (int db = 0; db < 4; ++db)
#pragma unroll
    for (int a = 0; a < 2; ++a) {
      uint32_t w[4];
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        const uint32_t x = T::pack(st.o[db][8 * a + 2 * j] * inv, st.o[db][8 * a + 2 * j + 1] * inv);
        const uint32_t y = T::pack(st.o[db][8 * a + 4 + 2 * j] * inv, st.o[db][8 * a + 5 + 2 * j] * inv);
        const auto p = __builtin_amdgcn_permlane32_swap(x, y, false, false);
        w[j] = p[0];
        w[2 + j] = p[1];
      }
      if (live)
        *reinterpret_cast<uint4v*>(row + 32 * db + 16 * a + 8 * (lane >> 5)) = uint4v{w[0], w[1], w[2], w[3]};
    }
}

// A split's record of a row: its output divided by its sum, with the maximum (log2 units) and the
// sum in fp32.  Splits of a row are joined by join_splits_kernel.  HALF: the output in fp16 (it lies
// within the values' range), for half the bytes written and read back, where a row has dozens of records:
// each one's rounding (half a step, 2^-11) is weighted by its share, so their sum stays below the result's
// own.
template <bool HALF>
__device__ __forceinline__ void store_record(const RowState& st, float l, void* o, float* ml, bool live, int lane) {
  const float inv = l == 0.0f ? 0.0f : 1.0f / l;
  if constexpr (HALF) {
    store_row<F16>(st, inv, static_cast<uint16_t*>(o), live, lane);
  } else if (live) {
#pragma unroll
    for (int db = 0; db < 4; ++db)
#pragma unroll
      for (int a = 0; a < 4; ++a) {
        const float4v x = {st.o[db][4 * a] * inv, st.o[db][4 * a + 1] * inv, st.o[db][4 * a + 2] * inv,
                           st.o[db][4 * a + 3] * inv};
        *reinterpret_cast<float4v*>(static_cast<float*>(o) + 32 * db + 8 * a + 4 * (lane >> 5)) = x;
      }
  }
  if (live && lane < 32) *reinterpret_cast<float2v*>(ml) = float2v{st.m, l};
}

// Where the splits' records are and where the joined rows go.  Rows are counted as
// (token, head of the group) per unit = (batch, kv head).
struct JoinArgs {
  const void* o;    // [units][rows][splits][128], fp16 or fp32
  const float* ml;  // [units][rows][splits][2]
  uint16_t* out;
  int64_t rows;     // per unit
  int64_t out_b, out_h, out_t;
  int32_t units, splits, g, hkv;
  const int32_t* rest_from;  // tokens from *rest_from on are left as they are (NULL: none)
};

int32_t launch_join(const JoinArgs& a, bool bf16, bool half_records, hipStream_t s);

}  // namespace tp
