// tp_page_tiles.h -- stored pages decoded into tiles of keys and values in LDS.
//
// Shared by the drafted-tree kernel (tp_tree.hip) and the shared-prefix kernel (tp_shared.hip): a
// workgroup reads a page's codes into registers (the next page's while it works on this one), decodes
// them in pieces into fp16 tiles and multiplies from those.  `Pages` is any struct with the fields of
// a page store: radii, radii_scales, angle_l1, angle_deep, v_codes, v_scales, l1_bits, deep_bits,
// split_half, l1_row, deep_row.
#pragma once

#include "tp_codes.h"
#include "tp_tiles.h"

namespace tp {

enum TreeKind { kTreeDefault = 0, kTreeFast = 1, kTreeAnyF16 = 2, kTreeAnyI8 = 3 };
constexpr bool tree_i8(int kind) { return kind == kTreeFast || kind == kTreeAnyI8; }
constexpr bool tree_any(int kind) { return kind == kTreeAnyF16 || kind == kTreeAnyI8; }

// The codes of one thread's part of a page: N runs of 8 pairs (16 dimensions) of a token,
// threads 8 to a token.
template <int KIND, int N>
struct PageRegs {
  uint4v r[tree_i8(KIND) ? 1 : N];  // fp16 radii
  uint2v r8[tree_i8(KIND) ? N : 1];
  uint2v c8[KIND == kTreeFast ? N : 1];
  uint32_t c4[KIND == kTreeDefault ? N : 1];
  uint32_t rows[tree_any(KIND) ? 2 * N : 1];  // dwords of the page's code rows, tid + threads i of them
  uint4v v[N];
  uint32_t vs[N];  // fp16 scale of the run's group
  uint32_t ls;     // fp16 page scale
};

template <int KIND, int N, int THREADS, class Pages>
__device__ __forceinline__ void load_page(const Pages& a, int64_t slot, int tid, PageRegs<KIND, N>& p) {
  const int c = tid & 7;
#pragma unroll
  for (int n = 0; n < N; ++n) {
    const int64_t row = slot * kPageTokens + (tid >> 3) + (THREADS / 8) * n;
    if constexpr (tree_i8(KIND))
      p.r8[n] = *reinterpret_cast<const uint2v*>(static_cast<const int8_t*>(a.radii) + row * kPairs + 8 * c);
    else
      p.r[n] = *reinterpret_cast<const uint4v*>(static_cast<const uint16_t*>(a.radii) + row * kPairs + 8 * c);
    if constexpr (KIND == kTreeFast)
      p.c8[n] = *reinterpret_cast<const uint2v*>(a.angle_deep + row * kPairs + 8 * c);
    else if constexpr (KIND == kTreeDefault)
      p.c4[n] = *reinterpret_cast<const uint32_t*>((c < 4 ? a.angle_l1 : a.angle_deep) + row * 16 + 4 * (c & 3));
    p.v[n] = *reinterpret_cast<const uint4v*>(a.v_codes + row * kHeadDim + 16 * c);
    p.vs[n] = a.v_scales[row * kVGroups + (c >> 1)];
  }
  if constexpr (tree_i8(KIND)) p.ls = a.radii_scales[slot];
  if constexpr (tree_any(KIND)) {  // at most 64 bytes of codes a token: 1,024 dwords, the level-1 rows first
    const int l1 = kPageTokens / 4 * a.l1_row, all = l1 + kPageTokens / 4 * a.deep_row;
    const uint32_t* l1_rows = reinterpret_cast<const uint32_t*>(a.angle_l1 + slot * kPageTokens * a.l1_row);
    const uint32_t* deep_rows = reinterpret_cast<const uint32_t*>(a.angle_deep + slot * kPageTokens * a.deep_row);
#pragma unroll
    for (int i = 0; i < 2 * N; ++i) {
      const int x = min(tid + THREADS * i, all - 1);  // threads past the last dword reread it
      p.rows[i] = *(x < l1 ? l1_rows + x : deep_rows + (x - l1));
    }
  }
}

template <int KIND, int N, int THREADS>
__device__ __forceinline__ void stage_rows(int tid, const PageRegs<KIND, N>& p, uint32_t* codes) {
  if constexpr (tree_any(KIND))
#pragma unroll
    for (int i = 0; i < 2 * N; ++i) codes[tid + THREADS * i] = p.rows[i];
}

// (cos, sin) in fp32 of the level-1 codes, then of the deep codes (the default layout's codes are of one width: the
// first 16).
struct TreeLut {
  float2v code[512];
};

// Of a code's decoded angle, the reference's (code_angle); an infinite radius meets no zero, as make_cs explains.
__device__ __forceinline__ float2v angle_pair(uint32_t code, int bits) {
  const float th = code_angle(code, bits);
  return float2v{cosf(th), sinf(th)};
}

// A pair's key, r (cos a, sin a), each rounded once.
__device__ __forceinline__ uint32_t key_pair(float r, float2v cs) { return F16::pack(r * cs.x, r * cs.y); }

// Of pair i of half h of run n: its code's place in the table, and its radius.  c is the thread's column, tid & 7.
template <int KIND, int N, class Pages>
__device__ __forceinline__ uint32_t pair_code(const Pages& a, const uint32_t* codes, const PageRegs<KIND, N>& p, int n,
                                              int h, int i, int c, int t) {
  if constexpr (KIND == kTreeDefault) {
    return (p.c4[n] >> (16 * h + 4 * i)) & 15u;
  } else if constexpr (KIND == kTreeFast) {
    return 256 + ((p.c8[n][h] >> (8 * i)) & 0xffu);
  } else {
    const int pair = 8 * c + 4 * h + i;
    const bool l1 = pair < a.split_half;
    const int bits = l1 ? a.l1_bits : a.deep_bits;
    const int bit = (l1 ? pair : pair - a.split_half) * bits;
    const int row = l1 ? t * a.l1_row : kPageTokens * a.l1_row + t * a.deep_row;
    const uint32_t byte = reinterpret_cast<const uint8_t*>(codes)[row + (bit >> 3)];
    return (l1 ? 0u : 256u) + ((byte >> (bit & 7)) & ((1u << bits) - 1u));
  }
}
template <int KIND, int N>
__device__ __forceinline__ float pair_radius(const PageRegs<KIND, N>& p, int n, int h, int i, float ls) {
  if constexpr (tree_i8(KIND))
    return __builtin_amdgcn_exp2f((float)(int)(int8_t)(p.r8[n][h] >> (8 * i)) * ls);
  else
    return h2f((uint16_t)(p.r[n][2 * h + (i >> 1)] >> (16 * (i & 1))));
}

// Half h of run n, 4 pairs: their codes' (cos, sin) out of the table, and the keys, 16 bytes, into a tile.  Between
// the two other work may go on, so that it does not wait for the table.
template <int KIND, int N, int THREADS, class Pages>
__device__ __forceinline__ void fetch_angles(const Pages& a, const TreeLut& lut, const uint32_t* codes, int tid,
                                             const PageRegs<KIND, N>& p, int n, int h, float2v* cs) {
  const int c = tid & 7, t = (tid >> 3) + (THREADS / 8) * n;
  int c0 = c;  // where a pair's code lies is computed anew: kept over the pages, it costs 30 registers
  if constexpr (tree_any(KIND)) asm volatile("" : "+v"(c0));
#pragma unroll
  for (int i = 0; i < 4; ++i) cs[i] = lut.code[pair_code<KIND, N>(a, codes, p, n, h, i, c0, t)];
}

template <int KIND, int N, int THREADS>
__device__ __forceinline__ void store_keys(int tid, const PageRegs<KIND, N>& p, int n, int h, const float2v* cs,
                                           char* kt) {
  const int c = tid & 7, t = (tid >> 3) + (THREADS / 8) * n;
  const float ls = tree_i8(KIND) ? h2f((uint16_t)p.ls) * kLog2e : 0.0f;  // rounded in fp32, as its products below
  uint32_t e[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) e[i] = key_pair(pair_radius<KIND, N>(p, n, h, i, ls), cs[i]);
  *reinterpret_cast<uint4v*>(kt + tile_at(t, 2 * c + h)) = uint4v{e[0], e[1], e[2], e[3]};
}

template <int KIND, int N, int THREADS, class Pages>
__device__ __forceinline__ void decode_keys(const Pages& a, const TreeLut& lut, const uint32_t* codes, int tid,
                                            const PageRegs<KIND, N>& p, int n, int h, char* kt) {
  const int c = tid & 7, t = (tid >> 3) + (THREADS / 8) * n;
  int c0 = c;  // as in fetch_angles
  if constexpr (tree_any(KIND)) asm volatile("" : "+v"(c0));
  const float ls = tree_i8(KIND) ? h2f((uint16_t)p.ls) * kLog2e : 0.0f;
  uint32_t e[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float2v cs = lut.code[pair_code<KIND, N>(a, codes, p, n, h, i, c0, t)];
    e[i] = key_pair(pair_radius<KIND, N>(p, n, h, i, ls), cs);
  }
  *reinterpret_cast<uint4v*>(kt + tile_at(t, 2 * c + h)) = uint4v{e[0], e[1], e[2], e[3]};
}

// And into a tile of values: 8 codes.
template <int KIND, int N, int THREADS>
__device__ __forceinline__ void decode_values(int tid, const PageRegs<KIND, N>& p, int n, int h, char* vt) {
  const int c = tid & 7, t = (tid >> 3) + (THREADS / 8) * n;
  const half2v scale = lo_lo(p.vs[n]);
  uint4v w;
#pragma unroll
  for (int j = 0; j < 2; ++j) {
    half2v lo, hi;
    i8x4_to_f16(p.v[n][2 * h + j], lo, hi);
    w[2 * j] = pack_h2(lo * scale);
    w[2 * j + 1] = pack_h2(hi * scale);
  }
  *reinterpret_cast<uint4v*>(vt + tile_at(t, 2 * c + h)) = w;
}

// Piece i of the 4 N that a page takes.
template <int KIND, int N, int THREADS, class Pages>
__device__ __forceinline__ void decode_piece(const Pages& a, const TreeLut& lut, const uint32_t* codes, int tid,
                                             const PageRegs<KIND, N>& p, int i, char* kt, char* vt) {
  if (i & 2)
    decode_values<KIND, N, THREADS>(tid, p, i >> 2, i & 1, vt);
  else
    decode_keys<KIND, N, THREADS>(a, lut, codes, tid, p, i >> 2, i & 1, kt);
}

// 64 dense tokens from k, v (t strides in elements) into the tiles; rows from `count` on repeat the
// last key (masked) and hold values of 0, as infinities and NaN among the values do, which are
// reported.
template <int THREADS>
__device__ __forceinline__ bool dense_tile(const uint16_t* k, const uint16_t* v, int64_t k_t, int64_t v_t, int count,
                                           int tid, char* kt, char* vt) {
  constexpr int N = kTileTokens * 16 / THREADS;
  uint4v kw[N], vw[N];
#pragma unroll
  for (int n = 0; n < N; ++n) {
    const int x = tid + THREADS * n, t = min(x >> 4, count - 1), c = x & 15;
    kw[n] = *reinterpret_cast<const uint4v*>(k + t * k_t + 8 * c);
    vw[n] = *reinterpret_cast<const uint4v*>(v + t * v_t + 8 * c);
  }
  bool flagged = false;
#pragma unroll
  for (int n = 0; n < N; ++n) {
    const int x = tid + THREADS * n, t = x >> 4, c = x & 15;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const uint32_t w = t < count ? vw[n][i] : 0u;
      flagged = flagged || pair_nonfinite<F16>(w);
      vw[n][i] = pair_finite<F16>(w);
    }
    *reinterpret_cast<uint4v*>(kt + tile_at(t, c)) = kw[n];
    *reinterpret_cast<uint4v*>(vt + tile_at(t, c)) = vw[n];
  }
  return flagged;
}

// Fills the table of a layout's angles; a barrier after it is the caller's.
template <int KIND, int THREADS, class Pages>
__device__ __forceinline__ void build_tree_lut(const Pages& a, TreeLut& lut, int tid) {
  for (int x = tid; x < 256; x += THREADS) {
    if constexpr (KIND == kTreeDefault) {
      if (x < 16) lut.code[x] = angle_pair(x, 4);
    } else if constexpr (KIND == kTreeFast) {
      lut.code[256 + x] = angle_pair(x, 8);
    } else {
      if (x < (1 << a.l1_bits)) lut.code[x] = angle_pair(x, a.l1_bits);
      if (x < (1 << a.deep_bits)) lut.code[256 + x] = angle_pair(x, a.deep_bits);
    }
  }
}

}  // namespace tp
