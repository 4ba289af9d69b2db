// tp_tree.hip -- attention of a tree of drafted tokens over a compressed cache.
//
//   out[b, h, i] = sum_j p_ij v_j,  p_ij = softmax_j(scale q[b, h, i] . k_j)
//
// over every stored page (decoded: k = r (cos a, sin a), v = code x scale), the dense tail, and
// of the drafted tokens node i itself and its ancestors.  A node that does not see itself is
// padding: its row is 0.
//
// The rows of a workgroup are (node, head of the group) pairs of one kv head, so a page is
// read and decoded once for up to 256 rows: its codes go through registers into an fp16 tile in
// LDS (the next page's codes in flight meanwhile), from which the waves multiply.  The cache is
// split over workgroups, the tail and the drafts go to one of their own, and a second launch
// joins their records.
#include <algorithm>

#include "tp_codes.h"
#include "tp_tiles.h"

namespace tp {

enum TreeKind { kTreeDefault = 0, kTreeFast = 1, kTreeAnyF16 = 2, kTreeAnyI8 = 3 };
constexpr bool tree_i8(int kind) { return kind == kTreeFast || kind == kTreeAnyI8; }
constexpr bool tree_any(int kind) { return kind == kTreeAnyF16 || kind == kTreeAnyI8; }

constexpr int kTreeMaxNodes = 256;
constexpr int kTreeTarget = 2048;  // waves that fill the GPU, two a SIMD

struct TreeArgs {
  const uint16_t* q;
  uint16_t* out;
  int64_t q_b, q_h, q_t, out_b, out_h, out_t;
  int32_t units, hkv, g, nodes, row_blocks;
  FastDiv div_units, div_blocks, div_hkv, div_g;
  const void* radii;
  const uint16_t* radii_scales;
  const uint8_t* angle_l1;
  const uint8_t* angle_deep;
  const int8_t* v_codes;
  const uint16_t* v_scales;
  int64_t capacity;
  int32_t n_pages, l1_bits, deep_bits, split_half, l1_row, deep_row;
  const uint16_t* tail_k;
  const uint16_t* tail_v;
  int64_t tail_stride;  // tokens
  int32_t tail_len;
  const uint16_t* draft_k;
  const uint16_t* draft_v;
  int64_t dk_b, dk_h, dk_t, dv_b, dv_h, dv_t;
  const uint64_t* mask;  // [batch or 1][nodes][words]: bit j of node i: i sees drafted token j
  int64_t mask_b;        // words between batch rows (0: one mask for all)
  int32_t words;
  float c;
  uint32_t flip;
  int32_t pages_per_split, page_splits, records;
  uint16_t* part_o;
  float* part_ml;
};

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

template <int KIND, int N, int THREADS>
__device__ __forceinline__ void load_page(const TreeArgs& a, int64_t slot, int tid, PageRegs<KIND, N>& p) {
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

// Decodes half h of run n into a tile of keys: 4 pairs, 16 bytes.
template <int KIND, int N, int THREADS>
__device__ __forceinline__ void decode_keys(const TreeArgs& a, const TreeLut& lut, const uint32_t* codes, int tid,
                                            const PageRegs<KIND, N>& p, int n, int h, char* kt) {
  const int c = tid & 7, t = (tid >> 3) + (THREADS / 8) * n;
  uint32_t e[4];
  const float ls = tree_i8(KIND) ? h2f((uint16_t)p.ls) * kLog2e : 0.0f;  // rounded in fp32, as its products below
  int c0 = c;  // where a pair's code lies is computed anew: kept over the pages, it costs 30 registers
  if constexpr (tree_any(KIND)) asm volatile("" : "+v"(c0));
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    uint32_t code;
    if constexpr (KIND == kTreeDefault) {
      code = (p.c4[n] >> (16 * h + 4 * i)) & 15u;
    } else if constexpr (KIND == kTreeFast) {
      code = 256 + ((p.c8[n][h] >> (8 * i)) & 0xffu);
    } else {
      const int pair = 8 * c0 + 4 * h + i;
      const bool l1 = pair < a.split_half;
      const int bits = l1 ? a.l1_bits : a.deep_bits;
      const int bit = (l1 ? pair : pair - a.split_half) * bits;
      const int row = l1 ? t * a.l1_row : kPageTokens * a.l1_row + t * a.deep_row;
      const uint32_t byte = reinterpret_cast<const uint8_t*>(codes)[row + (bit >> 3)];
      code = (l1 ? 0u : 256u) + ((byte >> (bit & 7)) & ((1u << bits) - 1u));
    }
    float r;
    if constexpr (tree_i8(KIND))
      r = __builtin_amdgcn_exp2f((float)(int)(int8_t)(p.r8[n][h] >> (8 * i)) * ls);
    else
      r = h2f((uint16_t)(p.r[n][2 * h + (i >> 1)] >> (16 * (i & 1))));
    e[i] = key_pair(r, lut.code[code]);
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
template <int KIND, int N, int THREADS>
__device__ __forceinline__ void decode_piece(const TreeArgs& a, const TreeLut& lut, const uint32_t* codes, int tid,
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

// RW waves of 32 rows each; TW waves share a row block and take a page's tokens in TW parts.  Two waves
// keep one tile in LDS, so that four such workgroups share a CU; more keep two.
template <int RW, int TW>
constexpr int kTreeThreads = 64 * RW * TW;

// The decode of a page (one product a pair of dimensions, one a pair of values) and the two products over it go
// on side by side: few rows are bound by the reads and the decode (5 nodes, 32 heads, 131,072 tokens of the fast
// layout: 63 us, 4.4 TB/s), 128 rows by decode and products alike (32 nodes over 32,805 tokens: 36.7 us, 2.1 TB/s and
// 0.46 PFLOP/s).
//
// A key component is rounded to fp16 once, from fp32 angles and radii, as the page decoder rounds it, so that what is
// attended is what the decoder hands out; a value, a weight, a record and the result once each; 32-bit sums.  An
// output's error, relative in L2, is 5.2e-4 (default layout, 1,000 tokens) to 7.0e-4 (fast layout, 131,072) by that,
// of which the keys alone give 3.7e-4 to 5.1e-4 (scores of a spread of 1.8); against attention in 64 bits over the
// decoder's numbers it is 3.5e-4.  Cosines, int8 radii and products in fp16 gave 5.9e-4 to 8.7e-4 for 2 % less time
// (32 nodes over 32,805 tokens with the join 40.6 us instead of 41.5).
template <int KIND, int RW, int TW>
__global__ __launch_bounds__((kTreeThreads<RW, TW>), 2) void tree_attention_kernel(TreeArgs a) {
  constexpr int THREADS = kTreeThreads<RW, TW>, N = 512 / THREADS, NB = 2 / TW, BUFS = RW * TW > 2 ? 2 : 1;
  __shared__ __align__(16) char tiles[BUFS][2][kTileBytes];
  __shared__ TreeLut lut;
  __shared__ uint32_t codes[tree_any(KIND) ? BUFS : 1][tree_any(KIND) ? 1024 : 1];  // any layout's code rows
  __shared__ float side_ml[TW == 2 ? RW : 1][2][64];
  __shared__ int flag;
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int rest = fast_div(blockIdx.x, a.div_units), unit = blockIdx.x - rest * a.units;
  const int record = fast_div(rest, a.div_blocks), block = rest - record * a.row_blocks;
  const int64_t slot0 = (int64_t)unit * a.capacity;
  int page = record * a.pages_per_split;
  const int page_end = record < a.page_splits ? min(page + a.pages_per_split, a.n_pages) : page;
  // The first page's loads before anything else; a record without pages has none to wait for.
  PageRegs<KIND, N> p;
  if (page < page_end) load_page<KIND, N, THREADS>(a, slot0 + page, tid, p);

  const int batch = fast_div(unit, a.div_hkv);
  const int64_t b = batch, kv = unit - batch * a.hkv;
  const int rw = wave / TW, tw = wave % TW;
  const int row = (block * RW + rw) * kWaveRows + (lane & 31);
  const int node = fast_div(row, a.div_g), head = row - node * a.g;
  const bool live = node < a.nodes;
  const int at_node = min(node, a.nodes - 1);  // loads of rows past the last node repeat it
  const uint64_t* mask = a.mask + b * a.mask_b + (int64_t)at_node * a.words;
  uint4v qs[8];
  load_query(a.q + b * a.q_b + (kv * a.g + head) * a.q_h + at_node * a.q_t, lane, qs);
  const uint64_t self = mask[at_node >> 6];
  const TileLane at(lane);
  RowState st;
  st.clear();

  if (tid == 0) flag = 0;
  if (page < page_end) {
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
    flip_query(a.flip, qs);
    __syncthreads();
    float16v s[NB];
    if constexpr (BUFS == 1) {
      static_assert(!tree_any(KIND), "any layout's codes are staged in the other form");
      for (; page < page_end; ++page) {
#pragma unroll
        for (int i = 0; i < 4 * N; ++i)
          decode_piece<KIND, N, THREADS>(a, lut, codes[0], tid, p, i, tiles[0][0], tiles[0][1]);
        __syncthreads();
        // The last page again rather than none: a load under a branch is waited for at its join.
        load_page<KIND, N, THREADS>(a, slot0 + min(page + 1, page_end - 1), tid, p);
        score_tile<F16, NB>(tiles[0][0], 32 * tw, at, qs, s, [](int) {});
        finish_tile<F16, NB>(tiles[0][1], 32 * tw, at, a.c, s, st);
        __syncthreads();
      }
    } else {
      // The next page is decoded under this one's first products.
      if constexpr (tree_any(KIND)) {
        stage_rows<KIND, N, THREADS>(tid, p, codes[0]);
        __syncthreads();
      }
#pragma unroll
      for (int i = 0; i < 4 * N; ++i)
        decode_piece<KIND, N, THREADS>(a, lut, codes[0], tid, p, i, tiles[0][0], tiles[0][1]);
      load_page<KIND, N, THREADS>(a, slot0 + min(page + 1, page_end - 1), tid, p);
      for (int buf = 0; page < page_end; ++page, buf ^= 1) {
        char *kt = tiles[buf ^ 1][0], *vt = tiles[buf ^ 1][1];
        const uint32_t* rows_of = codes[tree_any(KIND) ? buf ^ 1 : 0];
        stage_rows<KIND, N, THREADS>(tid, p, codes[tree_any(KIND) ? buf ^ 1 : 0]);
        __syncthreads();
        score_tile<F16, NB>(tiles[buf][0], 32 * tw, at, qs, s, [&](int i) {
          constexpr int kProducts = 8 * NB, kPieces = 4 * N;
#pragma unroll
          for (int x = i * kPieces / kProducts; x < (i + 1) * kPieces / kProducts; ++x)
            decode_piece<KIND, N, THREADS>(a, lut, rows_of, tid, p, x, kt, vt);
        });
        load_page<KIND, N, THREADS>(a, slot0 + min(page + 2, page_end - 1), tid, p);
        finish_tile<F16, NB>(tiles[buf][1], 32 * tw, at, a.c, s, st);
      }
    }
  }
  const bool real = live && ((self >> (at_node & 63)) & 1u);
  if (record == a.records - 1) {  // the tail and the drafts
    if (record >= a.page_splits) flip_query(a.flip, qs);  // not turned above
    const int first = a.tail_len > 0 ? -1 : 0;
    for (int j = first; j < a.words; ++j) {
      const uint16_t *k, *v;
      int64_t k_t, v_t;
      int count;
      if (j < 0) {
        k = a.tail_k + unit * a.tail_stride * kHeadDim, v = a.tail_v + unit * a.tail_stride * kHeadDim;
        k_t = v_t = kHeadDim;
        count = a.tail_len;
      } else {
        k = a.draft_k + b * a.dk_b + kv * a.dk_h + 64 * j * a.dk_t;
        v = a.draft_v + b * a.dv_b + kv * a.dv_h + 64 * j * a.dv_t;
        k_t = a.dk_t, v_t = a.dv_t;
        count = min(a.nodes - 64 * j, kTileTokens);
      }
      __syncthreads();  // the tile before is read
      if (dense_tile<THREADS>(k, v, k_t, v_t, count, tid, tiles[0][0], tiles[0][1])) flag = 1;
      __syncthreads();
      {
        const uint64_t there = count < 64 ? (1ull << count) - 1ull : ~0ull;
        const uint64_t sees = !real ? 0ull : j < 0 ? there : mask[j] & there;
        auto seen = [&](int x) { return ((sees >> x) & 1u) != 0; };
        float16v s[NB];
        score_tile<F16, NB>(tiles[0][0], 32 * tw, at, qs, s, [](int) {});
#pragma unroll
        for (int x = 0; x < 16 * NB; ++x)
          if (!seen(32 * (tw + (x >> 4)) + 8 * ((x & 15) >> 2) + (x & 3) + 4 * (lane >> 5))) s[x >> 4][x & 15] = -INFINITY;
        finish_tile<F16, NB>(tiles[0][1], 32 * tw, at, a.c, s, st);
        if (flag)
          add_nonfinite<F16>(st, lane, count, [&](int x) { return seen(x) && (TW == 1 || (x >> 5) == tw); },
                             [&](int x) { return v + x * v_t; });
      }
    }
  }
  if constexpr (TW == 2) {  // the second half's rows join the first's
    __syncthreads();
    static_assert(RW * 64 * 64 * sizeof(float) <= sizeof(tiles), "the second half's rows lie over the tiles");
    float* side = reinterpret_cast<float*>(&tiles[0][0][0]) + rw * 64 * 64 + lane;
    if (tw == 1) {
#pragma unroll
      for (int db = 0; db < 4; ++db)
#pragma unroll
        for (int i = 0; i < 16; ++i) side[(16 * db + i) * 64] = st.o[db][i];
      side_ml[rw][0][lane] = st.m;
      side_ml[rw][1][lane] = st.l;
    }
    __syncthreads();
    if (tw == 0) {
      const float m1 = side_ml[rw][0][lane], l1 = side_ml[rw][1][lane];
      const float m = fmaxf(st.m, m1), base = m == -INFINITY ? 0.0f : m;
      const float w0 = __builtin_amdgcn_exp2f(st.m - base), w1 = __builtin_amdgcn_exp2f(m1 - base);
#pragma unroll
      for (int db = 0; db < 4; ++db)
#pragma unroll
        for (int i = 0; i < 16; ++i) st.o[db][i] = st.o[db][i] * w0 + side[(16 * db + i) * 64] * w1;
      st.l = st.l * w0 + l1 * w1;
      st.m = m;
    }
  }
  if (tw != 0) return;
  if (!real) st.clear();  // padding: its queries were 0, its page tokens seen
  const float l = across_halves(st.l, [](float x, float y) { return x + y; });
  if (a.records > 1) {
    const int64_t rec = ((int64_t)unit * a.nodes * a.g + row) * a.records + record;
    // fp16: records of 32 bits lower the error from 6.1e-4 to 5.7e-4 and cost a tenth of the time (41.5 -> 45.2 us).
    store_record<true>(st, l, a.part_o + rec * kHeadDim, a.part_ml + rec * 2, live, lane);
  } else {
    store_row<F16>(st, l == 0.0f ? 0.0f : 1.0f / l, a.out + b * a.out_b + (kv * a.g + head) * a.out_h + node * a.out_t,
                   live, lane);
  }
}

// Rows of a workgroup, and how the pages are split: into as many workgroups as fill the GPU (two waves a
// SIMD).  Measured with 32/8 heads, us without the join:
//   up to 32 rows: two waves, four workgroups a CU, 63 over 131,072 tokens (four waves, two of them decoding only,
//     77); layouts whose codes go through LDS take the four of 64 rows, since a thread of two waves decodes four
//     runs, for which they have no registers (2-bit deep codes over 32,768 tokens 33 instead of 54);
//   up to 128 rows: four waves, 35 over 32,768 tokens (eight, each with half of a page's tokens, 40); the layouts
//     through LDS, which spill at four, the eight (split at pair 23: 51 instead of 88).
// The tail and the drafts take one more record, unless there is but one split of pages.
struct TreePlan {
  int32_t row_waves, row_blocks, pages_per_split, page_splits, records;
};
static TreePlan plan_tree(int64_t units, int64_t rows, int32_t n_pages, bool any) {
  TreePlan p;
  p.row_waves = rows <= 32 && !any ? 1 : rows <= 64 ? 2 : rows <= 128 ? 4 : 8;
  p.row_blocks = (int32_t)((rows + p.row_waves * kWaveRows - 1) / (p.row_waves * kWaveRows));
  const int64_t target = kTreeTarget / (p.row_waves == 8 || (p.row_waves == 4 && any) ? 8 : p.row_waves == 1 ? 2 : 4);
  const int64_t splits = std::max<int64_t>(1, std::min<int64_t>(target / (units * p.row_blocks), n_pages));
  p.pages_per_split = (int32_t)std::max<int64_t>(1, (n_pages + splits - 1) / splits);
  p.page_splits = (n_pages + p.pages_per_split - 1) / p.pages_per_split;
  p.records = p.page_splits <= 1 ? 1 : p.page_splits + 1;
  return p;
}

template <int KIND>
static void launch_tree(const TreeArgs& a, int row_waves, dim3 grid, hipStream_t s) {
  switch (row_waves) {
    case 1:
      if constexpr (!tree_any(KIND))
        hipLaunchKernelGGL((tree_attention_kernel<KIND, 1, 2>), grid, dim3(kTreeThreads<1, 2>), 0, s, a);
      break;
    case 2: hipLaunchKernelGGL((tree_attention_kernel<KIND, 2, 2>), grid, dim3(kTreeThreads<2, 2>), 0, s, a); break;
    case 4:
      if constexpr (tree_any(KIND))
        hipLaunchKernelGGL((tree_attention_kernel<KIND, 4, 2>), grid, dim3(kTreeThreads<4, 2>), 0, s, a);
      else
        hipLaunchKernelGGL((tree_attention_kernel<KIND, 4, 1>), grid, dim3(kTreeThreads<4, 1>), 0, s, a);
      break;
    default: hipLaunchKernelGGL((tree_attention_kernel<KIND, 8, 1>), grid, dim3(kTreeThreads<8, 1>), 0, s, a); break;
  }
}

}  // namespace tp

using namespace tp;

extern "C" size_t tp_tree_workspace_bytes(int64_t batch, int32_t hq, int32_t hkv, int32_t nodes, int32_t n_pages) {
  if (batch < 1 || hkv < 1 || hq < hkv || hq % hkv || nodes < 1 || nodes > kTreeMaxNodes || n_pages < 0) return 0;
  // Of the layouts, those with workgroups of two waves have the most splits.
  const TreePlan p = plan_tree(batch * hkv, (int64_t)nodes * (hq / hkv), n_pages, false);
  return p.records == 1 ? 0 : (size_t)batch * hq * nodes * p.records * (kHeadDim * sizeof(uint16_t) + 2 * sizeof(float));
}

extern "C" int32_t tp_tree_attention(const void* q, void* out, int64_t batch, int32_t hq, int32_t hkv, int32_t nodes,
                                     const tp_page_layout* layout, const tp_pages* pages, int32_t n_pages,
                                     const void* tail_k, const void* tail_v, int32_t tail_len, int64_t tail_stride,
                                     const void* draft_k, const void* draft_v, const int64_t* strides,
                                     const uint64_t* mask, int64_t mask_stride, float scale, void* workspace,
                                     size_t workspace_bytes, void* stream) {
  clear_error();
  int l1_row = 0, deep_row = 0;
  if (!check_layout(layout, &l1_row, &deep_row)) return TP_ERR_UNSUPPORTED;
  if (batch < 1 || hq < 1 || hkv < 1 || hq % hkv != 0 || batch > INT32_MAX / hkv) {
    set_error("bad query shape: batch=%lld hq=%d hkv=%d (hq must be a multiple of hkv)", (long long)batch, hq, hkv);
    return TP_ERR_INVALID;
  }
  if (nodes < 1 || nodes > kTreeMaxNodes || (int64_t)nodes * (hq / hkv) > INT32_MAX / 2) {
    set_error("nodes must be in [1, %d], got %d", kTreeMaxNodes, nodes);
    return TP_ERR_INVALID;
  }
  if (n_pages < 0 || (n_pages > 0 && (!pages || pages->capacity < n_pages))) {
    set_error("n_pages=%d exceeds page capacity", n_pages);
    return TP_ERR_INVALID;
  }
  if (n_pages > 0) {
    if (!pages->radii || !pages->v_codes || !pages->v_scales || (l1_row > 0 && !pages->angle_l1) ||
        (deep_row > 0 && !pages->angle_deep) || (layout->int8_radii && !pages->radii_scales)) {
      set_error("page buffers missing for this layout");
      return TP_ERR_INVALID;
    }
    if (((uintptr_t)pages->radii & 15u) || ((uintptr_t)pages->v_codes & 15u) || ((uintptr_t)pages->angle_l1 & 7u) ||
        ((uintptr_t)pages->angle_deep & 15u) || ((uintptr_t)pages->v_scales & 3u)) {
      set_error("page buffers are not aligned");
      return TP_ERR_INVALID;
    }
  }
  if (tail_len < 0 || tail_len >= kPageTokens) {
    set_error("tail_len must be in [0, 64), got %d", tail_len);
    return TP_ERR_INVALID;
  }
  if (tail_len > 0 && (!tail_k || !tail_v || tail_stride < tail_len || ((uintptr_t)tail_k & 15u) ||
                       ((uintptr_t)tail_v & 15u))) {
    set_error("tail buffers missing, misaligned or tail_stride < tail_len");
    return TP_ERR_INVALID;
  }
  if (!q || !out || !draft_k || !draft_v || !mask || ((uintptr_t)q & 15u) || ((uintptr_t)out & 15u) ||
      ((uintptr_t)draft_k & 15u) || ((uintptr_t)draft_v & 15u) || ((uintptr_t)mask & 7u) || mask_stride < 0) {
    set_error("q, out, draft_k and draft_v must be non-NULL 16-byte aligned buffers, mask an 8-byte aligned one");
    return TP_ERR_INVALID;
  }
  if (!strides) {
    set_error("strides is NULL");
    return TP_ERR_INVALID;
  }
  for (int i = 0; i < 12; ++i)
    if (strides[i] < 0 || (strides[i] & 7)) {
      set_error("strides must be non-negative multiples of 8 elements");
      return TP_ERR_INVALID;
    }
  if (!(scale == scale) || scale - scale != 0.0f) {
    set_error("scale must be finite");
    return TP_ERR_INVALID;
  }
  const int64_t units = batch * hkv, rows = (int64_t)nodes * (hq / hkv);
  const bool is_default = !layout->int8_radii && layout->l1_bits == 4 && layout->deep_bits == 4 && layout->split_dim == 64;
  const bool is_fast = layout->int8_radii && layout->deep_bits == 8 && layout->split_dim == 0;
  const TreePlan p = plan_tree(units, rows, n_pages, !is_default && !is_fast);
  if ((double)units * p.row_blocks * p.records > (double)INT32_MAX) {
    set_error("too many workgroups for one launch");
    return TP_ERR_INVALID;
  }
  TreeArgs a{};
  a.q = static_cast<const uint16_t*>(q);
  a.out = static_cast<uint16_t*>(out);
  int64_t* const to[12] = {&a.q_b, &a.q_h, &a.q_t, &a.dk_b, &a.dk_h, &a.dk_t, &a.dv_b, &a.dv_h, &a.dv_t, &a.out_b, &a.out_h, &a.out_t};
  for (int i = 0; i < 12; ++i) *to[i] = strides[i];
  a.units = (int32_t)units;
  a.hkv = hkv;
  a.g = hq / hkv;
  a.nodes = nodes;
  a.row_blocks = p.row_blocks;
  if (n_pages > 0) {
    a.radii = pages->radii;
    a.radii_scales = static_cast<const uint16_t*>(pages->radii_scales);
    a.angle_l1 = pages->angle_l1;
    a.angle_deep = pages->angle_deep;
    a.v_codes = pages->v_codes;
    a.v_scales = static_cast<const uint16_t*>(pages->v_scales);
    a.capacity = pages->capacity;
  }
  a.n_pages = n_pages;
  a.l1_bits = layout->l1_bits;
  a.deep_bits = layout->deep_bits;
  a.split_half = layout->split_dim / 2;
  a.l1_row = l1_row;
  a.deep_row = deep_row;
  a.tail_k = static_cast<const uint16_t*>(tail_k);
  a.tail_v = static_cast<const uint16_t*>(tail_v);
  a.tail_stride = tail_stride;
  a.tail_len = tail_len;
  a.draft_k = static_cast<const uint16_t*>(draft_k);
  a.draft_v = static_cast<const uint16_t*>(draft_v);
  a.mask = mask;
  a.mask_b = mask_stride;
  a.words = (nodes + 63) / 64;
  a.c = std::max(fabsf(scale) * kLog2e, 1.17549435e-38f);  // 2^-126 stands for 0: see tp_prompt_attention
  a.flip = scale < 0.0f ? 0x80008000u : 0u;
  a.pages_per_split = p.pages_per_split;
  a.page_splits = p.page_splits;
  a.records = p.records;
  if (a.records > 1) {
    const size_t need = tp_tree_workspace_bytes(batch, hq, hkv, nodes, n_pages);
    if (!workspace || workspace_bytes < need || ((uintptr_t)workspace & 255u)) {
      set_error("workspace of %zu bytes (256-byte aligned) required, got %zu", need, workspace_bytes);
      return TP_ERR_WORKSPACE;
    }
    a.part_o = static_cast<uint16_t*>(workspace);
    a.part_ml = reinterpret_cast<float*>(a.part_o + (size_t)units * rows * a.records * kHeadDim);
  }
  a.div_units = make_fastdiv((uint32_t)units);
  a.div_blocks = make_fastdiv((uint32_t)p.row_blocks);
  a.div_hkv = make_fastdiv((uint32_t)hkv);
  a.div_g = make_fastdiv((uint32_t)a.g);
  hipStream_t s = static_cast<hipStream_t>(stream);
  const dim3 grid((unsigned)(units * p.row_blocks * p.records));
  if (is_default)
    launch_tree<kTreeDefault>(a, p.row_waves, grid, s);
  else if (is_fast)
    launch_tree<kTreeFast>(a, p.row_waves, grid, s);
  else if (layout->int8_radii)
    launch_tree<kTreeAnyI8>(a, p.row_waves, grid, s);
  else
    launch_tree<kTreeAnyF16>(a, p.row_waves, grid, s);
  const int32_t st = launch_status("tp_tree_attention");
  if (st != TP_OK || a.records == 1) return st;
  JoinArgs j{};
  j.o = a.part_o;
  j.ml = a.part_ml;
  j.out = a.out;
  j.rows = rows;
  j.out_b = a.out_b, j.out_h = a.out_h, j.out_t = a.out_t;
  j.units = a.units, j.splits = a.records, j.g = a.g, j.hkv = hkv;
  return launch_join(j, false, true, s);
}
