// tp_prompt.hip -- attention over a whole prompt: causal or not, grouped query heads,
// sequences of one length or packed ones of different lengths.
//
//   out[b, h, i] = sum_j p_ij v[b, h / g, j],  p_ij = softmax_j(scale q[b, h, i] . k[b, h / g, j])
//
// over the keys j that query i sees: all nk of its sequence, or, causal, the first nk - nq
// + i + 1 (the queries are the last nq positions); a query that sees none gives 0.
//
// The rows of a workgroup are (token, head of the group) pairs of one kv head, so the
// g heads of a group share every tile of keys and values, and the rows of a workgroup
// span few tokens: little of the causal border is computed and masked.  A workgroup walks
// the keys in tiles of 64, the next tile's loads in flight over this one's products.
// Few tiles of rows: the keys are split over workgroups too, and joined by a second
// launch.
#include <algorithm>

#include "tp_tiles.h"

namespace tp {

constexpr int kPromptTarget = 256;  // workgroups that fill the GPU
// Packed sequences of a call.  Each adds a workgroup a kv head, and every workgroup looks its own up in the list, so
// their time grows with the square of their number.
constexpr int kMaxSequences = 65536;

struct PromptArgs {
  const uint16_t* q;
  const uint16_t* k;
  const uint16_t* v;
  uint16_t* out;
  int64_t q_b, q_h, q_t, k_b, k_h, k_t, v_b, v_h, v_t, out_b, out_h, out_t;  // strides in elements
  int32_t units, hkv, g, tq, tk;
  int32_t causal;
  const int32_t* q_starts;
  const int32_t* k_starts;
  int32_t n_seq;  // 0: one sequence a batch row
  int32_t keep_rest;
  int32_t tiles, splits;
  FastDiv div_units, div_splits, div_hkv, div_g;
  float c;        // |scale| log2(e)
  uint32_t flip;  // sign bits of a pair where the scale is negative
  float* part_o;
  float* part_ml;
};

// A tile of rows: queries [q0, q0 + nq) and keys [k0, k0 + nk) of its sequence, its first row.
struct PromptTile {
  int q0, nq, k0, nk, row0;
  bool rest;  // tokens behind the last sequence
};

template <int ROWS>
__device__ __forceinline__ PromptTile find_tile(const PromptArgs& a, int tile, int lane) {
  PromptTile t;
  t.rest = false;
  if (a.n_seq == 0) {
    t.q0 = 0, t.nq = a.tq, t.k0 = 0, t.nk = a.tk;
    t.row0 = (a.causal ? a.tiles - 1 - tile : tile) * ROWS;  // the longest first
    return t;
  }
  int before = 0;  // tiles of the sequences before
  for (int base = 0; base < a.n_seq; base += 64) {
    const int i = base + lane;
    int q0 = 0, q1 = 0;
    if (i < a.n_seq) {
      q0 = min(max(a.q_starts[i], 0), a.tq);
      q1 = min(max(a.q_starts[i + 1], q0), a.tq);
    }
    const int mine = (int)(((int64_t)(q1 - q0) * a.g + ROWS - 1) / ROWS);
    int upto = mine;
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) {
      const int x = __shfl_up(upto, d);
      if (lane >= d) upto += x;
    }
    const uint64_t found = __ballot(before + upto > tile);
    if (found) {
      const int w = __builtin_amdgcn_readfirstlane(__ffsll((unsigned long long)found) - 1);
      // Values of one lane for all: scalar from here on.
      t.q0 = __builtin_amdgcn_readlane(q0, w);
      t.nq = __builtin_amdgcn_readlane(q1, w) - t.q0;
      const int count = __builtin_amdgcn_readlane(mine, w);
      const int first = before + __builtin_amdgcn_readlane(upto, w) - count;
      t.k0 = min(max(a.k_starts[base + w], 0), a.tk);
      t.nk = min(max(a.k_starts[base + w + 1], t.k0), a.tk) - t.k0;
      t.row0 = (a.causal ? count - 1 - (tile - first) : tile - first) * ROWS;
      return t;
    }
    before += __builtin_amdgcn_readlane(upto, 63);
  }
  t.rest = true;
  t.q0 = min(max(a.q_starts[a.n_seq], 0), a.tq);
  t.nq = a.tq - t.q0;
  t.k0 = 0, t.nk = 0;
  t.row0 = (tile - before) * ROWS;
  return t;
}

// A thread's part of a tile of keys or values is 16-byte chunks tid + THREADS i of 64 rows of 16.
// Chunk i of tile j of the n tokens of x, `stride` bytes (below 2^24) apart.  Tiles past the last one
// repeat it and rows past the last token repeat that: no load is under a branch, at whose join it would
// be waited for.  The base is scalar, a lane's offset one 24-bit multiply-add.
template <int THREADS>
__device__ __forceinline__ uint4v load_chunk(const uint16_t* x, uint32_t stride, int j, int n, int tid, int i) {
  const int t0 = min(j, (n - 1) / kTileTokens) * kTileTokens, last = min(n - 1 - t0, kTileTokens - 1);
  const char* base = reinterpret_cast<const char*>(x) + (int64_t)t0 * stride;
  const uint32_t row = min((tid + THREADS * i) >> 4, last);
  return *reinterpret_cast<const uint4v*>(base + (__umul24(row, stride) + 16u * (tid & 15)));
}

template <int THREADS>
__device__ __forceinline__ void store_chunk(char* tile, int tid, int i, uint4v x) {
  const int at = tid + THREADS * i;
  *reinterpret_cast<uint4v*>(tile + tile_at(at >> 4, at & 15)) = x;
}

// Values of a tile that some row does not see whole: 0 past the last key (their weights are 0, and
// 0 times an infinity is not), and for infinities and NaN, which are reported.
template <class T, int THREADS>
__device__ __forceinline__ bool clean_part(int t0, int n, int tid, uint4v* r) {
  bool flagged = false;
#pragma unroll
  for (int j = 0; j < kTileTokens * 16 / THREADS; ++j)
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const uint32_t w = t0 + ((tid + THREADS * j) >> 4) < n ? r[j][i] : 0u;
      flagged = flagged || pair_nonfinite<T>(w);
      r[j][i] = pair_finite<T>(w);
    }
  return flagged;
}

// The products of a step: the next tile's scores in turn with a tile's weights and values, so that four
// products lie between two that add to the same registers.  Reads from LDS go out kAhead pairs before the
// products that take them.  Past the last tile the scores are of whatever the LDS holds, and not used: a
// second form without them would cost 64 registers more, where the two meet.  beside(i): what is issued under the products of pair i.
template <class T, class Beside>
__device__ __forceinline__ void multiply_tile(const char* kt, const char* vt, const TileLane& at, const uint4v* q,
                                              const uint4v* p, float16v* s, RowState& st, Beside beside) {
  constexpr int kAhead = 3;  // 4 would take 8 registers more than there are
  auto key = [&](int i) { return read_key<2>(kt, 0, at, i); };
  auto value = [&](int i) { return read_value(vt, 0, at, i); };
  uint4v k[kAhead], v[kAhead];
#pragma unroll
  for (int i = 0; i < kAhead; ++i) k[i] = key(i), v[i] = value(i);
  __builtin_amdgcn_sched_barrier(0);
#pragma unroll
  for (int i = 0; i < 16; ++i) {
    float16v& sum = s[i & 1];
    if (i < 2)
#pragma unroll
      for (int j = 0; j < 16; ++j) sum[j] = 0.0f;
    sum = T::mfma(k[i % kAhead], q[i >> 1], sum);
    if (i + kAhead < 16) k[i % kAhead] = key(i + kAhead);
    __builtin_amdgcn_sched_barrier(0);
    st.o[i & 3] = T::mfma(v[i % kAhead], p[i >> 2], st.o[i & 3]);
    if (i + kAhead < 16) v[i % kAhead] = value(i + kAhead);
    beside(i);
    __builtin_amdgcn_sched_barrier(0);
  }
}

// S^T = K Q^T and O^T += V^T P^T, so that a query is a column: its scores, maximum, sum and output stay with one
// pair of lanes, and P goes from the first product to the second in registers.  The work is 4 x 128 operations a
// query and key; the matrix units bind long prompts (32/8 heads, causal, fp16 4,096 tokens 151 us, 0.91 PFLOP/s;
// bf16 16,384 tokens 1.9 to 2.1 ms, 1.05 to 1.15, where the clock falls to 1.7 GHz; a large library product 1.2 to
// 1.3).  Where one wave of a SIMD computes its softmax, its partner multiplies (8 waves in two phases a tile).
template <class T, int WAVES>
__global__ __launch_bounds__(WAVES * 64, 2) void prompt_attention_kernel(PromptArgs a) {
  constexpr int ROWS = WAVES * kWaveRows, THREADS = WAVES * 64;
  __shared__ __align__(16) char kts[2][kTileBytes], vts[2][kTileBytes];
  __shared__ int flag;
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int rest = fast_div(blockIdx.x, a.div_units), unit = blockIdx.x - rest * a.units;
  const int tile = fast_div(rest, a.div_splits), split = rest - tile * a.splits;
  const PromptTile t = find_tile<ROWS>(a, tile, lane);
  const int batch = fast_div(unit, a.div_hkv);
  const int64_t b = batch, kv = unit - batch * a.hkv;
  auto token_of = [&](int row) { return (int)fast_div(row, a.div_g); };

  // The lane's row, and how many keys of its sequence it sees.
  auto keys_of = [&](int i) { return i >= t.nq ? 0 : a.causal ? min(max(t.nk - t.nq + i + 1, 0), t.nk) : t.nk; };
  const int wave_row = t.row0 + kWaveRows * wave, row = wave_row + (lane & 31);
  const int tok = token_of(row), head = row - tok * a.g;
  const int limit = keys_of(tok);
  // Of the workgroup's rows: the fewest and the most (the last live row's).  Rows past the last
  // query compute what they like and are not stored.
  const int last_tok = min(token_of(t.row0 + ROWS - 1), t.nq - 1);
  const int most = last_tok < 0 ? 0 : keys_of(last_tok), fewest = keys_of(token_of(t.row0));
  // Of the wave's.
  const int wave_most = token_of(wave_row) >= t.nq ? 0 : keys_of(min(token_of(wave_row + kWaveRows - 1), t.nq - 1));
  const int wave_fewest = keys_of(token_of(wave_row));

  // This split's tiles of keys, of those that the whole sequence has; the wave's end of them.
  const int all = (t.nk + kTileTokens - 1) / kTileTokens, each = (all + a.splits - 1) / a.splits;
  const int first = split * each, end = min(min(first + each, all), (most + kTileTokens - 1) / kTileTokens);
  const int wave_end = min(end, (wave_most + kTileTokens - 1) / kTileTokens);

  RowState st;
  st.clear();
  if (first < end) {
    const uint16_t* k = a.k + b * a.k_b + kv * a.k_h + (int64_t)t.k0 * a.k_t;
    const uint16_t* v = a.v + b * a.v_b + kv * a.v_h + (int64_t)t.k0 * a.v_t;
    const uint32_t k_t = (uint32_t)a.k_t * 2, v_t = (uint32_t)a.v_t * 2;
    constexpr int C = kTileTokens * 16 / THREADS;
    uint4v kr[2 * C], vr[C];
#pragma unroll
    for (int i = 0; i < 2 * C; ++i) kr[i] = load_chunk<THREADS>(k, k_t, first + i / C, t.nk, tid, i % C);
#pragma unroll
    for (int i = 0; i < C; ++i) vr[i] = load_chunk<THREADS>(v, v_t, first, t.nk, tid, i);
    uint4v q[8];
    const int64_t qt = t.q0 + min(tok, t.nq - 1);  // first < end: there is a query
    load_query(a.q + b * a.q_b + (kv * a.g + head) * a.q_h + qt * a.q_t, lane, q);
    const TileLane at(lane);
    auto clean = [&](int j) {  // where some row does not see all of tile j
      if ((j + 1) * kTileTokens > fewest && clean_part<T, THREADS>(j * kTileTokens, t.nk, tid, vr)) flag = 1;
    };
    // Tile j + 2's keys and j + 1's values to LDS, and the loads of those after them: piece i of 4 C.
    auto stage = [&](int j, int i) {
      const int c = i % C;
      if (i < C)
        store_chunk<THREADS>(kts[j & 1], tid, c, kr[c]);
      else if (i < 2 * C)
        store_chunk<THREADS>(vts[(j + 1) & 1], tid, c, vr[c]);
      else if (i < 3 * C)
        kr[c] = load_chunk<THREADS>(k, k_t, j + 3, t.nk, tid, c);
      else
        vr[c] = load_chunk<THREADS>(v, v_t, j + 2, t.nk, tid, c);
    };
    // Of 8 waves, w and w + 4 share a SIMD: the second four run one phase behind the first.
    const int behind = WAVES == 8 ? __builtin_amdgcn_readfirstlane(tid / (THREADS / 2)) : 0;
    if (tid == 0) flag = 0;
    __syncthreads();
    clean(first);
#pragma unroll
    for (int i = 0; i < 2 * C; ++i) store_chunk<THREADS>(kts[(first + i / C) & 1], tid, i % C, kr[i]);
#pragma unroll
    for (int i = 0; i < C; ++i) {
      store_chunk<THREADS>(vts[first & 1], tid, i, vr[i]);
      kr[i] = load_chunk<THREADS>(k, k_t, first + 2, t.nk, tid, i);
      vr[i] = load_chunk<THREADS>(v, v_t, first + 1, t.nk, tid, i);
    }
    __syncthreads();
    flip_query(a.flip, q);
    float16v s[2];
    if (first < wave_end) score_tile<T, 2>(kts[first & 1], 0, at, q, s, [](int) {});
    if (behind) lds_barrier();
    // Two phases a tile, a barrier after each (which waits for LDS accesses, not for loads from memory): the softmax,
    // and the products.  While one wave of a SIMD
    // multiplies, the other runs its softmax (in step, 41 % of the time went to products and almost all of
    // the rest to softmax).  The next tiles go to LDS under the products, into the buffers that both
    // halves of the waves have left by then.
    for (int j = first; j < end; ++j) {
      uint4v p[4];
      if (j < wave_end) {
        if ((j + 1) * kTileTokens > wave_fewest) mask_scores<2>(s, limit - 4 * (lane >> 5) - j * kTileTokens);
        rescale<2>(s, a.c, st);
        weigh<T, 2>(s, a.c, p, st);
      }
      clean(j + 1);
      lds_barrier();
      if (j < wave_end) {
        __builtin_amdgcn_s_setprio(1);
        multiply_tile<T>(kts[(j + 1) & 1], vts[j & 1], at, q, p, s, st, [&](int i) {
          if (i * C / 2 < 4 * C)
#pragma unroll
            for (int x = i * C / 2; x < (i + 1) * C / 2; ++x) stage(j, x);
        });
        __builtin_amdgcn_s_setprio(0);
      } else {
#pragma unroll
        for (int i = 0; i < 4 * C; ++i) stage(j, i);
      }
      lds_barrier();
    }
    if (!behind) lds_barrier();
    if (flag) {
      const int t0 = max(fewest / kTileTokens, first) * kTileTokens;  // the first tile with a border
      add_nonfinite<T>(st, lane, min(end * kTileTokens, t.nk) - t0, [&](int x) { return t0 + x < limit; },
                       [&](int x) { return v + (int64_t)(t0 + x) * a.v_t; });
    }
  }
  const float l = across_halves(st.l, [](float x, float y) { return x + y; });
  const int64_t out_t = t.q0 + tok;
  const bool live = tok < t.nq;
  if (a.splits > 1) {
    const int64_t rec = (((int64_t)unit * a.tq + out_t) * a.g + head) * a.splits + split;
    store_record<false>(st, l, a.part_o + rec * kHeadDim, a.part_ml + rec * 2, live, lane);
  } else if (!(t.rest && a.keep_rest)) {
    store_row<T>(st, l == 0.0f ? 0.0f : 1.0f / l, a.out + b * a.out_b + (kv * a.g + head) * a.out_h + out_t * a.out_t,
                 live, lane);
  }
}

// Joins the splits of a row: weights l_s 2^(m_s - max) over their sum.  A record's 16 bytes a lane: 16 lanes
// (fp16) or 32 (fp32) take one, so 4 or 2 records go by side by side and are folded at the end, kAhead such
// steps in flight.  WAVES waves a row, each a part of its records: one, or four where there are few rows of
// many records (129 records of 256 rows 8.4 -> 5.1 us, 65 of 1,024 7.4 -> 6.2).
template <class T, bool HALF, int kAhead, int WAVES>
__global__ __launch_bounds__(256) void join_splits_kernel(JoinArgs a) {
  constexpr int kLanes = HALF ? 16 : 32, kSide = 64 / kLanes, kDims = kHeadDim / kLanes;
  __shared__ float part_acc[WAVES > 1 ? WAVES : 1][kHeadDim], part_ml[WAVES][2];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, part = lane / kLanes, d0 = lane % kLanes * kDims;
  const int64_t i = WAVES > 1 ? (int64_t)blockIdx.x : (int64_t)blockIdx.x * 4 + wave;
  if (i >= (int64_t)a.units * a.rows) return;
  const int64_t unit = i / a.rows, row = i - unit * a.rows;
  const int64_t tok = row / a.g, head = row - tok * a.g;
  if (a.rest_from && tok >= *a.rest_from) return;
  const int each = (a.splits + WAVES - 1) / WAVES;
  const int first = WAVES > 1 ? min(wave * each, a.splits) : 0, end = min(first + each, a.splits);
  const float* ml = a.ml + i * a.splits * 2;
  const char* o = static_cast<const char*>(a.o) + (i * a.splits * kHeadDim + d0) * (HALF ? 2 : 4);
  float m = -INFINITY, l = 0.0f, acc[kDims] = {};
  for (int base = first; base < end; base += 64) {
    const int n = min(64, end - base);
    float2v mine = {-INFINITY, 0.0f};
    if (lane < n) mine = *reinterpret_cast<const float2v*>(ml + 2 * (base + lane));
    if (mine.y == 0.0f) mine.x = -INFINITY;  // saw nothing
    float top = mine.x;
#pragma unroll
    for (int d = 32; d; d >>= 1) top = fmaxf(top, __shfl_xor(top, d));
    const float next = fmaxf(m, top), to = next == -INFINITY ? 0.0f : next;
    const float w = mine.y == 0.0f ? 0.0f : mine.y * __builtin_amdgcn_exp2f(mine.x - to);
    float sum = w;
#pragma unroll
    for (int d = 32; d; d >>= 1) sum += __shfl_xor(sum, d);
    const float alpha = __builtin_amdgcn_exp2f(m - to);
#pragma unroll
    for (int d = 0; d < kDims; ++d) acc[d] *= alpha;
    l = l * alpha + sum;
    m = next;
    for (int s0 = 0; s0 < n; s0 += kAhead * kSide) {
      uint4v x[kAhead];
#pragma unroll
      for (int j = 0; j < kAhead; ++j) {
        const int s = min(s0 + kSide * j + part, n - 1);
        x[j] = *reinterpret_cast<const uint4v*>(o + (int64_t)(base + s) * kHeadDim * (HALF ? 2 : 4));
      }
#pragma unroll
      for (int j = 0; j < kAhead; ++j) {
        const int s = s0 + kSide * j + part;
        const float of_lane = __shfl(w, s & 63);  // with every lane taking part
        const float ws = s < n ? of_lane : 0.0f;
#pragma unroll
        for (int d = 0; d < kDims; ++d) {
          float v;
          if constexpr (HALF)
            v = h2f((uint16_t)(x[j][d >> 1] >> (16 * (d & 1))));
          else
            v = __uint_as_float(x[j][d]);
          acc[d] += ws != 0.0f ? ws * v : 0.0f;
        }
      }
    }
  }
#pragma unroll
  for (int d = 0; d < kDims; ++d)
#pragma unroll
    for (int step = kLanes; step < 64; step <<= 1) acc[d] += __shfl_xor(acc[d], step);
  if constexpr (WAVES > 1) {
    if (part == 0)
#pragma unroll
      for (int d = 0; d < kDims; ++d) part_acc[wave][d0 + d] = acc[d];
    if (lane == 0) part_ml[wave][0] = m, part_ml[wave][1] = l;
    __syncthreads();
    if (wave != 0) return;
    float top = -INFINITY;
#pragma unroll
    for (int w = 0; w < WAVES; ++w) top = fmaxf(top, part_ml[w][0]);
    if (top == -INFINITY) top = 0.0f;
    l = 0.0f;
#pragma unroll
    for (int d = 0; d < kDims; ++d) acc[d] = 0.0f;
#pragma unroll
    for (int w = 0; w < WAVES; ++w) {
      const float scale = __builtin_amdgcn_exp2f(part_ml[w][0] - top);
      l += part_ml[w][1] * scale;
#pragma unroll
      for (int d = 0; d < kDims; ++d) acc[d] += part_acc[w][d0 + d] * scale;
    }
  }
  const float inv = l == 0.0f ? 0.0f : 1.0f / l;
  if (part != 0) return;
  uint16_t* out = a.out + (unit / a.hkv) * a.out_b + ((unit % a.hkv) * a.g + head) * a.out_h + tok * a.out_t + d0;
  uint32_t y[kDims / 2];
#pragma unroll
  for (int d = 0; d < kDims / 2; ++d) y[d] = T::pack(acc[2 * d] * inv, acc[2 * d + 1] * inv);
  if constexpr (HALF)
    *reinterpret_cast<uint4v*>(out) = uint4v{y[0], y[1], y[2], y[3]};
  else
    *reinterpret_cast<uint2v*>(out) = uint2v{y[0], y[1]};
}

template <class T, bool HALF>
static void launch_join_of(const JoinArgs& a, hipStream_t s) {
  const int64_t rows = (int64_t)a.units * a.rows;
  const int steps = (a.splits + (HALF ? 3 : 1)) / (HALF ? 4 : 2);
  const dim3 grid((unsigned)((rows + 3) / 4));
  if (steps <= 2)
    hipLaunchKernelGGL((join_splits_kernel<T, HALF, 2, 1>), grid, dim3(256), 0, s, a);
  else if (steps > 5 && rows <= 4096)
    hipLaunchKernelGGL((join_splits_kernel<T, HALF, 5, 4>), dim3((unsigned)rows), dim3(256), 0, s, a);
  else
    hipLaunchKernelGGL((join_splits_kernel<T, HALF, 5, 1>), grid, dim3(256), 0, s, a);
}

int32_t launch_join(const JoinArgs& a, bool bf16, bool half_records, hipStream_t s) {
  if (half_records)
    launch_join_of<F16, true>(a, s);
  else if (bf16)
    launch_join_of<BF16, false>(a, s);
  else
    launch_join_of<F16, false>(a, s);
  return launch_status("join of the splits");
}

// Waves a workgroup, tiles of rows per unit (an upper bound where sequences are packed: each has one that
// it does not fill, and so have the tokens behind them) and splits of the keys.  256 rows (8 waves) read
// keys and values half as often as 128; where they leave part of the GPU idle, 128 rows do not, start
// sooner and fit a CU twice: 32/8 heads, 64 queries of 64 tokens 8.7 us (256 rows 10.9), but 8,192 causal tokens
// 609 (256 rows 549).  Few tiles all the same: each is given to as many workgroups as fill the GPU, of 4 tiles of
// keys at least, since the join takes as long as some 4 of them: 64 queries over 1,024 keys, us with the join,
// at least 2, 4 or 8 tiles: 18.2, 18.2, 22.1; over 4,096 keys 32.8, 26.8, 25.0; over 512 keys (4 or 8) 17.1, 16.4.
struct PromptPlan {
  int64_t waves, tiles, splits;
};
static int64_t prompt_tiles(int64_t rows, int64_t tile, int32_t n_seq) {
  return n_seq ? rows / tile + n_seq + 1 : (rows + tile - 1) / tile;
}
static PromptPlan plan_prompt(int64_t units, int32_t g, int64_t tq, int64_t tk, int32_t n_seq) {
  PromptPlan p;
  p.waves = units * prompt_tiles(tq * g, 256, n_seq) < kPromptTarget ? 4 : 8;
  p.tiles = prompt_tiles(tq * g, p.waves * kWaveRows, n_seq);
  const int64_t all = units * p.tiles, key_tiles = (tk + kTileTokens - 1) / kTileTokens;
  const int64_t target = p.waves == 8 ? kPromptTarget : 2 * kPromptTarget;
  p.splits = std::max<int64_t>(1, std::min<int64_t>(target / std::max<int64_t>(all, 1), key_tiles / 4));
  return p;
}

static bool strides_ok(const int64_t* s, int n) {
  for (int i = 0; i < n; ++i)
    if (s[i] < 0 || (s[i] & 7)) return false;
  return true;
}

}  // namespace tp

using namespace tp;

extern "C" size_t tp_prompt_workspace_bytes(int64_t batch, int32_t hq, int32_t hkv, int64_t tq, int64_t tk,
                                            int32_t n_seq) {
  if (batch < 1 || hkv < 1 || hq < hkv || hq % hkv || tq < 1 || tk < 1 || n_seq < 0) return 0;
  const PromptPlan p = plan_prompt(batch * hkv, hq / hkv, tq, tk, n_seq);
  if (p.splits == 1) return 0;
  return (size_t)batch * hq * tq * p.splits * (kHeadDim + 2) * sizeof(float);
}

extern "C" int32_t tp_prompt_attention(const void* q, const void* k, const void* v, void* out, int32_t dtype,
                                       int64_t batch, int32_t hq, int32_t hkv, int64_t tq, int64_t tk,
                                       const int64_t* strides, int32_t causal, const int32_t* q_starts,
                                       const int32_t* k_starts, int32_t n_seq, int32_t keep_rest, float scale,
                                       void* workspace, size_t workspace_bytes, void* stream) {
  clear_error();
  if (dtype != 0 && dtype != 1) {
    set_error("dtype must be 0 (fp16) or 1 (bf16), got %d", dtype);
    return TP_ERR_INVALID;
  }
  if (batch < 1 || hq < 1 || hkv < 1 || hq % hkv != 0 || tq < 0 || tk < 0 || n_seq < 0) {
    set_error("bad shape: batch=%lld hq=%d hkv=%d (hq must be a multiple of hkv) tq=%lld tk=%lld n_seq=%d",
              (long long)batch, hq, hkv, (long long)tq, (long long)tk, n_seq);
    return TP_ERR_INVALID;
  }
  const int32_t g = hq / hkv;
  // Rows, tokens and workgroups are counted in 32 bits.
  if (tk > INT32_MAX - 2 * kTileTokens || tq > (INT32_MAX - 512) / g || batch > INT32_MAX / hkv) {
    set_error("tq=%lld x %d heads a group, tk=%lld or batch * hkv exceeds 2^31 rows", (long long)tq, g, (long long)tk);
    return TP_ERR_INVALID;
  }
  if (n_seq && (batch != 1 || !q_starts || !k_starts || ((uintptr_t)q_starts & 3u) || ((uintptr_t)k_starts & 3u))) {
    set_error("packed sequences need a batch of 1 and both start arrays");
    return TP_ERR_INVALID;
  }
  if (n_seq > kMaxSequences) {
    set_error("a call takes at most %d packed sequences, got %d", kMaxSequences, n_seq);
    return TP_ERR_INVALID;
  }
  if (tq == 0) return TP_OK;
  if (!q || !out || (tk && (!k || !v)) || ((uintptr_t)q & 15u) || ((uintptr_t)k & 15u) || ((uintptr_t)v & 15u) ||
      ((uintptr_t)out & 15u)) {
    set_error("q, k, v and out must be non-NULL 16-byte aligned buffers");
    return TP_ERR_INVALID;
  }
  // Keys' and values' offsets within a tile are 24-bit products.
  if (!strides || !strides_ok(strides, 12) || strides[5] >= (1 << 23) || strides[8] >= (1 << 23)) {
    set_error("strides must be non-negative multiples of 8 elements, the token strides of k and v below 2^23");
    return TP_ERR_INVALID;
  }
  if (!(scale == scale) || scale - scale != 0.0f) {
    set_error("scale must be finite");
    return TP_ERR_INVALID;
  }
  const PromptPlan p = plan_prompt(batch * hkv, g, tq, std::max<int64_t>(tk, 1), n_seq);
  // Rows are counted in 32 bits up to the end of the last tile, workgroups too.
  if (p.tiles * p.waves * kWaveRows > INT32_MAX ||
      (double)batch * hkv * (double)p.tiles * (double)p.splits > (double)INT32_MAX) {
    set_error("too many tiles of rows for one launch");
    return TP_ERR_INVALID;
  }
  PromptArgs a{};
  a.q = static_cast<const uint16_t*>(q);
  a.k = static_cast<const uint16_t*>(k);
  a.v = static_cast<const uint16_t*>(v);
  a.out = static_cast<uint16_t*>(out);
  int64_t* const to[12] = {&a.q_b, &a.q_h, &a.q_t, &a.k_b, &a.k_h, &a.k_t, &a.v_b, &a.v_h, &a.v_t, &a.out_b, &a.out_h, &a.out_t};
  for (int i = 0; i < 12; ++i) *to[i] = strides[i];
  a.units = (int32_t)(batch * hkv);
  a.hkv = hkv;
  a.g = g;
  a.tq = (int32_t)tq;
  a.tk = (int32_t)tk;
  a.causal = causal != 0;
  a.q_starts = q_starts;
  a.k_starts = k_starts;
  a.n_seq = n_seq;
  a.keep_rest = keep_rest != 0;
  a.tiles = (int32_t)p.tiles;
  a.splits = (int32_t)p.splits;
  // A scale of 0 weighs every key alike; 2^-126 does so too and leaves a masked score at -inf.
  a.c = std::max(fabsf(scale) * kLog2e, 1.17549435e-38f);
  a.flip = scale < 0.0f ? 0x80008000u : 0u;
  if (a.splits > 1) {
    const size_t need = tp_prompt_workspace_bytes(batch, hq, hkv, tq, tk, n_seq);
    if (!workspace || workspace_bytes < need || ((uintptr_t)workspace & 255u)) {
      set_error("workspace of %zu bytes (256-byte aligned) required, got %zu", need, workspace_bytes);
      return TP_ERR_WORKSPACE;
    }
    a.part_o = static_cast<float*>(workspace);
    a.part_ml = a.part_o + (size_t)batch * hq * tq * a.splits * kHeadDim;
  }
  hipStream_t s = static_cast<hipStream_t>(stream);
  a.div_units = make_fastdiv((uint32_t)a.units);
  a.div_splits = make_fastdiv((uint32_t)a.splits);
  a.div_hkv = make_fastdiv((uint32_t)hkv);
  a.div_g = make_fastdiv((uint32_t)g);
  const dim3 grid((unsigned)(a.units * p.tiles * p.splits)), threads((unsigned)p.waves * 64);
  if (dtype && p.waves == 8)
    hipLaunchKernelGGL((prompt_attention_kernel<BF16, 8>), grid, threads, 0, s, a);
  else if (dtype)
    hipLaunchKernelGGL((prompt_attention_kernel<BF16, 4>), grid, threads, 0, s, a);
  else if (p.waves == 8)
    hipLaunchKernelGGL((prompt_attention_kernel<F16, 8>), grid, threads, 0, s, a);
  else
    hipLaunchKernelGGL((prompt_attention_kernel<F16, 4>), grid, threads, 0, s, a);
  const int32_t st = launch_status("tp_prompt_attention");
  if (st != TP_OK || a.splits == 1) return st;
  JoinArgs j{};
  j.o = a.part_o;
  j.ml = a.part_ml;
  j.out = a.out;
  j.rows = tq * g;
  j.out_b = a.out_b, j.out_h = a.out_h, j.out_t = a.out_t;
  j.units = a.units, j.splits = a.splits, j.g = g, j.hkv = hkv;
  j.rest_from = n_seq && keep_rest ? q_starts + n_seq : nullptr;
  return launch_join(j, dtype != 0, false, s);
}
