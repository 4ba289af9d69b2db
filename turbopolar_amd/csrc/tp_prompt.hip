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

constexpr int kPromptWaves = 8;
constexpr int kPromptRows = kPromptWaves * kWaveRows;
constexpr int kPromptThreads = kPromptWaves * 64;
constexpr int kPromptTarget = 256;  // workgroups that fill the GPU

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

__device__ __forceinline__ PromptTile find_tile(const PromptArgs& a, int tile, int lane) {
  PromptTile t;
  t.rest = false;
  if (a.n_seq == 0) {
    t.q0 = 0, t.nq = a.tq, t.k0 = 0, t.nk = a.tk;
    t.row0 = (a.causal ? a.tiles - 1 - tile : tile) * kPromptRows;  // the longest first
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
    const int mine = (int)(((int64_t)(q1 - q0) * a.g + kPromptRows - 1) / kPromptRows);
    int upto = mine;
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) {
      const int x = __shfl_up(upto, d);
      if (lane >= d) upto += x;
    }
    const uint64_t found = __ballot(before + upto > tile);
    if (found) {
      const int w = __ffsll((unsigned long long)found) - 1;
      t.q0 = __shfl(q0, w);
      t.nq = __shfl(q1, w) - t.q0;
      const int first = before + __shfl(upto, w) - __shfl(mine, w), count = __shfl(mine, w);
      t.k0 = min(max(a.k_starts[base + w], 0), a.tk);
      t.nk = min(max(a.k_starts[base + w + 1], t.k0), a.tk) - t.k0;
      t.row0 = (a.causal ? count - 1 - (tile - first) : tile - first) * kPromptRows;
      return t;
    }
    before += __shfl(upto, 63);
  }
  t.rest = true;
  t.q0 = min(max(a.q_starts[a.n_seq], 0), a.tq);
  t.nq = a.tq - t.q0;
  t.k0 = 0, t.nk = 0;
  t.row0 = (tile - before) * kPromptRows;
  return t;
}

// A tile's loads of one thread: 16-byte chunks tid + 512 j of 64 rows of 16, keys, then values.
constexpr int kChunksPerThread = kTileTokens * 16 / kPromptThreads;
struct PromptLoads {
  uint4v k[kChunksPerThread], v[kChunksPerThread];
};

__device__ __forceinline__ void load_tile(const uint16_t* k, const uint16_t* v, int64_t k_t, int64_t v_t, int t0,
                                          int nk, int tid, PromptLoads& r) {
#pragma unroll
  for (int j = 0; j < kChunksPerThread; ++j) {
    const int x = tid + kPromptThreads * j, c = x & 15;
    const int64_t t = min(t0 + (x >> 4), nk - 1);
    r.k[j] = *reinterpret_cast<const uint4v*>(k + t * k_t + 8 * c);
    r.v[j] = *reinterpret_cast<const uint4v*>(v + t * v_t + 8 * c);
  }
}

// Into LDS.  Values past the last key are 0 (their weights are 0, and 0 times an infinity is
// not); BORDER: infinities and NaN of the others are 0 too, and flagged.
template <class T, bool BORDER>
__device__ __forceinline__ bool store_tile(char* kt, char* vt, int t0, int nk, int tid, PromptLoads& r) {
  bool flagged = false;
#pragma unroll
  for (int j = 0; j < kChunksPerThread; ++j) {
    const int x = tid + kPromptThreads * j, at = tile_at(x >> 4, x & 15);
    *reinterpret_cast<uint4v*>(kt + at) = r.k[j];
    if constexpr (BORDER) {
      const bool in = t0 + (x >> 4) < nk;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const uint32_t w = in ? r.v[j][i] : 0u;
        flagged = flagged || pair_nonfinite<T>(w);
        r.v[j][i] = pair_finite<T>(w);
      }
    }
    *reinterpret_cast<uint4v*>(vt + at) = r.v[j];
  }
  return flagged;
}

template <class T>
__global__ __launch_bounds__(kPromptThreads, 2) void prompt_attention_kernel(PromptArgs a) {
  __shared__ __align__(16) char tiles[2][2][kTileBytes];
  __shared__ int flags[2];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int unit = blockIdx.x % a.units, rest = blockIdx.x / a.units;
  const int split = rest % a.splits;
  const PromptTile t = find_tile(a, rest / a.splits, lane);
  const int64_t b = unit / a.hkv, kv = unit % a.hkv;

  // The lane's row, and how many keys of its sequence it sees.
  const int row = t.row0 + kWaveRows * wave + (lane & 31);
  const int tok = row / a.g, head = row - tok * a.g;
  const bool live = tok < t.nq;
  auto keys_of = [&](int i) { return i >= t.nq ? 0 : a.causal ? min(max(t.nk - t.nq + i + 1, 0), t.nk) : t.nk; };
  const int limit = keys_of(tok);
  // Of the workgroup's rows: the fewest and the most (the last live row's).
  const int last_tok = min((t.row0 + kPromptRows - 1) / a.g, t.nq - 1);
  const int most = last_tok < 0 ? 0 : keys_of(last_tok), fewest = keys_of(t.row0 / a.g);
  // Of the wave's.
  const int wave_row = t.row0 + kWaveRows * wave;
  const int wave_last = min((wave_row + kWaveRows - 1) / a.g, t.nq - 1);
  const int wave_most = wave_row / a.g >= t.nq ? 0 : keys_of(wave_last);
  const int wave_fewest = (wave_row + kWaveRows - 1) / a.g >= t.nq ? 0 : keys_of(wave_row / a.g);

  // This split's tiles of keys, of those that the whole sequence has.
  const int all = (t.nk + kTileTokens - 1) / kTileTokens, each = (all + a.splits - 1) / a.splits;
  const int first = split * each, end = min(min(first + each, all), (most + kTileTokens - 1) / kTileTokens);

  RowState st;
  st.clear();
  if (first < end) {
    const uint16_t* k = a.k + b * a.k_b + kv * a.k_h + (int64_t)t.k0 * a.k_t;
    const uint16_t* v = a.v + b * a.v_b + kv * a.v_h + (int64_t)t.k0 * a.v_t;
    uint4v q[8];
    const int64_t qt = t.q0 + (live ? tok : 0);
    load_query(a.q + b * a.q_b + (kv * a.g + head) * a.q_h + qt * a.q_t, live, a.flip, lane, q);
    const TileLane at(lane);
    if (tid < 2) flags[tid] = 0;
    PromptLoads r;
    load_tile(k, v, a.k_t, a.v_t, first * kTileTokens, t.nk, tid, r);
    __syncthreads();
    for (int j = first; j < end; ++j) {
      const int t0 = j * kTileTokens, buf = j & 1;
      char *kt = tiles[buf][0], *vt = tiles[buf][1];
      const bool border = t0 + kTileTokens > fewest;  // some row of the workgroup does not see all of it
      if (border) {
        if (store_tile<T, true>(kt, vt, t0, t.nk, tid, r)) flags[buf] = 1;
      } else {
        store_tile<T, false>(kt, vt, t0, t.nk, tid, r);
      }
      __syncthreads();
      if (j + 1 < end) load_tile(k, v, a.k_t, a.v_t, t0 + kTileTokens, t.nk, tid, r);
      if (t0 < wave_most) {
        if (t0 + kTileTokens <= wave_fewest)
          attend_tile<T, 2, false>(kt, vt, 0, at, q, a.c, st, lane, [](int) { return true; });
        else
          attend_tile<T, 2, true>(kt, vt, 0, at, q, a.c, st, lane, [&](int x) { return t0 + x < limit; });
        if (border && flags[buf])
          add_nonfinite<T>(st, lane, min(kTileTokens, t.nk - t0), [&](int x) { return t0 + x < limit; },
                           [&](int x) { return v + (int64_t)(t0 + x) * a.v_t; });
      }
    }
  }
  const float l = across_halves(st.l, [](float x, float y) { return x + y; });
  const int64_t out_t = t.q0 + tok;
  if (a.splits > 1) {
    const int64_t rec = (((int64_t)unit * a.tq + out_t) * a.g + head) * a.splits + split;
    store_record(st, l, a.part_o + rec * kHeadDim, a.part_ml + rec * 2, live, lane);
  } else if (!(t.rest && a.keep_rest)) {
    store_row<T>(st, l == 0.0f ? 0.0f : 1.0f / l, a.out + b * a.out_b + (kv * a.g + head) * a.out_h + out_t * a.out_t,
                 live, lane);
  }
}

// Joins the splits of a row: weights l_s 2^(m_s - max) over their sum, two dimensions a lane, a
// wave a row.  Records with a sum of 0 (nothing seen) are not read.
template <class T>
__global__ __launch_bounds__(256) void join_splits_kernel(JoinArgs a) {
  const int lane = threadIdx.x & 63;
  const int64_t i = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6);
  if (i >= (int64_t)a.units * a.rows) return;
  const int64_t unit = i / a.rows, row = i - unit * a.rows;
  const int64_t tok = row / a.g, head = row - tok * a.g;
  if (a.rest_from && tok >= *a.rest_from) return;
  const float* ml = a.ml + i * a.splits * 2;
  const float* o = a.o + i * a.splits * kHeadDim + 2 * lane;
  float m = -INFINITY, l = 0.0f;
  float2v acc = {0.0f, 0.0f};
  for (int base = 0; base < a.splits; base += 64) {
    const int n = min(64, a.splits - base);
    float2v mine = {-INFINITY, 0.0f};
    if (lane < n) mine = *reinterpret_cast<const float2v*>(ml + 2 * (base + lane));
    if (mine.y == 0.0f) mine.x = -INFINITY;
    float top = mine.x;
#pragma unroll
    for (int d = 32; d; d >>= 1) top = fmaxf(top, __shfl_xor(top, d));
    const float next = fmaxf(m, top), to = next == -INFINITY ? 0.0f : next;
    const float w = mine.y == 0.0f ? 0.0f : mine.y * __builtin_amdgcn_exp2f(mine.x - to);
    float sum = w;
#pragma unroll
    for (int d = 32; d; d >>= 1) sum += __shfl_xor(sum, d);
    const float alpha = __builtin_amdgcn_exp2f(m - to);
    acc *= alpha;
    l = l * alpha + sum;
    m = next;
    for (int s = 0; s < n; ++s) {
      const float ws = __uint_as_float(__builtin_amdgcn_readlane(__float_as_uint(w), s));
      if (ws != 0.0f) acc += ws * *reinterpret_cast<const float2v*>(o + (int64_t)(base + s) * kHeadDim);
    }
  }
  const float inv = l == 0.0f ? 0.0f : 1.0f / l;
  uint16_t* out = a.out + (unit / a.hkv) * a.out_b + ((unit % a.hkv) * a.g + head) * a.out_h + tok * a.out_t;
  *reinterpret_cast<uint32_t*>(out + 2 * lane) = T::pack(acc.x * inv, acc.y * inv);
}

int32_t launch_join(const JoinArgs& a, bool bf16, hipStream_t s) {
  const int64_t rows = (int64_t)a.units * a.rows;
  const dim3 grid((unsigned)((rows + 3) / 4));
  if (bf16)
    hipLaunchKernelGGL((join_splits_kernel<BF16>), grid, dim3(256), 0, s, a);
  else
    hipLaunchKernelGGL((join_splits_kernel<F16>), grid, dim3(256), 0, s, a);
  return launch_status("join of the splits");
}

// Tiles of rows per unit (an upper bound where sequences are packed: each has one that it does
// not fill, and so have the tokens behind them) and splits of the keys: few tiles leave most of
// the GPU idle, so each is given to as many workgroups as fill it, of two tiles of keys at least.
struct PromptPlan {
  int64_t tiles, splits;
};
static PromptPlan plan_prompt(int64_t units, int32_t g, int64_t tq, int64_t tk, int32_t n_seq) {
  PromptPlan p;
  p.tiles = n_seq ? tq * g / kPromptRows + n_seq + 1 : (tq * g + kPromptRows - 1) / kPromptRows;
  const int64_t all = units * p.tiles, key_tiles = (tk + kTileTokens - 1) / kTileTokens;
  p.splits = std::max<int64_t>(1, std::min<int64_t>(kPromptTarget / std::max<int64_t>(all, 1), key_tiles / 2));
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
  if (tk > INT32_MAX - 2 * kTileTokens || tq > (INT32_MAX - 2 * kPromptRows) / g || batch > INT32_MAX / hkv) {
    set_error("tq=%lld x %d heads a group, tk=%lld or batch * hkv exceeds 2^31 rows", (long long)tq, g, (long long)tk);
    return TP_ERR_INVALID;
  }
  if (n_seq && (batch != 1 || !q_starts || !k_starts || ((uintptr_t)q_starts & 3u) || ((uintptr_t)k_starts & 3u))) {
    set_error("packed sequences need a batch of 1 and both start arrays");
    return TP_ERR_INVALID;
  }
  if (tq == 0) return TP_OK;
  if (!q || !out || (tk && (!k || !v)) || ((uintptr_t)q & 15u) || ((uintptr_t)k & 15u) || ((uintptr_t)v & 15u) ||
      ((uintptr_t)out & 15u)) {
    set_error("q, k, v and out must be non-NULL 16-byte aligned buffers");
    return TP_ERR_INVALID;
  }
  if (!strides || !strides_ok(strides, 12)) {
    set_error("strides must be non-negative multiples of 8 elements");
    return TP_ERR_INVALID;
  }
  if (!(scale == scale) || scale - scale != 0.0f) {
    set_error("scale must be finite");
    return TP_ERR_INVALID;
  }
  const PromptPlan p = plan_prompt(batch * hkv, g, tq, std::max<int64_t>(tk, 1), n_seq);
  if ((double)batch * hkv * (double)p.tiles * (double)p.splits > (double)INT32_MAX) {
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
  const dim3 grid((unsigned)(a.units * p.tiles * p.splits));
  if (dtype)
    hipLaunchKernelGGL((prompt_attention_kernel<BF16>), grid, dim3(kPromptThreads), 0, s, a);
  else
    hipLaunchKernelGGL((prompt_attention_kernel<F16>), grid, dim3(kPromptThreads), 0, s, a);
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
  return launch_join(j, dtype != 0, s);
}
