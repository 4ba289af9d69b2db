// tp_shared.hip -- one decode step's attention of sequences that share a prefix.
//
//   out[b, h] = sum_j p_j v_j,  p_j = softmax_j(scale q[b, h] . k_j)
//
// over the tokens of the prefix (one cache, stored once) and those of row b's own cache.  The softmax of a
// union is joined from the softmaxes of its parts, (m, l, o) each, so the prefix is attended by every row of
// the batch together: its rows are the (sequence, head of the group) pairs of one kv head, up to 256 of them
// for one read and one decode of a page.  A row's own pages are attended by its own heads.  Both are split into
// runs of tiles (a page, or the dense tail) and go on in one launch, or one each (plan_shared); a last one joins
// the records.
#include <algorithm>

#include "tp_page_tiles.h"

namespace tp {

// One of the two caches: its pages and tail, and the workgroups over it.
struct SharedPart {
  const void* radii;
  const uint16_t* radii_scales;
  const uint8_t* angle_l1;
  const uint8_t* angle_deep;
  const int8_t* v_codes;
  const uint16_t* v_scales;
  int32_t l1_bits, deep_bits, split_half, l1_row, deep_row;
  int64_t capacity;
  const uint16_t* tail_k;
  const uint16_t* tail_v;
  int64_t tail_stride;  // tokens
  int32_t n_pages, tail_len;
  int32_t units;       // hkv, or batch * hkv
  int32_t rows;        // batch * g, or g
  int32_t row_blocks;  // of the workgroup's rows
  int32_t tiles_per_split, records, first_record;
  FastDiv div_units, div_blocks;
};

struct SharedArgs {
  const uint16_t* q;
  uint16_t* out;
  int64_t q_b, q_h, out_b, out_h;
  int32_t hkv, g;
  FastDiv div_hkv, div_g;
  SharedPart part[2];  // the prefix, the rows' own
  int32_t prefix_groups;  // workgroups over the prefix, the launch's first
  int32_t records;
  float c;
  uint32_t flip;
  uint16_t* part_o;
  float* part_ml;
};

template <int RW, int TW>
constexpr int kSharedThreads = 64 * RW * TW;

// RW waves of 32 rows each; TW waves share a row block and take a tile's tokens in TW parts (as the
// drafted-tree kernel's).  Roundings: a key component once, from fp32 angles and radii, a value, a weight, a
// record and the result once each; sums in 32 bits.  The keys', which makes them the page decoder's, is most of the
// result's error (relative L2 5.7e-4 to 7.1e-4 over a long prefix): with keys in two parts it was 3.5e-4, and the kernel
// took 49 us where it took 38.7.
// A page is decoded in 1.7 us a workgroup on its own CU, under the products of the page before: 32 sequences of 32/8
// heads, 300 tokens each behind 32,805 (103 MB, 17.4 GFLOP) take 40.4 us and the join of the records 5.7 (42.9 in all,
// pass behind pass): bound by the
// decode, vector operations and table reads, rather than by the bytes (20 us of a copy's time) or the products (14.5 at
// a large product's rate).
template <int KIND, int RW, int TW>
__global__ __launch_bounds__((kSharedThreads<RW, TW>), 2) void shared_attention_kernel(SharedArgs a) {
  constexpr int THREADS = kSharedThreads<RW, TW>, N = 512 / THREADS, NB = 2 / TW, BUFS = RW * TW > 2 ? 2 : 1;
  __shared__ __align__(16) char tiles[BUFS][2][kTileBytes];
  __shared__ TreeLut lut;
  __shared__ uint32_t codes[tree_any(KIND) ? BUFS : 1][tree_any(KIND) ? 1024 : 1];
  __shared__ float side_ml[TW == 2 ? RW : 1][2][64];
  __shared__ int flag;
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const bool own = (int)blockIdx.x >= a.prefix_groups;
  const SharedPart& src = a.part[own ? 1 : 0];
  const int index = own ? (int)blockIdx.x - a.prefix_groups : (int)blockIdx.x;
  const int rest = fast_div(index, src.div_units), unit = index - rest * src.units;
  const int split = fast_div(rest, src.div_blocks), block = rest - split * src.row_blocks;
  const int64_t slot0 = (int64_t)unit * src.capacity;
  int page = split * src.tiles_per_split;
  const int page_end = min(page + src.tiles_per_split, src.n_pages);
  PageRegs<KIND, N> p;
  if (page < page_end) load_page<KIND, N, THREADS>(src, slot0 + page, tid, p);

  // Own rows fill a wave or two of the workgroup's; which ones goes round, so that those of neighbours lie on
  // different SIMDs, and the others only decode.
  const int tw = wave % TW, rw = (wave / TW + (own ? index : 0)) & (RW - 1);
  const bool busy = (block * RW + rw) * kWaveRows < src.rows;
  const int row = (block * RW + rw) * kWaveRows + (lane & 31);
  const bool live = row < src.rows;
  const int at_row = min(row, src.rows - 1);  // loads of rows past the last repeat it
  const int of_unit = fast_div(unit, a.div_hkv);
  const int seq_in = fast_div(at_row, a.div_g);
  const int64_t b = own ? of_unit : seq_in, kv = own ? unit - of_unit * a.hkv : unit;
  const int64_t head = kv * a.g + (own ? at_row : at_row - seq_in * a.g);
  uint4v qs[8];
  load_query(a.q + b * a.q_b + head * a.q_h, lane, qs);
  flip_query(a.flip, qs);
  const TileLane at(lane);
  RowState st;
  st.clear();

  if (tid == 0) flag = 0;
  if (page < page_end) {
    build_tree_lut<KIND, THREADS>(src, lut, tid);
    lds_barrier();
    float16v s[NB];
    if constexpr (BUFS == 1) {
      static_assert(!tree_any(KIND), "any layout's codes are staged in the other form");
      for (; page < page_end; ++page) {
#pragma unroll
        for (int i = 0; i < 4 * N; ++i)
          decode_piece<KIND, N, THREADS>(src, lut, codes[0], tid, p, i, tiles[0][0], tiles[0][1]);
        lds_barrier();
        // The last page again rather than none: a load under a branch is waited for at its join.
        load_page<KIND, N, THREADS>(src, slot0 + min(page + 1, page_end - 1), tid, p);
        score_tile<F16, NB>(tiles[0][0], 32 * tw, at, qs, s, [](int) {});
        finish_tile<F16, NB>(tiles[0][1], 32 * tw, at, a.c, s, st);
        lds_barrier();
      }
    } else {
      // The next page is decoded under this one's first products.
      if constexpr (tree_any(KIND)) {
        stage_rows<KIND, N, THREADS>(tid, p, codes[0]);
        lds_barrier();
      }
#pragma unroll
      for (int i = 0; i < 4 * N; ++i)
        decode_piece<KIND, N, THREADS>(src, lut, codes[0], tid, p, i, tiles[0][0], tiles[0][1]);
      load_page<KIND, N, THREADS>(src, slot0 + min(page + 1, page_end - 1), tid, p);
      for (int buf = 0; page < page_end; ++page, buf ^= 1) {
        char *kt = tiles[buf ^ 1][0], *vt = tiles[buf ^ 1][1];
        const uint32_t* rows_of = codes[tree_any(KIND) ? buf ^ 1 : 0];
        stage_rows<KIND, N, THREADS>(tid, p, codes[tree_any(KIND) ? buf ^ 1 : 0]);
        lds_barrier();
        if (busy) {
          // Of each key piece the table is read, a piece of values decoded, and the keys then.
          constexpr int kSlots = 8 * NB / (2 * N);
          float2v cs[4];
          score_tile<F16, NB>(tiles[buf][0], 32 * tw, at, qs, s, [&](int i) {
            const int piece = i / kSlots, at_slot = i % kSlots, n = piece >> 1, h = piece & 1;
            if (at_slot == 0) fetch_angles<KIND, N, THREADS>(src, lut, rows_of, tid, p, n, h, cs);
            if (at_slot == kSlots / 2) decode_values<KIND, N, THREADS>(tid, p, n, h, vt);
            if (at_slot == kSlots - 1) store_keys<KIND, N, THREADS>(tid, p, n, h, cs, kt);
          });
        } else {
#pragma unroll
          for (int i = 0; i < 4 * N; ++i) decode_piece<KIND, N, THREADS>(src, lut, rows_of, tid, p, i, kt, vt);
        }
        load_page<KIND, N, THREADS>(src, slot0 + min(page + 2, page_end - 1), tid, p);
        if (busy) finish_tile<F16, NB>(tiles[buf][1], 32 * tw, at, a.c, s, st);
      }
    }
  }
  if (split == src.records - 1 && src.tail_len > 0) {
    const int count = src.tail_len;
    const uint16_t* k = src.tail_k + unit * src.tail_stride * kHeadDim;
    const uint16_t* v = src.tail_v + unit * src.tail_stride * kHeadDim;
    lds_barrier();  // the tile before is read
    if (dense_tile<THREADS>(k, v, kHeadDim, kHeadDim, count, tid, tiles[0][0], tiles[0][1])) flag = 1;
    lds_barrier();
    if (busy) {
      float16v s[NB];
      score_tile<F16, NB>(tiles[0][0], 32 * tw, at, qs, s, [](int) {});
      mask_scores<NB>(s, count - 32 * tw - 4 * (lane >> 5));
      finish_tile<F16, NB>(tiles[0][1], 32 * tw, at, a.c, s, st);
      if (flag)
        add_nonfinite<F16>(st, lane, count, [&](int x) { return TW == 1 || (x >> 5) == tw; },
                           [&](int x) { return v + x * kHeadDim; });
    }
  }
  if constexpr (TW == 2) {  // the second half's rows join the first's
    lds_barrier();
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
    lds_barrier();
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
  const float l = across_halves(st.l, [](float x, float y) { return x + y; });
  if (a.records > 1) {
    const int64_t rec = (b * a.hkv * a.g + head) * a.records + src.first_record + split;
    store_record<true>(st, l, a.part_o + rec * kHeadDim, a.part_ml + rec * 2, live, lane);
  } else {
    store_row<F16>(st, l == 0.0f ? 0.0f : 1.0f / l, a.out + b * a.out_b + head * a.out_h, live, lane);
  }
}

constexpr int kSharedWaves = 2048;  // that fill the GPU, two a SIMD
constexpr int kSharedCus = 256;

struct SharedPlan {
  int32_t row_waves[2];
  int64_t tiles[2], row_blocks[2], tiles_per_split[2], records[2];
  bool apart;  // a launch for either part
};

// Splits of parts [begin, end), which are one launch.
static void plan_splits(SharedPlan& p, const int64_t* units, int64_t rows, int begin, int end, bool any) {
  const int rw = p.row_waves[begin];
  const int64_t slots = kSharedWaves / (rw == 8 || (rw == 4 && any) ? 8 : rw == 1 ? 2 : 4);
  int64_t total = 0;
  for (int i = begin; i < end; ++i) total += units[i] * p.row_blocks[i] * p.tiles[i];
  // In tiles of 1.7 us: a CU works on those it is dealt (workgroups go round the CUs) hardly faster for being two
  // (32,805 tokens for 32 rows of 32/8 heads, 17 tiles each on 248 CUs 38.7 us, 9 on 456 places 42.0), small
  // workgroups rather so (512 of two waves, 4 tiles each 16.8 us, 1,024 of 2 tiles 13.9); a round of workgroups
  // starts and ends in 6 us; the records are written and read at 3 TB/s.
  const double shared = rw == 1 ? 0.33 : 0.8, alone = rw == 1 ? 0.75 : 0.2;
  const int64_t even = (total + kSharedCus - 1) / kSharedCus;
  const int64_t step = std::max<int64_t>(1, even / 16);
  double best = INFINITY;
  int64_t chosen = 1;
  for (int64_t each = std::max<int64_t>(1, even / 4); each <= 2 * even + 2; each += step) {
    int64_t dealt = 0, groups = 0, records = 0, longest = 0;
    for (int i = begin; i < end; ++i) {
      const int64_t splits = (p.tiles[i] + each - 1) / each, n = units[i] * p.row_blocks[i] * splits;
      dealt += (n + kSharedCus - 1) / kSharedCus * std::min(each, p.tiles[i]);
      longest = std::max(longest, std::min(each, p.tiles[i]));
      groups += n;
      records += splits;
    }
    const double cost = shared * (double)dealt + alone * (double)longest + 3.5 * (double)((groups + slots - 1) / slots) +
                        (double)(rows * records) * (2.0 * 264.0 / 3.0e6 / 1.7);
    if (cost < best) best = cost, chosen = each;
  }
  for (int i = begin; i < end; ++i) {
    p.tiles_per_split[i] = chosen;
    p.records[i] = (p.tiles[i] + chosen - 1) / chosen;
  }
}

// Rows of a workgroup by the prefix's rows, as the drafted-tree kernel takes them (see plan_tree).  The rows' own
// tokens go along in workgroups of that size, of which one wave multiplies, or get a launch of workgroups of their
// size: where the prefix's have eight waves (us, one launch and two: 64 sequences of 32/8 heads, 1,000 tokens behind
// 16,000, 77 and 59; of 64/8 heads, 200 behind 4,000, 38 both), or where they are more than 24 tiles a CU (32
// sequences of 32/8 heads behind 16,000, 1,000 tokens each 41 and 42, 2,000 56 and 53, 4,000 92 and 81).
static SharedPlan plan_shared(int64_t batch, int32_t hkv, int32_t g, int64_t prefix_tiles, int64_t own_tiles, bool any) {
  SharedPlan p;
  auto waves_for = [&](int64_t rows) { return rows <= 32 && !any ? 1 : rows <= 64 ? 2 : rows <= 128 ? 4 : 8; };
  const int64_t units[2] = {hkv, batch * hkv}, rows[2] = {batch * g, g};
  p.tiles[0] = prefix_tiles, p.tiles[1] = own_tiles;
  p.row_waves[0] = p.row_waves[1] = waves_for(prefix_tiles ? rows[0] : rows[1]);
  p.apart = prefix_tiles && own_tiles &&
            (p.row_waves[0] == 8 || (p.row_waves[0] == 4 && any) ||
             (p.row_waves[0] != waves_for(rows[1]) && units[1] * own_tiles > 24 * kSharedCus));
  if (p.apart) p.row_waves[1] = waves_for(rows[1]);
  for (int i = 0; i < 2; ++i)
    p.row_blocks[i] = (rows[i] + p.row_waves[i] * kWaveRows - 1) / (p.row_waves[i] * kWaveRows);
  if (p.apart) {
    plan_splits(p, units, batch * hkv * g, 0, 1, any);
    plan_splits(p, units, batch * hkv * g, 1, 2, any);
  } else {
    plan_splits(p, units, batch * hkv * g, 0, 2, any);
  }
  return p;
}

template <int KIND>
static void launch_shared(const SharedArgs& a, int row_waves, dim3 grid, hipStream_t s) {
  switch (row_waves) {
    case 1:
      if constexpr (!tree_any(KIND))
        hipLaunchKernelGGL((shared_attention_kernel<KIND, 1, 2>), grid, dim3(kSharedThreads<1, 2>), 0, s, a);
      break;
    case 2: hipLaunchKernelGGL((shared_attention_kernel<KIND, 2, 2>), grid, dim3(kSharedThreads<2, 2>), 0, s, a); break;
    case 4:
      if constexpr (tree_any(KIND))
        hipLaunchKernelGGL((shared_attention_kernel<KIND, 4, 2>), grid, dim3(kSharedThreads<4, 2>), 0, s, a);
      else
        hipLaunchKernelGGL((shared_attention_kernel<KIND, 4, 1>), grid, dim3(kSharedThreads<4, 1>), 0, s, a);
      break;
    default: hipLaunchKernelGGL((shared_attention_kernel<KIND, 8, 1>), grid, dim3(kSharedThreads<8, 1>), 0, s, a); break;
  }
}

static bool is_default_layout(const tp_page_layout* l) {
  return !l->int8_radii && l->l1_bits == 4 && l->deep_bits == 4 && l->split_dim == 64;
}
static bool is_fast_layout(const tp_page_layout* l) { return l->int8_radii && l->deep_bits == 8 && l->split_dim == 0; }

// One cache's arguments into `p`; false with the error set.
static bool fill_part(SharedPart& p, const char* what, const tp_page_layout* layout, int l1_row, int deep_row,
                      const tp_pages* pages, int32_t n_pages, const void* tail_k, const void* tail_v, int32_t tail_len,
                      int64_t tail_stride) {
  if (n_pages < 0 || (n_pages > 0 && (!pages || pages->capacity < n_pages))) {
    set_error("%s: n_pages=%d exceeds page capacity", what, n_pages);
    return false;
  }
  if (n_pages > 0) {
    if (!pages->radii || !pages->v_codes || !pages->v_scales || (l1_row > 0 && !pages->angle_l1) ||
        (deep_row > 0 && !pages->angle_deep) || (layout->int8_radii && !pages->radii_scales)) {
      set_error("%s: page buffers missing for this layout", what);
      return false;
    }
    if (((uintptr_t)pages->radii & 15u) || ((uintptr_t)pages->v_codes & 15u) || ((uintptr_t)pages->angle_l1 & 7u) ||
        ((uintptr_t)pages->angle_deep & 15u) || ((uintptr_t)pages->v_scales & 3u)) {
      set_error("%s: page buffers are not aligned", what);
      return false;
    }
    p.radii = pages->radii;
    p.radii_scales = static_cast<const uint16_t*>(pages->radii_scales);
    p.angle_l1 = pages->angle_l1, p.angle_deep = pages->angle_deep;
    p.v_codes = pages->v_codes, p.v_scales = static_cast<const uint16_t*>(pages->v_scales);
    p.capacity = pages->capacity;
  }
  if (tail_len < 0 || tail_len >= kPageTokens) {
    set_error("%s: tail_len must be in [0, 64), got %d", what, tail_len);
    return false;
  }
  if (tail_len > 0 && (!tail_k || !tail_v || tail_stride < tail_len || ((uintptr_t)tail_k & 15u) ||
                       ((uintptr_t)tail_v & 15u))) {
    set_error("%s: tail buffers missing, misaligned or tail_stride < tail_len", what);
    return false;
  }
  p.tail_k = static_cast<const uint16_t*>(tail_k), p.tail_v = static_cast<const uint16_t*>(tail_v);
  p.tail_stride = tail_stride, p.tail_len = tail_len, p.n_pages = n_pages;
  p.l1_bits = layout->l1_bits, p.deep_bits = layout->deep_bits, p.split_half = layout->split_dim / 2;
  p.l1_row = l1_row, p.deep_row = deep_row;
  return true;
}

}  // namespace tp

using namespace tp;

extern "C" size_t tp_shared_workspace_bytes(int64_t batch, int32_t hq, int32_t hkv, const tp_page_layout* layout,
                                            int32_t prefix_pages, int32_t prefix_tail, int32_t n_pages,
                                            int32_t tail_len) {
  if (batch < 1 || hkv < 1 || hq < hkv || hq % hkv || batch > INT32_MAX / hq || !layout || prefix_pages < 0 || n_pages < 0)
    return 0;
  const SharedPlan p = plan_shared(batch, hkv, hq / hkv, (int64_t)prefix_pages + (prefix_tail > 0), (int64_t)n_pages + (tail_len > 0),
                                   !is_default_layout(layout) && !is_fast_layout(layout));
  const int64_t records = p.records[0] + p.records[1];
  return records <= 1 ? 0 : (size_t)batch * hq * records * (kHeadDim * sizeof(uint16_t) + 2 * sizeof(float));
}

extern "C" int32_t tp_shared_attention(const void* q, void* out, int64_t batch, int32_t hq, int32_t hkv,
                                       const tp_page_layout* layout, const tp_pages* prefix, int32_t prefix_pages,
                                       const void* prefix_tail_k, const void* prefix_tail_v, int32_t prefix_tail,
                                       int64_t prefix_tail_stride, const tp_pages* pages, int32_t n_pages,
                                       const void* tail_k, const void* tail_v, int32_t tail_len, int64_t tail_stride,
                                       const int64_t* strides, float scale, void* workspace, size_t workspace_bytes,
                                       void* stream) {
  clear_error();
  int l1_row = 0, deep_row = 0;
  if (!check_layout(layout, &l1_row, &deep_row)) return TP_ERR_UNSUPPORTED;
  if (batch < 1 || hq < 1 || hkv < 1 || hq % hkv != 0 || batch > INT32_MAX / 512 / hq) {
    set_error("bad query shape: batch=%lld hq=%d hkv=%d (hq must be a multiple of hkv)", (long long)batch, hq, hkv);
    return TP_ERR_INVALID;
  }
  SharedArgs a{};
  if (!fill_part(a.part[0], "prefix", layout, l1_row, deep_row, prefix, prefix_pages, prefix_tail_k, prefix_tail_v,
                 prefix_tail, prefix_tail_stride) ||
      !fill_part(a.part[1], "own tokens", layout, l1_row, deep_row, pages, n_pages, tail_k, tail_v, tail_len, tail_stride))
    return TP_ERR_INVALID;
  if (prefix_pages + prefix_tail + n_pages + tail_len == 0) {
    set_error("nothing to attend: no pages and no tail");
    return TP_ERR_INVALID;
  }
  if (!q || !out || ((uintptr_t)q & 15u) || ((uintptr_t)out & 15u)) {
    set_error("q and out must be non-NULL 16-byte aligned buffers");
    return TP_ERR_INVALID;
  }
  if (!strides) {
    set_error("strides is NULL");
    return TP_ERR_INVALID;
  }
  for (int i = 0; i < 4; ++i)
    if (strides[i] < 0 || (strides[i] & 7)) {
      set_error("strides must be non-negative multiples of 8 elements");
      return TP_ERR_INVALID;
    }
  if (!(scale == scale) || scale - scale != 0.0f) {
    set_error("scale must be finite");
    return TP_ERR_INVALID;
  }
  const bool def = is_default_layout(layout), fast = is_fast_layout(layout);
  const int32_t g = hq / hkv;
  const SharedPlan p = plan_shared(batch, hkv, g, (int64_t)prefix_pages + (prefix_tail > 0), (int64_t)n_pages + (tail_len > 0),
                                   !def && !fast);
  const int64_t units[2] = {hkv, batch * hkv}, rows[2] = {batch * g, g};
  int64_t groups[2];
  for (int i = 0; i < 2; ++i) {
    SharedPart& x = a.part[i];
    groups[i] = units[i] * p.row_blocks[i] * p.records[i];
    x.units = (int32_t)units[i], x.rows = (int32_t)rows[i], x.row_blocks = (int32_t)p.row_blocks[i];
    x.tiles_per_split = (int32_t)p.tiles_per_split[i], x.records = (int32_t)p.records[i];
    x.div_units = make_fastdiv((uint32_t)units[i]), x.div_blocks = make_fastdiv((uint32_t)p.row_blocks[i]);
  }
  a.part[1].first_record = (int32_t)p.records[0];
  const int rw = std::max(p.row_waves[0], p.row_waves[1]);
  if ((groups[0] + groups[1]) * (rw == 8 ? 512 : 128 * rw) > (int64_t)UINT32_MAX) {
    set_error("too many workgroups for one launch, whose threads are less than 2^32");
    return TP_ERR_INVALID;
  }
  a.q = static_cast<const uint16_t*>(q);
  a.out = static_cast<uint16_t*>(out);
  a.q_b = strides[0], a.q_h = strides[1], a.out_b = strides[2], a.out_h = strides[3];
  a.hkv = hkv, a.g = g;
  a.div_hkv = make_fastdiv((uint32_t)hkv), a.div_g = make_fastdiv((uint32_t)g);
  a.records = (int32_t)(p.records[0] + p.records[1]);
  a.c = std::max(fabsf(scale) * kLog2e, 1.17549435e-38f);  // 2^-126 stands for 0: see tp_prompt_attention
  a.flip = scale < 0.0f ? 0x80008000u : 0u;
  if (a.records > 1) {
    const size_t need = tp_shared_workspace_bytes(batch, hq, hkv, layout, prefix_pages, prefix_tail, n_pages, tail_len);
    if (!workspace || workspace_bytes < need || ((uintptr_t)workspace & 255u)) {
      set_error("workspace of %zu bytes (256-byte aligned) required, got %zu", need, workspace_bytes);
      return TP_ERR_WORKSPACE;
    }
    a.part_o = static_cast<uint16_t*>(workspace);
    a.part_ml = reinterpret_cast<float*>(a.part_o + (size_t)batch * hq * a.records * kHeadDim);
  }
  hipStream_t s = static_cast<hipStream_t>(stream);
  for (int i = 0; i < (p.apart ? 2 : 1); ++i) {
    a.prefix_groups = i == 0 ? (int32_t)groups[0] : 0;
    const dim3 grid((unsigned)(p.apart ? groups[i] : groups[0] + groups[1]));
    if (def)
      launch_shared<kTreeDefault>(a, p.row_waves[i], grid, s);
    else if (fast)
      launch_shared<kTreeFast>(a, p.row_waves[i], grid, s);
    else if (layout->int8_radii)
      launch_shared<kTreeAnyI8>(a, p.row_waves[i], grid, s);
    else
      launch_shared<kTreeAnyF16>(a, p.row_waves[i], grid, s);
  }
  const int32_t st = launch_status("tp_shared_attention");
  if (st != TP_OK || a.records == 1) return st;
  JoinArgs j{};
  j.o = a.part_o;
  j.ml = a.part_ml;
  j.out = a.out;
  j.rows = g;
  j.out_b = a.out_b, j.out_h = a.out_h;
  j.units = (int32_t)(batch * hkv), j.splits = a.records, j.g = g, j.hkv = hkv;
  return launch_join(j, false, true, s);
}
