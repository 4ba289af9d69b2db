// tp_select.hip -- which stored pages a query is likely to need.
//
// The bounds of a page are the smallest and the largest of each key component over its 64 tokens,
// lo_d <= k_d <= hi_d (of the keys r (cos a, sin a), fp32 products rounded to fp16; the page decoder rounds
// them in one step, which differs in the last bit where the fp32 product is a tie).  So no key of the page has a larger
// product with q than
//
//   u(q, page) = sum_d max(q_d lo_d, q_d hi_d),
//
// and a page's score is the largest u over the query heads of its group.  Selected are the first and the last
// pages asked for and those of the others with the largest scores, ties to the lower index, in ascending order.
//
// Scores are sums of exact products (fp16 by fp16 fits fp32) in fp64, so that two pages change places only if
// their scores differ by less than 2^-46 of their terms, whatever the order of the sum: which pages are attended
// does not depend on rounding.
#include <algorithm>

#include "tp_page_tiles.h"

namespace tp {

struct BoundsArgs {
  const void* radii;
  const uint16_t* radii_scales;
  const uint8_t* angle_l1;
  const uint8_t* angle_deep;
  int64_t capacity, bounds_capacity;
  int32_t page_begin, l1_bits, deep_bits, split_half, l1_row, deep_row;
  uint16_t* bounds;  // [bh][bounds_capacity][2][128]
};

constexpr int kBoundsThreads = 256;

// A workgroup a page.  Thread (c, t0) decodes pairs 8 c .. + 7 of tokens t0 and t0 + 32; the running bounds are
// joined over the wave's tokens by shuffles and over the waves in LDS.  Bound by the reads of the key fields.
template <bool I8>
__global__ __launch_bounds__(kBoundsThreads) void page_bounds_kernel(BoundsArgs a) {
  __shared__ float2v lut[512];
  __shared__ half2v side[4][2][kPairs];
  __shared__ float radius[I8 ? 256 : 1];  // of int8 codes, from -128 on, as the page decoder computes them
  const int tid = threadIdx.x, c = tid & 7, lane = tid & 63, wave = tid >> 6;
  const int64_t bh = blockIdx.y, page = (int64_t)a.page_begin + blockIdx.x, slot = bh * a.capacity + page;
  if (tid < (1 << a.l1_bits)) lut[tid] = angle_pair(tid, a.l1_bits);
  if (tid < (1 << a.deep_bits)) lut[256 + tid] = angle_pair(tid, a.deep_bits);
  if constexpr (I8) radius[tid] = expf((float)(tid - 128) * h2f(a.radii_scales[slot]));
  half2v lo[8], hi[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) lo[i] = half2v{(f16)INFINITY, (f16)INFINITY}, hi[i] = -lo[i];
  __syncthreads();
#pragma unroll
  for (int n = 0; n < 2; ++n) {
    const int64_t row = slot * kPageTokens + (tid >> 3) + 32 * n;
    float r[8];
    if constexpr (I8) {
      const uint2v w = *reinterpret_cast<const uint2v*>(static_cast<const int8_t*>(a.radii) + row * kPairs + 8 * c);
#pragma unroll
      for (int i = 0; i < 8; ++i) r[i] = radius[((w[i >> 2] >> (8 * (i & 3))) + 128u) & 0xffu];
    } else {
      const uint4v w = *reinterpret_cast<const uint4v*>(static_cast<const uint16_t*>(a.radii) + row * kPairs + 8 * c);
#pragma unroll
      for (int i = 0; i < 8; ++i) r[i] = h2f((uint16_t)(w[i >> 1] >> (16 * (i & 1))));
    }
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const int pair = 8 * c + i;
      const bool l1 = pair < a.split_half;
      const int bits = l1 ? a.l1_bits : a.deep_bits, bit = (l1 ? pair : pair - a.split_half) * bits;
      const uint32_t byte = l1 ? a.angle_l1[row * a.l1_row + (bit >> 3)] : a.angle_deep[row * a.deep_row + (bit >> 3)];
      const float2v cs = lut[(l1 ? 0u : 256u) + ((byte >> (bit & 7)) & ((1u << bits) - 1u))];
      // Rounded to fp16 before they are compared: rounding keeps the order.
      const half2v k = __builtin_convertvector((float2v{r[i] * cs.x, r[i] * cs.y}), half2v);
      lo[i] = __builtin_elementwise_min(lo[i], k), hi[i] = __builtin_elementwise_max(hi[i], k);
    }
  }
  auto other = [](half2v x, int d) { return __builtin_bit_cast(half2v, __shfl_xor(__builtin_bit_cast(int, x), d)); };
#pragma unroll
  for (int i = 0; i < 8; ++i)
#pragma unroll
    for (int d = 8; d < 64; d <<= 1) {
      lo[i] = __builtin_elementwise_min(lo[i], other(lo[i], d));
      hi[i] = __builtin_elementwise_max(hi[i], other(hi[i], d));
    }
  if (lane < 8)
#pragma unroll
    for (int i = 0; i < 8; ++i) side[wave][0][8 * c + i] = lo[i], side[wave][1][8 * c + i] = hi[i];
  __syncthreads();
  if (tid >= 128) return;
  const int which = tid >> 6, d = tid & 63;
  half2v x = side[0][which][d];
#pragma unroll
  for (int w = 1; w < 4; ++w)
    x = which ? __builtin_elementwise_max(x, side[w][1][d]) : __builtin_elementwise_min(x, side[w][0][d]);
  reinterpret_cast<half2v*>(a.bounds + (bh * a.bounds_capacity + page) * 2 * kHeadDim)[tid] = x;
}

struct SelectArgs {
  const uint16_t* q;       // [units][g][128]
  const uint16_t* bounds;  // [units][capacity][2][128]
  uint64_t* keys;          // [units][count]
  uint32_t* tickets;       // [units], 0 before and after
  int32_t* selected;       // [units][first + take + last]
  int64_t capacity;
  int32_t g, first, last, count, take, n_pages;  // scored: pages [first, first + count), of which `take` are selected
  uint32_t flip;                                 // negative scales: the queries' signs turned
};

constexpr int kSelectThreads = 512;
constexpr int kSelectWaves = kSelectThreads / 64;
constexpr int kScorePages = kSelectThreads / 8;
constexpr int kScoreHeads = 16;

// A score as a whole number of the same order.
__device__ __forceinline__ uint64_t score_key(double s) {
  s = s != s ? (double)INFINITY : s + 0.0;  // NaN (infinities of both signs): attended, as any infinity; -0 is 0
  const uint64_t u = __builtin_bit_cast(uint64_t, s);
  return u >> 63 ? ~u : u | (1ull << 63);
}

// The key of the thread's page: 8 lanes a page, 16 dimensions a lane, the group's queries in LDS.
__device__ __forceinline__ uint64_t page_key(const SelectArgs& a, int64_t unit, int page, int tid, float (*qs)[kHeadDim]) {
  const int c = tid & 7;
  const uint16_t* b = a.bounds + (unit * a.capacity + page) * 2 * kHeadDim + 16 * c;
  uint4v w[4];
#pragma unroll
  for (int j = 0; j < 4; ++j) w[j] = *reinterpret_cast<const uint4v*>(b + (j >> 1) * kHeadDim + 8 * (j & 1));
  double best = -INFINITY;
  bool any_nan = false;
  for (int h0 = 0; h0 < a.g; h0 += kScoreHeads) {
    const int heads = min(kScoreHeads, a.g - h0);
    __syncthreads();
    for (int x = tid; x < heads * kHeadDim; x += kSelectThreads)
      qs[0][x] = h2f((uint16_t)(a.q[(unit * a.g + h0) * kHeadDim + x] ^ a.flip));
    __syncthreads();
    for (int h = 0; h < heads; ++h) {
      double s = 0.0;
#pragma unroll
      for (int j = 0; j < 16; ++j) {
        const float x = qs[h][16 * c + j];
        const uint32_t lo = (w[j >> 3][(j >> 1) & 3] >> (16 * (j & 1))) & 0xffffu;
        const uint32_t hi = (w[2 + (j >> 3)][(j >> 1) & 3] >> (16 * (j & 1))) & 0xffffu;
        s += (double)fmaxf(x * h2f((uint16_t)lo), x * h2f((uint16_t)hi));
      }
#pragma unroll
      for (int d = 1; d < 8; d <<= 1) s += __shfl_xor(s, d);
      any_nan = any_nan || s != s;
      best = s > best ? s : best;
    }
  }
  return score_key(any_nan ? (double)INFINITY : best);
}

// A workgroup of each 64 pages of a (batch, kv head) scores them; the last of them to be done selects: the `take`-th
// largest key by its digits of 8 bits from the first in which the keys differ, then the pages above it, and the first
// of those that equal it, in their order.  PER: keys of a thread, held in registers (0: more, read anew each time).
// Keys go out and come back past the caches of the XCDs (agent scope), between them a ticket.
template <int PER>
__global__ __launch_bounds__(kSelectThreads) void select_pages_kernel(SelectArgs a) {
  __shared__ __align__(16) float qs[kScoreHeads][kHeadDim];
  __shared__ uint32_t hist[256];
  __shared__ uint64_t ends[2][kSelectWaves];
  __shared__ uint64_t found;
  __shared__ int32_t found_rest, found_all, is_last;
  __shared__ int32_t counts[2][kSelectWaves];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int64_t unit = blockIdx.y;
  uint64_t* keys = a.keys + unit * a.count;
  int32_t* out = a.selected + unit * (a.first + a.take + a.last);
  if (a.take > 0 && a.take < a.count) {
    const int i = (int)blockIdx.x * kScorePages + (tid >> 3);
    const uint64_t key = page_key(a, unit, a.first + min(i, a.count - 1), tid, qs);  // those past the last repeat it
    if ((tid & 7) == 0 && i < a.count) __hip_atomic_store(keys + i, key, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");  // the stores are where every XCD sees them
    __syncthreads();
    if (tid == 0)
      is_last = __hip_atomic_fetch_add(a.tickets + unit, 1u, __ATOMIC_ACQUIRE, __HIP_MEMORY_SCOPE_AGENT) + 1u == gridDim.x;
    __syncthreads();
    if (!is_last) return;
    if (tid == 0) __hip_atomic_store(a.tickets + unit, 0u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
  }
  for (int i = tid; i < a.first; i += kSelectThreads) out[i] = i;
  for (int i = tid; i < a.last; i += kSelectThreads) out[a.first + a.take + i] = a.n_pages - a.last + i;
  if (a.take == 0) return;
  out += a.first;
  if (a.take == a.count) {
    for (int i = tid; i < a.count; i += kSelectThreads) out[i] = a.first + i;
    return;
  }
  auto load = [&](int i) { return __hip_atomic_load(keys + i, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT); };
  uint64_t mine[PER ? PER : 1];
  if constexpr (PER)
#pragma unroll
    for (int j = 0; j < PER; ++j) mine[j] = load(min(tid + kSelectThreads * j, a.count - 1));
  auto each_key = [&](auto use) {
    if constexpr (PER) {
#pragma unroll
      for (int j = 0; j < PER; ++j)
        if (tid + kSelectThreads * j < a.count) use(mine[j]);
    } else {
      for (int i = tid; i < a.count; i += kSelectThreads) use(load(i));
    }
  };
  uint64_t low = ~0ull, high = 0;
  each_key([&](uint64_t k) {
    low = k < low ? k : low;
    high = k > high ? k : high;
  });
#pragma unroll
  for (int d = 1; d < 64; d <<= 1) {
    const uint64_t x = __shfl_xor((unsigned long long)low, d), y = __shfl_xor((unsigned long long)high, d);
    low = x < low ? x : low;
    high = y > high ? y : high;
  }
  if (lane == 0) ends[0][wave] = low, ends[1][wave] = high;
  __syncthreads();
  for (int w = 0; w < kSelectWaves; ++w) {
    low = ends[0][w] < low ? ends[0][w] : low;
    high = ends[1][w] > high ? ends[1][w] : high;
  }
  // Keys agree above bit `shift`; the digits found so far are `prefix`, the keys' bits from there on.
  int shift = low == high ? 0 : 64 - __builtin_clzll(low ^ high);
  uint64_t prefix = shift == 64 ? 0 : high >> shift;
  int32_t rest = a.take;
  bool all = false;  // whether every key with the prefix is taken
  while (shift > 0 && !all) {
    const int width = min(shift, 8), next = shift - width;
    if (tid < 256) hist[tid] = 0;
    __syncthreads();
    each_key([&](uint64_t k) {
      if (shift == 64 || (k >> shift) == prefix) atomicAdd(&hist[(uint32_t)(k >> next) & ((1u << width) - 1u)], 1u);
    });
    __syncthreads();
    if (wave == 0) {  // the digit in which the rest-th key from the top lies
      uint32_t n[4], sum = 0;
#pragma unroll
      for (int j = 0; j < 4; ++j) n[j] = hist[255 - 4 * lane - j], sum += n[j];
      uint32_t above = sum;
#pragma unroll
      for (int d = 1; d < 64; d <<= 1) {
        const uint32_t x = __shfl_up(above, d);
        above += lane >= d ? x : 0u;
      }
      above -= sum;
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        if (above < (uint32_t)rest && (uint32_t)rest <= above + n[j]) {
          found = (shift == 64 ? 0 : prefix << width) | (uint64_t)(255 - 4 * lane - j);
          found_rest = rest - (int32_t)above;
          found_all = n[j] == (uint32_t)rest - above;
        }
        above += n[j];
      }
    }
    __syncthreads();
    prefix = found;
    rest = found_rest;
    all = found_all != 0;
    shift = next;
  }
  // Above the prefix: taken; equal to it: the first `rest` of them (all of them where `all`).
  int32_t base = 0, equal_base = 0;
  auto place = [&](int i, uint64_t key) {
    const uint64_t k = key >> shift;
    const bool over = i < a.count && k > prefix, equal = i < a.count && k == prefix;
    const uint64_t equals = __ballot(equal), below = (1ull << lane) - 1ull;
    if (lane == 0) counts[0][wave] = __popcll(equals);
    __syncthreads();
    int32_t rank = equal_base + __popcll(equals & below), equal_all = 0;
    for (int w = 0; w < kSelectWaves; ++w) {
      rank += w < wave ? counts[0][w] : 0;
      equal_all += counts[0][w];
    }
    const bool taken = over || (equal && rank < rest);
    const uint64_t takes = __ballot(taken);
    if (lane == 0) counts[1][wave] = __popcll(takes);
    __syncthreads();
    int32_t at = base + __popcll(takes & below), taken_all = 0;
    for (int w = 0; w < kSelectWaves; ++w) {
      at += w < wave ? counts[1][w] : 0;
      taken_all += counts[1][w];
    }
    if (taken) out[at] = a.first + i;
    base += taken_all;
    equal_base += equal_all;
  };
  if constexpr (PER) {
#pragma unroll
    for (int j = 0; j < PER; ++j) place(tid + kSelectThreads * j, mine[j]);
  } else {
    for (int i0 = 0; i0 < a.count; i0 += kSelectThreads) place(i0 + tid, load(min(i0 + tid, a.count - 1)));
  }
}

}  // namespace tp

using namespace tp;

extern "C" int32_t tp_page_bounds(const tp_page_layout* layout, const tp_pages* pages, int64_t bh, int32_t page_begin,
                                  int32_t n_pages, void* bounds, int64_t bounds_capacity, void* stream) {
  clear_error();
  int l1_row = 0, deep_row = 0;
  if (!check_layout(layout, &l1_row, &deep_row)) return TP_ERR_UNSUPPORTED;
  if (bh < 1 || bh > 65535 || page_begin < 0 || n_pages < 0 || page_begin > INT32_MAX - n_pages) {
    set_error("bad page range: %lld rows (at most 65535), pages %d and the next %d", (long long)bh, page_begin, n_pages);
    return TP_ERR_INVALID;
  }
  if (n_pages == 0) return TP_OK;
  if (!pages || pages->capacity < page_begin + n_pages || bounds_capacity < page_begin + n_pages) {
    set_error("pages %d to %d exceed the pages' or the bounds' capacity", page_begin, page_begin + n_pages);
    return TP_ERR_INVALID;
  }
  if (!bounds || !pages->radii || (l1_row > 0 && !pages->angle_l1) || (deep_row > 0 && !pages->angle_deep) ||
      (layout->int8_radii && !pages->radii_scales)) {
    set_error("page buffers missing for this layout");
    return TP_ERR_INVALID;
  }
  if (((uintptr_t)pages->radii & 15u) || ((uintptr_t)bounds & 15u) || ((uintptr_t)pages->radii_scales & 1u)) {
    set_error("page buffers and bounds are not aligned");
    return TP_ERR_INVALID;
  }
  BoundsArgs a{};
  a.radii = pages->radii;
  a.radii_scales = static_cast<const uint16_t*>(pages->radii_scales);
  a.angle_l1 = pages->angle_l1, a.angle_deep = pages->angle_deep;
  a.capacity = pages->capacity, a.bounds_capacity = bounds_capacity;
  a.page_begin = page_begin;
  a.l1_bits = layout->l1_bits, a.deep_bits = layout->deep_bits, a.split_half = layout->split_dim / 2;
  a.l1_row = l1_row, a.deep_row = deep_row;
  a.bounds = static_cast<uint16_t*>(bounds);
  const dim3 grid((unsigned)n_pages, (unsigned)bh);
  hipStream_t s = static_cast<hipStream_t>(stream);
  if (layout->int8_radii)
    hipLaunchKernelGGL(page_bounds_kernel<true>, grid, dim3(kBoundsThreads), 0, s, a);
  else
    hipLaunchKernelGGL(page_bounds_kernel<false>, grid, dim3(kBoundsThreads), 0, s, a);
  return launch_status("tp_page_bounds");
}

extern "C" size_t tp_select_workspace_bytes(int64_t batch, int32_t hq, int32_t hkv, int32_t n_pages) {
  if (batch < 1 || hkv < 1 || hq < hkv || n_pages < 0) return 0;
  return tp_decode_counter_bytes(batch, hq, hkv) + (size_t)batch * hkv * n_pages * sizeof(uint64_t);
}

extern "C" int32_t tp_select_pages(const void* q, int64_t batch, int32_t hq, int32_t hkv, const void* bounds,
                                   int64_t bounds_capacity, int32_t n_pages, int32_t first, int32_t last, int32_t count,
                                   float scale, int32_t* selected, void* workspace, size_t workspace_bytes,
                                   void* stream) {
  clear_error();
  if (batch < 1 || hq < 1 || hkv < 1 || hq % hkv != 0 || batch > 65535 / hkv) {
    set_error("bad query shape: batch=%lld hq=%d hkv=%d (hq must be a multiple of hkv, batch * hkv at most 65535)",
              (long long)batch, hq, hkv);
    return TP_ERR_INVALID;
  }
  if (n_pages < 1 || bounds_capacity < n_pages || n_pages > INT32_MAX / 2) {
    set_error("n_pages=%d is not within the bounds' capacity", n_pages);
    return TP_ERR_INVALID;
  }
  if (first < 0 || last < 0 || count < 1 || count > n_pages || first > count || last > count - first) {
    set_error("cannot select %d of %d pages, the first %d and the last %d among them", count, n_pages, first, last);
    return TP_ERR_INVALID;
  }
  if (!(scale == scale) || scale - scale != 0.0f) {
    set_error("scale must be finite");
    return TP_ERR_INVALID;
  }
  if (!q || !bounds || !selected || ((uintptr_t)q & 1u) || ((uintptr_t)bounds & 15u) || ((uintptr_t)selected & 3u)) {
    set_error("q, bounds (16-byte aligned) and selected must be non-NULL buffers");
    return TP_ERR_INVALID;
  }
  const size_t need = tp_select_workspace_bytes(batch, hq, hkv, n_pages);
  if (!workspace || workspace_bytes < need || ((uintptr_t)workspace & 255u)) {
    set_error("workspace of %zu bytes (256-byte aligned) required, got %zu", need, workspace_bytes);
    return TP_ERR_WORKSPACE;
  }
  SelectArgs a{};
  a.q = static_cast<const uint16_t*>(q);
  a.bounds = static_cast<const uint16_t*>(bounds);
  a.tickets = static_cast<uint32_t*>(workspace);
  a.keys = reinterpret_cast<uint64_t*>(static_cast<char*>(workspace) + tp_decode_counter_bytes(batch, hq, hkv));
  a.selected = selected;
  a.capacity = bounds_capacity;
  a.g = hq / hkv, a.first = first, a.last = last, a.count = n_pages - first - last, a.take = count - first - last;
  a.n_pages = n_pages;
  a.flip = scale < 0.0f ? 0x8000u : 0u;
  const bool scored = a.take > 0 && a.take < a.count;
  const dim3 grid(scored ? (unsigned)((a.count + kScorePages - 1) / kScorePages) : 1u, (unsigned)(batch * hkv));
  hipStream_t s = static_cast<hipStream_t>(stream);
  if (a.count <= kSelectThreads)
    hipLaunchKernelGGL(select_pages_kernel<1>, grid, dim3(kSelectThreads), 0, s, a);
  else if (a.count <= 4 * kSelectThreads)
    hipLaunchKernelGGL(select_pages_kernel<4>, grid, dim3(kSelectThreads), 0, s, a);
  else
    hipLaunchKernelGGL(select_pages_kernel<0>, grid, dim3(kSelectThreads), 0, s, a);
  return launch_status("tp_select_pages");
}
