// tp_select.hip -- which stored pages a query is likely to need.
//
// The bounds of a page are the smallest and the largest of each key component over its 64 tokens,
// lo_d <= k_d <= hi_d (of the keys r (cos a, sin a), fp32 products rounded to fp16; the page decoder rounds
// them in one step, which differs in the last bit where the fp32 product is a tie).  So none of these keys has a larger
// product with q than
//
//   u(q, page) = sum_d max(q_d lo_d, q_d hi_d)
//
// (those that tp_selected_attention multiplies are not rounded so far, and their products may exceed it by half a step of
// fp16 of each component), and a page's score is the largest u over the query heads of its group.  Selected are the
// first and the last pages asked for and those of the others with the largest scores, ties to the lower index, in
// ascending order.
//
// Scores are sums of exact products (fp16 by fp16 fits fp32) in fp64, so that two pages change places only if
// their scores differ by less than 2^-46 of their terms, whatever the order of the sum: which pages are attended
// does not depend on rounding.
#include <algorithm>
#include <type_traits>

#include "tp_page_tiles.h"

namespace tp {

struct BoundsArgs {
  const void* radii;
  const uint16_t* radii_scales;
  const uint8_t* angle_l1;
  const uint8_t* angle_deep;
  int64_t capacity, bounds_capacity;
  int32_t page_begin, n_pages, l1_bits, deep_bits, split_half, l1_row, deep_row;
  uint16_t* bounds;  // [bh][bounds_capacity][2][128]
};

constexpr int kBoundsThreads = 256;

// A thread's part of a page's key fields: pairs 8 c .. + 7 of tokens t0 and t0 + 32.
template <int KIND>
struct BoundsRegs {
  uint4v r[tree_i8(KIND) ? 1 : 2];
  uint2v r8[tree_i8(KIND) ? 2 : 1];
  uint2v codes[2];  // the run's 8 codes, as bytes, or as nibbles in the first word
  uint32_t ls;
};

template <int KIND>
__device__ __forceinline__ void load_bounds(const BoundsArgs& a, int64_t slot, int tid, BoundsRegs<KIND>& p) {
  const int c = tid & 7;
#pragma unroll
  for (int n = 0; n < 2; ++n) {
    const int64_t row = slot * kPageTokens + (tid >> 3) + 32 * n;
    if constexpr (tree_i8(KIND))
      p.r8[n] = *reinterpret_cast<const uint2v*>(static_cast<const int8_t*>(a.radii) + row * kPairs + 8 * c);
    else
      p.r[n] = *reinterpret_cast<const uint4v*>(static_cast<const uint16_t*>(a.radii) + row * kPairs + 8 * c);
    if constexpr (KIND == kTreeDefault) {
      p.codes[n].x = *reinterpret_cast<const uint32_t*>((c < 4 ? a.angle_l1 : a.angle_deep) + row * 16 + 4 * (c & 3));
    } else if constexpr (KIND == kTreeFast) {
      p.codes[n] = *reinterpret_cast<const uint2v*>(a.angle_deep + row * kPairs + 8 * c);
    } else {
      uint32_t w[2] = {0u, 0u};
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const int pair = 8 * c + i;
        const bool l1 = pair < a.split_half;
        const int bits = l1 ? a.l1_bits : a.deep_bits, bit = (l1 ? pair : pair - a.split_half) * bits;
        const uint32_t byte = l1 ? a.angle_l1[row * a.l1_row + (bit >> 3)] : a.angle_deep[row * a.deep_row + (bit >> 3)];
        w[i >> 2] |= ((byte >> (bit & 7)) & ((1u << bits) - 1u)) << (8 * (i & 3));
      }
      p.codes[n] = uint2v{w[0], w[1]};
    }
  }
  if constexpr (tree_i8(KIND)) p.ls = a.radii_scales[slot];
}

// The smallest of a wave's lanes of one c (lane % 8) for 16 registers: a swap of half of the lanes of two registers
// joins them in one, which then holds the one's result in some lanes and the other's in the rest.  Register m of the
// four that remain holds, in row r = lane / 16, that of x[4 m + joined_register(r)].
__device__ __forceinline__ int joined_register(int row) { return ((row & 1) << 1) | (row >> 1); }
__device__ __forceinline__ void smallest_of_tokens(const half2v (&x)[16], half2v (&z)[4]) {
  auto smaller = [](uint32_t u, uint32_t w) {
    return __builtin_bit_cast(uint32_t, __builtin_elementwise_min(__builtin_bit_cast(half2v, u), __builtin_bit_cast(half2v, w)));
  };
  uint32_t y[8];
#pragma unroll
  for (int k = 0; k < 8; ++k) {
    const auto p = __builtin_amdgcn_permlane32_swap(__builtin_bit_cast(uint32_t, x[2 * k]),
                                                    __builtin_bit_cast(uint32_t, x[2 * k + 1]), false, false);
    y[k] = smaller(p[0], p[1]);
  }
#pragma unroll
  for (int m = 0; m < 4; ++m) {
    const auto p = __builtin_amdgcn_permlane16_swap(y[2 * m], y[2 * m + 1], false, false);
    const uint32_t w = smaller(p[0], p[1]);
    z[m] = __builtin_bit_cast(half2v, smaller(w, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)w, 0x128, 0xf, 0xf, true)));  // row_ror:8
  }
}

// A workgroup walks over pages of a (batch, head) row, one ahead in registers; the bounds are joined over the wave's
// tokens in registers and over the waves in LDS.  Every key field is read once, 10 KB a page of the default layout, and
// 512 bytes are written: 4,096 pages (512 of 8 rows, 44 MB) take 11.6 us, 3.8 TB/s, 5.1 of a copy's; bound by that and
// by the arithmetic, 8,192 products, roundings and comparisons a page (20.6 us with bytes read one by one and joined by
// shuffles, 16 with whole words and a page ahead).  128 pages take 3.3 us, mostly a launch.
template <int KIND>
__global__ __launch_bounds__(kBoundsThreads) void page_bounds_kernel(BoundsArgs a) {
  __shared__ TreeLut lut;
  __shared__ half2v side[2][4][2 * kPairs];  // smallest keys, then smallest negated keys
  __shared__ float radius[tree_i8(KIND) ? 2 : 1][tree_i8(KIND) ? 256 : 1];  // of int8 codes, from -128 on
  const int tid = threadIdx.x, c = tid & 7, lane = tid & 63, wave = tid >> 6;
  const int64_t bh = blockIdx.y;
  const int step = (int)gridDim.x;
  BoundsRegs<KIND> next;
  load_bounds<KIND>(a, bh * a.capacity + a.page_begin + blockIdx.x, tid, next);
  build_tree_lut<KIND, kBoundsThreads>(a, lut, tid);
  for (int i = blockIdx.x, buf = 0; i < a.n_pages; i += step, buf ^= 1) {
    const BoundsRegs<KIND> p = next;
    load_bounds<KIND>(a, bh * a.capacity + a.page_begin + min(i + step, a.n_pages - 1), tid, next);
    if constexpr (tree_i8(KIND)) radius[buf][tid] = expf((float)(tid - 128) * h2f((uint16_t)p.ls));
    if (tree_i8(KIND) || i == (int)blockIdx.x) lds_barrier();
    half2v x[16];
#pragma unroll
    for (int n = 0; n < 2; ++n)
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        float r;
        if constexpr (tree_i8(KIND))
          r = radius[buf][((p.r8[n][j >> 2] >> (8 * (j & 3))) + 128u) & 0xffu];
        else
          r = h2f((uint16_t)(p.r[n][j >> 1] >> (16 * (j & 1))));
        uint32_t code;
        if constexpr (KIND == kTreeDefault)
          code = (p.codes[n].x >> (4 * j)) & 15u;
        else
          code = (KIND == kTreeFast || 8 * c + j >= a.split_half ? 256u : 0u) + ((p.codes[n][j >> 2] >> (8 * (j & 3))) & 0xffu);
        const float2v cs = lut.code[code];
        // Rounded to fp16 before they are compared: rounding keeps the order.
        const half2v k = __builtin_convertvector((float2v{r * cs.x, r * cs.y}), half2v);
        x[j] = n ? __builtin_elementwise_min(x[j], k) : k;
        x[8 + j] = n ? __builtin_elementwise_min(x[8 + j], -k) : -k;
      }
    half2v z[4];
    smallest_of_tokens(x, z);
#pragma unroll
    for (int m = 0; m < 4; ++m) {
      const int at = 4 * m + joined_register(lane >> 4);
      if (!(lane & 8)) side[buf][wave][(at & 8) * (kPairs / 8) + 8 * c + (at & 7)] = z[m];
    }
    lds_barrier();
    if (tid < 2 * kPairs) {
      half2v y = side[buf][0][tid];
#pragma unroll
      for (int w = 1; w < 4; ++w) y = __builtin_elementwise_min(y, side[buf][w][tid]);
      reinterpret_cast<half2v*>(a.bounds + (bh * a.bounds_capacity + a.page_begin + i) * 2 * kHeadDim)[tid] = tid < kPairs ? y : -y;
    }
  }
}

struct SelectArgs {
  const uint16_t* q;       // [units][g][128]
  const uint16_t* bounds;  // [units][capacity][2][128]
  uint64_t* keys;          // [units][count]
  uint32_t* tickets;       // one of each row of the launch, 0 before and after
  int32_t* selected;       // [units][first + take + last]
  int64_t capacity;
  int32_t first_unit;
  int32_t g, first, last, count, take, n_pages;  // scored: pages [first, first + count), of which `take` are selected
  uint32_t flip;                                 // negative scales: the queries' signs turned
};

constexpr int kSelectThreads = 512;
constexpr int kSelectWaves = kSelectThreads / 64;
constexpr int kScorePages = kSelectThreads / 8;
constexpr int kScoreHeads = 16;
// Rows of a launch: as many as the counter area of the smallest workspace has tickets for.  What lies behind it is other
// calls' keys and records, so a row's ticket never does.
constexpr int64_t kTicketRows = 65536 / sizeof(uint32_t);

// A score as a whole number of the same order.
__device__ __forceinline__ uint64_t score_key(double s) {
  s = s != s ? (double)INFINITY : s + 0.0;  // NaN (infinities of both signs): attended, as any infinity; -0 is 0
  const uint64_t u = __builtin_bit_cast(uint64_t, s);
  return u >> 63 ? ~u : u | (1ull << 63);
}

template <int CTRL>
__device__ __forceinline__ double moved(double x) {
  const uint64_t u = __builtin_bit_cast(uint64_t, x);
  const uint32_t lo = (uint32_t)__builtin_amdgcn_update_dpp(0, (int)u, CTRL, 0xf, 0xf, true);
  const uint32_t hi = (uint32_t)__builtin_amdgcn_update_dpp(0, (int)(u >> 32), CTRL, 0xf, 0xf, true);
  return __builtin_bit_cast(double, (uint64_t)hi << 32 | lo);
}

// The key of the thread's page: 8 lanes a page, 16 dimensions a lane, the group's queries in LDS.  Two heads at a time,
// whose sums are chains of their own, joined by lane moves: 16 rows of 32/8 heads and 2,045 pages (134 MB of bounds) 57
// us against 68 with one head and shuffles.
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
#pragma unroll 2
    for (int h = 0; h < heads; ++h) {
      double s = 0.0;
#pragma unroll
      for (int j = 0; j < 16; ++j) {
        const float x = qs[h][16 * c + j];
        const uint32_t lo = (w[j >> 3][(j >> 1) & 3] >> (16 * (j & 1))) & 0xffffu;
        const uint32_t hi = (w[2 + (j >> 3)][(j >> 1) & 3] >> (16 * (j & 1))) & 0xffffu;
        s += (double)fmaxf(x * h2f((uint16_t)lo), x * h2f((uint16_t)hi));  // of 0 times infinity, NaN, and a number: that
      }
      s += moved<0xb1>(s);   // quad_perm 1 0 3 2
      s += moved<0x4e>(s);   // quad_perm 2 3 0 1
      s += moved<0x141>(s);  // row_half_mirror: a lane of the other four
      any_nan = any_nan || s != s;
      best = s > best ? s : best;
    }
  }
  return score_key(any_nan ? (double)INFINITY : best);
}

// The sum over lanes 0 .. this one.
__device__ __forceinline__ uint32_t wave_sum_up_to(uint32_t x) {
  auto add = [&](auto ctrl, auto rows) {
    x += (uint32_t)__builtin_amdgcn_update_dpp(0, (int)x, decltype(ctrl)::value, decltype(rows)::value, 0xf, false);
  };
  using std::integral_constant;
  add(integral_constant<int, 0x111>(), integral_constant<int, 0xf>());  // row_shr:1, 2, 4, 8
  add(integral_constant<int, 0x112>(), integral_constant<int, 0xf>());
  add(integral_constant<int, 0x114>(), integral_constant<int, 0xf>());
  add(integral_constant<int, 0x118>(), integral_constant<int, 0xf>());
  add(integral_constant<int, 0x142>(), integral_constant<int, 0xa>());  // row_bcast:15, to rows 1 and 3
  add(integral_constant<int, 0x143>(), integral_constant<int, 0xc>());  // row_bcast:31, to rows 2 and 3
  return x;
}

// All lanes' bits, in every lane.
__device__ __forceinline__ uint32_t wave_or(uint32_t x) {
  x |= (uint32_t)__builtin_amdgcn_update_dpp(0, (int)x, 0x121, 0xf, 0xf, true);  // row_ror:1, 2, 4, 8
  x |= (uint32_t)__builtin_amdgcn_update_dpp(0, (int)x, 0x122, 0xf, 0xf, true);
  x |= (uint32_t)__builtin_amdgcn_update_dpp(0, (int)x, 0x124, 0xf, 0xf, true);
  x |= (uint32_t)__builtin_amdgcn_update_dpp(0, (int)x, 0x128, 0xf, 0xf, true);
  const auto p = __builtin_amdgcn_permlane16_swap(x, x, false, false);
  const uint32_t y = p[0] | p[1];
  const auto q = __builtin_amdgcn_permlane32_swap(y, y, false, false);
  return q[0] | q[1];
}

// A workgroup of each 64 pages of a (batch, kv head) scores them; the last of them to be done selects: the `take`-th
// largest key by its digits of 8 bits from the first in which the keys differ, then the pages above it, and the first
// of those that equal it, in their order.  PER: keys of a thread, held in registers (0: more, read anew each time).
// Keys go out and come back past the caches of the XCDs (agent scope), between them a ticket.
// Bound by its latencies: for one sequence of 32/8 heads 513 pages take 6.7 us, 2,045 pages (8.4 MB of bounds, 1.6 us
// of a copy's time) 10.7, 4,096 17.5 and 8,192 30.6, of which the last workgroup's selection is 2 us a thousand pages;
// two launches, one to score and one to select, took 11.2 and 14.8 us for the first two.  Keys in registers against
// PER 0, us: 4,096 pages 17.5 (PER 8), 20.8 (16), 21.9; 8,192 30.6 (16), 41.0; 2,100 13.2 (8), 16.1 (16).
template <int PER>
__global__ __launch_bounds__(kSelectThreads) void select_pages_kernel(SelectArgs a) {
  __shared__ __align__(16) float qs[kScoreHeads][kHeadDim];
  __shared__ uint32_t hist[256];
  __shared__ uint32_t ends[2][kSelectWaves];
  __shared__ uint64_t found;
  __shared__ int32_t found_rest, found_all, is_last;
  __shared__ int32_t counts[2][PER ? PER : 2][kSelectWaves];  // pages above the prefix, and equal to it
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int64_t unit = a.first_unit + (int64_t)blockIdx.y;
  uint32_t* ticket = a.tickets + blockIdx.y;
  uint64_t* keys = a.keys + unit * a.count;
  int32_t* out = a.selected + unit * (a.first + a.take + a.last);
  if (a.take > 0 && a.take < a.count) {
    const int i = (int)blockIdx.x * kScorePages + (tid >> 3);
    const uint64_t key = page_key(a, unit, a.first + min(i, a.count - 1), tid, qs);  // those past the last repeat it
    if ((tid & 7) == 0 && i < a.count) __hip_atomic_store(keys + i, key, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");  // the stores are where every XCD sees them
    __syncthreads();
    if (tid == 0)
      is_last = __hip_atomic_fetch_add(ticket, 1u, __ATOMIC_ACQUIRE, __HIP_MEMORY_SCOPE_AGENT) + 1u == gridDim.x;
    __syncthreads();
    if (!is_last) return;
    if (tid == 0) __hip_atomic_store(ticket, 0u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
  }
  if (tid < 256) hist[tid] = 0;
  for (int i = tid; i < a.first; i += kSelectThreads) out[i] = i;
  for (int i = tid; i < a.last; i += kSelectThreads) out[a.first + a.take + i] = a.n_pages - a.last + i;
  if (a.take == 0) return;
  out += a.first;
  if (a.take == a.count) {
    for (int i = tid; i < a.count; i += kSelectThreads) out[i] = a.first + i;
    return;
  }
  __syncthreads();
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
  const uint64_t one = load(0);
  uint64_t differ = 0;
  each_key([&](uint64_t k) { differ |= k ^ one; });
  const uint32_t differ_lo = wave_or((uint32_t)differ), differ_hi = wave_or((uint32_t)(differ >> 32));
  if (lane == 0) ends[0][wave] = differ_lo, ends[1][wave] = differ_hi;
  __syncthreads();
  differ = 0;
  for (int w = 0; w < kSelectWaves; ++w) differ |= (uint64_t)ends[1][w] << 32 | ends[0][w];
  // Keys agree above bit `shift`; the digits found so far are `prefix`, the keys' bits from there on.
  int shift = differ ? 64 - __builtin_clzll(differ) : 0;
  uint64_t prefix = shift == 64 ? 0 : one >> shift;
  int32_t rest = a.take;
  bool all = false;  // whether every key with the prefix is taken
  while (shift > 0 && !all) {
    const int width = min(shift, 8), next = shift - width;
    each_key([&](uint64_t k) {
      if (shift == 64 || (k >> shift) == prefix) atomicAdd(&hist[(uint32_t)(k >> next) & ((1u << width) - 1u)], 1u);
    });
    __syncthreads();
    if (wave == 0) {  // the digit in which the rest-th key from the top lies
      uint32_t n[4], sum = 0;
#pragma unroll
      for (int j = 0; j < 4; ++j) n[j] = hist[255 - 4 * lane - j], sum += n[j];
      uint32_t above = wave_sum_up_to(sum);
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
    if (shift > 0 && !all) {
      if (tid < 256) hist[tid] = 0;
      __syncthreads();
    }
  }
  // Above the prefix: taken; equal to it: the first `rest` of them (all of them where `all`).
  const uint64_t below = (1ull << lane) - 1ull;
  auto compare = [&](int i, uint64_t key, uint64_t& over, uint64_t& equal) {
    const uint64_t k = key >> shift;
    over = __ballot(i < a.count && k > prefix);
    equal = __ballot(i < a.count && k == prefix);
  };
  // Page i, with `over` and `equal` the wave's, and how many of either lie before the wave.
  auto place = [&](int i, uint64_t over, uint64_t equal, int32_t overs, int32_t equals) {
    overs += __popcll(over & below);
    equals += __popcll(equal & below);
    const bool is_equal = (equal >> lane) & 1u;
    if (((over >> lane) & 1u) || (is_equal && equals < rest)) out[overs + min(equals, rest)] = a.first + i;
  };
  if constexpr (PER) {
    uint64_t over[PER], equal[PER];
#pragma unroll
    for (int j = 0; j < PER; ++j) {
      compare(tid + kSelectThreads * j, mine[j], over[j], equal[j]);
      if (lane == 0) counts[0][j][wave] = __popcll(over[j]), counts[1][j][wave] = __popcll(equal[j]);
    }
    __syncthreads();
    int32_t overs = 0, equals = 0;
#pragma unroll
    for (int j = 0; j < PER; ++j) {
      int32_t before[2] = {overs, equals};
      for (int w = 0; w < kSelectWaves; ++w) {
        const int32_t x = counts[0][j][w], y = counts[1][j][w];
        before[0] += w < wave ? x : 0, before[1] += w < wave ? y : 0;
        overs += x, equals += y;
      }
      place(tid + kSelectThreads * j, over[j], equal[j], before[0], before[1]);
    }
  } else {
    int32_t overs = 0, equals = 0;
    for (int i0 = 0, buf = 0; i0 < a.count; i0 += kSelectThreads, buf ^= 1) {
      uint64_t over, equal;
      compare(i0 + tid, load(min(i0 + tid, a.count - 1)), over, equal);
      if (lane == 0) counts[0][buf][wave] = __popcll(over), counts[1][buf][wave] = __popcll(equal);
      __syncthreads();
      int32_t before[2] = {overs, equals};
      for (int w = 0; w < kSelectWaves; ++w) {
        const int32_t x = counts[0][buf][w], y = counts[1][buf][w];
        before[0] += w < wave ? x : 0, before[1] += w < wave ? y : 0;
        overs += x, equals += y;
      }
      place(i0 + tid, over, equal, before[0], before[1]);
    }
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
  a.n_pages = n_pages;
  // As many workgroups as the GPU holds, eight a CU.
  const int64_t most = std::max<int64_t>(1, 2048 / bh);
  const dim3 grid((unsigned)std::min<int64_t>(n_pages, most), (unsigned)bh);
  hipStream_t s = static_cast<hipStream_t>(stream);
  // The runtime's two layouts; their code words are read whole.
  const bool def = !layout->int8_radii && layout->l1_bits == 4 && layout->deep_bits == 4 && layout->split_dim == 64 &&
                   !(((uintptr_t)pages->angle_l1 | (uintptr_t)pages->angle_deep) & 3u);
  const bool fast = layout->int8_radii && layout->deep_bits == 8 && layout->split_dim == 0 && !((uintptr_t)pages->angle_deep & 7u);
  if (def)
    hipLaunchKernelGGL(page_bounds_kernel<kTreeDefault>, grid, dim3(kBoundsThreads), 0, s, a);
  else if (fast)
    hipLaunchKernelGGL(page_bounds_kernel<kTreeFast>, grid, dim3(kBoundsThreads), 0, s, a);
  else if (layout->int8_radii)
    hipLaunchKernelGGL(page_bounds_kernel<kTreeAnyI8>, grid, dim3(kBoundsThreads), 0, s, a);
  else
    hipLaunchKernelGGL(page_bounds_kernel<kTreeAnyF16>, grid, dim3(kBoundsThreads), 0, s, a);
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
  if (n_pages < 1 || bounds_capacity < n_pages || n_pages > INT32_MAX / 8) {  // 8 threads a page, less than 2^32 a launch
    set_error("n_pages=%d is not within the bounds' capacity, or past 2^28", n_pages);
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
  hipStream_t s = static_cast<hipStream_t>(stream);
  int32_t st = TP_OK;
  for (int64_t unit = 0; unit < batch * hkv && st == TP_OK; unit += kTicketRows) {
    a.first_unit = (int32_t)unit;
    const dim3 grid(scored ? (unsigned)((a.count + kScorePages - 1) / kScorePages) : 1u,
                    (unsigned)std::min(kTicketRows, batch * hkv - unit));
    if (a.count <= kSelectThreads)
      hipLaunchKernelGGL(select_pages_kernel<1>, grid, dim3(kSelectThreads), 0, s, a);
    else if (a.count <= 4 * kSelectThreads)
      hipLaunchKernelGGL(select_pages_kernel<4>, grid, dim3(kSelectThreads), 0, s, a);
    else if (a.count <= 8 * kSelectThreads)
      hipLaunchKernelGGL(select_pages_kernel<8>, grid, dim3(kSelectThreads), 0, s, a);
    else if (a.count <= 16 * kSelectThreads)
      hipLaunchKernelGGL(select_pages_kernel<16>, grid, dim3(kSelectThreads), 0, s, a);
    else
      hipLaunchKernelGGL(select_pages_kernel<0>, grid, dim3(kSelectThreads), 0, s, a);
    st = launch_status("tp_select_pages");
  }
  return st;
}
