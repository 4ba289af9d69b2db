// tp_rotate.hip -- queries and keys turned by their positions, on their way into a cache.
//
//   y_a = x_a cos_a - x_b sin_a,  y_b = x_b cos_b + x_a sin_b
//
// over the pairs (a, b) = (d, d + 64), or (2 d, 2 d + 1) interleaved.  Queries and keys are rounded to fp16,
// values cast to it; keys and values go straight to where the cache wants them (its dense tail, or a
// [batch][heads][tokens] buffer that the page encoder reads next), whatever the projections' strides.
//
// A result is the rounding of the exact sum: a page's codes are chosen from these keys, so that whoever turns
// the same keys gets the same codes.  With tables and inputs of 16 bits the products are exact in fp32 and one
// FMA rounds their sum; with 32 bits on either side they are exact in fp64.  Then fp32, then fp16, as a cast does.
#include <algorithm>

#include "tp_common.h"

namespace tp {

typedef uint32_t uint4v __attribute__((ext_vector_type(4)));

enum RotateType { kRotF16 = 0, kRotF32 = 1, kRotBF16 = 2 };

struct RotateArgs {
  const char* q;
  const char* k;
  const char* v;
  const char* cos;
  const char* sin;
  uint16_t* q_out;
  uint16_t* k_out;
  uint16_t* v_out;
  int64_t q_b, q_h, q_t, k_b, k_h, k_t, v_b, v_h, v_t;  // elements
  int64_t c_b, c_t, o_b, o_h, o_t;
  int64_t kv_row, kv_pos;  // tokens between (batch, head) rows of k_out and v_out, and of their first one
  int32_t hq, hkv, columns;
  int64_t tokens;
  int64_t first;  // token of the launch's first workgroup, rows counted one behind the other
  uint32_t* flag;
  uint32_t epoch;
  int32_t check, reports;
};

template <int TYPE>
__device__ __forceinline__ void load8(const char* base, int64_t at, float* x) {
  if constexpr (TYPE == kRotF32) {
    const float4v lo = *reinterpret_cast<const float4v*>(base + at * 4);
    const float4v hi = *reinterpret_cast<const float4v*>(base + at * 4 + 16);
#pragma unroll
    for (int i = 0; i < 4; ++i) x[i] = lo[i], x[4 + i] = hi[i];
  } else {
    const uint4v w = *reinterpret_cast<const uint4v*>(base + at * 2);
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const uint32_t h = (w[i >> 1] >> (16 * (i & 1))) & 0xffffu;
      x[i] = TYPE == kRotF16 ? h2f((uint16_t)h) : __uint_as_float(h << 16);
    }
  }
}

// x c + y s of one component, s with its sign.
template <bool WIDE>
__device__ __forceinline__ float turn(float x, float c, float y, float s) {
  if constexpr (WIDE)
    return (float)__builtin_fma((double)y, (double)s, (double)x * (double)c);
  else
    return __builtin_fmaf(y, s, x * c);
}

__device__ __forceinline__ uint4v pack8(const float* y) {
  uint4v w;
#pragma unroll
  for (int i = 0; i < 4; ++i) w[i] = (uint32_t)f2h(y[2 * i]) | ((uint32_t)f2h(y[2 * i + 1]) << 16);
  return w;
}

__device__ __forceinline__ bool any_nonfinite(uint4v w) {
  bool bad = false;
#pragma unroll
  for (int i = 0; i < 4; ++i) bad = bad || (w[i] & 0x7c00u) == 0x7c00u || (w[i] & 0x7c000000u) == 0x7c000000u;
  return bad;
}

// A workgroup a token: 8 lanes share a head's row, each with 8 dimensions of either half of it (or 16 in a row),
// and walk over the heads, 32 at a time, so that the token's tables are read once.  Every element is read and written
// once: bound by that.  4,100 tokens of 32/8 heads in bf16 (103 MB) take 18.2 us, 5.65 TB/s (partly in the caches);
// 32,773 in fp16 with fp32 tables (839 MB) 175 us, 4.8 TB/s, where a copy reaches 5.1; a token 4 us, a launch's.  No faster:
// accesses past the caches (187 us), runs of neighbouring tokens on one XCD (172 to 177).
constexpr int kRotThreads = 256;
constexpr int kRotRows = kRotThreads / 8;
constexpr int64_t kRotLaunch = 1 << 23;  // tokens of a launch: a grid holds less than 2^32 threads

template <int TYPE, int TABLE, bool INTER>
__global__ __launch_bounds__(kRotThreads) void rotate_tokens_kernel(RotateArgs a) {
  constexpr bool WIDE = TYPE == kRotF32 || TABLE == kRotF32;
  const int c = threadIdx.x & 7, slot = threadIdx.x >> 3;
  const int64_t index = a.first + blockIdx.x, b = index / a.tokens, t = index - b * a.tokens;
  const int lo = INTER ? 16 * c : 8 * c, hi = INTER ? 16 * c + 8 : kHeadDim / 2 + 8 * c;
  float cl[8], ch[8], sl[8], sh[8];
  const int64_t row = b * a.c_b + t * a.c_t;
  if (a.columns == kHeadDim) {
    load8<TABLE>(a.cos, row + lo, cl);
    load8<TABLE>(a.cos, row + hi, ch);
    load8<TABLE>(a.sin, row + lo, sl);
    load8<TABLE>(a.sin, row + hi, sh);
  } else {  // one column a pair
    float x[8], y[8];
    load8<TABLE>(a.cos, row + 8 * c, x);
    load8<TABLE>(a.sin, row + 8 * c, y);
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      cl[i] = INTER ? x[i >> 1] : x[i];
      ch[i] = INTER ? x[4 + (i >> 1)] : x[i];
      sl[i] = INTER ? y[i >> 1] : y[i];
      sh[i] = INTER ? y[4 + (i >> 1)] : y[i];
    }
  }
  bool bad = false;
  const int heads = a.hq + 2 * a.hkv;
  for (int h = slot; h < heads; h += kRotRows) {
    const bool is_q = h < a.hq, is_v = h >= a.hq + a.hkv;
    const int64_t head = is_q ? h : is_v ? h - a.hq - a.hkv : h - a.hq;
    const char* from = is_q ? a.q : is_v ? a.v : a.k;
    const int64_t at = is_q   ? b * a.q_b + head * a.q_h + t * a.q_t
                       : is_v ? b * a.v_b + head * a.v_h + t * a.v_t
                              : b * a.k_b + head * a.k_h + t * a.k_t;
    float x[8], y[8];
    load8<TYPE>(from, at + lo, x);
    load8<TYPE>(from, at + hi, y);
    if (!is_v) {
      float u[8], w[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        if constexpr (INTER) {
          const int o = i ^ 1;
          u[i] = turn<WIDE>(x[i], cl[i], x[o], i & 1 ? sl[i] : -sl[i]);
          w[i] = turn<WIDE>(y[i], ch[i], y[o], i & 1 ? sh[i] : -sh[i]);
        } else {
          u[i] = turn<WIDE>(x[i], cl[i], y[i], -sl[i]);
          w[i] = turn<WIDE>(y[i], ch[i], x[i], sh[i]);
        }
      }
#pragma unroll
      for (int i = 0; i < 8; ++i) x[i] = u[i], y[i] = w[i];
    }
    const uint4v pl = pack8(x), ph = pack8(y);
    uint16_t* to;
    if (is_q) {
      to = a.q_out + b * a.o_b + head * a.o_h + t * a.o_t;
    } else {
      to = (is_v ? a.v_out : a.k_out) + ((b * a.hkv + head) * a.kv_row + a.kv_pos + t) * kHeadDim;
      bad = bad || any_nonfinite(pl) || any_nonfinite(ph);
    }
    *reinterpret_cast<uint4v*>(to + lo) = pl;
    *reinterpret_cast<uint4v*>(to + hi) = ph;
  }
  if (!a.check) return;
  // Each workgroup reports its verdict on a line of its own once its reads and writes are issued, and the host
  // polls them; or, where there are more than lines or than a launch's, only a non-finite value.
  const bool any_bad = __syncthreads_or(bad);
  if (threadIdx.x != 0) return;
  if (a.reports)
    __hip_atomic_store(a.flag + (int64_t)kReportStride * blockIdx.x, any_bad ? a.epoch + 1u : a.epoch, __ATOMIC_RELEASE,
                       __HIP_MEMORY_SCOPE_SYSTEM);
  else if (any_bad)
    __hip_atomic_store(a.flag, a.epoch + 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_SYSTEM);
}

template <int TYPE, int TABLE>
static void launch_rotate(const RotateArgs& a, bool interleaved, dim3 grid, hipStream_t s) {
  if (interleaved)
    hipLaunchKernelGGL((rotate_tokens_kernel<TYPE, TABLE, true>), grid, dim3(kRotThreads), 0, s, a);
  else
    hipLaunchKernelGGL((rotate_tokens_kernel<TYPE, TABLE, false>), grid, dim3(kRotThreads), 0, s, a);
}

// The verdict of `n` workgroups that report one word each.
static int32_t wait_reports(const uint32_t* flag, uint32_t epoch, int64_t n, hipStream_t s) {
  const volatile uint32_t* vf = flag;
  bool done = false, bad = false;
  const int64_t spins = (1 << 22) / (1 + n);
  for (int64_t spin = 0; spin < spins && !done; ++spin) {
    done = true, bad = false;
    for (int64_t i = 0; i < n; ++i) {
      const uint32_t w = vf[kReportStride * i];
      done = done && (w == epoch || w == epoch + 1u);
      bad = bad || w == epoch + 1u;
    }
  }
  if (!done) {
    if (hipStreamSynchronize(s) != hipSuccess) {
      set_error("tp_rotate_tokens: synchronising the stream failed");
      return TP_ERR_HIP;
    }
    bad = false;
    for (int64_t i = 0; i < n; ++i) bad = bad || vf[kReportStride * i] == epoch + 1u;
  }
  if (bad) {
    set_error("append() inputs must contain finite values");
    return TP_ERR_NONFINITE;
  }
  return TP_OK;
}

}  // namespace tp

using namespace tp;

extern "C" int32_t tp_rotate_tokens(const void* q, const void* k, const void* v, int32_t dtype, int64_t batch,
                                    int32_t hq, int32_t hkv, int64_t tokens, const int64_t* strides, const void* cos,
                                    const void* sin, int32_t table_dtype, int32_t columns, const int64_t* table_strides,
                                    int32_t interleaved, void* q_out, const int64_t* q_out_strides, void* k_out,
                                    void* v_out, int64_t out_tokens, int64_t out_pos, int32_t check, uint32_t* flag,
                                    int64_t flag_words, uint32_t epoch, void* stream) {
  clear_error();
  if (dtype < 0 || dtype > 2 || (table_dtype != dtype && table_dtype != kRotF32)) {
    set_error("dtype must be 0 (fp16), 1 (fp32) or 2 (bf16) and the tables' the same or 1, got %d and %d", dtype,
              table_dtype);
    return TP_ERR_INVALID;
  }
  if (batch < 1 || hq < 1 || hkv < 1 || tokens < 0 || hq > INT32_MAX / 4 || hkv > INT32_MAX / 4 ||
      (tokens > 0 && batch > INT32_MAX / tokens)) {
    set_error("bad shape: batch=%lld hq=%d hkv=%d tokens=%lld (at most 2^31 tokens in all)", (long long)batch, hq, hkv,
              (long long)tokens);
    return TP_ERR_INVALID;
  }
  if (columns != kHeadDim && columns != kHeadDim / 2) {
    set_error("tables must have 64 or 128 columns, got %d", columns);
    return TP_ERR_INVALID;
  }
  if (out_pos < 0 || out_tokens < 0 || out_pos > out_tokens - tokens) {
    set_error("%lld tokens do not fit at %lld of %lld", (long long)tokens, (long long)out_pos, (long long)out_tokens);
    return TP_ERR_INVALID;
  }
  if ((check != 0 && check != 2) || (check && (!flag || (epoch & 1u) || flag_words < 1))) {
    set_error("check must be 0, or 2 with a pinned host flag and an even epoch");
    return TP_ERR_INVALID;
  }
  if (tokens == 0) return TP_OK;
  const uintptr_t all = (uintptr_t)q | (uintptr_t)k | (uintptr_t)v | (uintptr_t)cos | (uintptr_t)sin | (uintptr_t)q_out |
                        (uintptr_t)k_out | (uintptr_t)v_out;
  if (!q || !k || !v || !cos || !sin || !q_out || !k_out || !v_out || (all & 15u)) {
    set_error("q, k, v, the tables and the outputs must be non-NULL 16-byte aligned buffers");
    return TP_ERR_INVALID;
  }
  if (!strides || !table_strides || !q_out_strides) {
    set_error("strides are NULL");
    return TP_ERR_INVALID;
  }
  for (int i = 0; i < 14; ++i) {
    const int64_t s = i < 9 ? strides[i] : i < 11 ? table_strides[i - 9] : q_out_strides[i - 11];
    if (s < 0 || (s & 7)) {
      set_error("strides must be non-negative multiples of 8 elements");
      return TP_ERR_INVALID;
    }
  }
  RotateArgs a{};
  a.q = static_cast<const char*>(q), a.k = static_cast<const char*>(k), a.v = static_cast<const char*>(v);
  a.cos = static_cast<const char*>(cos), a.sin = static_cast<const char*>(sin);
  a.q_out = static_cast<uint16_t*>(q_out), a.k_out = static_cast<uint16_t*>(k_out), a.v_out = static_cast<uint16_t*>(v_out);
  int64_t* const to[9] = {&a.q_b, &a.q_h, &a.q_t, &a.k_b, &a.k_h, &a.k_t, &a.v_b, &a.v_h, &a.v_t};
  for (int i = 0; i < 9; ++i) *to[i] = strides[i];
  a.c_b = table_strides[0], a.c_t = table_strides[1];
  a.o_b = q_out_strides[0], a.o_h = q_out_strides[1], a.o_t = q_out_strides[2];
  a.kv_row = out_tokens, a.kv_pos = out_pos;
  a.hq = hq, a.hkv = hkv, a.columns = columns, a.tokens = tokens;
  a.flag = flag, a.epoch = epoch, a.check = check;
  const int64_t groups = batch * tokens;
  a.reports = groups <= std::min(flag_words / kReportStride, kRotLaunch);
  hipStream_t s = static_cast<hipStream_t>(stream);
  const bool inter = interleaved != 0;
  int32_t st = TP_OK;
  for (; a.first < groups && st == TP_OK; a.first += kRotLaunch) {
    const dim3 grid((unsigned)std::min(kRotLaunch, groups - a.first));
    if (dtype == kRotF32)
      launch_rotate<kRotF32, kRotF32>(a, inter, grid, s);
    else if (dtype == kRotF16 && table_dtype == kRotF16)
      launch_rotate<kRotF16, kRotF16>(a, inter, grid, s);
    else if (dtype == kRotF16)
      launch_rotate<kRotF16, kRotF32>(a, inter, grid, s);
    else if (table_dtype == kRotBF16)
      launch_rotate<kRotBF16, kRotBF16>(a, inter, grid, s);
    else
      launch_rotate<kRotBF16, kRotF32>(a, inter, grid, s);
    st = launch_status("tp_rotate_tokens");
  }
  if (st != TP_OK || !check) return st;
  return a.reports ? wait_reports(flag, epoch, groups, s) : wait_verdict(flag, epoch, s, false, "tp_rotate_tokens");
}
