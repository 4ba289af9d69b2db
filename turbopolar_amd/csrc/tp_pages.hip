// tp_pages.hip -- pages of a cache copied into another one, and drafted tokens taken into its tail.
//
// Both move bytes and compute nothing, so a copy is bound by HBM (each kept byte read and
// written once) and the taking of a few tokens by its launch.
#include <algorithm>

#include "tp_common.h"

namespace tp {

typedef uint32_t uint4v __attribute__((ext_vector_type(4)));

constexpr int kCopyBuffers = 8;
constexpr int kCopyIndex = 768;  // index entries that travel with the launch
struct CopyArgs {
  struct Buffer {
    const char* src;
    char* dst;
    int64_t page_bytes;
  } wide[kCopyBuffers], narrow[kCopyBuffers];  // of 16-byte chunks; of any size
  int32_t first[kCopyBuffers + 1];             // first chunk of each wide buffer's page, and the end
  int32_t n_wide, n_narrow;
  int64_t src_capacity, dst_capacity;
  int32_t heads, batch_in, n_stored, keep;
  const int32_t* rows;   // source batch row of each copied one (NULL: the same)
  const int32_t* pages;  // source page of each copied one (NULL: the same)
  int32_t rows_at, pages_at;  // where they begin in `index` instead (-1: they do not)
  int32_t index[kCopyIndex];
  const char* tail_k;
  const char* tail_v;
  char* tail_k_out;
  char* tail_v_out;
  int64_t tail_bytes, tail_row;  // copied of each row, and between rows
};

// One workgroup a page slot of a (batch, head) row, over all of its buffers as one run of 16-byte
// chunks; slots past the kept ones are cleared.  The last workgroups of a row copy its tail.  Bound by
// HBM: 78 MB read and written in 27 to 36 us, 4.4 to 5.8 TB/s (a copy of 1 GiB 5.1).
__global__ __launch_bounds__(256) void copy_pages_kernel(CopyArgs a) {
  const int tid = threadIdx.x;
  const int64_t bh = blockIdx.y, slot = blockIdx.x;
  const int batch = (int)(bh / a.heads);
  const int from = a.rows_at >= 0 ? a.index[a.rows_at + batch]
                   : a.rows       ? min(max(a.rows[batch], 0), a.batch_in - 1)
                                  : batch;
  const int64_t src_bh = (int64_t)from * a.heads + (bh - (int64_t)batch * a.heads);
  if (slot == a.dst_capacity) {
    for (int64_t i = 16 * tid; i < a.tail_bytes; i += 16 * 256) {
      *reinterpret_cast<uint4v*>(a.tail_k_out + bh * a.tail_row + i) =
          *reinterpret_cast<const uint4v*>(a.tail_k + src_bh * a.tail_row + i);
      *reinterpret_cast<uint4v*>(a.tail_v_out + bh * a.tail_row + i) =
          *reinterpret_cast<const uint4v*>(a.tail_v + src_bh * a.tail_row + i);
    }
    return;
  }
  const bool kept = slot < a.keep;
  int64_t page = slot;
  if (kept && a.pages_at >= 0)
    page = a.index[a.pages_at + slot];
  else if (kept && a.pages)
    page = min(max(a.pages[slot], 0), a.n_stored - 1);
  const int64_t src_page = src_bh * a.src_capacity + page, dst_page = bh * a.dst_capacity + slot;
  constexpr int kUnroll = 5;
  const int total = a.first[a.n_wide];
  for (int i0 = tid; i0 < total; i0 += 256 * kUnroll) {
    uint4v w[kUnroll];
    char* to[kUnroll];
#pragma unroll
    for (int u = 0; u < kUnroll; ++u) {
      const int i = i0 + 256 * u;
      w[u] = uint4v{0u, 0u, 0u, 0u};
      to[u] = nullptr;
      if (i < total) {
        int n = 0;
        while (i >= a.first[n + 1]) ++n;
        const int64_t at = 16 * (int64_t)(i - a.first[n]);
        to[u] = a.wide[n].dst + dst_page * a.wide[n].page_bytes + at;
        if (kept) w[u] = *reinterpret_cast<const uint4v*>(a.wide[n].src + src_page * a.wide[n].page_bytes + at);
      }
    }
#pragma unroll
    for (int u = 0; u < kUnroll; ++u)
      if (to[u]) *reinterpret_cast<uint4v*>(to[u]) = w[u];
  }
  for (int n = 0; n < a.n_narrow; ++n) {
    const CopyArgs::Buffer& b = a.narrow[n];
    for (int64_t i = tid; i < b.page_bytes; i += 256)
      b.dst[dst_page * b.page_bytes + i] = kept ? b.src[src_page * b.page_bytes + i] : (char)0;
  }
}

constexpr int kTakeMax = 1024;
struct TakeArgs {
  const char* k;
  const char* v;
  char* out_k;
  char* out_v;
  int64_t k_b, k_h, k_t, v_b, v_h, v_t;  // bytes
  int64_t out_row;                       // bytes between (batch, head) rows of the outputs
  int32_t batch, heads, n, per_batch, token_bytes, f32;
  uint32_t* flag;
  uint32_t epoch;
  int32_t check;
  uint16_t index[kTakeMax];
};

// Tokens index[0 .. n) of every (batch, head) row of k and v, in that order.  16 bytes of each a
// thread; the verdict as append_stage_kernel reports it (one workgroup reports a finite input
// too, once all of its reads are through).  Latency: 3.4 us for 5 tokens, most of it the launch.
__global__ __launch_bounds__(1024) void take_tokens_kernel(TakeArgs a) {
  const int chunks = a.token_bytes / 16;
  const int64_t total = (int64_t)a.batch * a.heads * a.n * chunks;
  const uint32_t ones = a.f32 ? 0x7f800000u : 0x7c00u;
  bool bad = false;
  for (int64_t x = (int64_t)blockIdx.x * 1024 + threadIdx.x; x < total; x += (int64_t)gridDim.x * 1024) {
    const int64_t y = x / chunks, bh = y / a.n;
    const int c = (int)(x - y * chunks), i = (int)(y - bh * a.n);
    const int64_t b = bh / a.heads, h = bh - b * a.heads;
    const int64_t t = a.index[(a.per_batch ? b * a.n : 0) + i];
    const uint4v kw = *reinterpret_cast<const uint4v*>(a.k + b * a.k_b + h * a.k_h + t * a.k_t + 16 * c);
    const uint4v vw = *reinterpret_cast<const uint4v*>(a.v + b * a.v_b + h * a.v_h + t * a.v_t + 16 * c);
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      bad = bad || (kw[j] & ones) == ones || (vw[j] & ones) == ones;
      if (!a.f32) bad = bad || ((kw[j] >> 16) & ones) == ones || ((vw[j] >> 16) & ones) == ones;
    }
    const int64_t to = bh * a.out_row + (int64_t)i * a.token_bytes + 16 * c;
    *reinterpret_cast<uint4v*>(a.out_k + to) = kw;
    *reinterpret_cast<uint4v*>(a.out_v + to) = vw;
  }
  if (!a.check) return;
  if (gridDim.x == 1) {
    const bool any_bad = __syncthreads_or(bad);
    if (threadIdx.x == 0)
      __hip_atomic_store(a.flag, any_bad ? a.epoch + 1u : a.epoch, __ATOMIC_RELEASE, __HIP_MEMORY_SCOPE_SYSTEM);
  } else if (bad) {
    __hip_atomic_store(a.flag, a.epoch + 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_SYSTEM);
  }
}

}  // namespace tp

using namespace tp;

extern "C" int32_t tp_copy_pages(const tp_page_copy* bufs, int32_t n_bufs, int64_t batch, int32_t heads,
                                 int64_t batch_in, const int32_t* rows, int64_t src_capacity, int64_t dst_capacity,
                                 int32_t n_stored, const int32_t* page_index, int32_t keep, int32_t host_index,
                                 const void* tail_k, const void* tail_v, void* tail_k_out, void* tail_v_out, int64_t tail_bytes,
                                 int64_t tail_row, void* stream) {
  clear_error();
  if (n_bufs < 0 || n_bufs > kCopyBuffers || (n_bufs && !bufs) || batch < 1 || heads < 1 || batch_in < 1 ||
      batch_in > INT32_MAX || batch > 65535 / heads) {
    set_error("tp_copy_pages takes up to %d buffers and 1 to 65535 (batch, head) rows, got %d and %lld x %d",
              kCopyBuffers, n_bufs, (long long)batch, heads);
    return TP_ERR_INVALID;
  }
  if (!rows && batch != batch_in) {
    set_error("%lld batch rows of %lld need a row index", (long long)batch, (long long)batch_in);
    return TP_ERR_INVALID;
  }
  if (keep < 0 || n_stored < 0 || n_stored > src_capacity || keep > dst_capacity || dst_capacity < 0 ||
      dst_capacity >= INT32_MAX || (page_index ? keep > 0 && n_stored < 1 : keep > n_stored)) {
    set_error("%d pages of %d stored ones (capacity %lld) do not fit a capacity of %lld", keep, n_stored,
              (long long)src_capacity, (long long)dst_capacity);
    return TP_ERR_INVALID;
  }
  if (tail_bytes < 0 || (tail_bytes & 15) || (tail_row & 15) || tail_row < tail_bytes ||
      (tail_bytes && (!tail_k || !tail_v || !tail_k_out || !tail_v_out))) {
    set_error("tails of %lld bytes in rows of %lld", (long long)tail_bytes, (long long)tail_row);
    return TP_ERR_INVALID;
  }
  if ((((uintptr_t)tail_k | (uintptr_t)tail_v | (uintptr_t)tail_k_out | (uintptr_t)tail_v_out) & 15u) ||
      (((uintptr_t)rows | (uintptr_t)page_index) & 3u)) {
    set_error("tails must be 16-byte, index arrays 4-byte aligned");
    return TP_ERR_INVALID;
  }
  CopyArgs a{};
  for (int i = 0; i < n_bufs; ++i) {
    const tp_page_copy& b = bufs[i];
    if (b.page_bytes < 0 || b.page_bytes > (1 << 24)) {
      set_error("buffer %d has pages of %lld bytes", i, (long long)b.page_bytes);
      return TP_ERR_INVALID;
    }
    if (b.page_bytes == 0 || dst_capacity == 0) continue;
    if (!b.dst || (keep > 0 && !b.src)) {
      set_error("buffer %d is missing", i);
      return TP_ERR_INVALID;
    }
    const CopyArgs::Buffer to = {static_cast<const char*>(b.src), static_cast<char*>(b.dst), b.page_bytes};
    if ((((uintptr_t)b.src | (uintptr_t)b.dst | (uint64_t)b.page_bytes) & 15u) == 0) {
      a.wide[a.n_wide] = to;
      a.first[a.n_wide + 1] = a.first[a.n_wide] + (int32_t)(b.page_bytes / 16);
      ++a.n_wide;
    } else {
      a.narrow[a.n_narrow++] = to;
    }
  }
  a.rows_at = a.pages_at = -1;
  if (host_index && (rows || page_index)) {
    const int64_t n_rows = rows ? batch : 0, n_pages = page_index ? keep : 0;
    if (n_rows + n_pages > kCopyIndex) {
      set_error("host indices hold at most %d entries, got %lld", kCopyIndex, (long long)(n_rows + n_pages));
      return TP_ERR_INVALID;
    }
    for (int64_t i = 0; i < n_rows + n_pages; ++i) {
      const bool row = i < n_rows;
      const int32_t x = row ? rows[i] : page_index[i - n_rows];
      const int64_t end = row ? batch_in : n_stored;
      if (x < 0 || x >= end) {
        set_error("%s %d outside the %lld there are", row ? "batch row" : "page", x, (long long)end);
        return TP_ERR_INVALID;
      }
      a.index[i] = x;
    }
    if (rows) a.rows_at = 0;
    if (page_index) a.pages_at = (int32_t)n_rows;
    rows = page_index = nullptr;
  }
  a.src_capacity = src_capacity;
  a.dst_capacity = dst_capacity;
  a.heads = heads;
  a.batch_in = (int32_t)batch_in;
  a.n_stored = n_stored;
  a.keep = keep;
  a.rows = rows;
  a.pages = page_index;
  a.tail_k = static_cast<const char*>(tail_k);
  a.tail_v = static_cast<const char*>(tail_v);
  a.tail_k_out = static_cast<char*>(tail_k_out);
  a.tail_v_out = static_cast<char*>(tail_v_out);
  a.tail_bytes = tail_bytes;
  a.tail_row = tail_row;
  const int64_t x = dst_capacity + (tail_bytes > 0);
  if (x == 0) return TP_OK;
  hipLaunchKernelGGL(copy_pages_kernel, dim3((unsigned)x, (unsigned)(batch * heads)), dim3(256), 0,
                     static_cast<hipStream_t>(stream), a);
  return launch_status("tp_copy_pages");
}

extern "C" int32_t tp_take_tokens(const void* k, const void* v, int32_t in_dtype, int64_t batch, int32_t heads,
                                  int64_t tokens, const int64_t* strides, const int32_t* index, int32_t n,
                                  int32_t per_batch, void* out_k, void* out_v, int64_t out_tokens, int64_t out_pos,
                                  int32_t check, uint32_t* flag, uint32_t epoch, void* stream) {
  clear_error();
  if (in_dtype != 0 && in_dtype != 1) {
    set_error("in_dtype must be 0 (fp16) or 1 (fp32), got %d", in_dtype);
    return TP_ERR_INVALID;
  }
  if (!k || !v || !out_k || !out_v || !strides || !index || batch < 1 || heads < 1 || batch > INT32_MAX / heads ||
      tokens < 1 || tokens > 65536) {
    set_error("bad input: %lld x %d rows of %lld tokens", (long long)batch, heads, (long long)tokens);
    return TP_ERR_INVALID;
  }
  const int64_t entries = per_batch ? batch * (int64_t)n : n;
  if (n < 1 || entries > kTakeMax) {
    set_error("the index must hold 1 to %d tokens, got %lld", kTakeMax, (long long)entries);
    return TP_ERR_INVALID;
  }
  if (out_pos < 0 || out_pos + n > out_tokens) {
    set_error("%d tokens at position %lld do not fit rows of %lld", n, (long long)out_pos, (long long)out_tokens);
    return TP_ERR_INVALID;
  }
  if ((check != 0 && check != 2) || (check && (!flag || (epoch & 1u)))) {
    set_error("check must be 0 or 2 (pinned host flag, even epoch)");
    return TP_ERR_INVALID;
  }
  TakeArgs a{};
  const int item = in_dtype ? 4 : 2;
  for (int i = 0; i < 6; ++i)
    if (strides[i] < 0 || (strides[i] * item) % 16) {
      set_error("strides must be non-negative multiples of 16 bytes");
      return TP_ERR_INVALID;
    }
  if (((uintptr_t)k | (uintptr_t)v | (uintptr_t)out_k | (uintptr_t)out_v) & 15u) {
    set_error("k, v and the outputs must be 16-byte aligned");
    return TP_ERR_INVALID;
  }
  for (int64_t i = 0; i < entries; ++i) {
    if (index[i] < 0 || index[i] >= tokens) {
      set_error("index %d outside the %lld tokens", index[i], (long long)tokens);
      return TP_ERR_INVALID;
    }
    a.index[i] = (uint16_t)index[i];
  }
  a.k = static_cast<const char*>(k);
  a.v = static_cast<const char*>(v);
  a.token_bytes = kHeadDim * item;
  a.out_row = out_tokens * a.token_bytes;
  a.out_k = static_cast<char*>(out_k) + out_pos * a.token_bytes;
  a.out_v = static_cast<char*>(out_v) + out_pos * a.token_bytes;
  a.k_b = strides[0] * item, a.k_h = strides[1] * item, a.k_t = strides[2] * item;
  a.v_b = strides[3] * item, a.v_h = strides[4] * item, a.v_t = strides[5] * item;
  a.batch = (int32_t)batch;
  a.heads = heads;
  a.n = n;
  a.per_batch = per_batch != 0;
  a.f32 = in_dtype;
  a.flag = flag;
  a.epoch = epoch;
  a.check = check;
  // One workgroup, which reports its own end, for up to 8 chunks a thread.
  const int64_t total = batch * heads * n * (a.token_bytes / 16);
  const unsigned blocks = total <= 8192 ? 1u : (unsigned)std::min<int64_t>((total + 1023) / 1024, 2048);
  hipStream_t s = static_cast<hipStream_t>(stream);
  hipLaunchKernelGGL(take_tokens_kernel, dim3(blocks), dim3(1024), 0, s, a);
  const int32_t st = launch_status("tp_take_tokens");
  if (st != TP_OK || !check) return st;
  return wait_verdict(flag, epoch, s, blocks == 1, "tp_take_tokens");
}
