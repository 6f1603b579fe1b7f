// The paged key/value cache: block tables and slot maps built on the GPU
// (bi_page_tables) and the write of new keys and values (bi_paged_update).
//
// A cache is num_pages pages of page_size rows; request r keeps its row i in
// page block_tables[r][i / page_size], row i % page_size. A slot is page *
// page_size + row, -1 for a token that has none.
#include <hip/hip_runtime.h>
#include <stdint.h>

#include "bi_div.h"
#include "bi_internal.h"

namespace {

using bi::Div;

constexpr int kThreads = 256;
constexpr int kReqs = 4;                 // requests per thread and tile of the scan
constexpr int kTile = kThreads * kReqs;  // requests per tile

struct TablesArgs {
  int32_t* table;
  const int32_t* ctx;
  const int32_t* fresh;
  const int32_t* pool;
  int32_t* slots;
  int32_t* positions;
  int32_t* qstart;
  int32_t* seq;
  int32_t* used;
  int64_t R, W, F, T, table_stride;
  Div page;
};

// Pages of the first `rows` rows, at most W.
__device__ __forceinline__ uint32_t pages_of(uint32_t rows, const Div& page, uint32_t W) {
  const uint32_t n = rows ? (int32_t)(rows - 1) / page + 1 : 0;
  return n < W ? n : W;
}
// A request's cached rows and all its rows (at most 2^31 - 1).
__device__ __forceinline__ void lengths(int32_t ctx, int32_t fresh, uint32_t& c, uint32_t& n) {
  c = ctx > 0 ? ctx : 0;
  n = c + (fresh > 0 ? fresh : 0);
  n = n < 0x7FFFFFFFu ? n : 0x7FFFFFFFu;
}

// One launch, no communication between workgroups: each takes a range of
// tokens, one per thread, and computes the sums over the requests for itself
// (one load of each length; 1024 requests are one pass of the scan), so
// nothing waits on another workgroup: what bounds it is the chain of a launch,
// two loads, the scan and a search. A new page's table entry is written by the
// thread of the page's first token, which is always a new token, straight from
// the free list: no thread reads an entry that this launch writes. Sums of
// tokens (low) and pages (high) are scanned together; every index that depends
// on them is checked, whatever the lengths hold.
__global__ void __launch_bounds__(kThreads) page_tables_kernel(TablesArgs p) {
  __shared__ uint32_t s_start[kTile];  // first token of a request
  __shared__ uint32_t s_page[kTile];   // first place in the free list
  __shared__ int32_t s_ctx[kTile];
  __shared__ uint64_t s_part[kThreads / 64];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const uint32_t W = (uint32_t)p.W, first = blockIdx.x * kThreads, stride = gridDim.x * kThreads;
  uint64_t before = 0;  // of the tiles so far
  for (int64_t r0 = 0; r0 < p.R; r0 += kTile) {
    const int count = (int)(p.R - r0 < kTile ? p.R - r0 : kTile);
    uint32_t c[kReqs], n[kReqs];
    uint64_t own[kReqs], sum = 0;
#pragma unroll
    for (int i = 0; i < kReqs; i++) {
      const int k = tid * kReqs + i;
      lengths(k < count ? p.ctx[r0 + k] : 0, k < count ? p.fresh[r0 + k] : 0, c[i], n[i]);
    }
#pragma unroll
    for (int i = 0; i < kReqs; i++) {
      own[i] = (uint64_t)(pages_of(n[i], p.page, W) - pages_of(c[i], p.page, W)) << 32 | (n[i] - c[i]);
      sum += own[i];
    }
    uint64_t upto = sum;
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) {
      const uint64_t y = __shfl_up(upto, d);
      if (lane >= d) upto += y;
    }
    if (lane == 63) s_part[wave] = upto;
    __syncthreads();
    uint64_t at = before + upto - sum;
#pragma unroll
    for (int w = 0; w < kThreads / 64; w++) {
      if (w < wave) at += s_part[w];
      before += s_part[w];
    }
#pragma unroll
    for (int i = 0; i < kReqs; i++) {
      const int k = tid * kReqs + i;
      s_start[k] = (uint32_t)at;
      s_page[k] = (uint32_t)(at >> 32);
      s_ctx[k] = (int32_t)c[i];
      if (k < count && blockIdx.x == 0) {
        p.qstart[r0 + k] = (int32_t)at;
        p.seq[r0 + k] = (int32_t)n[i];
      }
      at += own[i];
    }
    __syncthreads();
    // The tile's tokens that this workgroup owns.
    const uint32_t t0 = s_start[0], t1 = (uint32_t)before;
    const uint32_t skip = t0 > first ? (t0 - first) / stride : 0;
    for (uint64_t b = first + (uint64_t)skip * stride; b < t1; b += stride) {
      const uint32_t t = (uint32_t)b + tid;
      if (t < t0 || t >= t1) continue;
      int lo = 0, hi = count - 1;  // the last request that starts at or before t
      while (lo < hi) {
        const int mid = (lo + hi + 1) >> 1;
        if (s_start[mid] <= t) lo = mid;
        else hi = mid - 1;
      }
      const uint32_t ctx = s_ctx[lo], pos = ctx + (t - s_start[lo]);
      int32_t id = -1;
      uint32_t row = 0;
      if (pos < 0x7FFFFFFFu) {
        const uint32_t pg = (int32_t)pos / p.page, have = pages_of(ctx, p.page, W);
        row = pos - pg * p.page.d;
        int32_t* entry = p.table + (r0 + lo) * p.table_stride + pg;
        if (pg < have) {
          id = *entry;
        } else if (pg < W) {
          const uint32_t f = s_page[lo] + pg - have;
          if (f < (uint32_t)p.F) id = p.pool[f];
          if (row == 0) *entry = id;
        }
      }
      if (t < p.T) {
        // (An entry that is no page of any cache has no slot, rather than another's.)
        const uint64_t slot = (uint64_t)(uint32_t)id * p.page.d + row;
        p.slots[t] = id < 0 || slot > INT32_MAX ? -1 : (int32_t)slot;
        p.positions[t] = (int32_t)pos;
      }
    }
    __syncthreads();
  }
  // Places behind the last request's tokens.
  const uint32_t end = (uint32_t)before;
  for (uint64_t b = first; b < (uint64_t)p.T; b += stride) {
    const uint64_t t = b + tid;
    if (t >= end && t < (uint64_t)p.T) p.slots[t] = p.positions[t] = -1;
  }
  if (blockIdx.x == 0 && tid == 0) {
    p.qstart[p.R] = (int32_t)end;
    *p.used = (int32_t)(before >> 32);
  }
}

struct UpdateArgs {
  const char* src[2];   // keys, values
  char* dst[2];
  const int32_t* slots;
  int64_t ss[2][2];     // source byte strides: token, head
  int64_t ds[2][3];     // cache byte strides: page, head, row
  int32_t T, slots_end;  // slots below num_pages * page_size
  int32_t keys, per_token;  // units of a token's keys; of keys and values
  Div page, wide;       // wide: threads side by side on a token
  Div units[2];         // copies of U bytes per row
};

// A copy: a thread moves one U-sized unit of one head's key or value row of one
// token. (What bounds it is how many loads are in flight as the launch ramps
// up: 8177 tokens of 4 KB took 16.6 us, 25 with two tokens a thread and 26.5
// with four; a plain copy of as many bytes 11.1.)
template <typename U>
__global__ void __launch_bounds__(kThreads) paged_update_kernel(UpdateArgs p) {
  const int each = kThreads / p.wide.d;  // tokens side by side
  const int sub = (int)threadIdx.x / p.wide;
  const int x = blockIdx.y * p.wide.d + (threadIdx.x - sub * (int)p.wide.d);
  if (sub >= each || x >= p.per_token) return;
  const int kv = x >= p.keys;
  const int y = kv ? x - p.keys : x;
  const int head = y / p.units[kv];
  const int64_t unit = (y - head * (int)p.units[kv].d) * (int64_t)sizeof(U);
  for (int64_t t = (int64_t)blockIdx.x * each + sub; t < p.T; t += (int64_t)gridDim.x * each) {
    const int32_t slot = p.slots[t];
    const U u = *reinterpret_cast<const U*>(p.src[kv] + t * p.ss[kv][0] + head * p.ss[kv][1] + unit);
    if (slot < 0 || slot >= p.slots_end) continue;
    const int32_t pg = slot / p.page, row = slot - pg * (int)p.page.d;
    *reinterpret_cast<U*>(p.dst[kv] + pg * p.ds[kv][0] + head * p.ds[kv][1] + row * p.ds[kv][2] + unit) = u;
  }
}

}  // namespace

extern "C" int bi_page_tables(int32_t* block_tables, const int32_t* context_lens,
                              const int32_t* new_lens, const int32_t* free_pages, int32_t* slots,
                              int32_t* positions, int32_t* query_start, int32_t* seq_lens,
                              int32_t* pages_used, int64_t R, int64_t W, int64_t table_stride,
                              int64_t F, int64_t T, int64_t page_size, void* hip_stream) {
  if (R < 0 || W < 0 || F < 0 || T < 0 || table_stride < 0)
    return bi::fail(BI_EINVAL, "bi_page_tables: negative size R=%lld W=%lld F=%lld T=%lld",
                    (long long)R, (long long)W, (long long)F, (long long)T);
  if (page_size <= 0 || page_size > INT32_MAX)
    return bi::fail(BI_EINVAL, "bi_page_tables: bad page size %lld", (long long)page_size);
  if (T > INT32_MAX || R > INT32_MAX || W > INT32_MAX || F > INT32_MAX)
    return bi::fail(BI_EINVAL, "bi_page_tables: sizes must fit 31 bits");
  if (!query_start || !pages_used || (R > 0 && (!context_lens || !new_lens || !seq_lens)) ||
      (R > 0 && W > 0 && !block_tables) || (F > 0 && !free_pages) || (T > 0 && (!slots || !positions)))
    return bi::fail(BI_EINVAL, "bi_page_tables: null pointer");
  TablesArgs p = {block_tables, context_lens, new_lens, free_pages, slots, positions, query_start,
                  seq_lens, pages_used, R, W, F, T, table_stride, bi::make_div(page_size)};
  int64_t blocks = (T + kThreads - 1) / kThreads;
  if (blocks < 1) blocks = 1;
  if (blocks > 1024) blocks = 1024;
  hipLaunchKernelGGL(page_tables_kernel, dim3((unsigned)blocks), dim3(kThreads), 0,
                     static_cast<hipStream_t>(hip_stream), p);
  const hipError_t e = hipGetLastError();
  return e == hipSuccess ? BI_OK : bi::launch_error(e, "bi_page_tables launch");
}

extern "C" int bi_paged_update(const void* k, const void* v, void* k_cache, void* v_cache,
                               const int32_t* slots, int64_t T, int64_t Hkv, int64_t D, int64_t V,
                               int64_t num_pages, int64_t page_size, const int64_t* strides,
                               int dtype, void* hip_stream) {
  const int esz = bi::elem_size(dtype);
  if (!esz) return bi::fail(BI_EINVAL, "bi_paged_update: unknown dtype %d", dtype);
  if (T < 0 || Hkv <= 0 || D <= 0 || V <= 0 || num_pages < 0 || page_size <= 0)
    return bi::fail(BI_EINVAL, "bi_paged_update: bad sizes T=%lld Hkv=%lld D=%lld V=%lld pages=%lld x %lld",
                    (long long)T, (long long)Hkv, (long long)D, (long long)V, (long long)num_pages,
                    (long long)page_size);
  if (Hkv > (1 << 20) || D > (1 << 20) || V > (1 << 20) || Hkv * (D + V) > (1 << 28) ||
      T > INT32_MAX || num_pages > INT32_MAX || page_size > INT32_MAX ||
      num_pages * page_size > INT32_MAX)
    return bi::fail(BI_EINVAL, "bi_paged_update: sizes too large");
  if (T == 0 || num_pages == 0) return BI_OK;
  if (!k || !v || !k_cache || !v_cache || !slots || !strides)
    return bi::fail(BI_EINVAL, "bi_paged_update: null pointer");
  UpdateArgs p;
  p.src[0] = static_cast<const char*>(k);
  p.src[1] = static_cast<const char*>(v);
  p.dst[0] = static_cast<char*>(k_cache);
  p.dst[1] = static_cast<char*>(v_cache);
  p.slots = slots;
  for (int i = 0; i < 2; i++) {
    for (int j = 0; j < 2; j++) p.ss[i][j] = strides[2 * i + j] * esz;
    for (int j = 0; j < 3; j++) p.ds[i][j] = strides[4 + 3 * i + j] * esz;
  }
  p.T = (int32_t)T;
  p.slots_end = (int32_t)(num_pages * page_size);
  p.page = bi::make_div(page_size);
  // The widest unit that every row's address and length is a multiple of.
  uint64_t bits = (uint64_t)(D * esz) | (uint64_t)(V * esz) | (uintptr_t)k | (uintptr_t)v |
                  (uintptr_t)k_cache | (uintptr_t)v_cache;
  for (int i = 0; i < 2; i++) {
    for (int j = 0; j < 2; j++) bits |= (uint64_t)p.ss[i][j];
    for (int j = 0; j < 3; j++) bits |= (uint64_t)p.ds[i][j];
  }
  const int unit = bits % 16 == 0 ? 16 : bits % 4 == 0 ? 4 : bits % 2 == 0 ? 2 : 1;
  if (unit < esz) return bi::fail(BI_EINVAL, "bi_paged_update: pointers not aligned to elements");
  p.units[0] = bi::make_div(D * esz / unit);
  p.units[1] = bi::make_div(V * esz / unit);
  p.keys = (int32_t)(Hkv * p.units[0].d);
  p.per_token = (int32_t)(p.keys + Hkv * p.units[1].d);
  const int64_t wide = p.per_token < kThreads ? p.per_token : kThreads;
  p.wide = bi::make_div(wide);
  const int64_t each = kThreads / wide, gy = (p.per_token + wide - 1) / wide;
  const int64_t tokens = (T + each - 1) / each, gx = tokens < 1 << 22 ? tokens : 1 << 22;
  if (gy > 65535) return bi::fail(BI_EINVAL, "bi_paged_update: rows too wide");
  const dim3 grid((unsigned)gx, (unsigned)gy);
  const hipStream_t s = static_cast<hipStream_t>(hip_stream);
  if (unit == 16) hipLaunchKernelGGL(paged_update_kernel<uint4>, grid, dim3(kThreads), 0, s, p);
  else if (unit == 4) hipLaunchKernelGGL(paged_update_kernel<uint32_t>, grid, dim3(kThreads), 0, s, p);
  else hipLaunchKernelGGL(paged_update_kernel<uint16_t>, grid, dim3(kThreads), 0, s, p);
  const hipError_t e = hipGetLastError();
  return e == hipSuccess ? BI_OK : bi::launch_error(e, "bi_paged_update launch");
}
