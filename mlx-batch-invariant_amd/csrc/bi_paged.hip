// The paged key/value cache: block tables and slot maps built on the GPU
// (bi_page_tables) and the write of new keys and values (bi_paged_update).
//
// A cache is num_pages pages of page_size rows; request r keeps its row i in
// page block_tables[r][i / page_size], row i % page_size. A slot is page *
// page_size + row, -1 for a token that has none.
#include <hip/hip_runtime.h>
#include <stdint.h>

#include "bi_internal.h"

namespace {

constexpr int kThreads = 256;
constexpr int kWave = 64;
constexpr int kReqs = 4;                       // requests per thread and tile of the scan
constexpr int kTile = kThreads * kReqs;        // requests per tile
constexpr int kTokens = 4;                     // tokens per thread
constexpr int kTokenTile = kThreads * kTokens;  // tokens per workgroup

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
  int32_t page;
};

__device__ __forceinline__ int64_t pages_of(int64_t rows, int32_t page, int64_t W) {
  const int64_t n = (int64_t)(((uint64_t)rows + (uint32_t)page - 1) / (uint32_t)page);
  return n < W ? n : W;
}

// Inclusive sums over the workgroup, 64-bit: over a wave by shuffles, over the
// waves through LDS. Returns this thread's exclusive sum; `total` the whole.
__device__ __forceinline__ int64_t block_scan(int64_t x, int64_t* part, int64_t& total) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  int64_t s = x;
#pragma unroll
  for (int d = 1; d < kWave; d <<= 1) {
    const int64_t y = __shfl_up(s, d);
    if (lane >= d) s += y;
  }
  if (lane == 63) part[wave] = s;
  __syncthreads();
  int64_t before = 0;
  total = 0;
#pragma unroll
  for (int w = 0; w < kThreads / kWave; w++) {
    if (w < wave) before += part[w];
    total += part[w];
  }
  __syncthreads();
  return before + s - x;
}

// One launch, no communication between workgroups: each takes a range of
// tokens and computes the sums over the requests for itself (R loads from the
// caches; with a few hundred requests one pass of the scan), so nothing waits
// on another workgroup. A new page's table entry is written by the thread of
// the page's first token, which is always a new token, straight from the free
// list: no thread reads an entry that this launch writes.
__global__ void __launch_bounds__(kThreads) page_tables_kernel(TablesArgs p) {
  __shared__ int64_t s_start[kTile];  // first token of a request
  __shared__ int64_t s_page[kTile];   // first place in the free list
  __shared__ int64_t s_part[kThreads / kWave];
  const int tid = threadIdx.x;
  const int64_t stride = (int64_t)gridDim.x * kTokenTile;
  int64_t t_base = 0, g_base = 0;  // tokens and pages of the requests before the tile
  for (int64_t r0 = 0; r0 < p.R; r0 += kTile) {
    int64_t n[kReqs], take[kReqs], sn = 0, st = 0;
    int32_t c[kReqs];
#pragma unroll
    for (int i = 0; i < kReqs; i++) {
      const int64_t r = r0 + tid * kReqs + i;
      c[i] = 0;
      n[i] = 0;
      if (r < p.R) {
        c[i] = p.ctx[r] > 0 ? p.ctx[r] : 0;
        n[i] = p.fresh[r] > 0 ? p.fresh[r] : 0;
      }
      take[i] = pages_of(c[i] + n[i], p.page, p.W) - pages_of(c[i], p.page, p.W);
      sn += n[i];
      st += take[i];
    }
    int64_t tn, tt;
    int64_t an = t_base + block_scan(sn, s_part, tn);
    int64_t at = g_base + block_scan(st, s_part, tt);
    const int count = (int)(p.R - r0 < kTile ? p.R - r0 : kTile);
#pragma unroll
    for (int i = 0; i < kReqs; i++) {
      const int64_t r = r0 + tid * kReqs + i;
      s_start[tid * kReqs + i] = an;
      s_page[tid * kReqs + i] = at;
      if (r < p.R && blockIdx.x == 0) {
        p.qstart[r] = (int32_t)an;
        p.seq[r] = (int32_t)(c[i] + n[i]);
      }
      an += n[i];
      at += take[i];
    }
    __syncthreads();
    // The tile's tokens t_base .. t_base + tn - 1 that this workgroup owns.
    const int64_t end = t_base + tn;
    for (int64_t b = (int64_t)blockIdx.x * kTokenTile; b < end; b += stride) {
      if (b + kTokenTile <= t_base) continue;
#pragma unroll
      for (int i = 0; i < kTokens; i++) {
        const int64_t t = b + i * kThreads + tid;
        if (t < t_base || t >= end) continue;
        int lo = 0, hi = count - 1;  // the last request that starts at or before t
        while (lo < hi) {
          const int mid = (lo + hi + 1) >> 1;
          if (s_start[mid] <= t) lo = mid;
          else hi = mid - 1;
        }
        const int64_t r = r0 + lo;
        const int32_t ctx = p.ctx[r] > 0 ? p.ctx[r] : 0;
        const int64_t pos = ctx + (t - s_start[lo]);
        const int64_t pg = pos / p.page, row = pos - pg * p.page;
        int32_t id = -1;
        if (pg < p.W) {
          const int64_t have = pages_of(ctx, p.page, p.W);
          if (pg < have) {
            id = p.table[r * p.table_stride + pg];
          } else {
            const int64_t f = s_page[lo] + pg - have;
            if (f < p.F) id = p.pool[f];
            if (row == 0) p.table[r * p.table_stride + pg] = id;
          }
        }
        if (t < p.T) {
          p.slots[t] = id < 0 ? -1 : (int32_t)((int64_t)id * p.page + row);
          p.positions[t] = (int32_t)pos;
        }
      }
    }
    t_base = end;
    g_base += tt;
    __syncthreads();
  }
  // Places behind the last request's tokens.
  for (int64_t b = (int64_t)blockIdx.x * kTokenTile; b < p.T; b += stride)
#pragma unroll
    for (int i = 0; i < kTokens; i++) {
      const int64_t t = b + i * kThreads + tid;
      if (t >= t_base && t < p.T) p.slots[t] = p.positions[t] = -1;
    }
  if (blockIdx.x == 0 && tid == 0) {
    p.qstart[p.R] = (int32_t)t_base;
    *p.used = (int32_t)g_base;
  }
}

struct UpdateArgs {
  const char* src[2];   // keys, values
  char* dst[2];
  const int32_t* slots;
  int64_t ss[2][2];     // source byte strides: token, head
  int64_t ds[2][3];     // cache byte strides: page, head, row
  int64_t T, slots_end;  // slots below num_pages * page_size
  int32_t page, heads;
  int32_t units[2];     // copies of U bytes per row
  int32_t per_token;    // heads * (units[0] + units[1])
};

// A copy: thread x of a token moves one U-sized unit of one head's key or
// value row. kRows tokens per thread keep several loads in flight.
constexpr int kRows = 4;
template <typename U>
__global__ void __launch_bounds__(kThreads) paged_update_kernel(UpdateArgs p) {
  const int wide = p.per_token < kThreads ? p.per_token : kThreads;  // units side by side
  const int each = kThreads / wide;                                 // tokens side by side
  const int sub = threadIdx.x / wide;
  const int x = blockIdx.y * wide + threadIdx.x % wide;
  if (sub >= each || x >= p.per_token) return;
  const int keys = p.heads * p.units[0];
  const int kv = x >= keys;
  const int y = kv ? x - keys : x;
  const int head = y / p.units[kv], unit = y - head * p.units[kv];
  const char* src = p.src[kv] + head * p.ss[kv][1] + (int64_t)unit * sizeof(U);
  char* dst = p.dst[kv] + head * p.ds[kv][1] + (int64_t)unit * sizeof(U);
  const int64_t step = (int64_t)gridDim.x * each * kRows;
  for (int64_t t0 = ((int64_t)blockIdx.x * kRows) * each + sub; t0 < p.T; t0 += step) {
    U u[kRows];
    int32_t slot[kRows];
#pragma unroll
    for (int i = 0; i < kRows; i++) {
      const int64_t t = t0 + i * each;
      slot[i] = t < p.T ? p.slots[t] : -1;
      if (t < p.T) u[i] = *reinterpret_cast<const U*>(src + t * p.ss[kv][0]);
    }
#pragma unroll
    for (int i = 0; i < kRows; i++) {
      if (slot[i] < 0 || slot[i] >= p.slots_end) continue;
      const int32_t pg = slot[i] / p.page, row = slot[i] - pg * p.page;
      *reinterpret_cast<U*>(dst + pg * p.ds[kv][0] + row * p.ds[kv][2]) = u[i];
    }
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
                  seq_lens, pages_used, R, W, F, T, table_stride, (int32_t)page_size};
  int64_t blocks = (T + kTokenTile - 1) / kTokenTile;
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
  p.T = T;
  p.slots_end = num_pages * page_size;
  p.page = (int32_t)page_size;
  p.heads = (int32_t)Hkv;
  // The widest unit that every row's address and length is a multiple of.
  uint64_t bits = (uint64_t)(D * esz) | (uint64_t)(V * esz) | (uintptr_t)k | (uintptr_t)v |
                  (uintptr_t)k_cache | (uintptr_t)v_cache;
  for (int i = 0; i < 2; i++) {
    for (int j = 0; j < 2; j++) bits |= (uint64_t)p.ss[i][j];
    for (int j = 0; j < 3; j++) bits |= (uint64_t)p.ds[i][j];
  }
  const int unit = bits % 16 == 0 ? 16 : bits % 4 == 0 ? 4 : bits % 2 == 0 ? 2 : 1;
  if (unit < esz) return bi::fail(BI_EINVAL, "bi_paged_update: pointers not aligned to elements");
  p.units[0] = (int32_t)(D * esz / unit);
  p.units[1] = (int32_t)(V * esz / unit);
  p.per_token = p.heads * (p.units[0] + p.units[1]);
  const int64_t wide = p.per_token < kThreads ? p.per_token : kThreads;
  const int64_t each = kThreads / wide, gy = (p.per_token + wide - 1) / wide;
  int64_t gx = (T + each * kRows - 1) / (each * kRows);
  if (gx > 65536) gx = 65536;
  if (gy > 65535) return bi::fail(BI_EINVAL, "bi_paged_update: rows too wide");
  const dim3 grid((unsigned)gx, (unsigned)gy);
  const hipStream_t s = static_cast<hipStream_t>(hip_stream);
  if (unit == 16) hipLaunchKernelGGL(paged_update_kernel<uint4>, grid, dim3(kThreads), 0, s, p);
  else if (unit == 4) hipLaunchKernelGGL(paged_update_kernel<uint32_t>, grid, dim3(kThreads), 0, s, p);
  else hipLaunchKernelGGL(paged_update_kernel<uint16_t>, grid, dim3(kThreads), 0, s, p);
  const hipError_t e = hipGetLastError();
  return e == hipSuccess ? BI_OK : bi::launch_error(e, "bi_paged_update launch");
}
