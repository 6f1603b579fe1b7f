// The paged cache in 8 bits: the write of new keys and values as codes with a
// scale for every token and head (bi_paged_update_q8), and the way back from a
// cache of any type to rows of tokens (bi_paged_read).
//
// Mathematics. A row x of one token and head is kept as whole numbers c in -127
// .. 127 and a scale s of 32 bits, its values being c * s: s = max |x| / 127,
// rounded once, and c = x / s rounded to the nearest, ties to even. (Exactly
// so, by a division and a look at its remainder: the codes are then a function
// of the row alone, whatever computes them.) A code is off by half a step at
// most, s / 2 = max |x| / 254. A scale belongs to one token: one that later
// tokens of a block could raise would make what a token attends to depend on
// how its prompt was cut.
#include <float.h>
#include <math.h>

#include <hip/hip_runtime.h>
#include <stdint.h>

#include "bi_div.h"
#include "bi_internal.h"

namespace {

using bi::Div;

constexpr int kThreads = 256;

struct Side {        // keys or values
  const char* src;   // tokens (update) or the cache (read)
  char* dst;
  float* scale;      // (num_pages, Hkv, page_size); NULL: read without
  int64_t ts, hs;    // byte strides of the tokens: token, head
  int64_t cp, ch, cr;  // of the cache: page, head, row
  int64_t sp, sh, sr;  // element strides of the scales
  int32_t D, units;  // elements of a row, and how many units these are
  int32_t lanes, shift;  // lanes of a row, 2^shift
  int32_t blocks;    // workgroups
};

struct Q8Args {
  Side side[2];
  const int32_t* slots;
  int64_t rows;      // T * Hkv
  int32_t T, slots_end;
  int32_t keep;      // scales are given
  Div Hkv, page;
};

template <typename T, int U> struct Vec {
  typedef T type __attribute__((ext_vector_type(U)));
};

// x / s to the nearest whole number, ties to even, within -127 .. 127.
__device__ __forceinline__ int8_t code_of(float x, float s) {
  float n = __builtin_rintf(x / s);
  // The quotient's own rounding may have made a tie of what is none.
  const float r = 2.f * __builtin_fmaf(-n, s, x);
  if (r > s) n += 1.f;
  if (r < -s) n -= 1.f;
  n = fminf(fmaxf(n, -127.f), 127.f);
  return (int8_t)(int)n;
}

// One row of a token and head by `lanes` lanes, U elements at a time each (16
// bytes, or one where rows are not aligned to that). What bounds it is memory.
template <typename T, int U>
__global__ void __launch_bounds__(kThreads) update_kernel(Q8Args p) {
  typedef typename Vec<T, U>::type In;
  typedef typename Vec<int8_t, U>::type Out;
  const int kv = (int)blockIdx.x >= p.side[0].blocks;
  const Side& w = p.side[kv];
  const int64_t block = blockIdx.x - (kv ? p.side[0].blocks : 0);
  const int lane = threadIdx.x & (w.lanes - 1);
  const int64_t id = (block * kThreads + threadIdx.x) >> w.shift;
  const bool real = id < p.rows;
  const int32_t t = real ? (int32_t)id / p.Hkv : 0, head = real ? (int32_t)id - t * (int32_t)p.Hkv.d : 0;
  const int32_t slot = p.slots[t];
  const bool write = real && slot >= 0 && slot < p.slots_end;
  const char* row = w.src + t * w.ts + head * w.hs;
  const int32_t pg = (write ? slot : 0) / p.page, at = (write ? slot : 0) - pg * (int32_t)p.page.d;
  float* scale = w.scale + pg * w.sp + head * w.sh + at * w.sr;

  // The first unit stays in registers: for most heads it is the only one.
  In first = {};
  float top = 0.f;
  bool odd = false;  // an infinity or NaN
  float s;
  if (p.keep) {
    if (lane < w.units) first = reinterpret_cast<const In*>(row)[lane];
    s = write ? *scale : 0.f;
  } else {
    for (int u = lane; u < w.units; u += w.lanes) {
      const In x = reinterpret_cast<const In*>(row)[u];
      if (u == lane) first = x;
#pragma unroll
      for (int i = 0; i < U; i++) {
        const float a = fabsf((float)x[i]);
        odd |= !(a <= FLT_MAX);
        top = fmaxf(top, a);
      }
    }
    top = odd ? INFINITY : top;
    for (int d = 1; d < w.lanes; d <<= 1) top = fmaxf(top, __shfl_xor(top, d));
    s = top <= FLT_MAX ? top / 127.f : NAN;
    if (write && lane == 0) *scale = s;
  }
  if (!write) return;
  Out* out = reinterpret_cast<Out*>(w.dst + pg * w.cp + head * w.ch + at * w.cr);
  for (int u = lane; u < w.units; u += w.lanes) {
    const In x = u == lane ? first : reinterpret_cast<const In*>(row)[u];
    Out c;
#pragma unroll
    for (int i = 0; i < U; i++) {
      const float v = (float)x[i];
      c[i] = s > 0.f && v == v ? code_of(v, s) : (int8_t)0;
    }
    out[u] = c;
  }
}

// The way back: unit by unit, a code's value c * s in 32 bits, rounded once
// more to the type; a cache of the type itself is copied.
template <typename C, typename T, int U>
__global__ void __launch_bounds__(kThreads) read_kernel(Q8Args p) {
  typedef typename Vec<C, U>::type In;
  typedef typename Vec<T, U>::type Out;
  const int kv = (int)blockIdx.x >= p.side[0].blocks;
  const Side& w = p.side[kv];
  const int64_t block = blockIdx.x - (kv ? p.side[0].blocks : 0);
  const int lane = threadIdx.x & (w.lanes - 1);
  const int64_t id = (block * kThreads + threadIdx.x) >> w.shift;
  if (id >= p.rows) return;
  const int32_t t = (int32_t)id / p.Hkv, head = (int32_t)id - t * (int32_t)p.Hkv.d;
  const int32_t slot = p.slots[t];
  const bool there = slot >= 0 && slot < p.slots_end;
  const int32_t pg = (there ? slot : 0) / p.page, at = (there ? slot : 0) - pg * (int32_t)p.page.d;
  const In* row = reinterpret_cast<const In*>(w.src + pg * w.cp + head * w.ch + at * w.cr);
  float s = 1.f;
  if constexpr (sizeof(C) == 1)
    if (there) s = w.scale[pg * w.sp + head * w.sh + at * w.sr];
  Out* out = reinterpret_cast<Out*>(w.dst + t * w.ts + head * w.hs);
  for (int u = lane; u < w.units; u += w.lanes) {
    Out y = {};
    if (there) {
      const In x = row[u];
#pragma unroll
      for (int i = 0; i < U; i++) {
        if constexpr (sizeof(C) == 1) y[i] = (T)((float)x[i] * s);
        else y[i] = x[i];
      }
    }
    out[u] = y;
  }
}

int shift_for(int64_t units) {
  int n = 0;
  while (1 << n < units && n < 6) n++;
  return n;
}

// Sizes and strides that update and read share.
int setup(const char* who, Q8Args& p, const void* slots, int64_t T, int64_t Hkv, int64_t D, int64_t V,
          int64_t num_pages, int64_t page_size, const int64_t* st, const int64_t* scale_st, int esz,
          int csz) {
  if (T < 0 || Hkv <= 0 || D <= 0 || V <= 0 || num_pages < 0 || page_size <= 0)
    return bi::fail(BI_EINVAL, "%s: bad sizes T=%lld Hkv=%lld D=%lld V=%lld pages=%lld x %lld", who,
                    (long long)T, (long long)Hkv, (long long)D, (long long)V, (long long)num_pages,
                    (long long)page_size);
  if (Hkv > (1 << 20) || D > (1 << 20) || V > (1 << 20) || T > INT32_MAX || T * Hkv > INT32_MAX ||
      num_pages > INT32_MAX || page_size > INT32_MAX || num_pages * page_size > INT32_MAX)
    return bi::fail(BI_EINVAL, "%s: sizes too large", who);
  p.slots = static_cast<const int32_t*>(slots);
  p.rows = T * Hkv;
  p.T = (int32_t)T;
  p.slots_end = (int32_t)(num_pages * page_size);
  p.Hkv = bi::make_div(Hkv);
  p.page = bi::make_div(page_size);
  for (int i = 0; i < 2; i++) {
    Side& w = p.side[i];
    w.D = (int32_t)(i ? V : D);
    w.ts = st[2 * i] * esz, w.hs = st[2 * i + 1] * esz;
    w.cp = st[4 + 3 * i] * csz, w.ch = st[5 + 3 * i] * csz, w.cr = st[6 + 3 * i] * csz;
    if (scale_st) w.sp = scale_st[3 * i], w.sh = scale_st[3 * i + 1], w.sr = scale_st[3 * i + 2];
  }
  return BI_OK;
}

// Whether rows can be taken `wide` elements at a time on both sides.
bool aligned(const Q8Args& p, const void* const* tokens, const void* const* cache, int wide, int esz,
             int csz) {
  for (int i = 0; i < 2; i++) {
    const Side& w = p.side[i];
    if (w.D % wide) return false;
    if (((uintptr_t)tokens[i] | (uint64_t)w.ts | (uint64_t)w.hs) % (wide * esz)) return false;
    if (((uintptr_t)cache[i] | (uint64_t)w.cp | (uint64_t)w.ch | (uint64_t)w.cr) % (wide * csz)) return false;
  }
  return true;
}

int start(const char* who, Q8Args& p, void (*kernel)(Q8Args), int unit, void* stream) {
  int64_t all = 0;
  for (int i = 0; i < 2; i++) {
    Side& w = p.side[i];
    w.units = w.D / unit;
    w.shift = shift_for(w.units);
    w.lanes = 1 << w.shift;
    const int64_t blocks = (p.rows * w.lanes + kThreads - 1) / kThreads;
    w.blocks = (int32_t)blocks;
    all += blocks;
  }
  if (all > INT32_MAX) return bi::fail(BI_EINVAL, "%s: sizes too large", who);
  hipLaunchKernelGGL(kernel, dim3((unsigned)all), dim3(kThreads), 0, static_cast<hipStream_t>(stream), p);
  const hipError_t e = hipGetLastError();
  return e == hipSuccess ? BI_OK : bi::launch_error(e, who);
}

template <typename C> void (*read_for(int dtype, bool wide))(Q8Args) {
  if constexpr (sizeof(C) == 1) {
    if (dtype == BI_F32) return wide ? read_kernel<C, float, 4> : read_kernel<C, float, 1>;
    if (dtype == BI_F16) return wide ? read_kernel<C, _Float16, 8> : read_kernel<C, _Float16, 1>;
    return wide ? read_kernel<C, __bf16, 8> : read_kernel<C, __bf16, 1>;
  } else {
    return wide ? read_kernel<C, C, 16 / sizeof(C)> : read_kernel<C, C, 1>;
  }
}

}  // namespace

extern "C" int bi_paged_update_q8(const void* k, const void* v, int8_t* k_cache, int8_t* v_cache,
                                  float* k_scales, float* v_scales, const int32_t* slots, int64_t T,
                                  int64_t Hkv, int64_t D, int64_t V, int64_t num_pages,
                                  int64_t page_size, const int64_t* strides,
                                  const int64_t* scale_strides, int keep_scales, int dtype,
                                  void* hip_stream) {
  const char* who = "bi_paged_update_q8";
  const int esz = bi::elem_size(dtype);
  if (!esz) return bi::fail(BI_EINVAL, "%s: unknown dtype %d", who, dtype);
  if (T > 0 && num_pages > 0 &&
      (!k || !v || !k_cache || !v_cache || !k_scales || !v_scales || !slots || !strides || !scale_strides))
    return bi::fail(BI_EINVAL, "%s: null pointer", who);
  const int64_t none[10] = {};
  Q8Args p = {};
  const int rc = setup(who, p, slots, T, Hkv, D, V, num_pages, page_size, strides ? strides : none,
                       scale_strides, esz, 1);
  if (rc) return rc;
  if (T == 0 || num_pages == 0) return BI_OK;
  const void* tokens[2] = {k, v};
  const void* cache[2] = {k_cache, v_cache};
  if (!aligned(p, tokens, cache, 1, esz, 1) || ((uintptr_t)k_scales | (uintptr_t)v_scales) % 4)
    return bi::fail(BI_EINVAL, "%s: pointers not aligned to elements", who);
  p.side[0].src = static_cast<const char*>(k), p.side[1].src = static_cast<const char*>(v);
  p.side[0].dst = reinterpret_cast<char*>(k_cache), p.side[1].dst = reinterpret_cast<char*>(v_cache);
  p.side[0].scale = k_scales, p.side[1].scale = v_scales;
  p.keep = keep_scales;
  const bool wide = aligned(p, tokens, cache, 16 / esz, esz, 1);
  void (*f)(Q8Args);
  if (dtype == BI_F32) f = wide ? update_kernel<float, 4> : update_kernel<float, 1>;
  else if (dtype == BI_F16) f = wide ? update_kernel<_Float16, 8> : update_kernel<_Float16, 1>;
  else f = wide ? update_kernel<__bf16, 8> : update_kernel<__bf16, 1>;
  return start(who, p, f, wide ? 16 / esz : 1, hip_stream);
}

extern "C" int bi_paged_read(const void* k_cache, const void* v_cache, const float* k_scales,
                             const float* v_scales, const int32_t* slots, void* k, void* v, int64_t T,
                             int64_t Hkv, int64_t D, int64_t V, int64_t num_pages, int64_t page_size,
                             const int64_t* strides, const int64_t* scale_strides, int dtype,
                             void* hip_stream) {
  const char* who = "bi_paged_read";
  const int esz = bi::elem_size(dtype);
  if (!esz) return bi::fail(BI_EINVAL, "%s: unknown dtype %d", who, dtype);
  const bool q8 = k_scales != nullptr;
  const int csz = q8 ? 1 : esz;
  if (T > 0 && (!k || !v || !slots || !strides || (num_pages > 0 && (!k_cache || !v_cache)) ||
                (q8 && (!v_scales || !scale_strides)) || (!q8 && v_scales)))
    return bi::fail(BI_EINVAL, "%s: null pointer", who);
  const int64_t none[10] = {};
  Q8Args p = {};
  const int rc = setup(who, p, slots, T, Hkv, D, V, num_pages, page_size, strides ? strides : none,
                       q8 ? scale_strides : nullptr, esz, csz);
  if (rc) return rc;
  if (T == 0) return BI_OK;
  const void* tokens[2] = {k, v};
  const void* cache[2] = {k_cache, v_cache};
  if (!aligned(p, tokens, cache, 1, esz, csz) || ((uintptr_t)k_scales | (uintptr_t)v_scales) % 4)
    return bi::fail(BI_EINVAL, "%s: pointers not aligned to elements", who);
  p.side[0].src = static_cast<const char*>(k_cache), p.side[1].src = static_cast<const char*>(v_cache);
  p.side[0].dst = static_cast<char*>(k), p.side[1].dst = static_cast<char*>(v);
  p.side[0].scale = const_cast<float*>(k_scales), p.side[1].scale = const_cast<float*>(v_scales);
  const bool wide = aligned(p, tokens, cache, 16 / esz, esz, csz);
  void (*f)(Q8Args);
  if (q8) f = read_for<int8_t>(dtype, wide);
  else if (dtype == BI_F32) f = read_for<float>(dtype, wide);
  else if (dtype == BI_F16) f = read_for<_Float16>(dtype, wide);
  else f = read_for<__bf16>(dtype, wide);
  return start(who, p, f, wide ? 16 / esz : 1, hip_stream);
}
