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
__device__ __forceinline__ float code_of(float x, float s) {
  float n = __builtin_rintf(x / s);
  // The quotient's own rounding may have made a tie of what is none.
  const float r = 2.f * __builtin_fmaf(-n, s, x);
  if (r > s) n += 1.f;
  if (r < -s) n -= 1.f;
  n = fminf(fmaxf(n, -127.f), 127.f);
  return x == x ? n : 0.f;
}
// The codes of U values with scale s above 0, `inv` about 1 / s: n = rint(x * inv)
// is the nearest whole number to x / s if |x - n s| is below s / 2, which it nearly
// always is; the fma rounds that difference once, and s / 2 is a number of 32 bits, so
// the comparison is exact. Else, next to a tie, the wave divides. (With a division for
// every value 8177 tokens took 25 us; memory would take 10.)
template <int U>
__device__ __forceinline__ void codes_of(const float (&x)[U], float s, float inv, bool keep, int8_t (&c)[U]) {
  float n[U], far = 0.f;
  bool odd = !(s > 1e-30f && s < 1e37f);
#pragma unroll
  for (int i = 0; i < U; i++) {
    n[i] = __builtin_rintf(x[i] * inv);
    far = fmaxf(far, fabsf(__builtin_fmaf(-n[i], s, x[i])));
    if (keep) {
      odd |= x[i] != x[i];
      n[i] = fminf(fmaxf(n[i], -127.f), 127.f);
    }
  }
  if (__builtin_amdgcn_ballot_w64(odd || !(2.f * far < s)) != 0)
#pragma unroll
    for (int i = 0; i < U; i++) n[i] = code_of(x[i], s);
#pragma unroll
  for (int i = 0; i < U; i++) c[i] = (int8_t)(int)n[i];
}

// The largest of `lanes` neighbouring lanes, a power of two, by moves within a
// register (a shuffle by way of the LDS takes ten times as long).
template <int CTRL> __device__ __forceinline__ float max_with(float x) {
  return fmaxf(x, __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(x), CTRL, 0xF, 0xF, true)));
}
__device__ __forceinline__ float row_max(float x, int lanes) {
  if (lanes > 1) x = max_with<0xB1>(x);   // lane ^ 1
  if (lanes > 2) x = max_with<0x4E>(x);   // lane ^ 2
  if (lanes > 4) x = max_with<0x141>(x);  // 7 - lane of eight
  if (lanes > 8) x = max_with<0x140>(x);  // 15 - lane of sixteen
  if (lanes > 16) {
    const auto r = __builtin_amdgcn_permlane16_swap(__float_as_uint(x), __float_as_uint(x), false, false);
    x = fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1]));
  }
  if (lanes > 32) {
    const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
    x = fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1]));
  }
  return x;
}

// n * stride: one multiplication of 32 bits by 32, and where a stride is past them
// (which all lanes know) the rest. (For the write, half of whose instructions were
// addresses and the search for the largest: 8177 tokens 19.8 -> 17.9 us with both
// mended; the read, bound by memory, gains nothing.)
__device__ __forceinline__ int64_t times(int32_t n, int64_t stride) {
  uint64_t x = (uint64_t)(uint32_t)n * (uint32_t)stride;
  const uint32_t high = (uint32_t)((uint64_t)stride >> 32);
  if (high) x += (uint64_t)((uint32_t)n * high) << 32;
  return (int64_t)x;
}

// A row's side, and its token and head, from the thread's place.
struct Place {
  int kv, lane;
  int32_t t, head;
  bool real;
};
__device__ __forceinline__ Place place(const Q8Args& p) {
  Place x;
  x.kv = (int)blockIdx.x >= p.side[0].blocks;
  const Side& w = p.side[x.kv];
  const uint32_t thread = (blockIdx.x - (x.kv ? p.side[0].blocks : 0)) * kThreads + threadIdx.x;
  x.lane = threadIdx.x & (w.lanes - 1);
  const uint32_t id = thread >> w.shift;
  x.real = id < p.rows;
  x.t = x.real ? (int32_t)id / p.Hkv : 0;
  x.head = x.real ? (int32_t)id - x.t * (int32_t)p.Hkv.d : 0;
  return x;
}

// The largest magnitude of U values, infinity where one is infinite or NaN: as whole
// numbers, without their sign, magnitudes have the order of their values, and those
// are above all. Of 16 bits two at a time.
template <typename T, int U> __device__ __forceinline__ float largest(const typename Vec<T, U>::type& y) {
  if constexpr (sizeof(T) == 4 || U == 1) {
    float top = 0.f;
#pragma unroll
    for (int i = 0; i < U; i++) {
      const float a = fabsf((float)y[i]);
      top = fmaxf(top, a <= FLT_MAX ? a : INFINITY);
    }
    return top;
  } else {
    typedef uint16_t u16x2 __attribute__((ext_vector_type(2)));
    typedef uint32_t Words __attribute__((ext_vector_type(U / 2)));
    const Words w = __builtin_bit_cast(Words, y);
    u16x2 m = {0, 0};
#pragma unroll
    for (int i = 0; i < U / 2; i++) m = __builtin_elementwise_max(m, __builtin_bit_cast(u16x2, w[i] & 0x7FFF7FFFu));
    const float a = (float)__builtin_bit_cast(T, m.x > m.y ? m.x : m.y);
    return a <= FLT_MAX ? a : INFINITY;
  }
}

// One row of a token and head by `lanes` lanes, U elements at a time each (16
// bytes, or one where rows are not aligned to that); ONE: each lane has one unit at
// most. What bounds it is memory, and the chain of a wave, of which there are few
// rounds: both rows of a token and head by the same lanes took 27 us for 8177 tokens
// of 4 KB, a row each 21 (17.9 now).
template <typename T, int U, bool ONE>
__global__ void __launch_bounds__(kThreads) update_kernel(Q8Args p) {
  typedef typename Vec<T, U>::type In;
  typedef typename Vec<int8_t, U>::type Out;
  const Place x = place(p);
  const Side& w = p.side[x.kv];
  // (The row is loaded before the slot is looked at, so that both are under way together.)
  const char* row = w.src + times(x.t, w.ts) + times(x.head, w.hs);
  In first = {};
  if (x.lane < w.units) first = reinterpret_cast<const In*>(row)[x.lane];
  const int32_t slot = p.slots[x.t];
  float top = 0.f;
  if (!p.keep) {
    auto look = [&](const In& y) __attribute__((always_inline)) { top = fmaxf(top, largest<T, U>(y)); };
    look(first);
    if (!ONE)
      for (int u = x.lane + w.lanes; u < w.units; u += w.lanes) look(reinterpret_cast<const In*>(row)[u]);
    top = row_max(top, w.lanes);
  }
  if (!x.real || slot < 0 || slot >= p.slots_end) return;
  const int32_t pg = slot / p.page, at = slot - pg * (int32_t)p.page.d;
  float* scale = w.scale + times(pg, w.sp) + times(x.head, w.sh) + times(at, w.sr);
  float s;
  if (p.keep) {
    s = *scale;
  } else {
    s = top <= FLT_MAX ? top / 127.f : NAN;
    if (x.lane == 0) *scale = s;
  }
  const float inv = __builtin_amdgcn_rcpf(s);
  Out* out = reinterpret_cast<Out*>(w.dst + times(pg, w.cp) + times(x.head, w.ch) + times(at, w.cr));
  auto put = [&](int u, const In& y) __attribute__((always_inline)) {
    float v[U];
    int8_t c[U] = {};
#pragma unroll
    for (int i = 0; i < U; i++) v[i] = (float)y[i];
    if (s > 0.f) codes_of<U>(v, s, inv, p.keep, c);
    Out z;
#pragma unroll
    for (int i = 0; i < U; i++) z[i] = c[i];
    out[u] = z;
  };
  if (x.lane < w.units) put(x.lane, first);
  if (!ONE)
    for (int u = x.lane + w.lanes; u < w.units; u += w.lanes) put(u, reinterpret_cast<const In*>(row)[u]);
}

// The way back: unit by unit, a code's value c * s in 32 bits, rounded once
// more to the type; a cache of the type itself is copied.
template <typename C, typename T, int U>
__global__ void __launch_bounds__(kThreads) read_kernel(Q8Args p) {
  typedef typename Vec<C, U>::type In;
  typedef typename Vec<T, U>::type Out;
  const Place x = place(p);
  if (!x.real) return;
  const Side& w = p.side[x.kv];
  const int32_t slot = p.slots[x.t];
  const bool there = slot >= 0 && slot < p.slots_end;
  const int32_t pg = (there ? slot : 0) / p.page, at = (there ? slot : 0) - pg * (int32_t)p.page.d;
  const In* row = reinterpret_cast<const In*>(w.src + pg * w.cp + x.head * w.ch + at * w.cr);
  float s = 1.f;
  if constexpr (sizeof(C) == 1)
    if (there) s = w.scale[pg * w.sp + x.head * w.sh + at * w.sr];
  Out* out = reinterpret_cast<Out*>(w.dst + x.t * w.ts + x.head * w.hs);
  for (int u = x.lane; u < w.units; u += w.lanes) {
    Out z = {};
    if (there) {
      const In y = row[u];
#pragma unroll
      for (int i = 0; i < U; i++) {
        if constexpr (sizeof(C) == 1) z[i] = (T)((float)y[i] * s);
        else z[i] = y[i];
      }
    }
    out[u] = z;
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
    if (blocks * kThreads > INT32_MAX) return bi::fail(BI_EINVAL, "%s: sizes too large", who);
    w.blocks = (int32_t)blocks;
    all += blocks;
  }
  hipLaunchKernelGGL(kernel, dim3((unsigned)all), dim3(kThreads), 0, static_cast<hipStream_t>(stream), p);
  const hipError_t e = hipGetLastError();
  return e == hipSuccess ? BI_OK : bi::launch_error(e, who);
}

template <typename T> void (*update_for(bool wide, bool one))(Q8Args) {
  constexpr int U = 16 / sizeof(T);
  return !wide ? update_kernel<T, 1, false> : one ? update_kernel<T, U, true> : update_kernel<T, U, false>;
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
  const bool one = D * esz <= 1024 && V * esz <= 1024;  // 64 lanes of 16 bytes
  void (*f)(Q8Args);
  if (dtype == BI_F32) f = update_for<float>(wide, one);
  else if (dtype == BI_F16) f = update_for<_Float16>(wide, one);
  else f = update_for<__bf16>(wide, one);
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
