// Rotary positions of queries and keys (bi_rotary).
//
// Mathematics. Pair i of a head at position p turns by the angle p * f_i:
// (x, y) -> scale * (x cos - y sin, x sin + y cos). Pair i is the dims
// offset + i and offset + n + i, or offset + 2i and offset + 2i + 1; the other
// dims of a head are copied.
//
// The angle is taken in turns and in 64 bits, where p * (f_i / 2 pi) is off by
// 2^-52 of itself (at position 10^6 by 4e-11 turns), reduced there to half a
// turn, and rounded to 32 bits once (2^-26 turns, 9e-8 in the sine and
// cosine). Products and their sum are in 32 bits, rounded once to the type.
//
// What bounds it is memory: every value is read and written once. A thread
// takes 16 bytes of the first and 16 of the second dims of the same pairs (or
// 32 adjacent bytes) of several heads in turn, which share the angles.
#include <hip/hip_runtime.h>
#include <stdint.h>

#include "bi_div.h"
#include "bi_internal.h"

namespace {

using bi::Div;

constexpr int kThreads = 256;

struct RotaryArgs {
  const char* src[2];  // queries, keys
  char* dst[2];
  const int32_t* positions;
  const double* freq;  // (n) radians per position
  int64_t ss[2][2];    // source byte strides: token, head
  int64_t threads;     // of the launch that have work
  int32_t H, heads;    // query heads; query and key heads
  int32_t D, n, offset;
  int32_t turns;       // items of a head that turn; the others copy
  int32_t per;         // heads of a thread
  Div items, groups;   // items of a head, groups of heads
  float scale;
};

template <typename T, int U> struct Unit {
  typedef T type __attribute__((ext_vector_type(U)));
};

// T: element, U: elements per unit (16 bytes, or one where rows are not
// aligned to that), PAIR: pairs are adjacent dims.
template <typename T, int U, bool PAIR>
__global__ void __launch_bounds__(kThreads) rotary_kernel(RotaryArgs p) {
  typedef typename Unit<T, U>::type Vec;
  const int64_t id = (int64_t)blockIdx.x * kThreads + threadIdx.x;
  if (id >= p.threads) return;
  const int32_t hi = (int32_t)id / p.items, item = (int32_t)id - hi * (int32_t)p.items.d;
  const int32_t t = hi / p.groups, group = hi - t * (int32_t)p.groups.d;
  const int h0 = group * p.per, h1 = h0 + p.per < p.heads ? h0 + p.per : p.heads;
  const bool turn = item < p.turns;

  // The item's two units, by their first element.
  int a, b;
  bool both = true;
  if (turn) {
    a = p.offset + (PAIR ? 2 * U : U) * item;
    b = PAIR ? a + U : a + p.n;
  } else {
    const int u = 2 * (item - p.turns), before = p.offset / U, units = (p.D - 2 * p.n) / U;
    a = (u < before ? u : u + 2 * p.n / U) * U;
    b = (u + 1 < before ? u + 1 : u + 1 + 2 * p.n / U) * U;
    both = u + 1 < units;
  }

  float c[U], s[U];
  if (turn) {
    const double pos = (double)p.positions[t];
#pragma unroll
    for (int i = 0; i < U; i++) {
      double r = pos * (p.freq[U * item + i] * 0.15915494309189535);
      r -= __builtin_rint(r);
      sincospif(2.f * (float)r, &s[i], &c[i]);
      s[i] *= p.scale;
      c[i] *= p.scale;
    }
  }
  for (int h = h0; h < h1; h++) {
    const int kv = h >= p.H, head = kv ? h - p.H : h;
    const T* from = reinterpret_cast<const T*>(p.src[kv] + t * p.ss[kv][0] + head * p.ss[kv][1]);
    T* to = reinterpret_cast<T*>(p.dst[kv]) + ((int64_t)t * (kv ? p.heads - p.H : p.H) + head) * p.D;
    Vec x = *reinterpret_cast<const Vec*>(from + a), y = {};
    if (both) y = *reinterpret_cast<const Vec*>(from + b);
    if (turn) {
      float v[2 * U], w[2 * U];
#pragma unroll
      for (int i = 0; i < U; i++) v[i] = (float)x[i], v[U + i] = (float)y[i];
#pragma unroll
      for (int i = 0; i < U; i++) {
        const int m = PAIR ? 2 * i : i, n = PAIR ? 2 * i + 1 : U + i;
        w[m] = __builtin_fmaf(v[m], c[i], -(v[n] * s[i]));
        w[n] = __builtin_fmaf(v[m], s[i], v[n] * c[i]);
      }
#pragma unroll
      for (int i = 0; i < U; i++) x[i] = (T)w[i], y[i] = (T)w[U + i];
    }
    *reinterpret_cast<Vec*>(to + a) = x;
    if (both) *reinterpret_cast<Vec*>(to + b) = y;
  }
}

typedef void (*Kernel)(RotaryArgs);
template <typename T> Kernel pick(bool wide, bool pair) {
  constexpr int U = 16 / sizeof(T);
  if (wide) return pair ? rotary_kernel<T, U, true> : rotary_kernel<T, U, false>;
  return pair ? rotary_kernel<T, 1, true> : rotary_kernel<T, 1, false>;
}

}  // namespace

extern "C" int bi_rotary(const void* q, const void* k, void* q_out, void* k_out,
                         const int32_t* positions, const double* inv_freq, int64_t T, int64_t H,
                         int64_t Hkv, int64_t D, int64_t n, int64_t offset, const int64_t* strides,
                         float scale, int interleaved, int dtype, void* hip_stream) {
  const char* who = "bi_rotary";
  const int esz = bi::elem_size(dtype);
  if (!esz) return bi::fail(BI_EINVAL, "%s: unknown dtype %d", who, dtype);
  if (T < 0 || H < 0 || Hkv < 0 || D <= 0 || n < 0 || offset < 0 || D > (1 << 20) ||
      H > (1 << 20) || Hkv > (1 << 20) || T > INT32_MAX)
    return bi::fail(BI_EINVAL, "%s: bad sizes T=%lld H=%lld Hkv=%lld D=%lld", who, (long long)T,
                    (long long)H, (long long)Hkv, (long long)D);
  if (n > D / 2 || offset > D - 2 * n)
    return bi::fail(BI_EINVAL, "%s: %lld pairs from dim %lld on do not fit a head of %lld", who,
                    (long long)n, (long long)offset, (long long)D);
  if (T == 0 || H + Hkv == 0) return BI_OK;
  if ((H > 0 && (!q || !q_out)) || (Hkv > 0 && (!k || !k_out)) || !positions || !strides ||
      (n > 0 && !inv_freq))
    return bi::fail(BI_EINVAL, "%s: null pointer", who);
  RotaryArgs p;
  p.src[0] = static_cast<const char*>(q);
  p.src[1] = static_cast<const char*>(k);
  p.dst[0] = static_cast<char*>(q_out);
  p.dst[1] = static_cast<char*>(k_out);
  p.positions = positions;
  p.freq = inv_freq;
  uint64_t bits = (uint64_t)(D * esz) | (uint64_t)(n * esz) | (uint64_t)(offset * esz);
  for (int i = 0; i < 2; i++) {
    for (int j = 0; j < 2; j++) p.ss[i][j] = strides[2 * i + j] * esz;
    if (i == 0 ? H > 0 : Hkv > 0)
      bits |= (uint64_t)p.ss[i][0] | (uint64_t)p.ss[i][1] | (uintptr_t)p.src[i] | (uintptr_t)p.dst[i];
  }
  if (bits % esz) return bi::fail(BI_EINVAL, "%s: pointers not aligned to elements", who);
  const bool wide = bits % 16 == 0;
  const int64_t U = wide ? 16 / esz : 1;
  p.H = (int32_t)H;
  p.heads = (int32_t)(H + Hkv);
  p.D = (int32_t)D;
  p.n = (int32_t)n;
  p.offset = (int32_t)offset;
  p.turns = (int32_t)(n / U);
  p.scale = scale;
  const int64_t items = n / U + ((D - 2 * n) / U + 1) / 2;
  // Heads of a thread: eight, which then share the angles (64 bits, and some 30
  // operations for each sine and cosine), but fewer where that leaves the GPU
  // short of threads.
  int64_t per = 8;
  if (T > (INT32_MAX - kThreads) / (items * ((H + Hkv + per - 1) / per)))
    return bi::fail(BI_EINVAL, "%s: sizes too large", who);
  while (per > 1 && T * items * ((H + Hkv + per - 1) / per) < 256 * 1024) per /= 2;
  const int64_t groups = (H + Hkv + per - 1) / per;
  p.per = (int32_t)per;
  p.items = bi::make_div(items);
  p.groups = bi::make_div(groups);
  p.threads = T * groups * items;
  const Kernel f = dtype == BI_F32 ? pick<float>(wide, interleaved)
                   : dtype == BI_F16 ? pick<_Float16>(wide, interleaved)
                                     : pick<__bf16>(wide, interleaved);
  hipLaunchKernelGGL(f, dim3((unsigned)((p.threads + kThreads - 1) / kThreads)), dim3(kThreads), 0,
                     static_cast<hipStream_t>(hip_stream), p);
  const hipError_t e = hipGetLastError();
  return e == hipSuccess ? BI_OK : bi::launch_error(e, "bi_rotary launch");
}
