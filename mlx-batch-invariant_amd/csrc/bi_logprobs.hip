// Log probabilities of given tokens, the entropy and the largest logits of
// every row (bi_token_logprobs).
//
// Mathematics. With M the row's largest logit, d_i = x_i - M, S = sum e^(d_i)
// and U = sum e^(d_i) d_i: log p_t = d_t - ln S, and the entropy -sum p ln p =
// ln S - U / S, two parts that are not negative, so nothing cancels. A logit of
// -inf is a token that is ruled out and counts for nothing; a row with a NaN or
// +inf, and one of -inf alone, is NaN. M, S and U are in 32 bits.
//
// The k largest, ties to the lowest id. The threads form 256 groups (64 for up to
// 32); the k-th largest of the groups' largest logits bounds the k-th largest
// logit of all from below. What is not below it, k to 1.4 k logits of most rows,
// is put in order wave by wave, by insertion into a list that the lanes hold, and
// what the waves' lists hold is counted against each other.
//
// A workgroup has a row to itself and keeps it in registers (longer rows than
// these hold pass by and only the threads with a large logit read theirs once
// more), so that the row is read once and its bits do not depend on other rows.
// What bounds many rows is reading them; a few rows, the chain of a launch, the
// load, two reductions and the insertions.
#include <math.h>

#include <hip/hip_runtime.h>
#include <stdint.h>

#include "bi_internal.h"

namespace {

constexpr int kMostTop = 64;

struct LogprobArgs {
  const void* logits;
  const void* tokens;
  float* logprobs;
  float* entropy;
  int64_t* top_ids;
  float* top_logprobs;
  int64_t stride;  // elements between rows
  int32_t V, top;
  int32_t wide_tokens;  // tokens are of 64 bits
};

// Logits as whole numbers in their order; a NaN above all, both zeros alike.
__device__ __forceinline__ int32_t order_of(float x) {
  const int32_t b = __float_as_int(x + 0.f);
  return x == x ? b ^ ((b >> 31) & 0x7FFFFFFF) : INT32_MAX;
}
__device__ __forceinline__ float logit_of(int32_t o) {
  return __int_as_float(o ^ ((o >> 31) & 0x7FFFFFFF));
}
__device__ __forceinline__ float larger(float a, float b) { return __builtin_elementwise_maximum(a, b); }

// A wave's value of all lanes, by moves within a register: op is the same of (a, b)
// and (b, a), so all lanes have the same bits.
template <int CTRL> __device__ __forceinline__ float moved(float x) {
  return __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(x), CTRL, 0xF, 0xF, true));
}
template <typename Op> __device__ __forceinline__ float of_wave(float x, const Op& op) {
  x = op(x, moved<0xB1>(x));   // lane ^ 1
  x = op(x, moved<0x4E>(x));   // lane ^ 2
  x = op(x, moved<0x141>(x));  // 7 - lane of eight
  x = op(x, moved<0x140>(x));  // 15 - lane of sixteen
  const auto r = __builtin_amdgcn_permlane16_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  x = op(__uint_as_float(r[0]), __uint_as_float(r[1]));
  const auto t = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  return op(__uint_as_float(t[0]), __uint_as_float(t[1]));
}

// NT threads of NU units of 16 bytes each; HELD: all of a row is in these.
template <typename T, int NT, int NU, bool HELD>
__global__ void __launch_bounds__(NT, NT == 1024 ? 8 : 6) logprobs_kernel(LogprobArgs p) {
  constexpr int U = 16 / sizeof(T), NW = NT / 64, GROUP = NT / 256;
  // (Rows begin at any element: the element's place decides which thread has
  // it, whatever the row's alignment.)
  typedef T Vec __attribute__((ext_vector_type(U), aligned(sizeof(T))));
  __shared__ float4 s_group[64];
  __shared__ float2 s_sum[NW];
  __shared__ int32_t s_list[NW * kMostTop], s_id[NW * kMostTop];
  __shared__ int s_count;

  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const T* row = static_cast<const T*>(p.logits) + blockIdx.x * p.stride;
  if (tid == 0) s_count = 0;

  // Unit u of the row; what lies behind its end is -inf.
  auto load = [&](int64_t u) __attribute__((always_inline)) -> Vec {
    Vec x;
    if ((u + 1) * U <= p.V) {
      x = *reinterpret_cast<const Vec*>(row + u * U);
    } else {
#pragma unroll
      for (int i = 0; i < U; i++) x[i] = u * U + i < p.V ? row[u * U + i] : (T)-INFINITY;
    }
    return x;
  };
  const int64_t units = ((int64_t)p.V + U - 1) / U;
  const int rounds = HELD ? 1 : (int)((units + NT * NU - 1) / (NT * NU));

  Vec x[NU];
  float unit[NU];  // the largest of each (HELD)
  float m = -INFINITY, s = 0.f, ud = 0.f;
  auto add = [&](const Vec& v, float base) __attribute__((always_inline)) {
#pragma unroll
    for (int i = 0; i < U; i++) {
      const float d = (float)v[i] - base;
      const float e = __builtin_amdgcn_exp2f(d * 1.4426950408889634f);
      s += e;
      ud = __builtin_fmaf(e, fmaxf(d, -200.f), ud);  // (e is 0 there, and d may be -inf)
    }
  };
  for (int r = 0; r < rounds; r++) {
#pragma unroll
    for (int i = 0; i < NU; i++) x[i] = load(((int64_t)r * NU + i) * NT + tid);
    float top = m;
#pragma unroll
    for (int i = 0; i < NU; i++) {
      unit[i] = -INFINITY;
#pragma unroll
      for (int j = 0; j < U; j++) unit[i] = larger(unit[i], (float)x[i][j]);
      top = larger(top, unit[i]);
    }
    if constexpr (!HELD) {
      // The thread's own base moves to its largest so far.
      const float d = m - top, f = __builtin_amdgcn_exp2f(d * 1.4426950408889634f);
      if (m > -INFINITY) {
        ud = __builtin_fmaf(s, fmaxf(d, -200.f), ud) * f;
        s *= f;
      }
      if (!(top == -INFINITY))
#pragma unroll
        for (int i = 0; i < NU; i++) add(x[i], top);
    }
    m = top;
  }

  // The groups' largest, four to a lane, and of them the row's.
  float g = m;
  static_assert(GROUP == 1 || GROUP == 4, "lanes of a group");
  if constexpr (GROUP == 4) g = larger(g, moved<0xB1>(g)), g = larger(g, moved<0x4E>(g));
  if (lane % GROUP == 0) reinterpret_cast<float*>(s_group)[tid / GROUP] = g;
  __syncthreads();
  const float4 four = s_group[lane];
  g = larger(larger(four.x, four.y), larger(four.z, four.w));
  const float M = of_wave(g, larger);

  if constexpr (HELD) {
#pragma unroll
    for (int i = 0; i < NU; i++) add(x[i], M);
  } else {
    const float d = m - M, f = __builtin_amdgcn_exp2f(d * 1.4426950408889634f);
    ud = __builtin_fmaf(s, fmaxf(d, -200.f), ud) * f;
    s *= f;
    if (M == -INFINITY) s = NAN;
  }
  const auto plus = [](float a, float b) __attribute__((always_inline)) { return a + b; };
  s = of_wave(s, plus);
  ud = of_wave(ud, plus);
  if (lane == 0) s_sum[wave] = make_float2(s, ud);

  if (p.top) {
    // A number that `top` groups reach, the largest of 16 bits: bit by bit. (With the
    // other 16, which bf16 has not, a row of fp32 would have a few candidates less.)
    auto key_of = [](float v) __attribute__((always_inline)) { return (uint32_t)order_of(v) ^ 0x80000000u; };
    uint32_t bound = 0;
    if (p.top <= 32) {
      const uint32_t key = key_of(g);
#pragma unroll
      for (int b = 31; b >= 16; b--) {
        const uint32_t t = bound | (1u << b);
        if (__popcll(__builtin_amdgcn_ballot_w64(key >= t)) >= p.top) bound = t;
      }
    } else {
      const uint32_t key[4] = {key_of(four.x), key_of(four.y), key_of(four.z), key_of(four.w)};
#pragma unroll
      for (int b = 31; b >= 16; b--) {
        const uint32_t t = bound | (1u << b);
        int n = 0;
#pragma unroll
        for (int i = 0; i < 4; i++) n += __popcll(__builtin_amdgcn_ballot_w64(key[i] >= t));
        if (n >= p.top) bound = t;
      }
    }
    // As a logit. (A bound that is NaN, where `top` groups have one, is below none; so is
    // one between -inf and the smallest number, where fewer groups than `top` have any.)
    const float least = logit_of((int32_t)(bound ^ 0x80000000u));
    // The wave's list: lane n has the n-th largest so far.
    int32_t lo = INT32_MIN, lid = INT32_MAX;
    const bool mine = !(m < least);
    if (__builtin_amdgcn_ballot_w64(mine) != 0) {
      for (int r = 0; r < rounds; r++) {
        uint64_t bits = 0;
        static_assert(NU * U <= 64, "a bit for each element");
        const int64_t first = (int64_t)r * NU * NT + tid;
#pragma unroll
        for (int i = 0; i < NU; i++) {  // (most units have no candidate in any lane)
          if (!(HELD ? !(unit[i] < least) : mine)) continue;
          const Vec v = HELD ? x[i] : load(first + (int64_t)i * NT);
#pragma unroll
          for (int j = 0; j < U; j++) bits |= (uint64_t)!((float)v[j] < least) << (i * U + j);
        }
        const bool one = HELD && __popcll(bits) == 1;  // then it is the thread's largest
        while (__builtin_amdgcn_ballot_w64(bits != 0) != 0) {
          // A candidate of every lane that has one, put in one after the other.
          int32_t o = INT32_MIN, id = INT32_MAX;
          if (bits) {
            const int b = __builtin_ctzll(bits);
            bits &= bits - 1;
            const int64_t at = (first + (int64_t)(b / U) * NT) * U + b % U;
            if (at < p.V) id = (int32_t)at, o = order_of(one ? m : (float)row[at]);
          }
          // (Of more candidates than `top`, as equal logits and ruled-out ones give, most do
          // not get past the list's last: one by one 32000 of them took 229 us.)
          const int32_t lasto = __builtin_amdgcn_readlane(lo, p.top - 1), lastid = __builtin_amdgcn_readlane(lid, p.top - 1);
          uint64_t todo = __builtin_amdgcn_ballot_w64(id != INT32_MAX && (o > lasto || (o == lasto && id < lastid)));
          while (todo) {
            const int from = __builtin_ctzll(todo);
            todo &= todo - 1;
            const int32_t co = __builtin_amdgcn_readlane(o, from), cid = __builtin_amdgcn_readlane(id, from);
            const bool before = lo > co || (lo == co && lid < cid);
            const int at = __popcll(__builtin_amdgcn_ballot_w64(before));
            if (at >= p.top) continue;
            // The lane before's (shifted through the whole wave).
            const int32_t po = __builtin_amdgcn_update_dpp(0, lo, 0x138, 0xF, 0xF, false);
            const int32_t pid = __builtin_amdgcn_update_dpp(0, lid, 0x138, 0xF, 0xF, false);
            lo = lane > at ? po : lane == at ? co : lo;
            lid = lane > at ? pid : lane == at ? cid : lid;
          }
        }
      }
    }
    const bool has = lid != INT32_MAX && lane < p.top;
    const int n = __popcll(__builtin_amdgcn_ballot_w64(has));
    int to = 0;
    if (lane == 0 && n) to = atomicAdd(&s_count, n);  // (in any order: their ranks decide)
    to = __builtin_amdgcn_readfirstlane(to);
    if (has) s_list[to + lane] = lo, s_id[to + lane] = lid;
  }
  __syncthreads();

  // What is left is one wave's, but for more candidates than it has lanes.
  const int n = p.top ? s_count : 0;
  if (n <= 64 && wave != 0) return;
  float S = 0.f, UD = 0.f;
#pragma unroll
  for (int w = 0; w < NW; w++) {
    S += s_sum[w].x;
    UD += s_sum[w].y;
  }
  const float ln = logf(S);
  const int64_t r = blockIdx.x;
  if (tid == 0) {
    const int64_t t = p.wide_tokens ? static_cast<const int64_t*>(p.tokens)[r]
                                    : static_cast<const int32_t*>(p.tokens)[r];
    p.logprobs[r] = t >= 0 && t < p.V ? (float)row[t] - M - ln : NAN;
    p.entropy[r] = ln - UD / S;
  }
  if (p.top) {
    auto put = [&](int32_t o, int32_t id, int rank) __attribute__((always_inline)) {
      if (rank >= p.top) return;
      p.top_ids[r * p.top + rank] = id;
      p.top_logprobs[r * p.top + rank] = logit_of(o) - M - ln;
    };
    if (n <= 64) {  // one wave, its lanes' candidates against each other
      const int32_t o = lane < n ? s_list[lane] : INT32_MIN, id = lane < n ? s_id[lane] : INT32_MAX;
      int rank = lane < n ? 0 : kMostTop;
      for (int j = 0; j < n; j++) {
        const int32_t oj = __builtin_amdgcn_readlane(o, j), idj = __builtin_amdgcn_readlane(id, j);
        rank += oj > o || (oj == o && idj < id);
      }
      put(o, id, rank);
    } else {
      for (int i = tid; i < n; i += NT) {
        const int32_t o = s_list[i], id = s_id[i];
        int rank = 0;
        for (int j = 0; j < n; j++) rank += s_list[j] > o || (s_list[j] == o && s_id[j] < id);
        put(o, id, rank);
      }
    }
  }
}

// Rows of a launch: its threads are counted in 32 bits, and of those that pass them it
// starts the rest of a division by 2^32, without an error.
constexpr int64_t kMostRows = 1 << 21;

template <typename T> int start(LogprobArgs p, int64_t rows, hipStream_t st) {
  constexpr int U = 16 / sizeof(T), NU = 32 / U;
  for (;;) {
    const int64_t n = rows < kMostRows ? rows : kMostRows;
    const dim3 grid((unsigned)n);
    // By the row's length alone, so that its bits are the same in every call.
    if (p.V <= 256 * 32) hipLaunchKernelGGL((logprobs_kernel<T, 256, NU, true>), grid, dim3(256), 0, st, p);
    else if (p.V <= 1024 * 32) hipLaunchKernelGGL((logprobs_kernel<T, 1024, NU, true>), grid, dim3(1024), 0, st, p);
    else hipLaunchKernelGGL((logprobs_kernel<T, 1024, NU, false>), grid, dim3(1024), 0, st, p);
    const hipError_t e = hipGetLastError();
    if (e != hipSuccess) return bi::launch_error(e, "bi_token_logprobs launch");
    if ((rows -= n) == 0) return BI_OK;
    p.logits = static_cast<const T*>(p.logits) + n * p.stride;
    p.tokens = static_cast<const char*>(p.tokens) + n * (p.wide_tokens ? 8 : 4);
    p.logprobs += n, p.entropy += n;
    if (p.top) p.top_ids += n * p.top, p.top_logprobs += n * p.top;
  }
}

}  // namespace

extern "C" int bi_token_logprobs(const void* logits, const void* tokens, float* logprobs, float* entropy,
                                 int64_t* top_ids, float* top_logprobs, int64_t rows, int64_t V,
                                 int64_t stride, int64_t top, int token_bytes, int dtype,
                                 void* hip_stream) {
  const char* who = "bi_token_logprobs";
  const int esz = bi::elem_size(dtype);
  if (!esz) return bi::fail(BI_EINVAL, "%s: unknown dtype %d", who, dtype);
  if (rows < 0 || V <= 0 || rows > INT32_MAX || V > (1 << 30) || stride < 0)
    return bi::fail(BI_EINVAL, "%s: bad sizes rows=%lld V=%lld", who, (long long)rows, (long long)V);
  if (top < 0 || top > kMostTop || top > V)
    return bi::fail(BI_EINVAL, "%s: top=%lld is not between 0 and %d and at most V=%lld", who,
                    (long long)top, kMostTop, (long long)V);
  if (token_bytes != 4 && token_bytes != 8)
    return bi::fail(BI_EINVAL, "%s: tokens are of 4 or 8 bytes, not %d", who, token_bytes);
  if (rows == 0) return BI_OK;
  if (!logits || !tokens || !logprobs || !entropy || (top > 0 && (!top_ids || !top_logprobs)))
    return bi::fail(BI_EINVAL, "%s: null pointer", who);
  if ((uintptr_t)logits % esz) return bi::fail(BI_EINVAL, "%s: logits not aligned to elements", who);
  LogprobArgs p = {logits, tokens, logprobs, entropy, top_ids, top_logprobs, stride, (int32_t)V,
                   (int32_t)top, token_bytes == 8};
  const hipStream_t st = static_cast<hipStream_t>(hip_stream);
  return dtype == BI_F32 ? start<float>(p, rows, st)
         : dtype == BI_F16 ? start<_Float16>(p, rows, st)
                           : start<__bf16>(p, rows, st);
}
