// Batch-invariant attention over a paged cache or over contiguous keys, with
// an optional sliding window and first tokens that stay visible: the kernel
// templates, included by one unit per head-dim pair (bi_paged_attn_d*.hip).
//
// Mathematics. A column is one (query head, token) pair; the columns of a
// request that share a kv head read the same keys. Scores are s_j = raw_j * a
// with raw_j = q . k_j and a = |scale| * log2 e (a negative scale negates q),
// and out = sum_j 2^(s_j) v_j / (sum_j 2^(s_j) + 2^(sink * log2 e)) over the
// rows j that the token sees.
//
// Fixed arithmetic of a column (what makes its bits independent of the call):
//   * Rows are taken by their position in the request: steps of kStep rows (64
//     where a row of keys and of values is at most 256 bytes, else 32), eight
//     steps (fp32: four) to a segment.
//   * raw_j is a chain of 32x32 matrix products over the head dim from +0.0:
//     of 16 dims for 16-bit types, of 2 for fp32; 16-byte chunks 2t and 2t + 1
//     of the rows enter product t (fp32: products 4t .. 4t + 3).
//   * Within a segment the running base m moves at a step whose largest seen
//     score M exceeds m + 6, to the next multiple of 4 from M on. p_j =
//     2^(fma(raw_j, a, -m)), 0 for an unseen row (whose raw_j is -inf); l =
//     l * f + (the step's sum of p, in a fixed order per lane half); o = o * f, then o += v . p by 32x32
//     products over the step's rows in ascending order, p rounded once to the
//     type (the products of bf16 and f16 take such operands), and l sums what
//     was rounded. f is a power of two, as every base is an integer.
//   * Segments start from nothing and are folded in ascending order: with M'
//     the larger base, O = fma(o, 2^(m - M'), O * 2^(M - M')), L alike.
//   * The sink enters last: out = (O * e) / (L * e + 2^(sink2 - X)) + 0.0, X the
//     larger of M and sink2, e = 2^(M - X), the division by a product with the
//     rounded inverse; rounded once to the type.
// A step or segment that a column sees nothing of leaves it as it is, so which
// of them a workgroup walks for its other columns changes no bits (a zero's
// sign would: hence the + 0.0).
// A value row that only some of a workgroup's tokens see is loaded, and p = 0
// times an infinity or NaN in it would be NaN for the others. The values of the
// steps that not all tokens see whole (a prompt's diagonal, a window's ends) are
// looked at as they pass; where one of them is infinite or NaN, the workgroup
// computes its tokens once more one by one (a split one by its own loop, a whole
// one by token_segment). The look costs 4096 tokens over 8192 rows 427 -> 434
// us, prompts of 8192 tokens under a window of 1024 188 -> 191, of 64 62.7 ->
// 65.7. (With NaN in every value the first takes 58 ms.)
//
// Two routes, the same bits:
//   * split: a workgroup per (request, kv head, up to 32 columns, segment),
//     whose four waves take a step each at a time; a second kernel folds the
//     segments. For few columns, where what bounds it is reading the cache.
//   * whole: a workgroup per 128 or 256 columns walks all their steps, 32
//     columns per wave, keys and values through a ring of LDS buffers. For
//     chunks of a prompt, where the matrix products and the exponentials bound
//     it.
// A segment is long enough that writing its results costs little beside
// reading it, and short enough that one long sequence fills the GPU.
#pragma once

#include <float.h>
#include <math.h>

#include <type_traits>

#include "bi_paged_attn.h"

namespace bi_paged {
namespace {

typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef short i16x4 __attribute__((ext_vector_type(4)));
typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef float f32x2 __attribute__((ext_vector_type(2)));
typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
typedef __attribute__((address_space(3))) void lds_void;
typedef __attribute__((address_space(3))) i16x4 lds_i16x4;

constexpr float kNone = -FLT_MAX;  // the base of a column that has seen nothing

// What loads of rows that nobody sees read: products with them are 0.
__device__ const uint4 g_zero_row[64] = {};

// One request: its tokens t0 .. t0 + L - 1 sit at rows n - L .. n - 1.
struct Request {
  int64_t t0;
  int32_t L, n;
  bool beyond;  // past max_query or max_seq
};
__device__ __forceinline__ Request request(const Args& p, int r) {
  Request q;
  if (p.qstart) {
    int32_t a = p.qstart[r], b = p.qstart[r + 1];
    a = a < 0 ? 0 : a > p.T ? p.T : a;
    b = b < a ? a : b > p.T ? p.T : b;
    q.t0 = a;
    q.L = b - a;
    q.n = p.seq[r] < 0 ? 0 : p.seq[r];
    q.beyond = q.L > p.max_query || q.n > p.max_seq;
  } else {
    q.t0 = 0;
    q.L = p.qL;
    q.n = p.N;
    q.beyond = false;
  }
  return q;
}

// The units (steps or segments of `size` rows) that tokens at positions lo ..
// hi see some row of: [0, a) and [b, e).
struct Walk {
  int32_t a, b, e;
  __device__ __forceinline__ int count() const { return a + (e - b); }
  __device__ __forceinline__ int unit(int i) const { return i < a ? i : b + (i - a); }
  // How many of them are before unit u.
  __device__ __forceinline__ int below(int u) const {
    const int late = (u < e ? u : e) - b;
    return (u < a ? u : a) + (late > 0 ? late : 0);
  }
};
__device__ __forceinline__ Walk walk(const Args& p, int32_t lo, int32_t hi, int size) {
  Walk w;
  w.e = hi < 0 ? 0 : hi / size + 1;
  w.a = w.b = 0;
  if (p.window) {
    const int32_t first = p.first < hi + 1 ? p.first : hi + 1;
    w.a = first <= 0 ? 0 : (first - 1) / size + 1;
    const int32_t start = lo - p.window + 1;
    w.b = start <= 0 ? 0 : start / size;
    if (w.b > w.e) w.b = w.e;
    if (w.b < w.a) w.b = w.a;
  }
  return w;
}
// Whether a token at lo .. hi may see one of rows j .. j + size - 1; whether all see all.
__device__ __forceinline__ bool any_seen(const Args& p, int32_t lo, int32_t hi, int32_t j, int size) {
  return j <= hi && (p.window == 0 || j + size - 1 > lo - p.window || j < p.first);
}
__device__ __forceinline__ bool all_seen(const Args& p, int32_t lo, int32_t hi, int32_t j, int size) {
  return j + size - 1 <= lo && (p.window == 0 || j > hi - p.window || j + size - 1 < p.first);
}
// Bits 0 .. d of 64 (none for d < 0).
__device__ __forceinline__ uint64_t bits_to(int32_t d) {
  return d < 0 ? 0ull : d >= 63 ? ~0ull : (2ull << d) - 1;
}
// Bit n: a token at `pos` sees row key0 + n, if it is mapped.
__device__ __forceinline__ uint64_t seen_bits(const Args& p, int32_t pos, int32_t key0, uint64_t mapped) {
  uint64_t b = bits_to(pos - key0);
  if (p.window) b &= ~bits_to(pos - p.window - key0) | bits_to(p.first - 1 - key0);
  return b & mapped;
}

// A row's table entry as it stands (loaded without a branch, so that nothing
// waits for it before it is used), and what it says: the row's page, the
// request for contiguous keys, -1 for none.
__device__ __forceinline__ int32_t table_column(const Args& p, int32_t key) {
  return (key < 0 ? 0 : key) / p.page;
}
__device__ __forceinline__ int32_t entry_of(const Args& p, int r, int32_t key) {
  if (!p.qstart || p.W == 0) return 0;
  const int32_t c = table_column(p, key);
  return p.table[r * p.table_stride + (c < p.W ? c : p.W - 1)];
}
__device__ __forceinline__ int32_t page_of(const Args& p, int r, int32_t entry, int32_t key) {
  if (!p.qstart) return r;
  return table_column(p, key) < p.W && entry < p.pages ? entry : -1;
}
__device__ __forceinline__ int32_t row_of(const Args& p, int32_t key) {
  if (!p.qstart) return key;
  return key - key / p.page * (int32_t)p.page.d;
}

// The kernel's arguments, read again: for what is needed seldom, so that it is not
// kept in registers meanwhile.
__device__ __forceinline__ const Args& args_again() {
  typedef __attribute__((address_space(4))) const Args KernelArgs;
  KernelArgs* args = (KernelArgs*)__builtin_amdgcn_kernarg_segment_ptr();
  asm volatile("" : "+s"(args));
  return *(const Args*)args;
}

__device__ __forceinline__ int opaque(int x) {
  asm volatile("" : "+v"(x));
  return x;
}
// Runs `use(n, operand)` for n = 0 .. N - 1 with the operands `read(n)` from LDS
// four products ahead. (Left to itself the compiler reads each operand right
// before its product, which then waits out the LDS latency.)
template <int N, typename Read, typename Use>
__device__ __forceinline__ void feed(const Read& read, const Use& use) {
  static_assert(N % 4 == 0, "groups of four");
  uint4 x[2][4];
#pragma unroll
  for (int i = 0; i < 4; i++) x[0][i] = read(i);
#pragma unroll
  for (int n = 0; n < N; n += 4) {
    __builtin_amdgcn_sched_barrier(0);
    if (n + 4 < N)
#pragma unroll
      for (int i = 0; i < 4; i++) x[(n / 4 + 1) & 1][i] = read(n + 4 + i);
    __builtin_amdgcn_sched_barrier(0);
#pragma unroll
    for (int i = 0; i < 4; i++) use(n + i, x[(n / 4) & 1][i]);
  }
}
__device__ __forceinline__ uint64_t uniform(uint64_t x) {
  return ((uint64_t)(uint32_t)__builtin_amdgcn_readfirstlane((uint32_t)(x >> 32)) << 32) |
         (uint32_t)__builtin_amdgcn_readfirstlane((uint32_t)x);
}
// 16 or 4 bytes from each lane's address to LDS at `to` + 16 or 4 * lane (`to` uniform),
// in flight until wait_loads(). As asm, since beside the builtin, which the
// compiler counts as an access of both memories, it waits for all LDS reads
// and all loads wherever it waits for one. It has no result that could be
// taken before it is there; the caller waits and meets a barrier before it
// reads the LDS. (M0, which nothing else here uses, holds the LDS address.)
template <int BYTES> __device__ __forceinline__ void load_to_lds(const void* from, void* to) {
  const uint32_t at = __builtin_amdgcn_readfirstlane((uint32_t)(uintptr_t)(lds_void*)to);
  if constexpr (BYTES == 16)
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, off"
                 :: "s"(at), "v"(from) : "memory");
  else
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dword %1, off"
                 :: "s"(at), "v"(from) : "memory");
}
template <int N> __device__ __forceinline__ void wait_loads_but() {  // all but the N youngest
  static_assert(N <= 63, "vmcnt range");
  asm volatile("s_waitcnt vmcnt(%0)" ::"i"(N) : "memory");
}
__device__ __forceinline__ void wait_loads() { asm volatile("s_waitcnt vmcnt(0)" ::: "memory"); }
// LDS written before is visible to the workgroup after; loads stay in flight.
__device__ __forceinline__ void barrier() {
  asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory");
}

__device__ __forceinline__ float half_swap_max(float x) {
  const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  return __builtin_elementwise_maximum(__uint_as_float(r[0]), __uint_as_float(r[1]));
}
__device__ __forceinline__ float half_swap_sum(float x) {
  const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  return __uint_as_float(r[0]) + __uint_as_float(r[1]);
}
// 2^e for an integer e that is at most 0 (0 far below).
__device__ __forceinline__ float pow2(float e) {
  return __builtin_amdgcn_ldexpf(1.f, (int)fmaxf(e, -300.f));
}
// The base after a step whose largest seen raw score is `top` (-inf: none seen):
// p is at most 2^kRise, and above 2^-4 for the largest score of a segment's
// first step (f16 holds p to 2^-25).
// A sum of rounded p up to kMostSum holds none of a score above the base +
// kRise, whose p is 64 and rounds to no less than 63.75 in any type, with the
// exponential's own error.
constexpr float kRise = 6.f, kMostSum = 63.f;
__device__ __forceinline__ float next_base(float m, float top, float a) {
  const float s = top * a;
  return top > -INFINITY && s > m + kRise ? ceilf(s * 0.25f) * 4.f : m;
}
// Folds a segment's (m, l) into the running (M, L); fa and fb scale O and o.
__device__ __forceinline__ void fold_base(float& M, float& L, float m, float l, float& fa, float& fb) {
  const float n = fmaxf(M, m);
  fa = pow2(M - n);
  fb = pow2(m - n);
  M = n;
  L = __builtin_fmaf(l, fb, L * fa);
}
// The sink's part: what scales O and the denominator.
__device__ __forceinline__ void finish(float M, float L, float sink2, bool has, float& e, float& den) {
  e = 1.f;
  den = L;
  if (has) {
    const float x = fmaxf(M, sink2);
    e = __builtin_amdgcn_exp2f(M - x);
    den = __builtin_fmaf(L, e, __builtin_amdgcn_exp2f(sink2 - x));
  }
}
__device__ __forceinline__ float inverse(float den) { return den == 0.f ? 0.f : 1.f / den; }
template <typename T> __device__ __forceinline__ T result(float O, float e, float inv) {
  return (T)__builtin_fmaf(O * e, inv, 0.f);
}

template <typename T, int D_, int V_>
struct Geo {
  static constexpr int D = D_, V = V_;
  static constexpr int E = sizeof(T);
  static constexpr int kStep = (D > V ? D : V) * E <= 256 ? 64 : 32;
  // Steps to a segment; half as many for fp32, whose rows and products take
  // twice as long and more.
  static constexpr int kSegSteps = E == 2 ? 8 : 4;
  static constexpr int kSeg = kSegSteps * kStep;
  static constexpr int KT = kStep / 32;       // score tiles per step
  static constexpr int CH = D * E / 16;       // 16-byte chunks per key row
  static constexpr int VCH = V * E / 16;      // per value row
  static constexpr int MCH = CH > VCH ? CH : VCH;
  static constexpr int NQ = CH / 2;           // chunks per lane half
  static constexpr int PU = E;                // 16-byte units of p per tile and lane
  static constexpr int DT = V / 32;           // tiles of output dims
  // Whole route: two waves per SIMD (256 registers each) hold o, O, the query
  // and a step's scores; LDS buffers that fit a CU with one workgroup.
  static constexpr bool kTwoWaves = V + 4 * NQ <= 192;
  static constexpr int kStepBytes = kStep * (CH + VCH) * 16;
  static constexpr int kDeep = kStepBytes <= 32768 ? 4 : 3;
  // Split workgroups of NC columns per CU: two where its 160 KB of LDS hold their
  // values (4 steps), p, row addresses, largest scores and sums twice.
  static constexpr int split_per_cu(int NC) {
    return 4 * kStep * MCH * 16 + 4 * KT * PU * 2 * NC * 16 + 2 * 4 * kStep * 8 + 4 * 3 * NC * 4 <= 81920 ? 2 : 1;
  }
  // Times for the choice of route, microseconds, fitted to both routes of every
  // head dim at two head layouts and 19 sizes (one to 64 requests of one to
  // 2048 tokens over 300 to 8192 rows). A row of a whole workgroup's walk: over
  // 8192 rows 16-bit 15.3, 18.6, 20.0, 31.7, 53.2 and 62.5 ns for 64/64, 96/96,
  // 128/128, 192/128, 192/192 and 256/256, fp32 (4096 rows) 68, 108, 136, 195,
  // 248 and 317: the products and, for 16 bits, the exponentials, more where
  // steps are of 32 rows, and twice that where one wave per SIMD has nothing
  // beside it.
  static constexpr double row_us() {
    return 1e-3 * (E == 4 ? 0.53 * (D + V) * (kTwoWaves ? 1.0 : 1.17)
                   : kTwoWaves ? (10.8 + 0.0345 * (D + V)) * (kStep == 64 ? 1.0 : 1.45)
                               : 26.0 + 0.071 * (D + V));
  }
  // A full segment's workgroups that a CU runs together, by the segment's size
  // (64 to 256 KB): 16-bit 10.8, 12.5, 11.8, 13.2, 16.2 and 20.3 us for the same
  // head dims at 32 columns, fp32 12.2, 14.3, 11.5, 14.1, 17.7 and 22.5, with
  // what their results cost.
  static constexpr double seg_us(int NC) {
    const double kb = kSeg * (D + V) * E / 1024.0;
    return E == 4 ? (3.0 + 0.06 * kb) * (split_per_cu(NC) == 2 ? 1.3 : 1.0) : 5.5 + 0.023 * kb;
  }

  // The lane's chunk pair t of keys and query: one product (fp32: four).
  __device__ __forceinline__ static f32x16 score(uint4 k, uint4 q, f32x16 c) {
    if constexpr (__is_same(T, __bf16)) {
      return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8, k),
                                                     __builtin_bit_cast(bf16x8, q), c, 0, 0, 0);
    } else if constexpr (__is_same(T, _Float16)) {
      return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(f16x8, k),
                                                    __builtin_bit_cast(f16x8, q), c, 0, 0, 0);
    } else {
      c = __builtin_amdgcn_mfma_f32_32x32x2f32(__uint_as_float(k.x), __uint_as_float(q.x), c, 0, 0, 0);
      c = __builtin_amdgcn_mfma_f32_32x32x2f32(__uint_as_float(k.y), __uint_as_float(q.y), c, 0, 0, 0);
      c = __builtin_amdgcn_mfma_f32_32x32x2f32(__uint_as_float(k.z), __uint_as_float(q.z), c, 0, 0, 0);
      return __builtin_amdgcn_mfma_f32_32x32x2f32(__uint_as_float(k.w), __uint_as_float(q.w), c, 0, 0, 0);
    }
  }
  // Element i of a tile is row 8 (i / 4) + 4 half + i % 4.
  __device__ __forceinline__ static int row(int i, int half) { return 8 * (i >> 2) + 4 * half + (i & 3); }
  // Row 32 kt + r's chunk 2 t + half. (Where a row's chunks are a power of two,
  // 2t only flips bits of the place at t = 0.)
  __device__ __forceinline__ static uint4 key_chunk(const uint4* k, int kt, int r, int t, int half) {
    const char* at = reinterpret_cast<const char*>(k + 32 * kt * CH);
    if constexpr ((CH & (CH - 1)) == 0) at += ((r * CH + (half ^ kswz(r))) * 16) ^ (32 * t);
    else at += (r * CH + ((2 * t + half) ^ kswz(r))) * 16;
    return __builtin_bit_cast(uint4, *reinterpret_cast<const u32x4*>(at));
  }
  // The largest score. (As the IEEE maximum, of which there is an instruction of
  // three operands; fmaxf would first quiet both of its own. A NaN score makes
  // its column NaN in any case.)
  __device__ __forceinline__ static float top(const f32x16 (&s)[KT]) {
    float m = -INFINITY;
#pragma unroll
    for (int kt = 0; kt < KT; kt++)
#pragma unroll
      for (int i = 0; i < 16; i += 2)
        m = __builtin_elementwise_maximum(__builtin_elementwise_maximum(m, s[kt][i]), s[kt][i + 1]);
    return half_swap_max(m);
  }
  // Scores of unseen rows become -inf; `seen` is shifted by the half's 4 rows.
  __device__ __forceinline__ static void hide(f32x16 (&s)[KT], uint64_t seen) {
#pragma unroll
    for (int kt = 0; kt < KT; kt++) {
      const uint32_t w = (uint32_t)(seen >> (32 * kt));
#pragma unroll
      for (int i = 0; i < 16; i++) s[kt][i] = w & (1u << row(i, 0)) ? s[kt][i] : -INFINITY;
    }
  }
  // p of a tile rounded to the type: unit u holds elements (16 / PU) u ...
  __device__ __forceinline__ static void pack(const f32x16& p, uint4 (&u)[PU]) {
    if constexpr (E == 2) {
#pragma unroll
      for (int j = 0; j < 2; j++) {
        uint32_t w[4];
#pragma unroll
        for (int i = 0; i < 4; i++) {
          const f32x2 d = {p[8 * j + 2 * i], p[8 * j + 2 * i + 1]};
          if constexpr (__is_same(T, __bf16)) {
            w[i] = __builtin_bit_cast(uint32_t, __builtin_convertvector(d, bf16x2));
          } else {
            w[i] = (uint32_t)__builtin_bit_cast(unsigned short, (_Float16)d[0]) |
                   ((uint32_t)__builtin_bit_cast(unsigned short, (_Float16)d[1]) << 16);
          }
        }
        u[j] = make_uint4(w[0], w[1], w[2], w[3]);
      }
    } else {
#pragma unroll
      for (int j = 0; j < 4; j++)
        u[j] = make_uint4(__float_as_uint(p[4 * j]), __float_as_uint(p[4 * j + 1]),
                          __float_as_uint(p[4 * j + 2]), __float_as_uint(p[4 * j + 3]));
    }
  }
  // A lane's sum of the step's p as they were rounded, so that what is divided
  // by is what was multiplied with: a chain per unit, units in pairs.
  __device__ __forceinline__ static float sum(const uint4 (&u)[KT][PU]) {
    float s[KT * PU];
#pragma unroll
    for (int i = 0; i < KT * PU; i++) {
      const uint4 x = u[i / PU][i % PU];
      const uint32_t w[4] = {x.x, x.y, x.z, x.w};
      s[i] = 0.f;
#pragma unroll
      for (int j = 0; j < 4; j++) {
        if constexpr (__is_same(T, __bf16))
          s[i] = __builtin_amdgcn_fdot2_f32_bf16(__builtin_bit_cast(bf16x2, w[j]),
                                                 __builtin_bit_cast(bf16x2, 0x3F803F80u), s[i], false);
        else if constexpr (__is_same(T, _Float16))
          s[i] = __builtin_amdgcn_fdot2(__builtin_bit_cast(f16x2, w[j]),
                                        __builtin_bit_cast(f16x2, 0x3C003C00u), s[i], false);
        else
          s[i] = j == 0 ? __uint_as_float(w[0]) : s[i] + __uint_as_float(w[j]);
      }
    }
#pragma unroll
    for (int d = 1; d < KT * PU; d *= 2)
#pragma unroll
      for (int i = 0; i + d < KT * PU; i += 2 * d) s[i] += s[i + d];
    return s[0];
  }

  // Sums of these over any elements have a bit of kOdd set if one of them is an
  // infinity or NaN.
  static constexpr uint32_t kExp = E == 4 ? 0x7F800000u : __is_same(T, __bf16) ? 0x7F807F80u : 0x7C007C00u;
  static constexpr uint32_t kOne = E == 4 ? 0x00800000u : __is_same(T, __bf16) ? 0x00800080u : 0x04000400u;
  static constexpr uint32_t kOdd = E == 4 ? 0x80000000u : 0x80008000u;
  __device__ __forceinline__ static uint32_t odd(uint4 x) {
    return ((x.x & kExp) + kOne) | ((x.y & kExp) + kOne) | ((x.z & kExp) + kOne) | ((x.w & kExp) + kOne);
  }
  // Values in LDS: row r's chunk c at chunk c ^ vswz(r). A transposing read
  // takes 4 consecutive rows, 64 bytes each, per pass (32 lanes of 8 bytes);
  // the exchange puts these in different quarters of the 64 banks. (Rows of
  // an odd multiple of 64 bytes lie so by themselves.)
  __device__ __forceinline__ static int vswz(int r) {
    if constexpr (E == 4) return 0;
    else if constexpr (VCH % 16 == 0) return (r & 3) << 2;
    else if constexpr (VCH % 8 == 0) return ((r >> 1) & 1) << 2;
    else return 0;
  }
  // Keys in LDS: a read takes one chunk of 16 rows per pass (16 lanes of 16 bytes).
  __device__ __forceinline__ static int kswz(int r) {
    if constexpr (CH % 16 == 0) return r & 15;
    else if constexpr (CH % 8 == 0) return (r >> 1) & 7;
    else return (r >> 2) & 3;
  }

  // The values' operand of product u of a tile: LDS rows row0 + 0 .. 31, those
  // of p's unit u, output dims 32 dt ...
  __device__ __forceinline__ static uint4 value(const uint4* v, int row0, int u, int dt, int lane) {
    const int half = lane >> 5;
    if constexpr (E == 2) {
      const int g = lane >> 4, i = lane & 15;
      const int rr = i >> 2, piece = i & 3;
      const int c = dt * 4 + (g & 1) * 2 + (piece >> 1);
      i16x4 a[2];
#pragma unroll
      for (int x = 0; x < 2; x++) {
        const int r = row0 + 16 * u + 8 * x + 4 * half + rr;
        const char* at = reinterpret_cast<const char*>(v + r * VCH + (c ^ vswz(r))) + 8 * (piece & 1);
        a[x] = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_i16x4*)at);
      }
      const uint2 lo = __builtin_bit_cast(uint2, a[0]), hi = __builtin_bit_cast(uint2, a[1]);
      return make_uint4(lo.x, lo.y, hi.x, hi.y);
    } else {
      uint32_t a[4];
#pragma unroll
      for (int e = 0; e < 4; e++)
        a[e] = reinterpret_cast<const uint32_t*>(v + (row0 + 8 * u + 4 * half + e) * VCH)[32 * dt + (lane & 31)];
      return make_uint4(a[0], a[1], a[2], a[3]);
    }
  }
};

// A load from device memory. (From a generic pointer, such as one kept in LDS,
// it would be a flat load, which counts as an LDS access too and makes every
// later wait one for all loads.)
__device__ __forceinline__ uint4 ld16(const void* p) {
  typedef __attribute__((address_space(1))) const u32x4 gvec;
  return __builtin_bit_cast(uint4, *(gvec*)p);
}
// One whose line is not wanted again.
__device__ __forceinline__ uint4 ld16_once(const void* p) {
  typedef __attribute__((address_space(1))) const u32x4 gvec;
  return __builtin_bit_cast(uint4, __builtin_nontemporal_load((gvec*)p));
}

__device__ __forceinline__ void st16(uint4* p, uint4 v) {
  *reinterpret_cast<u32x4*>(p) = __builtin_bit_cast(u32x4, v);
}

// A column's query as the products' operand: chunks 2t + half.
template <typename G>
__device__ __forceinline__ void load_query(const char* q, int half, uint4 (&out)[G::NQ]) {
#pragma unroll
  for (int t = 0; t < G::NQ; t++) out[t] = ld16(q + (2 * t + half) * 16);
}
template <typename G>
__device__ __forceinline__ void sign_query(const Args& p, uint4 (&q)[G::NQ]) {
#pragma unroll
  for (int t = 0; t < G::NQ; t++)
    q[t] = make_uint4(q[t].x ^ p.qsign, q[t].y ^ p.qsign, q[t].z ^ p.qsign, q[t].w ^ p.qsign);
}
template <typename T>
__device__ __forceinline__ const char* query_at(const Args& p, int r, const Request& rq, int i, int head) {
  const int64_t off = p.qstart ? (rq.t0 + i) * p.qt : r * p.qb + i * p.qt;
  return static_cast<const char*>(p.q) + (off + head * p.qh) * (int64_t)sizeof(T);
}
template <typename T>
__device__ __forceinline__ T* out_at(const Args& p, int r, const Request& rq, int i, int head) {
  const int64_t off = p.qstart ? (rq.t0 + i) * p.ot : r * p.ob + i * p.ot;
  return static_cast<T*>(p.out) + off + head * p.oh;
}

// The lane's number, not taken from a register that the caller would keep for it.
__device__ __forceinline__ int lane_anew() {
  return __builtin_amdgcn_mbcnt_hi(~0u, __builtin_amdgcn_mbcnt_lo(~0u, opaque(0)));
}
// Column c's (m, l of its lane half, o of the dims 32 dt ..) over one segment, by
// one wave whose lanes hold the columns of one token: the arithmetic of the
// kernels below with zeros for every row that the token does not see, for
// tokens of a whole workgroup beside others that see a row of values with an
// infinity or NaN. (Slow and rare: it keeps little in registers.) `lds`: 32 rows
// of values.
template <typename T, int D, int V>
__device__ __forceinline__ f32x16 token_segment(const Args& p, int r, const Request& rq, int kvh, int c, int dt,
                                                int segment, uint4* lds, float& m, float& l) {
  using G = Geo<T, D, V>;
  constexpr int S = G::kStep, KT = G::KT, PU = G::PU;
  const int lane = lane_anew(), half = lane >> 5;
  const int token = c / p.G;
  const int32_t pos = rq.n - rq.L + token;
  const char* q = query_at<T>(p, r, rq, token, kvh * (int)p.G.d + c - token * (int)p.G.d);
  auto row_at = [&](const void* base, int64_t page, int64_t head, int64_t row, int32_t key)
      __attribute__((always_inline)) -> const char* {
    const int32_t id = any_seen(p, pos, pos, key, 1) ? page_of(p, r, entry_of(p, r, key), key) : -1;
    const char* at = static_cast<const char*>(base) +
                     (kvh * head + id * page + row_of(p, key) * row) * (int64_t)sizeof(T);
    return id >= 0 ? at : reinterpret_cast<const char*>(g_zero_row);
  };
  m = kNone, l = 0.f;
  f32x16 o = {};
#pragma unroll 1
  for (int32_t key0 = segment * G::kSeg; key0 < (segment + 1) * G::kSeg; key0 += S) {
    if (!any_seen(p, pos, pos, key0, S)) continue;
    f32x16 s[KT];
#pragma unroll
    for (int kt = 0; kt < KT; kt++) {
      const char* k = row_at(p.k, p.kb, p.kh, p.kn, key0 + 32 * kt + (lane & 31));
      s[kt] = f32x16{};
#pragma unroll 1
      for (int t = 0; t < G::NQ; t++) {
        uint4 x = ld16(q + (2 * t + half) * 16);
        x = make_uint4(x.x ^ p.qsign, x.y ^ p.qsign, x.z ^ p.qsign, x.w ^ p.qsign);
        s[kt] = G::score(ld16(k + (2 * t + half) * 16), x, s[kt]);
      }
    }
    const int32_t key = key0 + (lane & (S - 1));
    const uint64_t mapped = __builtin_amdgcn_ballot_w64(page_of(p, r, entry_of(p, r, key), key) >= 0);
    G::hide(s, seen_bits(p, pos, key0, mapped) >> (4 * half));
    const float base = next_base(m, G::top(s), p.scale2), f = pow2(m - base);
    m = base;
    uint4 pu[KT][PU];
#pragma unroll
    for (int kt = 0; kt < KT; kt++) {
      f32x16 e;
#pragma unroll
      for (int i = 0; i < 16; i++) e[i] = __builtin_amdgcn_exp2f(__builtin_fmaf(s[kt][i], p.scale2, -m));
      G::pack(e, pu[kt]);
    }
    l = __builtin_fmaf(l, f, G::sum(pu));
#pragma unroll
    for (int i = 0; i < 16; i++) o[i] *= f;
#pragma unroll
    for (int kt = 0; kt < KT; kt++) {
#pragma unroll 1
      for (int at = lane; at < 32 * G::VCH; at += 64) {
        const int row = at / G::VCH, chunk = at - row * G::VCH;
        const char* v = row_at(p.v, p.vb, p.vh, p.vn, key0 + 32 * kt + row);
        st16(lds + row * G::VCH + (chunk ^ G::vswz(row)), ld16(v + chunk * 16));
      }
      __builtin_amdgcn_wave_barrier();
#pragma unroll
      for (int u = 0; u < PU; u++) o = G::score(G::value(lds, 0, u, dt, lane), pu[kt][u], o);
      __builtin_amdgcn_wave_barrier();
    }
  }
  return o;
}
// Runs use(column, valid) for the columns c0 .. clast of a token, 32 lanes at a
// time; a lane without one has the first one's.
template <typename Use>
__device__ __forceinline__ void for_columns(const Args& p, int token, int c0, int clast, const Use& use) {
  const int lane = lane_anew() & 31;
  const int first = token * (int)p.G.d, end = first + (int)p.G.d <= clast ? first + (int)p.G.d : clast + 1;
  for (int c = first < c0 ? c0 : first; c < end; c += 32) use(c + lane < end ? c + lane : c, c + lane < end);
}
// A token's columns c0 .. clast, output dims 32 dt .., of all segments.
template <typename T, int D, int V>
__device__ __forceinline__ void walk_token(const Args& p, int r, const Request& rq, int kvh, int token, int dt, int c0, int clast,
                           uint4* lds) {
  using G = Geo<T, D, V>;
  const int half = lane_anew() >> 5;
  const int32_t pos = rq.n - rq.L + token;
  const Walk w = walk(p, pos, pos, G::kSeg);
  for_columns(p, token, c0, clast, [&](int c, bool valid) __attribute__((always_inline)) {
    float M = kNone, L = 0.f;
    f32x16 O = {};
#pragma unroll 1
    for (int i = 0; i < w.count(); i++) {
      float m, l, fa, fb;
      const f32x16 o = token_segment<T, D, V>(p, r, rq, kvh, c, dt, w.unit(i), lds, m, l);
      fold_base(M, L, m, half_swap_sum(l), fa, fb);
#pragma unroll
      for (int e = 0; e < 16; e++) O[e] = __builtin_fmaf(o[e], fb, O[e] * fa);
    }
    const int head = kvh * (int)p.G.d + c - token * (int)p.G.d;
    float e, den;
    finish(M, L, p.sinks ? (float)static_cast<const T*>(p.sinks)[head] * 1.4426950408889634f : 0.f,
           p.sinks != nullptr, e, den);
    const float inv = inverse(den);
    T* out = out_at<T>(p, r, rq, token, head);
    if (valid)
#pragma unroll
      for (int i = 0; i < 16; i++) out[32 * dt + G::row(i, half)] = result<T>(O[i], e, inv);
  });
}

// Split route: a segment's (m, l, o) of NC columns, four steps to a pass, one
// per wave. What bounds it is reading the cache, which it does 64 KB at a
// time: a step's values are on their way while its scores are computed, the
// next pass's keys while the values are used, both through the same registers
// (the table's entries are loaded two passes ahead). The same loads without
// any computation read 64 requests of 8191 rows in pages of 16 in 350 us (6.1
// TB/s); this kernel and its fold take 365 to 390, 5 % more with loads that
// keep their lines in the caches. (32 loads a wave in flight, keys and values
// together, were no faster: alone they read 4.7 TB/s, 16 a wave 6.0-6.4.)
// ONE: no request has more than one token, so that no row is seen by some only
// (the code for these costs one request of 8192 rows 1.0 us of 18.7, 64 1.4 %).
template <typename T, int D, int V, int NC, bool ONE>
__global__ void __launch_bounds__(256, (Geo<T, D, V>::split_per_cu(NC))) split_kernel(Args p) {
  using G = Geo<T, D, V>;
  constexpr int S = G::kStep, KT = G::KT, PU = G::PU;
  __shared__ uint4 s_kv[4 * S * G::MCH];  // a step per wave: its keys, then its values
  __shared__ uint4 s_p[4 * KT * PU * 2 * NC];
  __shared__ const char* s_row[2][4 * S];
  __shared__ float s_max[4][NC];
  __shared__ float s_sum[4][2 * NC];
  __shared__ int s_odd[2];

  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int col = lane & 31, half = lane >> 5, cn = col & (NC - 1);
  // Workgroup -> kv head, columns, segment of the walk, request. A segment's
  // column tiles are next to each other, with 8 kv heads on one XCD: they read
  // the same rows; but one after the other where most requests have only the
  // first (beside chunks: 30 of 32 requests, 70 us the other way, 47 so).
  // Request by request; under a window, where every request has the same few
  // segments and the first and the last are cut, segment by segment (16
  // requests that see 1024 rows 24.1 -> 21.4 us; 64 of 1000 to 8191 rows 271
  // -> 279).
  const int x = blockIdx.x, xc = x / p.Hkv, kvh = x - xc * (int)p.Hkv.d;
  const int xq = xc / (p.once ? p.slots : p.ctiles);
  const int xr = xc - xq * (int)(p.once ? p.slots : p.ctiles).d;
  const int xs = p.once ? xr : xq, c0 = (p.once ? xq : xr) * NC;
  const int outer = xs / (p.window ? p.reqs : p.gseg);
  const int inner = xs - outer * (int)(p.window ? p.reqs : p.gseg).d;
  const int r = p.window ? inner : outer, part0 = p.window ? outer : inner;
  // Without a window the walk's entries are the segments themselves, and the
  // table's entries can be on their way before the request is known.
  constexpr int PS = 4 * S, PN = G::kSeg / PS;
  int32_t entry0 = 0, entry = 0;
  if (!p.window) {
    entry0 = entry_of(p, r, part0 * G::kSeg + wave * S + (lane & (S - 1)));
    entry = entry_of(p, r, part0 * G::kSeg + PS + wave * S + (lane & (S - 1)));
  }
  const Request rq = request(p, r);
  const int ncol = rq.L * (int)p.G.d;
  if (rq.beyond || ncol > p.split_cols || c0 >= ncol) return;
  const int clast = (c0 + NC < ncol ? c0 + NC : ncol) - 1;
  int32_t lo = rq.n - rq.L + c0 / p.G, hi = rq.n - rq.L + clast / p.G;
  // The segment's passes (4 steps each) that some column sees.
  const Walk w = walk(p, lo, hi, G::kSeg);
  const int parts = w.count() < (int)p.nseg.d ? w.count() : p.nseg.d;
  if (part0 >= parts) return;
  const bool several = !ONE && lo != hi;  // tokens, which may see different rows
  if (several && threadIdx.x < 2) s_odd[threadIdx.x] = 0;
  int turn = 0, token = -1;  // token: the one whose results are computed once more

  // Column; one without a token takes the first one's query and sees nothing.
  const int cc = c0 + col;
  const bool cv = col < NC && cc < ncol;
  const int cq = cv ? cc : c0;
  const int tok = cq / p.G, head = kvh * (int)p.G.d + (cq - tok * (int)p.G.d);
  const int32_t pos = cv ? rq.n - rq.L + tok : -1;
  const char* kh = static_cast<const char*>(p.k) + kvh * p.kh * (int64_t)sizeof(T);
  const char* vh = static_cast<const char*>(p.v) + kvh * p.vh * (int64_t)sizeof(T);
  // In vector registers: scalar ones are short, and what is left of them decides
  // how the compiler orders the loads and products of a pass (128 tokens over 8192
  // rows 107 us, 117 with these and the arguments of the results' store kept
  // there; 104 without computing tokens once more).
  if (!ONE) asm volatile("" : "+v"(kh), "+v"(vh));

  int part = part0, s0, s1;
  // Row addresses of the wave's step of a segment; a row that no column sees,
  // or that has no page, is a row of zeros. Without branches, so that the
  // loads in flight are counted exactly.
  auto key_of = [&](int si) __attribute__((always_inline)) { return si * PS + wave * S; };
  auto entry_for = [&](int si) __attribute__((always_inline)) -> int32_t {
    return entry_of(p, r, key_of(si) + (lane & (S - 1)));
  };
  auto put_rows = [&](int si, int32_t entry) __attribute__((always_inline)) -> uint64_t {
    const int32_t key = key_of(si) + (lane & (S - 1));
    const int32_t id = si < s1 && any_seen(p, lo, hi, key, 1) ? page_of(p, r, entry, key) : -1;
    const int64_t row = row_of(p, key);
    const char* zero = reinterpret_cast<const char*>(g_zero_row);
    const char* ka = kh + (id * p.kb + row * p.kn) * (int64_t)sizeof(T);
    const char* va = vh + (id * p.vb + row * p.vn) * (int64_t)sizeof(T);
    s_row[0][wave * S + (lane & (S - 1))] = id >= 0 ? ka : zero;
    s_row[1][wave * S + (lane & (S - 1))] = id >= 0 ? va : zero;
    __builtin_amdgcn_wave_barrier();
    return __builtin_amdgcn_ballot_w64(id >= 0);
  };
  // Rows are loaded whole, consecutive lanes taking consecutive chunks. Lane
  // numbers go by way of opaque(): addresses are computed where they are used,
  // not kept across segments in registers that the loads need.
  constexpr int KL = S * G::CH / 64, VL = S * G::VCH / 64;
  uint4 x16[KL > VL ? KL : VL], q[G::NQ];
  auto load_rows = [&](const char* const* rows, auto chunks, auto load) __attribute__((always_inline)) {
    constexpr int C = decltype(chunks)::value;
    const int ln = opaque(lane);
#pragma unroll
    for (int j = 0; j < S * C / 64; j++) {
      const int at = j * 64 + ln, row = at / C;
      x16[j] = load(rows[wave * S + row] + (at - row * C) * 16);
    }
  };
  auto load_keys = [&]() __attribute__((always_inline)) {
    if (p.once) load_rows(s_row[0], std::integral_constant<int, G::CH>(), ld16_once);
    else load_rows(s_row[0], std::integral_constant<int, G::CH>(), ld16);
  };
  auto load_values = [&]() __attribute__((always_inline)) {
    if (p.once) load_rows(s_row[1], std::integral_constant<int, G::VCH>(), ld16_once);
    else load_rows(s_row[1], std::integral_constant<int, G::VCH>(), ld16);
  };

  // The grid has p.gseg places for a request's segments: a few are enough
  // where there are many workgroups, and empty ones are not free (64 requests
  // of 250 rows under a bound of 65536 53 us, 128 with a place for each).
  for (;;) {
    s0 = w.unit(part) * PN, s1 = s0 + PN;
    if (!ONE && token >= 0 && !any_seen(p, lo, hi, s0 * PS, G::kSeg)) s1 = s0;  // one token may see none of it
    while (s0 < s1 && !any_seen(p, lo, hi, s0 * PS, PS)) s0++;
    while (s0 < s1 && !any_seen(p, lo, hi, (s1 - 1) * PS, PS)) s1--;
    if (p.window || part != part0 || token >= 0) {
      entry0 = entry_for(s0);
      entry = entry_for(s0 + 1);
    }
    load_query<G>(query_at<T>(p, r, rq, tok, head), half, q);
    uint64_t mapped = put_rows(s0, entry0);
    load_keys();
    sign_query<G>(p, q);

    constexpr int TW = (G::DT + 3) / 4;  // tiles of output dims per wave
    float m = kNone, l = 0.f;
    f32x16 o[TW];
#pragma unroll
    for (int i = 0; i < TW; i++) o[i] = f32x16{};
    for (int si = s0; si < s1; si++) {
      const int32_t pass0 = si * PS, key0 = pass0 + wave * S;
      const int32_t entry2 = entry_for(si + 2);
      // Scores of the wave's step and their largest. The keys change from rows to
      // the products' operands by way of the LDS where the wave's values go next.
      f32x16 s[KT];
      const int lk = opaque(lane);
#pragma unroll
      for (int j = 0; j < KL; j++) {
        const int at = j * 64 + lk, row = at / G::CH, c = (at - row * G::CH) ^ G::kswz(row);
        st16(s_kv + wave * S * G::MCH + row * G::CH + c, x16[j]);
      }
      load_values();
      __builtin_amdgcn_wave_barrier();
#pragma unroll
      for (int kt = 0; kt < KT; kt++) {
        f32x16 c = {};
#pragma unroll
        for (int t = 0; t < G::NQ; t++)
          c = G::score(G::key_chunk(s_kv + wave * S * G::MCH, kt, lk & 31, t, lk >> 5), q[t], c);
        s[kt] = c;
      }
      const bool full = mapped == ~0ull && all_seen(p, lo, hi, key0, S) && c0 + NC <= ncol;
      if (!full) G::hide(s, seen_bits(p, pos, key0, mapped) >> (4 * half));
      const float top = G::top(s);
      if (lane < NC) s_max[wave][lane] = top;
      barrier();

      // The bases of the pass's steps; this wave's p.
      float base[4], f[4];
#pragma unroll
      for (int i = 0; i < 4; i++) {
        base[i] = next_base(m, s_max[i][cn], p.scale2);
        f[i] = pow2(m - base[i]);
        m = base[i];
      }
      const float mw = wave == 0 ? base[0] : wave == 1 ? base[1] : wave == 2 ? base[2] : base[3];
      uint4 pu[KT][PU];
#pragma unroll
      for (int kt = 0; kt < KT; kt++) {
        f32x16 e;
#pragma unroll
        for (int i = 0; i < 16; i++)
          e[i] = __builtin_amdgcn_exp2f(__builtin_fmaf(s[kt][i], p.scale2, -mw));
        G::pack(e, pu[kt]);
        if (col < NC)
#pragma unroll
          for (int j = 0; j < PU; j++) s_p[((wave * KT + kt) * PU + j) * 2 * NC + half * NC + col] = pu[kt][j];
      }
      const float psum = G::sum(pu);
      if (col < NC) s_sum[wave][half * NC + col] = psum;
      const int ln = opaque(lane);
#pragma unroll
      for (int j = 0; j < VL; j++) {
        const int at = j * 64 + ln, row = at / G::VCH, c = (at - row * G::VCH) ^ G::vswz(row);
        st16(s_kv + wave * S * G::MCH + row * G::VCH + c, x16[j]);
      }
      mapped = put_rows(si + 1, entry);
      entry = entry2;
      load_keys();
      barrier();

      // The sum, and the wave's tiles of output dims over the pass's steps.
#pragma unroll
      for (int i = 0; i < 4; i++) l = __builtin_fmaf(l, f[i], s_sum[i][half * NC + cn]);
#pragma unroll
      for (int x = 0; x < TW; x++) {
        const int dt = wave + 4 * x;
        if (dt >= G::DT) break;
#pragma unroll
        for (int i = 0; i < 4; i++) {
          if (!any_seen(p, lo, hi, pass0 + i * S, S)) continue;
          if (__builtin_amdgcn_ballot_w64(f[i] != 1.f) != 0)
#pragma unroll
            for (int e = 0; e < 16; e++) o[x][e] *= f[i];
#pragma unroll
          for (int kt = 0; kt < KT; kt++) {
            uint4 u[PU];
#pragma unroll
            for (int j = 0; j < PU; j++) u[j] = s_p[((i * KT + kt) * PU + j) * 2 * NC + (ln >> 5) * NC + (ln & (NC - 1))];
#pragma unroll
            for (int j = 0; j < PU; j++)
              o[x] = G::score(G::value(s_kv + i * S * G::MCH, kt * 32, j, dt, ln), u[j], o[x]);
          }
        }
      }
      if (several && token < 0) {
        if (ln == 0) s_odd[~turn & 1] = 0;  // of the last part, of which all know
        if (!all_seen(p, lo, hi, key0, S)) {
          uint32_t odd = 0;
          for (int j = 0; j < VL; j++) odd |= G::odd(s_kv[wave * S * G::MCH + j * 64 + ln]);
          if (__builtin_amdgcn_ballot_w64((odd & G::kOdd) != 0) != 0) s_odd[turn & 1] = 1;
        }
      }
      barrier();  // everyone is done with the values and p
    }

    l = half_swap_sum(l);
    const Args& again = ONE ? p : args_again();
    if (cv && (ONE || token < 0 || (c0 + col) / again.G == token)) {
      const int64_t slot = (((int64_t)r * again.Hkv.d + kvh) * again.nseg.d + part) * again.ccap.d + cc;
      if (wave == 0 && half == 0) again.pml[slot] = make_float2(m, l);
#pragma unroll
      for (int x = 0; x < TW; x++) {
        if (wave + 4 * x >= G::DT) break;
        float* to = again.po + slot * V + 32 * (wave + 4 * x);
#pragma unroll
        for (int b = 0; b < 4; b++)
          *reinterpret_cast<f32x4*>(to + 8 * b + 4 * half) =
              f32x4{o[x][4 * b], o[x][4 * b + 1], o[x][4 * b + 2], o[x][4 * b + 3]};
      }
    }
    if (several) {
      // Some values that not all tokens see are infinities or NaN: the segment once
      // more, token by token; the columns of others are computed as they come and
      // not stored. (Each pass ends with a barrier.)
      if (token >= 0 ? token < clast / again.G
                     : __builtin_expect_with_probability(__builtin_amdgcn_readfirstlane(s_odd[turn & 1]), 1, 0.0)) {
        token = token < 0 ? c0 / again.G : token + 1;
        lo = hi = rq.n - rq.L + token;
        continue;
      }
      if (token >= 0) lo = rq.n - rq.L + c0 / again.G, hi = rq.n - rq.L + clast / again.G, token = -1;
      turn++;
    }
    if ((part += again.gseg.d) >= parts) return;
  }
}

// Tokens that no kernel computes: 0 where no request owns them, NaN where the
// request is beyond a bound. `block` of p.fill_blocks workgroups.
template <typename T, int V>
__device__ void fill(const Args& p, int block) {
  const int64_t row = (int64_t)p.H * V;
  T* out = static_cast<T*>(p.out);
  const int64_t tid = (int64_t)block * blockDim.x + threadIdx.x, all = (int64_t)p.fill_blocks * blockDim.x;
  int32_t a = p.R > 0 ? p.qstart[0] : p.T, b = p.R > 0 ? p.qstart[p.R] : p.T;
  a = a < 0 ? 0 : a > p.T ? p.T : a;
  b = b < a ? a : b > p.T ? p.T : b;
  for (int64_t i = tid; i < a * row; i += all) out[i] = (T)0.f;
  for (int64_t i = b * row + tid; i < p.T * row; i += all) out[i] = (T)0.f;
  for (int r0 = 0; r0 < p.R; r0 += blockDim.x) {
    const int r = r0 + threadIdx.x;
    const bool mine = r < p.R && request(p, r).beyond;
    if (!__syncthreads_or(mine)) continue;
    for (int k = r0; k < p.R && k < r0 + (int)blockDim.x; k++) {
      const Request rq = request(p, k);
      if (!rq.beyond) continue;
      for (int64_t i = rq.t0 * row + tid; i < (rq.t0 + rq.L) * row; i += all) out[i] = (T)NAN;
    }
  }
}

// Split route: folds a column's segments; one wave per column. Beside chunks a
// wave takes every G-th column of a request, most of which have no more (30
// single tokens beside two chunks 4.8 us, 10.0 with a wave per column).
template <typename T, int D, int V, int SEG>
__global__ void __launch_bounds__(256) combine_kernel(Args p) {
  constexpr int NV = (V + 127) / 128;
  if ((int)blockIdx.x < p.fill_blocks) {
    fill<T, V>(p, blockIdx.x);
    return;
  }
  const int lane = threadIdx.x & 63;
  const int x = (blockIdx.x - p.fill_blocks) * 4 + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int xh = x / p.cstep;
  const int r = xh / p.Hkv, kvh = xh - r * (int)p.Hkv.d;
  if (r >= p.R) return;
  const Request rq = request(p, r);
  const int ncol = rq.L * (int)p.G.d;
  if (rq.beyond || ncol > p.split_cols) return;
  auto fold = [&](int cc) __attribute__((always_inline)) {
    // The columns that shared a workgroup, and with them its segments.
    const int c0 = cc & -p.nc, clast = (c0 + p.nc < ncol ? c0 + p.nc : ncol) - 1;
    const Walk w = walk(p, rq.n - rq.L + c0 / p.G, rq.n - rq.L + clast / p.G, SEG);
    const int n = w.count() < (int)p.nseg.d ? w.count() : p.nseg.d;
    const int tok = cc / p.G, head = kvh * (int)p.G.d + cc - tok * (int)p.G.d;
    const int64_t slot = (int64_t)xh * p.nseg.d * p.ccap.d + cc;  // segments ccap apart
    // Dims 2 lane, 2 lane + 1 and those 128 further; 16 segments' loads in flight.
    constexpr int NB = 16;
    float M = kNone, L = 0.f;
    f32x2 O[NV] = {};
    for (int i0 = 0; i0 < n; i0 += NB) {
      f32x2 o[NB][NV];
      float2 ml[NB];
#pragma unroll
      for (int i = 0; i < NB; i++) {
        const bool in = i0 + i < n;
        const int64_t at = slot + (int64_t)(i0 + i) * p.ccap.d;
        ml[i] = in ? p.pml[at] : make_float2(kNone, 0.f);
#pragma unroll
        for (int j = 0; j < NV; j++)
          o[i][j] = in && 2 * lane + 128 * j < V
                        ? *reinterpret_cast<const f32x2*>(p.po + at * V + 2 * lane + 128 * j)
                        : f32x2{0.f, 0.f};
      }
#pragma unroll
      for (int i = 0; i < NB; i++) {
        float fa, fb;
        fold_base(M, L, ml[i].x, ml[i].y, fa, fb);
#pragma unroll
        for (int j = 0; j < NV; j++)
#pragma unroll
          for (int k = 0; k < 2; k++) O[j][k] = __builtin_fmaf(o[i][j][k], fb, O[j][k] * fa);
      }
    }
    float e, den;
    finish(M, L, p.sinks ? (float)static_cast<const T*>(p.sinks)[head] * 1.4426950408889634f : 0.f,
           p.sinks != nullptr, e, den);
    const float inv = inverse(den);
    T* out = out_at<T>(p, r, rq, tok, head);
#pragma unroll
    for (int j = 0; j < NV; j++)
      if (2 * lane + 128 * j < V) {
        typedef T T2 __attribute__((ext_vector_type(2)));
        *reinterpret_cast<T2*>(out + 2 * lane + 128 * j) =
            T2{result<T>(O[j][0], e, inv), result<T>(O[j][1], e, inv)};
      }
  };
  // (The first one apart: as the loop's body alone it took 1 us more.)
  int cc = x - xh * (int)p.cstep.d;
  if (cc >= ncol) return;
  fold(cc);
  while ((cc += p.cstep.d) < ncol) fold(cc);
}

// Whole route: NW waves of 32 columns each walk the steps that some column of
// the workgroup sees. Keys and values go through a ring of NB LDS buffers, NB -
// 1 steps ahead of their use, by loads that LW waves more do nothing but issue
// (LW = 0: the NW waves themselves). A wave spends about 150 cycles on issuing
// a load that writes LDS, 8 a step: with another wave on its SIMD that is
// hidden, alone it is a quarter of the step (512 tokens over 8192 keys 244 us,
// 173 with loading waves; 1024 over 5120 167 and 125). (Four more computing
// waves on every second segment of the same columns, whose results go through
// LDS, took 185: matrix products and exponentials do not overlap on a SIMD, and
// one wave already fills it.)
template <typename T, int D, int V, int NW, int LW, int NB>
__global__ void __launch_bounds__(64 * (NW + LW), (Geo<T, D, V>::kTwoWaves ? 2 : 1))
    whole_kernel(Args p) {
  using G = Geo<T, D, V>;
  constexpr int S = G::kStep, KT = G::KT, PU = G::PU, DT = G::DT, COLS = 32 * NW;
  constexpr int KU = S * G::CH, VU = S * G::VCH, AHEAD = NB - 1;
  constexpr int NT = 64 * (LW ? LW : NW);  // threads that load
  // Loads per wave and step: its share of the keys and of the values.
  constexpr int LPS = (KU + NT - 1) / NT + (VU + NT - 1) / NT;
  __shared__ uint4 s_kv[NB * (KU + VU)];
  __shared__ uint4 s_dump[KU % NT || VU % NT ? 64 : 1];  // of waves that have no share
  __shared__ const char* s_row[NB][2][S];
  __shared__ int32_t s_entry[8][64];
  __shared__ uint64_t s_map[8];
  __shared__ int s_odd;
  __shared__ int s_scan[NW + LW + 3];
  __shared__ float s_ml[2][64 * NW];  // each lane's own M and L

  if ((int)blockIdx.x < p.fill_blocks) {
    fill<T, V>(p, blockIdx.x);
    return;
  }
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int col = lane & 31, half = lane >> 5;

  // Workgroup -> kv head (neighbours in the grid land on different XCDs, so
  // with 8 kv heads each XCD's L2 holds one of them), request, column tile;
  // a request's last tiles, which see the most rows, start first.
  const int x = blockIdx.x - p.fill_blocks;
  int tile = x / p.Hkv, r = 0;
  const int kvh = x - tile * (int)p.Hkv.d;
  if (!p.qstart) {
    const int per = (p.qL * (int)p.G.d + COLS - 1) / COLS;
    r = tile / per;
    tile = per - 1 - (tile - r * per);
  } else {
    int before = 0, found = -1;
    for (int r0 = 0; r0 < p.R; r0 += 64 * (NW + LW)) {
      int n = 0;
      if (r0 + tid < p.R) {
        const Request rq = request(p, r0 + tid);
        const int ncol = rq.L * (int)p.G.d;
        n = rq.beyond || ncol <= p.split_cols ? 0 : (ncol + COLS - 1) / COLS;
      }
      int sum = n;
#pragma unroll
      for (int d = 1; d < 64; d <<= 1) {
        const int y = __shfl_up(sum, d);
        if (lane >= d) sum += y;
      }
      if (lane == 63) s_scan[wave] = sum;
      if (tid == 0) s_scan[NW + LW] = -1;
      __syncthreads();
      int all = 0;
#pragma unroll
      for (int i = 0; i < NW + LW; i++) {
        if (i < wave) sum += s_scan[i];
        all += s_scan[i];
      }
      if (tile >= before + sum - n && tile < before + sum) {
        s_scan[NW + LW] = r0 + tid;
        s_scan[NW + LW + 1] = n - 1 - (tile - (before + sum - n));
      }
      __syncthreads();
      found = s_scan[NW + LW];
      if (found >= 0) break;
      before += all;
      __syncthreads();
    }
    if (found < 0) return;
    r = found;
    tile = s_scan[NW + LW + 1];
  }
  r = __builtin_amdgcn_readfirstlane(r);
  tile = __builtin_amdgcn_readfirstlane(tile);
  const Request rq = request(p, r);
  const int ncol = rq.L * (int)p.G.d;
  const int c0 = tile * COLS, cw = c0 + 32 * wave;
  const int clast = (c0 + COLS < ncol ? c0 + COLS : ncol) - 1;
  const int32_t p0 = rq.n - rq.L;
  const int32_t lo = p0 + c0 / p.G, hi = p0 + clast / p.G;
  // The wave's own columns; a wave without one only loads.
  const int wlast = cw + 31 < ncol ? cw + 31 : ncol - 1;
  const int32_t wlo = cw < ncol ? p0 + cw / p.G : INT32_MAX / 2, whi = cw < ncol ? p0 + wlast / p.G : -1;

  const bool loads = LW == 0 || wave >= NW;
  const int lw = LW ? wave - NW : wave;  // which of the loading waves

  const int cc = cw + col;
  const bool cv = cc < ncol;
  const int tok = cv ? cc / p.G : 0;
  const bool whole_tile = cw + 32 <= ncol;
  uint4 q[G::NQ];
  load_query<G>(query_at<T>(p, r, rq, tok, kvh * (int)p.G.d + (cv ? cc - tok * (int)p.G.d : 0)), half, q);
  sign_query<G>(p, q);

  const Walk w = walk(p, lo, hi, S);
  const int steps = w.count();
  const char* kh = static_cast<const char*>(p.k) + kvh * p.kh * (int64_t)sizeof(T);
  const char* vh = static_cast<const char*>(p.v) + kvh * p.vh * (int64_t)sizeof(T);

  // A step's way into LDS: the table's entries of its rows, NB + AHEAD steps
  // before, and from them the rows' addresses, NB steps before, both by the
  // first loading wave; then keys and values, AHEAD steps before. A wave issues
  // the same number of loads every step, so that it can wait by their count.
  auto load_entries = [&](int j) __attribute__((always_inline)) {
    const int32_t* at = reinterpret_cast<const int32_t*>(g_zero_row);
    if (p.qstart && p.W > 0) {
      const int32_t c = table_column(p, w.unit(j) * S + (opaque(lane) & (S - 1)));
      at = p.table + r * p.table_stride + (c < p.W ? c : p.W - 1);
    }
    load_to_lds<4>(at, s_entry[j & 7]);
  };
  auto put_rows = [&](int j, int32_t entry) __attribute__((always_inline)) {
    if (j >= steps) return;
    const int ln = opaque(lane) & (S - 1);
    const int32_t key = w.unit(j) * S + ln;
    const int32_t id = any_seen(p, lo, hi, key, 1) ? page_of(p, r, entry, key) : -1;
    const int64_t row = row_of(p, key);
    const char* zero = reinterpret_cast<const char*>(g_zero_row);
    s_row[j % NB][0][ln] = id >= 0 ? kh + (id * p.kb + row * p.kn) * (int64_t)sizeof(T) : zero;
    s_row[j % NB][1][ln] = id >= 0 ? vh + (id * p.vb + row * p.vn) * (int64_t)sizeof(T) : zero;
    s_map[j & 7] = __builtin_amdgcn_ballot_w64(id >= 0);  // S = 32: both halves alike
  };
  auto load_rows = [&](const char* const* rows, auto ch, auto swizzle, uint4* to)
      __attribute__((always_inline)) {
    constexpr int C = decltype(ch)::value, U = S * C;
    const int td = opaque(64 * lw + lane);
    // Chunk i NT + td of the step; all addresses before the first load.
    constexpr int N = (U + NT - 1) / NT;
    const char* from[N];
#pragma unroll
    for (int i = 0; i < N; i++) {
      const int row = NT % C == 0 ? i * (NT / C) + td / C : (i * NT + td) / C;
      const int c = NT % C == 0 ? td % C : (i * NT + td) % C;
      from[i] = rows[U % NT == 0 || i * NT + td < U ? row : 0] + (c ^ swizzle(row)) * 16;
    }
#pragma unroll
    for (int i = 0; i < N; i++)
      load_to_lds<16>(from[i], U % NT == 0 || i * NT + lw * 64 < U ? to + i * NT + lw * 64 : s_dump);
  };
  auto load_step = [&](int j) __attribute__((always_inline)) {
    uint4* to = s_kv + j % NB * (KU + VU);
    load_rows(s_row[j % NB][0], std::integral_constant<int, G::CH>(), G::kswz, to);
    load_rows(s_row[j % NB][1], std::integral_constant<int, G::VCH>(), G::vswz, to + KU);
  };

  // The segment's o and the result's O are in registers, the result's base and
  // sum, which are touched once a segment, in LDS. (O in scratch memory cost
  // 490 us of 1060 over 8192 keys: what the waves keep there exceeds the L2.)
  float m = kNone, l = 0.f;
  bool fresh = true;  // the segment has no step yet
  f32x16 O[DT], o[DT];
#pragma unroll
  for (int dt = 0; dt < DT; dt++) O[dt] = f32x16{}, o[dt] = f32x16{};
  if (wave < NW) {
    s_ml[0][tid] = kNone;
    s_ml[1][tid] = 0.f;
  }

  // Loads of step j, and for the first wave the entries of the step whose
  // addresses are written when step j is waited for.
  auto start_step = [&](int j) __attribute__((always_inline)) {
    if (j >= steps) return;
    if (lw == 0) load_entries(j + NB);
    load_step(j);
  };
  // This wave's part of step j: all but the loads of the AHEAD - 1 later ones.
  auto await_step = [&](int j) __attribute__((always_inline)) {
    if (j + AHEAD > steps) wait_loads();
    else if (lw == 0) wait_loads_but<(AHEAD - 1) * (LPS + 1)>();
    else wait_loads_but<(AHEAD - 1) * LPS>();
  };
  // Steps all_b .. all_e - 1 are seen whole by every token. (As are some with
  // first tokens: a look at those costs little.) `next_look`: the next other one.
  int all_b = 0, all_e = steps;
  if (lo != hi) {
    const int32_t start = p.window ? hi - p.window + 1 : 0, past = lo < 0 ? 0 : (lo + 1) / S;
    const int skip = (start > 0 ? (start + S - 1) / S : 0) - w.b;
    all_b = w.a + (skip > 0 ? skip : 0);
    all_e = w.a + past - w.b;
    if (all_e < all_b) all_e = all_b;
  }
  int next_look = all_b > 0 ? 0 : all_e;
  // Before the barrier of step j: whether this wave's part of its values, which
  // some tokens may not see, holds an infinity or NaN.
  auto look_at_values = [&](int j) __attribute__((always_inline)) {
    if (j != next_look) return;
    next_look = j + 1 == all_b ? all_e : j + 1;
    const uint4* at = s_kv + j % NB * (KU + VU) + KU + 64 * lw + opaque(lane);
    uint32_t odd = 0;
#pragma unroll
    for (int i = 0; i < (VU + NT - 1) / NT; i++)
      if (VU % NT == 0 || i * NT + 64 * lw < VU) odd |= G::odd(at[i * NT]);
    if (__builtin_amdgcn_ballot_w64((odd & G::kOdd) != 0) != 0) s_odd = 1;
  };
  if (tid == 0) s_odd = 0;
  if (loads && lw == 0) {
    int32_t entry[NB];
#pragma unroll
    for (int i = 0; i < NB; i++) entry[i] = entry_of(p, r, w.unit(i) * S + (lane & (S - 1)));
#pragma unroll
    for (int i = 0; i < NB; i++) put_rows(i, entry[i]);
  }
  __syncthreads();
  if (loads)
#pragma unroll
    for (int i = 0; i < AHEAD; i++) start_step(i);
  if constexpr (LW != 0)
    if (loads) {
      for (int j = 0; j < steps; j++) {
        await_step(j);
        look_at_values(j);
        barrier();
        start_step(j + AHEAD);
        if (lw == 0) put_rows(j + NB, s_entry[(j + NB) & 7][opaque(lane)]);
      }
      return;
    }
  for (int j = 0; j < steps; j++) {
    // LDS addresses are computed anew each step: kept across steps they take
    // the registers that o and O need.
    const int ln = opaque(lane), hf = ln >> 5;
    if constexpr (LW == 0) {
      await_step(j);
      look_at_values(j);
    }
    barrier();  // step j is there, and everyone is done with step j - 1's buffer
    if constexpr (LW == 0) start_step(j + AHEAD);
    const uint4 *kd = s_kv + j % NB * (KU + VU), *vd = kd + KU;
    const int32_t unit = w.unit(j), key0 = unit * S;
    if (any_seen(p, wlo, whi, key0, S)) {
      const uint64_t mapped = uniform(s_map[j & 7]);
      const bool full = whole_tile && mapped == ~0ull && all_seen(p, wlo, whi, key0, S);
      f32x16 s[KT];
#pragma unroll
      for (int kt = 0; kt < KT; kt++) s[kt] = f32x16{};
      feed<KT * G::NQ>(
          [&](int n) __attribute__((always_inline)) {
            return G::key_chunk(kd, n % KT, ln & 31, n / KT, hf);
          },
          [&](int n, uint4 k) __attribute__((always_inline)) {
            s[n % KT] = G::score(k, q[n / KT], s[n % KT]);
          });
      if (!full) {
        // (The column's position anew: it would take a register.)
        const int c = cw + (opaque(lane) & 31);
        G::hide(s, seen_bits(p, c < ncol ? p0 + c / p.G : -1, key0, mapped) >> (4 * hf));
      }
      // A lane's sum of at most kMostSum holds no score that moves the base;
      // else, and at a segment's first step, the largest score decides.
      uint4 pu[KT][PU];
      float psum;
      bool look = fresh;
      for (;;) {
        if (look) {
          const float mn = next_base(m, G::top(s), p.scale2);
          if (!fresh && __builtin_amdgcn_ballot_w64(mn != m) != 0) {
            const float f = pow2(m - mn);
            l *= f;  // exact, as in the sum's fma(l, f, .)
#pragma unroll
            for (int dt = 0; dt < DT; dt++)
#pragma unroll
              for (int i = 0; i < 16; i++) o[dt][i] *= f;
          }
          m = mn;
        }
#pragma unroll
        for (int kt = 0; kt < KT; kt++) {
          f32x16 e;
#pragma unroll
          for (int i = 0; i < 16; i++)
            e[i] = __builtin_amdgcn_exp2f(__builtin_fmaf(s[kt][i], p.scale2, -m));
          G::pack(e, pu[kt]);
        }
        psum = G::sum(pu);
        if (look || __builtin_amdgcn_ballot_w64(psum > kMostSum) == 0) break;
        look = true;
      }
      l += psum;
      fresh = false;
      // Products of one output tile are a chain: those of the others go between.
      feed<DT * KT * PU>(
          [&](int n) __attribute__((always_inline)) {
            return G::value(vd, n / DT / PU * 32, n / DT % PU, n % DT, ln);
          },
          [&](int n, uint4 v) __attribute__((always_inline)) {
            o[n % DT] = G::score(v, pu[n / DT / PU][n / DT % PU], o[n % DT]);
          });
    }
    // The segment's end: fold it.
    if (j + 1 == steps || w.unit(j + 1) / G::kSegSteps != unit / G::kSegSteps) {
      if (!fresh) {
        const int td = opaque(tid);
        float M = s_ml[0][td], L = s_ml[1][td], fa, fb;
        fold_base(M, L, m, half_swap_sum(l), fa, fb);
        s_ml[0][td] = M;
        s_ml[1][td] = L;
        if (__builtin_amdgcn_ballot_w64(fa != 1.f) != 0)
#pragma unroll
          for (int dt = 0; dt < DT; dt++)
#pragma unroll
            for (int i = 0; i < 16; i++) O[dt][i] *= fa;
#pragma unroll
        for (int dt = 0; dt < DT; dt++) {
#pragma unroll
          for (int i = 0; i < 16; i++) O[dt][i] = __builtin_fmaf(o[dt][i], fb, O[dt][i]);
          o[dt] = f32x16{};
        }
        m = kNone;
        l = 0.f;
        fresh = true;
      }
    }
    if constexpr (LW == 0)
      if (lw == 0) put_rows(j + NB, s_entry[(j + NB) & 7][opaque(lane)]);
  }

  // The column anew (kept, it would take registers that the loop needs).
  const int lane2 = opaque(lane), cc2 = cw + (lane2 & 31), half2 = lane2 >> 5;
  if (cc2 < ncol) {
    const int tok2 = cc2 / p.G, head = kvh * (int)p.G.d + cc2 - tok2 * (int)p.G.d;
    const float M = s_ml[0][wave * 64 + lane2], L = s_ml[1][wave * 64 + lane2];
    float e, den;
    finish(M, L, p.sinks ? (float)static_cast<const T*>(p.sinks)[head] * 1.4426950408889634f : 0.f,
           p.sinks != nullptr, e, den);
    const float inv = inverse(den);
    T* out = out_at<T>(p, r, rq, tok2, head);
#pragma unroll
    for (int dt = 0; dt < DT; dt++) {
#pragma unroll
      for (int b = 0; b < 4; b++) {
        typedef T T4 __attribute__((ext_vector_type(4)));
        T4 y;
#pragma unroll
        for (int i = 0; i < 4; i++) y[i] = result<T>(O[dt][4 * b + i], e, inv);
        *reinterpret_cast<T4*>(out + 32 * dt + 8 * b + 4 * half2) = y;
      }
    }
  }
  // (Set before the last step's barrier, if at all.)
  // (With no probability: else what follows costs the loop above its registers,
  // 1 % of its time.)
  if (__builtin_expect_with_probability(!__builtin_amdgcn_readfirstlane(s_odd), 1, 1.0)) return;
  __syncthreads();
  // Waves that have room for 32 rows of values each. (All from the arguments
  // again: what is kept for this takes registers from the loop.)
  constexpr int FIT = NB * (KU + VU) / (32 * G::VCH), RW = FIT < NW ? FIT : NW;
  const Args& again = args_again();
  const Request rq2 = request(again, r);
  const int from = tile * COLS, all = rq2.L * (int)again.G.d, to = (from + COLS < all ? from + COLS : all) - 1;
  const int t0 = from / again.G, tasks = (to / again.G - t0 + 1) * DT;
  if (wave < RW)
#pragma unroll 1
    for (int i = wave; i < tasks; i += RW)
      walk_token<T, D, V>(again, r, rq2, kvh, t0 + i / DT, i % DT, from, to, s_kv + wave * 32 * G::VCH);
}

template <typename T, int D, int V>
Kernels kernels_of() {
  Kernels k;
  k.split16 = split_kernel<T, D, V, 16, false>;
  k.split32 = split_kernel<T, D, V, 32, false>;
  k.split16_one = split_kernel<T, D, V, 16, true>;
  k.split32_one = split_kernel<T, D, V, 32, true>;
  using G = Geo<T, D, V>;
  k.combine = combine_kernel<T, D, V, G::kSeg>;
  k.seg = G::kSeg, k.pass = 4 * G::kStep;
  k.row_us = G::row_us();
  k.seg16_us = G::seg_us(16), k.seg32_us = G::seg_us(32);
  k.per_cu16 = G::split_per_cu(16), k.per_cu32 = G::split_per_cu(32);
  if constexpr (G::kTwoWaves) {
    k.whole4 = whole_kernel<T, D, V, 4, 4, G::kDeep>;
    k.whole4_pair = whole_kernel<T, D, V, 4, 0, 2>;
    k.whole8 = whole_kernel<T, D, V, 8, 0, 2>;
  } else {
    k.whole4 = whole_kernel<T, D, V, 4, 0, 2>;
    k.whole4_pair = k.whole8 = nullptr;
  }
  k.whole4_threads = G::kTwoWaves ? 512 : 256;
  return k;
}

}  // namespace
}  // namespace bi_paged

#define BI_PAGED_KERNELS(D, V)                                      \
  bi_paged::Kernels bi_paged::kernels_d##D##_v##V(int dtype) {      \
    return dtype == BI_F32 ? kernels_of<float, D, V>()              \
           : dtype == BI_F16 ? kernels_of<_Float16, D, V>()         \
                             : kernels_of<__bf16, D, V>();          \
  }
