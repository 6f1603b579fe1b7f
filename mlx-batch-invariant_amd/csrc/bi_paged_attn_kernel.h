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
//     where a row of keys and of values is at most 256 bytes, else 32), four
//     steps to a segment.
//   * raw_j is a chain of 32x32 matrix products over the head dim from +0.0:
//     of 16 dims for 16-bit types, of 2 for fp32; 16-byte chunks 2t and 2t + 1
//     of the rows enter product t (fp32: products 4t .. 4t + 3).
//   * Within a segment the running base m moves at a step whose largest seen
//     score M exceeds m + 8, to the multiple of 8 nearest M. p_j =
//     2^(fma(raw_j, a, -m)), 0 for an unseen row; l = l * f + (the step's sum,
//     in a fixed tree per lane half); o = o * f, then o += v . p by 32x32
//     products over the step's rows in ascending order, p rounded once to the
//     type (the products of bf16 and f16 take such operands; l sums the
//     unrounded p). f is a power of two, as every base is an integer.
//   * Segments start from nothing and are folded in ascending order: with M'
//     the larger base, O = fma(o, 2^(m - M'), O * 2^(M - M')), L alike.
//   * The sink enters last: out = (O * e) / (L * e + 2^(sink2 - X)) + 0.0, X the
//     larger of M and sink2, e = 2^(M - X), the division by a product with the
//     rounded inverse; rounded once to the type.
// A step or segment that a column sees nothing of leaves it as it is, so which
// of them a workgroup walks for its other columns changes no bits (a zero's
// sign would: hence the + 0.0).
//
// Two routes, the same bits:
//   * split: a workgroup per (request, kv head, up to 32 columns, segment); its
//     four waves take a step each, so a segment's keys and values are all in
//     flight at once, and a second kernel folds the segments. For few columns,
//     where what bounds it is reading the cache.
//   * whole: a workgroup per 128 columns walks all their steps, 32 columns per
//     wave, keys and values through two LDS buffers. For chunks of a prompt,
//     where the matrix products and the exponentials bound it.
#pragma once

#include <float.h>
#include <math.h>

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
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
typedef __attribute__((address_space(3))) void lds_void;
typedef __attribute__((address_space(3))) i16x4 lds_i16x4;
typedef __attribute__((address_space(1))) const void global_void;

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

// A row's page, or -1; contiguous keys: the request.
__device__ __forceinline__ int32_t page_of(const Args& p, int r, int32_t key) {
  if (!p.qstart) return r;
  const int32_t pg = p.page_shift >= 0 ? key >> p.page_shift : (int32_t)((uint32_t)key / (uint32_t)p.page);
  if (pg >= p.W) return -1;
  const int32_t id = p.table[r * p.table_stride + pg];
  return id < p.pages ? id : -1;
}
__device__ __forceinline__ int32_t row_of(const Args& p, int32_t key) {
  if (!p.qstart) return key;
  return p.page_shift >= 0 ? key & (p.page - 1) : (int32_t)((uint32_t)key % (uint32_t)p.page);
}

__device__ __forceinline__ int opaque(int x) {
  asm volatile("" : "+v"(x));
  return x;
}
__device__ __forceinline__ uint64_t uniform(uint64_t x) {
  return ((uint64_t)(uint32_t)__builtin_amdgcn_readfirstlane((uint32_t)(x >> 32)) << 32) |
         (uint32_t)__builtin_amdgcn_readfirstlane((uint32_t)x);
}
// Loads that write LDS are not covered by a barrier's own waits.
__device__ __forceinline__ void wait_loads() { asm volatile("s_waitcnt vmcnt(0)" ::: "memory"); }

__device__ __forceinline__ float half_swap_max(float x) {
  const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  return fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1]));
}
__device__ __forceinline__ float half_swap_sum(float x) {
  const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  return __uint_as_float(r[0]) + __uint_as_float(r[1]);
}
// 2^e for an integer e that is at most 0 (0 far below).
__device__ __forceinline__ float pow2(float e) {
  return __builtin_amdgcn_ldexpf(1.f, (int)fmaxf(e, -300.f));
}
// The base after a step whose largest seen raw score is `top` (-inf: none seen).
__device__ __forceinline__ float next_base(float m, float top, float a) {
  const float s = top * a;
  return top > -INFINITY && s > m + 8.f ? rintf(s * 0.125f) * 8.f : m;
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
  static constexpr int kSeg = 4 * kStep;
  static constexpr int KT = kStep / 32;       // score tiles per step
  static constexpr int CH = D * E / 16;       // 16-byte chunks per key row
  static constexpr int VCH = V * E / 16;      // per value row
  static constexpr int NQ = CH / 2;           // chunks per lane half
  static constexpr int PU = E;                // 16-byte units of p per tile and lane
  static constexpr int DT = V / 32;           // tiles of output dims

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
  __device__ __forceinline__ static float sum(const f32x16& p) {
    float s[8];
#pragma unroll
    for (int i = 0; i < 8; i++) s[i] = p[2 * i] + p[2 * i + 1];
    return ((s[0] + s[1]) + (s[2] + s[3])) + ((s[4] + s[5]) + (s[6] + s[7]));
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

  // o += values of rows `row0` + 0 .. 31 (LDS `v`) times p, output dims 32 dt ...
  __device__ __forceinline__ static void accumulate(const uint4* v, int row0, int dt, int lane,
                                                    const uint4 (&pu)[PU], f32x16& o) {
    const int half = lane >> 5;
    if constexpr (E == 2) {
      const int g = lane >> 4, i = lane & 15;
      const int rr = i >> 2, piece = i & 3;
      const int c = dt * 4 + (g & 1) * 2 + (piece >> 1);
#pragma unroll
      for (int u = 0; u < 2; u++) {
        i16x4 a[2];
#pragma unroll
        for (int x = 0; x < 2; x++) {
          const int r = row0 + 16 * u + 8 * x + 4 * half + rr;
          const char* at = reinterpret_cast<const char*>(v + r * VCH + (c ^ vswz(r))) + 8 * (piece & 1);
          a[x] = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_i16x4*)at);
        }
        const uint2 lo = __builtin_bit_cast(uint2, a[0]), hi = __builtin_bit_cast(uint2, a[1]);
        o = score(make_uint4(lo.x, lo.y, hi.x, hi.y), pu[u], o);
      }
    } else {
#pragma unroll
      for (int u = 0; u < 4; u++) {
        float a[4];
#pragma unroll
        for (int e = 0; e < 4; e++)
          a[e] = reinterpret_cast<const float*>(v + (row0 + 8 * u + 4 * half + e) * VCH)[32 * dt + (lane & 31)];
        o = score(make_uint4(__float_as_uint(a[0]), __float_as_uint(a[1]), __float_as_uint(a[2]),
                             __float_as_uint(a[3])), pu[u], o);
      }
    }
  }
};

__device__ __forceinline__ uint4 ld16(const void* p) {
  return __builtin_bit_cast(uint4, *reinterpret_cast<const u32x4*>(p));
}

// A column's query as products' operand: chunks 2t + half.
template <typename G>
__device__ __forceinline__ void load_query(const Args& p, const char* q, bool valid, int half,
                                           uint4 (&out)[G::NQ]) {
#pragma unroll
  for (int t = 0; t < G::NQ; t++) {
    uint4 x = valid ? ld16(q + (2 * t + half) * 16) : make_uint4(0, 0, 0, 0);
    out[t] = make_uint4(x.x ^ p.qsign, x.y ^ p.qsign, x.z ^ p.qsign, x.w ^ p.qsign);
  }
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

// Split route: partial result of NC columns over one segment; wave w takes
// step w of the segment.
template <typename T, int D, int V, int NC>
__global__ void __launch_bounds__(256) split_kernel(Args p) {
  using G = Geo<T, D, V>;
  constexpr int S = G::kStep, KT = G::KT, PU = G::PU;
  __shared__ uint4 s_v[G::kSeg * G::VCH];
  __shared__ uint4 s_p[4 * KT * PU * 2 * NC];
  __shared__ const char* s_row[2][G::kSeg];
  __shared__ float s_max[4][NC];
  __shared__ float s_sum[4][2 * NC];

  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int col = lane & 31, half = lane >> 5;
  int x = blockIdx.x;
  const int kvh = x % p.Hkv;
  x /= p.Hkv;
  const int si = x % p.nseg;
  const int r = x / p.nseg;
  const Request rq = request(p, r);
  const int ncol = rq.L * p.G;
  const int c0 = blockIdx.y * NC;
  if (rq.beyond || ncol > p.split_cols || c0 >= ncol) return;
  const int clast = (c0 + NC < ncol ? c0 + NC : ncol) - 1;
  const int32_t lo = rq.n - rq.L + c0 / p.G, hi = rq.n - rq.L + clast / p.G;
  const Walk w = walk(p, lo, hi, G::kSeg);
  if (si >= w.count()) return;  // at most p.nseg of them
  const int32_t seg0 = w.unit(si) * G::kSeg;
  const int32_t key0 = seg0 + wave * S;
  const bool live = any_seen(p, lo, hi, key0, S);

  // Column.
  const int cc = c0 + col;
  const bool cv = col < NC && cc < ncol;
  const int tok = cv ? cc / p.G : 0, head = kvh * p.G + (cv ? cc - tok * p.G : 0);
  const int32_t pos = cv ? rq.n - rq.L + tok : -1;

  uint64_t mapped = 0;
  uint4 kr[KT][G::NQ], q[G::NQ];
  if (live) {
    const int32_t key = key0 + lane;
    const char *ka = reinterpret_cast<const char*>(g_zero_row), *va = ka;
    bool ok = lane < S && any_seen(p, lo, hi, key, 1);
    const int32_t id = ok ? page_of(p, r, key) : -1;
    ok = id >= 0;
    if (ok) {
      const int64_t row = row_of(p, key);
      ka = static_cast<const char*>(p.k) + (id * p.kb + kvh * p.kh + row * p.kn) * (int64_t)sizeof(T);
      va = static_cast<const char*>(p.v) + (id * p.vb + kvh * p.vh + row * p.vn) * (int64_t)sizeof(T);
    }
    mapped = __builtin_amdgcn_ballot_w64(ok);
    if (lane < S) {
      s_row[0][wave * S + lane] = ka;
      s_row[1][wave * S + lane] = va;
    }
    load_query<G>(p, query_at<T>(p, r, rq, tok, head), cv, half, q);
    __builtin_amdgcn_wave_barrier();
#pragma unroll
    for (int kt = 0; kt < KT; kt++) {
      const char* ra = s_row[0][wave * S + kt * 32 + col];
#pragma unroll
      for (int t = 0; t < G::NQ; t++) kr[kt][t] = ld16(ra + (2 * t + half) * 16);
    }
#pragma unroll
    for (int j = 0; j < S * G::VCH / 64; j++) {
      const int at = j * 64 + lane, row = at / G::VCH, c = (at - row * G::VCH) ^ G::vswz(row);
      const char* ra = s_row[1][wave * S + row];
      __builtin_amdgcn_global_load_lds((global_void*)(ra + c * 16),
                                       (lds_void*)(s_v + wave * S * G::VCH + j * 64), 16, 0, 0);
    }
  }

  // Scores of the wave's step and their largest.
  f32x16 s[KT];
  float top = -INFINITY;
  if (live) {
    const bool full = mapped == (S == 64 ? ~0ull : 0xFFFFFFFFull) && all_seen(p, lo, hi, key0, S) && c0 + NC <= ncol;
#pragma unroll
    for (int kt = 0; kt < KT; kt++) {
      f32x16 c = {};
#pragma unroll
      for (int t = 0; t < G::NQ; t++) c = G::score(kr[kt][t], q[t], c);
      s[kt] = c;
    }
    if (!full) G::hide(s, seen_bits(p, pos, key0, mapped) >> (4 * half));
#pragma unroll
    for (int kt = 0; kt < KT; kt++)
#pragma unroll
      for (int i = 0; i < 16; i++) top = fmaxf(top, s[kt][i]);
    top = half_swap_max(top);
  }
  if (lane < NC) s_max[wave][lane] = top;
  __syncthreads();

  // The bases of the segment's steps; this wave's p.
  const int cn = col & (NC - 1);
  float base[4], m = kNone;
#pragma unroll
  for (int i = 0; i < 4; i++) base[i] = m = next_base(m, s_max[i][cn], p.scale2);
  float psum = 0.f;
  if (live) {
    const float mw = wave == 0 ? base[0] : wave == 1 ? base[1] : wave == 2 ? base[2] : base[3];
#pragma unroll
    for (int kt = 0; kt < KT; kt++) {
      f32x16 e;
#pragma unroll
      for (int i = 0; i < 16; i++)
        e[i] = s[kt][i] == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(__builtin_fmaf(s[kt][i], p.scale2, -mw));
      psum = kt == 0 ? G::sum(e) : psum + G::sum(e);
      uint4 u[PU];
      G::pack(e, u);
      if (col < NC)
#pragma unroll
        for (int j = 0; j < PU; j++) s_p[((wave * KT + kt) * PU + j) * 2 * NC + half * NC + col] = u[j];
    }
  }
  if (col < NC) s_sum[wave][half * NC + col] = psum;
  wait_loads();
  __syncthreads();

  // The wave's tiles of output dims over the segment's steps.
  const int64_t slot = (((int64_t)r * p.Hkv + kvh) * p.ccap + cc) * p.nseg + si;
  if (wave == 0) {
    float l = 0.f;
    m = kNone;
#pragma unroll
    for (int i = 0; i < 4; i++) {
      l = __builtin_fmaf(l, pow2(m - base[i]), s_sum[i][half * NC + cn]);
      m = base[i];
    }
    l = half_swap_sum(l);
    if (cv && half == 0) p.pml[slot] = make_float2(m, l);
  }
  for (int dt = wave; dt < G::DT; dt += 4) {
    f32x16 o = {};
    m = kNone;
#pragma unroll
    for (int i = 0; i < 4; i++) {
      if (!any_seen(p, lo, hi, seg0 + i * S, S)) continue;
      const float f = pow2(m - base[i]);
      m = base[i];
#pragma unroll
      for (int e = 0; e < 16; e++) o[e] *= f;
#pragma unroll
      for (int kt = 0; kt < KT; kt++) {
        uint4 u[PU];
#pragma unroll
        for (int j = 0; j < PU; j++) u[j] = s_p[((i * KT + kt) * PU + j) * 2 * NC + half * NC + cn];
        G::accumulate(s_v, i * S + kt * 32, dt, lane, u, o);
      }
    }
    if (cv) {
      float* to = p.po + slot * V + 32 * dt;
#pragma unroll
      for (int b = 0; b < 4; b++)
        *reinterpret_cast<f32x4*>(to + 8 * b + 4 * half) = f32x4{o[4 * b], o[4 * b + 1], o[4 * b + 2], o[4 * b + 3]};
    }
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

// Split route: folds a column's segments; one wave per column.
template <typename T, int D, int V>
__global__ void __launch_bounds__(256) combine_kernel(Args p) {
  using G = Geo<T, D, V>;
  constexpr int NV = (V + 63) / 64;
  if ((int)blockIdx.x < p.fill_blocks) {
    fill<T, V>(p, blockIdx.x);
    return;
  }
  const int lane = threadIdx.x & 63;
  int64_t x = ((int64_t)blockIdx.x - p.fill_blocks) * 4 + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int cc = (int)(x % p.ccap);
  x /= p.ccap;
  const int kvh = (int)(x % p.Hkv), r = (int)(x / p.Hkv);
  if (r >= p.R) return;
  const Request rq = request(p, r);
  const int ncol = rq.L * p.G;
  if (rq.beyond || ncol > p.split_cols || cc >= ncol) return;
  // The columns that shared a workgroup, and with them its segments.
  const int NC = p.ccap <= 16 ? 16 : 32;
  const int c0 = cc / NC * NC, clast = (c0 + NC < ncol ? c0 + NC : ncol) - 1;
  const Walk w = walk(p, rq.n - rq.L + c0 / p.G, rq.n - rq.L + clast / p.G, G::kSeg);
  const int n = w.count() < p.nseg ? w.count() : p.nseg;
  const int tok = cc / p.G, head = kvh * p.G + cc - tok * p.G;
  const int64_t slot = (((int64_t)r * p.Hkv + kvh) * p.ccap + cc) * p.nseg;
  float M = kNone, L = 0.f, O[NV] = {};
  for (int i0 = 0; i0 < n; i0 += 8) {
    float o[8][NV];
    float2 ml[8];
#pragma unroll
    for (int i = 0; i < 8; i++) {
      const bool in = i0 + i < n;
      ml[i] = in ? p.pml[slot + i0 + i] : make_float2(kNone, 0.f);
#pragma unroll
      for (int j = 0; j < NV; j++)
        o[i][j] = in && lane + 64 * j < V ? p.po[(slot + i0 + i) * V + lane + 64 * j] : 0.f;
    }
#pragma unroll
    for (int i = 0; i < 8; i++) {
      float fa, fb;
      fold_base(M, L, ml[i].x, ml[i].y, fa, fb);
#pragma unroll
      for (int j = 0; j < NV; j++) O[j] = __builtin_fmaf(o[i][j], fb, O[j] * fa);
    }
  }
  float e, den;
  finish(M, L, p.sinks ? (float)static_cast<const T*>(p.sinks)[head] * 1.4426950408889634f : 0.f,
         p.sinks != nullptr, e, den);
  const float inv = inverse(den);
  T* out = out_at<T>(p, r, rq, tok, head);
#pragma unroll
  for (int j = 0; j < NV; j++)
    if (lane + 64 * j < V) out[lane + 64 * j] = result<T>(O[j], e, inv);
}

// Whole route: NW waves of 32 columns each walk the steps that some column of
// the workgroup sees, two LDS buffers ahead of each other.
template <typename T, int D, int V, int NW>
__global__ void __launch_bounds__(64 * NW, (D > 128 || V > 128) ? 1 : 2) whole_kernel(Args p) {
  using G = Geo<T, D, V>;
  constexpr int S = G::kStep, KT = G::KT, PU = G::PU, DT = G::DT, NT = 64 * NW, COLS = 32 * NW;
  constexpr int KU = S * G::CH, VU = S * G::VCH;
  __shared__ uint4 s_k0[KU], s_k1[KU], s_v0[VU], s_v1[VU];
  __shared__ const char* s_row[2][2][S];
  __shared__ uint64_t s_map[4];
  __shared__ int s_scan[NW + 3];

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
  const int kvh = x % p.Hkv;
  int tile = x / p.Hkv, r = 0;
  if (!p.qstart) {
    const int per = (p.qL * p.G + COLS - 1) / COLS;
    r = tile / per;
    tile = per - 1 - (tile - r * per);
  } else {
    int before = 0, found = -1;
    for (int r0 = 0; r0 < p.R; r0 += NT) {
      int n = 0;
      if (r0 + tid < p.R) {
        const Request rq = request(p, r0 + tid);
        const int ncol = rq.L * p.G;
        n = rq.beyond || ncol <= p.split_cols ? 0 : (ncol + COLS - 1) / COLS;
      }
      int sum = n;
#pragma unroll
      for (int d = 1; d < 64; d <<= 1) {
        const int y = __shfl_up(sum, d);
        if (lane >= d) sum += y;
      }
      if (lane == 63) s_scan[wave] = sum;
      if (tid == 0) s_scan[NW] = -1;
      __syncthreads();
      int all = 0;
#pragma unroll
      for (int i = 0; i < NW; i++) {
        if (i < wave) sum += s_scan[i];
        all += s_scan[i];
      }
      if (tile >= before + sum - n && tile < before + sum) {
        s_scan[NW] = r0 + tid;
        s_scan[NW + 1] = n - 1 - (tile - (before + sum - n));
      }
      __syncthreads();
      found = s_scan[NW];
      if (found >= 0) break;
      before += all;
      __syncthreads();
    }
    if (found < 0) return;
    r = found;
    tile = s_scan[NW + 1];
  }
  r = __builtin_amdgcn_readfirstlane(r);
  tile = __builtin_amdgcn_readfirstlane(tile);
  const Request rq = request(p, r);
  const int ncol = rq.L * p.G;
  const int c0 = tile * COLS, cw = c0 + 32 * wave;
  const int clast = (c0 + COLS < ncol ? c0 + COLS : ncol) - 1;
  const int32_t p0 = rq.n - rq.L;
  const int32_t lo = p0 + c0 / p.G, hi = p0 + clast / p.G;
  // The wave's own columns; a wave without one only loads.
  const int wlast = cw + 31 < ncol ? cw + 31 : ncol - 1;
  const int32_t wlo = cw < ncol ? p0 + cw / p.G : INT32_MAX / 2, whi = cw < ncol ? p0 + wlast / p.G : -1;

  const int cc = cw + col;
  const bool cv = cc < ncol;
  const int tok = cv ? cc / p.G : 0, head = kvh * p.G + (cv ? cc - tok * p.G : 0);
  const int32_t pos = cv ? p0 + tok : -1;
  const bool whole_tile = cw + 32 <= ncol;
  uint4 q[G::NQ];
  load_query<G>(p, query_at<T>(p, r, rq, tok, head), cv, half, q);

  const Walk w = walk(p, lo, hi, S);
  const int steps = w.count();
  const char* kh = static_cast<const char*>(p.k) + kvh * p.kh * (int64_t)sizeof(T);
  const char* vh = static_cast<const char*>(p.v) + kvh * p.vh * (int64_t)sizeof(T);

  // Row addresses of a step, by the first wave: the page's number is loaded a
  // step before they are written, which is a step before they are used.
  auto page_for = [&](int j) __attribute__((always_inline)) -> int32_t {
    if (j >= steps || lane >= S) return -1;
    const int32_t key = w.unit(j) * S + lane;
    return any_seen(p, lo, hi, key, 1) ? page_of(p, r, key) : -1;
  };
  auto put_rows = [&](int j, int32_t id) __attribute__((always_inline)) {
    if (j >= steps) return;
    const char *ka = reinterpret_cast<const char*>(g_zero_row), *va = ka;
    if (id >= 0) {
      const int64_t row = row_of(p, w.unit(j) * S + lane);
      ka = kh + (id * p.kb + row * p.kn) * (int64_t)sizeof(T);
      va = vh + (id * p.vb + row * p.vn) * (int64_t)sizeof(T);
    }
    const uint64_t m = __builtin_amdgcn_ballot_w64(id >= 0);
    if (lane < S) {
      s_row[j & 1][0][lane] = ka;
      s_row[j & 1][1][lane] = va;
    }
    if (lane == 0) s_map[j & 3] = m;
  };
  auto load_step = [&](int j, uint4* kd, uint4* vd) __attribute__((always_inline)) {
    const int td = opaque(tid);
#pragma unroll
    for (int i = 0; i < (KU + NT - 1) / NT; i++) {
      const int at = i * NT + td, row = at / G::CH, c = (at - row * G::CH) ^ G::kswz(row);
      if (KU % NT == 0 || at < KU)
        __builtin_amdgcn_global_load_lds((global_void*)(s_row[j & 1][0][row] + c * 16),
                                         (lds_void*)(kd + i * NT + wave * 64), 16, 0, 0);
    }
#pragma unroll
    for (int i = 0; i < (VU + NT - 1) / NT; i++) {
      const int at = i * NT + td, row = at / G::VCH, c = (at - row * G::VCH) ^ G::vswz(row);
      if (VU % NT == 0 || at < VU)
        __builtin_amdgcn_global_load_lds((global_void*)(s_row[j & 1][1][row] + c * 16),
                                         (lds_void*)(vd + i * NT + wave * 64), 16, 0, 0);
    }
  };

  float M = kNone, L = 0.f, m = kNone, l = 0.f;
  f32x16 O[DT], o[DT];
#pragma unroll
  for (int dt = 0; dt < DT; dt++) O[dt] = f32x16{}, o[dt] = f32x16{};

  if (steps > 0) {
    if (wave == 0) {
      put_rows(0, page_for(0));
      put_rows(1, page_for(1));
    }
    __syncthreads();
    load_step(0, s_k0, s_v0);
  }
  auto step = [&](int j, const uint4* kd, const uint4* vd, uint4* kn, uint4* vn)
      __attribute__((always_inline)) {
    // LDS addresses are computed anew each step: kept across steps they, for
    // two buffers, take the registers that o and O need.
    const int ln = opaque(lane), hf = ln >> 5;
    wait_loads();     // this wave's part of step j
    __syncthreads();  // everyone's, and everyone is done with the other buffers
    int32_t id = -1;
    if (wave == 0) id = page_for(j + 2);
    if (j + 1 < steps) load_step(j + 1, kn, vn);
    const int32_t unit = w.unit(j), key0 = unit * S;
    if (any_seen(p, wlo, whi, key0, S)) {
      const uint64_t mapped = uniform(s_map[j & 3]);
      const bool full = whole_tile && mapped == (S == 64 ? ~0ull : 0xFFFFFFFFull) &&
                        all_seen(p, wlo, whi, key0, S);
      f32x16 s[KT];
      float top = -INFINITY;
#pragma unroll
      for (int kt = 0; kt < KT; kt++) {
        f32x16 c = {};
        const int row = kt * 32 + (ln & 31), sw = G::kswz(row);
#pragma unroll
        for (int t = 0; t < G::NQ; t++) c = G::score(kd[row * G::CH + ((2 * t + hf) ^ sw)], q[t], c);
        s[kt] = c;
      }
      if (!full) G::hide(s, seen_bits(p, pos, key0, mapped) >> (4 * half));
#pragma unroll
      for (int kt = 0; kt < KT; kt++)
#pragma unroll
        for (int i = 0; i < 16; i++) top = fmaxf(top, s[kt][i]);
      top = half_swap_max(top);
      const float mn = next_base(m, top, p.scale2);
      const float f = pow2(m - mn);
      if (__builtin_amdgcn_ballot_w64(mn != m) != 0) {
#pragma unroll
        for (int dt = 0; dt < DT; dt++)
#pragma unroll
          for (int i = 0; i < 16; i++) o[dt][i] *= f;
        m = mn;
      }
      uint4 pu[KT][PU];
      float psum = 0.f;
#pragma unroll
      for (int kt = 0; kt < KT; kt++) {
        f32x16 e;
#pragma unroll
        for (int i = 0; i < 16; i++)
          e[i] = __builtin_amdgcn_exp2f(__builtin_fmaf(s[kt][i], p.scale2, -m));
        if (!full) {
#pragma unroll
          for (int i = 0; i < 16; i++) e[i] = s[kt][i] == -INFINITY ? 0.f : e[i];
        }
        psum = kt == 0 ? G::sum(e) : psum + G::sum(e);
        G::pack(e, pu[kt]);
      }
      l = __builtin_fmaf(l, f, psum);
#pragma unroll
      for (int dt = 0; dt < DT; dt++)
#pragma unroll
        for (int kt = 0; kt < KT; kt++) G::accumulate(vd, kt * 32, dt, ln, pu[kt], o[dt]);
    }
    // The segment's end: fold it.
    if (j + 1 == steps || w.unit(j + 1) / 4 != unit / 4) {
      if (__builtin_amdgcn_ballot_w64(m != kNone) != 0) {
        float fa, fb;
        fold_base(M, L, m, half_swap_sum(l), fa, fb);
        if (__builtin_amdgcn_ballot_w64(fa != 1.f || fb != 1.f) == 0) {
#pragma unroll
          for (int dt = 0; dt < DT; dt++)
#pragma unroll
            for (int i = 0; i < 16; i++) O[dt][i] += o[dt][i];
        } else {
#pragma unroll
          for (int dt = 0; dt < DT; dt++)
#pragma unroll
            for (int i = 0; i < 16; i++) O[dt][i] = __builtin_fmaf(o[dt][i], fb, O[dt][i] * fa);
        }
#pragma unroll
        for (int dt = 0; dt < DT; dt++) o[dt] = f32x16{};
        m = kNone;
        l = 0.f;
      }
    }
    if (wave == 0) put_rows(j + 2, id);
  };
  for (int j = 0; j < steps; j += 2) {
    step(j, s_k0, s_v0, s_k1, s_v1);
    if (j + 1 < steps) step(j + 1, s_k1, s_v1, s_k0, s_v0);
  }

  if (!cv) return;
  float e, den;
  finish(M, L, p.sinks ? (float)static_cast<const T*>(p.sinks)[head] * 1.4426950408889634f : 0.f,
         p.sinks != nullptr, e, den);
  const float inv = inverse(den);
  T* out = out_at<T>(p, r, rq, tok, head);
#pragma unroll
  for (int dt = 0; dt < DT; dt++)
#pragma unroll
    for (int b = 0; b < 4; b++) {
      typedef T T4 __attribute__((ext_vector_type(4)));
      T4 y;
#pragma unroll
      for (int i = 0; i < 4; i++) y[i] = result<T>(O[dt][4 * b + i], e, inv);
      *reinterpret_cast<T4*>(out + 32 * dt + 8 * b + 4 * half) = y;
    }
}

template <typename T, int D, int V>
Kernels kernels_of() {
  Kernels k;
  k.split16 = split_kernel<T, D, V, 16>;
  k.split32 = split_kernel<T, D, V, 32>;
  k.combine = combine_kernel<T, D, V>;
  k.whole = whole_kernel<T, D, V, 4>;
  k.step = Geo<T, D, V>::kStep;
  k.whole_cols = 128;
  k.whole_threads = 256;
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
