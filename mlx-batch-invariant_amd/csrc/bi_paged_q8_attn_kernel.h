// Batch-invariant attention over a paged cache of 8 bits: the kernel templates,
// included by one unit per head-dim pair (bi_paged_q8_attn_d*.hip). What is said
// in bi_paged_attn_kernel.h of columns, walks, segments, their fold, routes and
// the ring holds here too; this is what differs.
//
// Mathematics. Row j has codes k_j and v_j in -127 .. 127 and scales ks_j and
// vs_j. Scores are s_j = raw_j * c_j with raw_j = q . k_j and c_j = ks_j * a, and
// out = sum_j (2^(s_j) vs_j) v_j / (sum_j 2^(s_j) + 2^(sink * log2 e)).
//
// Fixed arithmetic of a column:
//   * Steps are of 64 rows for all head dims, eight to a segment.
//   * A code is a whole number, which bf16 and f16 hold exactly: raw_j is a
//     chain of 16x16x32 products of codes and the query over the head dim. The
//     lanes' quarter g takes the codes of 16-byte chunk 4 c + g in products 2 c
//     and 2 c + 1, eight each (what is left of 96 dims: of 8-byte piece 8 + g).
//   * c_j is rounded once to 32 bits; p_j = 2^(fma(raw_j, c_j, -m)); l sums the p
//     of 32 bits, in a fixed order per quarter.
//   * bf16: the weights p_j * vs_j are rounded to bf16, whose range holds any
//     scale: half a step of 2^-8 of a weight whose value's code is off by as much
//     as 2^-8 of the largest. f16: the scale's power of two 2^e, kept to 2^-14 ..
//     2^9, goes with the codes, which stay exact (127 * 2^9 is below f16's
//     largest, 2^-14 its smallest normal number), and the weights p_j * (vs_j /
//     2^e), of p's own size for scales in that range, are rounded to f16. (Scales
//     past 2^19, of values past 6e7, overflow them.)
// A row that a column does not see has the raw score -inf, and with it p and
// weight 0, whatever its codes, which are finite. Its scales are made so too: a row
// whose scales are infinite or NaN, or negative for keys, gets c_j above 0 and vs_j =
// 0, and a mark by which the sum, and with it the result, of every column that sees
// the row is NaN. So no row's content reaches a token that does not see it, and there
// is no case of values to look for.
//
// (Products of 16 columns, not of 32 as in the kernels of the other types: single
// tokens have 4 or 8, and what a wave spends its time on there is the issue of
// vector instructions, one in 5 cycles, for conversions, exponentials and
// addresses. Half the columns are half of these, and half the registers, so that
// more waves share a SIMD.)
#pragma once

#include "bi_paged_attn_kernel.h"

namespace bi_paged {
namespace {

typedef int i32x2 __attribute__((ext_vector_type(2)));
typedef __attribute__((address_space(3))) i32x2 lds_i32x2;
typedef __attribute__((address_space(3))) const u32x4 lds_u32x4;

// Four codes as two dwords of bf16 or f16.
template <typename T> __device__ __forceinline__ uint2 codes4(uint32_t w) {
  if constexpr (__is_same(T, __bf16)) {
    const f32x2 a = {(float)(int8_t)w, (float)(int8_t)(w >> 8)};
    const f32x2 b = {(float)(int8_t)(w >> 16), (float)(int8_t)(w >> 24)};
    return make_uint2(__builtin_bit_cast(uint32_t, __builtin_convertvector(a, bf16x2)),
                      __builtin_bit_cast(uint32_t, __builtin_convertvector(b, bf16x2)));
  } else {
    // 0x6400 + n is 1024 + n for n = code + 128; the subtraction is exact.
    // (An instruction takes one constant: the other is put into a register here, not
    // kept in one that others need.)
    w ^= 0x80808080u;
    const uint32_t high = (uint32_t)opaque(0x64646464);
    const f16x2 bias = {(_Float16)1152.f, (_Float16)1152.f};
    const f16x2 a = __builtin_bit_cast(f16x2, __builtin_amdgcn_perm(high, w, 0x04010400u)) - bias;
    const f16x2 b = __builtin_bit_cast(f16x2, __builtin_amdgcn_perm(high, w, 0x04030402u)) - bias;
    return make_uint2(__builtin_bit_cast(uint32_t, a), __builtin_bit_cast(uint32_t, b));
  }
}
template <typename T> __device__ __forceinline__ uint4 codes8(uint32_t lo, uint32_t hi) {
  const uint2 a = codes4<T>(lo), b = codes4<T>(hi);
  return make_uint4(a.x, a.y, b.x, b.y);
}
// f16 times powers of two, two to a dword.
__device__ __forceinline__ uint4 times(uint4 x, uint4 f) {
  auto mul = [](uint32_t a, uint32_t b) __attribute__((always_inline)) {
    return __builtin_bit_cast(uint32_t, __builtin_bit_cast(f16x2, a) * __builtin_bit_cast(f16x2, b));
  };
  return make_uint4(mul(x.x, f.x), mul(x.y, f.y), mul(x.z, f.z), mul(x.w, f.w));
}
// The part of a value's scale that goes with its codes, as f16, and what is left.
__device__ __forceinline__ uint16_t scale_power(float vs, float& left) {
  int e = __builtin_amdgcn_frexp_expf(vs) - 1;
  e = e < -14 ? -14 : e > 9 ? 9 : e;
  left = __builtin_amdgcn_ldexpf(vs, -e);
  return (uint16_t)((e + 15) << 10);
}

// The largest, and the sum, of a column's four quarters.
__device__ __forceinline__ float quarters_max(float x) {
  const auto r = __builtin_amdgcn_permlane16_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  return half_swap_max(__builtin_elementwise_maximum(__uint_as_float(r[0]), __uint_as_float(r[1])));
}
__device__ __forceinline__ float quarters_sum(float x) {
  const auto r = __builtin_amdgcn_permlane16_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  return half_swap_sum(__uint_as_float(r[0]) + __uint_as_float(r[1]));
}

// A segment's sum, NaN where its base is so far from 0 that a score's own rounding,
// which the base has and the exponent has not, is beyond what a weight holds. Half a
// step of a score is 64 from 2^30 on, with which an exponential may leave bf16's range
// (at twice that it is 2^128), and 16 from 2^28 on, with which it leaves f16's
// (below, p is at most 2^12 and the largest at least 2^-8).
template <typename T> __device__ __forceinline__ float within(float m, float l) {
  constexpr float kFar = __is_same(T, _Float16) ? 268435456.f : 1073741824.f;
  return fabsf(m) < kFar || m == kNone ? l : NAN;
}

template <typename T, int D_, int V_>
struct Geo8 {
  static constexpr int D = D_, V = V_;
  static constexpr int kStep = 64, RT = kStep / 16, kSegSteps = 8, kSeg = kSegSteps * kStep;
  static constexpr int CH = D / 16, VCH = V / 16;  // 16-byte chunks of a row of codes
  static constexpr int MCH = CH > VCH ? CH : VCH;
  static constexpr int NQ = D / 32;                // products of a score
  static constexpr int DT = V / 16;                // tiles of output dims
  static constexpr int TCH = D / 8, TVCH = V / 8;  // chunks of a row in the type
  static constexpr bool kPower = __is_same(T, _Float16);  // values' codes carry 2^e
  static constexpr bool kTwoWaves = V + D / 4 <= 160;     // whole route: two waves per SIMD
  // Whole route: products of a wave's second 16 columns whose query waits in LDS
  // (128 dims: with all in registers, of which 234 are in use at once, some were
  // kept in scratch memory).
  static constexpr int kFarQuery = D == 128 && V == 128 ? NQ : 0;
  // Whole route, a step as it lies in LDS: 16-byte units of keys, of values (both in
  // the type), then c_j, what values are multiplied with, and the masks of the rows
  // that have a page and that spoil. Laid out in memory the same.
  static constexpr int KU = kStep * TCH, VU = kStep * TVCH, FU = kStep / 4;
  static constexpr int IU = (KU + VU + 2 * FU + 1 + 31) / 32 * 32;  // (whole rows: LDS addresses are multiples of these)
  // Steps of them in LDS.
  static constexpr int kDeep = 3 * IU * 16 <= 150 * 1024 ? 3 : 2;
  // Split route: workgroups of NC columns that a compute unit's registers hold.
  static constexpr int split_per_cu(int NC) {
    return NC == 16 ? (D + V <= 128 ? 4 : D + V <= 256 ? 3 : 2) : (D + V <= 128 ? 3 : D + V <= 320 ? 2 : 1);
  }

  // Prices of a row and of a segment (for the choice of route), fitted to the times
  // of 666 sizes with each route: rows whose chunks are no power of two cost the
  // whole workgroups, where all waves share the loads, and small splits more.
  static constexpr bool kPow2 = (CH & (CH - 1)) == 0 && (VCH & (VCH - 1)) == 0;
  static constexpr double row_us() {
    return 1e-3 * (kTwoWaves ? 14.0 + 0.047 * (D + V) + (kPow2 ? 0.0 : 10.0) : 24.0 + 0.0725 * (D + V));
  }
  static constexpr double laid_row_us() { return 1e-3 * (10.0 + 0.051 * (D + V)); }
  // (One workgroup's ends are beside another's rows where a compute unit has two.)
  static constexpr double laid_tile_us() { return D + V <= 192 ? 3.0 : 7.5; }
  static constexpr double seg_us(int NC) {
    if (NC == 32) return 9.2 + 0.0135 * (D + V);
    return kTwoWaves ? 4.0 + 0.006 * (D + V) + (kPow2 ? 0.0 : 2.0) : 2.0 + 0.026 * (D + V);
  }

  __device__ __forceinline__ static f32x4 product(uint4 a, uint4 b, f32x4 c) {
    if constexpr (kPower)
      return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
    else
      return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
  }
  // The 16-byte piece (eight dims in the type) that quarter g takes in product n.
  __device__ __forceinline__ static int piece(int n, int g) {
    return NQ % 2 && n + 1 == NQ ? 4 * n + g : 2 * (4 * (n >> 1) + g) + (n & 1);
  }

  // Rows in LDS, of C chunks: row r's chunk c at chunk c ^ swz<C>(r). A read takes
  // one chunk of 16 rows per pass, which the exchange spreads over all banks.
  template <int C> __device__ __forceinline__ static uint32_t swz(uint32_t r) {
    if constexpr (C % 16 == 0) return r & 15;
    else if constexpr (C % 8 == 0) return (r >> 1) & 7;
    else if constexpr (C % 4 == 0) return (r >> 2) & 3;
    else return (r >> 3) & 1;
  }
  // Values of codes: row r at place vplace(r), which puts the eight rows of a
  // product's quarter (4 g .. and 16 + 4 g ..) side by side.
  __device__ __forceinline__ static uint32_t vplace(uint32_t r) {
    return (r & 35) | ((r >> 2) & 4) | ((r << 1) & 24);
  }
  // Values in the type (whole route): a transposing read takes four rows, of two
  // quarters 32 bytes of eight rows per pass. (The lowest bit is for the stores.)
  __device__ __forceinline__ static uint32_t tswz(uint32_t r) {
    if constexpr (TVCH % 16 == 0) return (r & 7) << 1 | (r & 1);
    else if constexpr (TVCH % 8 == 0) return ((r >> 1) & 3) << 1 | (r & 1);
    else return ((r >> 2) & 1) << 1 | (r & 1);
  }
  // Row and chunk of the unit that thread `t` of N takes in turn j, rows of C chunks.
  template <int C, int N> struct Unit {
    uint32_t row, chunk;
    __device__ __forceinline__ Unit(int j, uint32_t t) {
      if constexpr (N % C == 0) row = j * (N / C) + t / C, chunk = t % C;
      else row = (j * N + t) / C, chunk = j * N + t - row * C;
    }
  };
  // Byte offset in LDS of a unit that lane `t` of a wave stores in turn j. Where
  // rows are a power of two of chunks, turns differ by constants: places and
  // exchanges are permutations of the row number's bits.
  template <int C, typename Place>
  __device__ __forceinline__ static uint32_t stored(int j, uint32_t t, const Place& place) {
    if constexpr ((C & (C - 1)) == 0) {
      const uint32_t at = place(t / C), turn = place(j * (64 / C));
      return ((at * C + ((t % C) ^ swz<C>(at))) * 16 ^ swz<C>(turn) * 16) + turn * C * 16;
    } else {
      const Unit<C, 64> x(j, t);
      const uint32_t at = place(x.row);
      return (at * C + (x.chunk ^ swz<C>(at))) * 16;
    }
  }
  __device__ __forceinline__ static uint32_t key_stored(int j, uint32_t t) {
    return stored<CH>(j, t, [](uint32_t r) { return r; });
  }
  __device__ __forceinline__ static uint32_t value_stored(int j, uint32_t t) {
    return stored<VCH>(j, t, [](uint32_t r) { return vplace(r); });
  }

  // Products 2 c and 2 c + 1 (one: the last of an odd number) of a tile of 16 rows
  // of codes, as operands.
  __device__ __forceinline__ static void keys(const uint4* k, int row0, int c, uint32_t ln, uint4 (&x)[2]) {
    const uint32_t own = ln & 15, g = ln >> 4;
    const char* row = reinterpret_cast<const char*>(k) + row0 * CH * 16 + own * CH * 16;
    if (NQ % 2 && 2 * c + 1 == NQ) {
      const uint2 w = *reinterpret_cast<const uint2*>(row + ((4 * c + (g >> 1)) ^ swz<CH>(own)) * 16 + 8 * (g & 1));
      x[0] = codes8<T>(w.x, w.y);
    } else {
      const u32x4 w = *reinterpret_cast<const u32x4*>(row + ((4 * c + g) ^ swz<CH>(own)) * 16);
      x[0] = codes8<T>(w[0], w[1]);
      x[1] = codes8<T>(w[2], w[3]);
    }
  }
  // The values' operand of product u of a step's codes, output dims 16 dt ..;
  // `power`: 2^e by place. (The exchange depends on the lane alone.)
  __device__ __forceinline__ static uint4 value(const uint4* v, const uint16_t* power, int u, int dt, uint32_t ln) {
    const uint32_t own = 8 * (ln >> 4) + ((ln & 15) >> 1);
    const char* from = reinterpret_cast<const char*>(v) + ((own * VCH + (dt ^ swz<VCH>(own))) * 16 + 8 * (ln & 1)) +
                       32 * u * VCH * 16;
    const i32x2 x = __builtin_amdgcn_ds_read_tr8_b64_v2i32((lds_i32x2*)from);
    const uint4 y = codes8<T>((uint32_t)x[0], (uint32_t)x[1]);
    if constexpr (!kPower) return y;
    else return times(y, *reinterpret_cast<const uint4*>(power + 32 * u + 8 * (ln >> 4)));
  }
  // The same operands from rows in the type. Which product or output tile it is turns
  // bits of the lane's chunk, which are bits of its address where rows are a power of
  // two long and the LDS address is a multiple of one: an instruction for each operand.
  struct OfType {
    uint32_t row, chunk;  // LDS address of the lane's row, and its chunk's place in it, in bytes
    template <int C> __device__ __forceinline__ uint32_t at(uint32_t turn) const {
      if constexpr ((C & (C - 1)) == 0) return (row + chunk) ^ turn;
      else return row + (chunk ^ turn);
    }
    __device__ __forceinline__ static uint32_t lds(const uint4* p) { return (uint32_t)(uintptr_t)(lds_void*)const_cast<uint4*>(p); }
  };
  __device__ __forceinline__ static OfType keys_of_type(const uint4* k, uint32_t ln) {
    const uint32_t own = ln & 15, g = ln >> 4;
    return {OfType::lds(k) + own * TCH * 16, ((2 * g) ^ swz<TCH>(own)) * 16};
  }
  __device__ __forceinline__ static uint4 key_of_type(const OfType& k, int row0, int n, uint32_t ln) {
    uint32_t at;
    if (NQ % 2 && n + 1 == NQ) at = k.row + (piece(n, ln >> 4) ^ swz<TCH>(ln & 15)) * 16;
    else at = k.template at<TCH>(piece(n, 0) * 16);
    return __builtin_bit_cast(uint4, *(lds_u32x4*)(uintptr_t)(at + row0 * TCH * 16));
  }
  __device__ __forceinline__ static OfType values_of_type(const uint4* v, uint32_t ln) {
    const uint32_t own = 4 * (ln >> 4) + ((ln & 15) >> 2), part = ln & 3;
    return {OfType::lds(v) + own * TVCH * 16, ((part >> 1) ^ tswz(own)) * 16 + 8 * (part & 1)};
  }
  __device__ __forceinline__ static uint4 value_of_type(const OfType& v, int u, int dt) {
    const uint32_t at = v.template at<TVCH>(dt * 32);
    i16x4 a[2];
#pragma unroll
    for (int x = 0; x < 2; x++)  // (tswz has bits 0 to 2 of the row: rows 16 on have the same)
      a[x] = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_i16x4*)(uintptr_t)(at + (32 * u + 16 * x) * TVCH * 16));
    const uint2 lo = __builtin_bit_cast(uint2, a[0]), hi = __builtin_bit_cast(uint2, a[1]);
    return make_uint4(lo.x, lo.y, hi.x, hi.y);
  }

  __device__ __forceinline__ static void load_query(const char* q, int g, uint4 (&out)[NQ]) {
#pragma unroll
    for (int n = 0; n < NQ; n++) out[n] = ld16(q + piece(n, g) * 16);
  }
  __device__ __forceinline__ static void sign_query(const Args& p, uint4 (&q)[NQ]) {
#pragma unroll
    for (int n = 0; n < NQ; n++)
      q[n] = make_uint4(q[n].x ^ p.qsign, q[n].y ^ p.qsign, q[n].z ^ p.qsign, q[n].w ^ p.qsign);
  }

  // A row's c_j, above 0 so that an unseen row's -inf stays one, and what its
  // values' weights are multiplied with; whether it spoils what sees it.
  __device__ __forceinline__ static bool factors(const Args& p, float ks, float vs, float& c, float& left, uint16_t& power) {
    c = ks * p.scale2;
    const bool good = ks >= 0.f && c < INFINITY && fabsf(vs) < INFINITY;
    c = good ? fmaxf(c, 1.2e-38f) : 1.f;
    left = good ? vs : 0.f;
    if constexpr (kPower) power = scale_power(left, left);
    return !good;
  }
  // Element i of row tile t is row 16 t + 4 g + i; `seen` is shifted by 4 g.
  __device__ __forceinline__ static f32x4 rows4(const float* at, int t, int g) {
    return *reinterpret_cast<const f32x4*>(at + 16 * t + 4 * g);
  }
  // Scores of unseen rows become -inf.
  template <int CT> __device__ __forceinline__ static void hide(f32x4 (&s)[RT][CT], const uint64_t (&seen)[CT]) {
#pragma unroll
    for (int t = 0; t < RT; t++)
#pragma unroll
      for (int k = 0; k < CT; k++) {
        const uint32_t w = (uint32_t)(seen[k] >> (16 * t));
#pragma unroll
        for (int i = 0; i < 4; i++) s[t][k][i] = w & (1u << i) ? s[t][k][i] : -INFINITY;
      }
  }
  // The largest scores of CT column tiles.
  template <int CT>
  __device__ __forceinline__ static void top(const f32x4 (&s)[RT][CT], const float* c, int g, float (&m)[CT]) {
#pragma unroll
    for (int k = 0; k < CT; k++) m[k] = -INFINITY;
#pragma unroll
    for (int t = 0; t < RT; t++) {
      const f32x4 f = rows4(c, t, g);
#pragma unroll
      for (int k = 0; k < CT; k++) {
        f32x4 x;
#pragma unroll
        for (int i = 0; i < 4; i++) x[i] = s[t][k][i] * f[i];
        m[k] = __builtin_elementwise_maximum(__builtin_elementwise_maximum(m[k], x[0]), x[1]);
        m[k] = __builtin_elementwise_maximum(__builtin_elementwise_maximum(m[k], x[2]), x[3]);
      }
    }
#pragma unroll
    for (int k = 0; k < CT; k++) m[k] = quarters_max(m[k]);
  }
  // A step's weights in the type, and the lane's sums of p: a chain for the eight
  // rows of a product, then both. (Four rows at a time: else the compiler reads all
  // factors first, into registers that there are not.)
  template <int CT, bool ALL = false>
  __device__ __forceinline__ static void weights(const f32x4 (&s)[RT][CT], const float* c, const float* vs, int g,
                                                 const float (&m)[CT], uint4 (&u)[RT / 2][CT], float (&sum)[CT]) {
#pragma unroll
    for (int j = 0; j < RT / 2; j++) {
      uint32_t d[CT][4];
      float l[CT];
#pragma unroll
      for (int b = 0; b < 2; b++) {
        const int t = 2 * j + b;
        const f32x4 f = rows4(c, t, g), h = rows4(vs, t, g);
#pragma unroll
        for (int k = 0; k < CT; k++) {
          f32x4 e;
#pragma unroll
          for (int i = 0; i < 4; i++) {
            e[i] = __builtin_amdgcn_exp2f(__builtin_fmaf(s[t][k][i], f[i], -m[k]));
            l[k] = b == 0 && i == 0 ? e[i] : l[k] + e[i];
          }
          f32x4 z;
#pragma unroll
          for (int i = 0; i < 4; i++) z[i] = e[i] * h[i];
#pragma unroll
          for (int i = 0; i < 2; i++) {
            const f32x2 two = {z[2 * i], z[2 * i + 1]};
            if constexpr (kPower) d[k][2 * b + i] = __builtin_bit_cast(uint32_t, __builtin_convertvector(two, f16x2));
            else d[k][2 * b + i] = __builtin_bit_cast(uint32_t, __builtin_convertvector(two, bf16x2));
          }
        }
        if constexpr (!ALL) __builtin_amdgcn_sched_barrier(0);
      }
#pragma unroll
      for (int k = 0; k < CT; k++) {
        u[j][k] = make_uint4(d[k][0], d[k][1], d[k][2], d[k][3]);
        sum[k] = j == 0 ? l[k] : sum[k] + l[k];
      }
    }
  }
  // Columns that see a row that spoils them.
  template <int CT> __device__ __forceinline__ static void spoil(const Args& p, const int32_t (&pos)[CT], int32_t key0, uint64_t bad, float (&sum)[CT]) {
#pragma unroll
    for (int k = 0; k < CT; k++)
      if (seen_bits(p, pos[k], key0, bad) != 0) sum[k] = NAN;
  }
};

// As feed(), with the operands A products ahead.
template <int N, int A, typename Read, typename Use>
__device__ __forceinline__ void feed_ahead(const Read& read, const Use& use) {
  static_assert(N % A == 0, "groups");
  uint4 x[2][A];
#pragma unroll
  for (int i = 0; i < A; i++) x[0][i] = read(i);
#pragma unroll
  for (int n = 0; n < N; n += A) {
    __builtin_amdgcn_sched_barrier(0);
    if (n + A < N)
#pragma unroll
      for (int i = 0; i < A; i++) x[(n / A + 1) & 1][i] = read(n + A + i);
    __builtin_amdgcn_sched_barrier(0);
#pragma unroll
    for (int i = 0; i < A; i++) use(n + i, x[(n / A) & 1][i]);
  }
}

// barrier(), N instruction words behind a multiple of the 32 bytes that are fetched at a
// time (behind s_nop 0).
template <int N> __device__ __forceinline__ void barrier_at() {
  asm volatile("s_waitcnt lgkmcnt(0)\n\t.p2align 5\n\t.fill %0, 4, 0xbf800000\n\ts_barrier" ::"i"(N) : "memory");
}
__device__ __forceinline__ uint2 ld8(const void* p) {
  typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));
  typedef __attribute__((address_space(1))) const u32x2 gvec;
  return __builtin_bit_cast(uint2, *(gvec*)p);
}
// A row of a page, and its scale from device memory, as ld16; zeros for a row
// without a page.
__device__ __forceinline__ const char* row_at(const char* base, int32_t id, uint32_t page, int32_t row, uint32_t step) {
  const char* at = base + ((uint64_t)(uint32_t)id * page + (uint64_t)(uint32_t)row * step);
  return id >= 0 ? at : reinterpret_cast<const char*>(g_zero_row);
}
__device__ __forceinline__ float ld_scale(const char* at) {
  typedef __attribute__((address_space(1))) const float gfloat;
  return *(gfloat*)at;
}

// Split route: a segment's (m, l, o) of NC columns, four steps to a pass, one
// per wave, as for the other types. Keys and values of the next pass are on their
// way through registers of their own while a pass is computed, across the ends of
// the workgroup's segments.
template <typename T, int D, int V, int NC>
__global__ void __launch_bounds__(256, (Geo8<T, D, V>::split_per_cu(NC))) split8_kernel(Args p) {
  using G8 = Geo8<T, D, V>;
  constexpr int S = G8::kStep, RT = G8::RT, CT = NC / 16, NU = RT / 2;
  __shared__ uint4 s_kv[4 * S * G8::MCH];  // a step per wave: its keys, then its values
  __shared__ uint4 s_p[4 * NU * CT * 64];
  __shared__ const char* s_row[2][4 * S];
  __shared__ __attribute__((aligned(16))) float s_c[4 * S], s_vs[4 * S];
  __shared__ __attribute__((aligned(16))) uint16_t s_pow[G8::kPower ? 4 * S : 8];
  __shared__ float s_max[4][NC];
  __shared__ float s_sum[4][CT * 64];

  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int col = lane & 15, g = lane >> 4;
  // Workgroup -> kv head, columns, segment of the walk, request. Neighbours in the
  // grid land on different XCDs: so do neighbouring heads, but for a cache whose
  // rows hold all heads side by side, which share lines, of scales above all: there
  // a row's heads go to one XCD (64 requests in a token-major cache, 128 dims 163 ->
  // 153 us, 64 dims 136 -> 114; in a head-major one it costs 132 -> 136, and with
  // 256 dims 150 -> 163).
  const int x = blockIdx.x;
  int xc = x / p.Hkv, kvh = x - xc * (int)p.Hkv.d;
  if (p.eight.d) {
    const int set = x / p.eight, at = x - set * (int)p.eight.d;
    kvh = at >> 3, xc = 8 * set + (at & 7);
    if (xc >= (int)(p.slots.d * p.ctiles.d)) return;  // (the grid is rounded up)
  }
  const int xq = xc / (p.once ? p.slots : p.ctiles);
  const int xr = xc - xq * (int)(p.once ? p.slots : p.ctiles).d;
  const int xs = p.once ? xr : xq, c0 = (p.once ? xq : xr) * NC;
  const int outer = xs / (p.window ? p.reqs : p.gseg);
  const int inner = xs - outer * (int)(p.window ? p.reqs : p.gseg).d;
  const int r = p.window ? inner : outer, part0 = p.window ? outer : inner;
  constexpr int PS = 4 * S, PN = G8::kSeg / PS;
  int32_t entry0 = 0, entry = 0;
  if (!p.window) {
    entry0 = entry_of(p, r, part0 * G8::kSeg + wave * S + lane);
    entry = entry_of(p, r, part0 * G8::kSeg + PS + wave * S + lane);
  }
  const Request rq = request(p, r);
  const int ncol = rq.L * (int)p.G.d;
  if (rq.beyond || ncol > p.split_cols || c0 >= ncol) return;
  const int clast = (c0 + NC < ncol ? c0 + NC : ncol) - 1;
  const int32_t lo = rq.n - rq.L + c0 / p.G, hi = rq.n - rq.L + clast / p.G;
  const Walk w = walk(p, lo, hi, G8::kSeg);
  const int parts = w.count() < (int)p.nseg.d ? w.count() : p.nseg.d;
  if (part0 >= parts) return;

  // Columns; one without a token takes the first one's query, and nobody its result.
  bool cv[CT];
  int32_t pos[CT];
  const char* qa[CT];
#pragma unroll
  for (int k = 0; k < CT; k++) {
    const int cc = c0 + 16 * k + col;
    cv[k] = cc < ncol;
    const int cq = cv[k] ? cc : c0, tok = cq / p.G;
    pos[k] = cv[k] ? rq.n - rq.L + tok : -1;
    qa[k] = query_at<T>(p, r, rq, tok, kvh * (int)p.G.d + (cq - tok * (int)p.G.d));
  }
  const char* kh = static_cast<const char*>(p.k) + kvh * p.kh;
  const char* vh = static_cast<const char*>(p.v) + kvh * p.vh;
  const char* ksh = reinterpret_cast<const char*>(p.ks + kvh * p.ksh);
  const char* vsh = reinterpret_cast<const char*>(p.vs + kvh * p.vsh);

  // A pass of the workgroup's parts of the walk, which it takes one after the
  // other as one run of passes: pass `si` (counted from the request's first row)
  // of segment `part`, whose passes that some column sees end before `s1`.
  struct At {
    int part, si, s1;
  };
  auto open = [&](At& t) __attribute__((always_inline)) {
    if (t.part >= parts) return;
    t.si = w.unit(t.part) * PN, t.s1 = t.si + PN;
    while (t.si < t.s1 && !any_seen(p, lo, hi, t.si * PS, PS)) t.si++;
    while (t.si < t.s1 && !any_seen(p, lo, hi, (t.s1 - 1) * PS, PS)) t.s1--;
  };
  auto after = [&](At t) __attribute__((always_inline)) -> At {
    if (t.part < parts && ++t.si >= t.s1) {
      t.part += p.gseg.d;
      open(t);
    }
    return t;
  };
  // Row addresses of the wave's step of a pass, and its scales, on their way; a row
  // that no column sees, or that has no page, is a row of zeros.
  float ks, vs;
  auto entry_for = [&](const At& t) __attribute__((always_inline)) -> int32_t {
    return entry_of(p, r, t.si * PS + wave * S + lane);
  };
  auto put_rows = [&](const At& t, int32_t entry) __attribute__((always_inline)) -> uint64_t {
    const int32_t key = t.si * PS + wave * S + lane;
    const int32_t id = t.part < parts && any_seen(p, lo, hi, key, 1) ? page_of(p, r, entry, key) : -1;
    const int32_t row = row_of(p, key);
    s_row[0][wave * S + lane] = row_at(kh, id, p.k8b, row, p.k8n);
    s_row[1][wave * S + lane] = row_at(vh, id, p.v8b, row, p.v8n);
    ks = ld_scale(row_at(ksh, id, p.ksb, row, p.ksn));
    vs = ld_scale(row_at(vsh, id, p.vsb, row, p.vsn));
    __builtin_amdgcn_wave_barrier();
    return __builtin_amdgcn_ballot_w64(id >= 0);
  };
  // Rows are loaded whole, consecutive lanes taking consecutive chunks.
  constexpr int KL = S * G8::CH / 64, VL = S * G8::VCH / 64;
  uint4 xk[KL], xv[VL], q[CT][G8::NQ];
  auto load_rows = [&](uint4* to, const char* const* rows, auto chunks, auto load) __attribute__((always_inline)) {
    constexpr int C = decltype(chunks)::value;
    const int ln = opaque(lane);
#pragma unroll
    for (int j = 0; j < S * C / 64; j++) {
      const typename G8::template Unit<C, 64> u(j, ln);
      to[j] = load(rows[wave * S + u.row] + u.chunk * 16);
    }
  };
  // (Past the caches, but for lines that hold parts of other heads' rows too.)
  const bool past = p.once && (!p.eight.d || (G8::CH % 8 == 0 && G8::VCH % 8 == 0));
  auto load_keys = [&]() __attribute__((always_inline)) {
    if (past) load_rows(xk, s_row[0], std::integral_constant<int, G8::CH>(), ld16_once);
    else load_rows(xk, s_row[0], std::integral_constant<int, G8::CH>(), ld16);
  };
  auto load_values = [&]() __attribute__((always_inline)) {
    if (past) load_rows(xv, s_row[1], std::integral_constant<int, G8::VCH>(), ld16_once);
    else load_rows(xv, s_row[1], std::integral_constant<int, G8::VCH>(), ld16);
  };

  // Keys and values of the next pass and the table's entries of the one after it
  // are on their way while a pass is computed, whichever segments these are of.
  At at = {part0, 0, 0};
  open(at);
  At next = after(at);
  if (p.window) entry0 = entry_for(at);
  if (p.window || next.part != part0) entry = entry_for(next);
#pragma unroll
  for (int k = 0; k < CT; k++) G8::load_query(qa[k], g, q[k]);
  uint64_t mapped = put_rows(at, entry0);
  load_keys();
  load_values();
#pragma unroll
  for (int k = 0; k < CT; k++) G8::sign_query(p, q[k]);

  constexpr int TW = (G8::DT + 3) / 4;  // tiles of output dims per wave
  float m[CT], l[CT];
  f32x4 o[TW][CT];
  auto begin = [&]() __attribute__((always_inline)) {
#pragma unroll
    for (int k = 0; k < CT; k++) {
      m[k] = kNone, l[k] = 0.f;
#pragma unroll
      for (int y = 0; y < TW; y++) o[y][k] = f32x4{};
    }
  };
  begin();
  for (;;) {
    const int32_t pass0 = at.si * PS, key0 = pass0 + wave * S;
    const At third = after(next);
    const int32_t entry2 = entry_for(third);
    const int lk = opaque(lane);
    uint4* own = s_kv + wave * S * G8::MCH;
#pragma unroll
    for (int j = 0; j < KL; j++)
      st16(reinterpret_cast<uint4*>(reinterpret_cast<char*>(own) + G8::key_stored(j, lk)), xk[j]);
    float c, left;
    uint16_t power = 0;
    const uint64_t bad = __builtin_amdgcn_ballot_w64(G8::factors(p, ks, vs, c, left, power));
    s_c[wave * S + lk] = c;
    s_vs[wave * S + lk] = left;
    if constexpr (G8::kPower) s_pow[wave * S + G8::vplace(lk)] = power;
    const uint64_t now = mapped;
    mapped = put_rows(next, entry);
    entry = entry2;
    load_keys();
    __builtin_amdgcn_wave_barrier();
    // Scores of the wave's step and their largest.
    f32x4 s[RT][CT];
#pragma unroll
    for (int t = 0; t < RT; t++) {
#pragma unroll
      for (int k = 0; k < CT; k++) s[t][k] = f32x4{};
#pragma unroll
      for (int c = 0; c < (G8::NQ + 1) / 2; c++) {
        uint4 x[2];
        G8::keys(own, 16 * t, c, lk, x);
#pragma unroll
        for (int n = 2 * c; n < 2 * c + 2 && n < G8::NQ; n++)
#pragma unroll
          for (int k = 0; k < CT; k++) s[t][k] = G8::product(x[n & 1], q[k][n], s[t][k]);
      }
    }
    const bool full = now == ~0ull && all_seen(p, lo, hi, key0, S);
    if (!full) {
      uint64_t seen[CT];
#pragma unroll
      for (int k = 0; k < CT; k++) seen[k] = seen_bits(p, pos[k], key0, now) >> (4 * g);
      G8::template hide<CT>(s, seen);
    }
    const float* cs = s_c + wave * S;
    float top[CT];
    G8::template top<CT>(s, cs, g, top);
    if (g == 0)
#pragma unroll
      for (int k = 0; k < CT; k++) s_max[wave][16 * k + col] = top[k];
    barrier();

    // The bases of the pass's steps; this wave's weights.
    float f[CT][4], mw[CT];
#pragma unroll
    for (int k = 0; k < CT; k++)
#pragma unroll
      for (int i = 0; i < 4; i++) {
        const float base = next_base(m[k], s_max[i][16 * k + col], 1.f);
        f[k][i] = pow2(m[k] - base);
        m[k] = base;
        if (i == 0 || i <= wave) mw[k] = base;
      }
    uint4 pu[NU][CT];
    float psum[CT];
    G8::template weights<CT>(s, cs, s_vs + wave * S, g, mw, pu, psum);
    if (bad & now) G8::template spoil<CT>(p, pos, key0, bad & now, psum);
    const int ln = opaque(lane);
#pragma unroll
    for (int k = 0; k < CT; k++) {
#pragma unroll
      for (int u = 0; u < NU; u++) s_p[((wave * NU + u) * CT + k) * 64 + ln] = pu[u][k];
      s_sum[wave][64 * k + ln] = psum[k];
    }
#pragma unroll
    for (int j = 0; j < VL; j++)
      st16(reinterpret_cast<uint4*>(reinterpret_cast<char*>(own) + G8::value_stored(j, ln)), xv[j]);
    load_values();
    barrier();

    // The sum, and the wave's tiles of output dims over the pass's steps.
#pragma unroll
    for (int i = 0; i < 4; i++) {
      if (!any_seen(p, lo, hi, pass0 + i * S, S)) continue;
#pragma unroll
      for (int k = 0; k < CT; k++) {
        if (wave == 0) l[k] = __builtin_fmaf(l[k], f[k][i], s_sum[i][64 * k + ln]);
        if (__builtin_amdgcn_ballot_w64(f[k][i] != 1.f) != 0)
#pragma unroll
          for (int y = 0; y < TW; y++)
#pragma unroll
            for (int e = 0; e < 4; e++) o[y][k][e] *= f[k][i];
      }
#pragma unroll
      for (int u = 0; u < NU; u++) {
        uint4 x[CT];
#pragma unroll
        for (int k = 0; k < CT; k++) x[k] = s_p[((i * NU + u) * CT + k) * 64 + ln];
#pragma unroll
        for (int y = 0; y < TW; y++) {
          const int dt = wave + 4 * y;
          if (G8::DT % 4 && dt >= G8::DT) break;
          const uint4 v = G8::value(s_kv + i * S * G8::MCH, s_pow + i * S, u, dt, ln);
#pragma unroll
          for (int k = 0; k < CT; k++) o[y][k] = G8::product(v, x[k], o[y][k]);
        }
      }
    }
    if (next.part != at.part) {  // the segment's last pass
#pragma unroll
      for (int k = 0; k < CT; k++) {
        const float sum = within<T>(m[k], quarters_sum(l[k]));
        if (!cv[k]) continue;
        const int64_t slot = (((int64_t)r * p.Hkv.d + kvh) * p.nseg.d + at.part) * p.ccap.d + c0 + 16 * k + col;
        if (wave == 0 && g == 0) p.pml[slot] = make_float2(m[k], sum);
#pragma unroll
        for (int y = 0; y < TW; y++) {
          if (wave + 4 * y >= G8::DT) break;
          *reinterpret_cast<f32x4*>(p.po + slot * V + 16 * (wave + 4 * y) + 4 * g) = o[y][k];
        }
      }
      if (next.part >= parts) return;
      begin();
    }
    barrier();  // everyone is done with the values and weights
    at = next;
    next = third;
  }
}

// Lays rows out as the whole route wants them in LDS: a unit of 16 bytes for each 8
// codes of a row, in the place it has there.
//
// What every workgroup of the whole route would do for the rows that it walks, looking
// up pages and making numbers of codes, is done once, where there is room for the
// result (4096 tokens over 8192 rows, 64 column tiles to a kv head, 128 dims: 576 ->
// 480 us; 192 dims 1342 -> 887, 256 1557 -> 912, where four waves of 32 columns gave
// way to eight of 16 as well). It costs a launch and three bytes of traffic a code:
// 12 us for these rows, and 8 requests of 64 tokens over 4000 rows would take 166 us
// for 116, so the host compares. The list of what is to do, steps of requests that are
// not split, is the same for all workgroups, which take from it in turn. Where not
// every step of every request can have a place, requests have theirs one behind the
// other, as far as there is room, and the first workgroup notes where; then those of one
// column tile, whose rows would be read once more for nothing, get none.
template <typename T, int D, int V>
__global__ void __launch_bounds__(256) lay8_kernel(Args p) {
  using G8 = Geo8<T, D, V>;
  constexpr int S = G8::kStep;
  __shared__ const char* s_row[2][S];
  __shared__ uint16_t s_pow[S];
  __shared__ int s_end[256], s_scan[4];
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  int next = blockIdx.x, before = 0;
  for (int r0 = 0; r0 < p.R; r0 += 256) {
    int sum = 0;
    bool whole = false;
    if (r0 + tid < p.R) {
      const Request rq = request(p, r0 + tid);
      whole = !rq.beyond && rq.L * (int)p.G.d > p.laid_cols;
      if (whole) {
        const int n = walk(p, rq.n - rq.L, rq.n - 1, S).count();
        sum = n > p.room / p.Hkv ? p.room + 1 : n * (int)p.Hkv.d;
      }
    }
    const int own = sum;
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) {
      const int y = __shfl_up(sum, d);
      if (lane >= d) sum += y;
    }
    if (lane == 63) s_scan[wave] = sum;
    __syncthreads();
#pragma unroll
    for (int i = 0; i < 4; i++)
      if (i < wave) sum += s_scan[i];
    s_end[tid] = before + sum;
    if (p.laid_at && blockIdx.x == 0 && r0 + tid < p.R)
      p.laid_at[r0 + tid] = whole && before + sum <= p.room ? before + sum - own : -1;
    __syncthreads();
    const int end = s_end[255];
    for (; next < end; next += gridDim.x) {
      int a = 0;  // requests whose steps all come before
#pragma unroll
      for (int d = 128; d; d >>= 1)
        if (s_end[a + d - 1] <= next) a += d;
      if (s_end[a] > p.room) break;
      const int r = r0 + a, start = a ? s_end[a - 1] : before, at = next - start;
      const int i = at / p.Hkv, kvh = at - i * (int)p.Hkv.d;
      const Request rq = request(p, r);
      const int32_t lo = rq.n - rq.L, hi = rq.n - 1;
      const Walk w = walk(p, lo, hi, S);
      const int unit = w.unit(i);
      const int to_step = p.laid_at ? start + kvh * w.count() + i : (r * (int)p.Hkv.d + kvh) * p.units + unit;
      char* to = p.laid + (int64_t)to_step * (G8::IU * 16);
      if (wave == 0) {
        const int32_t key = unit * S + lane;
        const int32_t id = any_seen(p, lo, hi, key, 1) ? page_of(p, r, entry_of(p, r, key), key) : -1;
        const int32_t row = row_of(p, key);
        s_row[0][lane] = row_at(static_cast<const char*>(p.k) + kvh * p.kh, id, p.k8b, row, p.k8n);
        s_row[1][lane] = row_at(static_cast<const char*>(p.v) + kvh * p.vh, id, p.v8b, row, p.v8n);
        const float ks = ld_scale(row_at(reinterpret_cast<const char*>(p.ks + kvh * p.ksh), id, p.ksb, row, p.ksn));
        const float vs = ld_scale(row_at(reinterpret_cast<const char*>(p.vs + kvh * p.vsh), id, p.vsb, row, p.vsn));
        float c, left;
        uint16_t power = 0;
        const uint64_t bad = __builtin_amdgcn_ballot_w64(G8::factors(p, ks, vs, c, left, power));
        const uint64_t mapped = __builtin_amdgcn_ballot_w64(id >= 0);
        s_pow[lane] = power;
        float* f = reinterpret_cast<float*>(to + (G8::KU + G8::VU) * 16);
        f[lane] = c;
        f[S + lane] = left;
        if (lane == 0) *reinterpret_cast<ulonglong2*>(f + 2 * S) = make_ulonglong2(mapped, bad);
      }
      __syncthreads();
#pragma unroll
      for (int j = 0; j < G8::KU / 256; j++) {
        const uint32_t n = j * 256 + tid, row = n / G8::TCH, c = (n % G8::TCH) ^ G8::template swz<G8::TCH>(row);
        const uint2 w = ld8(s_row[0][row] + c * 8);
        reinterpret_cast<uint4*>(to)[n] = codes8<T>(w.x, w.y);
      }
#pragma unroll
      for (int j = 0; j < G8::VU / 256; j++) {
        const uint32_t n = j * 256 + tid, row = n / G8::TVCH, c = (n % G8::TVCH) ^ G8::tswz(row);
        const uint2 w = ld8(s_row[1][row] + c * 8);
        uint4 y = codes8<T>(w.x, w.y);
        if constexpr (G8::kPower) {
          const uint32_t f = s_pow[row] * 0x10001u;
          y = times(y, make_uint4(f, f, f, f));
        }
        reinterpret_cast<uint4*>(to)[G8::KU + n] = y;
      }
      __syncthreads();
    }
    before = end <= p.room ? end : p.room + 1;
    __syncthreads();
  }
}

// Whole route: NW waves of 16 CT columns each walk the steps that some column of
// the workgroup sees. LAID: these lie in memory as they are wanted in LDS, and go there
// past the registers, two steps ahead where three fit. Else each step's codes go from
// device memory to registers a step before they become bf16 or f16 in LDS, each by one
// lane of the workgroup, and from there to all waves' products; LW waves more do
// nothing but that (LW = 0: the NW waves themselves).
//
// What bounds it (laid out, 256 columns, 128 dims, 4096 tokens over 8192 rows): a
// step's 2.4 us are 6000 cycles, of which each SIMD's two waves have products in 35 %
// and issue vector instructions in 47 %, the LDS is busy in 25 %; what is left is waits.
// Operands read further ahead, or half of the waves half a step behind the others,
// changed nothing; 16 waves of 16 columns, four a SIMD, took 531 us for 485.
template <typename T, int D, int V, int NW, int LW, int CT, bool LAID>
__global__ void __launch_bounds__(64 * (NW + LW), (Geo8<T, D, V>::kTwoWaves || NW == 8 ? 2 : 1)) whole8_kernel(Args p) {
  using G8 = Geo8<T, D, V>;
  constexpr int S = G8::kStep, RT = G8::RT, NU = RT / 2, DT = G8::DT, WC = 16 * CT, COLS = WC * NW;  // columns of a wave, of all
  constexpr int kFar = CT == 2 ? G8::kFarQuery : 0;
  constexpr bool kEasy = CT == 1 && D + V <= 384 && D % 64 == 0 && V % 64 == 0;  // registers are left
  constexpr int KU = G8::KU, VU = G8::VU, IU = LAID ? G8::IU : KU + VU;
  constexpr int NLW = LW ? LW : NW, NT = 64 * NLW, NB = LAID ? G8::kDeep : 2;  // waves and threads that load
  constexpr int KN = (S * G8::CH + NT - 1) / NT, VN = (S * G8::VCH + NT - 1) / NT;  // loads per thread
  __shared__ __attribute__((aligned(512))) uint4 s_kv[NB * IU];
  constexpr int RING = LAID ? 1 : 2 * NLW;
  __shared__ const char* s_row[RING][2][S];
  __shared__ __attribute__((aligned(16))) float s_c[RING][S], s_vs[RING][S];
  __shared__ uint16_t s_pow[RING][G8::kPower ? S : 1];
  __shared__ uint64_t s_map[2 * RING], s_bad[RING];
  __shared__ uint4 s_q[kFar ? NW : 1][kFar ? kFar : 1][kFar ? 64 : 1];
  __shared__ int s_scan[NW + LW + 3];
  __shared__ float s_ml[CT][2][64 * NW];  // each lane's own M and L

  if ((int)blockIdx.x < p.fill_blocks) {
    fill<T, V>(p, blockIdx.x);
    return;
  }
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int col = lane & 15;

  // Workgroup -> kv head, request, column tile; a request's last tiles first.
  const int x = blockIdx.x - p.fill_blocks;
  int tile = x / p.Hkv, r = -1;
  const int kvh = x - tile * (int)p.Hkv.d;
  int before = 0;
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
    r = s_scan[NW + LW];
    if (r >= 0) break;
    before += all;
    __syncthreads();
  }
  if (r < 0) return;
  tile = s_scan[NW + LW + 1];
  r = __builtin_amdgcn_readfirstlane(r);
  tile = __builtin_amdgcn_readfirstlane(tile);
  // (With rows laid out as far as there is room: the others' by a launch of their own.)
  if (p.laid_at && (p.laid_at[r] >= 0) != LAID) return;
  const Request rq = request(p, r);
  const int ncol = rq.L * (int)p.G.d;
  const int c0 = tile * COLS, cw = c0 + WC * wave;
  const int clast = (c0 + COLS < ncol ? c0 + COLS : ncol) - 1;
  const int32_t p0 = rq.n - rq.L;
  const int32_t lo = p0 + c0 / p.G, hi = p0 + clast / p.G;
  // The wave's own columns; a wave without one only loads.
  const int wlast = cw + WC - 1 < ncol ? cw + WC - 1 : ncol - 1;
  const int32_t wlo = cw < ncol ? p0 + cw / p.G : INT32_MAX / 2, whi = cw < ncol ? p0 + wlast / p.G : -1;

  const bool loads = LW == 0 || wave >= NW;
  const int lw = LW ? wave - NW : wave;  // which of the loading waves

  uint4 q[CT][G8::NQ];
#pragma unroll
  for (int k = 0; k < CT; k++) {
    const int cc = cw + 16 * k + col, cq = cc < ncol ? cc : 0, tok = cq / p.G;
    G8::load_query(query_at<T>(p, r, rq, tok, kvh * (int)p.G.d + (cq - tok * (int)p.G.d)), lane >> 4, q[k]);
    G8::sign_query(p, q[k]);
    if (k == 1 && wave < NW)
#pragma unroll
      for (int n = 0; n < kFar; n++) s_q[wave][n][lane] = q[k][n];
  }

  const Walk w = walk(p, lo, hi, S);
  const int steps = w.count();

  // A step's way into LDS: its rows' addresses from the table's entries, 2 NLW steps
  // before it is computed, and their scales NLW before, both by the loading wave
  // whose turn it is; then by all, its codes into registers two steps before, and in
  // the type into LDS one before.
  int32_t entry = 0;
  float ks = 0.f, vs = 0.f;
  auto entry_for = [&](int j) __attribute__((always_inline)) -> int32_t {
    return entry_of(args_again(), r, w.unit(j) * S + opaque(lane));
  };
  auto put_rows = [&](int j) __attribute__((always_inline)) {  // takes `entry`, leaves ks and vs
    // (The arguments again: kept, they would take more scalar registers than
    // there are, and what those overflow into, vector registers that there are not.)
    const Args& a = args_again();
    const int ln = opaque(lane);
    const int32_t key = w.unit(j) * S + ln;
    const int32_t id = j < steps && any_seen(a, lo, hi, key, 1) ? page_of(a, r, entry, key) : -1;
    const int32_t row = row_of(a, key);
    s_row[j % RING][0][ln] = row_at(static_cast<const char*>(a.k) + kvh * a.kh, id, a.k8b, row, a.k8n);
    s_row[j % RING][1][ln] = row_at(static_cast<const char*>(a.v) + kvh * a.vh, id, a.v8b, row, a.v8n);
    ks = ld_scale(row_at(reinterpret_cast<const char*>(a.ks + kvh * a.ksh), id, a.ksb, row, a.ksn));
    vs = ld_scale(row_at(reinterpret_cast<const char*>(a.vs + kvh * a.vsh), id, a.vsb, row, a.vsn));
    s_map[j % (2 * RING)] = __builtin_amdgcn_ballot_w64(id >= 0);
  };
  auto put_scales = [&](int j) __attribute__((always_inline)) {
    const int ln = opaque(lane);
    float c, left;
    uint16_t power = 0;
    const uint64_t bad = __builtin_amdgcn_ballot_w64(G8::factors(args_again(), ks, vs, c, left, power));
    s_c[j % RING][ln] = c;
    s_vs[j % RING][ln] = left;
    if constexpr (G8::kPower) s_pow[j % RING][ln] = power;
    s_bad[j % RING] = bad;
  };
  // (Between steps j - 1 and j: everyone is done with the rows of step j + 1 and the
  // scales of step j - 1, whose places these take.)
  auto prepare = [&](int j) __attribute__((always_inline)) {
    if (j % NLW != lw) return;
    put_scales(j + NLW);
    put_rows(j + 2 * NLW);
    entry = entry_for(j + 3 * NLW);
  };
  uint4 xk[KN], xv[VN];
  auto load_codes = [&](uint4* to, const char* const* rows, auto chunks) __attribute__((always_inline)) {
    constexpr int C = decltype(chunks)::value, U = S * C, N = (U + NT - 1) / NT;
    const int td = opaque(64 * lw + lane);
#pragma unroll
    for (int i = 0; i < N; i++) {
      const typename G8::template Unit<C, NT> u(i, td);
      if (U % NT == 0 || i * NT + td < U) to[i] = ld16(rows[u.row] + u.chunk * 16);
    }
  };
  auto load_step = [&](int j) __attribute__((always_inline)) {
    load_codes(xk, s_row[j % RING][0], std::integral_constant<int, G8::CH>());
    load_codes(xv, s_row[j % RING][1], std::integral_constant<int, G8::VCH>());
  };
  auto put_step = [&](int j) __attribute__((always_inline)) {
    uint4 *kd = s_kv + (j & 1) * (KU + VU), *vd = kd + KU;
    const int td = opaque(64 * lw + lane);
#pragma unroll
    for (int i = 0; i < KN; i++) {
      const typename G8::template Unit<G8::CH, NT> u(i, td);
      const uint32_t row = u.row, c = 2 * u.chunk;
      if (S * G8::CH % NT == 0 || i * NT + td < S * G8::CH) {
        st16(kd + row * G8::TCH + (c ^ G8::template swz<G8::TCH>(row)), codes8<T>(xk[i].x, xk[i].y));
        st16(kd + row * G8::TCH + ((c + 1) ^ G8::template swz<G8::TCH>(row)), codes8<T>(xk[i].z, xk[i].w));
      }
    }
#pragma unroll
    for (int i = 0; i < VN; i++) {
      const typename G8::template Unit<G8::VCH, NT> u(i, td);
      const uint32_t row = u.row, c = 2 * u.chunk;
      if (S * G8::VCH % NT == 0 || i * NT + td < S * G8::VCH) {
        uint4 a = codes8<T>(xv[i].x, xv[i].y), b = codes8<T>(xv[i].z, xv[i].w);
        if constexpr (G8::kPower) {
          const uint32_t f = s_pow[j % RING][row] * 0x10001u;
          a = times(a, make_uint4(f, f, f, f)), b = times(b, make_uint4(f, f, f, f));
        }
        st16(vd + row * G8::TVCH + (c ^ G8::tswz(row)), a);
        st16(vd + row * G8::TVCH + ((c + 1) ^ G8::tswz(row)), b);
      }
    }
  };

  float m[CT], l[CT];
  bool fresh = true;  // the segment has no step yet
  f32x4 O[DT][CT], o[DT][CT];
#pragma unroll
  for (int k = 0; k < CT; k++) {
    m[k] = kNone, l[k] = 0.f;
#pragma unroll
    for (int dt = 0; dt < DT; dt++) O[dt][k] = o[dt][k] = f32x4{};
    if (wave < NW) {
      s_ml[k][0][tid] = kNone;
      s_ml[k][1][tid] = 0.f;
    }
  }

  // LAID: a step's way into LDS, NB - 1 steps ahead.
  constexpr int MU = KU + VU + 2 * G8::FU + 1, NL = (MU + NT - 1) / NT;  // units that are wanted
  const char* laid = nullptr;
  Walk place = w;
  if constexpr (LAID) {
    int start = (r * (int)p.Hkv.d + kvh) * p.units;
    if (p.laid_at) {  // (only what the request walks has a place)
      const Walk all = walk(p, p0, rq.n - 1, S);
      start = p.laid_at[r] + kvh * all.count();
      place.b -= all.b - all.a;
    }
    laid = p.laid + (int64_t)start * (IU * 16);
  }
  auto fetch = [&](int j) __attribute__((always_inline)) {
    const char* from = laid + (uint64_t)(uint32_t)place.unit(j) * (IU * 16);
    uint4* to = s_kv + j % NB * IU + 64 * wave;
#pragma unroll
    for (int i = 0; i < NL; i++)
      if (i * NT + NT <= MU || i * NT + tid < MU)
        load_to_lds<16>(from + (i * NT + opaque(tid)) * 16, to + i * NT);
  };

  if constexpr (LAID) {
#pragma unroll
    for (int j = 0; j < NB - 1; j++)
      if (j < steps) fetch(j);
  } else {
    if (loads) {
      entry = entry_for(lw);
      put_rows(lw);
      put_scales(lw);
      entry = entry_for(lw + NLW);
      put_rows(lw + NLW);
      entry = entry_for(lw + 2 * NLW);
    }
    __syncthreads();
    if (loads) {
      load_step(0);
      put_step(0);
      load_step(1);
    }
    if constexpr (LW != 0)
      if (loads) {
        for (int j = 0; j < steps; j++) {
          barrier();
          if (j + 1 < steps) put_step(j + 1);
          prepare(j);  // (before the loads that the next step waits for, and with them for its own)
          if (j + 2 < steps) load_step(j + 2);
        }
        return;
      }
  }
  // (Where the loop's instructions lie within the 32 bytes that are fetched at a time: the
  // same ones take, 128 dims, by the place of the step's barrier 221 to 230 us laid out in
  // 128 columns, for 512 tokens over 8192 rows, in 256 463 to 475, for 4096, and not laid
  // out 407 to 421, for 4 requests of 512. In 256 columns instructions that do nothing
  // cost as much within the loop: there they are before it. 64 and 256 dims gain nothing.)
  constexpr bool kPlaced = D == 128 && V == 128;
  if constexpr (kPlaced && LAID && CT == 2) asm volatile(".p2align 5\n\t.fill 2, 4, 0xbf800000");
  for (int j = 0; j < steps; j++) {
    const uint32_t ln = opaque(lane);
    const int g = ln >> 4;
    if constexpr (LAID) {  // (the loads of the NB - 2 steps after it may be on their way still)
      if (j + NB - 2 < steps) wait_loads_but<(MU / NT) * (NB - 2)>();
      else wait_loads();
    }
    // Step j is there, and everyone is done with step j - 1's buffer.
    if constexpr (kPlaced && !(LAID && CT == 2)) barrier_at<LAID ? 0 : 3>();
    else barrier();
    if constexpr (LAID) {
      if (j + NB - 1 < steps) fetch(j + NB - 1);
    } else if constexpr (LW == 0) {
      if (j + 1 < steps) put_step(j + 1);
      prepare(j);
    }
    const uint4 *kd = s_kv + j % NB * IU, *vd = kd + KU;
    const float *cs = s_c[j % RING], *gs = s_vs[j % RING];
    const uint64_t *maps = &s_map[j % (2 * RING)], *bads = &s_bad[j % RING];
    if constexpr (LAID) {
      cs = reinterpret_cast<const float*>(vd + VU), gs = cs + S;
      maps = reinterpret_cast<const uint64_t*>(gs + S), bads = maps + 1;
    }
    const int32_t unit = w.unit(j), key0 = unit * S;
    const bool mine = any_seen(p, wlo, whi, key0, S);
    uint4 pu[NU][CT];
    if (mine) {
      const uint64_t mapped = uniform(*maps);
      const bool full = mapped == ~0ull && all_seen(p, wlo, whi, key0, S);
      f32x4 s[RT][CT];
#pragma unroll
      for (int t = 0; t < RT; t++)
#pragma unroll
        for (int k = 0; k < CT; k++) s[t][k] = f32x4{};
      uint4 far[2];
      auto far_query = [&](int n) __attribute__((always_inline)) { far[n & 1] = s_q[wave][n][ln]; };
      if (kFar) far_query(0);
      const auto keys = G8::keys_of_type(kd, ln);
      feed_ahead<RT * G8::NQ, kEasy ? 8 : 2>(
          [&](int n) __attribute__((always_inline)) { return G8::key_of_type(keys, 16 * (n % RT), n / RT, ln); },
          [&](int n, uint4 x) __attribute__((always_inline)) {
            const int i = n / RT;
            if (n % RT == 0 && i + 1 < kFar) far_query(i + 1);
#pragma unroll
            for (int k = 0; k < CT; k++) s[n % RT][k] = G8::product(x, k == 1 && i < kFar ? far[i & 1] : q[k][i], s[n % RT][k]);
          });
      const uint64_t bad = uniform(*bads) & mapped;
      auto positions = [&](int32_t(&pos)[CT]) __attribute__((always_inline)) {
#pragma unroll
        for (int k = 0; k < CT; k++) {
          const int c = cw + 16 * k + (opaque(lane) & 15);
          pos[k] = c < ncol ? p0 + c / p.G : -1;
        }
      };
      if (!full) {
        int32_t pos[CT];
        uint64_t seen[CT];
        positions(pos);
#pragma unroll
        for (int k = 0; k < CT; k++) seen[k] = seen_bits(p, pos[k], key0, mapped) >> (4 * g);
        G8::template hide<CT>(s, seen);
      }
      // A lane's sum of at most kMostSum holds no score that moves the base;
      // else, and at a segment's first step, the largest score decides.
      float psum[CT];
      bool look = fresh;
      for (;;) {
        const int h = opaque(g);  // (so that no row's factor is read before the loop, into registers)
        if (look) {
          float t[CT];
          G8::template top<CT>(s, cs, h, t);
#pragma unroll
          for (int k = 0; k < CT; k++) {
            const float mn = next_base(m[k], t[k], 1.f);
            if (!fresh && __builtin_amdgcn_ballot_w64(mn != m[k]) != 0) {
              const float f = pow2(m[k] - mn);
              l[k] *= f;  // exact, as in the sum's fma(l, f, .)
#pragma unroll
              for (int dt = 0; dt < DT; dt++)
#pragma unroll
                for (int i = 0; i < 4; i++) o[dt][k][i] *= f;
            }
            m[k] = mn;
          }
        }
        G8::template weights<CT, kEasy>(s, cs, gs, h, m, pu, psum);
        bool more = false;
#pragma unroll
        for (int k = 0; k < CT; k++) more |= psum[k] > kMostSum;
        if (look || __builtin_amdgcn_ballot_w64(more) == 0) break;
        look = true;
      }
      if (bad) {
        int32_t pos[CT];
        positions(pos);
        G8::template spoil<CT>(p, pos, key0, bad, psum);
      }
#pragma unroll
      for (int k = 0; k < CT; k++) l[k] += psum[k];
      fresh = false;
    }
    // (Not before the scores, whose operands need the registers.)
    if constexpr (LW == 0 && !LAID)
      if (j + 2 < steps) load_step(j + 2);
    if (mine) {
      // Products of one output tile are a chain: those of the others go between.
      const auto values = G8::values_of_type(vd, ln);
      feed_ahead<DT * NU, kEasy ? 8 : 4>(
          [&](int n) __attribute__((always_inline)) { return G8::value_of_type(values, n / DT, n % DT); },
          [&](int n, uint4 v) __attribute__((always_inline)) {
#pragma unroll
            for (int k = 0; k < CT; k++) o[n % DT][k] = G8::product(v, pu[n / DT][k], o[n % DT][k]);
          });
    }
    // The segment's end: fold it.
    if (j + 1 == steps || w.unit(j + 1) / G8::kSegSteps != unit / G8::kSegSteps) {
      if (!fresh) {
        const int td = opaque(tid);
#pragma unroll
        for (int k = 0; k < CT; k++) {
          float M = s_ml[k][0][td], L = s_ml[k][1][td], fa, fb;
          fold_base(M, L, m[k], within<T>(m[k], quarters_sum(l[k])), fa, fb);
          s_ml[k][0][td] = M;
          s_ml[k][1][td] = L;
          if (__builtin_amdgcn_ballot_w64(fa != 1.f) != 0)
#pragma unroll
            for (int dt = 0; dt < DT; dt++)
#pragma unroll
              for (int i = 0; i < 4; i++) O[dt][k][i] *= fa;
#pragma unroll
          for (int dt = 0; dt < DT; dt++) {
#pragma unroll
            for (int i = 0; i < 4; i++) O[dt][k][i] = __builtin_fmaf(o[dt][k][i], fb, O[dt][k][i]);
            o[dt][k] = f32x4{};
          }
          m[k] = kNone;
          l[k] = 0.f;
        }
        fresh = true;
      }
    }
  }

#pragma unroll
  for (int k = 0; k < CT; k++) {
    const int lane2 = opaque(lane), cc = cw + 16 * k + (lane2 & 15);
    if (cc >= ncol) continue;
    const int tok = cc / p.G, head = kvh * (int)p.G.d + cc - tok * (int)p.G.d;
    const float M = s_ml[k][0][wave * 64 + lane2], L = s_ml[k][1][wave * 64 + lane2];
    float e, den;
    finish(M, L, p.sinks ? (float)static_cast<const T*>(p.sinks)[head] * 1.4426950408889634f : 0.f,
           p.sinks != nullptr, e, den);
    const float inv = inverse(den);
    T* out = out_at<T>(p, r, rq, tok, head);
#pragma unroll
    for (int dt = 0; dt < DT; dt++) {
      typedef T T4 __attribute__((ext_vector_type(4)));
      T4 y;
#pragma unroll
      for (int i = 0; i < 4; i++) y[i] = result<T>(O[dt][k][i], e, inv);
      *reinterpret_cast<T4*>(out + 16 * dt + 4 * (lane2 >> 4)) = y;
    }
  }
}

template <typename T, int D, int V>
Kernels kernels8_of() {
  using G8 = Geo8<T, D, V>;
  Kernels k;
  k.split16 = k.split16_one = split8_kernel<T, D, V, 16>;
  k.split32 = k.split32_one = split8_kernel<T, D, V, 32>;
  k.combine = combine_kernel<T, D, V, G8::kSeg>;
  k.seg = G8::kSeg, k.pass = 4 * G8::kStep;
  k.row_us = G8::row_us();
  k.seg16_us = G8::seg_us(16), k.seg32_us = G8::seg_us(32);
  k.laid_row_us = G8::laid_row_us(), k.laid_tile_us = G8::laid_tile_us();
  k.per_cu16 = G8::split_per_cu(16), k.per_cu32 = G8::split_per_cu(32);
  k.whole4_pair = nullptr;
  if constexpr (G8::kTwoWaves) {
    k.whole4 = whole8_kernel<T, D, V, 4, 4, 2, false>;
    k.laid8 = whole8_kernel<T, D, V, 8, 0, 2, true>;
  } else {
    k.whole4 = whole8_kernel<T, D, V, 4, 0, 2, false>;
  }
  k.laid4 = whole8_kernel<T, D, V, 8, 0, 1, true>;
  k.lay = lay8_kernel<T, D, V>;
  k.step = G8::kStep, k.step_bytes = G8::IU * 16;
  k.whole8 = nullptr;
  k.whole4_threads = G8::kTwoWaves ? 512 : 256;
  // (64 requests of 1000 to 8056 rows of a token-major cache 154 us, with 1024 to 8192
  // places 160 to 163; 250 rows under a bound of 65536 36, with 8192 43.)
  k.places = 2048;
  return k;
}

}  // namespace
}  // namespace bi_paged

#define BI_PAGED_Q8_KERNELS(D, V)                                 \
  bi_paged::Kernels bi_paged::kernels8_d##D##_v##V(int dtype) {   \
    return dtype == BI_F16 ? kernels8_of<_Float16, D, V>()        \
                           : kernels8_of<__bf16, D, V>();         \
  }
