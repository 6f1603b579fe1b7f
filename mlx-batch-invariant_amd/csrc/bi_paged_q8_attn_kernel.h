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
//     chain of 32x32x16 products of codes and the query over the head dim. The
//     lane half h takes the codes of 16-byte chunk 2 c + h in products 2 c and 2
//     c + 1, eight each.
//   * c_j is rounded once to 32 bits; p_j = 2^(fma(raw_j, c_j, -m)); l sums the p
//     of 32 bits, in a fixed order per lane half.
//   * bf16: the weights p_j * vs_j are rounded to bf16, whose range holds any
//     scale: half a step of 2^-8 of a weight whose value's code is off by as much
//     as 2^-8 of the largest. f16: the scale's power of two 2^e, kept to 2^-14 ..
//     2^9, goes with the codes, which stay exact (127 * 2^9 is below f16's
//     largest, 2^-14 its smallest normal number), and the weights p_j * (vs_j /
//     2^e), of p's own size for scales in that range, are rounded to f16. (Scales
//     past 2^19, of values past 6e7, overflow them.)
// A row that a column does not see has p and weight 0 by selection, whatever its
// codes and scales, and codes are finite: so no row's content reaches a token that
// does not see it, and there is no case of values to look for. A negative scale
// of keys gives NaN.
#pragma once

#include "bi_paged_attn_kernel.h"

namespace bi_paged {
namespace {

typedef int i32x2 __attribute__((ext_vector_type(2)));
typedef __attribute__((address_space(3))) i32x2 lds_i32x2;

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

template <typename T, int D_, int V_>
struct Geo8 {
  static constexpr int D = D_, V = V_;
  using G = Geo<T, D, V>;
  static constexpr int kStep = 64, KT = 2, kSegSteps = 8, kSeg = kSegSteps * kStep;
  static constexpr int CH = D / 16, VCH = V / 16;  // 16-byte chunks of a row of codes
  static constexpr int MCH = CH > VCH ? CH : VCH;
  static constexpr int NQ = D / 16;                // products of a score
  static constexpr int DT = V / 32;
  static constexpr int PU = 2;                     // units of eight weights per tile and lane
  static constexpr bool kPower = __is_same(T, _Float16);  // values' codes carry 2^e
  static constexpr bool kTwoWaves = V + D / 4 <= 160;
  static constexpr int split_per_cu() { return D + V <= 256 ? 2 : 1; }

  static constexpr double row_us() { return 1e-3 * (kTwoWaves ? 13.0 + 0.04 * (D + V) : 28.0 + 0.08 * (D + V)); }
  static constexpr double seg_us() { return 5.0 + 0.023 * (kSeg * (D + V) / 1024.0); }

  // Codes of keys in LDS (split route): row r's chunk c at chunk c ^ kswz(r). A
  // read takes one chunk of 16 rows per pass; the exchange spreads them over all
  // banks.
  __device__ __forceinline__ static int kswz(int r) {
    if constexpr (CH % 16 == 0) return r & 15;
    else if constexpr (CH % 8 == 0) return (r >> 1) & 7;
    else if constexpr (CH % 4 == 0) return (r >> 2) & 3;
    else return (r >> 3) & 1;
  }
  // Codes of values: row r at place vplace(r), which puts the eight rows of a
  // product's lane half side by side, its chunk c at chunk c ^ vswz(place): 32
  // lanes read 32 bytes of eight rows per pass.
  __device__ __forceinline__ static int vplace(int r) {
    return (r & ~12) | ((r >> 1) & 4) | ((r << 1) & 8);
  }
  __device__ __forceinline__ static int vswz(int at) {
    if constexpr (VCH == 16) return (at & 7) << 1;
    else if constexpr (VCH == 8) return ((at >> 1) & 3) << 1;
    else if constexpr (VCH == 12 || VCH == 4) return ((at >> 2) & 1) << 1;
    else return 0;
  }
  // The values' operand of product u of the tile at row0, output dims 32 dt ..;
  // `power`: 2^e by place.
  __device__ __forceinline__ static uint4 value(const uint4* v, const uint16_t* power, int row0, int u, int dt,
                                                int lane) {
    const int i = lane & 15, at = row0 + 16 * u + 8 * (lane >> 5) + (i >> 1);
    const int c = 2 * dt + ((lane >> 4) & 1);
    const char* from = reinterpret_cast<const char*>(v + at * VCH + (c ^ vswz(at))) + 8 * (i & 1);
    const i32x2 x = __builtin_amdgcn_ds_read_tr8_b64_v2i32((lds_i32x2*)from);
    const uint4 y = codes8<T>((uint32_t)x[0], (uint32_t)x[1]);
    if constexpr (!kPower) return y;
    else return times(y, *reinterpret_cast<const uint4*>(power + row0 + 16 * u + 8 * (lane >> 5)));
  }
  // A column's query: chunk 4 c + 2 half + j for product 2 c + j.
  __device__ __forceinline__ static void load_query(const char* q, int half, uint4 (&out)[NQ]) {
#pragma unroll
    for (int n = 0; n < NQ; n++) out[n] = ld16(q + (4 * (n >> 1) + 2 * half + (n & 1)) * 16);
  }
  __device__ __forceinline__ static void sign_query(const Args& p, uint4 (&q)[NQ]) {
#pragma unroll
    for (int n = 0; n < NQ; n++)
      q[n] = make_uint4(q[n].x ^ p.qsign, q[n].y ^ p.qsign, q[n].z ^ p.qsign, q[n].w ^ p.qsign);
  }

  // c_j from a row's scale: above 0, so that an unseen row's -inf stays one.
  __device__ __forceinline__ static float factor(const Args& p, float ks) {
    return ks >= 0.f ? fmaxf(ks * p.scale2, 1.2e-38f) : NAN;
  }
  // The rows' numbers of a tile's elements 4 b .. 4 b + 3 from LDS.
  __device__ __forceinline__ static f32x4 rows4(const float* at, int kt, int b, int half) {
    return *reinterpret_cast<const f32x4*>(at + 32 * kt + 8 * b + 4 * half);
  }
  // The largest score; `seen` (shifted by the half's four rows) says which count.
  template <bool FULL>
  __device__ __forceinline__ static float top(const f32x16 (&s)[KT], const float* c, int half, uint64_t seen) {
    float m = -INFINITY;
#pragma unroll
    for (int kt = 0; kt < KT; kt++) {
      const uint32_t w = (uint32_t)(seen >> (32 * kt));
#pragma unroll
      for (int b = 0; b < 4; b++) {
        const f32x4 f = rows4(c, kt, b, half);
#pragma unroll
        for (int i = 0; i < 4; i++) {
          float x = s[kt][4 * b + i] * f[i];
          if (!FULL) x = w & (1u << (8 * b + i)) ? x : -INFINITY;
          m = __builtin_elementwise_maximum(m, x);
        }
      }
    }
    return half_swap_max(m);
  }
  // A step's weights in the type, and the lane's sum of p: a chain for eight
  // rows, then these in pairs. (Eight rows at a time: else the compiler reads
  // all factors first, into registers that there are not.)
  template <bool FULL>
  __device__ __forceinline__ static float weights(const f32x16 (&s)[KT], const float* c, const float* vs,
                                                  int half, uint64_t seen, float m, uint4 (&u)[KT][PU]) {
    float sum[KT * PU];
#pragma unroll
    for (int kt = 0; kt < KT; kt++) {
      const uint32_t w = (uint32_t)(seen >> (32 * kt));
#pragma unroll
      for (int j = 0; j < PU; j++) {
        float l = 0.f;
        uint32_t d[4];
#pragma unroll
        for (int b = 0; b < 2; b++) {
          const f32x4 f = rows4(c, kt, 2 * j + b, half), g = rows4(vs, kt, 2 * j + b, half);
          f32x4 z;
#pragma unroll
          for (int i = 0; i < 4; i++) {
            float e = __builtin_amdgcn_exp2f(__builtin_fmaf(s[kt][8 * j + 4 * b + i], f[i], -m));
            if (!FULL) e = w & (1u << (16 * j + 8 * b + i)) ? e : 0.f;
            l = b == 0 && i == 0 ? e : l + e;
            z[i] = e * g[i];
            if (!FULL) z[i] = w & (1u << (16 * j + 8 * b + i)) ? z[i] : 0.f;
          }
#pragma unroll
          for (int i = 0; i < 2; i++) {
            const f32x2 two = {z[2 * i], z[2 * i + 1]};
            if constexpr (kPower) d[2 * b + i] = __builtin_bit_cast(uint32_t, __builtin_convertvector(two, f16x2));
            else d[2 * b + i] = __builtin_bit_cast(uint32_t, __builtin_convertvector(two, bf16x2));
          }
        }
        sum[kt * PU + j] = l;
        u[kt][j] = make_uint4(d[0], d[1], d[2], d[3]);
        __builtin_amdgcn_sched_barrier(0);
      }
    }
    return (sum[0] + sum[1]) + (sum[2] + sum[3]);
  }
};

// A row's scale, 0 for one without a page; from device memory, as ld16.
__device__ __forceinline__ float ld_scale(const float* at, bool there) {
  typedef __attribute__((address_space(1))) const float gfloat;
  return *(gfloat*)(there ? at : reinterpret_cast<const float*>(g_zero_row));
}

// Split route: a segment's (m, l, o) of NC columns, four steps to a pass, one
// per wave, as for the other types. Keys and values of the next pass are on their
// way through registers of their own while a pass is computed.
template <typename T, int D, int V, int NC>
__global__ void __launch_bounds__(256, (Geo8<T, D, V>::split_per_cu())) split8_kernel(Args p) {
  using G8 = Geo8<T, D, V>;
  using G = typename G8::G;
  constexpr int S = G8::kStep, KT = G8::KT, PU = G8::PU;
  __shared__ uint4 s_kv[4 * S * G8::MCH];  // a step per wave: its keys, then its values
  __shared__ uint4 s_p[4 * KT * PU * 2 * NC];
  __shared__ const char* s_row[2][4 * S];
  __shared__ __attribute__((aligned(16))) float s_c[4 * S], s_vs[4 * S];
  __shared__ __attribute__((aligned(16))) uint16_t s_pow[G8::kPower ? 4 * S : 8];
  __shared__ float s_max[4][NC];
  __shared__ float s_sum[4][2 * NC];

  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int col = lane & 31, half = lane >> 5, cn = col & (NC - 1);
  // Workgroup -> kv head, columns, segment of the walk, request.
  const int x = blockIdx.x, xc = x / p.Hkv, kvh = x - xc * (int)p.Hkv.d;
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

  // Column; one without a token takes the first one's query and sees nothing.
  const int cc = c0 + col;
  const bool cv = col < NC && cc < ncol;
  const int cq = cv ? cc : c0;
  const int tok = cq / p.G, head = kvh * (int)p.G.d + (cq - tok * (int)p.G.d);
  const int32_t pos = cv ? rq.n - rq.L + tok : -1;
  const char* kh = static_cast<const char*>(p.k) + kvh * p.kh;
  const char* vh = static_cast<const char*>(p.v) + kvh * p.vh;
  const float* ksh = p.ks + kvh * p.ksh;
  const float* vsh = p.vs + kvh * p.vsh;

  int s0, s1;
  // Row addresses of the wave's step of a segment, and its scales, on their way; a
  // row that no column sees, or that has no page, is a row of zeros.
  float ks, vs;
  auto key_of = [&](int si) __attribute__((always_inline)) { return si * PS + wave * S; };
  auto entry_for = [&](int si) __attribute__((always_inline)) -> int32_t {
    return entry_of(p, r, key_of(si) + lane);
  };
  auto put_rows = [&](int si, int32_t entry) __attribute__((always_inline)) -> uint64_t {
    const int32_t key = key_of(si) + lane;
    const int32_t id = si < s1 && any_seen(p, lo, hi, key, 1) ? page_of(p, r, entry, key) : -1;
    const int64_t row = row_of(p, key);
    const char* zero = reinterpret_cast<const char*>(g_zero_row);
    s_row[0][wave * S + lane] = id >= 0 ? kh + id * p.kb + row * p.kn : zero;
    s_row[1][wave * S + lane] = id >= 0 ? vh + id * p.vb + row * p.vn : zero;
    ks = ld_scale(ksh + id * p.ksb + row * p.ksn, id >= 0);
    vs = ld_scale(vsh + id * p.vsb + row * p.vsn, id >= 0);
    __builtin_amdgcn_wave_barrier();
    return __builtin_amdgcn_ballot_w64(id >= 0);
  };
  // Rows are loaded whole, consecutive lanes taking consecutive chunks.
  constexpr int KL = S * G8::CH / 64, VL = S * G8::VCH / 64;
  uint4 xk[KL], xv[VL], q[G8::NQ];
  auto load_rows = [&](uint4* to, const char* const* rows, auto chunks, auto load) __attribute__((always_inline)) {
    constexpr int C = decltype(chunks)::value;
    const int ln = opaque(lane);
#pragma unroll
    for (int j = 0; j < S * C / 64; j++) {
      const uint32_t at = j * 64 + ln, row = at / C;
      to[j] = load(rows[wave * S + row] + (at - row * C) * 16);
    }
  };
  auto load_keys = [&]() __attribute__((always_inline)) {
    if (p.once) load_rows(xk, s_row[0], std::integral_constant<int, G8::CH>(), ld16_once);
    else load_rows(xk, s_row[0], std::integral_constant<int, G8::CH>(), ld16);
  };
  auto load_values = [&]() __attribute__((always_inline)) {
    if (p.once) load_rows(xv, s_row[1], std::integral_constant<int, G8::VCH>(), ld16_once);
    else load_rows(xv, s_row[1], std::integral_constant<int, G8::VCH>(), ld16);
  };

  for (int part = part0; part < parts; part += p.gseg.d) {
    s0 = w.unit(part) * PN, s1 = s0 + PN;
    while (s0 < s1 && !any_seen(p, lo, hi, s0 * PS, PS)) s0++;
    while (s0 < s1 && !any_seen(p, lo, hi, (s1 - 1) * PS, PS)) s1--;
    if (p.window || part != part0) {
      entry0 = entry_for(s0);
      entry = entry_for(s0 + 1);
    }
    G8::load_query(query_at<T>(p, r, rq, tok, head), half, q);
    uint64_t mapped = put_rows(s0, entry0);
    load_keys();
    load_values();
    G8::sign_query(p, q);

    constexpr int TW = (G8::DT + 3) / 4;  // tiles of output dims per wave
    float m = kNone, l = 0.f;
    f32x16 o[TW];
#pragma unroll
    for (int i = 0; i < TW; i++) o[i] = f32x16{};
    for (int si = s0; si < s1; si++) {
      const int32_t pass0 = si * PS, key0 = pass0 + wave * S;
      const int32_t entry2 = entry_for(si + 2);
      const int lk = opaque(lane);
#pragma unroll
      for (int j = 0; j < KL; j++) {
        const uint32_t at = j * 64 + lk, row = at / G8::CH, c = (at - row * G8::CH) ^ G8::kswz(row);
        st16(s_kv + wave * S * G8::MCH + row * G8::CH + c, xk[j]);
      }
      s_c[wave * S + lk] = G8::factor(p, ks);
      float left = vs;
      if constexpr (G8::kPower) s_pow[wave * S + G8::vplace(lk)] = scale_power(vs, left);
      s_vs[wave * S + lk] = left;
      const uint64_t now = mapped;
      mapped = put_rows(si + 1, entry);
      entry = entry2;
      load_keys();
      __builtin_amdgcn_wave_barrier();
      // Scores of the wave's step and their largest.
      f32x16 s[KT];
#pragma unroll
      for (int kt = 0; kt < KT; kt++) {
        f32x16 c = {};
        const int row = 32 * kt + (lk & 31);
#pragma unroll
        for (int t = 0; t < G8::NQ / 2; t++) {
          const uint4 k = s_kv[wave * S * G8::MCH + row * G8::CH + ((2 * t + (lk >> 5)) ^ G8::kswz(row))];
          c = G::score(codes8<T>(k.x, k.y), q[2 * t], c);
          c = G::score(codes8<T>(k.z, k.w), q[2 * t + 1], c);
        }
        s[kt] = c;
      }
      const bool full = now == ~0ull && all_seen(p, lo, hi, key0, S) && c0 + NC <= ncol;
      const uint64_t seen = full ? 0 : seen_bits(p, pos, key0, now) >> (4 * half);
      const float* cs = s_c + wave * S;
      const float top = full ? G8::template top<true>(s, cs, half, seen) : G8::template top<false>(s, cs, half, seen);
      if (lane < NC) s_max[wave][lane] = top;
      barrier();

      // The bases of the pass's steps; this wave's weights.
      float base[4], f[4];
#pragma unroll
      for (int i = 0; i < 4; i++) {
        base[i] = next_base(m, s_max[i][cn], 1.f);
        f[i] = pow2(m - base[i]);
        m = base[i];
      }
      const float mw = wave == 0 ? base[0] : wave == 1 ? base[1] : wave == 2 ? base[2] : base[3];
      uint4 pu[KT][PU];
      const float psum = full ? G8::template weights<true>(s, cs, s_vs + wave * S, half, seen, mw, pu)
                              : G8::template weights<false>(s, cs, s_vs + wave * S, half, seen, mw, pu);
      if (col < NC) {
#pragma unroll
        for (int kt = 0; kt < KT; kt++)
#pragma unroll
          for (int j = 0; j < PU; j++) s_p[((wave * KT + kt) * PU + j) * 2 * NC + half * NC + col] = pu[kt][j];
        s_sum[wave][half * NC + col] = psum;
      }
      const int ln = opaque(lane);
#pragma unroll
      for (int j = 0; j < VL; j++) {
        const uint32_t at = j * 64 + ln, row = at / G8::VCH, place = G8::vplace(row);
        const int c = (at - row * G8::VCH) ^ G8::vswz(place);
        st16(s_kv + wave * S * G8::MCH + place * G8::VCH + c, xv[j]);
      }
      load_values();
      barrier();

      // The sum, and the wave's tiles of output dims over the pass's steps.
#pragma unroll
      for (int i = 0; i < 4; i++) l = __builtin_fmaf(l, f[i], s_sum[i][half * NC + cn]);
#pragma unroll
      for (int y = 0; y < TW; y++) {
        const int dt = wave + 4 * y;
        if (dt >= G8::DT) break;
#pragma unroll
        for (int i = 0; i < 4; i++) {
          if (!any_seen(p, lo, hi, pass0 + i * S, S)) continue;
          if (__builtin_amdgcn_ballot_w64(f[i] != 1.f) != 0)
#pragma unroll
            for (int e = 0; e < 16; e++) o[y][e] *= f[i];
#pragma unroll
          for (int kt = 0; kt < KT; kt++) {
#pragma unroll
            for (int j = 0; j < PU; j++) {
              const uint4 v = G8::value(s_kv + i * S * G8::MCH, s_pow + i * S, 32 * kt, j, dt, ln);
              const uint4 u = s_p[((i * KT + kt) * PU + j) * 2 * NC + (ln >> 5) * NC + (ln & (NC - 1))];
              o[y] = G::score(v, u, o[y]);
            }
          }
        }
      }
      barrier();  // everyone is done with the values and weights
    }

    l = half_swap_sum(l);
    if (cv) {
      const int64_t slot = (((int64_t)r * p.Hkv.d + kvh) * p.nseg.d + part) * p.ccap.d + cc;
      if (wave == 0 && half == 0) p.pml[slot] = make_float2(m, l);
#pragma unroll
      for (int y = 0; y < TW; y++) {
        if (wave + 4 * y >= G8::DT) break;
        float* to = p.po + slot * V + 32 * (wave + 4 * y);
#pragma unroll
        for (int b = 0; b < 4; b++)
          *reinterpret_cast<f32x4*>(to + 8 * b + 4 * half) =
              f32x4{o[y][4 * b], o[y][4 * b + 1], o[y][4 * b + 2], o[y][4 * b + 3]};
      }
    }
  }
}

// Whole route: NW waves of 32 columns each walk the steps that some column of
// the workgroup sees. Each step's codes go from device memory to registers a step
// before they become bf16 or f16 in LDS, each by one lane of the workgroup, and
// from there to all waves' products. LW waves more do nothing but that (LW = 0:
// the NW waves themselves).
template <typename T, int D, int V, int NW, int LW>
__global__ void __launch_bounds__(64 * (NW + LW), (Geo8<T, D, V>::kTwoWaves ? 2 : 1)) whole8_kernel(Args p) {
  using G8 = Geo8<T, D, V>;
  using G = typename G8::G;
  constexpr int S = G8::kStep, KT = G8::KT, PU = G8::PU, DT = G8::DT, COLS = 32 * NW;
  constexpr int KU = S * G::CH, VU = S * G::VCH;  // 16-byte units of a step in LDS
  constexpr int NT = 64 * (LW ? LW : NW), NB = 2;  // NT: threads that load
  constexpr int KN = (S * G8::CH + NT - 1) / NT, VN = (S * G8::VCH + NT - 1) / NT;  // loads per thread
  __shared__ uint4 s_kv[NB * (KU + VU)];
  __shared__ const char* s_row[4][2][S];
  __shared__ __attribute__((aligned(16))) float s_c[4][S], s_vs[4][S];
  __shared__ uint16_t s_pow[4][G8::kPower ? S : 1];
  __shared__ uint64_t s_map[8];
  __shared__ int s_scan[NW + LW + 3];
  __shared__ float s_ml[2][64 * NW];  // each lane's own M and L

  if ((int)blockIdx.x < p.fill_blocks) {
    fill<T, V>(p, blockIdx.x);
    return;
  }
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int col = lane & 31, half = lane >> 5;

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
  uint4 q[G8::NQ];
  G8::load_query(query_at<T>(p, r, rq, tok, kvh * (int)p.G.d + (cv ? cc - tok * (int)p.G.d : 0)), half, q);
  G8::sign_query(p, q);

  const Walk w = walk(p, lo, hi, S);
  const int steps = w.count();

  // A step's way into LDS, by the first wave: its rows' addresses from the table's
  // entries three steps before it is computed, and their scales from registers two
  // before; then by all, its codes into registers two steps before, and as bf16 or
  // f16 into LDS one before.
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
    const int64_t row = row_of(a, key);
    const char* zero = reinterpret_cast<const char*>(g_zero_row);
    const char *k = static_cast<const char*>(a.k) + kvh * a.kh, *v = static_cast<const char*>(a.v) + kvh * a.vh;
    s_row[j & 3][0][ln] = id >= 0 ? k + id * a.kb + row * a.kn : zero;
    s_row[j & 3][1][ln] = id >= 0 ? v + id * a.vb + row * a.vn : zero;
    ks = ld_scale(a.ks + kvh * a.ksh + id * a.ksb + row * a.ksn, id >= 0);
    vs = ld_scale(a.vs + kvh * a.vsh + id * a.vsb + row * a.vsn, id >= 0);
    s_map[j & 7] = __builtin_amdgcn_ballot_w64(id >= 0);
  };
  auto put_scales = [&](int j) __attribute__((always_inline)) {
    const int ln = opaque(lane);
    s_c[j & 3][ln] = G8::factor(p, ks);
    float left = vs;
    if constexpr (G8::kPower) s_pow[j & 3][ln] = scale_power(vs, left);
    s_vs[j & 3][ln] = left;
  };
  uint4 xk[KN], xv[VN];
  auto load_codes = [&](uint4* to, const char* const* rows, auto chunks) __attribute__((always_inline)) {
    constexpr int C = decltype(chunks)::value, U = S * C, N = (U + NT - 1) / NT;
    const int td = opaque(64 * lw + lane);
#pragma unroll
    for (int i = 0; i < N; i++) {
      const uint32_t at = i * NT + td, row = at / C;
      if (U % NT == 0 || at < U) to[i] = ld16(rows[row] + (at - row * C) * 16);
    }
  };
  auto load_step = [&](int j) __attribute__((always_inline)) {
    load_codes(xk, s_row[j & 3][0], std::integral_constant<int, G8::CH>());
    load_codes(xv, s_row[j & 3][1], std::integral_constant<int, G8::VCH>());
  };
  auto put_step = [&](int j) __attribute__((always_inline)) {
    uint4 *kd = s_kv + (j & 1) * (KU + VU), *vd = kd + KU;
    const int td = opaque(64 * lw + lane);
#pragma unroll
    for (int i = 0; i < KN; i++) {
      const uint32_t at = i * NT + td, row = at / G8::CH, c = 2 * (at - row * G8::CH);
      if (S * G8::CH % NT == 0 || at < S * G8::CH) {
        st16(kd + row * G::CH + (c ^ G::kswz(row)), codes8<T>(xk[i].x, xk[i].y));
        st16(kd + row * G::CH + ((c + 1) ^ G::kswz(row)), codes8<T>(xk[i].z, xk[i].w));
      }
    }
#pragma unroll
    for (int i = 0; i < VN; i++) {
      const uint32_t at = i * NT + td, row = at / G8::VCH, c = 2 * (at - row * G8::VCH);
      if (S * G8::VCH % NT == 0 || at < S * G8::VCH) {
        uint4 a = codes8<T>(xv[i].x, xv[i].y), b = codes8<T>(xv[i].z, xv[i].w);
        if constexpr (G8::kPower) {
          const uint32_t f = s_pow[j & 3][row] * 0x10001u;
          a = times(a, make_uint4(f, f, f, f)), b = times(b, make_uint4(f, f, f, f));
        }
        st16(vd + row * G::VCH + (c ^ G::vswz(row)), a);
        st16(vd + row * G::VCH + ((c + 1) ^ G::vswz(row)), b);
      }
    }
  };

  float m = kNone, l = 0.f;
  bool fresh = true;  // the segment has no step yet
  f32x16 O[DT], o[DT];
#pragma unroll
  for (int dt = 0; dt < DT; dt++) O[dt] = f32x16{}, o[dt] = f32x16{};
  if (wave < NW) {
    s_ml[0][tid] = kNone;
    s_ml[1][tid] = 0.f;
  }

  if (loads && lw == 0) {
#pragma unroll
    for (int j = 0; j < 3; j++) {
      entry = entry_for(j);
      put_rows(j);
      if (j < 2) put_scales(j);
    }
    entry = entry_for(3);
  }
  __syncthreads();
  if (loads) {
    load_step(0);
    put_step(0);
    load_step(1);
  }
  auto ahead = [&](int j) __attribute__((always_inline)) {
    if (lw == 0) {
      put_scales(j + 2);
      put_rows(j + 3);
      entry = entry_for(j + 4);
    }
  };
  if constexpr (LW != 0)
    if (loads) {
      for (int j = 0; j < steps; j++) {
        barrier();
        if (j + 1 < steps) put_step(j + 1);
        if (j + 2 < steps) load_step(j + 2);
        ahead(j);
      }
      return;
    }
  for (int j = 0; j < steps; j++) {
    const int ln = opaque(lane), hf = ln >> 5;
    barrier();  // step j is there, and everyone is done with step j - 1's buffer
    if constexpr (LW == 0) {
      if (j + 1 < steps) put_step(j + 1);
      ahead(j);
    }
    const uint4 *kd = s_kv + (j & 1) * (KU + VU), *vd = kd + KU;
    const int32_t unit = w.unit(j), key0 = unit * S;
    const bool mine = any_seen(p, wlo, whi, key0, S);
    uint4 pu[KT][PU];
    if (mine) {
      const uint64_t mapped = uniform(s_map[j & 7]);
      const bool full = whole_tile && mapped == ~0ull && all_seen(p, wlo, whi, key0, S);
      f32x16 s[KT];
#pragma unroll
      for (int kt = 0; kt < KT; kt++) s[kt] = f32x16{};
      feed<KT * G8::NQ>(
          [&](int n) __attribute__((always_inline)) {
            const int t = n / KT, row = 32 * (n % KT) + (ln & 31);
            return kd[row * G::CH + ((4 * (t >> 1) + 2 * hf + (t & 1)) ^ G::kswz(row))];
          },
          [&](int n, uint4 k) __attribute__((always_inline)) {
            s[n % KT] = G::score(k, q[n / KT], s[n % KT]);
          });
      uint64_t seen = 0;
      if (!full) {
        const int c = cw + (opaque(lane) & 31);
        seen = seen_bits(p, c < ncol ? p0 + c / p.G : -1, key0, mapped) >> (4 * hf);
      }
      const float *cs = s_c[j & 3], *gs = s_vs[j & 3];
      // A lane's sum of at most kMostSum holds no score that moves the base;
      // else, and at a segment's first step, the largest score decides.
      float psum;
      bool look = fresh;
      for (;;) {
        if (look) {
          const float t = full ? G8::template top<true>(s, cs, hf, seen) : G8::template top<false>(s, cs, hf, seen);
          const float mn = next_base(m, t, 1.f);
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
        psum = full ? G8::template weights<true>(s, cs, gs, hf, seen, m, pu)
                    : G8::template weights<false>(s, cs, gs, hf, seen, m, pu);
        if (look || __builtin_amdgcn_ballot_w64(psum > kMostSum) == 0) break;
        look = true;
      }
      l += psum;
      fresh = false;
    }
    // (Not before the scores, whose operands need the registers.)
    if constexpr (LW == 0)
      if (j + 2 < steps) load_step(j + 2);
    if (mine) {
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
    if (j + 1 == steps || w.unit(j + 1) / G8::kSegSteps != unit / G8::kSegSteps) {
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
  }

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
  k.seg16_us = k.seg32_us = G8::seg_us();
  k.per_cu16 = k.per_cu32 = G8::split_per_cu();
  k.whole4_pair = nullptr;
  if constexpr (G8::kTwoWaves) {
    k.whole4 = whole8_kernel<T, D, V, 4, 4>;
    k.whole8 = whole8_kernel<T, D, V, 8, 0>;
  } else {
    k.whole4 = whole8_kernel<T, D, V, 4, 0>;
    k.whole8 = nullptr;
  }
  k.whole4_threads = G8::kTwoWaves ? 512 : 256;
  return k;
}

}  // namespace
}  // namespace bi_paged

#define BI_PAGED_Q8_KERNELS(D, V)                                 \
  bi_paged::Kernels bi_paged::kernels8_d##D##_v##V(int dtype) {   \
    return dtype == BI_F16 ? kernels8_of<_Float16, D, V>()        \
                           : kernels8_of<__bf16, D, V>();         \
  }
