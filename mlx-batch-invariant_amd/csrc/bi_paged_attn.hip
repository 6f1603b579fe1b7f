// Attention over a paged cache and windowed attention over contiguous keys:
// the C entry points and the choice of route (contract in include/bi.h, kernels
// in bi_paged_attn_kernel.h).
#include <math.h>

#include "bi_paged_attn.h"

namespace {

using namespace bi_paged;

bool dims_built(int64_t D, int64_t V) {
#define BI_CASE(d, v) if (D == d && V == v) return true;
  BI_PAGED_DIM_PAIRS(BI_CASE)
#undef BI_CASE
  return false;
}

Kernels kernels(int64_t D, int64_t V, int dtype) {
#define BI_CASE(d, v) if (D == d && V == v) return kernels_d##d##_v##v(dtype);
  BI_PAGED_DIM_PAIRS(BI_CASE)
#undef BI_CASE
  return Kernels{};
}

// Tokens, lengths and windows past this are not computed with (positions
// minus a window stay in 32 bits).
constexpr int64_t kMost = (int64_t)1 << 30;

// How a call is split: the columns up to which a request is (0: none), and the
// memory of its partial results. `exact`: every request has max_query tokens.
struct Plan {
  int64_t split_cols, ccap, nc, nseg, bytes;
};
Plan plan(int64_t R, int64_t G, int64_t Hkv, int64_t V, int64_t window, int64_t first,
          int64_t max_query, int64_t max_seq, bool exact, const Kernels& k) {
  Plan s = {0, 0, 0, 0, 0};
  const int64_t cols = max_query * G;
  if (R <= 0 || cols <= 0 || max_seq <= 0) return s;
  s.split_cols = 32;
  if (exact && cols > s.split_cols) return Plan{0, 0, 0, 0, 0};
  s.ccap = cols < s.split_cols ? cols : s.split_cols;
  // Beside requests of more columns those of few are mostly single tokens: then
  // two workgroups of 16 columns, of which such a request needs one.
  s.nc = s.ccap > 16 && cols <= s.split_cols ? 32 : 16;
  const int64_t part = k.seg;
  s.nseg = (max_seq + part - 1) / part;
  if (window) {
    // Tokens of a workgroup's columns, rows that they see between them.
    const int64_t span = window + (s.nc - 1) / G + 1;
    const int64_t n = (span + part - 2) / part + 1 + (first + part - 1) / part;
    if (n < s.nseg) s.nseg = n;
  }
  s.bytes = R * Hkv * s.ccap * s.nseg * (V + 2) * (int64_t)sizeof(float);
  if (s.bytes > (int64_t)1 << 31 || R * Hkv * s.nseg > INT32_MAX ||
      R * Hkv * s.ccap > INT32_MAX) return Plan{0, 0, 0, 0, 0};
  return s;
}

int launch(const char* who, Args& p, int64_t D, int64_t V, int dtype, void* ws, int64_t ws_bytes,
           void* stream) {
  const Kernels k = kernels(D, V, dtype);
  const hipStream_t st = static_cast<hipStream_t>(stream);
  const int64_t most = p.qstart ? p.max_query : p.qL;
  Plan s = plan(p.R, p.G.d, p.Hkv.d, V, p.window, p.first, most, p.qstart ? p.max_seq : p.N,
                !p.qstart, k);
  if (!ws || (uintptr_t)ws % 16 || ws_bytes < s.bytes) s = Plan{0, 0, 0, 0, 0};
  hipError_t e;
  if (s.split_cols) {
    p.split_cols = (int32_t)s.split_cols;
    p.ccap = make_div(s.ccap);
    p.nseg = make_div(s.nseg);
    p.reqs = make_div(p.R);
    p.nc = (int32_t)s.nc;
    p.po = static_cast<float*>(ws);
    p.pml = reinterpret_cast<float2*>(p.po + (int64_t)p.R * p.Hkv.d * s.ccap * s.nseg * V);
    const dim3 grid((unsigned)(p.R * p.Hkv.d * s.nseg), (unsigned)((s.ccap + s.nc - 1) / s.nc));
    hipLaunchKernelGGL(s.nc == 16 ? k.split16 : k.split32, grid, dim3(256), 0, st, p);
    if ((e = hipGetLastError()) != hipSuccess) return bi::launch_error(e, who);
  }
  const bool whole = most * p.G.d > s.split_cols;
  p.fill_blocks = p.qstart ? 16 : 0;
  if (s.split_cols) {
    const int64_t cols = (int64_t)p.R * p.Hkv.d * s.ccap;
    hipLaunchKernelGGL(k.combine, dim3((unsigned)((cols + 3) / 4 + p.fill_blocks)), dim3(256), 0,
                       st, p);
    if ((e = hipGetLastError()) != hipSuccess) return bi::launch_error(e, who);
    p.fill_blocks = 0;
  }
  if (whole || p.fill_blocks) {
    // Eight waves share their keys' and values' loads and addresses where that
    // leaves a workgroup for every compute unit (4096 tokens over 8192 keys 517
    // -> 496 us); with fewer, four of them fill more (two chunks of 511 tokens
    // beside 30 decodes 161 us, 175 with eight), two to a compute unit where
    // there are more than these.
    const int64_t cols = p.qstart ? (int64_t)p.T * p.G.d : (int64_t)p.R * p.qL * p.G.d;
    const int cus = bi::device_cus();
    const bool eight = k.whole8 && cols / 256 * p.Hkv.d >= cus;
    const bool pair = !eight && k.whole4_pair && cols / 128 * p.Hkv.d > cus;
    const int64_t wc = eight ? 256 : 128;
    // Column tiles: every request with tokens may end in a part of one.
    int64_t tiles = p.qstart ? cols / wc + (p.T < p.R ? p.T : p.R)
                             : (int64_t)p.R * (((int64_t)p.qL * p.G.d + wc - 1) / wc);
    if (!whole) tiles = 0;
    const int64_t blocks = tiles * p.Hkv.d + p.fill_blocks;
    if (blocks > INT32_MAX) return bi::fail(BI_EINVAL, "%s: grid too large", who);
    if (blocks == 0) return BI_OK;
    hipLaunchKernelGGL(eight ? k.whole8 : pair ? k.whole4_pair : k.whole4, dim3((unsigned)blocks),
                       dim3(eight ? 512 : pair ? 256 : k.whole4_threads), 0, st, p);
    if ((e = hipGetLastError()) != hipSuccess) return bi::launch_error(e, who);
  }
  return BI_OK;
}

// The checks that both entry points share.
int check(const char* who, int64_t H, int64_t Hkv, int64_t D, int64_t V, float scale,
          int64_t window, int64_t sink_tokens, int dtype) {
  if (!bi::elem_size(dtype)) return bi::fail(BI_EINVAL, "%s: unknown dtype %d", who, dtype);
  if (H <= 0 || Hkv <= 0 || H > 65535 || H % Hkv)
    return bi::fail(BI_EINVAL, "%s: H=%lld is not a multiple of Hkv=%lld (at most 65535)", who,
                    (long long)H, (long long)Hkv);
  if (window < 0 || sink_tokens < 0)
    return bi::fail(BI_EINVAL, "%s: negative window or sink_tokens", who);
  if (scale != scale) return bi::fail(BI_EINVAL, "%s: scale is NaN", who);
  if (!dims_built(D, V))
    return bi::fail(BI_EUNSUPPORTED, "%s: head dims D=%lld V=%lld are not built (built: 64, 96, "
                    "128, 192 and 256 for both, and (192, 128))", who, (long long)D, (long long)V);
  return BI_OK;
}

bool aligned16(const void* a, const void* b, const void* c, const int64_t* strides, int n, int esz) {
  if (((uintptr_t)a | (uintptr_t)b | (uintptr_t)c) % 16) return false;
  for (int i = 0; i < n; i++)
    if (strides[i] * esz % 16) return false;
  return true;
}

int32_t clamp32(int64_t x) { return x > kMost ? (int32_t)kMost : (int32_t)x; }

void common(Args& p, int64_t H, int64_t Hkv, float scale, int64_t window, int64_t sink_tokens,
            int dtype) {
  p.H = (int32_t)H;
  p.Hkv = make_div(Hkv);
  p.G = make_div(H / Hkv);
  p.window = clamp32(window);
  p.first = clamp32(sink_tokens);
  // Not 0, with which an unseen row's -inf would not stay one.
  p.scale2 = fmaxf(fabsf(scale) * 1.4426950408889634f, 1.2e-38f);
  p.qsign = scale < 0.f ? (dtype == BI_F32 ? 0x80000000u : 0x80008000u) : 0u;
}

}  // namespace

extern "C" int bi_paged_attention(const void* q, const void* k_cache, const void* v_cache,
                                  const int32_t* block_tables, const int32_t* query_start,
                                  const int32_t* seq_lens, const void* sinks, void* out, int64_t T,
                                  int64_t R, int64_t H, int64_t Hkv, int64_t D, int64_t V,
                                  int64_t num_pages, int64_t page_size, int64_t W,
                                  const int64_t* strides, float scale, int64_t window,
                                  int64_t sink_tokens, int64_t max_query, int64_t max_seq,
                                  int dtype, void* workspace, int64_t workspace_bytes,
                                  void* hip_stream) {
  const char* who = "bi_paged_attention";
  int rc = check(who, H, Hkv, D, V, scale, window, sink_tokens, dtype);
  if (rc) return rc;
  if (T < 0 || R < 0 || num_pages < 0 || page_size <= 0 || W < 0 || max_query < 0 || max_seq < 0 ||
      T > kMost || T * H > INT32_MAX || R > kMost || num_pages > INT32_MAX || page_size > INT32_MAX ||
      W > INT32_MAX)
    return bi::fail(BI_EINVAL, "%s: bad sizes T=%lld R=%lld pages=%lld x %lld W=%lld", who,
                    (long long)T, (long long)R, (long long)num_pages, (long long)page_size,
                    (long long)W);
  if (T == 0) return BI_OK;
  if (!q || !out || !query_start || (R > 0 && !seq_lens) || !strides ||
      (R > 0 && W > 0 && !block_tables) || (num_pages > 0 && (!k_cache || !v_cache)))
    return bi::fail(BI_EINVAL, "%s: null pointer", who);
  const int esz = bi::elem_size(dtype);
  if (!aligned16(q, k_cache, v_cache, strides, 8, esz))
    return bi::fail(BI_EINVAL, "%s: q and caches must be 16-byte aligned, with strides of "
                    "multiples of 16 bytes", who);
  Args p = {};
  common(p, H, Hkv, scale, window, sink_tokens, dtype);
  p.q = q;
  p.k = k_cache;
  p.v = v_cache;
  p.sinks = sinks;
  p.out = out;
  p.table = block_tables;
  p.qstart = query_start;
  p.seq = seq_lens;
  p.qt = strides[0], p.qh = strides[1];
  p.ot = H * V, p.oh = V;
  p.kb = strides[2], p.kh = strides[3], p.kn = strides[4];
  p.vb = strides[5], p.vh = strides[6], p.vn = strides[7];
  p.table_stride = strides[8];
  p.R = (int32_t)R;
  p.W = (int32_t)W;
  p.pages = (int32_t)num_pages;
  p.T = (int32_t)T;
  p.max_query = clamp32(max_query);
  p.max_seq = clamp32(max_seq);
  p.page = make_div(page_size);
  return launch(who, p, D, V, dtype, workspace, workspace_bytes, hip_stream);
}

extern "C" int64_t bi_paged_attention_workspace(int64_t T, int64_t R, int64_t H, int64_t Hkv,
                                                int64_t D, int64_t V, int64_t window,
                                                int64_t sink_tokens, int64_t max_query,
                                                int64_t max_seq, int dtype) {
  if (T <= 0 || R <= 0 || H <= 0 || Hkv <= 0 || H % Hkv || !bi::elem_size(dtype) ||
      !dims_built(D, V) || T > kMost || R > kMost || window < 0 || sink_tokens < 0)
    return 0;
  return plan(R, H / Hkv, Hkv, V, clamp32(window), clamp32(sink_tokens),
              clamp32(max_query), clamp32(max_seq), false, kernels(D, V, dtype)).bytes;
}

extern "C" int bi_window_attention(const void* q, const void* k, const void* v, const void* sinks,
                                   void* out, int64_t B, int64_t H, int64_t Hkv, int64_t qL,
                                   int64_t N, int64_t D, int64_t V, const int64_t* strides,
                                   float scale, int64_t window, int64_t sink_tokens, int dtype,
                                   void* workspace, int64_t workspace_bytes, void* hip_stream) {
  const char* who = "bi_window_attention";
  int rc = check(who, H, Hkv, D, V, scale, window, sink_tokens, dtype);
  if (rc) return rc;
  if (B < 0 || qL < 0 || N < 0 || N > kMost || qL > kMost || B > kMost || B * qL > kMost ||
      B * qL * H > INT32_MAX)
    return bi::fail(BI_EINVAL, "%s: bad sizes B=%lld qL=%lld N=%lld", who, (long long)B,
                    (long long)qL, (long long)N);
  if (B == 0 || qL == 0) return BI_OK;
  if (!q || !out || !strides || (N > 0 && (!k || !v)))
    return bi::fail(BI_EINVAL, "%s: null pointer", who);
  if (!aligned16(q, N > 0 ? k : nullptr, N > 0 ? v : nullptr, strides, 9, bi::elem_size(dtype)))
    return bi::fail(BI_EINVAL, "%s: q, k and v must be 16-byte aligned, with strides of multiples "
                    "of 16 bytes", who);
  Args p = {};
  common(p, H, Hkv, scale, window, sink_tokens, dtype);
  p.q = q;
  p.k = k;
  p.v = v;
  p.sinks = sinks;
  p.out = out;
  p.qb = strides[0], p.qh = strides[1], p.qt = strides[2];
  p.ob = H * qL * V, p.oh = qL * V, p.ot = V;
  p.kb = strides[3], p.kh = strides[4], p.kn = strides[5];
  p.vb = strides[6], p.vh = strides[7], p.vn = strides[8];
  p.R = (int32_t)B;
  p.qL = (int32_t)qL;
  p.N = (int32_t)N;
  return launch(who, p, D, V, dtype, workspace, workspace_bytes, hip_stream);
}

extern "C" int64_t bi_window_attention_workspace(int64_t B, int64_t H, int64_t Hkv, int64_t qL,
                                                 int64_t N, int64_t D, int64_t V, int64_t window,
                                                 int64_t sink_tokens, int dtype) {
  if (B <= 0 || H <= 0 || Hkv <= 0 || H % Hkv || qL <= 0 || N <= 0 || !bi::elem_size(dtype) ||
      !dims_built(D, V) || qL > kMost || N > kMost || B > kMost || window < 0 || sink_tokens < 0)
    return 0;
  return plan(B, H / Hkv, Hkv, V, clamp32(window), clamp32(sink_tokens), qL, N, true,
              kernels(D, V, dtype)).bytes;
}
