// Attention over a paged cache and windowed attention over contiguous keys:
// the C entry points and the kernels (contract in include/bi.h).
#include <float.h>
#include <math.h>

#include "bi_paged_attn.h"

namespace {

using namespace bi_paged;

template <typename T> __device__ __forceinline__ float up(T x) { return (float)x; }

// One wave per (token, head): 64 keys at a time, a key per lane, then a value
// dim per lane.
template <typename T, int D, int V>
__global__ void __launch_bounds__(64) attend_simple(Args p) {
  const int lane = threadIdx.x;
  const int h = blockIdx.y, kvh = h / p.G;
  int r = 0, i = 0;
  int64_t qoff, ooff;
  Request rq;
  constexpr int NV = (V + 63) / 64;
  if (p.qstart) {
    const int t = blockIdx.x;
    qoff = t * p.qt + h * p.qh;
    ooff = t * p.ot + h * p.oh;
    bool owned = false;
    for (r = 0; r < p.R; r++) {
      rq = request(p, r);
      if (t >= rq.t0 && t < rq.t0 + rq.L) {
        owned = true;
        break;
      }
    }
    if (!owned) {
      for (int j = 0; j < NV; j++)
        if (lane + 64 * j < V) static_cast<T*>(p.out)[ooff + lane + 64 * j] = (T)0.f;
      return;
    }
    i = (int)(t - rq.t0);
  } else {
    r = blockIdx.x / p.qL;
    i = blockIdx.x % p.qL;
    rq = request(p, r);
    qoff = r * p.qb + i * p.qt + h * p.qh;
    ooff = r * p.ob + i * p.ot + h * p.oh;
  }
  const T* q = static_cast<const T*>(p.q) + qoff;
  T* out = static_cast<T*>(p.out) + ooff;
  const int32_t pos = rq.n - rq.L + i;
  float m = -INFINITY, l = 0.f, o[NV] = {};
  if (p.sinks) {
    m = up(static_cast<const T*>(p.sinks)[h]) * 1.4426950408889634f;
    l = 1.f;
  }
  for (int32_t j0 = 0; j0 <= pos; j0 += 64) {
    const int32_t j = j0 + lane;
    bool use = sees(p, pos, j);
    int64_t ko = 0, vo = 0;
    if (use) {
      if (p.qstart) {
        const int32_t pg = j / p.page, row = j - pg * p.page;
        const int32_t id = pg < p.W ? p.table[r * p.table_stride + pg] : -1;
        use = id >= 0 && id < p.pages;
        ko = id * p.kb + kvh * p.kh + row * p.kn;
        vo = id * p.vb + kvh * p.vh + row * p.vn;
      } else {
        ko = r * p.kb + kvh * p.kh + j * p.kn;
        vo = r * p.vb + kvh * p.vh + j * p.vn;
      }
    }
    float s = -INFINITY;
    if (use) {
      const T* k = static_cast<const T*>(p.k) + ko;
      float a = 0.f;
      for (int d = 0; d < D; d++) a = fmaf(up(q[d]), up(k[d]), a);
      s = (p.qneg ? -a : a) * p.scale2;
    }
    float bm = s;
    for (int x = 1; x < 64; x <<= 1) bm = fmaxf(bm, __shfl_xor(bm, x));
    const float mn = fmaxf(m, bm);
    if (mn == -INFINITY) continue;
    const float f = exp2f(m - mn);
    const float w = use ? exp2f(s - mn) : 0.f;
    float bs = w;
    for (int x = 1; x < 64; x <<= 1) bs += __shfl_xor(bs, x);
    l = l * f + bs;
    m = mn;
    for (int jv = 0; jv < NV; jv++) o[jv] *= f;
    for (int x = 0; x < 64; x++) {
      const float wx = __shfl(w, x);
      const int64_t vx = __shfl(vo, x);
      if (!__shfl((int)use, x)) continue;
      const T* v = static_cast<const T*>(p.v) + vx;
      for (int jv = 0; jv < NV; jv++)
        if (lane + 64 * jv < V) o[jv] = fmaf(wx, up(v[lane + 64 * jv]), o[jv]);
    }
  }
  for (int jv = 0; jv < NV; jv++)
    if (lane + 64 * jv < V)
      out[lane + 64 * jv] = rq.beyond ? (T)NAN : (T)(l == 0.f ? 0.f : o[jv] / l);
}

typedef void (*Kernel)(Args);
template <int D, int V> Kernel kernel_of(int dtype) {
  return dtype == BI_F32 ? attend_simple<float, D, V>
         : dtype == BI_F16 ? attend_simple<_Float16, D, V>
                           : attend_simple<__bf16, D, V>;
}

#define BI_PAGED_DIM_PAIRS(X) X(64, 64) X(96, 96) X(128, 128) X(192, 128) X(192, 192) X(256, 256)

bool dims_built(int64_t D, int64_t V) {
#define BI_CASE(d, v) if (D == d && V == v) return true;
  BI_PAGED_DIM_PAIRS(BI_CASE)
#undef BI_CASE
  return false;
}

int launch(const char* who, const Args& p, int64_t D, int64_t V, int dtype, void* stream) {
  Kernel fn = nullptr;
#define BI_CASE(d, v) if (D == d && V == v) fn = kernel_of<d, v>(dtype);
  BI_PAGED_DIM_PAIRS(BI_CASE)
#undef BI_CASE
  const int64_t rows = p.qstart ? p.T : (int64_t)p.R * p.qL;
  hipLaunchKernelGGL(fn, dim3((unsigned)rows, (unsigned)p.H), dim3(64), 0,
                     static_cast<hipStream_t>(stream), p);
  const hipError_t e = hipGetLastError();
  return e == hipSuccess ? BI_OK : bi::launch_error(e, who);
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

int32_t clamp32(int64_t x) { return x > INT32_MAX ? INT32_MAX : (int32_t)x; }

void common(Args& p, int64_t H, int64_t Hkv, float scale, int64_t window, int64_t sink_tokens) {
  p.H = (int32_t)H;
  p.Hkv = (int32_t)Hkv;
  p.G = (int32_t)(H / Hkv);
  p.window = clamp32(window);
  p.first = clamp32(sink_tokens);
  p.scale2 = fabsf(scale) * 1.4426950408889634f;
  p.qneg = scale < 0.f;
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
      T > INT32_MAX || R > INT32_MAX || num_pages > INT32_MAX || page_size > INT32_MAX ||
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
  common(p, H, Hkv, scale, window, sink_tokens);
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
  p.page = (int32_t)page_size;
  p.pages = (int32_t)num_pages;
  p.T = (int32_t)T;
  p.max_query = clamp32(max_query);
  p.max_seq = clamp32(max_seq);
  return launch(who, p, D, V, dtype, hip_stream);
}

extern "C" int64_t bi_paged_attention_workspace(int64_t T, int64_t R, int64_t H, int64_t Hkv,
                                                int64_t D, int64_t V, int64_t window,
                                                int64_t sink_tokens, int64_t max_query,
                                                int64_t max_seq, int dtype) {
  return 0;
}

extern "C" int bi_window_attention(const void* q, const void* k, const void* v, const void* sinks,
                                   void* out, int64_t B, int64_t H, int64_t Hkv, int64_t qL,
                                   int64_t N, int64_t D, int64_t V, const int64_t* strides,
                                   float scale, int64_t window, int64_t sink_tokens, int dtype,
                                   void* workspace, int64_t workspace_bytes, void* hip_stream) {
  const char* who = "bi_window_attention";
  int rc = check(who, H, Hkv, D, V, scale, window, sink_tokens, dtype);
  if (rc) return rc;
  if (B < 0 || qL < 0 || N < 0 || N > INT32_MAX - 4096 || qL > INT32_MAX || B > INT32_MAX ||
      B * qL > INT32_MAX)
    return bi::fail(BI_EINVAL, "%s: bad sizes B=%lld qL=%lld N=%lld", who, (long long)B,
                    (long long)qL, (long long)N);
  if (B == 0 || qL == 0) return BI_OK;
  if (!q || !out || !strides || (N > 0 && (!k || !v)))
    return bi::fail(BI_EINVAL, "%s: null pointer", who);
  if (!aligned16(q, N > 0 ? k : nullptr, N > 0 ? v : nullptr, strides, 9, bi::elem_size(dtype)))
    return bi::fail(BI_EINVAL, "%s: q, k and v must be 16-byte aligned, with strides of multiples "
                    "of 16 bytes", who);
  Args p = {};
  common(p, H, Hkv, scale, window, sink_tokens);
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
  p.max_query = p.max_seq = INT32_MAX;
  return launch(who, p, D, V, dtype, hip_stream);
}

extern "C" int64_t bi_window_attention_workspace(int64_t B, int64_t H, int64_t Hkv, int64_t qL,
                                                 int64_t N, int64_t D, int64_t V, int64_t window,
                                                 int64_t sink_tokens, int dtype) {
  return 0;
}
