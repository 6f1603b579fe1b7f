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

// `q8`: over a cache of 8 bits.
Kernels kernels(int64_t D, int64_t V, int dtype, bool q8) {
#define BI_CASE(d, v) if (D == d && V == v) return q8 ? kernels8_d##d##_v##v(dtype) : kernels_d##d##_v##v(dtype);
  BI_PAGED_DIM_PAIRS(BI_CASE)
#undef BI_CASE
  return Kernels{};
}

// Tokens, lengths and windows past this are not computed with (positions
// minus a window stay in 32 bits).
constexpr int64_t kMost = (int64_t)1 << 29;
// Workspaces are not larger.
constexpr int64_t kMostBytes = (int64_t)1 << 32;
// Rows that are laid out have a place for every row that a request may have where that
// takes no more than this; else for as many as are expected, or as fit in this.
constexpr int64_t kLaidBytes = (int64_t)1 << 27;

// A call as the host knows it; `exact`: every request has max_query tokens.
struct Call {
  int64_t R, tokens, G, Hkv, D, V, window, first, max_query, max_seq;
  bool exact;
  double bytes;  // of a cached element
};

// How a call is split: the columns up to which a request is (0: none), columns
// kept per request and kv head, columns per workgroup, segments, workgroups for
// these, and the bytes of the partial results. Of the others' rows that are laid
// out (a cache of 8 bits): the steps of a request, those that one walks at most,
// places for all (0: `units` for each), and the bytes, 0 for none.
struct Plan {
  int64_t split_cols, ccap, nc, nseg, gseg, bytes, units, walked, room, laid;
  int64_t laid_at() const { return (bytes + 15) / 16 * 16; }
  int64_t workspace() const { return laid ? laid_at() + laid : bytes; }
};
// Bytes of a note for each request where its steps are.
int64_t notes(int64_t R) { return (4 * R + 511) / 512 * 512; }

// Column tiles of all requests that can have a token (one of each request is
// not full).
int64_t full_tiles(const Call& c, const Plan& s) {
  const int64_t all = c.R * ((s.ccap + s.nc - 1) / s.nc), full = c.tokens * c.G / s.nc + c.R;
  return all < full ? all : full;
}

// A plan that splits requests of up to `most` columns.
Plan split_up_to(const Call& c, int64_t most, const Kernels& k) {
  const int64_t seg = k.seg;
  Plan s = {};
  const int64_t cols = c.max_query * c.G;
  s.split_cols = most;
  s.ccap = cols < most ? cols : most;
  // Beside requests of more columns those of few are mostly single tokens: then
  // workgroups of 16 columns, of which such a request needs one.
  s.nc = s.ccap > 16 && (cols <= most || c.G > 16) ? 32 : 16;
  s.nseg = (c.max_seq + seg - 1) / seg;
  if (c.window) {
    // Tokens of a workgroup's columns, rows that they see between them.
    const int64_t span = c.window + (s.nc - 1) / c.G + 1;
    const int64_t n = (span + seg - 2) / seg + 1 + (c.first + seg - 1) / seg;
    if (n < s.nseg) s.nseg = n;
  }
  // Places for a request's segments: k.places workgroups in all, not counting
  // columns that no token has.
  const int64_t places = k.places / (c.Hkv * full_tiles(c, s));
  s.gseg = places < 1 ? 1 : places < s.nseg ? places : s.nseg;
  s.bytes = c.R * c.Hkv * s.ccap * s.nseg * (c.V + 2) * (int64_t)sizeof(float);
  return s;
}
int64_t split_grid(const Call& c, const Plan& s) {
  return c.R * c.Hkv * s.gseg * ((s.ccap + s.nc - 1) / s.nc);
}
bool fits(const Call& c, const Plan& s) {
  return s.bytes <= kMostBytes && split_grid(c, s) <= 1 << 23 && c.R * c.Hkv * s.ccap <= 1 << 24;
}

// Requests are split where that is estimated to take less time than to walk
// them whole; beside chunks of more than 2048 columns, and where the bounds are
// far above the average request, those of single tokens and a few (32 columns)
// are. Microseconds, from times of every head dim and type (prices of a row and
// of a segment: Geo in bi_paged_attn_kernel.h): a whole workgroup 7.5 and the
// rows it walks, one per compute unit at a time; the split ones that a compute
// unit runs together as much as a full segment costs, half of it for a segment
// and half by its passes of four steps (0.85 of it for one alone where two fit;
// 0.4 of a round more, as the last is rarely full), an empty one 3.3; reading
// the cache once at 5 TB/s; the partial results' way through memory and back at
// 4 TB/s; a launch 2, two with their chain 10. Tokens of a chunk see all but
// half of the chunk's rows on average. (whole / split, 32/8 heads: bf16, D = V =
// 128, over 8192 rows 16 tokens 157 / 21.5, 64 162 / 59, 128 164 / 107, 256 163
// / 199; 64 requests of one token and 300 rows 31.8 / 27.8, 32 of 16 and 1024
// 33.3 / 70.6; 16 under a window of 1024 33.9 / 23.0, of 512 21.5 / 19.5, 64 of
// 512 43.1 / 44.0. 64/64, 128 tokens over 8192 rows 125 / 55; 256/256, 256 513 /
// 344, 512 513 / 659. fp32, 128/128, 64 requests of 2048 rows 570 / 284, 256
// tokens over 4096 rows 559 / 368, 512 559 / 670; 256/256, 1000 tokens of a
// prompt, 8/8 heads 331 / 124. Of 822 sizes timed both ways it picks the one
// that takes 8 % more or worse four times, 29 % at most; over a cache of 8 bits, of
// 666 sizes timed each way, with its rows laid out too, 1 % on average, 20 % or worse
// seven times, mostly over 200 rows. 64 single tokens under a
// bound of 64 229, with all these columns split 1030.)
Plan plan(const Call& c, const Kernels& k) {
  const Plan none = {};
  const int64_t cols = c.max_query * c.G;
  if (c.R <= 0 || cols <= 0 || c.max_seq <= 0) return none;
  const int64_t few = c.G > 32 ? c.G : 32;
  const double cus = bi::device_cus(), H = (double)(c.G * c.Hkv), seq = (double)c.max_seq;
  // Rows that a token sees at most; `cut`: under a window.
  const double wide = (double)(c.window + c.first);
  const bool cut = c.window && wide < seq;
  const double rows = cut ? wide : seq;
  const double chunk = (double)(c.max_query < c.max_seq ? c.max_query : c.max_seq);
  const double read = (double)c.R * rows * c.Hkv * (c.D + c.V) * c.bytes / 5e6;
  const double all = (double)c.R * ((cols + 127) / 128), full = (double)c.tokens * c.G / 128.0 + c.R;
  const double tiles = (all < full ? all : full) * c.Hkv / cus;
  auto walk_us = [&](double row_us, double tile_us) {
    const double walked = (cut ? rows + 128.0 / c.G + 64.0 : rows) * row_us;
    const double first = 7.5 + walked, most = tiles * (tile_us + walked * (cut ? 1.0 : 1.0 - 0.5 * chunk / seq));
    const double us = first > most ? first : most;
    return 2.0 + (us > 1.1 * read ? us : 1.1 * read);
  };
  double whole = walk_us(k.row_us, 7.5);
  // Whether the rows that are walked whole are laid out first: a launch, and their
  // codes through memory, three bytes for each, at 4 TB/s.
  Plan lay = none;
  if (k.lay) {
    const double requests = (double)c.tokens / (double)c.max_query, part = (double)c.max_query + wide;
    const double laid = (cut && part < seq ? part : seq) * (requests < 1.0 ? 1.0 : requests < c.R ? requests : c.R);
    const double us = walk_us(k.laid_row_us, k.laid_tile_us) + 4.0 + laid * c.Hkv * (c.D + c.V) * 3.0 / 4e6;
    lay.units = (c.max_seq + k.step - 1) / k.step;
    double bytes = (double)c.R * (double)(c.Hkv * lay.units * k.step_bytes);
    if (bytes > (double)kLaidBytes) {
      // As if the tokens were of requests with max_query each: 64 requests of up to 8192
      // rows, of which one brings a chunk, would have places for all of theirs in 2.2 GB.
      const int64_t most = (c.max_query + c.window + c.first) / k.step + 4;  // (a window's ends, the first tokens')
      lay.walked = c.window && most < lay.units ? most : lay.units;
      const int64_t n = c.tokens / c.max_query + (c.tokens % c.max_query != 0), each = c.Hkv * lay.walked;
      const double least = (double)(kLaidBytes / k.step_bytes), some = (double)(n < c.R ? n : c.R) * (double)each;
      const double room = some > least ? some : least, some_bytes = room * k.step_bytes + (double)notes(c.R);
      if (some_bytes < bytes) bytes = some_bytes, lay.room = bytes <= (double)kMostBytes ? (int64_t)room : 0;
    }
    if (us < whole && bytes <= (double)kMostBytes) {
      whole = us;
      lay.laid = (int64_t)bytes;
    } else {
      lay = none;
    }
  }
  auto beside = [&](Plan s) {
    if (cols > s.split_cols && s.bytes + lay.laid <= kMostBytes)
      s.units = lay.units, s.walked = lay.walked, s.room = lay.room, s.laid = lay.laid;
    return s;
  };
  auto split = [&](const Plan& s) {
    const double busy = (double)full_tiles(c, s) * c.Hkv, n = (double)s.nseg;
    const int per_cu = s.nc == 16 ? k.per_cu16 : k.per_cu32;
    const double slots = per_cu * cus, seg = s.nc == 16 ? k.seg16_us : k.seg32_us;
    // Segments and passes of a column tile, on average under a window, which
    // begins and ends inside of them.
    const double span = rows + (double)s.nc / c.G - 1.0, more = c.first ? 2.0 : 1.0;
    double segs = cut ? span / k.seg + more : n, passes = cut ? span / k.pass + more : ceil(seq / k.pass);
    const double in = (double)(k.seg / k.pass);
    if (segs > n) segs = n;
    if (passes > n * in) passes = n * in;
    const double later = seq > k.seg ? 1.0 - k.seg / seq : 0.0, mean = cut ? 1.0 : 1.0 - 0.5 * chunk / seq * later;
    const double rounds = busy * 0.5 * (segs + passes / in) / slots * mean;
    const double part = rows < k.seg ? rows / k.seg : 1.0;
    const double alone = (0.5 + 0.5 * part) * (per_cu == 2 ? 0.85 : 1.0);
    double walk = rounds + (rounds < 1.0 ? 0.4 * rounds : 0.4);
    walk = (walk > alone ? walk : alone) * seg;
    const double idle = ((double)split_grid(c, s) - busy * s.gseg * mean) / slots * 3.3;
    return 10.0 + (walk > 0.9 * read ? walk : 0.9 * read) +
           (double)c.tokens * H * segs * (c.V + 2) * 8.0 / 4e6 + idle;
  };
  // Bounds far above the average request: most have a few columns.
  const bool loose = cols > few && c.tokens * c.G <= c.R * (few / 2);
  if (cols <= few || (cols <= 2048 && !loose)) {
    const Plan s = split_up_to(c, cols > few ? cols : few, k);
    if (fits(c, s) && split(s) < whole) return s;
    if (cols <= few && whole <= split(s)) return lay;
  }
  // All requests have max_query tokens, or what is missing is padding (else
  // two launches that find nothing, 3 to 4 us each).
  if (c.exact || c.tokens >= c.R * c.max_query) return lay;
  // Beside whole chunks; where the results would take too much, single tokens.
  Plan s = split_up_to(c, few, k);
  if (!fits(c, s)) s = split_up_to(c, c.G, k);
  return fits(c, s) ? beside(s) : lay;
}

int launch(const char* who, Args& p, int64_t D, int64_t V, int dtype, bool q8, void* ws, int64_t ws_bytes,
           void* stream) {
  const Kernels k = kernels(D, V, dtype, q8);
  const hipStream_t st = static_cast<hipStream_t>(stream);
  const int64_t most = p.qstart ? p.max_query : p.qL;
  const Call c = {p.R, p.qstart ? p.T : (int64_t)p.R * p.qL, p.G.d, p.Hkv.d, D, V, p.window, p.first,
                  most, p.qstart ? p.max_seq : p.N, !p.qstart, q8 ? 1.0 : (double)bi::elem_size(dtype)};
  Plan s = plan(c, k);
  if (!ws || (uintptr_t)ws % 16 || ws_bytes < s.bytes) s = Plan{};
  if (ws_bytes < s.workspace()) s.laid = 0;
  // What is walked whole.
  const bool whole = most * p.G.d > s.split_cols;
  // Eight waves share their keys' and values' loads and addresses where that
  // leaves a workgroup for every compute unit and the walk is long (4096
  // tokens over 8192 keys 476 us, 510 with two workgroups of four; 4096 alone
  // 174 and 189). Over a short one a second workgroup, which starts while the
  // first works, gains more: 2048 tokens alone 76 us with eight, 71 with
  // twice four; 8192 under a window of 64 73 and 63, of 512 135 and 131, of
  // 1024 197 and 201. With fewer columns four waves fill more (two chunks of
  // 511 tokens beside 30 decodes 161 us, 175 with eight), two workgroups to a
  // compute unit where there are more than these.
  const int64_t cols = p.qstart ? (int64_t)p.T * p.G.d : (int64_t)p.R * p.qL * p.G.d;
  const int cus = bi::device_cus();
  // Rows that a tile walks, on average: 64 tokens see 63 more than the window.
  const int64_t longest = p.qstart ? p.max_seq : p.N;
  const int64_t seen = (int64_t)p.window + p.first + 63, causal = longest - most / 2;
  const bool far = (p.window && seen < causal ? seen : causal) > 1024;
  const Kernel whole8 = s.laid ? k.laid8 : k.whole8, whole4 = s.laid ? k.laid4 : k.whole4;
  const bool eight = whole8 && far && cols / 256 * p.Hkv.d >= cus;
  const bool pair = !eight && k.whole4_pair && cols / 128 * p.Hkv.d > cus;
  const int64_t wc = eight ? 256 : 128, threads = eight || s.laid ? 512 : pair ? 256 : k.whole4_threads;
  // Column tiles: every request with tokens may end in a part of one.
  const int64_t requests = p.T < p.R ? p.T : p.R;
  const int64_t tiles = !whole ? 0 : p.qstart ? cols / wc + requests
                                              : (int64_t)p.R * (((int64_t)p.qL * p.G.d + wc - 1) / wc);
  const int32_t fill = p.qstart && !s.split_cols ? 16 : 0;
  const int64_t blocks = tiles * p.Hkv.d + fill;
  // Beside rows laid out, requests that are not: of one column tile, or for which there
  // may be no room, each of which has more than split_cols columns (a launch that finds
  // nothing takes some 4 us).
  const int64_t least = s.split_cols / p.G.d + 1, n = p.T / least < p.R ? p.T / least : p.R;
  const bool more = whole && s.laid && s.room && (s.split_cols < 128 || n * p.Hkv.d * s.walked > s.room);
  const int64_t rest = more ? (cols / 128 + requests) * p.Hkv.d : 0;
  if (bi::grid_too_large(blocks, threads) || bi::grid_too_large(rest, k.whole4_threads))
    return bi::fail(BI_EINVAL, "%s: grid too large", who);
  hipError_t e;
  if (s.split_cols) {
    p.split_cols = (int32_t)s.split_cols;
    p.ccap = make_div(s.ccap);
    p.cstep = make_div(most * p.G.d > s.split_cols && p.G.d < s.ccap ? (int64_t)p.G.d : s.ccap);
    p.nseg = make_div(s.nseg);
    p.reqs = make_div(p.R);
    p.nc = (int32_t)s.nc;
    p.po = static_cast<float*>(ws);
    p.pml = reinterpret_cast<float2*>(p.po + (int64_t)p.R * p.Hkv.d * s.ccap * s.nseg * V);
    const int64_t ctiles = (s.ccap + s.nc - 1) / s.nc;
    p.ctiles = make_div(ctiles);
    p.gseg = make_div(s.gseg);
    p.slots = make_div(p.R * s.gseg);
    // (Beside larger requests split ones mostly have one column tile.)
    p.once = ctiles == 1 || most * p.G.d > s.split_cols;
    const Kernel split = most > 1 ? (s.nc == 16 ? k.split16 : k.split32)
                                  : (s.nc == 16 ? k.split16_one : k.split32_one);
    int64_t grid = split_grid(c, s);
    if (p.eight.d) grid = (grid / p.Hkv.d + 7) / 8 * 8 * p.Hkv.d;
    hipLaunchKernelGGL(split, dim3((unsigned)grid), dim3(256), 0, st, p);
    if ((e = hipGetLastError()) != hipSuccess) return bi::launch_error(e, who);
    p.fill_blocks = p.qstart ? 16 : 0;
    const int64_t waves = (int64_t)p.R * p.Hkv.d * p.cstep.d;
    hipLaunchKernelGGL(k.combine, dim3((unsigned)((waves + 3) / 4 + p.fill_blocks)), dim3(256), 0,
                       st, p);
    if ((e = hipGetLastError()) != hipSuccess) return bi::launch_error(e, who);
  }
  p.fill_blocks = fill;
  if (blocks) {
    if (s.laid && whole) {
      p.laid = static_cast<char*>(ws) + s.laid_at();
      p.units = (int32_t)s.units;
      p.room = (int32_t)(s.room ? s.room : (int64_t)p.R * p.Hkv.d * s.units);
      p.laid_cols = p.split_cols;
      if (s.room) {
        if (p.laid_cols < 128) p.laid_cols = 128;
        p.laid_at = reinterpret_cast<int32_t*>(p.laid);
        p.laid += notes(p.R);
      }
      const int64_t most_groups = 8 * (int64_t)cus;
      hipLaunchKernelGGL(k.lay, dim3((unsigned)(p.room < most_groups ? p.room : most_groups)), dim3(256), 0, st, p);
      if ((e = hipGetLastError()) != hipSuccess) return bi::launch_error(e, who);
    }
    hipLaunchKernelGGL(eight ? whole8 : pair ? k.whole4_pair : whole4, dim3((unsigned)blocks),
                       dim3((unsigned)threads), 0, st, p);
    if ((e = hipGetLastError()) != hipSuccess) return bi::launch_error(e, who);
    if (more) {
      p.fill_blocks = 0;
      hipLaunchKernelGGL(k.whole4, dim3((unsigned)rest), dim3(k.whole4_threads), 0, st, p);
      if ((e = hipGetLastError()) != hipSuccess) return bi::launch_error(e, who);
    }
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

// What bi_paged_attention and bi_paged_attention_q8 (`scale_strides`) share.
int paged_attention(const char* who, const void* q, const void* k_cache, const void* v_cache,
                    const float* k_scales, const float* v_scales, const int32_t* block_tables,
                    const int32_t* query_start, const int32_t* seq_lens, const void* sinks, void* out,
                    int64_t T, int64_t R, int64_t H, int64_t Hkv, int64_t D, int64_t V,
                    int64_t num_pages, int64_t page_size, int64_t W, const int64_t* strides,
                    const int64_t* scale_strides, float scale, int64_t window, int64_t sink_tokens,
                    int64_t max_query, int64_t max_seq, int dtype, bool q8, void* workspace,
                    int64_t workspace_bytes, void* hip_stream) {
  int rc = check(who, H, Hkv, D, V, scale, window, sink_tokens, dtype);
  if (rc) return rc;
  if (q8 && dtype == BI_F32)
    return bi::fail(BI_EUNSUPPORTED, "%s: fp32 queries over a cache of 8 bits are not built (f16 and "
                    "bf16 are)", who);
  if (T < 0 || R < 0 || num_pages < 0 || page_size <= 0 || W < 0 || max_query < 0 || max_seq < 0 ||
      T > kMost || T * H > INT32_MAX || R > kMost || num_pages > INT32_MAX || page_size > INT32_MAX ||
      W > INT32_MAX)
    return bi::fail(BI_EINVAL, "%s: bad sizes T=%lld R=%lld pages=%lld x %lld W=%lld", who,
                    (long long)T, (long long)R, (long long)num_pages, (long long)page_size,
                    (long long)W);
  if (T == 0) return BI_OK;
  if (!q || !out || !query_start || (R > 0 && !seq_lens) || !strides ||
      (R > 0 && W > 0 && !block_tables) || (num_pages > 0 && (!k_cache || !v_cache)) ||
      (q8 && (!scale_strides || (num_pages > 0 && (!k_scales || !v_scales)))))
    return bi::fail(BI_EINVAL, "%s: null pointer", who);
  const int esz = bi::elem_size(dtype);
  if (!aligned16(q, nullptr, nullptr, strides, 2, esz) ||
      !aligned16(nullptr, k_cache, v_cache, strides + 2, 6, q8 ? 1 : esz))
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
  if (q8) {
    if (((uintptr_t)k_scales | (uintptr_t)v_scales) % 4)
      return bi::fail(BI_EINVAL, "%s: scales not aligned to elements", who);
    // Pages and rows, whose numbers a kernel multiplies row by row, in 32 bits.
    uint32_t* const to[8] = {&p.k8b, &p.k8n, &p.v8b, &p.v8n, &p.ksb, &p.ksn, &p.vsb, &p.vsn};
    const int64_t from[8] = {strides[2], strides[4], strides[5], strides[7], scale_strides[0] * 4,
                             scale_strides[2] * 4, scale_strides[3] * 4, scale_strides[5] * 4};
    for (int i = 0; i < 8; i++) {
      if (from[i] < 0 || from[i] > UINT32_MAX)
        return bi::fail(BI_EUNSUPPORTED, "%s: pages and rows lie less than 4 GiB apart", who);
      *to[i] = (uint32_t)from[i];
    }
    p.ks = k_scales;
    p.vs = v_scales;
    p.ksh = scale_strides[1], p.vsh = scale_strides[4];
    if (Hkv > 1 && D + V <= 256 && strides[3] < strides[4]) p.eight = make_div(8 * Hkv);
  }
  return launch(who, p, D, V, dtype, q8, workspace, workspace_bytes, hip_stream);
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
  return paged_attention("bi_paged_attention", q, k_cache, v_cache, nullptr, nullptr, block_tables,
                         query_start, seq_lens, sinks, out, T, R, H, Hkv, D, V, num_pages, page_size, W,
                         strides, nullptr, scale, window, sink_tokens, max_query, max_seq, dtype, false,
                         workspace, workspace_bytes, hip_stream);
}

extern "C" int64_t bi_paged_attention_workspace(int64_t T, int64_t R, int64_t H, int64_t Hkv,
                                                int64_t D, int64_t V, int64_t window,
                                                int64_t sink_tokens, int64_t max_query,
                                                int64_t max_seq, int dtype) {
  if (T <= 0 || R <= 0 || H <= 0 || Hkv <= 0 || H > 65535 || H % Hkv || !bi::elem_size(dtype) ||
      !dims_built(D, V) || T > kMost || R > kMost || window < 0 || sink_tokens < 0)
    return 0;
  const Call c = {R, T, H / Hkv, Hkv, D, V, clamp32(window), clamp32(sink_tokens), clamp32(max_query),
                  clamp32(max_seq), false, (double)bi::elem_size(dtype)};
  return plan(c, kernels(D, V, dtype, false)).bytes;
}

extern "C" int bi_paged_attention_q8(const void* q, const int8_t* k_cache, const int8_t* v_cache,
                                     const float* k_scales, const float* v_scales,
                                     const int32_t* block_tables, const int32_t* query_start,
                                     const int32_t* seq_lens, const void* sinks, void* out, int64_t T,
                                     int64_t R, int64_t H, int64_t Hkv, int64_t D, int64_t V,
                                     int64_t num_pages, int64_t page_size, int64_t W,
                                     const int64_t* strides,
                                     const int64_t* scale_strides, float scale, int64_t window,
                                     int64_t sink_tokens, int64_t max_query, int64_t max_seq,
                                     int dtype, void* workspace, int64_t workspace_bytes,
                                     void* hip_stream) {
  return paged_attention("bi_paged_attention_q8", q, k_cache, v_cache, k_scales, v_scales, block_tables,
                         query_start, seq_lens, sinks, out, T, R, H, Hkv, D, V, num_pages, page_size, W,
                         strides, scale_strides, scale, window, sink_tokens, max_query, max_seq, dtype,
                         true, workspace, workspace_bytes, hip_stream);
}

namespace {

Plan q8_plan(int64_t T, int64_t R, int64_t H, int64_t Hkv, int64_t D, int64_t V, int64_t window,
             int64_t sink_tokens, int64_t max_query, int64_t max_seq, int dtype) {
  if (T <= 0 || R <= 0 || H <= 0 || Hkv <= 0 || H > 65535 || H % Hkv || (dtype != BI_F16 && dtype != BI_BF16) ||
      !dims_built(D, V) || T > kMost || R > kMost || window < 0 || sink_tokens < 0)
    return Plan{};
  const Call c = {R, T, H / Hkv, Hkv, D, V, clamp32(window), clamp32(sink_tokens), clamp32(max_query),
                  clamp32(max_seq), false, 1.0};
  return plan(c, kernels(D, V, dtype, true));
}

}  // namespace

extern "C" int64_t bi_paged_attention_q8_workspace(int64_t T, int64_t R, int64_t H, int64_t Hkv,
                                                   int64_t D, int64_t V, int64_t window,
                                                   int64_t sink_tokens, int64_t max_query,
                                                   int64_t max_seq, int dtype) {
  return q8_plan(T, R, H, Hkv, D, V, window, sink_tokens, max_query, max_seq, dtype).workspace();
}

extern "C" int64_t bi_paged_attention_q8_least_workspace(int64_t T, int64_t R, int64_t H, int64_t Hkv,
                                                         int64_t D, int64_t V, int64_t window,
                                                         int64_t sink_tokens, int64_t max_query,
                                                         int64_t max_seq, int dtype) {
  return q8_plan(T, R, H, Hkv, D, V, window, sink_tokens, max_query, max_seq, dtype).bytes;
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
  return launch(who, p, D, V, dtype, false, workspace, workspace_bytes, hip_stream);
}

extern "C" int64_t bi_window_attention_workspace(int64_t B, int64_t H, int64_t Hkv, int64_t qL,
                                                 int64_t N, int64_t D, int64_t V, int64_t window,
                                                 int64_t sink_tokens, int dtype) {
  if (B <= 0 || H <= 0 || Hkv <= 0 || H > 65535 || H % Hkv || qL <= 0 || N <= 0 || !bi::elem_size(dtype) ||
      !dims_built(D, V) || qL > kMost || N > kMost || B > kMost || window < 0 || sink_tokens < 0)
    return 0;
  const Call c = {B, B * qL, H / Hkv, Hkv, D, V, clamp32(window), clamp32(sink_tokens), qL, N, true,
                  (double)bi::elem_size(dtype)};
  return plan(c, kernels(D, V, dtype, false)).bytes;
}
