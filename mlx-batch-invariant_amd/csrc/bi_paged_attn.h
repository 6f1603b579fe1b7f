// Attention over a paged cache, or over contiguous keys with a window: launch
// arguments shared by the kernels (bi_paged_attn_kernel.h) and the C entry
// points (bi_paged_attn.hip).
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

#include "bi_div.h"
#include "bi_internal.h"

namespace bi_paged {

using bi::Div;
using bi::make_div;

struct Args {
  const void* q;
  const void* k;
  const void* v;
  const void* sinks;
  void* out;
  const int32_t* table;   // (R, W)
  const int32_t* qstart;  // (R + 1); NULL: contiguous keys, qL tokens and N rows each
  const int32_t* seq;     // (R)
  int64_t qb, qt, qh;     // q element strides: request (contiguous only), token, head
  int64_t ob, ot, oh;     // out
  int64_t kb, kh, kn;     // keys: page or request, head, row
  int64_t vb, vh, vn;
  int64_t table_stride;
  int32_t R, H, W, pages;
  Div Hkv, G, page;       // G: query heads of a kv head
  int32_t qL, N;          // contiguous
  int32_t T;              // tokens of a paged call
  int32_t window, first;  // window 0: none
  int32_t max_query, max_seq;
  float scale2;           // |scale| * log2(e)
  uint32_t qsign;         // negative scale: the sign bits of a query dword
  // The split route: partial results of (request, kv head, segment, column).
  float* po;              // [V] each
  float2* pml;            // base and sum
  Div nseg, ccap;         // segments and columns kept per (request, kv head)
  Div gseg;               // workgroups for a request's segments, which each takes in turn
  Div cstep;              // columns between those that a wave folds
  Div reqs;               // R
  int32_t nc;             // columns per workgroup, 16 or 32
  Div ctiles;             // workgroups of them
  Div slots;              // R * gseg
  int32_t once;           // keys and values are read by one of these only
  int32_t split_cols;     // requests of at most this many columns are split
  int32_t fill_blocks;    // workgroups that fill tokens no kernel computes
};

typedef void (*Kernel)(Args);
struct Kernels {
  Kernel split16, split32;  // 16 or 32 columns per workgroup
  Kernel split16_one, split32_one;  // where no request has more than one token
  Kernel combine;
  // 4 or 8 waves of 32 columns per workgroup, one to a CU, or 4 waves two to a
  // CU (the last two where the registers allow two waves per SIMD, else NULL).
  Kernel whole4, whole8, whole4_pair;
  int whole4_threads;       // its loading waves among them
  int seg, pass;            // rows per segment and per pass of the split route (four steps)
  // For the choice of route, in microseconds: what a row costs a whole
  // workgroup, and a full segment the split ones of 16 and 32 columns that a
  // CU runs together, per_cu of them.
  double row_us, seg16_us, seg32_us;
  int per_cu16, per_cu32;
};

#define BI_PAGED_DIM_PAIRS(X) X(64, 64) X(96, 96) X(128, 128) X(192, 128) X(192, 192) X(256, 256)
#define BI_PAGED_DECLARE(D, V) Kernels kernels_d##D##_v##V(int dtype);
BI_PAGED_DIM_PAIRS(BI_PAGED_DECLARE)
#undef BI_PAGED_DECLARE

}  // namespace bi_paged
