// Attention over a paged cache, or over contiguous keys with a window: launch
// arguments and the visibility rule shared by its kernels.
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

#include "bi_internal.h"

namespace bi_paged {

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
  int32_t R, H, Hkv, G, W, page, pages;
  int32_t qL, N;          // contiguous
  int32_t T;              // tokens of a paged call
  int32_t window, first;  // window 0: none
  int32_t max_query, max_seq;
  float scale2;           // |scale| * log2(e)
  uint32_t qneg;          // nonzero: negate the scores
};

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

__device__ __forceinline__ bool sees(const Args& p, int32_t pos, int32_t key) {
  return key <= pos && (p.window == 0 || key > pos - p.window || key < p.first);
}

}  // namespace bi_paged
