// Attention over a paged cache of 8 bits for D = 192, V = 192 (bi_paged_q8_attn_kernel.h).
#include "bi_paged_q8_attn_kernel.h"

BI_PAGED_Q8_KERNELS(192, 192)
