// Attention over a paged cache of 8 bits for D = 96, V = 96 (bi_paged_q8_attn_kernel.h).
#include "bi_paged_q8_attn_kernel.h"

BI_PAGED_Q8_KERNELS(96, 96)
