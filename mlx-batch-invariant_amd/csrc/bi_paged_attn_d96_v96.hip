// Paged and windowed attention for D = 96, V = 96 (bi_paged_attn_kernel.h).
#include "bi_paged_attn_kernel.h"

BI_PAGED_KERNELS(96, 96)
