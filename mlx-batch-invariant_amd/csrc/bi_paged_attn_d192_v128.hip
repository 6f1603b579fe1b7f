// Paged and windowed attention for D = 192, V = 128 (bi_paged_attn_kernel.h).
#include "bi_paged_attn_kernel.h"

BI_PAGED_KERNELS(192, 128)
