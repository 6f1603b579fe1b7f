// Paged and windowed attention for D = 64, V = 64 (bi_paged_attn_kernel.h).
#include "bi_paged_attn_kernel.h"

BI_PAGED_KERNELS(64, 64)
