// Paged and windowed attention for D = 256, V = 256 (bi_paged_attn_kernel.h).
#include "bi_paged_attn_kernel.h"

BI_PAGED_KERNELS(256, 256)
