// Attention over a shared prefix, f32 (prefix_attention.h).
#include "prefix_attention.h"

namespace paella {
AttentionKernel attention_kernel_f32(int dim, int rp, int ro) { return attention_kernel<F32>(dim, rp, ro); }
}  // namespace paella
