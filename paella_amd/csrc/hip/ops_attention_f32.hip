// Attention over a shared prefix, f32 (prefix_attention.h).
#include "prefix_attention.h"

namespace paella {
AttentionKernel attention_kernel_f32(int dim, int rp, int ro) { return attention_kernel<F32>(dim, rp, ro); }
AttentionKernel attention_join_f32(int dim) { return attention_join<F32>(dim); }
}  // namespace paella
