// Attention over a shared prefix, bf16 (prefix_attention.h).
#include "prefix_attention.h"

namespace paella {
AttentionKernel attention_kernel_bf16(int dim, int rp, int ro) { return attention_kernel<Bf16>(dim, rp, ro); }
AttentionKernel attention_join_bf16(int dim) { return attention_join<Bf16>(dim); }
}  // namespace paella
