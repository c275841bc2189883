// Attention over a shared prefix, f16 (prefix_attention.h).
#include "prefix_attention.h"

namespace paella {
AttentionKernel attention_kernel_f16(int dim, int rp, int ro) { return attention_kernel<F16>(dim, rp, ro); }
AttentionKernel attention_join_f16(int dim) { return attention_join<F16>(dim); }
}  // namespace paella
