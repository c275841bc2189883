// Attention over picked pages and the weights that tokens gather, bf16 (long_attention.h).
#include "long_attention.h"

namespace paella {
PageAttentionKernel page_attention_bf16(int dim) { return page_attention_kernel_of<Bf16>(dim); }
WeighKernel key_sums_bf16(int dim, bool few) { return key_sums<Bf16>(dim, few); }
WeighKernel key_weights_bf16(int dim, bool few) { return key_weights<Bf16>(dim, few); }
}  // namespace paella
