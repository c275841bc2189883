// Attention over picked pages and the weights that tokens gather, fp32 (long_attention.h).
#include "long_attention.h"

namespace paella {
PageAttentionKernel page_attention_f32(int dim) { return page_attention_kernel_of<F32>(dim); }
WeighKernel key_sums_f32(int dim, bool few) { return key_sums<F32>(dim, few); }
WeighKernel key_weights_f32(int dim, bool few) { return key_weights<F32>(dim, few); }
}  // namespace paella
