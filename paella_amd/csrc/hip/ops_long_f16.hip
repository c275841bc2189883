// Attention over picked pages and the weights that tokens gather, fp16 (long_attention.h).
#include "long_attention.h"

namespace paella {
PageAttentionKernel page_attention_f16(int dim) { return page_attention_kernel_of<F16>(dim); }
WeighKernel key_sums_f16(int dim, bool few) { return key_sums<F16>(dim, few); }
WeighKernel key_weights_f16(int dim, bool few) { return key_weights<F16>(dim, few); }
}  // namespace paella
