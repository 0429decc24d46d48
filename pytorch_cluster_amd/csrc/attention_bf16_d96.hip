// Attention kernels: bf16, heads of up to 96.
#include "attention_impl.hpp"

namespace pca {
hipError_t attention_bf16_d96(const AttentionCall &c, int pass, int rows,
                              hipStream_t stream) {
  return attn::launch<__bf16, 96>(c, pass, rows, stream);
}
} // namespace pca
