// Attention kernels: f32, heads of up to 128.
#include "attention_impl.hpp"

namespace pca {
hipError_t attention_f32_d128(const AttentionCall &c, int pass, int rows,
                              hipStream_t stream) {
  return attn::launch<float, 128>(c, pass, rows, stream);
}
} // namespace pca
