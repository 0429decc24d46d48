// Attention kernels: f16, heads of up to 128.
#include "attention_impl.hpp"

namespace pca {
hipError_t attention_f16_d128(const AttentionCall &c, int pass, int rows,
                              hipStream_t stream) {
  return attn::launch<_Float16, 128>(c, pass, rows, stream);
}
} // namespace pca
