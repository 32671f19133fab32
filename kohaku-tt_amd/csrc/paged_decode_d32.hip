// Attention over a paged cache, padded head dim 32 (kernels in paged_decode.hpp).
#include "paged_decode.hpp"

namespace kmi {
namespace paged {
template hipError_t launch_decode<bf16, 32>(const AttnParams&, int, bool, hipStream_t);
template hipError_t launch_decode<f16, 32>(const AttnParams&, int, bool, hipStream_t);
}  // namespace paged
}  // namespace kmi
