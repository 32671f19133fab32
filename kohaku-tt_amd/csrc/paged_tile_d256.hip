// Attention over a paged cache on 32x32x16 MFMA tiles, padded head dim 256 (paged_tile.hpp).
#include "paged_tile.hpp"

namespace kmi {
namespace paged {
template hipError_t launch_tile<bf16, 256>(const AttnParams&, int, hipStream_t);
template hipError_t launch_tile<f16, 256>(const AttnParams&, int, hipStream_t);
}  // namespace paged
}  // namespace kmi
