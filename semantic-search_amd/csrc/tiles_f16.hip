// The matrix products of float16 operands.
#include <math.h>

#include "tiles.h"

namespace ssmap {

template void launch_product<SSMAP_F16, SSMAP_F16>(Product, hipStream_t);
template void launch_product<SSMAP_F16, SSMAP_F32>(Product, hipStream_t);

}  // namespace ssmap
