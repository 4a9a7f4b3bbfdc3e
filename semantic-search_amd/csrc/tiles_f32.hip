// The matrix products of float32 operands.
#include <math.h>

#include "tiles.h"

namespace ssmap {

template void launch_product<SSMAP_F32, SSMAP_F32>(Product, hipStream_t);

}  // namespace ssmap
