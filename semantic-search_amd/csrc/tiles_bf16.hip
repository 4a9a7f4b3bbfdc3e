// The matrix products of bfloat16 operands.
#include <math.h>

#include "tiles.h"

namespace ssmap {

template void launch_product<SSMAP_BF16, SSMAP_BF16>(Product, hipStream_t);
template void launch_product<SSMAP_BF16, SSMAP_F32>(Product, hipStream_t);

}  // namespace ssmap
