// proj4_g0.hip -- MXFP4 projections (proj4_impl.hpp).
#include "proj4_impl.hpp"

namespace grim {
GRIM_PROJ4(0)
}  // namespace grim
