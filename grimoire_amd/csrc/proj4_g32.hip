// proj4_g32.hip -- INT4 projections in groups of 32 (proj4_impl.hpp).
#include "proj4_impl.hpp"

namespace grim {
GRIM_PROJ4(32)
}  // namespace grim
