// proj4_g128.hip -- INT4 projections in groups of 128 and 256 (proj4_impl.hpp).
#include "proj4_impl.hpp"

namespace grim {
GRIM_PROJ4(128)
}  // namespace grim
