// proj4_g64.hip -- INT4 projections in groups of 64 (proj4_impl.hpp).
#include "proj4_impl.hpp"

namespace grim {
GRIM_PROJ4(64)
}  // namespace grim
