// The walk's builds with 4 scales to a chunk of 128 columns (groups of 32).
#include "ftk_w4_walk.h"

namespace ftk {

hipError_t launch_w4_s4(const W4Args& a, const W4Shape& s, hipStream_t stream) {
  return w4::launch_shape<4>(a, s, stream);
}

}  // namespace ftk
