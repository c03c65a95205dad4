// The walk's builds with 1 scale to a chunk of 128 columns (groups of 128).
#include "ftk_w4_walk.h"

namespace ftk {

hipError_t launch_w4_s1(const W4Args& a, const W4Shape& s, hipStream_t stream) {
  return w4::launch_shape<1>(a, s, stream);
}

}  // namespace ftk
