// state_m64.hip -- the matrix form of the attention over the state cache, channel groups of 64.
#include "dgs_attend.cuh"

namespace dgs {

void attend_matrix_64(const AttendArgs &a, int waves, int type, hipStream_t st) {
  switch (a.c.dim / 64) {
    case 1: launch_matrix<1, 64>(a, waves, type, st); break;
    case 2: launch_matrix<2, 64>(a, waves, type, st); break;
    case 4: launch_matrix<4, 64>(a, waves, type, st); break;
    default: throw Error("attend: no matrix form for this head_dim and group");
  }
}

}  // namespace dgs
