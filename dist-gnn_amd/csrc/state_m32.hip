// state_m32.hip -- the matrix form of the attention over the state cache, channel groups of 32.
#include "dgs_attend.cuh"

namespace dgs {

void attend_matrix_32(const AttendArgs &a, int waves, int type, hipStream_t st) {
  switch (a.c.dim / 32) {
    case 1: launch_matrix<1, 32>(a, waves, type, st); break;
    case 2: launch_matrix<2, 32>(a, waves, type, st); break;
    case 4: launch_matrix<4, 32>(a, waves, type, st); break;
    default: throw Error("attend: no matrix form for this head_dim and group");
  }
}

}  // namespace dgs
