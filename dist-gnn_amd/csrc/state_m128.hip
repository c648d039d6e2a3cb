// state_m128.hip -- the matrix form of the attention over the state cache, channel groups of 128.
#include "dgs_attend.cuh"

namespace dgs {

void attend_matrix_128(const AttendArgs &a, int waves, int type, hipStream_t st) {
  switch (a.c.dim / 128) {
    case 1: launch_matrix<1, 128>(a, waves, type, st); break;
    case 2: launch_matrix<2, 128>(a, waves, type, st); break;
    default: throw Error("attend: no matrix form for this head_dim and group");
  }
}

}  // namespace dgs
