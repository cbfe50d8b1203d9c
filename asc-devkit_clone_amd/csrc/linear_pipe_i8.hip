// linear_pipe_i8.hip -- the int8 instances of linear_pipe.h
#include "linear_pipe.h"

namespace ascq {

hipError_t launch_linear_pipe_i8(const LinearArgs& a, hipStream_t st)
{
    return a.w_trans ? launch_linear_layout<OP_I8, false>(a, st) : launch_linear_layout<OP_I8, true>(a, st);
}

}  // namespace ascq
