// linear_pipe_f8.hip -- the fp8 e4m3 instances of linear_pipe.h
#include "linear_pipe.h"

namespace ascq {

hipError_t launch_linear_pipe_f8(const LinearArgs& a, hipStream_t st)
{
    return a.w_trans ? launch_linear_layout<OP_F8, false>(a, st) : launch_linear_layout<OP_F8, true>(a, st);
}

}  // namespace ascq
