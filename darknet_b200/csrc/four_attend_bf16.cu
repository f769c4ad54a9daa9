// The attention kernels of four_attend.cuh for __nv_bfloat16.
#include "four_attend.cuh"

int xnor::launch_attend_bf16(const AttendParams & p, const AttendPlan & plan, cudaStream_t stream) { return launch_attend_shape<__nv_bfloat16>(p, plan, stream); }
