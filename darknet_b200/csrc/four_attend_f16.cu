// The attention kernels of four_attend.cuh for __half.
#include "four_attend.cuh"

int xnor::launch_attend_f16(const AttendParams & p, const AttendPlan & plan, cudaStream_t stream) { return launch_attend_shape<__half>(p, plan, stream); }
