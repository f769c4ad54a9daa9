// The attention kernels of four_attend.cuh for float.
#include "four_attend.cuh"

int xnor::launch_attend_f32(const AttendParams & p, const AttendPlan & plan, cudaStream_t stream) { return launch_attend_shape<float>(p, plan, stream); }
