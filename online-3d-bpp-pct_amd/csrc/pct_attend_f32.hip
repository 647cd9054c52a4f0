// pct_attend_f32.hip -- the attention kernels (pct_attend.cuh) for one element type.
#include "pct_attend.cuh"

namespace pct {
int64_t attend_workspace_f32(const AttendParams& p, bool backward) { return Attend<float>::workspace(p, backward); }
int attend_forward_f32(AttendParams& p, char* ws, hipStream_t s) { return Attend<float>::forward(p, ws, s); }
int attend_backward_f32(AttendParams& p, char* ws, hipStream_t s) { return Attend<float>::backward(p, ws, s); }
}  // namespace pct
