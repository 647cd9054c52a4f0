// pct_attend_f16.hip -- the attention kernels (pct_attend.cuh) for one element type.
#include "pct_attend.cuh"

namespace pct {
int64_t attend_workspace_f16(const AttendParams& p, bool backward) { return Attend<f16>::workspace(p, backward); }
int attend_forward_f16(AttendParams& p, char* ws, hipStream_t s) { return Attend<f16>::forward(p, ws, s); }
int attend_backward_f16(AttendParams& p, char* ws, hipStream_t s) { return Attend<f16>::backward(p, ws, s); }
}  // namespace pct
