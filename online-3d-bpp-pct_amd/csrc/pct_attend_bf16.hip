// pct_attend_bf16.hip -- the attention kernels (pct_attend.cuh) for one element type.
#include "pct_attend.cuh"

namespace pct {
int64_t attend_workspace_bf16(const AttendParams& p, bool backward) { return Attend<bf16>::workspace(p, backward); }
int attend_forward_bf16(AttendParams& p, char* ws, hipStream_t s) { return Attend<bf16>::forward(p, ws, s); }
int attend_backward_bf16(AttendParams& p, char* ws, hipStream_t s) { return Attend<bf16>::backward(p, ws, s); }
}  // namespace pct
