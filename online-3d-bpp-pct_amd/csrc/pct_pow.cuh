// pct_pow.cuh -- `tri_base_len ** 2` of the lever rule.
//
// Reference: pct_envs/PctContinuous0/space.py:108,206 (PctDiscrete0/space.py:112,210): `tri_base_line /= tri_base_len ** 2`
// with tri_base_len an np.float64 -- NumPy's scalar power, which is the C library's pow(len, 2.0).  The library's pow is not
// correctly rounded: comparing its results with len * len shows another last bit on about 0.08 % of the lengths the
// continuous env produces, and on none of the lengths a discrete env of up to 43 units per axis can produce.  On the device
// the square is the correctly rounded one, so a stability verdict of the continuous env (or of a bin of more than 31 units per
// axis) that hangs on that bit may differ from a reference run; the host build of this source calls the library's function.
#ifndef PCT_POW_CUH
#define PCT_POW_CUH
#include <math.h>

namespace pct {

#if defined(__HIPCC__)
__device__ __forceinline__ double lever_square(double len) { return len * len; }
#else
static inline double pow_glibc_fma(double x, double y) {
  volatile double e = y;  // (a literal exponent of 2 would be folded into x * x)
  return ::pow(x, e);
}
static inline double lever_square(double len) { return pow_glibc_fma(len, 2.0); }
#endif

}  // namespace pct
#endif
