// pct_policy.cuh -- what the policy operators' translation units share: element types, mask entries, wavefront reductions.
#ifndef PCT_POLICY_CUH
#define PCT_POLICY_CUH
#include <hip/hip_runtime.h>
#include <stdint.h>

#include "../../include/pct_env.h"
#include "../../include/pct_policy.h"

namespace pct {

int policy_fail(int code, const char* text);  // pct_env.hip: the text behind pct_last_error()
int policy_launched(const char* what);        // the launch error of the calling thread, as a status

using bf16 = __bf16;
using f16 = _Float16;

constexpr float kLog2e = 1.44269504088896340736f, kLn2 = 0.69314718055994530942f;

// loads and stores of 16 (8) bytes where only the element's own alignment is known: the hardware takes any address
struct __attribute__((packed, aligned(1))) Bytes8 { uint32_t w[2]; };
struct __attribute__((packed, aligned(2))) Half8 { uint32_t w[4]; };
struct __attribute__((packed, aligned(4))) Float8 { uint32_t w[8]; };

template <typename T> struct Vec8 { using raw = Half8; };
template <> struct Vec8<float> { using raw = Float8; };

template <typename T>
__device__ __forceinline__ void unpack8(const typename Vec8<T>::raw& r, float (&o)[8]) {
  if constexpr (sizeof(T) == 4) {
#pragma unroll
    for (int i = 0; i < 8; i++) o[i] = __uint_as_float(r.w[i]);
  } else {
#pragma unroll
    for (int i = 0; i < 4; i++) {
      if constexpr (__is_same(T, bf16)) {
        o[2 * i] = __uint_as_float(r.w[i] << 16);
        o[2 * i + 1] = __uint_as_float(r.w[i] & 0xffff0000u);
      } else {
        o[2 * i] = (float)__builtin_bit_cast(f16, (uint16_t)(r.w[i] & 0xffffu));
        o[2 * i + 1] = (float)__builtin_bit_cast(f16, (uint16_t)(r.w[i] >> 16));
      }
    }
  }
}

template <typename T>
__device__ __forceinline__ void load8(const T* p, float (&o)[8]) { unpack8<T>(*(const typename Vec8<T>::raw*)p, o); }

// two values rounded to nearest even and packed
template <typename T>
__device__ __forceinline__ uint32_t pack2(float a, float b) {
  typedef float f2 __attribute__((ext_vector_type(2)));
  typedef T t2 __attribute__((ext_vector_type(2)));
  f2 v = {a, b};
  return __builtin_bit_cast(uint32_t, __builtin_convertvector(v, t2));
}

template <typename T>
__device__ __forceinline__ void store8(T* p, const float (&v)[8]) {
  typename Vec8<T>::raw r;
  if constexpr (sizeof(T) == 4) {
#pragma unroll
    for (int i = 0; i < 8; i++) r.w[i] = __float_as_uint(v[i]);
  } else {
#pragma unroll
    for (int i = 0; i < 4; i++) r.w[i] = pack2<T>(v[2 * i], v[2 * i + 1]);
  }
  *(typename Vec8<T>::raw*)p = r;
}

// a mask entry of any type: a zero float of either sign forbids
struct Mask {
  const void* p;
  int64_t row, col;
  int type;
  __device__ __forceinline__ bool at(int64_t r, int64_t c) const {
    const int64_t o = r * row + c * col;
    if (type == PCT_MASK_U8) return ((const uint8_t*)p)[o] != 0;
    if (type == PCT_MASK_F16) return (((const uint16_t*)p)[o] & 0x7fffu) != 0;
    const uint32_t w = ((const uint32_t*)p)[o];
    return (type == PCT_MASK_F32 ? w << 1 : w) != 0;
  }
};

// ---- reductions over the 64 lanes, by the data-parallel primitives (no LDS): the result stands in every lane ----
template <int CTRL, int ROWS, typename F>
__device__ __forceinline__ float dpp_step(float v, float idle, F f) {
  return f(v, __int_as_float(__builtin_amdgcn_update_dpp(__float_as_int(idle), __float_as_int(v), CTRL, ROWS, 0xf, false)));
}
__device__ __forceinline__ float lane63(float v) { return __int_as_float(__builtin_amdgcn_readlane(__float_as_int(v), 63)); }

template <typename F>
__device__ __forceinline__ float wave_reduce(float v, float idle, F f) {
  v = dpp_step<0x111, 0xf>(v, idle, f);  // row_shr 1, 2, 4, 8: the last lane of each row of 16 holds the row's
  v = dpp_step<0x112, 0xf>(v, idle, f);
  v = dpp_step<0x114, 0xf>(v, idle, f);
  v = dpp_step<0x118, 0xf>(v, idle, f);
  v = dpp_step<0x142, 0xa>(v, idle, f);  // row_bcast 15, 31
  v = dpp_step<0x143, 0xc>(v, idle, f);
  return lane63(v);
}
__device__ __forceinline__ float wave_sum(float v) { return wave_reduce(v, 0.f, [](float a, float b) { return a + b; }); }
__device__ __forceinline__ float wave_max(float v) { return wave_reduce(v, -INFINITY, [](float a, float b) { return fmaxf(a, b); }); }

template <int CTRL, int ROWS>
__device__ __forceinline__ uint64_t dpp_max_u64(uint64_t v) {
  const uint32_t lo = __builtin_amdgcn_update_dpp(0, (int)(uint32_t)v, CTRL, ROWS, 0xf, false);
  const uint32_t hi = __builtin_amdgcn_update_dpp(0, (int)(uint32_t)(v >> 32), CTRL, ROWS, 0xf, false);
  const uint64_t o = ((uint64_t)hi << 32) | lo;
  return o > v ? o : v;
}
__device__ __forceinline__ uint64_t readlane_u64(uint64_t v, int lane) {
  const uint32_t lo = __builtin_amdgcn_readlane((int)(uint32_t)v, lane), hi = __builtin_amdgcn_readlane((int)(uint32_t)(v >> 32), lane);
  return ((uint64_t)hi << 32) | lo;
}
__device__ __forceinline__ uint64_t wave_max_u64(uint64_t v) {  // (0 is the idle value)
  v = dpp_max_u64<0x111, 0xf>(v);
  v = dpp_max_u64<0x112, 0xf>(v);
  v = dpp_max_u64<0x114, 0xf>(v);
  v = dpp_max_u64<0x118, 0xf>(v);
  v = dpp_max_u64<0x142, 0xa>(v);
  v = dpp_max_u64<0x143, 0xc>(v);
  return readlane_u64(v, 63);
}

}  // namespace pct
#endif
