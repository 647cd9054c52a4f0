// pct_attend.cuh -- attention of the queries of a batch to its allowed keys, and the gradients.
//
// For the rows r = (l, g) of one key/value head (g counts the heads that share it), over the n allowed keys j of the batch:
//     S_rj = q_r . k_j,  P_rj = e^(scale S_rj) / sum_j e^(scale S_rj),  O_r = sum_j P_rj v_j   (n = 0: O = 0, no gradients)
//     D_r = dO_r . O_r = sum_j P_rj dP_rj,  dP_rj = dO_r . v_j,  dS_rj = P_rj (dP_rj - D_r),
//     dq_r = scale sum_j dS_rj k_j,   dk_j = scale sum_r dS_rj q_r,   dv_j = sum_r P_rj dO_r.
//
// A mask allows a key for every query of its batch, so the allowed keys are listed once (pct_attend_list_kernel) and only they
// are read: the work falls with their share, nothing masked is multiplied, and a value that must not count is never loaded.
//
// One layout carries the three kernels.  A wavefront keeps 32 "resident" rows, one to a lane column (rows of q in the forward
// and the dq kernel, keys in the dk/dv kernel), and walks over tiles of "streamed" rows that the workgroup stages in LDS.  With
// 32x32x16 matrix instructions a product streamed x resident^T leaves in lane (c, h) = (lane % 32, lane / 32) column c and the
// rows {8 i + 4 h .. + 3}.  The second product contracts over these rows, and the order of a contraction is free as long as
// both operands share it: registers 8 b .. 8 b + 7 of the lane ARE its operand for the block of 16 rows b, where slot (h, e)
// means row 16 b + 8 (e / 4) + 4 h + e % 4.  So P and dS never pass through LDS or another lane; the other operand is read from
// the staged tile transposed (ds_read_b64_tr_b16), in that row order.  The sum of a row and its maximum are a lane's own
// registers and one exchange between the halves.
//
// float32 runs the same code with eight 32x32x2 instructions in place of one 32x32x16 (slot e of both halves each).
//
// Roundings: S, P, dP, dS, all sums and statistics are float32.  P and dS are rounded to the tensors' type as operands of the
// second product (half a step, as the result itself is); float32 tensors stay float32.  In float16, whose range is small, P
// carries a power of two, and dS one that follows the largest entry met so far (pct_attend: F16 below).
#ifndef PCT_ATTEND_CUH
#define PCT_ATTEND_CUH
#include <type_traits>

#include "pct_policy.cuh"

namespace pct {

// n / d for n < 2^31 by a multiplication: m = 2^32 (2^s - d) / d + 1 with s = ceil(log2 d)
struct Divisor {
  uint32_t d, m, s;
  Divisor() : d(1), m(1), s(0) {}
  explicit Divisor(uint32_t by) : d(by), s(0) {
    while (((uint64_t)1 << s) < by) s++;
    m = (uint32_t)((((uint64_t)1 << 32) * (((uint64_t)1 << s) - by)) / by + 1);
  }
  __device__ __forceinline__ uint32_t of(uint32_t n) const { return (__umulhi(m, n) + n) >> s; }
};

struct AttendParams {
  const void *q, *k, *v, *d_out, *o;
  int64_t qs[3], ks[3], vs[3], ds[3];  // batch, length, head
  const int32_t* list;                 // [batch, k_len + 1]: the count, the allowed keys, then the others
  const void* lengths;
  int lengths_type;
  int batch, q_len, k_len, heads, kv_heads, dim, group, rows;  // rows = q_len * group
  float scale, c;                      // c = scale log2 e
  int tiles, splits;                   // workgroups along the resident rows / along the streamed ones
  bool tail;                           // the last tiles may find nothing to do
  Divisor by_tiles, by_splits, by_kv, by_group, by_die;
  void* out;
  float2* stats;                       // [batch, kv_heads, rows]: reference point (log2), sum
  float* delta;                        // [batch, kv_heads, rows]
  void *dq, *dk, *dv;
  float* part;                         // splits > 1: float32 partial results
  float2* part_stats;
};

namespace {

constexpr float kLowest = -3.402823466e38f;
// What fills up a tile behind the last row: a row's second product meets P = 0 there, which must not make NaN of an infinite value.
__device__ uint4 kZeroRow[32];  // (128 float32)
template <typename T>
__device__ __forceinline__ const T* zero_row() {
  uint64_t p = (uint64_t)kZeroRow;
  asm volatile("" : "+s"(p));  // (asked for where it is used: kept in registers over a tile it costs a wavefront of 5 to a SIMD)
  return (const T*)p;
}

template <typename T> using Frag = T __attribute__((ext_vector_type(8)));
typedef float Acc __attribute__((ext_vector_type(16)));

__device__ __forceinline__ Acc mfma(Frag<bf16> a, Frag<bf16> b, Acc c) { return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, c, 0, 0, 0); }
__device__ __forceinline__ Acc mfma(Frag<f16> a, Frag<f16> b, Acc c) { return __builtin_amdgcn_mfma_f32_32x32x16_f16(a, b, c, 0, 0, 0); }
__device__ __forceinline__ Acc mfma(Frag<float> a, Frag<float> b, Acc c) {
#pragma unroll
  for (int e = 0; e < 8; e++) c = __builtin_amdgcn_mfma_f32_32x32x2f32(a[e], b[e], c, 0, 0, 0);
  return c;
}

template <typename T> struct Type {
  static constexpr int CE = 16 / sizeof(T);           // elements to a 16-byte chunk
  static constexpr int ROWS = sizeof(T) == 2 ? 64 : 32;  // streamed rows to a tile
  static constexpr bool F16 = __is_same(T, f16);
};

#define LDS_PTR(T, p) ((__attribute__((address_space(3))) T*)(p))

// A staged tile: rows of DP elements in 16-byte chunks; a chunk's place within its row is XORed with bits of the row.  Two reads
// must meet all 64 banks once: 16 adjacent rows at one chunk (row8), and 4 adjacent rows at 4 (32 lanes of col8), so the row's
// low bits go where the chunk's low bits are not.  (With row & 15 for 16 chunks to a row the second read met 4 rows on a bank:
// 4 x 16 heads x 2048 x 4096, bfloat16: 358 -> 331 us forward, 651 -> 611 dk and dv.)
template <typename T, int DP, int R = Type<T>::ROWS>
struct Tile {
  static constexpr int CE = Type<T>::CE, CPR = DP / CE, ROWS = R, BYTES = ROWS * DP * (int)sizeof(T);
  static __device__ __forceinline__ int swz(int row) {
    if (CPR % 16 == 0) return ((row & 3) << 2) | ((row >> 2) & 3);
    if (CPR % 8 == 0) return ((row & 2) << 1) | ((row >> 2) & 3);  // (two rows to the 64 banks)
    return (row >> 2) & 3;
  }
  static __device__ __forceinline__ int at(int row, int d) { return row * DP + ((d / CE) ^ swz(row)) * CE + d % CE; }

  // 8 elements along d: the first product's operand
  static __device__ __forceinline__ Frag<T> row8(const T* t, int row, int d) {
    if constexpr (sizeof(T) == 2) {
      return *(const Frag<T>*)(t + at(row, d));
    } else {
      typedef float f4 __attribute__((ext_vector_type(4)));
      const f4 a = *(const f4*)(t + at(row, d)), b = *(const f4*)(t + at(row, d + 4));
      return __builtin_shufflevector(a, b, 0, 1, 2, 3, 4, 5, 6, 7);
    }
  }
  // 8 rows of column d0 + lane % 32, in the order of the second product's slots: rows r0 + 4 h + {0..3, 8..11}
  static __device__ __forceinline__ Frag<T> col8(const T* t, int r0, int d0, int lane) {
    const int h = lane >> 5;
    if constexpr (sizeof(T) == 2) {
      typedef short s4 __attribute__((ext_vector_type(4)));
      const int i = lane & 15, row = r0 + 4 * h + (i >> 2), d = d0 + (lane & 16) + 4 * (i & 3);
      const s4 a = __builtin_amdgcn_ds_read_tr16_b64_v4i16(LDS_PTR(s4, (T*)t + at(row, d)));
      const s4 b = __builtin_amdgcn_ds_read_tr16_b64_v4i16(LDS_PTR(s4, (T*)t + at(row + 8, d)));
      return __builtin_bit_cast(Frag<T>, __builtin_shufflevector(a, b, 0, 1, 2, 3, 4, 5, 6, 7));
    } else {
      Frag<T> f;
#pragma unroll
      for (int e = 0; e < 8; e++) f[e] = t[at(r0 + 8 * (e >> 2) + 4 * h + (e & 3), d0 + (lane & 31))];
      return f;
    }
  }
  // starts the copy of the rows of two tensors from global memory straight into their tiles, 64 chunks to an instruction; the
  // caller waits.  What lies behind `dim` in a row is left as it is (zero from the start).
  template <typename Row>
  static __device__ __forceinline__ void stage2(T* t, T* u, int dim, int wave, int waves, int lane, Row rows) {
#pragma unroll 4
    for (int i = wave; i < ROWS * CPR / 64; i += waves) {
      const int c = i * 64 + lane, row = c / CPR, d = ((c % CPR) ^ swz(row)) * CE;
      const T *a, *b;
      rows(row, a, b);
      if (d < dim) {
        __builtin_amdgcn_global_load_lds((const __attribute__((address_space(1))) void*)(a + d), LDS_PTR(void, t + i * 64 * CE), 16, 0, 0);
        __builtin_amdgcn_global_load_lds((const __attribute__((address_space(1))) void*)(b + d), LDS_PTR(void, u + i * 64 * CE), 16, 0, 0);
      }
    }
  }
};

template <typename T>
__device__ __forceinline__ Frag<T> load_frag(const T* p) {
  struct __attribute__((packed, aligned(sizeof(T)))) Raw { T v[8]; };
  const Raw r = *(const Raw*)p;
  return __builtin_bit_cast(Frag<T>, r);
}
template <typename T>
__device__ __forceinline__ Frag<T> zero_frag() {
  Frag<T> f;
#pragma unroll
  for (int e = 0; e < 8; e++) f[e] = (T)0.f;
  return f;
}
template <typename T>
__device__ __forceinline__ Frag<T> to_frag(const float* v) {
  if constexpr (sizeof(T) == 4) {
    Frag<T> f;
#pragma unroll
    for (int e = 0; e < 8; e++) f[e] = v[e];
    return f;
  } else {
    typedef uint32_t u4 __attribute__((ext_vector_type(4)));
    const u4 w = {pack2<T>(v[0], v[1]), pack2<T>(v[2], v[3]), pack2<T>(v[4], v[5]), pack2<T>(v[6], v[7])};
    return __builtin_bit_cast(Frag<T>, w);
  }
}
// 4 adjacent elements of an output row
template <typename T>
__device__ __forceinline__ void store4(T* p, float a, float b, float c, float d) {
  if constexpr (sizeof(T) == 4) {
    *(float4*)p = make_float4(a, b, c, d);
  } else {
    *(uint2*)p = make_uint2(pack2<T>(a, b), pack2<T>(c, d));
  }
}
// The lane's 16 elements of 32 output elements (register j of an accumulator is element 8 (j / 4) + 4 h + j % 4), f times them:
// 16-bit elements change places with the other half, so that a lane stores 8 in a row.
template <typename T>
__device__ __forceinline__ void store_row(T* dst, const Acc& a, float f, int room, int h) {  // room: elements of the row from dst on
#pragma unroll
  for (int j = 0; j < 4; j += sizeof(T) == 4 ? 1 : 2) {
    if constexpr (sizeof(T) == 4) {
      const int d = 8 * j + 4 * h;
      if (d < room) store4<T>(dst + d, a[4 * j] * f, a[4 * j + 1] * f, a[4 * j + 2] * f, a[4 * j + 3] * f);
    } else {
      uint32_t x[2], y[2];
#pragma unroll
      for (int e = 0; e < 2; e++) {
        auto r = __builtin_amdgcn_permlane32_swap(pack2<T>(a[4 * j + 2 * e] * f, a[4 * j + 2 * e + 1] * f),
                                                  pack2<T>(a[4 * j + 4 + 2 * e] * f, a[4 * j + 5 + 2 * e] * f), false, false);
        x[e] = r[0];  // of the lower half: elements 0 .. 3 of block j, of the upper: of block j + 1
        y[e] = r[1];  // elements 4 .. 7
      }
      const int d = 8 * (j + h);
      if (d < room) *(uint4*)(dst + d) = make_uint4(x[0], x[1], y[0], y[1]);
    }
  }
}
__device__ __forceinline__ float other_half(float v) {
  auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  return __uint_as_float((threadIdx.x & 32) ? r[0] : r[1]);
}
__device__ __forceinline__ int allowed_keys(const AttendParams& p, int b) {
  if (p.list) return p.list[(int64_t)b * (p.k_len + 1)];
  if (!p.lengths) return p.k_len;
  const int64_t n = p.lengths_type == 8 ? ((const int64_t*)p.lengths)[b] : ((const int32_t*)p.lengths)[b];
  return (int)(n < 0 ? 0 : (n > p.k_len ? p.k_len : n));
}

// the row of register j of an accumulator
__device__ __forceinline__ int acc_row(int j, int h) { return (j & 3) + 8 * (j >> 2) + 4 * h; }

struct Work { int b, kh, tile, split; };
// Workgroups go to the 8 dies in turn, and each die has an L2 of its own: the workgroups that stream the same rows are numbered
// so that they meet on one die.
// Where part of the tiles may find nothing to do (p.tail), their workgroups come last on each die: numbered side by side with
// the others they would meet the same compute units every time.  Heads stay side by side, since they share cache lines.
__device__ __forceinline__ Work decode(const AttendParams& p) {
  Work k;
  uint32_t w;
  if (p.tail) {
    const uint32_t slot = blockIdx.x >> 3, x = p.by_die.of(slot), bh = (blockIdx.x & 7) * p.by_die.d + (slot - x * p.by_die.d);
    k.tile = (int)p.by_splits.of(x);
    k.split = (int)(x - k.tile * p.splits);
    const bool in = bh < (uint32_t)p.batch * p.kv_heads;
    k.b = in ? (int)p.by_kv.of(bh) : -1;
    k.kh = in ? (int)(bh - k.b * p.kv_heads) : 0;
    return k;
  }
  const uint32_t total = gridDim.x, die = blockIdx.x & 7, slot = blockIdx.x >> 3, per = total >> 3, rest = total & 7;
  w = die * per + (die < rest ? die : rest) + slot;
  uint32_t x = p.by_tiles.of(w);
  k.tile = (int)(w - x * p.tiles);
  w = p.by_splits.of(x);
  k.split = (int)(x - w * p.splits);
  k.b = (int)p.by_kv.of(w);
  k.kh = (int)(w - k.b * p.kv_heads);
  return k;
}
// the part of `all` tiles that is split k of n
__device__ __forceinline__ int split_at(const AttendParams& p, int all, int k) {
  return p.splits == 1 ? (k ? all : 0) : (int)p.by_splits.of((uint32_t)all * (uint32_t)k);
}

// element offset of row r = (l, g) of a [batch, length, head, dim] tensor behind its head's first row
__device__ __forceinline__ int64_t row_offset(int64_t ls, int64_t hs, const AttendParams& p, int r) {
  if (p.group == 1) return r * ls;
  const int l = (int)p.by_group.of(r), g = r - l * p.group;
  return l * ls + g * hs;
}
template <typename T>
__device__ __forceinline__ T* head_of(T* t, const int64_t (&s)[3], const AttendParams& p, const Work& w) {
  return t + (w.b * s[0] + (int64_t)w.kh * p.group * s[2]);
}
// the same in a result, which is contiguous
__device__ __forceinline__ int64_t out_head(const AttendParams& p, const Work& w) {
  return ((int64_t)w.b * p.q_len * p.heads + w.kh * p.group) * p.dim;
}
__device__ __forceinline__ int64_t out_row(const AttendParams& p, int r) { return row_offset((int64_t)p.heads * p.dim, p.dim, p, r); }

template <int N>
__device__ __forceinline__ void zero_lds(void* p, int tid, int threads) {
  for (int i = tid; i < N / 16; i += threads) ((float4*)p)[i] = make_float4(0.f, 0.f, 0.f, 0.f);
}

// the staged tile is there, the other one is free: every wavefront waits for its own copies, then for the others
__device__ __forceinline__ void tile_barrier() {
  asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)" ::: "memory");
  __syncthreads();
}

// F16: the power of two that dS carries into its product, one for the wavefront.  It starts high and falls so that the largest
// entry met so far stays below 2^14; when it falls, the sums so far are scaled with it.
struct Power {
  int e;
  float f;  // 2^e
  __device__ __forceinline__ void start() { e = 100; f = __builtin_amdgcn_exp2f(100.f); }
  template <int N>
  __device__ __forceinline__ float follow(float largest, Acc (&acc)[N]) {
    // (whether it has to fall is asked of all lanes at once; the wavefront's maximum is needed only then: dq and dk/dv of
    // 3 x 517 x 1999: 62 and 73 us with the maximum every time, 59 and 69 so)
    if (__ballot(largest >= __builtin_amdgcn_exp2f((float)(14 - e)))) {
      const float m = wave_max(largest);
      const int x = (int)((__float_as_uint(m) >> 23) & 255) - 127;  // 2^x <= m < 2^(x + 1)
      int want = 13 - x;
      want = want < -100 ? -100 : want;
      if (want < e) {
        const float g = __builtin_amdgcn_exp2f((float)(want - e));
#pragma unroll
        for (int i = 0; i < N; i++) acc[i] *= g;
        e = want;
        f = __builtin_amdgcn_exp2f((float)e);
      }
    }
    return f;
  }
};

// ------------------------------------------------------------------------------------------------------------- forward
// Measured: 4 x 16 heads x 2048 x 4096 x 128 bfloat16 331 us, 830 TFLOP/s (a library product of 8192^3: 1134) -- two wavefronts to a
// SIMD that wait for their own products and exponentials in turn; 2048 x 4 x 200 x 401 x 32 with 29 % of the keys 128 us, where
// vector instructions are 59 % busy and HBM moves 2.6 TB/s; 4096 x 131 x 131 x 64 float32 163 us, its matrix instructions at 35 % of
// their peak; single queries, 16 x 8 heads x 16384 x 128, 156 us, 5.2 TB/s.
template <typename T, int DP, int MAXW, int R>
__global__ __launch_bounds__(64 * MAXW) void pct_attend_kernel(AttendParams p) {
  using L = Tile<T, DP, R>;
  constexpr int KT = L::ROWS, SUB = KT / 32, KS = DP / 16, DB = DP / 32;
  extern __shared__ __attribute__((aligned(16))) char lds[];
  T* const buf = (T*)lds;  // [2][k, v] tiles
  __shared__ int keys[2][KT];
  const int tid = threadIdx.x, lane = tid & 63, waves = blockDim.x >> 6, c32 = lane & 31, h = lane >> 5;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const Work w = decode(p);
  const int row = (w.tile * waves + wave) * 32 + c32;
  const bool active = (w.tile * waves + wave) * 32 < p.rows;
  const int32_t* list = p.list ? p.list + (int64_t)w.b * (p.k_len + 1) + 1 : nullptr;
  const T* kb = (const T*)p.k + w.b * p.ks[0] + w.kh * p.ks[2];
  const T* vb = (const T*)p.v + w.b * p.vs[0] + w.kh * p.vs[2];

  const T* qr = head_of((const T*)p.q, p.qs, p, w) + row_offset(p.qs[1], p.qs[2], p, row);
  Frag<T> qf[KS];
#pragma unroll
  for (int s = 0; s < KS; s++) {
    const int d = 16 * s + 8 * h;
    qf[s] = row < p.rows && d < p.dim ? load_frag(qr + d) : zero_frag<T>();
  }
  // (unsplit, the first entries of the list are asked for together with the count: behind it, the first one stands in for them)
  const bool ahead_of_count = list && p.splits == 1;
  int early[2 * KT / 64], early0 = 0;
  if (ahead_of_count) {
    early0 = list[0];
#pragma unroll
    for (int x = 0; x < 2 * KT / 64; x++) {
      const int i = x * (int)blockDim.x + tid;
      early[x] = list[i < p.k_len ? i : 0];
    }
  }
  const int n = allowed_keys(p, w.b), all = (n + KT - 1) / KT;
  const int t0 = split_at(p, all, w.split), t1 = split_at(p, all, w.split + 1);
  auto key_at = [&](int i) { i = i < n ? i : n - 1; return list ? list[i] : i; };
  auto stage = [&](int t) {
    T* k = buf + (t & 1) * 2 * KT * DP;
    L::stage2(k, k + KT * DP, p.dim, wave, waves, lane, [&](int r, const T*& a, const T*& b) {
      const int64_t key = keys[t & 1][r];
      a = kb + key * p.ks[1];
      b = t * KT + r >= n ? zero_row<T>() : vb + key * p.vs[1];
    });
  };
  if (p.dim != DP) zero_lds<4 * L::BYTES>(lds, tid, blockDim.x);
  if (t0 < t1) {
#pragma unroll
    for (int x = 0; x < 2 * KT / 64; x++) {
      const int i = x * (int)blockDim.x + tid;
      if (i < 2 * KT) keys[(t0 + i / KT) & 1][i % KT] = ahead_of_count ? (i < n ? early[x] : early0) : key_at(t0 * KT + i);
    }
  }
  __syncthreads();
  if (t0 < t1) stage(t0);
  if (t0 + 1 < t1) stage(t0 + 1);
  Acc o[DB];
#pragma unroll
  for (int i = 0; i < DB; i++) o[i] = Acc{};
  // exponents are taken against `ref`, which follows the maximum only when it is left behind by more than 2^6 (P then stays
  // small enough for every type, and the sums are rarely scaled); float16 lifts P by 2^8 out of its denormals
  constexpr float LIFT = Type<T>::F16 ? 8.f : 0.f;
  // (it starts at the lowest number, not at -infinity: a tile of scores that are all -infinity then weighs 0, not NaN)
  float ref = kLowest, sum = 0.f;
  for (int t = t0; t < t1; t++) {
    tile_barrier();
    int ahead = 0;
    if (t > t0 && t + 1 < t1) stage(t + 1);  // (the first two are on their way already)
    if (t + 2 < t1 && tid < KT) ahead = key_at((t + 2) * KT + tid);
    if (active) {
      const T* kt = buf + (t & 1) * 2 * KT * DP;
      const T* vt = kt + KT * DP;
      Acc s[SUB];
#pragma unroll
      for (int i = 0; i < SUB; i++) {
        s[i] = Acc{};
#pragma unroll
        for (int x = 0; x < KS; x++) s[i] = mfma(L::row8(kt, 32 * i + c32, 16 * x + 8 * h), qf[x], s[i]);
      }
      if ((t + 1) * KT > n) {
#pragma unroll
        for (int i = 0; i < SUB; i++)
#pragma unroll
          for (int j = 0; j < 16; j++) s[i][j] = t * KT + 32 * i + acc_row(j, h) < n ? s[i][j] : -INFINITY;
      }
      float top = s[0][0];
#pragma unroll
      for (int i = 0; i < SUB; i++)
#pragma unroll
        for (int j = 0; j < 16; j++) top = fmaxf(top, s[i][j]);
      top = fmaxf(top, other_half(top)) * p.c - LIFT;
      if (__ballot(top > ref + 6.f)) {
        const float to = fmaxf(ref, top), f = __builtin_amdgcn_exp2f(ref - to);
#pragma unroll
        for (int i = 0; i < DB; i++) o[i] *= f;
        sum *= f;
        ref = to;
      }
#pragma unroll
      for (int i = 0; i < SUB; i++)
#pragma unroll
        for (int j = 0; j < 16; j++) {
          s[i][j] = __builtin_amdgcn_exp2f(fmaf(s[i][j], p.c, -ref));
          sum += s[i][j];
        }
#pragma unroll
      for (int i = 0; i < SUB; i++)
#pragma unroll
        for (int b = 0; b < 2; b++) {
          float e8[8];
#pragma unroll
          for (int e = 0; e < 8; e++) e8[e] = s[i][8 * b + e];
          const Frag<T> pf = to_frag<T>(e8);
#pragma unroll
          for (int d = 0; d < DB; d++) o[d] = mfma(L::col8(vt, 32 * i + 16 * b, 32 * d, lane), pf, o[d]);
        }
    }
    if (t + 2 < t1) {  // (every wavefront has read the keys of tile t before the barrier above)
      if (tid < KT) keys[t & 1][tid] = ahead;
      for (int i = tid + (int)blockDim.x; i < KT; i += blockDim.x) keys[t & 1][i] = key_at((t + 2) * KT + i);
    }
  }
  if (row >= p.rows) return;
  sum += other_half(sum);
  const int64_t at = ((int64_t)w.b * p.kv_heads + w.kh) * p.rows + row;
  if (p.splits > 1) {
    const int64_t sp = (int64_t)w.split * p.batch * p.kv_heads * p.rows + at;
    if (h == 0) p.part_stats[sp] = make_float2(ref, sum);
    float* dst = p.part + sp * p.dim;
#pragma unroll
    for (int i = 0; i < DB; i++)
#pragma unroll
      for (int j = 0; j < 4; j++) {
        const int d = 32 * i + 8 * j + 4 * h;
        if (d < p.dim) *(float4*)(dst + d) = make_float4(o[i][4 * j], o[i][4 * j + 1], o[i][4 * j + 2], o[i][4 * j + 3]);
      }
    return;
  }
  const float inv = n > 0 ? 1.f / sum : 0.f;
  if (h == 0 && p.stats) p.stats[at] = n > 0 ? make_float2(ref, sum) : make_float2(0.f, INFINITY);
  T* dst = (T*)p.out + out_head(p, w) + out_row(p, row);
#pragma unroll
  for (int i = 0; i < DB; i++) store_row<T>(dst + 32 * i, o[i], inv, p.dim - 32 * i, h);
}

// Joins the splits of the forward pass: a thread to 4 elements of a row walks over them, four in flight.  Bound by latency: 512 rows of
// 128 in 16 parts 6.3 us, in 64 parts 13.2, 2048 rows in 32 parts 9.0.  (A wavefront to a row with all of its reads in flight was no
// faster anywhere: 7.0, 13.0, 9.4, and 10.8 against 8.8 for one row in 64 parts.)
template <typename T>
__global__ __launch_bounds__(256) void pct_attend_join_kernel(AttendParams p) {
  const int per = p.dim / 4;
  const int64_t rows = (int64_t)p.batch * p.kv_heads * p.rows, i = (int64_t)blockIdx.x * 256 + threadIdx.x;
  if (i >= rows * per) return;
  const int64_t at = i / per;
  const int d = (int)(i % per) * 4, r = (int)(at % p.rows), bh = (int)(at / p.rows);
  float ref = kLowest, sum = 0.f;
#pragma unroll 4
  for (int s = 0; s < p.splits; s++) ref = fmaxf(ref, p.part_stats[s * rows + at].x);
  float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 4
  for (int s = 0; s < p.splits; s++) {
    const float2 st = p.part_stats[s * rows + at];
    const float f = __builtin_amdgcn_exp2f(st.x - ref);
    const float4 x = *(const float4*)(p.part + (s * rows + at) * p.dim + d);
    sum += f * st.y;
    o.x += f * x.x; o.y += f * x.y; o.z += f * x.z; o.w += f * x.w;
  }
  const bool none = allowed_keys(p, bh / p.kv_heads) == 0;
  const float inv = none ? 0.f : 1.f / sum;
  if (d == 0 && p.stats) p.stats[at] = none ? make_float2(0.f, INFINITY) : make_float2(ref, sum);
  const Work w = {bh / p.kv_heads, bh % p.kv_heads, 0, 0};
  store4<T>((T*)p.out + out_head(p, w) + out_row(p, r) + d, o.x * inv, o.y * inv, o.z * inv, o.w * inv);
}

// P of the backward pass: float32 keeps the forward's reference point and sum apart (their logarithm's rounding would be a
// common factor of the row), the others fold them, and float16 lifts P by 2^14 (P <= 1)
template <typename T> constexpr float p_lift() { return Type<T>::F16 ? 14.f : 0.f; }
// (a lone key has P = 1: asked for with c = 0 and these terms it is that to the last bit, so that dP - D is 0 as it should be)
template <typename T>
__device__ __forceinline__ float2 p_alone() { return make_float2(-p_lift<T>(), 1.f); }
template <typename T>
__device__ __forceinline__ float2 p_terms(float2 st) {
  if constexpr (sizeof(T) == 4) return make_float2(st.x, 1.f / st.y);
  else return make_float2(st.x + log2f(st.y) - p_lift<T>(), 1.f);
}
template <typename T>
__device__ __forceinline__ float p_value(float s, float c, float2 t) {
  const float e = __builtin_amdgcn_exp2f(fmaf(s, c, -t.x));
  return sizeof(T) == 4 ? e * t.y : e;
}

// ---------------------------------------------------------------------------------------------------------------- dq, D
// D_r = dO_r . O_r, where O_r has been rounded to the tensors' type: over many keys that error vanishes beside dP, over few it
// would not, so where all keys fit one tile of 16-bit elements D is summed from P dP itself.  So is that of a lone key, in every
// type: its dS is then exactly 0.
// Measured: 4 x 16 x 2048 x 4096 x 128 bfloat16 460 us, 895 TFLOP/s over three products; 2048 x 4 x 200 x 401 x 32 188 us; 4096 x 131 x
// 131 x 64 float32 252 us, 34 % of the matrix peak at two wavefronts to a SIMD (more would spill).
template <typename T, int DP, int MAXW>
__global__ __launch_bounds__(64 * MAXW) void pct_attend_dq_kernel(AttendParams p) {
  using L = Tile<T, DP>;
  constexpr int KT = L::ROWS, SUB = KT / 32, KS = DP / 16, DB = DP / 32;
  constexpr bool EXACT = sizeof(T) == 2;
  extern __shared__ __attribute__((aligned(16))) char lds[];
  T* const buf = (T*)lds;
  __shared__ int keys[2][KT];
  const int tid = threadIdx.x, lane = tid & 63, waves = blockDim.x >> 6, c32 = lane & 31, h = lane >> 5;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const Work w = decode(p);
  const int row = (w.tile * waves + wave) * 32 + c32;
  const bool active = (w.tile * waves + wave) * 32 < p.rows;
  const int32_t* list = p.list ? p.list + (int64_t)w.b * (p.k_len + 1) + 1 : nullptr;
  const T* kb = (const T*)p.k + w.b * p.ks[0] + w.kh * p.ks[2];
  const T* vb = (const T*)p.v + w.b * p.vs[0] + w.kh * p.vs[2];
  const int64_t at = ((int64_t)w.b * p.kv_heads + w.kh) * p.rows + row;

  const T* qr = head_of((const T*)p.q, p.qs, p, w) + row_offset(p.qs[1], p.qs[2], p, row);
  const T* dr = head_of((const T*)p.d_out, p.ds, p, w) + row_offset(p.ds[1], p.ds[2], p, row);
  Frag<T> qf[KS], df[KS];
#pragma unroll
  for (int s = 0; s < KS; s++) {
    const int d = 16 * s + 8 * h;
    const bool in = row < p.rows && d < p.dim;
    qf[s] = in ? load_frag(qr + d) : zero_frag<T>();
    df[s] = in ? load_frag(dr + d) : zero_frag<T>();
  }
  float2 st = row < p.rows ? p.stats[at] : make_float2(INFINITY, INFINITY);
  // (unsplit, the first entries of the list are asked for together with the count: behind it, the first one stands in for them)
  const bool ahead_of_count = list && p.splits == 1;
  int early[2 * KT / 64], early0 = 0;
  if (ahead_of_count) {
    early0 = list[0];
#pragma unroll
    for (int x = 0; x < 2 * KT / 64; x++) {
      const int i = x * (int)blockDim.x + tid;
      early[x] = list[i < p.k_len ? i : 0];
    }
  }
  const int n = allowed_keys(p, w.b), all = (n + KT - 1) / KT;
  const int t0 = split_at(p, all, w.split), t1 = split_at(p, all, w.split + 1);
  auto key_at = [&](int i) { i = i < n ? i : n - 1; return list ? list[i] : i; };
  auto stage = [&](int t) {
    T* k = buf + (t & 1) * 2 * KT * DP;
    L::stage2(k, k + KT * DP, p.dim, wave, waves, lane, [&](int r, const T*& a, const T*& b) {
      const int64_t key = keys[t & 1][r];
      a = kb + key * p.ks[1];
      b = vb + key * p.vs[1];
    });
  };
  if (p.dim != DP) zero_lds<4 * L::BYTES>(lds, tid, blockDim.x);
  if (t0 < t1) {
#pragma unroll
    for (int x = 0; x < 2 * KT / 64; x++) {
      const int i = x * (int)blockDim.x + tid;
      if (i < 2 * KT) keys[(t0 + i / KT) & 1][i % KT] = ahead_of_count ? (i < n ? early[x] : early0) : key_at(t0 * KT + i);
    }
  }
  __syncthreads();
  if (t0 < t1) stage(t0);
  if (t0 + 1 < t1) stage(t0 + 1);
  st = n == 1 ? p_alone<T>() : p_terms<T>(st);
  const float c = n == 1 ? 0.f : p.c;
  const bool few = n == 1 || (EXACT && n <= KT);
  float D = 0.f;
  if (row < p.rows && n > 0 && !few) {
#pragma unroll
    for (int s = 0; s < KS; s++) {
      const int d = 16 * s + 8 * h;
      if (d >= p.dim) break;
      const Frag<T> of = load_frag((const T*)p.o + out_head(p, w) + out_row(p, row) + d);
#pragma unroll
      for (int e = 0; e < 8; e++) D = fmaf((float)df[s][e], (float)of[e], D);
    }
  }
  Acc dq[DB];
#pragma unroll
  for (int i = 0; i < DB; i++) dq[i] = Acc{};
  Power power;
  power.start();
  auto products = [&](const T* kt, const T* vt, int first, Acc& s, Acc& dp) {  // P in s, dP in dp, of 32 keys
    s = Acc{};
    dp = Acc{};
#pragma unroll
    for (int x = 0; x < KS; x++) {
      s = mfma(L::row8(kt, first % KT + c32, 16 * x + 8 * h), qf[x], s);
      dp = mfma(L::row8(vt, first % KT + c32, 16 * x + 8 * h), df[x], dp);
    }
#pragma unroll
    for (int j = 0; j < 16; j++) s[j] = first + acc_row(j, h) < n ? p_value<T>(s[j], c, st) : 0.f;
  };
  for (int t = t0; t < t1; t++) {
    tile_barrier();
    int ahead = 0;
    if (t > t0 && t + 1 < t1) stage(t + 1);  // (the first two are on their way already)
    if (t + 2 < t1 && tid < KT) ahead = key_at((t + 2) * KT + tid);
    if (active) {
      const T* kt = buf + (t & 1) * 2 * KT * DP;
      const T* vt = kt + KT * DP;
      if (few) {
#pragma unroll 1
        for (int i = 0; i < SUB; i++) {
          Acc s, dp;
          products(kt, vt, 32 * i, s, dp);
#pragma unroll
          for (int j = 0; j < 16; j++) D = fmaf(s[j], dp[j], D);
        }
        D *= __builtin_amdgcn_exp2f(-p_lift<T>());
      }
      if (t == t0) D += other_half(D);
#pragma unroll 1
      for (int i = 0; i < SUB; i++) {
        if (t * KT + 32 * i >= n) break;
        Acc s, dp;
        products(kt, vt, t * KT + 32 * i, s, dp);
        float e16[16], big = 0.f;
#pragma unroll
        for (int j = 0; j < 16; j++) {
          e16[j] = s[j] * (dp[j] - D);
          if (Type<T>::F16) big = fmaxf(big, fabsf(e16[j]));
        }
        if (Type<T>::F16) {
          const float f = power.follow(big, dq);
#pragma unroll
          for (int j = 0; j < 16; j++) e16[j] *= f;
        }
#pragma unroll
        for (int b = 0; b < 2; b++) {
          const Frag<T> sf = to_frag<T>(e16 + 8 * b);
#pragma unroll
          for (int d = 0; d < DB; d++) dq[d] = mfma(L::col8(kt, 32 * i + 16 * b, 32 * d, lane), sf, dq[d]);
        }
      }
    }
    if (t + 2 < t1) {  // (every wavefront has read the keys of tile t before the barrier above)
      if (tid < KT) keys[t & 1][tid] = ahead;
      for (int i = tid + (int)blockDim.x; i < KT; i += blockDim.x) keys[t & 1][i] = key_at((t + 2) * KT + i);
    }
  }
  if (row >= p.rows) return;
  if (h == 0 && t0 == 0 && t1 > 0) p.delta[at] = D;  // (one split of them has the first tile; without keys nobody reads it)
  const float f = Type<T>::F16 ? p.scale * __builtin_amdgcn_exp2f(-(float)power.e - p_lift<T>()) : p.scale;
  float* part = p.splits > 1 ? p.part + (int64_t)w.split * p.batch * p.q_len * p.heads * p.dim + out_head(p, w) + out_row(p, row) : nullptr;
  T* dst = (T*)p.dq + out_head(p, w) + out_row(p, row);
#pragma unroll
  for (int i = 0; i < DB; i++) {
    if (part) store_row<float>(part + 32 * i, dq[i], f, p.dim - 32 * i, h);
    else store_row<T>(dst + 32 * i, dq[i], f, p.dim - 32 * i, h);
  }
}

// --------------------------------------------------------------------------------------------------------------- dk, dv
// The same tiles with the sides changed: keys stay, q and d_out pass.  S and dP are computed a second time, which costs two products
// of seven and needs neither atomics nor dS in memory.  Measured: 4 x 16 x 2048 x 4096 x 128 bfloat16 611 us, 900 TFLOP/s over four
// products; 2048 x 4 x 200 x 401 x 32 160 us; 4096 x 131 x 131 x 64 float32 250 us, 46 % of the matrix peak.
template <typename T, int DP, int MAXW>
__global__ __launch_bounds__(64 * MAXW) void pct_attend_dkv_kernel(AttendParams p) {
  using L = Tile<T, DP>;
  constexpr int QT = L::ROWS, SUB = QT / 32, KS = DP / 16, DB = DP / 32;
  extern __shared__ __attribute__((aligned(16))) char lds[];
  T* const buf = (T*)lds;  // [2][q, d_out] tiles
  __shared__ __attribute__((aligned(16))) float terms[2][3][QT];  // of the staged rows: p_terms, D
  const int tid = threadIdx.x, lane = tid & 63, waves = blockDim.x >> 6, c32 = lane & 31, h = lane >> 5;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const Work w = decode(p);
  if (w.b < 0) return;
  const int32_t* list = p.list ? p.list + (int64_t)w.b * (p.k_len + 1) + 1 : nullptr;
  const int first = (w.tile * waves + wave) * 32, i = first + c32;  // place in the list
  const int key = i < p.k_len ? (list ? list[i] : i) : 0;
  const int n = allowed_keys(p, w.b);
  const bool active = first < n, valid = i < n;
  if (w.tile * waves * 32 >= n) return;  // (the whole workgroup; pct_attend_clear_kernel writes the rows of such keys)
  const int all = (p.rows + QT - 1) / QT;
  const int t0 = split_at(p, all, w.split), t1 = split_at(p, all, w.split + 1);
  const T* qb = head_of((const T*)p.q, p.qs, p, w);
  const T* db = head_of((const T*)p.d_out, p.ds, p, w);
  const float2* stats = p.stats + ((int64_t)w.b * p.kv_heads + w.kh) * p.rows;
  const float* delta = p.delta + ((int64_t)w.b * p.kv_heads + w.kh) * p.rows;

  auto stage = [&](int t) {
    T* q = buf + (t & 1) * 2 * QT * DP;
    L::stage2(q, q + QT * DP, p.dim, wave, waves, lane, [&](int r, const T*& a, const T*& b) {
      const bool in = t * QT + r < p.rows;
      const int x = in ? t * QT + r : p.rows - 1, l = p.group == 1 ? x : (int)p.by_group.of(x), g = x - l * p.group;
      a = qb + l * p.qs[1] + g * p.qs[2];
      b = in ? db + l * p.ds[1] + g * p.ds[2] : zero_row<T>();
    });
  };
  // (a workgroup has at least 64 threads: one to a staged row)
  struct Terms { float2 p; float d; };
  auto get_terms = [&](int t) {
    const int row = t * QT + tid;
    Terms x = {make_float2(INFINITY, INFINITY), 0.f};
    if (tid < QT && row < p.rows) { x.p = stats[row]; x.d = delta[row]; }
    return x;
  };
  auto put_terms = [&](int t, const Terms& y) {
    if (tid < QT) {
      const float2 x = n == 1 && t * QT + tid < p.rows ? p_alone<T>() : p_terms<T>(y.p);
      terms[t & 1][0][tid] = x.x;
      terms[t & 1][1][tid] = x.y;
      terms[t & 1][2][tid] = y.d;
    }
  };
  if (p.dim != DP) {
    zero_lds<4 * L::BYTES>(lds, tid, blockDim.x);
    __syncthreads();
  }
  const float c = n == 1 ? 0.f : p.c;
  Terms next = {};
  Frag<T> kf[KS], vf[KS];
  if (t0 < t1) {
    const Terms x = get_terms(t0);
    next = get_terms(t0 + 1);
    stage(t0);
    if (t0 + 1 < t1) stage(t0 + 1);
#pragma unroll
    for (int s = 0; s < KS; s++) {
      const int d = 16 * s + 8 * h;
      const bool in = valid && d < p.dim;
      kf[s] = in ? load_frag((const T*)p.k + w.b * p.ks[0] + key * p.ks[1] + w.kh * p.ks[2] + d) : zero_frag<T>();
      vf[s] = in ? load_frag((const T*)p.v + w.b * p.vs[0] + key * p.vs[1] + w.kh * p.vs[2] + d) : zero_frag<T>();
    }
    put_terms(t0, x);
    put_terms(t0 + 1, next);
  }
  Acc dk[DB], dv[DB];
#pragma unroll
  for (int d = 0; d < DB; d++) { dk[d] = Acc{}; dv[d] = Acc{}; }
  Power power;
  power.start();
  for (int t = t0; t < t1; t++) {
    tile_barrier();
    const bool more = t > t0 && t + 1 < t1;
    if (more) {
      next = get_terms(t + 1);
      stage(t + 1);
    }
    if (active) {
    const T* qt = buf + (t & 1) * 2 * QT * DP;
    const T* dt = qt + QT * DP;
#pragma unroll 1
    for (int u = 0; u < SUB; u++) {
      if (t * QT + 32 * u >= p.rows) break;
      Acc s = {}, dp = {};
#pragma unroll
      for (int x = 0; x < KS; x++) {
        s = mfma(L::row8(qt, 32 * u + c32, 16 * x + 8 * h), kf[x], s);
        dp = mfma(L::row8(dt, 32 * u + c32, 16 * x + 8 * h), vf[x], dp);
      }
      float p16[16], e16[16], big = 0.f;
#pragma unroll
      for (int g = 0; g < 4; g++) {
        const int r = 32 * u + 8 * g + 4 * h;
        const float4 a = *(const float4*)&terms[t & 1][0][r], D = *(const float4*)&terms[t & 1][2][r];
        float4 b = make_float4(1.f, 1.f, 1.f, 1.f);
        if (sizeof(T) == 4) b = *(const float4*)&terms[t & 1][1][r];
#pragma unroll
        for (int e = 0; e < 4; e++) {
          const int j = 4 * g + e;
          p16[j] = p_value<T>(s[j], c, make_float2((&a.x)[e], (&b.x)[e]));
          e16[j] = p16[j] * (dp[j] - (&D.x)[e]);
          if (Type<T>::F16) big = fmaxf(big, fabsf(e16[j]));
        }
      }
      if (Type<T>::F16) {
        const float f = power.follow(valid ? big : 0.f, dk);
#pragma unroll
        for (int j = 0; j < 16; j++) e16[j] *= f;
      }
#pragma unroll
      for (int b = 0; b < 2; b++) {
        const Frag<T> pf = to_frag<T>(p16 + 8 * b), sf = to_frag<T>(e16 + 8 * b);
#pragma unroll
        for (int d = 0; d < DB; d++) {
          dv[d] = mfma(L::col8(dt, 32 * u + 16 * b, 32 * d, lane), pf, dv[d]);
          dk[d] = mfma(L::col8(qt, 32 * u + 16 * b, 32 * d, lane), sf, dk[d]);
        }
      }
    }
    }
    if (more) put_terms(t + 1, next);
  }
  if (!valid) return;
  const float fk = Type<T>::F16 ? p.scale * __builtin_amdgcn_exp2f(-(float)power.e - p_lift<T>()) : p.scale;
  const float fv = __builtin_amdgcn_exp2f(-p_lift<T>());
  const int64_t at = ((int64_t)w.b * p.k_len * p.kv_heads + w.kh) * p.dim + key * ((int64_t)p.kv_heads * p.dim);
  const int64_t whole = (int64_t)p.batch * p.k_len * p.kv_heads * p.dim;
  float* part = p.splits > 1 ? p.part + (int64_t)w.split * 2 * whole + at : nullptr;
#pragma unroll
  for (int x = 0; x < DB; x++) {
    const int room = p.dim - 32 * x;
    if (part) {
      store_row<float>(part + 32 * x, dk[x], fk, room, h);
      store_row<float>(part + whole + 32 * x, dv[x], fv, room, h);
    } else {
      store_row<T>((T*)p.dk + at + 32 * x, dk[x], fk, room, h);
      store_row<T>((T*)p.dv + at + 32 * x, dv[x], fv, room, h);
    }
  }
}

// clears dk and dv of the keys that are not allowed, all heads of one at a time: a workgroup to a batch, 16 bytes to a thread
// (2048 x 401 keys of 4 x 32, 71 % of them: 41 us, 7 TB/s)
template <typename T>
__global__ __launch_bounds__(256) void pct_attend_clear_kernel(AttendParams p, int chunks, int b0) {
  const int b = b0 + blockIdx.x, n = allowed_keys(p, b);
  const int32_t* list = p.list ? p.list + (int64_t)b * (p.k_len + 1) + 1 : nullptr;
  const int64_t bytes = (int64_t)p.kv_heads * p.dim * (int64_t)sizeof(T), base = b * p.k_len * bytes;
  const int per = (int)(bytes / 16), rows = p.k_len - n;
  // (a row's chunks are shared out in powers of two of threads, so that no division is needed)
  const int x0 = threadIdx.x % chunks;
  for (int r = threadIdx.x / chunks + blockIdx.y * (256 / chunks); r < rows; r += gridDim.y * (256 / chunks)) {
    const int64_t at = base + (list ? list[n + r] : n + r) * bytes;
    for (int x = x0; x < per; x += chunks) {
      *(uint4*)((char*)p.dk + at + 16 * x) = make_uint4(0, 0, 0, 0);
      *(uint4*)((char*)p.dv + at + 16 * x) = make_uint4(0, 0, 0, 0);
    }
  }
}

// adds the splits' partial gradients, laid out as the results are: 4 elements to a thread
template <typename T>
__global__ __launch_bounds__(256) void pct_attend_sum_kernel(const float* part, int64_t stride, int splits, int64_t count, T* a, T* b) {
  const int64_t i = ((int64_t)blockIdx.x * 256 + threadIdx.x) * 4;
  if (i >= count) return;
  float4 s = *(const float4*)(part + blockIdx.y * count + i);
#pragma unroll 4
  for (int k = 1; k < splits; k++) {
    const float4 x = *(const float4*)(part + k * stride + blockIdx.y * count + i);
    s.x += x.x; s.y += x.y; s.z += x.z; s.w += x.w;
  }
  store4<T>((blockIdx.y ? b : a) + i, s.x, s.y, s.z, s.w);
}

// How the work is cut.  Resident rows: 32 to a wavefront, as many wavefronts to a workgroup as there are rows for (they share a
// staged tile), 8 or at most 4 (5 to 7 load a compute unit's four SIMDs unevenly and leave no room for another workgroup: 90 heads x
// 1300, D = 128, bfloat16, forward 150 us with 7, 112 with 4), and fewer while that leaves compute units without a workgroup.  Streamed rows: split over workgroups until
// about eight wavefronts per compute unit are there, in parts of at least four tiles (64 x 50 x 131, float32: 5 tiles in two parts
// 12.2 + 4.0 us for the join, in one 14); the partial results are joined after.
struct Cut { int waves, tiles, splits; };
inline Cut cut(int64_t resident, int64_t streamed_tiles, int64_t heads, int max_waves) {
  const int64_t t = (resident + 31) / 32;
  int64_t w = t < max_waves ? t : max_waves, blocks = (t + w - 1) / w;
  w = (t + blocks - 1) / blocks;
  if (w > 4 && w < 8) {
    w = 4;
    blocks = (t + w - 1) / w;
  }
  while (heads * blocks < 256 && w > 1) {
    w = (w + 1) / 2;
    blocks = (t + w - 1) / w;
  }
  int64_t s = (2048 + heads * t - 1) / (heads * t);
  s = s < streamed_tiles / 4 ? s : streamed_tiles / 4;
  s = s < 1 ? 1 : (s > 64 ? 64 : s);
  return Cut{(int)w, (int)blocks, (int)s};
}

// the wavefronts to a workgroup that a kernel is compiled for: 8, two to a SIMD, where a wavefront's registers allow it (256 each)
template <typename T, int DP> constexpr int max_waves() { return sizeof(T) == 4 && DP > 64 ? 4 : 8; }

// a launch with the LDS of four tiles, which may be more than the runtime's default limit of 64 KiB
template <int BYTES>
void launch(void (*kernel)(AttendParams), dim3 grid, int waves, hipStream_t s, const AttendParams& p) {
  if (BYTES > 60 * 1024) (void)hipFuncSetAttribute((const void*)kernel, hipFuncAttributeMaxDynamicSharedMemorySize, BYTES);
  kernel<<<grid, 64 * waves, BYTES, s>>>(p);
}

template <typename T> struct Attend {
  template <typename F>
  static auto by_dim(int dim, F f) {
    if (dim <= 32) return f(std::integral_constant<int, 32>());
    if (dim <= 64) return f(std::integral_constant<int, 64>());
    if (dim <= 96) return f(std::integral_constant<int, 96>());
    return f(std::integral_constant<int, 128>());
  }
  // Wavefronts to a workgroup: 4, from which two or three workgroups fit a compute unit and wait for each other's products.  Times below
  // are us with up to 2 / 4 / 8, over 131 to 5000 rows, every type and four head sizes; fewer than 256 workgroups are cut further (cut).
  //  * forward, 16-bit, 1024 rows and more: 8 read a tile half as often.  64 heads x 2048 x 2048: D = 32 158 / 123 / 115, 64 234 / 183 /
  //    170, 128 461 / 328 / 306, but 96 336 / 253 / 282 (its registers).  Below 1024 rows they gain nothing (512: 132 / 97 / 100).
  //  * dq, dk and dv, 16-bit, D = 128, 1024 rows and more, all keys allowed: of the whole backward pass 4 x 16 heads x 2048 x 4096
  //    1528 / 1099 / 1083 by dq's, 1793 / 1145 / 1100 by dk's and dv's; with a mask 4 (64 heads x 2048: 1183 / 818 / 930).
  //  * dq of float32, up to 512 rows: 2, since few rows to a head leave the last workgroup half empty -- 4096 x 131 x 131, D = 64 531 /
  //    605 / 641, 200 rows 662 / 660 / 685, 450 rows 1325 / 1294 / 1346.
  //  * dk and dv of float32, up to 512 keys of which not all are allowed: 2, whose workgroups end at once behind the allowed ones --
  //    4096 x 131 530 / 601 / 741, 512 x 450 1326 / 1357 / 1466; 16-bit 2048 x 4 x 401, D = 32 414 / 389 / 428, 512 x 450, D = 128 741 /
  //    559 / 600, so 4 there.
  static Cut cut_q(const AttendParams& p, bool dq) {
    const bool all = !p.list && !p.lengths;
    int mw = 4;
    if (sizeof(T) == 2 && p.rows >= 1024 && (dq ? all && p.dim > 96 : p.dim <= 64 || p.dim > 96)) mw = 8;
    if (sizeof(T) == 4 && dq && p.rows <= 512) mw = 2;
    return cut(p.rows, (p.k_len + Type<T>::ROWS - 1) / Type<T>::ROWS, (int64_t)p.batch * p.kv_heads, mw);
  }
  static Cut cut_k(const AttendParams& p) {
    const bool all = !p.list && !p.lengths;
    int mw = 4;
    if (sizeof(T) == 2 && all && p.dim > 96 && p.k_len >= 1024) mw = 8;
    if (sizeof(T) == 4 && !all && p.k_len <= 512) mw = 2;
    return cut(p.k_len, (p.rows + Type<T>::ROWS - 1) / Type<T>::ROWS, (int64_t)p.batch * p.kv_heads, mw);
  }
  // the partial statistics, up to where the partial results start (those are read 16 bytes at a time)
  static int64_t stats_bytes(int splits, int64_t rows) { return (splits * rows * 8 + 15) / 16 * 16; }
  static int64_t workspace(const AttendParams& p, bool backward) {
    const int64_t rows = (int64_t)p.batch * p.kv_heads * p.rows;
    const Cut q = cut_q(p, backward);
    if (!backward) return q.splits > 1 ? stats_bytes(q.splits, rows) + q.splits * rows * 4 * (int64_t)p.dim : 0;
    const Cut k = cut_k(p);
    const int64_t a = q.splits > 1 ? q.splits * rows * p.dim * 4 : 0;
    const int64_t b = k.splits > 1 ? k.splits * 2 * (int64_t)p.batch * p.k_len * p.kv_heads * p.dim * 4 : 0;
    return (rows * 4 + 255) / 256 * 256 + (a > b ? a : b);
  }
  static void set(AttendParams& p, const Cut& c, bool tail) {
    p.tiles = c.tiles;
    p.splits = c.splits;
    p.tail = tail;
    p.by_tiles = Divisor(c.tiles);
    p.by_splits = Divisor(c.splits);
    p.by_kv = Divisor(p.kv_heads);
    p.by_group = Divisor(p.group);
    p.by_die = Divisor((unsigned)(((int64_t)p.batch * p.kv_heads + 7) / 8));
  }
  // (a head's workgroups all meet on one die then, so there have to be enough heads for every die)
  static bool tail(const AttendParams& p) { return (p.list || p.lengths) && p.k_len <= 512 && (int64_t)p.batch * p.kv_heads >= 64; }
  static int grid(const AttendParams& p, const Cut& c, bool by_die, dim3& g) {
    const int64_t heads = (int64_t)p.batch * p.kv_heads, n = (int64_t)c.tiles * c.splits * (by_die ? (heads + 7) / 8 * 8 : heads);
    if (n * c.waves * 64 >= (int64_t)1 << 32) return policy_fail(PCT_ERR_UNSUPPORTED, "attention: more workgroups than a launch can hold");
    g = dim3((unsigned)n);
    return PCT_OK;
  }
  static int forward(AttendParams& p, char* ws, hipStream_t s) {
    const Cut c = cut_q(p, false);
    const int64_t rows = (int64_t)p.batch * p.kv_heads * p.rows;
    set(p, c, false);
    p.part_stats = (float2*)ws;
    p.part = (float*)(ws + stats_bytes(c.splits, rows));
    dim3 g;
    if (int rc = grid(p, c, false, g)) return rc;
    by_dim(p.dim, [&](auto d) {
      constexpr int DP = d.value, W = max_waves<T, DP>();
      // a lone wavefront or two are bound by what is in flight: smaller tiles let more of them onto a compute unit
      if (c.waves <= 2) launch<4 * Tile<T, DP, 32>::BYTES>(pct_attend_kernel<T, DP, W, 32>, g, c.waves, s, p);
      else launch<4 * Tile<T, DP>::BYTES>(pct_attend_kernel<T, DP, W, Type<T>::ROWS>, g, c.waves, s, p);
    });
    if (c.splits > 1) pct_attend_join_kernel<T><<<(unsigned)((rows * (p.dim / 4) + 255) / 256), 256, 0, s>>>(p);
    return policy_launched("attention kernel");
  }
  static int backward(AttendParams& p, char* ws, hipStream_t s) {
    const Cut q = cut_q(p, true), k = cut_k(p);
    const int64_t rows = (int64_t)p.batch * p.kv_heads * p.rows;
    p.delta = (float*)ws;
    p.part = (float*)(ws + (rows * 4 + 255) / 256 * 256);
    dim3 gq, gk;
    int rc = grid(p, q, false, gq);
    if (!rc) rc = grid(p, k, tail(p), gk);
    if (rc) return rc;
    by_dim(p.dim, [&](auto d) {
      constexpr int DP = d.value, W = max_waves<T, DP>();
      set(p, q, false);
      launch<4 * Tile<T, DP>::BYTES>(pct_attend_dq_kernel<T, DP, W>, gq, q.waves, s, p);
      if (q.splits > 1) {
        const int64_t n = (int64_t)p.batch * p.q_len * p.heads * p.dim;
        pct_attend_sum_kernel<T><<<(unsigned)((n / 4 + 255) / 256), 256, 0, s>>>(p.part, n, q.splits, n, (T*)p.dq, (T*)nullptr);
      }
      set(p, k, tail(p));
      launch<4 * Tile<T, DP>::BYTES>(pct_attend_dkv_kernel<T, DP, W>, gk, k.waves, s, p);
      if (k.splits > 1) {
        const int64_t n = (int64_t)p.batch * p.k_len * p.kv_heads * p.dim;
        pct_attend_sum_kernel<T><<<dim3((unsigned)((n / 4 + 255) / 256), 2), 256, 0, s>>>(p.part, 2 * n, k.splits, n, (T*)p.dk, (T*)p.dv);
      }
      if (p.list || p.lengths) {
        int chunks = 1;  // threads to a row
        while (chunks < 64 && 2 * chunks * 16 <= p.kv_heads * p.dim * (int)sizeof(T)) chunks *= 2;
        const int64_t per = p.k_len / (256 / chunks) / 8 + 1;
        constexpr int SLICE = 1 << 17;  // batches to a launch, which holds fewer than 2^32 threads
        for (int64_t b = 0; b < p.batch; b += SLICE)
          pct_attend_clear_kernel<T><<<dim3((unsigned)(p.batch - b < SLICE ? p.batch - b : SLICE), (unsigned)(per < 64 ? per : 64)), 256, 0, s>>>(p, chunks, (int)b);
      }
    });
    return policy_launched("attention gradient kernels");
  }
};

}  // namespace
}  // namespace pct
#endif
