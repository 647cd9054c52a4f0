// pct_choice.hip -- the masked choice that ends a policy: pick, log-probabilities with entropy and alternatives, gradient.
//
// A row x of logits allows choice j where its mask entry is not zero and x_j != -inf.  Over the allowed choices
//     M = max x,  s = sum e^(x - M),  t = sum e^(x - M) (x - M) log2 e,
//     log p_j = (x_j - M) - ln s,  H = ln s - ln 2 t / s,
// and the gradient, given d_g for the listed choices a_g (given ones and alternatives) and dH for the entropy, is
//     dx_j = sum_g d_g (1[j = a_g] - p_j) - dH p_j (log p_j + H).
// A row that allows nothing has H = 0, log p = 0 and a zero gradient.
//
// Forward: one pass.  A lane carries (M, s, t) of what it has seen and rescales when its maximum rises, 8 elements to a 16-byte
// load (two for float32), 4 loads in flight; lanes, wavefronts and workgroups are joined by rescaling to the common maximum.
// Sums are float32: a lane adds at most a few thousand terms, the rest is a tree.  Both passes are bound by HBM where rows x
// choices is large -- 8192 x 65536 bfloat16 240 us forward (4.5 TB/s, with some ten vector instructions to an element), 387 us
// backward (5.5 TB/s) -- and by latency where it is not: 64 x 50 3.7 us, 16 x 131072 with the 20 best 12.5 + 5.2 us for the join.
#include "pct_policy.cuh"

namespace pct {

// orders by value, the lower index first among equal values; 0 stands for "none"
__device__ __forceinline__ uint64_t choice_key(float v, int idx) {
  const uint32_t b = __float_as_uint(v + 0.0f);
  const uint32_t o = (b >> 31) ? ~b : (b | 0x80000000u);
  return ((uint64_t)o << 32) | (0xffffffffu - (uint32_t)idx);
}
__device__ __forceinline__ float key_value(uint64_t k) {
  const uint32_t o = (uint32_t)(k >> 32);
  return __uint_as_float((o >> 31) ? (o & 0x7fffffffu) : ~o);
}
__device__ __forceinline__ int key_index(uint64_t k) { return (int)(0xffffffffu - (uint32_t)k); }

// (x - M) log2 e below this adds nothing in float32; the bound keeps 0 * inf out of the sums
constexpr float kFloor = -200.f;
__device__ __forceinline__ float rel(float x, float m) { return (x - m) * kLog2e; }

struct Sums {
  float m, s, t;
  __device__ __forceinline__ void start() { m = -INFINITY; s = 0.f; t = 0.f; }
  __device__ __forceinline__ void raise(float to) {  // to >= m, to > -inf
    const float d = fmaxf(rel(m, to), kFloor), f = __builtin_amdgcn_exp2f(d);
    t = fmaf(d, s, t) * f;
    s = s * f;
    m = to;
  }
  __device__ __forceinline__ void add(float x, float at) {  // at = m, or 0 while nothing is allowed
    const float y = rel(x, at), e = __builtin_amdgcn_exp2f(y);
    s += e;
    t = fmaf(e, fmaxf(y, kFloor), t);
  }
};

// ---- the best K <= 64 keys of a wavefront, lane i holding the i-th ----
__device__ __forceinline__ uint64_t shfl_u64(uint64_t v, int lane) { return (uint64_t)__shfl((unsigned long long)v, lane); }
__device__ __forceinline__ uint64_t shfl_xor_u64(uint64_t v, int m) { return (uint64_t)__shfl_xor((unsigned long long)v, m); }

__device__ __forceinline__ uint64_t sort64(uint64_t k, int lane) {
#pragma unroll
  for (int n = 2; n <= 64; n *= 2)
#pragma unroll
    for (int j = n / 2; j; j /= 2) {
      const uint64_t o = shfl_xor_u64(k, j);
      const bool hi = ((lane & j) == 0) == ((lane & n) == 0);
      k = (o > k) == hi ? o : k;
    }
  return k;
}
__device__ __forceinline__ uint64_t merge64(uint64_t a, uint64_t b, int lane) {  // both in falling order
  const uint64_t r = shfl_u64(b, 63 - lane);
  uint64_t k = r > a ? r : a;
#pragma unroll
  for (int j = 32; j; j /= 2) {
    const uint64_t o = shfl_xor_u64(k, j);
    k = (o > k) == ((lane & j) == 0) ? o : k;
  }
  return k;
}
struct Best {
  uint64_t list, least;  // least: the K-th key, in every lane
  __device__ __forceinline__ void start() { list = 0; least = 0; }
  __device__ __forceinline__ void offer(uint64_t key, int K, int lane) {  // one key (or 0) per lane
    uint64_t in = __ballot(key > least);
    if (!in) return;
    if (__popcll(in) > 3) {
      list = merge64(list, sort64(key, lane), lane);
    } else {
      for (; in; in &= in - 1) {
        const uint64_t x = readlane_u64(key, __ffsll((unsigned long long)in) - 1);
        const uint64_t up = (uint64_t)__shfl_up((unsigned long long)list, 1);
        const int pos = __popcll(__ballot(list > x));
        list = lane < pos ? list : (lane == pos ? x : up);
      }
    }
    least = readlane_u64(list, K - 1);
  }
};

struct ChoiceParams {
  const void* x;
  int64_t x_row;
  Mask mask;
  const float* noise;
  int64_t noise_row;
  int rows, choices, given_count, top, splits, chunk, row0;
  const int64_t* given;
  int64_t* actions;
  float *log_probs, *entropy, *top_log_probs;
  int64_t* top_actions;
  float4* stats;
  char* ws;
};

struct Part {  // what a workgroup leaves for the join, followed by `top` keys
  float m, s, t, pad;
  uint64_t key, pad2;
};
__host__ __device__ __forceinline__ int64_t part_bytes(int top) { return (int64_t)sizeof(Part) + 8 * (int64_t)top; }

enum { PICK = 0, LOGP = 1, LOGP_TOP = 2 };
enum { M_NONE = 0, M_BYTES = 1, M_ANY = 2 };  // how a mask is read: not at all, 8 adjacent bytes at once, one by one

// one entry of the mask (of bytes without a look at its type: with it the 16-bit variants took 243 registers, and 4000 x 30000
// bfloat16 208 us in place of 99)
template <int MASK>
__device__ __forceinline__ bool allows(const Mask& m, int64_t row, int64_t i) {
  return MASK == M_BYTES ? ((const uint8_t*)m.p)[row * m.row + i] != 0 : m.at(row, i);
}

// a whole wavefront writes what a row's sums, best key and best list say
template <typename T, int MASK, int MODE>
__device__ __forceinline__ void finish_row(const ChoiceParams& p, int row, float m, float s, float t, uint64_t key, uint64_t list, int lane) {
  const bool empty = m == -INFINITY && s == 0.f;
  const float l2 = empty ? 0.f : log2f(s), ls = empty ? 0.f : logf(s);
  const float H = empty ? 0.f : ls - kLn2 * (t / s);
  const T* x = (const T*)p.x + (int64_t)row * p.x_row;
  if (lane == 0) {
    if (p.entropy) p.entropy[row] = H;
    if (MODE != PICK && p.stats) p.stats[row] = make_float4(empty ? INFINITY : m, l2, H, 0.f);
  }
  if (MODE == PICK) {
    if (lane == 0) {
      const int a = empty || !key ? 0 : key_index(key);
      p.actions[row] = a;
      if (p.log_probs) p.log_probs[row] = empty ? 0.f : ((float)x[a] - m) - ls;
    }
    return;
  }
  for (int g = lane; g < p.given_count; g += 64) {
    const int64_t id = p.given[(int64_t)row * p.given_count + g];
    float v = 0.f;
    if (id < -1 || id >= p.choices) v = NAN;
    else if (id >= 0 && !empty) v = MASK && !p.mask.at(row, id) ? -INFINITY : ((float)x[id] - m) - ls;
    p.log_probs[(int64_t)row * p.given_count + g] = v;
  }
  if (MODE == LOGP_TOP && lane < p.top) {
    const int64_t o = (int64_t)row * p.top + lane;
    p.top_log_probs[o] = list ? (key_value(list) - m) - ls : -INFINITY;
    p.top_actions[o] = list ? key_index(list) : -1;
  }
}

// TEAM wavefronts to a row.  TEAM 1: four rows to a workgroup, no barrier -- rows of up to 2048.  TEAM 8: one row, or one of
// p.splits chunks of one, to a workgroup.  VEC 1 (adjacent lanes read adjacent elements) is for rows of up to 128, which 8
// elements to a lane would leave to a few lanes.
template <typename T, int MASK, int MODE, int VEC, int TEAM>
__global__ __launch_bounds__(TEAM == 1 ? 256 : 64 * TEAM) void pct_choice_kernel(ChoiceParams p) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int row = p.row0 + (TEAM == 1 ? (int)blockIdx.x * 4 + wave : (int)blockIdx.x);
  if (row >= p.rows) return;
  const int c0 = TEAM == 1 ? 0 : (int)blockIdx.y * p.chunk;
  const int c1 = TEAM == 1 ? p.choices : min(p.choices - c0, p.chunk) + c0;
  constexpr int U = VEC == 1 || MODE == LOGP_TOP ? 2 : 4, STEP = TEAM * 64 * VEC;
  const T* x = (const T*)p.x + (int64_t)row * p.x_row;
  const float* nz = p.noise ? p.noise + (int64_t)row * p.noise_row : nullptr;
  Sums a;
  a.start();
  Best best;
  best.start();
  float score = 0.f;
  int pick = -1;
  // 16-bit rows: the next step's logits (and bytes of the mask) are on their way while this step's are worked on.  8192 x 65536
  // bfloat16: 265 us without, 240 so (4.5 TB/s); no gain where a list is kept (the sorts hide it) or for float32 (twice the bytes to
  // the same work).
  constexpr bool AHEAD = VEC == 8 && sizeof(T) == 2 && MODE != LOGP_TOP;
  // (the mask's only without noise, whose loads take the registers: 4000 x 30000 98 -> 87 us, but 5000 x 20000 with noise 133 -> 147)
  constexpr bool MASK_AHEAD = AHEAD && MASK == M_BYTES && MODE == LOGP;
  using Raw = typename Vec8<T>::raw;
  Raw ahead[AHEAD ? U : 1];
  Bytes8 ahead_mask[MASK_AHEAD ? U : 1];
  auto fetch = [&](int64_t base) {
    if constexpr (AHEAD) {
      const int64_t i0 = base + (int64_t)(TEAM == 1 ? lane : (int)threadIdx.x) * VEC;
#pragma unroll
      for (int u = 0; u < U; u++)
        if (i0 + u * STEP + VEC <= c1) {
          ahead[u] = *(const Raw*)(x + i0 + u * STEP);
          if constexpr (MASK_AHEAD) ahead_mask[u] = *(const Bytes8*)((const uint8_t*)p.mask.p + (int64_t)row * p.mask.row + i0 + u * STEP);
        }
    }
  };
  fetch(c0);
  // (the loop runs the same number of times in every lane: the top list needs whole wavefronts)
#pragma unroll 1
  for (int64_t base = c0; base < c1; base += (int64_t)STEP * U) {
    float v[U][VEC];
    const int64_t i0 = base + (int64_t)(TEAM == 1 ? lane : (int)threadIdx.x) * VEC;
#pragma unroll
    for (int u = 0; u < U; u++) {
      const int64_t i = i0 + u * STEP;
      bool whole = false;
      if constexpr (VEC == 8) {
        if (i + VEC <= c1) {
          whole = true;
          if constexpr (AHEAD) unpack8<T>(ahead[u], v[u]);
          else load8(x + i, v[u]);
          if (MASK == M_BYTES) {
            Bytes8 b;
            if constexpr (MASK_AHEAD) b = ahead_mask[u];
            else b = *(const Bytes8*)((const uint8_t*)p.mask.p + (int64_t)row * p.mask.row + i);
#pragma unroll
            for (int e = 0; e < VEC; e++) v[u][e] = (b.w[e / 4] & (0xffu << (8 * (e % 4)))) ? v[u][e] : -INFINITY;
          } else if (MASK == M_ANY) {
#pragma unroll
            for (int e = 0; e < VEC; e++) v[u][e] = p.mask.at(row, i + e) ? v[u][e] : -INFINITY;
          }
        }
      }
      if (!whole) {
#pragma unroll
        for (int e = 0; e < VEC; e++) {
          v[u][e] = -INFINITY;
          if (i + e < c1) {
            v[u][e] = (float)x[i + e];
            if (MASK && !allows<MASK>(p.mask, row, i + e)) v[u][e] = -INFINITY;
          }
        }
      }
    }
    fetch(base + (int64_t)STEP * U);
    float top = -INFINITY;
#pragma unroll
    for (int u = 0; u < U; u++)
#pragma unroll
      for (int e = 0; e < VEC; e++) top = fmaxf(top, v[u][e]);
    if (top > a.m) a.raise(top);
    const float at = a.m == -INFINITY ? 0.f : a.m;
#pragma unroll
    for (int u = 0; u < U; u++)
#pragma unroll
      for (int e = 0; e < VEC; e++) a.add(v[u][e], at);
    if constexpr (MODE == PICK) {
#pragma unroll
      for (int u = 0; u < U; u++) {
        const int64_t i = i0 + u * STEP;
        float n[VEC];
#pragma unroll
        for (int e = 0; e < VEC; e++) n[e] = 0.f;
        if (nz) {
          bool whole = false;
          if constexpr (VEC == 8) {
            if (i + VEC <= c1) { whole = true; load8(nz + i, n); }
          }
          if (!whole) {
#pragma unroll
            for (int e = 0; e < VEC; e++)
              if (i + e < c1) n[e] = nz[i + e];
          }
        }
#pragma unroll
        for (int e = 0; e < VEC; e++) {
          const float sc = v[u][e] + n[e];
          if (v[u][e] != -INFINITY && (pick < 0 || sc > score)) { score = sc; pick = (int)(i + e); }
        }
      }
    }
    if constexpr (MODE == LOGP_TOP) {
      // An empty list starts with each lane's own best: the K-th of these 64 bounds the K-th of all, and little is left above it.
      // Then a comparison of values says whether an element may come in (a NaN may), and only those are made into keys.
      uint64_t mine = 0;
      float bar = best.least ? key_value(best.least) : -INFINITY;
      if (__ballot(!(top < bar))) {
        if (!best.least) {
#pragma unroll
          for (int u = 0; u < U; u++)
#pragma unroll
            for (int e = 0; e < VEC; e++) {
              const uint64_t k = v[u][e] != -INFINITY ? choice_key(v[u][e], (int)(i0 + u * STEP + e)) : 0;
              mine = k > mine ? k : mine;
            }
          best.offer(mine, p.top, lane);
          bar = best.least ? key_value(best.least) : -INFINITY;
        }
#pragma unroll
        for (int u = 0; u < U; u++)
#pragma unroll
          for (int e = 0; e < VEC; e++) {
            const bool in = !(v[u][e] < bar) && v[u][e] != -INFINITY;
            if (__ballot(in)) {
              const uint64_t k = choice_key(v[u][e], (int)(i0 + u * STEP + e));
              best.offer(in && k != mine ? k : 0, p.top, lane);
              bar = best.least ? key_value(best.least) : -INFINITY;
            }
          }
      }
    }
  }
  // the lanes' sums at the wavefront's maximum
  uint64_t key = MODE == PICK ? wave_max_u64(pick < 0 ? 0 : choice_key(score, pick)) : 0;
  float m = wave_max(a.m);
  if (m > -INFINITY) a.raise(m);
  float s = wave_sum(a.s), t = wave_sum(a.t);
  if constexpr (TEAM > 1) {
    __shared__ float sm[TEAM], ss[TEAM], st[TEAM];
    __shared__ uint64_t sk[TEAM];
    __shared__ uint64_t sl[MODE == LOGP_TOP ? TEAM * 64 : 1];
    if (lane == 0) { sm[wave] = m; ss[wave] = s; st[wave] = t; sk[wave] = key; }
    if constexpr (MODE == LOGP_TOP) {
      for (int half = TEAM / 2; half; half /= 2) {
        if (wave >= half && wave < 2 * half) sl[wave * 64 + lane] = best.list;
        __syncthreads();
        if (wave < half) best.list = merge64(best.list, sl[(wave + half) * 64 + lane], lane);
      }
    }
    __syncthreads();
    if (wave) return;
    a.m = lane < TEAM ? sm[lane % TEAM] : -INFINITY;
    a.s = lane < TEAM ? ss[lane % TEAM] : 0.f;
    a.t = lane < TEAM ? st[lane % TEAM] : 0.f;
    if (MODE == PICK) key = wave_max_u64(lane < TEAM ? sk[lane % TEAM] : 0);
    m = wave_max(a.m);
    if (m > -INFINITY) a.raise(m);
    s = wave_sum(a.s);
    t = wave_sum(a.t);
    if (p.splits > 1) {
      char* w = p.ws + ((int64_t)row * p.splits + blockIdx.y) * part_bytes(p.top);
      if (lane == 0) {
        Part* q = (Part*)w;
        q->m = m; q->s = s; q->t = t; q->key = key;
      }
      if (MODE == LOGP_TOP && lane < p.top) ((uint64_t*)(w + sizeof(Part)))[lane] = best.list;
      return;
    }
  }
  if (MODE == LOGP_TOP && lane >= p.top) best.list = 0;
  finish_row<T, MASK, MODE>(p, row, m, s, t, key, best.list, lane);
}

// joins the chunks of a row (at most 64, a lane to each); with a top list 8 wavefronts merge the chunks' lists as a tree
template <typename T, int MASK, int MODE>
__global__ __launch_bounds__(MODE == LOGP_TOP ? 512 : 64) void pct_choice_join_kernel(ChoiceParams p) {
  constexpr int TEAM = MODE == LOGP_TOP ? 8 : 1;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, row = p.row0 + blockIdx.x;
  const char* w = p.ws + (int64_t)row * p.splits * part_bytes(p.top);
  uint64_t list = 0;
  if constexpr (MODE == LOGP_TOP) {
    __shared__ uint64_t sl[TEAM * 64];
    for (int c = wave; c < p.splits; c += TEAM) {
      const uint64_t o = lane < p.top ? ((const uint64_t*)(w + c * part_bytes(p.top) + sizeof(Part)))[lane] : 0;
      list = c < TEAM ? o : merge64(list, o, lane);
    }
    for (int half = TEAM / 2; half; half /= 2) {
      if (wave >= half && wave < 2 * half) sl[wave * 64 + lane] = list;
      __syncthreads();
      if (wave < half) list = merge64(list, sl[(wave + half) * 64 + lane], lane);
    }
    if (wave) return;
    if (lane >= p.top) list = 0;
  }
  Sums a;
  a.start();
  uint64_t key = 0;
  if (lane < p.splits) {
    const Part* q = (const Part*)(w + lane * part_bytes(p.top));
    a.m = q->m; a.s = q->s; a.t = q->t; key = q->key;
  }
  const float m = wave_max(a.m);
  if (m > -INFINITY) a.raise(m);
  const float s = wave_sum(a.s), t = wave_sum(a.t);
  if (MODE == PICK) key = wave_max_u64(key);
  finish_row<T, MASK, MODE>(p, row, m, s, t, key, list, lane);
}

struct ChoiceGradParams {
  const void* x;
  int64_t x_row;
  Mask mask;
  int rows, choices, given_count, top, chunk, row0;
  const int64_t *given, *top_actions;
  const float4* stats;
  const float *d_log_probs, *d_entropy, *d_top;
  void* dx;
};

// Backward: reads the logits once more and writes the gradient -- the statistics of the forward pass make the rows' chunks
// independent.  With A = sum_g d_g + dH H and B = dH ln 2 every allowed element is -p (A + B log2 p); the few listed choices
// are then computed again with their own d added (in float32, rounded once) and written over, after a barrier that orders the
// two stores.  A choice that is listed twice is written by its first entry, which adds up all of its entries in order.
template <typename T, int MASK, int VEC, int TEAM>
__global__ __launch_bounds__(TEAM == 1 ? 256 : 64 * TEAM) void pct_choice_grad_kernel(ChoiceGradParams p) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int row = p.row0 + (TEAM == 1 ? (int)blockIdx.x * 4 + wave : (int)blockIdx.x);
  if (row >= p.rows) return;
  const int c0 = TEAM == 1 ? 0 : (int)blockIdx.y * p.chunk;
  const int c1 = TEAM == 1 ? p.choices : min(p.choices - c0, p.chunk) + c0;
  constexpr int U = VEC == 1 ? 2 : 4, STEP = TEAM * 64 * VEC;
  const T* x = (const T*)p.x + (int64_t)row * p.x_row;
  T* dx = (T*)p.dx + (int64_t)row * p.choices;
  const float4 st = p.stats[row];
  const float m = st.x, l2 = st.y, H = st.z;
  const bool empty = m == INFINITY && l2 == 0.f;
  // the listed choices: two to a lane at most
  int id[2];
  float d[2], sum = 0.f;
  const int listed = p.given_count + p.top;
#pragma unroll
  for (int h = 0; h < 2; h++) {
    const int e = lane + 64 * h;
    id[h] = -1;
    d[h] = 0.f;
    if (e < listed && !empty) {
      const bool g = e < p.given_count;
      const float* src = g ? p.d_log_probs : p.d_top;
      if (src) {
        const int64_t j = g ? p.given[(int64_t)row * p.given_count + e] : p.top_actions[(int64_t)row * p.top + e - p.given_count];
        if (j >= 0 && j < p.choices && (float)x[j] != -INFINITY && (!MASK || p.mask.at(row, j))) {
          id[h] = (int)j;
          d[h] = g ? src[(int64_t)row * p.given_count + e] : src[(int64_t)row * p.top + e - p.given_count];
        }
      }
    }
    if (64 * h < listed) sum += wave_sum(d[h]);
  }
  const float dH = p.d_entropy && !empty ? p.d_entropy[row] : 0.f;
  const float A = sum + dH * H, B = dH * kLn2;
  auto slope = [&](float v) {
    const float y = rel(v, m) - l2;
    return -__builtin_amdgcn_exp2f(y) * fmaf(B, fmaxf(y, kFloor), A);
  };
  for (int64_t i0 = c0 + (int64_t)(TEAM == 1 ? lane : (int)threadIdx.x) * VEC; i0 < c1; i0 += (int64_t)STEP * U) {
    float v[U][VEC];
#pragma unroll
    for (int u = 0; u < U; u++) {
      const int64_t i = i0 + u * STEP;
      bool whole = false;
      if constexpr (VEC == 8) {
        if (i + VEC <= c1) {
          whole = true;
          load8(x + i, v[u]);
          if (MASK == M_BYTES) {
            const Bytes8 b = *(const Bytes8*)((const uint8_t*)p.mask.p + (int64_t)row * p.mask.row + i);
#pragma unroll
            for (int e = 0; e < VEC; e++) v[u][e] = (b.w[e / 4] & (0xffu << (8 * (e % 4)))) ? v[u][e] : -INFINITY;
          } else if (MASK == M_ANY) {
#pragma unroll
            for (int e = 0; e < VEC; e++) v[u][e] = p.mask.at(row, i + e) ? v[u][e] : -INFINITY;
          }
        }
      }
      if (!whole) {
#pragma unroll
        for (int e = 0; e < VEC; e++) {
          v[u][e] = -INFINITY;
          if (i + e < c1) {
            v[u][e] = (float)x[i + e];
            if (MASK && !allows<MASK>(p.mask, row, i + e)) v[u][e] = -INFINITY;
          }
        }
      }
    }
#pragma unroll
    for (int u = 0; u < U; u++) {
      const int64_t i = i0 + u * STEP;
#pragma unroll
      for (int e = 0; e < VEC; e++) v[u][e] = v[u][e] == -INFINITY || empty ? 0.f : slope(v[u][e]);
      bool whole = false;
      if constexpr (VEC == 8) {
        if (i + VEC <= c1) { whole = true; store8(dx + i, v[u]); }
      }
      if (!whole) {
#pragma unroll
        for (int e = 0; e < VEC; e++)
          if (i + e < c1) dx[i + e] = (T)v[u][e];
      }
    }
  }
  if (!listed) return;
  if constexpr (TEAM > 1) {
    __syncthreads();
    if (wave) return;
  } else {
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "workgroup");
    __builtin_amdgcn_wave_barrier();
  }
  float total[2] = {0.f, 0.f};
  bool first[2] = {true, true};
  for (int e = 0; e < listed; e++) {
    const int j = e < 64 ? __builtin_amdgcn_readlane(id[0], e) : __builtin_amdgcn_readlane(id[1], e - 64);
    const float dj = __int_as_float(e < 64 ? __builtin_amdgcn_readlane(__float_as_int(d[0]), e) : __builtin_amdgcn_readlane(__float_as_int(d[1]), e - 64));
#pragma unroll
    for (int h = 0; h < 2; h++)
      if (j == id[h]) {
        total[h] += dj;
        if (e < lane + 64 * h) first[h] = false;
      }
  }
#pragma unroll
  for (int h = 0; h < 2; h++)
    if (id[h] >= c0 && id[h] < c1 && first[h]) dx[id[h]] = (T)(slope((float)x[id[h]]) + total[h]);
}

namespace {
// Rows of more than 2048 choices are cut until about four workgroups of 8 wavefronts per compute unit stand ready, in chunks of
// at least 4096 (a workgroup's fixed costs are those of about 2000 elements) and, for the join's one lane to a chunk, at most 64.
int choice_splits(int rows, int choices) {
  if (choices <= 2048) return 1;
  int64_t s = (1024 + (int64_t)rows - 1) / rows;
  const int64_t most = ((int64_t)choices + 4095) / 4096;
  s = s < most ? s : most;
  return s < 1 ? 1 : (s > 64 ? 64 : (int)s);
}
int choice_chunk(int choices, int splits) {  // a multiple of 512 unless it is the whole row
  const int64_t c = (((int64_t)choices + splits - 1) / splits + 511) / 512 * 512;
  return c < choices ? (int)c : choices;
}

constexpr int SLICE = 1 << 22;  // rows to a launch, which holds fewer than 2^32 threads; a multiple of a workgroup's rows

template <typename T, int MASK, int MODE>
void launch_choice(ChoiceParams& p, hipStream_t s) {
  for (p.row0 = 0; p.row0 < p.rows; p.row0 += SLICE) {
    const int n = p.rows - p.row0 < SLICE ? p.rows - p.row0 : SLICE;
    if (p.choices <= 128) {
      pct_choice_kernel<T, MASK, MODE, 1, 1><<<(n + 3) / 4, 256, 0, s>>>(p);
    } else if (p.choices <= 2048) {
      pct_choice_kernel<T, MASK, MODE, 8, 1><<<(n + 3) / 4, 256, 0, s>>>(p);
    } else {
      pct_choice_kernel<T, MASK, MODE, 8, 8><<<dim3(n, p.splits), 512, 0, s>>>(p);
      if (p.splits > 1) pct_choice_join_kernel<T, MASK, MODE><<<n, MODE == LOGP_TOP ? 512 : 64, 0, s>>>(p);
    }
    if (p.rows - p.row0 <= SLICE) return;  // (row0 + SLICE may pass 2^31)
  }
}
template <typename T, int MASK>
void launch_choice(ChoiceParams& p, int mode, hipStream_t s) {
  if (mode == PICK) launch_choice<T, MASK, PICK>(p, s);
  else if (mode == LOGP) launch_choice<T, MASK, LOGP>(p, s);
  else launch_choice<T, MASK, LOGP_TOP>(p, s);
}
template <typename T>
void launch_choice(ChoiceParams& p, int mode, hipStream_t s) {
  if (!p.mask.p) launch_choice<T, M_NONE>(p, mode, s);
  else if (p.mask.type == PCT_MASK_U8 && p.mask.col == 1) launch_choice<T, M_BYTES>(p, mode, s);
  else launch_choice<T, M_ANY>(p, mode, s);
}
template <typename T, int MASK>
void launch_grad(ChoiceGradParams& p, hipStream_t s) {
  const int splits = choice_splits(p.rows, p.choices);
  p.chunk = choice_chunk(p.choices, splits);
  for (p.row0 = 0; p.row0 < p.rows; p.row0 += SLICE) {
    const int n = p.rows - p.row0 < SLICE ? p.rows - p.row0 : SLICE;
    if (p.choices <= 128) pct_choice_grad_kernel<T, MASK, 1, 1><<<(n + 3) / 4, 256, 0, s>>>(p);
    else if (p.choices <= 2048) pct_choice_grad_kernel<T, MASK, 8, 1><<<(n + 3) / 4, 256, 0, s>>>(p);
    else pct_choice_grad_kernel<T, MASK, 8, 8><<<dim3(n, splits), 512, 0, s>>>(p);
    if (p.rows - p.row0 <= SLICE) return;
  }
}
template <typename T>
void launch_grad(ChoiceGradParams& p, hipStream_t s) {
  if (!p.mask.p) launch_grad<T, M_NONE>(p, s);
  else if (p.mask.type == PCT_MASK_U8 && p.mask.col == 1) launch_grad<T, M_BYTES>(p, s);
  else launch_grad<T, M_ANY>(p, s);
}

template <typename C>
int check_choice(const C* c, const char* what) {
  if (!c || c->struct_size != (int)sizeof(C)) return policy_fail(PCT_ERR_INVALID_ARG, what);
  if (c->dtype < PCT_F32 || c->dtype > PCT_F16) return policy_fail(PCT_ERR_INVALID_ARG, "unknown dtype of the logits");
  if (c->rows < 0 || c->choices < 1) return policy_fail(PCT_ERR_INVALID_ARG, "rows must be >= 0 and choices >= 1");
  if (c->given_count < 0 || c->given_count > PCT_CHOICE_MAX_GIVEN || c->top < 0 || c->top > PCT_CHOICE_MAX_TOP)
    return policy_fail(PCT_ERR_INVALID_ARG, "given_count and top must be 0 .. 64");
  if (c->mask && (c->mask_type < PCT_MASK_U8 || c->mask_type > PCT_MASK_I32)) return policy_fail(PCT_ERR_INVALID_ARG, "unknown mask type");
  if (c->rows && (!c->logits || (c->given_count && !c->given))) return policy_fail(PCT_ERR_INVALID_ARG, "null logits or given choices");
  return PCT_OK;
}

int run_choice(const pct_choice* c, int mode, hipStream_t s) {
  if (!c->rows) return PCT_OK;
  ChoiceParams p = {};
  p.x = c->logits; p.x_row = c->logits_row;
  p.mask = Mask{c->mask, c->mask_row, c->mask_col, c->mask_type};
  p.noise = c->noise; p.noise_row = c->noise_row;
  p.rows = c->rows; p.choices = c->choices; p.given_count = c->given_count; p.top = mode == PICK ? 0 : c->top;
  p.given = c->given; p.actions = c->actions; p.log_probs = c->log_probs; p.entropy = c->entropy;
  p.top_log_probs = c->top_log_probs; p.top_actions = c->top_actions; p.stats = (float4*)c->stats;
  p.splits = choice_splits(c->rows, c->choices);
  p.chunk = choice_chunk(c->choices, p.splits);
  p.ws = (char*)c->workspace;
  if (p.splits > 1 && (!c->workspace || c->workspace_bytes < pct_choice_workspace(c->rows, c->choices, p.top)))
    return policy_fail(PCT_ERR_INVALID_ARG, "the workspace is smaller than pct_choice_workspace() says");
  if (c->dtype == PCT_F32) launch_choice<float>(p, mode, s);
  else if (c->dtype == PCT_BF16) launch_choice<bf16>(p, mode, s);
  else launch_choice<f16>(p, mode, s);
  return policy_launched("choice kernel");
}
}  // namespace
}  // namespace pct

extern "C" {
int64_t pct_choice_workspace(int32_t rows, int32_t choices, int32_t top) {
  if (rows < 1 || choices < 1 || top < 0) return 0;
  const int s = pct::choice_splits(rows, choices);
  return s > 1 ? (int64_t)rows * s * pct::part_bytes(top) : 0;
}

int pct_choice_pick(const pct_choice* c, void* stream) {
  int rc = pct::check_choice(c, "pct_choice size mismatch");
  if (rc) return rc;
  if (c->rows && !c->actions) return pct::policy_fail(PCT_ERR_INVALID_ARG, "pick: null actions");
  return pct::run_choice(c, pct::PICK, (hipStream_t)stream);
}

int pct_choice_log_probs(const pct_choice* c, void* stream) {
  int rc = pct::check_choice(c, "pct_choice size mismatch");
  if (rc) return rc;
  if (c->rows && ((c->given_count && !c->log_probs) || (c->top && (!c->top_log_probs || !c->top_actions))))
    return pct::policy_fail(PCT_ERR_INVALID_ARG, "log_probs: null outputs");
  return pct::run_choice(c, c->top ? pct::LOGP_TOP : pct::LOGP, (hipStream_t)stream);
}

int pct_choice_backward(const pct_choice_grad* c, void* stream) {
  int rc = pct::check_choice(c, "pct_choice_grad size mismatch");
  if (rc || !c->rows) return rc;
  if (!c->stats || !c->d_logits || (c->top && !c->top_actions)) return pct::policy_fail(PCT_ERR_INVALID_ARG, "backward: null statistics or outputs");
  pct::ChoiceGradParams p = {};
  p.x = c->logits; p.x_row = c->logits_row;
  p.mask = pct::Mask{c->mask, c->mask_row, c->mask_col, c->mask_type};
  p.rows = c->rows; p.choices = c->choices; p.given_count = c->given_count; p.top = c->top;
  p.given = c->given; p.top_actions = c->top_actions; p.stats = (const float4*)c->stats;
  p.d_log_probs = c->d_log_probs; p.d_entropy = c->d_entropy; p.d_top = c->d_top_log_probs;
  p.dx = c->d_logits;
  hipStream_t s = (hipStream_t)stream;
  if (c->dtype == PCT_F32) pct::launch_grad<float>(p, s);
  else if (c->dtype == PCT_BF16) pct::launch_grad<pct::bf16>(p, s);
  else pct::launch_grad<pct::f16>(p, s);
  return pct::policy_launched("choice gradient kernel");
}
}
