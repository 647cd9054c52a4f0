// pct_attend.hip -- attention: the list of allowed keys, the checks of the C entries, the choice of the element type.
#include "pct_attend.cuh"

namespace pct {
#define PCT_ATTEND_TYPE(n)                                             \
  int64_t attend_workspace_##n(const AttendParams& p, bool backward); \
  int attend_forward_##n(AttendParams& p, char* ws, hipStream_t s);   \
  int attend_backward_##n(AttendParams& p, char* ws, hipStream_t s);
PCT_ATTEND_TYPE(f32)
PCT_ATTEND_TYPE(bf16)
PCT_ATTEND_TYPE(f16)

namespace {
constexpr int SLICE = 1 << 22;  // batches to a launch, which holds fewer than 2^32 threads

// A batch's keys in the order: allowed ones, then the others, both rising; the count of the allowed ones in front.  One workgroup
// to a batch reads its mask twice (the second time from L2): to count, and to place.  2048 x 401 entries, a column of 36-byte rows:
// 13 us, bound by the 64-byte lines that hold one entry or two.
__global__ __launch_bounds__(256) void pct_attend_list_kernel(Mask mask, AttendParams p, int32_t* lists, int b0) {
  __shared__ int part[4];
  const int b = b0 + blockIdx.x, tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  int32_t* out = lists + (int64_t)b * (p.k_len + 1);
  p.list = nullptr;
  const int limit = allowed_keys(p, b);  // by the lengths
  int mine = 0;
  for (int j = tid; j < limit; j += 256) mine += mask.at(b, j) ? 1 : 0;
  for (int o = 32; o; o /= 2) mine += __shfl_xor(mine, o);
  if (lane == 0) part[wave] = mine;
  __syncthreads();
  const int n = part[0] + part[1] + part[2] + part[3];
  __syncthreads();
  if (tid == 0) out[0] = n;
  int before = 0;  // allowed keys before this step's
  for (int j0 = 0; j0 < p.k_len; j0 += 256) {
    const int j = j0 + tid;
    const bool in = j < limit && mask.at(b, j);
    const uint64_t bits = __ballot(in);
    if (lane == 0) part[wave] = __popcll(bits);
    __syncthreads();
    int at = before + __popcll(bits & (((uint64_t)1 << lane) - 1));
    for (int k = 0; k < 4; k++) {
      if (k < wave) at += part[k];
      before += part[k];
    }
    if (j < p.k_len) out[1 + (in ? at : n + j - at)] = j;
    __syncthreads();
  }
}

bool aligned16(const void* p, const int64_t* strides, int size) {
  if ((uintptr_t)p % 16) return false;
  for (int i = 0; i < 3; i++)
    if (strides[i] * size % 16) return false;
  return true;
}

int check_attention(const pct_attention* a, AttendParams& p) {
  if (!a || a->struct_size != (int)sizeof(pct_attention)) return policy_fail(PCT_ERR_INVALID_ARG, "pct_attention size mismatch");
  if (a->dtype < PCT_F32 || a->dtype > PCT_F16) return policy_fail(PCT_ERR_INVALID_ARG, "attention: unknown dtype");
  if (a->batch < 0 || a->q_len < 0 || a->k_len < 0 || a->heads < 1 || a->kv_heads < 1 || a->heads % a->kv_heads)
    return policy_fail(PCT_ERR_INVALID_ARG, "attention: bad sizes (heads must be a multiple of kv_heads)");
  if (a->dim < 8 || a->dim > 128 || a->dim % 8) return policy_fail(PCT_ERR_UNSUPPORTED, "attention: dim must be a multiple of 8 up to 128");
  if (!(a->scale > 0.f) || a->scale > 1e30f) return policy_fail(PCT_ERR_INVALID_ARG, "attention: scale must be positive and finite");
  const int64_t rows = (int64_t)a->q_len * (a->heads / a->kv_heads);
  if (rows >= (int64_t)1 << 29 || a->k_len >= 1 << 29) return policy_fail(PCT_ERR_UNSUPPORTED, "attention: lengths beyond 2^29 rows");
  if (a->key_mask && (a->mask_type < PCT_MASK_U8 || a->mask_type > PCT_MASK_I32)) return policy_fail(PCT_ERR_INVALID_ARG, "unknown mask type");
  if (a->key_lengths && a->lengths_type != 4 && a->lengths_type != 8) return policy_fail(PCT_ERR_INVALID_ARG, "key lengths must be int32 or int64");
  p = AttendParams{};
  p.q = a->q; p.k = a->k; p.v = a->v; p.d_out = a->d_out; p.o = a->out;
  for (int i = 0; i < 3; i++) { p.qs[i] = a->q_stride[i]; p.ks[i] = a->k_stride[i]; p.vs[i] = a->v_stride[i]; p.ds[i] = a->d_out_stride[i]; }
  p.list = a->key_mask ? a->key_list : nullptr;
  p.lengths = a->key_lengths; p.lengths_type = a->lengths_type;
  p.batch = a->batch; p.q_len = a->q_len; p.k_len = a->k_len; p.heads = a->heads; p.kv_heads = a->kv_heads; p.dim = a->dim;
  p.group = a->heads / a->kv_heads; p.rows = (int)rows;
  p.scale = a->scale; p.c = a->scale * kLog2e;
  p.out = a->out; p.stats = (float2*)a->stats;
  p.dq = a->d_q; p.dk = a->d_k; p.dv = a->d_v;
  return PCT_OK;
}

int check_pointers(const pct_attention* a, bool backward) {
  const int size = a->dtype == PCT_F32 ? 4 : 2;
  const bool q = a->batch && a->q_len, k = a->batch && a->k_len;
  if (a->key_mask && a->batch && a->k_len && !a->key_list) return policy_fail(PCT_ERR_INVALID_ARG, "attention: a key mask needs a key_list");
  if ((q && (!a->q || !a->out)) || (k && (!a->k || !a->v))) return policy_fail(PCT_ERR_INVALID_ARG, "attention: null tensor");
  if ((q && !aligned16(a->q, a->q_stride, size)) || (k && (!aligned16(a->k, a->k_stride, size) || !aligned16(a->v, a->v_stride, size))))
    return policy_fail(PCT_ERR_INVALID_ARG, "attention: the rows of q, k and v must start on 16 bytes");
  if (!backward) return PCT_OK;
  if ((q && (!a->d_out || !a->d_q || !a->stats)) || (k && (!a->d_k || !a->d_v))) return policy_fail(PCT_ERR_INVALID_ARG, "attention backward: null tensor");
  if (q && !aligned16(a->d_out, a->d_out_stride, size)) return policy_fail(PCT_ERR_INVALID_ARG, "attention: the rows of d_out must start on 16 bytes");
  return PCT_OK;
}

int64_t workspace(const pct_attention* a, const AttendParams& p, bool backward) {
  if (!p.batch || !p.rows || !p.k_len) return 0;
  return a->dtype == PCT_F32 ? attend_workspace_f32(p, backward) : (a->dtype == PCT_BF16 ? attend_workspace_bf16(p, backward) : attend_workspace_f16(p, backward));
}

// (clears with a kernel: a memset recorded into a graph is avoided)
__global__ __launch_bounds__(256) void pct_attend_zero_kernel(uint4* p, int64_t n) {
  for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < n; i += (int64_t)gridDim.x * 256) p[i] = make_uint4(0, 0, 0, 0);
}
void zero(void* p, int64_t elements, int size, hipStream_t s) {
  const int64_t n = elements * size / 16;  // (dim is a multiple of 8)
  if (n) pct_attend_zero_kernel<<<(unsigned)(n < 262144 ? (n + 255) / 256 : 1024), 256, 0, s>>>((uint4*)p, n);
}
}  // namespace
}  // namespace pct

extern "C" {
int64_t pct_attend_workspace(const pct_attention* a, int32_t backward) {
  pct::AttendParams p;
  return pct::check_attention(a, p) ? 0 : pct::workspace(a, p, backward != 0);
}

int pct_attend(const pct_attention* a, void* stream) {
  pct::AttendParams p;
  if (int rc = pct::check_attention(a, p)) return rc;
  if (int rc = pct::check_pointers(a, false)) return rc;
  hipStream_t s = (hipStream_t)stream;
  if (!p.batch || !p.rows) return PCT_OK;
  if (!p.k_len) {
    pct::zero(a->out, (int64_t)p.batch * p.rows * p.kv_heads * p.dim, a->dtype == PCT_F32 ? 4 : 2, s);
    return pct::policy_launched("attention clear kernel");
  }
  const int64_t need = pct::workspace(a, p, false);
  if (need && (!a->workspace || a->workspace_bytes < need)) return pct::policy_fail(PCT_ERR_INVALID_ARG, "the workspace is smaller than pct_attend_workspace() says");
  if (a->key_mask)
    for (int b = 0; b < p.batch; b += pct::SLICE) {
      pct::pct_attend_list_kernel<<<p.batch - b < pct::SLICE ? p.batch - b : pct::SLICE, 256, 0, s>>>(
          pct::Mask{a->key_mask, a->mask_row, a->mask_col, a->mask_type}, p, a->key_list, b);
      if (p.batch - b <= pct::SLICE) break;  // (b + SLICE may pass 2^31)
    }
  char* ws = (char*)a->workspace;
  return a->dtype == PCT_F32 ? pct::attend_forward_f32(p, ws, s) : (a->dtype == PCT_BF16 ? pct::attend_forward_bf16(p, ws, s) : pct::attend_forward_f16(p, ws, s));
}

int pct_attend_backward(const pct_attention* a, void* stream) {
  pct::AttendParams p;
  if (int rc = pct::check_attention(a, p)) return rc;
  if (int rc = pct::check_pointers(a, true)) return rc;
  hipStream_t s = (hipStream_t)stream;
  if (!p.batch) return PCT_OK;
  if (!p.rows || !p.k_len) {
    const int size = a->dtype == PCT_F32 ? 4 : 2;
    const int64_t nk = (int64_t)p.batch * p.k_len * p.kv_heads * p.dim;
    if (p.rows) pct::zero(a->d_q, (int64_t)p.batch * p.rows * p.kv_heads * p.dim, size, s);
    if (p.k_len) { pct::zero(a->d_k, nk, size, s); pct::zero(a->d_v, nk, size, s); }
    return pct::policy_launched("attention clear kernel");
  }
  const int64_t need = pct::workspace(a, p, true);
  if (!a->workspace || a->workspace_bytes < need) return pct::policy_fail(PCT_ERR_INVALID_ARG, "the workspace is smaller than pct_attend_workspace() says");
  char* ws = (char*)a->workspace;
  return a->dtype == PCT_F32 ? pct::attend_backward_f32(p, ws, s) : (a->dtype == PCT_BF16 ? pct::attend_backward_bf16(p, ws, s) : pct::attend_backward_f16(p, ws, s));
}
}
