// Entry points of the attention operators: argument checks, and which kernels take a call.
#include "attention_sm100.cuh"

namespace lsr {
namespace {

constexpr int kMaxHeadDim = 128;

bool dtype_ok(int d) { return d == LSR_DTYPE_F32 || d == LSR_DTYPE_BF16 || d == LSR_DTYPE_F16; }

int check_args(const lsr_attention_args* a) {
  if (!a || !dtype_ok(a->dtype)) return LSR_ERR_ARG;
  if (a->batch < 0 || a->q_len < 0 || a->kv_len < 0 || a->heads < 1 || a->kv_heads < 1 || a->head_dim < 1) return LSR_ERR_ARG;
  if (a->causal != 0 && a->causal != 1) return LSR_ERR_ARG;
  if (a->heads % a->kv_heads || a->head_dim > kMaxHeadDim) return LSR_ERR_SHAPE;
  // row numbers and block counts stay within 31 bits
  if ((long long)a->batch * a->heads > (1ll << 24) || a->q_len > (1 << 30) || a->kv_len > (1 << 30)) return LSR_ERR_SHAPE;
  return LSR_OK;
}

// Whether the tensors are aligned to their entries.
bool aligned(const lsr_attention_args* a) {
  const uintptr_t entry = a->dtype == LSR_DTYPE_F32 ? 4 : 2;
  uintptr_t bits = 0;
  for (const void* t : {a->q, a->k, a->v, (const void*)a->out, a->dout, (const void*)a->dq, (const void*)a->dk, (const void*)a->dv})
    bits |= reinterpret_cast<uintptr_t>(t);
  return bits % entry == 0 && reinterpret_cast<uintptr_t>(a->lse) % 4 == 0;
}

AttnStride stride_of(const long long* s) { return AttnStride{s[0], s[1], s[2]}; }

AttnParams params_of(const lsr_attention_args* a) {
  AttnParams p{};
  p.batch = a->batch;
  p.q_len = a->q_len;
  p.kv_len = a->kv_len;
  p.heads = a->heads;
  p.kv_heads = a->kv_heads;
  p.head_dim = a->head_dim;
  p.causal = a->causal;
  p.group = a->heads / a->kv_heads;
  p.scale = a->scale;
  p.q = a->q;
  p.k = a->k;
  p.v = a->v;
  p.out = a->out;
  p.dout = a->dout;
  p.dq = a->dq;
  p.dk = a->dk;
  p.dv = a->dv;
  p.sq = stride_of(a->q_stride);
  p.sk = stride_of(a->k_stride);
  p.sv = stride_of(a->v_stride);
  p.so = stride_of(a->out_stride);
  p.sdo = stride_of(a->dout_stride);
  p.sdq = stride_of(a->dq_stride);
  p.sdk = stride_of(a->dk_stride);
  p.sdv = stride_of(a->dv_stride);
  p.mask = a->key_mask;
  p.mask_stride = a->key_mask_stride;
  p.lse = a->lse;
  return p;
}

// The tensor-core kernels read by TMA: 16-bit types, 16-byte addresses, strides and rows. They take the
// row maximum of unscaled scores, which is that of the scaled ones for a positive scale.
bool fast_forward(const AttnParams& p, int dtype) {
  return dtype != LSR_DTYPE_F32 && p.scale > 0.f && p.kv_len > 0 &&
         rows_ok(p.q, p.sq, p.batch, p.heads, p.q_len, p.head_dim) &&
         rows_ok(p.k, p.sk, p.batch, p.kv_heads, p.kv_len, p.head_dim) &&
         rows_ok(p.v, p.sv, p.batch, p.kv_heads, p.kv_len, p.head_dim) &&
         rows_ok(p.out, p.so, p.batch, p.heads, p.q_len, p.head_dim);
}

bool fast_backward(const AttnParams& p, int dtype) {
  return p.q_len > 0 && fast_forward(p, dtype) && rows_ok(p.dout, p.sdo, p.batch, p.heads, p.q_len, p.head_dim) &&
         rows_ok(p.dq, p.sdq, p.batch, p.heads, p.q_len, p.head_dim) &&
         rows_ok(p.dk, p.sdk, p.batch, p.kv_heads, p.kv_len, p.head_dim) &&
         rows_ok(p.dv, p.sdv, p.batch, p.kv_heads, p.kv_len, p.head_dim);
}

}  // namespace
}  // namespace lsr

extern "C" {

size_t lsr_attention_forward_workspace_bytes(const lsr_attention_args* a) {
  using namespace lsr;
  if (check_args(a) != LSR_OK || a->batch == 0 || a->q_len == 0) return 0;
  const AttnParams p = params_of(a);
  return fast_forward(p, a->dtype) ? attention_forward_sm100_ws(p) : 0;
}

size_t lsr_attention_backward_workspace_bytes(const lsr_attention_args* a) {
  using namespace lsr;
  if (check_args(a) != LSR_OK || a->batch == 0) return 0;
  const AttnParams p = params_of(a);
  if (fast_backward(p, a->dtype)) return attention_backward_sm100_ws(p, a->dtype);
  return (size_t)a->batch * a->heads * a->q_len * sizeof(float) + 16;
}

int lsr_attention_forward(const lsr_attention_args* a, void* ws, size_t ws_bytes, lsr_stream_t stream) {
  using namespace lsr;
  int rc = check_args(a);
  if (rc != LSR_OK) return rc;
  if (a->batch == 0 || a->q_len == 0) return LSR_OK;
  if (!a->q || !a->out || !a->lse || (a->kv_len && (!a->k || !a->v))) return LSR_ERR_ARG;
  if (!aligned(a)) return LSR_ERR_SHAPE;
  if ((rc = check_device()) != LSR_OK) return rc;
  AttnParams p = params_of(a);
  if (!fast_forward(p, a->dtype)) return attention_forward_general(p, a->dtype, static_cast<cudaStream_t>(stream));
  const size_t need = attention_forward_sm100_ws(p);
  if (need && (!ws || ws_bytes < need || (reinterpret_cast<uintptr_t>(ws) & 15))) return LSR_ERR_WORKSPACE;
  if (!(p.status = status_ptr())) return LSR_ERR_LAUNCH;
  return attention_forward_sm100(p, a->dtype, ws, static_cast<cudaStream_t>(stream));
}

int lsr_attention_backward(const lsr_attention_args* a, void* ws, size_t ws_bytes, lsr_stream_t stream) {
  using namespace lsr;
  int rc = check_args(a);
  if (rc != LSR_OK) return rc;
  if (a->batch == 0 || (a->q_len == 0 && a->kv_len == 0)) return LSR_OK;
  if (a->q_len && (!a->q || !a->dout || !a->out || !a->lse || !a->dq)) return LSR_ERR_ARG;
  if (a->kv_len && (!a->k || !a->v || !a->dk || !a->dv)) return LSR_ERR_ARG;
  if (!aligned(a)) return LSR_ERR_SHAPE;
  if (!ws || ws_bytes < lsr_attention_backward_workspace_bytes(a) || (reinterpret_cast<uintptr_t>(ws) & 15))
    return LSR_ERR_WORKSPACE;
  if ((rc = check_device()) != LSR_OK) return rc;
  AttnParams p = params_of(a);
  if (fast_backward(p, a->dtype)) {
    if (!(p.status = status_ptr())) return LSR_ERR_LAUNCH;
    return attention_backward_sm100(p, a->dtype, ws, static_cast<cudaStream_t>(stream));
  }
  p.delta = static_cast<float*>(ws);
  return attention_backward_general(p, a->dtype, static_cast<cudaStream_t>(stream));
}

}  // extern "C"
