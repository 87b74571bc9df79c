// Attention: the C entry points, their checks and the choice by type.
#include "attention.hpp"
#include "mhc_launch.hpp"

namespace mhc {

template <typename S> int att_fwd(const AttArgs&, hipStream_t);
template <typename S> int att_bwd(const AttArgs&, hipStream_t);
extern template int att_fwd<float>(const AttArgs&, hipStream_t);
extern template int att_fwd<bf16_t>(const AttArgs&, hipStream_t);
extern template int att_fwd<f16_t>(const AttArgs&, hipStream_t);
extern template int att_bwd<float>(const AttArgs&, hipStream_t);
extern template int att_bwd<bf16_t>(const AttArgs&, hipStream_t);
extern template int att_bwd<f16_t>(const AttArgs&, hipStream_t);

namespace {

// Rows are counted in 32 bits, with a tile's rows past the last one.
constexpr int64_t kMaxRows = 1ll << 30;
// Bytes from a row to the next: a tile of 128 rows stays below 2^31.
constexpr int64_t kMaxRowBytes = 1ll << 24;

int check_rows(const char* who, const char* name, const void* p, const int64_t* stride, int64_t rows, int es, int d) {
  if (rows == 0) return MHC_OK;
  if (!p) return set_error(MHC_ERR_INVALID, "%s: null pointer", who);
  if (!aligned16(p) || (stride[0] * es) % 16 || (stride[1] * es) % 16 || (stride[2] * es) % 16)
    return set_error(MHC_ERR_INVALID, "%s: %s has an address or a stride that is no multiple of 16 bytes", who, name);
  if (stride[0] < 0 || stride[2] < 0 || stride[1] < d || stride[1] * es > kMaxRowBytes)
    return set_error(MHC_ERR_INVALID, "%s: %s has strides %lld, %lld, %lld for rows of %d elements", who, name,
                     (long long)stride[0], (long long)stride[1], (long long)stride[2], d);
  return MHC_OK;
}

int check_att(const char* who, const mhc_attention_args* c, AttArgs& a) {
  if (!c) return set_error(MHC_ERR_INVALID, "%s: null arguments", who);
  if (c->dtype != MHC_DTYPE_F32 && c->dtype != MHC_DTYPE_BF16 && c->dtype != MHC_DTYPE_F16)
    return set_error(MHC_ERR_UNSUPPORTED, "%s: dtype %d not supported", who, c->dtype);
  const int es = c->dtype == MHC_DTYPE_F32 ? 4 : 2;
  if (c->heads < 1 || c->heads_k < 1 || c->heads % c->heads_k || c->d < 1 || c->sequences < 0 || c->rows_q < 0 || c->rows_k < 0)
    return set_error(MHC_ERR_INVALID, "%s: heads=%d heads_k=%d d=%d sequences=%d rows_q=%lld rows_k=%lld", who, c->heads,
                     c->heads_k, c->d, c->sequences, (long long)c->rows_q, (long long)c->rows_k);
  if (c->d * es > 512 || (c->d * es) % 16)
    return set_error(MHC_ERR_UNSUPPORTED, "%s: d=%d, expected whole 16 bytes and at most 512", who, c->d);
  if (c->rows_q > kMaxRows || c->rows_k > kMaxRows || c->heads > 65535 || c->sequences > kMaxRows)
    return set_error(MHC_ERR_UNSUPPORTED, "%s: rows_q=%lld rows_k=%lld heads=%d sequences=%d above the supported sizes", who,
                     (long long)c->rows_q, (long long)c->rows_k, c->heads, c->sequences);
  // (the kernels take scale * log2(e), which has to be a number too: an infinite one makes NaN of scores of 0)
  if (!(c->scale > 0.f) || !(c->scale * kLog2e <= __FLT_MAX__))
    return set_error(MHC_ERR_INVALID, "%s: scale %g", who, (double)c->scale);
  if (c->reserved) return set_error(MHC_ERR_INVALID, "%s: reserved=%d, expected 0", who, c->reserved);
  if (c->cu_seqlens_k && c->lengths_k) return set_error(MHC_ERR_INVALID, "%s: cu_seqlens_k and lengths_k", who);
  if ((!c->cu_seqlens_q && c->sequences == 0 && c->rows_q) || (!c->cu_seqlens_k && c->sequences == 0 && c->rows_k) ||
      (!c->cu_seqlens_q && c->sequences && c->rows_q % c->sequences) || (!c->cu_seqlens_k && c->sequences && c->rows_k % c->sequences))
    return set_error(MHC_ERR_INVALID, "%s: rows_q=%lld rows_k=%lld are no %d sequences", who, (long long)c->rows_q,
                     (long long)c->rows_k, c->sequences);
  if (const int rc = check_rows(who, "q", c->q, c->q_stride, c->rows_q, es, c->d)) return rc;
  if (const int rc = check_rows(who, "k", c->k, c->k_stride, c->rows_k, es, c->d)) return rc;
  if (const int rc = check_rows(who, "v", c->v, c->v_stride, c->rows_k, es, c->d)) return rc;
  a = {};
  a.q = {c->q, c->q_stride[0], c->q_stride[1], c->q_stride[2]};
  a.k = {c->k, c->k_stride[0], c->k_stride[1], c->k_stride[2]};
  a.v = {c->v, c->v_stride[0], c->v_stride[1], c->v_stride[2]};
  a.n = {c->cu_seqlens_q, c->cu_seqlens_k, c->lengths_k, c->rows_q, c->rows_k, c->sequences,
         c->sequences ? (int)(c->rows_q / c->sequences) : 0, c->sequences ? (int)(c->rows_k / c->sequences) : 0,
         c->heads, c->heads_k, c->d, c->causal ? 1 : 0};
  a.scale = c->scale;
  a.scale2 = c->scale * kLog2e;
  return MHC_OK;
}

}  // namespace
}  // namespace mhc

using namespace mhc;

extern "C" size_t mhc_attention_fwd_workspace_size(const mhc_attention_args* c) {
  AttArgs a;
  if (check_att("", c, a)) return 0;
  return att_split(a.n, device_cu_count()).bytes(a.n);
}

extern "C" int mhc_attention_fwd(const mhc_attention_args* c, void* out, float* lse, void* workspace, size_t workspace_bytes,
                                 void* stream) {
  clear_error();
  AttArgs a;
  if (const int rc = check_att("attention", c, a)) return rc;
  if (c->rows_q == 0) return MHC_OK;
  if (!out || !aligned16(out)) return set_error(MHC_ERR_INVALID, "attention: out is null or not 16-byte aligned");
  const size_t need = att_split(a.n, device_cu_count()).bytes(a.n);
  if (need && (!workspace || workspace_bytes < need || !aligned16(workspace)))
    return set_error(MHC_ERR_INVALID, "attention: workspace too small or not 16-byte aligned (%zu < %zu bytes)",
                     workspace ? workspace_bytes : (size_t)0, need);
  a.out = out;
  a.lse = lse;
  a.part = static_cast<float*>(workspace);
  hipStream_t st = static_cast<hipStream_t>(stream);
  if (c->dtype == MHC_DTYPE_F32) return att_fwd<float>(a, st);
  if (c->dtype == MHC_DTYPE_BF16) return att_fwd<bf16_t>(a, st);
  return att_fwd<f16_t>(a, st);
}

static AttBwdPlan bwd_plan(const mhc_attention_args* c, const AttArgs& a) {
  const bool fp32 = c->dtype == MHC_DTYPE_F32;
  return att_bwd_plan(a.n, fp32, att_big_head(a.n, fp32), device_cu_count());
}

extern "C" size_t mhc_attention_bwd_workspace_size(const mhc_attention_args* c) {
  AttArgs a;
  if (check_att("", c, a)) return 0;
  const AttBwdPlan p = bwd_plan(c, a);
  return p.delta_bytes + p.part_bytes;
}

extern "C" int mhc_attention_bwd(const mhc_attention_args* c, const void* grad_out, const int64_t* grad_stride, const void* out,
                                 const float* lse, void* grad_q, void* grad_k, void* grad_v, void* workspace,
                                 size_t workspace_bytes, void* stream) {
  clear_error();
  AttArgs a;
  if (const int rc = check_att("attention_backward", c, a)) return rc;
  const int es = c->dtype == MHC_DTYPE_F32 ? 4 : 2;
  if (!grad_stride) return set_error(MHC_ERR_INVALID, "attention_backward: null pointer");
  if (const int rc = check_rows("attention_backward", "grad_out", grad_out, grad_stride, c->rows_q, es, c->d)) return rc;
  if (c->rows_q && (!out || !lse || !grad_q || !aligned16(out) || !aligned16(grad_q)))
    return set_error(MHC_ERR_INVALID, "attention_backward: out, lse or grad_q is null or not 16-byte aligned");
  const bool keys = grad_k || grad_v;
  if (c->rows_k && keys && (!grad_k || !grad_v || !aligned16(grad_k) || !aligned16(grad_v)))
    return set_error(MHC_ERR_INVALID, "attention_backward: grad_k or grad_v is null or not 16-byte aligned");
  const AttBwdPlan plan = bwd_plan(c, a);
  const size_t need = keys ? plan.delta_bytes + plan.part_bytes : plan.delta_bytes;
  if (need && (!workspace || workspace_bytes < need || !aligned16(workspace)))
    return set_error(MHC_ERR_INVALID, "attention_backward: workspace too small or not 16-byte aligned (%zu < %zu bytes)",
                     workspace ? workspace_bytes : (size_t)0, need);
  const int64_t row = (int64_t)c->heads * c->d;
  a.go = {grad_out, grad_stride[0], grad_stride[1], grad_stride[2]};
  a.o = {out, a.n.Sq * row, row, c->d};
  a.out = grad_q;
  a.dk = grad_k;
  a.dv = grad_v;
  a.lse = const_cast<float*>(lse);
  a.delta = static_cast<float*>(workspace);
  a.part = reinterpret_cast<float*>(static_cast<char*>(workspace) + plan.delta_bytes);
  hipStream_t st = static_cast<hipStream_t>(stream);
  if (c->dtype == MHC_DTYPE_F32) return att_bwd<float>(a, st);
  if (c->dtype == MHC_DTYPE_BF16) return att_bwd<bf16_t>(a, st);
  return att_bwd<f16_t>(a, st);
}
