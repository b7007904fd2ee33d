// Attention over packed sequences (bfb_packed_attention, forward and
// backward): host side, checks and the choice of the kernels.
//
//   S = scale q k^T over the keys a query sees, P = softmax(S), o = P v,
//   lse = log sum exp S
//   dV = P^T dO, dP = dO V^T, delta = rowsum(dO o) - dlse,
//   dS = P (dP - delta), dQ = scale dS K, dK = scale dS^T Q
#include <algorithm>
#include <cfloat>

#include "attention.cuh"

namespace bfb {

namespace {

using Attn = attn::Args;

int check_args(const Attn& a, int dtype) {
  if (dtype != BFB_F16 && dtype != BFB_BF16) return BFB_ERR_UNSUPPORTED_DTYPE;
  if (a.total_q < 0 || a.total_k < 0 || a.heads < 1 || a.kv_heads < 1 || a.heads % a.kv_heads || a.dim < 8 ||
      a.dim > 128 || a.dim % 8 || a.seqs < 0)
    return BFB_ERR_INVALID_ARG;
  if (a.total_q > 0x7fffff00 || a.total_k > 0x7fffff00 || a.heads > 65535) return BFB_ERR_TOO_LARGE;
  if (!(a.scale == a.scale) || !(a.scale <= FLT_MAX && a.scale >= -FLT_MAX)) return BFB_ERR_INVALID_ARG;
  if (a.seqs > 0 && (!a.cu_q || !a.cu_k)) return BFB_ERR_INVALID_ARG;
  if (a.total_q > 0 && (!a.q || !a.out || !a.lse)) return BFB_ERR_INVALID_ARG;
  if (a.total_k > 0 && (!a.k || !a.v)) return BFB_ERR_INVALID_ARG;
  // rows and heads start on 16 bytes
  const int64_t strides = a.q_row | a.q_head | a.k_row | a.k_head | a.v_row | a.v_head;
  const uintptr_t bases = reinterpret_cast<uintptr_t>(a.q) | reinterpret_cast<uintptr_t>(a.k) |
                          reinterpret_cast<uintptr_t>(a.v) | reinterpret_cast<uintptr_t>(a.out);
  if (strides % 8 || bases % 16) return BFB_ERR_INVALID_ARG;
  return BFB_OK;
}

// Whether the queries are few enough for the kernel that is split over the
// keys: up to two of its 16-row tiles for the average sequence and key head.
// Split kernel / tile kernel, us, 32/8 heads of 128, bf16, causal, by rows (queries x query heads of a key head):
//   sequences x keys     4 rows         32            64            128
//       4 x   128        12 /  12      12 /  12      12 /  12      16 /  12
//       4 x 20000        72 / 261     116 / 261     202 / 261     368 / 260
//      32 x   128        13 /  50      23 /  53      38 /  54      60 /  55
//      32 x  8000       172 / 746     332 / 748     644 / 747    1310 / 747
// Heads of 64 cross between 32 and 64 (32 x 128: 20 / 23 at 32, 34 / 23 at 64; 32 x 8000: 326 / 367 at 64), so the limit
// stays below what 128 alone would take.  Lengths are on the device, so the rule sees their average, and one kernel takes
// a whole batch: a prompt of 4000 with 100 single queries on 2000 keys each 825 us (tiles; apart 136 + 142), with 600 on
// 500 keys 2195 us (split; apart 136 + 285).  Two calls avoid it.
bool few_rows(int64_t total_q, int64_t heads, int64_t kv_heads, int64_t seqs) {
  return total_q * (heads / kv_heads) <= 32 * seqs;
}

Attn make(const void* q, const void* k, const void* v, const int64_t* strides, int64_t total_q, int64_t total_k,
          int64_t heads, int64_t kv_heads, int64_t dim, int64_t seqs, const int32_t* cu_q, const int32_t* cu_k,
          const int32_t* kv_lengths, int causal, double scale) {
  Attn a = {};
  a.q = q; a.k = k; a.v = v;
  a.q_row = strides[0]; a.q_head = strides[1];
  a.k_row = strides[2]; a.k_head = strides[3];
  a.v_row = strides[4]; a.v_head = strides[5];
  a.total_q = total_q; a.total_k = total_k;
  auto narrow = [](int64_t x) { return x < 0 || x > 0x7fffffff ? -1 : (int)x; };  // -1 is refused by check_args
  a.heads = narrow(heads); a.kv_heads = narrow(kv_heads); a.dim = narrow(dim); a.seqs = narrow(seqs);
  a.cu_q = cu_q; a.cu_k = cu_k; a.kv_lengths = kv_lengths;
  a.causal = causal != 0;
  a.scale = (float)scale;
  return a;
}

}  // namespace
}  // namespace bfb

using namespace bfb;

extern "C" int bfb_packed_attention_workspace_size(int64_t total_q, int64_t total_k, int64_t heads, int64_t kv_heads,
                                                   int64_t dim, int64_t seqs, int backward, size_t* bytes) {
  if (!bytes || total_q < 0 || total_k < 0 || heads < 1 || kv_heads < 1 || dim < 1 || seqs < 0)
    return BFB_ERR_INVALID_ARG;
  Carver c(nullptr);
  if (backward) {
    for (int i = 0; i < 3; ++i) c.take<float>((size_t)(total_q * heads));
    c.take<float>((size_t)(total_k * kv_heads));
  } else if (few_rows(total_q, heads, kv_heads, seqs)) {
    c.take<float>(attn::rows_record_floats((int)dim));
  }
  *bytes = c.bytes();
  return BFB_OK;
}

extern "C" int bfb_packed_attention(const void* q_dev, const void* k_dev, const void* v_dev, const int64_t* strides,
                                    int dtype, int64_t total_q, int64_t total_k, int64_t heads, int64_t kv_heads,
                                    int64_t dim, int64_t seqs, const int32_t* cu_q_dev, const int32_t* cu_k_dev,
                                    const int32_t* kv_lengths_dev, int causal, double scale, void* out_dev,
                                    float* lse_dev, void* workspace_dev, size_t workspace_bytes, void* stream) {
  BFB_INJECT_POINT();
  if (!strides) return BFB_ERR_INVALID_ARG;
  Attn a = make(q_dev, k_dev, v_dev, strides, total_q, total_k, heads, kv_heads, dim, seqs, cu_q_dev, cu_k_dev,
                kv_lengths_dev, causal, scale);
  a.out = out_dev;
  a.lse = lse_dev;
  BFB_TRY(check_args(a, dtype));
  if (total_q == 0) return BFB_OK;
  if (few_rows(total_q, heads, kv_heads, seqs)) {
    size_t need = 0;
    BFB_TRY(bfb_packed_attention_workspace_size(total_q, total_k, heads, kv_heads, dim, seqs, 0, &need));
    if (!workspace_dev || workspace_bytes < need) return BFB_ERR_WORKSPACE;
    Carver c(workspace_dev);
    return attn::forward_rows(a, dtype, c.take<float>(attn::rows_record_floats(a.dim)), as_stream(stream));
  }
  return attn::forward_sm100(a, dtype, as_stream(stream));
}

extern "C" int bfb_attention_timeouts(uint64_t* count, int reset) {
  if (!count) return BFB_ERR_INVALID_ARG;
  *count = 0;
  BFB_TRY(attn::timeouts_forward(count, reset));
  return attn::timeouts_backward(count, reset);
}

extern "C" int bfb_packed_attention_backward(
    const void* out_grad_dev, const float* lse_grad_dev, const void* q_dev, const void* k_dev, const void* v_dev,
    const int64_t* strides, const void* out_dev, const float* lse_dev, int dtype, int64_t total_q, int64_t total_k,
    int64_t heads, int64_t kv_heads, int64_t dim, int64_t seqs, const int32_t* cu_q_dev, const int32_t* cu_k_dev,
    const int32_t* kv_lengths_dev, int causal, double scale, void* q_grad_dev, void* k_grad_dev, void* v_grad_dev,
    void* workspace_dev, size_t workspace_bytes, void* stream) {
  BFB_INJECT_POINT();
  if (!strides) return BFB_ERR_INVALID_ARG;
  Attn a = make(q_dev, k_dev, v_dev, strides, total_q, total_k, heads, kv_heads, dim, seqs, cu_q_dev, cu_k_dev,
                kv_lengths_dev, causal, scale);
  a.out = const_cast<void*>(out_dev);
  a.lse = const_cast<float*>(lse_dev);
  a.dout = out_grad_dev;
  a.dlse = lse_grad_dev;
  a.dq = q_grad_dev;
  a.dk = k_grad_dev;
  a.dv = v_grad_dev;
  BFB_TRY(check_args(a, dtype));
  if ((total_q > 0 && (!out_grad_dev || !q_grad_dev)) || (total_k > 0 && (!k_grad_dev || !v_grad_dev)))
    return BFB_ERR_INVALID_ARG;
  if ((reinterpret_cast<uintptr_t>(out_grad_dev) | reinterpret_cast<uintptr_t>(q_grad_dev) |
       reinterpret_cast<uintptr_t>(k_grad_dev) | reinterpret_cast<uintptr_t>(v_grad_dev)) % 16)
    return BFB_ERR_INVALID_ARG;
  size_t need = 0;
  BFB_TRY(bfb_packed_attention_workspace_size(total_q, total_k, heads, kv_heads, dim, seqs, 1, &need));
  if (need > 0 && (!workspace_dev || workspace_bytes < need)) return BFB_ERR_WORKSPACE;
  Carver c(workspace_dev);
  a.lse2 = c.take<float>((size_t)(total_q * heads));
  a.delta = c.take<float>((size_t)(total_q * heads));
  a.norm_g = c.take<float>((size_t)(total_q * heads));
  a.norm_v = c.take<float>((size_t)(total_k * kv_heads));
  if (total_q == 0 && total_k == 0) return BFB_OK;
  return attn::backward_sm100(a, dtype, as_stream(stream));
}
