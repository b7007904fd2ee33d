// Attention over packed sequences (bfb_packed_attention, forward and
// backward): host side and the kernels that need no tensor core.
//
//   S = scale q k^T over the keys a query sees, P = softmax(S), o = P v,
//   lse = log sum exp S
//   dV = P^T dO, dP = dO V^T, delta = rowsum(dO o) - dlse,
//   dS = P (dP - delta), dQ = scale dS K, dK = scale dS^T Q
#include <algorithm>
#include <cfloat>

#include "attention.cuh"

namespace bfb {

BFB_DEBUG_COUNTER();
BFB_DEBUG_READER(debug_violations_attention)

namespace {

using Attn = attn::Args;

struct Span {
  int64_t q0, k0;
  int lq, lk, room;
};

__device__ __forceinline__ Span span_of(const Attn& a, int seq) {
  Span s;
  const int64_t q0 = min(max((int64_t)a.cu_q[seq], (int64_t)0), a.total_q);
  const int64_t q1 = min(max((int64_t)a.cu_q[seq + 1], q0), a.total_q);
  const int64_t k0 = min(max((int64_t)a.cu_k[seq], (int64_t)0), a.total_k);
  const int64_t k1 = min(max((int64_t)a.cu_k[seq + 1], k0), a.total_k);
  s.q0 = q0;
  s.k0 = k0;
  s.lq = (int)(q1 - q0);
  s.room = (int)(k1 - k0);
  s.lk = a.kv_lengths ? min(max(a.kv_lengths[seq], 0), s.room) : s.room;
  return s;
}

// The sequence that holds row r, or -1.
__device__ __forceinline__ int seq_of(const int32_t* cu, int seqs, int64_t r) {
  int lo = 0, hi = seqs;  // the last start <= r
  while (lo < hi) {
    const int mid = (lo + hi) >> 1;
    if (cu[mid + 1] <= r) lo = mid + 1; else hi = mid;
  }
  return lo < seqs && cu[lo] <= r ? lo : -1;
}

__device__ __forceinline__ float warp_sum(float x) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) x += __shfl_xor_sync(0xffffffffu, x, o);
  return x;
}

template <class T>
__device__ __forceinline__ void row_load(const T* p, int dim, float (&v)[4]) {
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int c = (threadIdx.x & 31) + 32 * i;
    v[i] = c < dim ? to_f32<T>(p[c]) : 0.f;
  }
}
template <class T>
__device__ __forceinline__ void row_store(T* p, int dim, const float (&v)[4]) {
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int c = (threadIdx.x & 31) + 32 * i;
    if (c < dim) p[c] = from_f32<T>(v[i]);
  }
}
__device__ __forceinline__ float dot4(const float (&a)[4], const float (&b)[4]) {
  return warp_sum(a[0] * b[0] + a[1] * b[1] + a[2] * b[2] + a[3] * b[3]);
}

// delta = rowsum(dO o) - dlse, one warp per (row, head).
template <class T>
__global__ void __launch_bounds__(128) delta_kernel(const T* out, const T* dout, const float* dlse, float* delta,
                                                    int64_t rows, int heads, int dim) {
  const int64_t unit = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 5);
  if (unit >= rows * heads) return;
  const int64_t r = unit / heads;
  const int h = (int)(unit % heads);
  float x[4], y[4];
  row_load<T>(out + unit * dim, dim, x);
  row_load<T>(dout + unit * dim, dim, y);
  const float d = dot4(x, y);
  if ((threadIdx.x & 31) == 0) delta[h * rows + r] = d - (dlse ? dlse[h * rows + r] : 0.f);
}

template <class T>
__global__ void __launch_bounds__(128) dq_kernel(const __grid_constant__ Attn a) {
  const int64_t unit = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 5);
  if (unit >= a.total_q * a.heads) return;
  const int64_t r = unit / a.heads;
  const int h = (int)(unit % a.heads), m = h / (a.heads / a.kv_heads);
  const int seq = seq_of(a.cu_q, a.seqs, r);
  float dq[4] = {};
  if (seq >= 0) {
    const Span s = span_of(a, seq);
    const int64_t i = r - s.q0;
    const int64_t n = a.causal ? min((int64_t)s.lk, i + s.lk - s.lq + 1) : s.lk;
    float q[4], g[4], k[4], v[4];
    row_load<T>(static_cast<const T*>(a.q) + r * a.q_row + h * a.q_head, a.dim, q);
    row_load<T>(static_cast<const T*>(a.dout) + unit * a.dim, a.dim, g);
    const float lse = a.lse[h * a.total_q + r], delta = a.delta[h * a.total_q + r];
    for (int64_t j = 0; j < n; ++j) {
      row_load<T>(static_cast<const T*>(a.k) + (s.k0 + j) * a.k_row + m * a.k_head, a.dim, k);
      row_load<T>(static_cast<const T*>(a.v) + (s.k0 + j) * a.v_row + m * a.v_head, a.dim, v);
      const float p = expf(dot4(q, k) * a.scale - lse), ds = p * (dot4(g, v) - delta) * a.scale;
#pragma unroll
      for (int c = 0; c < 4; ++c) dq[c] += ds * k[c];
    }
  }
  row_store<T>(static_cast<T*>(a.dq) + unit * a.dim, a.dim, dq);
}

// One warp per (key row, key head).
template <class T>
__global__ void __launch_bounds__(128) dkv_kernel(const __grid_constant__ Attn a) {
  const int64_t unit = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 5);
  if (unit >= a.total_k * a.kv_heads) return;
  const int64_t r = unit / a.kv_heads;
  const int m = (int)(unit % a.kv_heads), group = a.heads / a.kv_heads;
  const int seq = seq_of(a.cu_k, a.seqs, r);
  float dk[4] = {}, dv[4] = {};
  if (seq >= 0) {
    const Span s = span_of(a, seq);
    const int64_t j = r - s.k0;
    if (j < s.lk) {
      float q[4], g[4], k[4], v[4];
      row_load<T>(static_cast<const T*>(a.k) + r * a.k_row + m * a.k_head, a.dim, k);
      row_load<T>(static_cast<const T*>(a.v) + r * a.v_row + m * a.v_head, a.dim, v);
      const int64_t first = a.causal ? max((int64_t)0, j - (s.lk - s.lq)) : 0;
      for (int h = m * group; h < (m + 1) * group; ++h) {
        for (int64_t i = first; i < s.lq; ++i) {
          const int64_t row = s.q0 + i;
          row_load<T>(static_cast<const T*>(a.q) + row * a.q_row + h * a.q_head, a.dim, q);
          row_load<T>(static_cast<const T*>(a.dout) + (row * a.heads + h) * a.dim, a.dim, g);
          const float p = expf(dot4(q, k) * a.scale - a.lse[h * a.total_q + row]);
          const float ds = p * (dot4(g, v) - a.delta[h * a.total_q + row]) * a.scale;
#pragma unroll
          for (int c = 0; c < 4; ++c) {
            dv[c] += p * g[c];
            dk[c] += ds * q[c];
          }
        }
      }
    }
  }
  row_store<T>(static_cast<T*>(a.dk) + unit * a.dim, a.dim, dk);
  row_store<T>(static_cast<T*>(a.dv) + unit * a.dim, a.dim, dv);
}

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
  if (backward) c.take<float>((size_t)(total_q * heads));
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
  return attn::forward_sm100(a, dtype, as_stream(stream));
}

extern "C" int bfb_attention_timeouts(uint64_t* count, int reset) {
  if (!count) return BFB_ERR_INVALID_ARG;
  *count = 0;
  return attn::timeouts_forward(count, reset);
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
  a.delta = c.take<float>((size_t)(total_q * heads));
  cudaStream_t st = as_stream(stream);
  if (total_q > 0) {
    const unsigned blocks = (unsigned)ceil_div(total_q * heads, 4);
    if (dtype == BFB_F16)
      delta_kernel<__half><<<blocks, 128, 0, st>>>(static_cast<const __half*>(a.out), static_cast<const __half*>(a.dout),
                                                   lse_grad_dev, a.delta, total_q, a.heads, a.dim);
    else
      delta_kernel<__nv_bfloat16><<<blocks, 128, 0, st>>>(static_cast<const __nv_bfloat16*>(a.out),
                                                          static_cast<const __nv_bfloat16*>(a.dout), lse_grad_dev,
                                                          a.delta, total_q, a.heads, a.dim);
    BFB_CHECK_LAUNCH();
    (dtype == BFB_F16 ? dq_kernel<__half> : dq_kernel<__nv_bfloat16>)<<<blocks, 128, 0, st>>>(a);
    BFB_CHECK_LAUNCH();
  }
  if (total_k > 0) {
    const unsigned blocks = (unsigned)ceil_div(total_k * kv_heads, 4);
    (dtype == BFB_F16 ? dkv_kernel<__half> : dkv_kernel<__nv_bfloat16>)<<<blocks, 128, 0, st>>>(a);
    BFB_CHECK_LAUNCH();
  }
  return BFB_OK;
}
