// Per-token operators of an attention block over active sites: the norm of
// each query and key head with its rotary position in one pass
// (bfb_qk_norm_rotary, forward and backward) and dropout onto the residual
// stream from a counter-based generator (bfb_residual_dropout).
//
// Both are bound by HBM: every value is read once, worked on in fp32
// registers, rounded once and written once.
#include <algorithm>
#include <cmath>

#include "common.cuh"

namespace bfb {

BFB_DEBUG_COUNTER();
BFB_DEBUG_READER(debug_violations_token_ops)

namespace {

constexpr int kThreads = 256;
constexpr int kMaxAxes = 8;
constexpr int kMaxDim = 256;

// 8 consecutive values as fp32 (16-byte aligned in memory).
template <class T>
__device__ __forceinline__ void load8(const T* p, float (&v)[8]) {
  const uint4 u = *reinterpret_cast<const uint4*>(p);
  const T* e = reinterpret_cast<const T*>(&u);
#pragma unroll
  for (int i = 0; i < 8; ++i) v[i] = to_f32<T>(e[i]);
}
template <>
__device__ __forceinline__ void load8<float>(const float* p, float (&v)[8]) {
  const float4 a = *reinterpret_cast<const float4*>(p), b = *reinterpret_cast<const float4*>(p + 4);
  v[0] = a.x; v[1] = a.y; v[2] = a.z; v[3] = a.w;
  v[4] = b.x; v[5] = b.y; v[6] = b.z; v[7] = b.w;
}
template <class T>
__device__ __forceinline__ void store8(T* p, const float (&v)[8]) {
  uint4 u;
  T* e = reinterpret_cast<T*>(&u);
#pragma unroll
  for (int i = 0; i < 8; ++i) e[i] = from_f32<T>(v[i]);
  *reinterpret_cast<uint4*>(p) = u;
}
template <>
__device__ __forceinline__ void store8<float>(float* p, const float (&v)[8]) {
  *reinterpret_cast<float4*>(p) = make_float4(v[0], v[1], v[2], v[3]);
  *reinterpret_cast<float4*>(p + 4) = make_float4(v[4], v[5], v[6], v[7]);
}

// ------------------------------------------------------------ norm + rotary
// x [T, H, D] -> rotate(x * rsqrt(mean(x^2) + eps) * w): a group of L lanes
// owns one (token, head) row, each lane 16 of its values as two chunks of 8.
// In the half form (value i pairs with i + R/2) the two chunks are the two
// sides of 8 pairs, in the interleaved form neighbours, so every pair is
// turned inside one thread; values past R pass through.
struct RotaryArgs {
  const void* x[2];       // q, k
  const void* g[2];       // backward: gradients of the outputs, contiguous
  void* y[2];             // forward: outputs; backward: dq, dk (contiguous)
  const float* w[2];      // norm weights [D], NULL: no norm
  int64_t row[2], head[2];  // element strides of x
  int heads[2];
  int64_t tokens;
  int dim, half;          // half = R / 2 pairs
  int lanes, lane_shift;  // lanes per row (a power of two)
  int rotary_lanes;       // half form: lanes that own pairs
  int interleaved;
  const void* pos;
  int pos_type;           // 0 int32, 1 int64, 2 fp32
  int64_t pos_row, pos_axis;
  const void* freq;
  int freq_f64;
  int axes, axis_end[kMaxAxes];
  float eps, inv_dim;
  int tile;               // tokens per block
  FastDiv per_token[2];   // units of one token: heads[0] / heads[1]
  FastDiv pairs;          // half
  float* partial;         // backward: [blocks][2][D] sums for the weights' gradients
};

__device__ __forceinline__ double position(const RotaryArgs& a, int64_t t, int axis) {
  const int64_t at = t * a.pos_row + axis * a.pos_axis;
  if (a.pos_type == 0) return static_cast<const int32_t*>(a.pos)[at];
  if (a.pos_type == 1) return static_cast<double>(static_cast<const int64_t*>(a.pos)[at]);
  return static_cast<const float*>(a.pos)[at];
}

// cos and sin of pos * inv_freq for the block's tokens, into shared memory.
// The angle of a far position (10^6 and more) has few fraction bits left in
// fp32, so it is formed in fp64 as turns, whose whole part is dropped before
// the rounding to fp32: the error is that of one fp32 rounding at any
// position.  Shared by all heads of a token, this costs half / (H * D) of the
// row work.
__device__ __forceinline__ void fill_turns(const RotaryArgs& a, int64_t t0, int count, float2* turns) {
  for (uint32_t i = threadIdx.x; i < (uint32_t)(count * a.half); i += kThreads) {
    const uint32_t t = a.pairs.div(i), f = i - t * a.half;
    int axis = 0;
    while (axis < a.axes - 1 && (int)f >= a.axis_end[axis]) ++axis;
    const double freq =
        a.freq_f64 ? static_cast<const double*>(a.freq)[f] : (double)static_cast<const float*>(a.freq)[f];
    const double turn = position(a, t0 + t, axis) * freq * 0.15915494309189533577;  // 1 / (2 pi)
    float s, c;
    sincospif((float)(2.0 * (turn - rint(turn))), &s, &c);
    turns[i] = make_float2(c, s);
  }
}

// The two chunks of a lane (element offsets, -1: none).
__device__ __forceinline__ void chunks_of(const RotaryArgs& a, int lane, int& c0, int& c1) {
  if (a.interleaved) {
    c0 = 16 * lane;
    c1 = c0 + 8;
  } else if (lane < a.rotary_lanes) {
    c0 = 8 * lane;
    c1 = c0 + a.half;
    return;
  } else {
    c0 = 2 * a.half + 16 * (lane - a.rotary_lanes);
    c1 = c0 + 8;
  }
  if (c0 >= a.dim) c0 = -1;
  if (c1 >= a.dim) c1 = -1;
}

template <bool kBack>
__device__ __forceinline__ void turn(const RotaryArgs& a, int lane, int c0, int c1, const float2* turns, float (&u)[8],
                                     float (&v)[8]) {
  auto rot = [](float& x, float& y, float2 cs) {
    const float s = kBack ? -cs.y : cs.y;
    const float p = x * cs.x - y * s, q = y * cs.x + x * s;
    x = p;
    y = q;
  };
  if (!a.interleaved) {
    if (lane < a.rotary_lanes) {
#pragma unroll
      for (int i = 0; i < 8; ++i) rot(u[i], v[i], turns[8 * lane + i]);
    }
    return;
  }
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    if (c0 >= 0 && c0 / 2 + i < a.half) rot(u[2 * i], u[2 * i + 1], turns[c0 / 2 + i]);
    if (c1 >= 0 && c1 / 2 + i < a.half) rot(v[2 * i], v[2 * i + 1], turns[c1 / 2 + i]);
  }
}

__device__ __forceinline__ float lane_sum(float x, int lanes) {
  for (int o = lanes >> 1; o > 0; o >>= 1) x += __shfl_xor_sync(0xffffffffu, x, o);
  return x;
}

template <class T>
__global__ void __launch_bounds__(kThreads) rotary_forward_kernel(const __grid_constant__ RotaryArgs a) {
  extern __shared__ float2 turns[];
  const int64_t t0 = (int64_t)blockIdx.x * a.tile;
  const int count = (int)min((int64_t)a.tile, a.tokens - t0);
  fill_turns(a, t0, count, turns);
  __syncthreads();
  const int lane = threadIdx.x & (a.lanes - 1);
  int c0, c1;
  chunks_of(a, lane, c0, c1);
#pragma unroll
  for (int side = 0; side < 2; ++side) {
    const int heads = a.heads[side], units = count * heads;
    const T* x = static_cast<const T*>(a.x[side]);
    T* y = static_cast<T*>(a.y[side]);
    float w0[8], w1[8];
    const bool norm = a.w[side] != nullptr;
    if (norm) {
      if (c0 >= 0) load8<float>(a.w[side] + c0, w0);
      if (c1 >= 0) load8<float>(a.w[side] + c1, w1);
    }
    // every thread of a warp takes every step: the shuffles need the full warp
    for (int base = 0; base < units; base += kThreads >> a.lane_shift) {
      const int unit = base + (threadIdx.x >> a.lane_shift);
      const bool live = unit < units;
      const uint32_t t = live ? a.per_token[side].div(unit) : 0;
      const int h = live ? unit - t * heads : 0;
      const T* row = x + (t0 + t) * a.row[side] + h * a.head[side];
      float u[8] = {}, v[8] = {};
      if (live && c0 >= 0) load8<T>(row + c0, u);
      if (live && c1 >= 0) load8<T>(row + c1, v);
      if (norm) {
        float ss = 0.f;
#pragma unroll
        for (int i = 0; i < 8; ++i) ss += u[i] * u[i] + v[i] * v[i];
        const float r = rsqrtf(lane_sum(ss, a.lanes) * a.inv_dim + a.eps);
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          if (c0 >= 0) u[i] *= r * w0[i];
          if (c1 >= 0) v[i] *= r * w1[i];
        }
      }
      turn<false>(a, lane, c0, c1, turns + t * a.half, u, v);
      T* out = y + ((t0 + t) * heads + h) * a.dim;
      if (live && c0 >= 0) store8<T>(out + c0, u);
      if (live && c1 >= 0) store8<T>(out + c1, v);
    }
  }
}

// g = R^T dy; dx = r (w g - xhat mean(w g xhat)), xhat = r x; the weights'
// gradients g xhat are summed in registers over the block's rows (each lane
// always owns the same columns), then over the block's warps and written as
// one partial per block: no atomics, so the sums' order is fixed.
template <class T>
__global__ void __launch_bounds__(kThreads) rotary_backward_kernel(const __grid_constant__ RotaryArgs a) {
  extern __shared__ float2 turns[];
  __shared__ float sums[kThreads / 32][kMaxDim];
  const int lane = threadIdx.x & (a.lanes - 1);
  int c0, c1;
  chunks_of(a, lane, c0, c1);
  float acc[2][16] = {};
  for (int64_t t0 = (int64_t)blockIdx.x * a.tile; t0 < a.tokens; t0 += (int64_t)gridDim.x * a.tile) {
    const int count = (int)min((int64_t)a.tile, a.tokens - t0);
    __syncthreads();
    fill_turns(a, t0, count, turns);
    __syncthreads();
#pragma unroll
    for (int side = 0; side < 2; ++side) {
      const int heads = a.heads[side], units = count * heads;
      const T* x = static_cast<const T*>(a.x[side]);
      const T* g = static_cast<const T*>(a.g[side]);
      T* y = static_cast<T*>(a.y[side]);
      const bool norm = a.w[side] != nullptr;
      float w0[8], w1[8];
      if (norm) {
        if (c0 >= 0) load8<float>(a.w[side] + c0, w0);
        if (c1 >= 0) load8<float>(a.w[side] + c1, w1);
      }
      for (int base = 0; base < units; base += kThreads >> a.lane_shift) {
        const int unit = base + (threadIdx.x >> a.lane_shift);
        const bool live = unit < units;
        const uint32_t t = live ? a.per_token[side].div(unit) : 0;
        const int h = live ? unit - t * heads : 0;
        const int64_t flat = ((t0 + t) * heads + h) * a.dim;
        float gu[8] = {}, gv[8] = {};
        if (live && c0 >= 0) load8<T>(g + flat + c0, gu);
        if (live && c1 >= 0) load8<T>(g + flat + c1, gv);
        float u[8] = {}, v[8] = {};
        if (norm) {
          const T* row = x + (t0 + t) * a.row[side] + h * a.head[side];
          if (live && c0 >= 0) load8<T>(row + c0, u);
          if (live && c1 >= 0) load8<T>(row + c1, v);
        }
        turn<true>(a, lane, c0, c1, turns + t * a.half, gu, gv);
        if (norm) {
          float ss = 0.f, dot = 0.f;
#pragma unroll
          for (int i = 0; i < 8; ++i) {
            ss += u[i] * u[i] + v[i] * v[i];
            if (c0 >= 0) dot += w0[i] * gu[i] * u[i];
            if (c1 >= 0) dot += w1[i] * gv[i] * v[i];
          }
          ss = lane_sum(ss, a.lanes);
          dot = lane_sum(dot, a.lanes);
          const float r = live ? rsqrtf(ss * a.inv_dim + a.eps) : 0.f, m = r * r * dot * a.inv_dim;
#pragma unroll
          for (int i = 0; i < 8; ++i) {
            acc[side][i] += r * gu[i] * u[i];  // zero for idle lanes
            acc[side][8 + i] += r * gv[i] * v[i];
            if (c0 >= 0) gu[i] = r * (w0[i] * gu[i] - u[i] * m);
            if (c1 >= 0) gv[i] = r * (w1[i] * gv[i] - v[i] * m);
          }
        }
        if (live && c0 >= 0) store8<T>(y + flat + c0, gu);
        if (live && c1 >= 0) store8<T>(y + flat + c1, gv);
      }
    }
  }
#pragma unroll
  for (int side = 0; side < 2; ++side) {
    if (a.w[side] == nullptr) continue;
    __syncthreads();
#pragma unroll
    for (int i = 0; i < 16; ++i) {
      float s = acc[side][i];
      for (int o = a.lanes; o < 32; o <<= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
      const int c = i < 8 ? c0 : c1;
      if ((threadIdx.x & 31) < a.lanes && c >= 0) sums[threadIdx.x >> 5][c + (i & 7)] = s;
    }
    __syncthreads();
    for (int c = threadIdx.x; c < a.dim; c += kThreads) {
      float s = 0.f;
#pragma unroll
      for (int i = 0; i < kThreads / 32; ++i) s += sums[i][c];
      a.partial[((int64_t)blockIdx.x * 2 + side) * a.dim + c] = s;
    }
  }
}

// Sum of the blocks' partials for 32 columns of one weight: 32 fixed
// interleaved row sets, then their sum in order.
__global__ void __launch_bounds__(1024) rotary_weight_kernel(const float* partial, int blocks, int dim, float* dqw,
                                                             float* dkw) {
  __shared__ float s[32][33];
  const int side = blockIdx.y, c = blockIdx.x * 32 + threadIdx.x;
  float* out = side ? dkw : dqw;
  if (out == nullptr) return;
  float v = 0.f;
  if (c < dim)
    for (int b = threadIdx.y; b < blocks; b += 32) v += partial[((int64_t)b * 2 + side) * dim + c];
  s[threadIdx.y][threadIdx.x] = v;
  __syncthreads();
  if (threadIdx.y == 0 && c < dim) {
    v = 0.f;
    for (int i = 0; i < 32; ++i) v += s[i][threadIdx.x];
    out[c] = v;
  }
}

constexpr int kBackBlocks = 148 * 4;

// Tokens per block: enough rows for four passes of the block's threads (the
// turns of a token are then computed once for all its heads), while small
// calls keep one token per block so that all SMs take part; the turns stay
// within 32 KB.
int tile_tokens(int64_t tokens, int heads, int lanes, int half) {
  const int64_t want = std::max<int64_t>(1, 4 * kThreads / ((int64_t)heads * lanes));
  const int64_t fit = std::max<int64_t>(1, (32 << 10) / (8 * std::max(1, half)));
  const int64_t spread = std::max<int64_t>(1, tokens / (148 * 4));
  return (int)std::min({want, fit, spread});
}

int fill_args(RotaryArgs& a, const void* q, const void* k, int64_t q_row, int64_t q_head, int64_t k_row,
              int64_t k_head, int dtype, int64_t tokens, int64_t heads, int64_t kv_heads, int64_t dim,
              int64_t rotated, const void* pos, int pos_type, int64_t pos_row, int64_t pos_axis, const void* freq,
              int freq_f64, int64_t axes, const int64_t* sections, const float* qw, const float* kw, double eps,
              int interleaved) {
  if (dtype_size(dtype) == 0) return BFB_ERR_UNSUPPORTED_DTYPE;
  if (tokens < 0 || heads < 1 || kv_heads < 1 || dim < 8 || dim > kMaxDim || dim % 8) return BFB_ERR_INVALID_ARG;
  if (rotated < 2 || rotated > dim || rotated % (interleaved ? 2 : 16)) return BFB_ERR_INVALID_ARG;
  if (axes < 1 || axes > kMaxAxes || !sections || !(eps >= 0.0)) return BFB_ERR_INVALID_ARG;
  if (pos_type < 0 || pos_type > 2) return BFB_ERR_UNSUPPORTED_DTYPE;
  if (heads > 4096 || kv_heads > 4096 || tokens > (int64_t)1 << 40) return BFB_ERR_TOO_LARGE;
  int64_t end = 0;
  for (int i = 0; i < axes; ++i) {
    if (sections[i] < 0 || sections[i] > dim) return BFB_ERR_INVALID_ARG;
    a.axis_end[i] = (int)(end += sections[i]);
  }
  if (end != rotated / 2) return BFB_ERR_INVALID_ARG;
  if (tokens > 0 && (!q || !k || !pos || !freq)) return BFB_ERR_INVALID_ARG;
  const int64_t per16 = 16 / dtype_size(dtype);
  if ((reinterpret_cast<uintptr_t>(q) | reinterpret_cast<uintptr_t>(k)) % 16 || q_row % per16 || q_head % per16 ||
      k_row % per16 || k_head % per16)
    return BFB_ERR_INVALID_ARG;
  if ((reinterpret_cast<uintptr_t>(qw) | reinterpret_cast<uintptr_t>(kw)) % 16) return BFB_ERR_INVALID_ARG;
  a.x[0] = q; a.x[1] = k;
  a.w[0] = qw; a.w[1] = kw;
  a.row[0] = q_row; a.row[1] = k_row;
  a.head[0] = q_head; a.head[1] = k_head;
  a.heads[0] = (int)heads; a.heads[1] = (int)kv_heads;
  a.tokens = tokens;
  a.dim = (int)dim;
  a.half = (int)rotated / 2;
  a.interleaved = interleaved;
  a.rotary_lanes = (int)rotated / 16;
  const int need = interleaved ? (int)(dim + 15) / 16 : a.rotary_lanes + (int)(dim - rotated + 15) / 16;
  a.lanes = 1;
  a.lane_shift = 0;
  while (a.lanes < need) a.lanes <<= 1, ++a.lane_shift;
  a.pos = pos; a.pos_type = pos_type; a.pos_row = pos_row; a.pos_axis = pos_axis;
  a.freq = freq; a.freq_f64 = freq_f64;
  a.axes = (int)axes;
  a.eps = (float)eps;
  a.inv_dim = 1.f / (float)dim;
  a.per_token[0] = FastDiv((uint32_t)heads);
  a.per_token[1] = FastDiv((uint32_t)kv_heads);
  a.pairs = FastDiv((uint32_t)a.half);
  a.tile = tile_tokens(tokens, (int)(heads + kv_heads), a.lanes, a.half);
  return BFB_OK;
}

// ---------------------------------------------------------------- dropout
// Philox4x32-10 (Salmon et al., "Parallel random numbers: as easy as 1, 2,
// 3", SC 2011): ten rounds of two 32 x 32 -> 64 bit products over a 128-bit
// counter with a 64-bit key.  Element i of the tensor uses word i % 4 at
// counter (i / 4, offset), so forward and backward draw the same mask from
// the seed alone and none is stored.
__device__ __forceinline__ uint4 philox(uint64_t block, uint64_t offset, uint64_t key) {
  uint32_t x0 = (uint32_t)block, x1 = (uint32_t)(block >> 32), x2 = (uint32_t)offset, x3 = (uint32_t)(offset >> 32);
  uint32_t k0 = (uint32_t)key, k1 = (uint32_t)(key >> 32);
#pragma unroll
  for (int i = 0; i < 10; ++i) {
    const uint64_t u = (uint64_t)x0 * 0xD2511F53u, w = (uint64_t)x2 * 0xCD9E8D57u;
    x0 = (uint32_t)(w >> 32) ^ x1 ^ k0;
    x2 = (uint32_t)(u >> 32) ^ x3 ^ k1;
    x1 = (uint32_t)w;
    x3 = (uint32_t)u;
    k0 += 0x9E3779B9u;
    k1 += 0xBB67AE85u;
  }
  return make_uint4(x0, x1, x2, x3);
}

// y = residual + keep * scale * x.  One thread takes 8 values: two Philox
// calls, 16-byte accesses.  A dropped value contributes an exact 0 whatever
// x holds there (a select, not a product).
template <class T, bool kAligned>
__global__ void __launch_bounds__(kThreads) dropout_kernel(const T* __restrict__ x, const T* __restrict__ residual,
                                                           T* __restrict__ y, int64_t n,
                                                           const int64_t* __restrict__ seed, uint32_t threshold,
                                                           int drop_all, float scale) {
  const int64_t i = ((int64_t)blockIdx.x * kThreads + threadIdx.x) * 8;
  if (i >= n) return;
  const bool whole = kAligned && i + 8 <= n;
  float v[8], r[8] = {};
  if (whole) {
    load8<T>(x + i, v);
    if (residual) load8<T>(residual + i, r);
  } else {
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      v[j] = i + j < n ? to_f32<T>(x[i + j]) : 0.f;
      if (residual && i + j < n) r[j] = to_f32<T>(residual[i + j]);
    }
  }
  const uint64_t key = (uint64_t)seed[0], offset = (uint64_t)seed[1];
  const uint4 a = philox((uint64_t)i / 4, offset, key), b = philox((uint64_t)i / 4 + 1, offset, key);
  const uint32_t word[8] = {a.x, a.y, a.z, a.w, b.x, b.y, b.z, b.w};
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    const bool keep = word[j] >= threshold && !drop_all;
    v[j] = keep ? fmaf(v[j], scale, r[j]) : r[j];
  }
  if (whole) {
    store8<T>(y + i, v);
  } else {
#pragma unroll
    for (int j = 0; j < 8; ++j)
      if (i + j < n) y[i + j] = from_f32<T>(v[j]);
  }
}

template <class T>
int dropout_launch(const void* x, const void* residual, void* y, int64_t n, const int64_t* seed, double p,
                   cudaStream_t stream) {
  const int drop_all = p >= 1.0;
  const uint32_t threshold = drop_all ? 0u : (uint32_t)(p * 4294967296.0);
  const float scale = drop_all ? 0.f : (float)(1.0 / (1.0 - p));
  const int64_t blocks = ceil_div(n, 8 * kThreads);
  const bool aligned =
      (reinterpret_cast<uintptr_t>(x) | reinterpret_cast<uintptr_t>(residual) | reinterpret_cast<uintptr_t>(y)) % 16 ==
      0;
  auto kernel = aligned ? dropout_kernel<T, true> : dropout_kernel<T, false>;
  kernel<<<(unsigned)blocks, kThreads, 0, stream>>>(static_cast<const T*>(x), static_cast<const T*>(residual),
                                                    static_cast<T*>(y), n, seed, threshold, drop_all, scale);
  BFB_CHECK_LAUNCH();
  return BFB_OK;
}

}  // namespace
}  // namespace bfb

using namespace bfb;

extern "C" int bfb_qk_norm_rotary(const void* q_dev, const void* k_dev, int64_t q_row, int64_t q_head, int64_t k_row,
                                  int64_t k_head, int dtype, int64_t tokens, int64_t heads, int64_t kv_heads,
                                  int64_t dim, int64_t rotated, const void* positions_dev, int position_type,
                                  int64_t position_row, int64_t position_axis, const void* inv_freq_dev,
                                  int inv_freq_f64, int64_t axes, const int64_t* sections, const float* q_weight_dev,
                                  const float* k_weight_dev, double eps, int interleaved, void* q_out_dev,
                                  void* k_out_dev, void* stream) {
  BFB_INJECT_POINT();
  RotaryArgs a = {};
  BFB_TRY(fill_args(a, q_dev, k_dev, q_row, q_head, k_row, k_head, dtype, tokens, heads, kv_heads, dim, rotated,
                    positions_dev, position_type, position_row, position_axis, inv_freq_dev, inv_freq_f64, axes,
                    sections, q_weight_dev, k_weight_dev, eps, interleaved));
  if (tokens == 0) return BFB_OK;
  if (!q_out_dev || !k_out_dev) return BFB_ERR_INVALID_ARG;
  a.y[0] = q_out_dev;
  a.y[1] = k_out_dev;
  const int64_t blocks = ceil_div(tokens, a.tile);
  if (blocks > 0x7fffffff) return BFB_ERR_TOO_LARGE;
  const size_t smem = sizeof(float2) * a.tile * a.half;
  auto kernel = dtype == BFB_F32 ? rotary_forward_kernel<float>
                : dtype == BFB_F16 ? rotary_forward_kernel<__half> : rotary_forward_kernel<__nv_bfloat16>;
  kernel<<<(unsigned)blocks, kThreads, smem, as_stream(stream)>>>(a);
  BFB_CHECK_LAUNCH();
  return BFB_OK;
}

extern "C" int bfb_qk_norm_rotary_backward_workspace_size(int64_t dim, size_t* bytes) {
  if (!bytes || dim < 8 || dim > kMaxDim || dim % 8) return BFB_ERR_INVALID_ARG;
  *bytes = align_up(sizeof(float) * kBackBlocks * 2 * (size_t)dim);
  return BFB_OK;
}

extern "C" int bfb_qk_norm_rotary_backward(
    const void* q_grad_dev, const void* k_grad_dev, const void* q_dev, const void* k_dev, int64_t q_row,
    int64_t q_head, int64_t k_row, int64_t k_head, int dtype, int64_t tokens, int64_t heads, int64_t kv_heads,
    int64_t dim, int64_t rotated, const void* positions_dev, int position_type, int64_t position_row,
    int64_t position_axis, const void* inv_freq_dev, int inv_freq_f64, int64_t axes, const int64_t* sections,
    const float* q_weight_dev, const float* k_weight_dev, double eps, int interleaved, void* q_input_grad_dev,
    void* k_input_grad_dev, float* q_weight_grad_dev, float* k_weight_grad_dev, void* workspace_dev,
    size_t workspace_bytes, void* stream) {
  BFB_INJECT_POINT();
  RotaryArgs a = {};
  BFB_TRY(fill_args(a, q_dev, k_dev, q_row, q_head, k_row, k_head, dtype, tokens, heads, kv_heads, dim, rotated,
                    positions_dev, position_type, position_row, position_axis, inv_freq_dev, inv_freq_f64, axes,
                    sections, q_weight_dev, k_weight_dev, eps, interleaved));
  if ((q_weight_dev && !q_weight_grad_dev) || (k_weight_dev && !k_weight_grad_dev)) return BFB_ERR_INVALID_ARG;
  const bool weights = q_weight_dev || k_weight_dev;
  size_t need = 0;
  BFB_TRY(bfb_qk_norm_rotary_backward_workspace_size(dim, &need));
  if (weights && (!workspace_dev || workspace_bytes < need)) return BFB_ERR_WORKSPACE;
  int64_t blocks = 0;
  if (tokens > 0) {
    if (!q_grad_dev || !k_grad_dev || !q_input_grad_dev || !k_input_grad_dev) return BFB_ERR_INVALID_ARG;
    if ((reinterpret_cast<uintptr_t>(q_grad_dev) | reinterpret_cast<uintptr_t>(k_grad_dev)) % 16)
      return BFB_ERR_INVALID_ARG;
    a.g[0] = q_grad_dev;
    a.g[1] = k_grad_dev;
    a.y[0] = q_input_grad_dev;
    a.y[1] = k_input_grad_dev;
    a.partial = static_cast<float*>(workspace_dev);
    blocks = std::min<int64_t>(kBackBlocks, ceil_div(tokens, a.tile));
    const size_t smem = sizeof(float2) * a.tile * a.half;
    auto kernel = dtype == BFB_F32 ? rotary_backward_kernel<float>
                  : dtype == BFB_F16 ? rotary_backward_kernel<__half> : rotary_backward_kernel<__nv_bfloat16>;
    kernel<<<(unsigned)blocks, kThreads, smem, as_stream(stream)>>>(a);
    BFB_CHECK_LAUNCH();
  }
  if (weights) {
    rotary_weight_kernel<<<dim3((unsigned)ceil_div(dim, 32), 2), dim3(32, 32), 0, as_stream(stream)>>>(
        static_cast<const float*>(workspace_dev), (int)blocks, (int)dim, q_weight_dev ? q_weight_grad_dev : nullptr,
        k_weight_dev ? k_weight_grad_dev : nullptr);
    BFB_CHECK_LAUNCH();
  }
  return BFB_OK;
}

extern "C" int bfb_residual_dropout(const void* x_dev, const void* residual_dev, int dtype, int64_t n,
                                    const int64_t* seed_dev, double p, void* out_dev, void* stream) {
  BFB_INJECT_POINT();
  if (dtype_size(dtype) == 0) return BFB_ERR_UNSUPPORTED_DTYPE;
  if (n < 0 || !(p >= 0.0 && p <= 1.0)) return BFB_ERR_INVALID_ARG;
  if (n == 0) return BFB_OK;
  if (!x_dev || !out_dev || !seed_dev) return BFB_ERR_INVALID_ARG;
  if (ceil_div(n, 8 * kThreads) > 0x7fffffff) return BFB_ERR_TOO_LARGE;
  switch (dtype) {
    case BFB_F32: return dropout_launch<float>(x_dev, residual_dev, out_dev, n, seed_dev, p, as_stream(stream));
    case BFB_F16: return dropout_launch<__half>(x_dev, residual_dev, out_dev, n, seed_dev, p, as_stream(stream));
    default: return dropout_launch<__nv_bfloat16>(x_dev, residual_dev, out_dev, n, seed_dev, p, as_stream(stream));
  }
}
