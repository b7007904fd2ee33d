// Per-token operators of an attention block over active sites: the norm of
// each query and key head with its rotary position in one pass
// (bfb_qk_norm_rotary, forward and backward) and dropout onto the residual
// stream from a counter-based generator (bfb_residual_dropout).
//
// Every value is read once, worked on in fp32 registers, rounded once and
// written once, so HBM is the floor; the instructions are close behind it.
// Measured: rotary, 24 k tokens of 16 + 4 heads of 128, bf16: forward 58 us,
// backward 90 us (HBM 41 and 46 % busy, issue 52 and 44 %, 30 and 23 % of the
// warps fit).  Dropout, 90 k x 512, bf16: with the residual 50 us (HBM 60 %,
// issue 56 %), its gradient 45 us (37 and 60 %: the generator's ten rounds).
#include <algorithm>
#include <cmath>
#include <type_traits>

#include "sm100.cuh"

namespace bfb {

BFB_DEBUG_COUNTER();
BFB_DEBUG_READER(debug_violations_token_ops)

namespace {

using sm100::fma2;
using sm100::mul2;

constexpr int kThreads = 256;
// Rows of a thread in flight and threads of an SM, of the rotary kernels.  Measured on 90 k tokens of 16 heads of 64
// (forward) and 24 k of 20 of 128 (forward and backward), bf16: forward 4 x 768 and 2 x 1024 78 us, 3 x 1024 99
// (spills), 4 x 512 84; both 2 x 512 154 us, 1 x 512 168, 3 x 512 170.
constexpr int kForwardSteps = 4, kForwardBlocks = 3;
constexpr int kBackSteps = 2, kBackBlocks = 2;
constexpr int kMaxAxes = 8;
constexpr int kMaxDim = 256;
constexpr int kMaxHeads = 4096;
// Shares of the heads: at most kMaxHeads of each side, 16 heads of 16 lanes to a block.
constexpr int kMostShares = 2 * kMaxHeads / 16;
// Blocks of the backward: a share of the heads fills at least half of kThreads, 4 blocks of which an SM holds at most.
constexpr int kMostPartials = 148 * 4 + kMostShares;
// Dynamic shared memory of a block: 256 rows' sums of 16 columns each, or the angles of up to 4 x 256 tokens of 16
// values (one lane a row): the rows of a step hold 16 * kThreads values at most.
constexpr int kMostAngles = 4 * kThreads * 16 * 4;
constexpr size_t kPlainSmem = 32 << 10;  // up to here (beside the static tables) no kernel has to ask

// 8 consecutive values as they lie in memory (16-byte aligned).
template <class T>
struct Eight {
  uint4 u[sizeof(T) / 2];
  __device__ __forceinline__ void load(const T* p) {
#pragma unroll
    for (int i = 0; i < (int)sizeof(T) / 2; ++i) u[i] = reinterpret_cast<const uint4*>(p)[i];
  }
  __device__ __forceinline__ void zero() {
#pragma unroll
    for (int i = 0; i < (int)sizeof(T) / 2; ++i) u[i] = make_uint4(0u, 0u, 0u, 0u);
  }
  __device__ __forceinline__ void get(float (&v)[8]) const {
    const T* e = reinterpret_cast<const T*>(u);
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = to_f32<T>(e[i]);
  }
  __device__ __forceinline__ void set(const float (&v)[8]) {
    T* e = reinterpret_cast<T*>(u);
#pragma unroll
    for (int i = 0; i < 8; ++i) e[i] = from_f32<T>(v[i]);
  }
  __device__ __forceinline__ void store(T* p) const {
#pragma unroll
    for (int i = 0; i < (int)sizeof(T) / 2; ++i) reinterpret_cast<uint4*>(p)[i] = u[i];
  }
  __device__ __forceinline__ void pairs(float2 (&v)[4]) const {
    float x[8];
    get(x);
#pragma unroll
    for (int i = 0; i < 4; ++i) v[i] = make_float2(x[2 * i], x[2 * i + 1]);
  }
  __device__ __forceinline__ void set(const float2 (&v)[4]) {
    const float x[8] = {v[0].x, v[0].y, v[1].x, v[1].y, v[2].x, v[2].y, v[3].x, v[3].y};
    set(x);
  }
};
// a bf16 is the upper half of its fp32
template <>
__device__ __forceinline__ void Eight<__nv_bfloat16>::get(float (&v)[8]) const {
  const uint32_t w[4] = {u[0].x, u[0].y, u[0].z, u[0].w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    v[2 * i] = __uint_as_float(w[i] << 16);
    v[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
  }
}
template <>
__device__ __forceinline__ void Eight<__half>::get(float (&v)[8]) const {
  const uint32_t w[4] = {u[0].x, u[0].y, u[0].z, u[0].w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&w[i]));
    v[2 * i] = f.x;
    v[2 * i + 1] = f.y;
  }
}
template <>
__device__ __forceinline__ void Eight<__nv_bfloat16>::set(const float (&v)[8]) {
  u[0] = make_uint4(sm100::pack2<__nv_bfloat16>(v[0], v[1]), sm100::pack2<__nv_bfloat16>(v[2], v[3]),
                    sm100::pack2<__nv_bfloat16>(v[4], v[5]), sm100::pack2<__nv_bfloat16>(v[6], v[7]));
}
template <>
__device__ __forceinline__ void Eight<__half>::set(const float (&v)[8]) {
  u[0] = make_uint4(sm100::pack2<__half>(v[0], v[1]), sm100::pack2<__half>(v[2], v[3]),
                    sm100::pack2<__half>(v[4], v[5]), sm100::pack2<__half>(v[6], v[7]));
}

__device__ __forceinline__ void read8(const float* p, float (&v)[8]) {
  Eight<float> e;
  e.load(p);
  e.get(v);
}

// ------------------------------------------------------------ norm + rotary
// x [T, H, D] -> rotate(x * rsqrt(mean(x^2) + eps) * w): a group of L lanes
// owns one (token, head) row, each lane 16 of its values as two chunks of 8.
// In the half form (value i pairs with i + R/2) the two chunks are the two
// sides of 8 pairs, in the interleaved form neighbours, so every pair is
// turned inside one thread; values past R pass through.  A block takes `k`
// whole tokens at a time (or a share of one token's heads), so a thread's head,
// side, addresses and columns stay the same from one step to the next, and a
// warp's rows lie one after another in memory.  A tile is kSteps such steps: the
// threads first ask for their rows of all of them, and while these are on the
// way compute the tile's angles, which all heads of a token share.
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
  int slots;              // heads of a block
  int k;                  // tokens of a step
  int steps;              // steps of a tile
  int stride;             // floats from one token's cosines to the next's
  FastDiv per_slot, pairs;  // slots, half
  float* partial;         // backward: [blocks][2][D] sums for the weights' gradients
};

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

// What a block's groups all read: inv_freq / (2 pi) as sums of two fp32 numbers,
// and the norms' weights.
struct Tables {
  float2 freq[kMaxDim / 2];
  float w[2][kMaxDim];
  int64_t axis[kMaxDim / 2];  // offset of each pair's axis in a row of positions
};

__device__ __forceinline__ double freq_at(const RotaryArgs& a, int f) {
  return (a.freq_f64 ? static_cast<const double*>(a.freq)[f] : (double)static_cast<const float*>(a.freq)[f]) *
         0.15915494309189533577;
}

__device__ __forceinline__ void fill_tables(const RotaryArgs& a, Tables& s) {
  for (int f = threadIdx.x; f < a.half; f += blockDim.x) {
    const double turn = freq_at(a, f);
    const float hi = (float)turn;
    s.freq[f] = make_float2(hi, (float)(turn - hi));
    int axis = 0;
    while (axis < a.axes - 1 && f >= a.axis_end[axis]) ++axis;
    s.axis[f] = axis * a.pos_axis;
  }
  for (int i = threadIdx.x; i < 2 * a.dim; i += blockDim.x) {
    const int side = i >= a.dim, c = i - side * a.dim;
    if (a.w[side]) s.w[side][c] = a.w[side][c];
  }
  __syncthreads();
}

// Turns of pos * inv_freq, less whole ones, where fp32 sums do not suffice.
__device__ __noinline__ float far_turn(double pos, double freq) {
  const double turn = pos * freq;
  return (float)(turn - rint(turn));
}

// cos and sin of pos * inv_freq for the tile's tokens.  The angle of a far
// position has few fraction bits left in fp32, so the turns pos * inv_freq /
// (2 pi) are formed to about 48 bits as a sum of fp32 numbers, p = pos hi
// rounded, its rounding error, and pos lo; p's whole turns are dropped exactly.
// Positions of more than 24 bits and angles of more than 2^21 turns take fp64.
// Sine and cosine of the fraction are the special-function pipe's where the
// results are rounded to 16 bits (absolute error below 2^-20), sincospif
// otherwise: with it the angles were most of the kernel's instructions (voxels,
// 90 k tokens, 16 heads of 64, bf16: 81 us, now 77).
template <bool kExact, class P>
__device__ __forceinline__ void fill_angles_of(const RotaryArgs& a, const Tables& s, const P* pos_at, int count,
                                               float* cosine, float* sine) {
  for (uint32_t i = threadIdx.x; i < (uint32_t)(count * a.half); i += blockDim.x) {
    const uint32_t t = a.pairs.div(i), f = i - t * a.half;
    const P at = pos_at[t * a.pos_row + s.axis[f]];
    const float pos = (float)at;
    bool fits = true;
    if (!std::is_same<P, float>::value) fits = at >= (P) - (1 << 24) && at <= (P)(1 << 24);
    const float2 w = s.freq[f];
    const float p = pos * w.x;
    float turn = p - rintf(p) + (fmaf(pos, w.x, -p) + pos * w.y);
    if (!(fits && fabsf(p) < 2097152.f)) turn = far_turn((double)at, freq_at(a, f));
    float sn, cs;
    if (kExact) {
      sincospif(2.f * turn, &sn, &cs);
    } else {
      turn = (turn - rintf(turn)) * 6.283185307179586f;
      sn = __sinf(turn);
      cs = __cosf(turn);
    }
    cosine[t * a.stride + f] = cs;
    sine[t * a.stride + f] = sn;
  }
}

template <bool kExact>
__device__ __forceinline__ void fill_angles(const RotaryArgs& a, const Tables& s, int64_t t0, int count, float* cosine,
                                            float* sine) {
  if (a.pos_type == 0)
    fill_angles_of<kExact>(a, s, static_cast<const int32_t*>(a.pos) + t0 * a.pos_row, count, cosine, sine);
  else if (a.pos_type == 1)
    fill_angles_of<kExact>(a, s, static_cast<const int64_t*>(a.pos) + t0 * a.pos_row, count, cosine, sine);
  else
    fill_angles_of<kExact>(a, s, static_cast<const float*>(a.pos) + t0 * a.pos_row, count, cosine, sine);
}

// Turns the pairs of u and v (half form: u[i] with v[i]) by the angles from
// pair `f0` on, `count` of them.
template <bool kBack, bool kInterleaved>
__device__ __forceinline__ void turn(const float* cosine, const float* sine, int count, float2 (&u)[4],
                                     float2 (&v)[4]) {
  if (kInterleaved) {
    auto rot = [](float2& x, float cs, float sn) {
      if (kBack) sn = -sn;
      x = make_float2(x.x * cs - x.y * sn, x.y * cs + x.x * sn);
    };
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      if (i < count) rot(u[i], cosine[i], sine[i]);
      if (i + 4 < count) rot(v[i], cosine[i + 4], sine[i + 4]);
    }
  } else if (count > 0) {  // 8
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const float4 c4 = reinterpret_cast<const float4*>(cosine)[h], s4 = reinterpret_cast<const float4*>(sine)[h];
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const float2 cs = i ? make_float2(c4.z, c4.w) : make_float2(c4.x, c4.y);
        float2 sn = i ? make_float2(s4.z, s4.w) : make_float2(s4.x, s4.y);
        float2 &x = u[2 * h + i], &y = v[2 * h + i];
        const float2 minus = make_float2(-sn.x, -sn.y);
        const float2 p = fma2(y, kBack ? sn : minus, mul2(x, cs));
        y = fma2(x, kBack ? minus : sn, mul2(y, cs));
        x = p;
      }
    }
  }
}

__device__ __forceinline__ float lane_sum(float x, int lanes) {
  if (lanes > 1) x += __shfl_xor_sync(0xffffffffu, x, 1);
  if (lanes > 2) x += __shfl_xor_sync(0xffffffffu, x, 2);
  if (lanes > 4) x += __shfl_xor_sync(0xffffffffu, x, 4);
  if (lanes > 8) x += __shfl_xor_sync(0xffffffffu, x, 8);
  return x;
}

// A thread's place: its lane, its token within a step, its side and head.
struct Place {
  int lane, token, side, head, c0, c1, count;
};
__device__ __forceinline__ Place place_of(const RotaryArgs& a) {
  Place p;
  p.lane = threadIdx.x & (a.lanes - 1);
  const int slot = threadIdx.x >> a.lane_shift;
  p.token = (int)a.per_slot.div(slot);
  const int h = blockIdx.y * a.slots + (slot - p.token * a.slots);
  p.side = h >= a.heads[0];
  p.head = p.side ? h - a.heads[0] : h;
  chunks_of(a, p.lane, p.c0, p.c1);
  if (p.token >= a.k || h >= a.heads[0] + a.heads[1]) p.c0 = p.c1 = -1;  // takes part in the shuffles alone
  p.count = min(max(a.half - 8 * p.lane, 0), 8);
  return p;
}

template <class T, bool kInterleaved>
__global__ void __launch_bounds__(kThreads, kForwardBlocks) rotary_forward_kernel(const __grid_constant__ RotaryArgs a) {
  constexpr int kSteps = sizeof(T) == 2 ? kForwardSteps : kForwardSteps / 2;
  __shared__ __align__(16) Tables s;
  extern __shared__ __align__(16) float cosine[];
  float* sine = cosine + a.steps * a.k * a.stride;
  const Place me = place_of(a);
  const int heads = me.side ? a.heads[1] : a.heads[0];
  const int64_t row = me.side ? a.row[1] : a.row[0];
  const T* x = static_cast<const T*>(me.side ? a.x[1] : a.x[0]) + me.token * row +
               me.head * (me.side ? a.head[1] : a.head[0]);
  T* y = static_cast<T*>(me.side ? a.y[1] : a.y[0]) + ((int64_t)me.token * heads + me.head) * a.dim;
  const int64_t out_row = (int64_t)heads * a.dim;
  const bool norm = me.side ? a.w[1] != nullptr : a.w[0] != nullptr;
  const float *w0 = s.w[me.side] + max(me.c0, 0), *w1 = s.w[me.side] + max(me.c1, 0);
  fill_tables(a, s);
  const int tile = a.steps * a.k;
  for (int64_t t0 = (int64_t)blockIdx.x * tile; t0 < a.tokens; t0 += (int64_t)gridDim.x * tile) {
    const int count = (int)min((int64_t)tile, a.tokens - t0);
    Eight<T> x0[kSteps], x1[kSteps];
#pragma unroll
    for (int i = 0; i < kSteps; ++i) {
      x0[i].zero();
      x1[i].zero();
      if (i >= a.steps || i * a.k + me.token >= count) continue;
      if (BFB_BAD(t0 + i * a.k + me.token < a.tokens && (me.c0 < 0 || me.head < heads))) continue;
      const T* from = x + (t0 + i * a.k) * row;
      if (me.c0 >= 0) x0[i].load(from + me.c0);
      if (me.c1 >= 0) x1[i].load(from + me.c1);
    }
    __syncthreads();  // the tables; the last tile's angles are read
    fill_angles<sizeof(T) == 4>(a, s, t0, count, cosine, sine);
    __syncthreads();
#pragma unroll
    for (int i = 0; i < kSteps; ++i) {
      if (i >= a.steps) break;
      float2 u[4], v[4];
      x0[i].pairs(u);
      x1[i].pairs(v);
      if (norm || a.w[0] != nullptr || a.w[1] != nullptr) {  // the whole warp, for the shuffles
        float2 ss = mul2(u[0], u[0]);
#pragma unroll
        for (int e = 1; e < 4; ++e) ss = fma2(u[e], u[e], ss);
#pragma unroll
        for (int e = 0; e < 4; ++e) ss = fma2(v[e], v[e], ss);
        const float r = rsqrtf(lane_sum(ss.x + ss.y, a.lanes) * a.inv_dim + a.eps);
        if (norm) {
          const float2 r2 = make_float2(r, r);
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            u[e] = mul2(u[e], mul2(r2, reinterpret_cast<const float2*>(w0)[e]));
            v[e] = mul2(v[e], mul2(r2, reinterpret_cast<const float2*>(w1)[e]));
          }
        }
      }
      const int t = i * a.k + me.token;
      if (t >= count) continue;
      turn<false, kInterleaved>(cosine + t * a.stride + 8 * me.lane, sine + t * a.stride + 8 * me.lane, me.count, u, v);
      T* to = y + (t0 + i * a.k) * out_row;
      if (me.c0 >= 0) {
        x0[i].set(u);
        x0[i].store(to + me.c0);
      }
      if (me.c1 >= 0) {
        x1[i].set(v);
        x1[i].store(to + me.c1);
      }
    }
  }
}

// g = R^T dy; dx = r (w g - xhat mean(w g xhat)), xhat = r x; the weights'
// gradients g xhat are summed in registers over a thread's rows (each thread
// always owns the same columns of the same side), then over the block's threads
// and written as one partial per block: no atomics, so the sums' order is fixed.
template <class T, bool kInterleaved>
__global__ void __launch_bounds__(kThreads, kBackBlocks) rotary_backward_kernel(const __grid_constant__ RotaryArgs a) {
  constexpr int kSteps = sizeof(T) == 2 ? kBackSteps : kBackSteps / 2;
  __shared__ __align__(16) Tables s;
  extern __shared__ __align__(16) float cosine[];
  float* sine = cosine + a.steps * a.k * a.stride;
  const Place me = place_of(a);
  const int heads = me.side ? a.heads[1] : a.heads[0];
  const int64_t row = me.side ? a.row[1] : a.row[0], out_row = (int64_t)heads * a.dim;
  const T* x = static_cast<const T*>(me.side ? a.x[1] : a.x[0]) + me.token * row +
               me.head * (me.side ? a.head[1] : a.head[0]);
  const int64_t mine = ((int64_t)me.token * heads + me.head) * a.dim;
  const T* g = static_cast<const T*>(me.side ? a.g[1] : a.g[0]) + mine;
  T* y = static_cast<T*>(me.side ? a.y[1] : a.y[0]) + mine;
  const bool norm = me.side ? a.w[1] != nullptr : a.w[0] != nullptr, norms = a.w[0] || a.w[1];
  const float *w0 = s.w[me.side] + max(me.c0, 0), *w1 = s.w[me.side] + max(me.c1, 0);
  fill_tables(a, s);
  float2 acc[8] = {};
  const int tile = a.steps * a.k;
  for (int64_t t0 = (int64_t)blockIdx.x * tile; t0 < a.tokens; t0 += (int64_t)gridDim.x * tile) {
    const int count = (int)min((int64_t)tile, a.tokens - t0);
    Eight<T> x0[kSteps], x1[kSteps], g0[kSteps], g1[kSteps];
#pragma unroll
    for (int i = 0; i < kSteps; ++i) {
      x0[i].zero();
      x1[i].zero();
      g0[i].zero();
      g1[i].zero();
      if (i >= a.steps || i * a.k + me.token >= count) continue;
      if (BFB_BAD(t0 + i * a.k + me.token < a.tokens && (me.c0 < 0 || me.head < heads))) continue;
      const T* gr = g + (t0 + i * a.k) * out_row;
      if (me.c0 >= 0) g0[i].load(gr + me.c0);
      if (me.c1 >= 0) g1[i].load(gr + me.c1);
      if (!norm) continue;
      const T* from = x + (t0 + i * a.k) * row;
      if (me.c0 >= 0) x0[i].load(from + me.c0);
      if (me.c1 >= 0) x1[i].load(from + me.c1);
    }
    __syncthreads();
    fill_angles<sizeof(T) == 4>(a, s, t0, count, cosine, sine);
    __syncthreads();
#pragma unroll
    for (int i = 0; i < kSteps; ++i) {
      if (i >= a.steps) break;
      const int t = i * a.k + me.token;
      const bool live = t < count;
      float2 gu[4], gv[4];
      g0[i].pairs(gu);
      g1[i].pairs(gv);
      if (live)
        turn<true, kInterleaved>(cosine + t * a.stride + 8 * me.lane, sine + t * a.stride + 8 * me.lane, me.count, gu,
                                 gv);
      if (norms) {
        float2 u[4], v[4], px[4], py[4], ss = make_float2(0.f, 0.f), dot = ss;  // idle lanes and rows hold zeros
        x0[i].pairs(u);
        x1[i].pairs(v);
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          ss = fma2(u[e], u[e], fma2(v[e], v[e], ss));
          const float2 gx = mul2(gu[e], u[e]), gy = mul2(gv[e], v[e]);
          if (norm) {
            const float2 a0 = reinterpret_cast<const float2*>(w0)[e], a1 = reinterpret_cast<const float2*>(w1)[e];
            dot = fma2(a0, gx, fma2(a1, gy, dot));
            gu[e] = mul2(gu[e], a0);
            gv[e] = mul2(gv[e], a1);
          }
          px[e] = gx;
          py[e] = gy;
        }
        const float sum = lane_sum(ss.x + ss.y, a.lanes), dots = lane_sum(dot.x + dot.y, a.lanes);
        if (norm && live) {
          const float r = rsqrtf(sum * a.inv_dim + a.eps), m = -r * r * dots * a.inv_dim;
          const float2 r2 = make_float2(r, r), m2 = make_float2(m, m);
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            acc[e] = fma2(r2, px[e], acc[e]);
            acc[4 + e] = fma2(r2, py[e], acc[4 + e]);
            gu[e] = mul2(r2, fma2(m2, u[e], gu[e]));
            gv[e] = mul2(r2, fma2(m2, v[e], gv[e]));
          }
        }
      }
      if (!live) continue;
      T* to = y + (t0 + i * a.k) * out_row;
      if (me.c0 >= 0) {
        g0[i].set(gu);
        g0[i].store(to + me.c0);
      }
      if (me.c1 >= 0) {
        g1[i].set(gv);
        g1[i].store(to + me.c1);
      }
    }
  }
  if (!norms) return;
  // every slot's sums in shared memory, then each column's in the order of the slots
  float* sums = cosine;  // [slots of the block][dim]
  __syncthreads();
  const int slot = threadIdx.x >> a.lane_shift;
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    if (me.c0 >= 0) reinterpret_cast<float2*>(sums + slot * a.dim + me.c0)[e] = acc[e];
    if (me.c1 >= 0) reinterpret_cast<float2*>(sums + slot * a.dim + me.c1)[e] = acc[4 + e];
  }
  __syncthreads();
  const int all = a.heads[0] + a.heads[1];
  if (BFB_BAD(gridDim.x * gridDim.y <= (unsigned)kMostPartials)) return;
  for (int i = threadIdx.x; i < 2 * a.dim; i += blockDim.x) {
    const int side = i >= a.dim, c = i - side * a.dim;
    float v = 0.f;
    for (int t = 0; t < a.k; ++t)
      for (int j = 0; j < a.slots; ++j) {
        const int h = blockIdx.y * a.slots + j;
        if (h < all && (h >= a.heads[0]) == side) v += sums[(t * a.slots + j) * a.dim + c];
      }
    a.partial[((int64_t)(blockIdx.y * gridDim.x + blockIdx.x) * 2 + side) * a.dim + c] = v;
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
#pragma unroll 4
    for (int b = threadIdx.y; b < blocks; b += 32) v += partial[((int64_t)b * 2 + side) * dim + c];
  s[threadIdx.y][threadIdx.x] = v;
  __syncthreads();
  if (threadIdx.y == 0 && c < dim) {
    v = 0.f;
    for (int i = 0; i < 32; ++i) v += s[i][threadIdx.x];
    out[c] = v;
  }
}

constexpr int kSms = 148;
constexpr int kForwardThreads = kForwardBlocks * kThreads, kBackThreads = kBackBlocks * kThreads;  // what an SM holds at once

// How the rows are shared out: the grid (x: tiles, y: shares of the heads, as
// even as they come) and a block's threads.
struct Shape {
  unsigned x, y, threads;
};
Shape rotary_shape(RotaryArgs& a, int steps, int sm_threads) {
  const int all = a.heads[0] + a.heads[1], most = kThreads >> a.lane_shift;
  Shape g;
  g.y = (unsigned)ceil_div(all, most);
  a.slots = (int)ceil_div(all, g.y);
  a.k = std::max(1, most / a.slots);
  g.threads = (unsigned)ceil_div((int64_t)a.k * a.slots << a.lane_shift, 32) * 32;
  const int64_t x = std::max<int64_t>(1, kSms * (sm_threads / g.threads) / g.y);
  // few tokens are spread over all SMs
  a.k = (int)std::min<int64_t>(a.k, std::max<int64_t>(1, a.tokens / x));
  a.steps = (int)std::min<int64_t>(steps, std::max<int64_t>(1, a.tokens / (x * a.k)));
  g.threads = (unsigned)ceil_div((int64_t)a.k * a.slots << a.lane_shift, 32) * 32;
  g.x = (unsigned)std::min<int64_t>(x, ceil_div(a.tokens, (int64_t)a.k * a.steps));
  a.stride = (a.half + 3) / 4 * 4;
  a.per_slot = FastDiv((uint32_t)a.slots);
  a.pairs = FastDiv((uint32_t)a.half);
  return g;
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
  if (heads > kMaxHeads || kv_heads > kMaxHeads || tokens > (int64_t)1 << 40) return BFB_ERR_TOO_LARGE;
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
  return BFB_OK;
}

// ---------------------------------------------------------------- dropout
// Philox4x32-10 (Salmon et al., "Parallel random numbers: as easy as 1, 2,
// 3", SC 2011): ten rounds of two 32 x 32 -> 64 bit products over a 128-bit
// counter with a 64-bit key.  Element i of the tensor uses word i % 4 at
// counter (i / 4, offset), so forward and backward draw the same mask from
// the seed alone and none is stored.
struct Philox {
  uint32_t k0[10], k1[10];  // the rounds' keys, shared by all of a thread's counters
  uint32_t o0, o1;
  __device__ __forceinline__ Philox(uint64_t key, uint64_t offset)
      : o0((uint32_t)offset), o1((uint32_t)(offset >> 32)) {
#pragma unroll
    for (int i = 0; i < 10; ++i) {
      k0[i] = (uint32_t)key + i * 0x9E3779B9u;
      k1[i] = (uint32_t)(key >> 32) + i * 0xBB67AE85u;
    }
  }
  __device__ __forceinline__ uint4 at(uint64_t block) const {
    uint32_t x0 = (uint32_t)block, x1 = (uint32_t)(block >> 32), x2 = o0, x3 = o1;
#pragma unroll
    for (int i = 0; i < 10; ++i) {
      const uint64_t u = (uint64_t)x0 * 0xD2511F53u, w = (uint64_t)x2 * 0xCD9E8D57u;
      x0 = (uint32_t)(w >> 32) ^ x1 ^ k0[i];
      x2 = (uint32_t)(u >> 32) ^ x3 ^ k1[i];
      x1 = (uint32_t)w;
      x3 = (uint32_t)u;
    }
    return make_uint4(x0, x1, x2, x3);
  }
};

// 8 values from element i on: y = residual + keep * scale * x.  A dropped value
// contributes an exact 0 whatever x holds there (a select, not a product).
template <bool kResidual>
__device__ __forceinline__ void drop8(const Philox& rng, int64_t i, float (&v)[8], const float (&r)[8],
                                      uint32_t threshold, float scale) {
#pragma unroll
  for (int half = 0; half < 2; ++half) {
    const uint4 w = rng.at((uint64_t)i / 4 + half);
    const uint32_t word[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int e = 4 * half + j;
      const float kept = kResidual ? fmaf(v[e], scale, r[e]) : v[e] * scale;
      v[e] = word[j] >= threshold ? kept : kResidual ? r[e] : 0.f;
    }
  }
}

constexpr int kDropUnits = 4;  // times 8 values of a thread, a block's width apart (1: 102 us, 2: 105, 4: 97, 8: 99 on
// 90 k x 512 bf16, forward and backward)

// Bound by the instructions of the generator (10 of about 15 for each value)
// as much as by HBM, so a thread's counters share the rounds' keys.
template <class T, bool kResidual>
__global__ void __launch_bounds__(kThreads) dropout_kernel(const T* __restrict__ x, const T* __restrict__ residual,
                                                           T* __restrict__ y, int64_t n,
                                                           const int64_t* __restrict__ seed, uint32_t threshold,
                                                           float scale) {
  const int64_t base = ((int64_t)blockIdx.x * kDropUnits * kThreads + threadIdx.x) * 8;
  Eight<T> a[kDropUnits], b[kDropUnits];
#pragma unroll
  for (int u = 0; u < kDropUnits; ++u) {
    const int64_t i = base + (int64_t)u * kThreads * 8;
    if (i + 8 > n) continue;
    a[u].load(x + i);
    if (kResidual) b[u].load(residual + i);
  }
  const Philox rng((uint64_t)seed[0], (uint64_t)seed[1]);
#pragma unroll
  for (int u = 0; u < kDropUnits; ++u) {
    const int64_t i = base + (int64_t)u * kThreads * 8;
    if (i >= n) return;
    float v[8], r[8] = {};
    if (i + 8 <= n) {
      a[u].get(v);
      if (kResidual) b[u].get(r);
      drop8<kResidual>(rng, i, v, r, threshold, scale);
      a[u].set(v);
      a[u].store(y + i);
    } else {
      for (int j = 0; j < 8; ++j) {
        v[j] = i + j < n ? to_f32<T>(x[i + j]) : 0.f;
        if (kResidual && i + j < n) r[j] = to_f32<T>(residual[i + j]);
      }
      drop8<kResidual>(rng, i, v, r, threshold, scale);
      for (int j = 0; j < 8; ++j)
        if (i + j < n) y[i + j] = from_f32<T>(v[j]);
    }
  }
}

// The same for tensors that do not start on 16 bytes, and for p = 1.
template <class T>
__global__ void __launch_bounds__(kThreads) dropout_any_kernel(const T* __restrict__ x,
                                                               const T* __restrict__ residual, T* __restrict__ y,
                                                               int64_t n, const int64_t* __restrict__ seed,
                                                               uint32_t threshold, int drop_all, float scale) {
  const int64_t i = ((int64_t)blockIdx.x * kThreads + threadIdx.x) * 4;
  if (i >= n) return;
  const Philox rng((uint64_t)seed[0], (uint64_t)seed[1]);
  const uint4 w = rng.at((uint64_t)i / 4);
  const uint32_t word[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    if (i + j >= n) return;
    const float r = residual ? to_f32<T>(residual[i + j]) : 0.f;
    y[i + j] = from_f32<T>(word[j] >= threshold && !drop_all ? fmaf(to_f32<T>(x[i + j]), scale, r) : r);
  }
}

template <class T>
int dropout_launch(const void* x, const void* residual, void* y, int64_t n, const int64_t* seed, double p,
                   cudaStream_t stream) {
  const int drop_all = p >= 1.0;
  const uint32_t threshold = drop_all ? 0u : (uint32_t)(p * 4294967296.0);
  const float scale = drop_all ? 0.f : (float)(1.0 / (1.0 - p));
  const T *xt = static_cast<const T*>(x), *rt = static_cast<const T*>(residual);
  const uintptr_t bases =
      reinterpret_cast<uintptr_t>(x) | reinterpret_cast<uintptr_t>(residual) | reinterpret_cast<uintptr_t>(y);
  if (drop_all || bases % 16) {
    dropout_any_kernel<T><<<(unsigned)ceil_div(n, 4 * kThreads), kThreads, 0, stream>>>(
        xt, rt, static_cast<T*>(y), n, seed, threshold, drop_all, scale);
  } else {
    const unsigned blocks = (unsigned)ceil_div(n, 8 * kThreads * kDropUnits);
    (residual ? dropout_kernel<T, true> : dropout_kernel<T, false>)<<<blocks, kThreads, 0, stream>>>(
        xt, rt, static_cast<T*>(y), n, seed, threshold, scale);
  }
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
  const Shape g = rotary_shape(a, dtype == BFB_F32 ? kForwardSteps / 2 : kForwardSteps, kForwardThreads);
  const size_t smem = sizeof(float) * 2 * a.steps * a.k * a.stride;
  auto kernel = dtype == BFB_F32   ? (interleaved ? rotary_forward_kernel<float, true> : rotary_forward_kernel<float, false>)
                : dtype == BFB_F16 ? (interleaved ? rotary_forward_kernel<__half, true> : rotary_forward_kernel<__half, false>)
                                   : (interleaved ? rotary_forward_kernel<__nv_bfloat16, true>
                                                  : rotary_forward_kernel<__nv_bfloat16, false>);
  if (smem > kPlainSmem) BFB_CUDA(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, kMostAngles));
  kernel<<<dim3(g.x, g.y), g.threads, smem, as_stream(stream)>>>(a);
  BFB_CHECK_LAUNCH();
  return BFB_OK;
}

extern "C" int bfb_qk_norm_rotary_backward_workspace_size(int64_t dim, size_t* bytes) {
  if (!bytes || dim < 8 || dim > kMaxDim || dim % 8) return BFB_ERR_INVALID_ARG;
  *bytes = align_up(sizeof(float) * 2 * kMostPartials * (size_t)dim);
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
  int blocks = 0;
  if (tokens > 0) {
    if (!q_grad_dev || !k_grad_dev || !q_input_grad_dev || !k_input_grad_dev) return BFB_ERR_INVALID_ARG;
    if ((reinterpret_cast<uintptr_t>(q_grad_dev) | reinterpret_cast<uintptr_t>(k_grad_dev)) % 16)
      return BFB_ERR_INVALID_ARG;
    a.g[0] = q_grad_dev;
    a.g[1] = k_grad_dev;
    a.y[0] = q_input_grad_dev;
    a.y[1] = k_input_grad_dev;
    a.partial = static_cast<float*>(workspace_dev);
    const Shape g = rotary_shape(a, dtype == BFB_F32 ? kBackSteps / 2 : kBackSteps, kBackThreads);
    blocks = (int)(g.x * g.y);
    const size_t smem = sizeof(float) * std::max(2 * a.steps * a.k * a.stride, weights ? a.k * a.slots * a.dim : 0);
    auto kernel = dtype == BFB_F32   ? (interleaved ? rotary_backward_kernel<float, true> : rotary_backward_kernel<float, false>)
                  : dtype == BFB_F16 ? (interleaved ? rotary_backward_kernel<__half, true> : rotary_backward_kernel<__half, false>)
                                     : (interleaved ? rotary_backward_kernel<__nv_bfloat16, true>
                                                    : rotary_backward_kernel<__nv_bfloat16, false>);
    if (smem > kPlainSmem) BFB_CUDA(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, kMostAngles));
    kernel<<<dim3(g.x, g.y), g.threads, smem, as_stream(stream)>>>(a);
    BFB_CHECK_LAUNCH();
  }
  if (weights) {
    rotary_weight_kernel<<<dim3((unsigned)ceil_div(dim, 32), 2), dim3(32, 32), 0, as_stream(stream)>>>(
        static_cast<const float*>(workspace_dev), blocks, (int)dim, q_weight_dev ? q_weight_grad_dev : nullptr,
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
  if (ceil_div(n, 4 * kThreads) > 0x7fffffff) return BFB_ERR_TOO_LARGE;
  switch (dtype) {
    case BFB_F32: return dropout_launch<float>(x_dev, residual_dev, out_dev, n, seed_dev, p, as_stream(stream));
    case BFB_F16: return dropout_launch<__half>(x_dev, residual_dev, out_dev, n, seed_dev, p, as_stream(stream));
    default: return dropout_launch<__nv_bfloat16>(x_dev, residual_dev, out_dev, n, seed_dev, p, as_stream(stream));
  }
}
