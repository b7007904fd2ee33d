// Packed attention, forward, on the tensor cores.
//
//   S = q k^T        (tcgen05, both operands in shared memory, S in tensor memory)
//   P = exp2(c (S - m)),  c = scale log2(e): one thread per row, rounded to 16
//                    bits and written to tensor memory
//   O += P v         (tcgen05, P from tensor memory)
// over the keys in tiles of 128; O stays in tensor memory.  Where a row's
// maximum grows, O and the sum have to be scaled down; here the maximum in use
// is only moved when it grows by more than 2^8, so the scaling is rare and its
// result the same (a published idea for this chip, not this file's).  In fp16 m is
// 7 below the maximum: P stays below 2^15, and the keys of a long tail (2^-14 of
// the largest and less) out of the subnormal numbers, where each counts for
// little but all of them together need not.
//
// Two kernels, by the width of a head:
// * up to 64 (one_tile_kernel): a block takes 128 query rows, two blocks fit an
//   SM.  Tensor memory has room for P beside S, so the next scores are made as
//   soon as the softmax has read the last ones and the softmax warps never wait
//   for a product; the two blocks fill each other's gaps.
// * up to 128 (two_tile_kernel): keys and values are twice as wide, and read for
//   128 rows only they would come from L2 faster than it delivers; so a block
//   takes two tiles of 128 rows and the SM.  P lies over S, and while one tile is
//   in its softmax the tensor core works on the other.
//
// Measured, one sequence of 8192 tokens, full.  8 heads of 64, fp16: 230 us, 598
// TFLOP/s; the special-function pipe (exponentials) is 67 % busy, the tensor pipe
// 29 %.  8/2 heads of 128, bf16: 272 us, 1011 TFLOP/s; 60 and 51 %: a tile's chain
// of product, softmax and product bounds it, with one block to an SM.
#include <cfloat>

#include "attention.cuh"

namespace bfb {

BFB_DEBUG_COUNTER();
BFB_DEBUG_READER(debug_violations_attention_fwd)

namespace attn {

namespace {

using namespace sm100;

__device__ unsigned long long g_timeouts = 0ull;

constexpr float kGrow = 8.f;  // log2 of the growth that moves the maximum

template <int DP>
struct Layout {
  static constexpr int kTileBytes = kTile * DP * 2;
  static constexpr int kPanel = kTile * 128;  // 64 columns of a tile
};

// c: positive, as a negative scale's sign goes into the product, and for 0 the
// smallest number (hidden scores stay -inf, and every other exponent 0).
__device__ __forceinline__ float exponent_factor(float scale) {
  return fmaxf(fabsf(scale) * 1.4426950408889634f, FLT_MIN);
}

// Scores from the `limit`-th column on are hidden: whatever they are, they
// become -inf.
__device__ __forceinline__ void hide(uint32_t (&x)[kTile], int limit) {
#pragma unroll
  for (int b = 0; b < kTile; ++b)
    if (b >= limit) x[b] = 0xff800000u;
}

__device__ __forceinline__ float row_max(const uint32_t (&x)[kTile]) {
  float best[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
  for (int b = 0; b < kTile; b += 8)
#pragma unroll
    for (int e = 0; e < 4; ++e)
      best[e] = fmaxf(best[e], fmaxf(__uint_as_float(x[b + 2 * e]), __uint_as_float(x[b + 2 * e + 1])));
  return fmaxf(fmaxf(best[0], best[1]), fmaxf(best[2], best[3]));
}

// Moves m, `top` here, to kBelow under a row's maximum `now` where it has to, and
// returns what O and the sum are to be scaled by.
template <class T>
__device__ __forceinline__ float move_top(float& top, float now) {
  constexpr float kBelow = std::is_same<T, __half>::value ? 7.f : 0.f;
  now -= kBelow;
  if (!(now > top + kGrow || top == -INFINITY)) return 1.f;
  const float keep = now == -INFINITY ? 1.f : exp2_approx(top - now);  // 0 at the first keys
  top = now;
  return keep;
}

// P = exp2(c S - top) to tensor memory; returns the row's sum.
template <class T>
__device__ __forceinline__ float write_p(const uint32_t (&x)[kTile], float c, float top, uint32_t to) {
  const float off = top == -INFINITY ? 0.f : -top;
  const float2 c2 = make_float2(c, c), off2 = make_float2(off, off);
  float2 part[2] = {};
#pragma unroll
  for (int b = 0; b < 4; ++b) {
    uint32_t p[16];
#pragma unroll
    for (int e = 0; e < 16; ++e) {
      float2 u = fma2(pair_of(x + 32 * b + 2 * e), c2, off2);
      u = make_float2(exp2_approx(u.x), exp2_approx(u.y));
      part[e & 1] = add2(part[e & 1], u);
      p[e] = pack2<T>(u.x, u.y);
    }
    tmem_st16(to + 16 * b, p);
  }
  part[0] = add2(part[0], part[1]);
  return part[0].x + part[0].y;
}

template <int DP>
__device__ __forceinline__ void scale_o(uint32_t o_at, float keep) {
#pragma unroll
  for (int b = 0; b < DP / 32; ++b) {
    uint32_t o[32];
    tmem_ld32(o_at + 32 * b, o);
    tmem_ld_wait32(o);
#pragma unroll
    for (int e = 0; e < 32; ++e) o[e] = __float_as_uint(__uint_as_float(o[e]) * keep);
    tmem_st32(o_at + 32 * b, o);
  }
  tmem_st_wait();
}

// One row of the output, zeros where it saw no key.
template <class T, int DP>
__device__ __forceinline__ void write_o(uint32_t o_at, float sum, T* out, int dim, bool any, bool live) {
  const float inv = !any || sum == 0.f ? 0.f : 1.f / sum;
#pragma unroll
  for (int b = 0; b < DP / 32; ++b) {
    uint32_t o[32];
    if (any) {
      tmem_ld32(o_at + 32 * b, o);
      tmem_ld_wait32(o);
    }
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      if (!live || 32 * b + 8 * e >= dim) continue;
      uint4 w = make_uint4(0, 0, 0, 0);
      if (inv != 0.f) {
        uint32_t* ww = reinterpret_cast<uint32_t*>(&w);
#pragma unroll
        for (int f = 0; f < 4; ++f)
          ww[f] = pack2<T>(__uint_as_float(o[8 * e + 2 * f]) * inv, __uint_as_float(o[8 * e + 2 * f + 1]) * inv);
      }
      *reinterpret_cast<uint4*>(out + 32 * b + 8 * e) = w;
    }
  }
}

__device__ __forceinline__ float lse_of(float top, float sum) {
  return sum == 0.f ? -INFINITY : (top + log2f(sum)) * 0.6931471805599453f;
}

// S = q k^T of one tile of each.
template <int DP>
__device__ __forceinline__ void score(uint32_t to, uint32_t q, uint32_t k, uint32_t desc) {
  const TileDesc qd(q, 16), kd(k, 16);
  if (elect_one()) {
#pragma unroll
    for (int c = 0; c < DP / 16; ++c) {
      const uint32_t off = (c / 4) * Layout<DP>::kPanel + (c % 4) * 32;
      mma_ss(to, qd.at(off), kd.at(off), desc, c > 0);
    }
  }
}
// O += P v.
template <int DP, bool kBf16>
__device__ __forceinline__ void output(uint32_t to, uint32_t p, uint32_t v, bool first) {
  const TileDesc vd(v, Layout<DP>::kPanel);
  if (elect_one()) {
#pragma unroll
    for (int c = 0; c < kTile / 16; ++c)
      mma_ts(to, p + c * 8, vd.at(c * 2048), mma_desc(kBf16, DP, true), !first || c > 0);
  }
}

// One warp's load of a tile of keys or values; the rows of v behind the last
// key are other sequences' (or anything): P is 0 there, but 0 * NaN is not, so
// they are cleared before the product may read them.  k needs none of this: its
// scores are replaced.  `tail` is used once, for the last tile.
template <int DP>
__device__ __forceinline__ void load_kv(uint8_t* dst, const CUtensorMap* map, int head, int64_t row, int valid,
                                        bool is_v, uint64_t* full, uint64_t* tail) {
  const int lane = threadIdx.x & 31;
  const bool clear = is_v && valid < kTile;
  uint64_t* bar = clear ? tail : full;
  if (lane == 0) {
    bar_expect(bar, Layout<DP>::kTileBytes);
#pragma unroll
    for (int c = 0; c < DP / 64; ++c) tma_load(dst + c * Layout<DP>::kPanel, map, 64 * c, head, (int)row, bar);
  }
  if (clear) {
    bar_wait_warp(tail, 0, &g_timeouts);
    for (int c = 0; c < DP / 64; ++c)
      for (int b = valid * 8 + lane; b < kTile * 8; b += 32)
        reinterpret_cast<uint4*>(dst + c * Layout<DP>::kPanel)[b] = make_uint4(0, 0, 0, 0);
    fence_async_smem();
    __syncwarp();
    if (lane == 0) bar_arrive(full);
  }
}

// ------------------------------------------------------------ heads up to 64
constexpr int kOneStages = 4;

struct OneShared {
  uint64_t q_full, kv_full[kOneStages], kv_empty[kOneStages], s_full, s_read, p_ready, pv_done, tail, drained;
  uint32_t tmem;
  Tile tile;
};
constexpr int kOneBytes = (1 + kOneStages) * Layout<64>::kTileBytes + 1024;

// Warps 0-3: softmax, scaling, output; 4: products; 5: loads.
template <class T>
__global__ void __launch_bounds__(256, 2)
    one_tile_kernel(const __grid_constant__ Args a, const __grid_constant__ CUtensorMap q_map,
                    const __grid_constant__ CUtensorMap k_map, const __grid_constant__ CUtensorMap v_map) {
  constexpr int DP = 64;
  using L = Layout<DP>;
  constexpr bool kBf16 = std::is_same<T, __nv_bfloat16>::value;
  extern __shared__ uint8_t raw[];
  __shared__ OneShared s;
  uint8_t* sq = raw + (1024 - (smem_u32(raw) & 1023)) % 1024;
  uint8_t* skv = sq + L::kTileBytes;
  const int warp = __shfl_sync(0xffffffffu, (int)(threadIdx.x >> 5), 0), lane = threadIdx.x & 31;
  const int h = blockIdx.x % a.heads, m = h / (a.heads / a.kv_heads);

  if (warp == 0) {
    const Tile t = find_tile<false>(a, kTile, blockIdx.x / a.heads);
    if (lane == 0) s.tile = t;
  } else if (warp == 1 && lane == 0) {
    bar_init(&s.q_full, 1);
    for (int i = 0; i < kOneStages; ++i) {
      bar_init(&s.kv_full[i], 1);
      bar_init(&s.kv_empty[i], 1);
    }
    bar_init(&s.s_full, 1);
    bar_init(&s.s_read, 4);  // a warp arrives once
    bar_init(&s.p_ready, 4);
    bar_init(&s.pv_done, 1);
    bar_init(&s.tail, 1);
    bar_init(&s.drained, 1);
    fence_bar_init();
  } else if (warp == 4) {
    tmem_alloc(&s.tmem, 256);
  } else if (warp == 5 && lane == 0) {
    tma_prefetch(&q_map);
    tma_prefetch(&k_map);
    tma_prefetch(&v_map);
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = s.tmem, ts = tmem, tp = tmem + kTile, to = tp + kTile / 2;
  const Tile place = s.tile;
  const int lq = place.part < 0 ? 0 : place.lq, lk = place.lk, i0 = place.index * kTile, shift = lk - lq;
  // keys that query row i of the sequence sees
  auto seen = [&](int i) { return a.causal ? max(0, min(lk, i + shift + 1)) : lk; };
  const int n = place.part < 0 ? 0 : (seen(min(lq, i0 + kTile) - 1) + kTile - 1) / kTile;

  if (warp < 4) {
    regs_grow<200>();
    const int row = threadIdx.x, i = i0 + row, sees = seen(i), warp_sees = seen(i - lane);
    const uint32_t lanes = (uint32_t)(warp * 32) << 16;
    const float c = exponent_factor(a.scale);
    float top = -INFINITY, sum = 0.f;
    bool ok = true;
    for (int j = 0; j < n; ++j) {
      if (!(ok = bar_wait_warp(&s.s_full, j & 1, &g_timeouts))) break;
      tc_fence_after();
      uint32_t x[kTile];
#pragma unroll
      for (int b = 0; b < 4; ++b) tmem_ld32(ts + lanes + 32 * b, x + 32 * b);
#pragma unroll
      for (int b = 0; b < 4; ++b) tmem_ld_wait32(x + 32 * b);
      tc_fence_before();
      bar_arrive_warp(&s.s_read);
      if ((j + 1) * kTile > warp_sees) hide(x, sees - j * kTile);
      const float keep = move_top<T>(top, row_max(x) * c);
      if (j > 0) {  // the last product has read P and left O
        if (!(ok = bar_wait_warp(&s.pv_done, (j - 1) & 1, &g_timeouts))) break;
        tc_fence_after();
        if (__any_sync(0xffffffffu, keep != 1.f)) scale_o<DP>(to + lanes, keep);
      }
      sum = sum * keep + write_p<T>(x, c, top, tp + lanes);
      tmem_st_wait();
      tc_fence_before();
      bar_arrive_warp(&s.p_ready);
    }
    if (ok && n > 0) {
      ok = bar_wait_warp(&s.pv_done, (n - 1) & 1, &g_timeouts);
      tc_fence_after();
    }
    if (ok) {
      const bool live = i < lq && !BFB_BAD(place.q0 + i < a.total_q);
      T* out = static_cast<T*>(a.out) + ((place.q0 + i) * a.heads + h) * a.dim;
      write_o<T, DP>(to + lanes, sum, out, a.dim, n > 0, live);
      if (live) a.lse[(int64_t)h * a.total_q + place.q0 + i] = lse_of(top, sum);
    }
  } else {
    regs_shrink<56>();
    if (warp == 4 && n > 0) {
      const uint32_t ds = mma_desc(kBf16, kTile, false) | (a.scale < 0.f ? kNegateA : 0u);
      const uint32_t q_addr = smem_u32(sq), kv_addr = smem_u32(skv);
      // tiles come as k0 k1 v0 k2 v1 ..: the scores run one tile ahead
      int stage = 0;
      uint32_t phase = 0;
      auto next = [&](int& at) {
        at = stage;
        if (!bar_wait_warp(&s.kv_full[stage], phase, &g_timeouts)) return false;
        if (++stage == kOneStages) {
          stage = 0;
          phase ^= 1;
        }
        return true;
      };
      int at = 0;
      bool ok = bar_wait_warp(&s.q_full, 0, &g_timeouts) && next(at);
      if (ok) {
        tc_fence_after();
        score<DP>(ts, q_addr, kv_addr, ds);
        if (elect_one()) {
          mma_commit(&s.s_full);
          mma_commit(&s.kv_empty[0]);
        }
      }
      for (int j = 0; j < n && ok; ++j) {
        if (j + 1 < n) {
          if (!(ok = next(at) && bar_wait_warp(&s.s_read, j & 1, &g_timeouts))) break;
          tc_fence_after();
          score<DP>(ts, q_addr, kv_addr + at * L::kTileBytes, ds);
          if (elect_one()) {
            mma_commit(&s.s_full);
            mma_commit(&s.kv_empty[at]);
          }
        }
        if (!(ok = next(at) && bar_wait_warp(&s.p_ready, j & 1, &g_timeouts))) break;
        tc_fence_after();
        output<DP, kBf16>(to, tp, kv_addr + at * L::kTileBytes, j == 0);
        if (elect_one()) {
          mma_commit(&s.pv_done);
          mma_commit(&s.kv_empty[at]);
        }
      }
      if (elect_one()) mma_commit(&s.drained);  // nothing leaves before its products are done
      bar_wait_warp(&s.drained, 0, &g_timeouts);
    } else if (warp == 5 && n > 0) {
      if (lane == 0) {
        bar_expect(&s.q_full, L::kTileBytes);
        tma_load(sq, &q_map, 0, h, (int)(place.q0 + i0), &s.q_full);
      }
      int it = 0;
      for (; it < 2 * n; ++it) {
        const bool last = it == 2 * n - 1, is_v = it > 0 && (it % 2 == 0 || last);
        const int j = last ? n - 1 : is_v ? it / 2 - 1 : (it + 1) / 2, stage = it % kOneStages;
        bool ok = true;
        if (lane == 0) ok = bar_wait(&s.kv_empty[stage], ((it / kOneStages) & 1) ^ 1, &g_timeouts);
        if (!__shfl_sync(0xffffffffu, ok, 0)) break;
        load_kv<DP>(skv + stage * L::kTileBytes, is_v ? &v_map : &k_map, m, place.k0 + (int64_t)j * kTile,
                    lk - j * kTile, is_v, &s.kv_full[stage], &s.tail);
      }
      if (lane == 0 && it < 2 * n) {  // nor before its loads have landed
        bar_wait(&s.q_full, 0, &g_timeouts);
        for (int i = max(0, it - kOneStages); i < it; ++i)
          bar_wait(&s.kv_full[i % kOneStages], (i / kOneStages) & 1, &g_timeouts);
      }
    }
  }
  tc_fence_before();
  __syncthreads();
  if (warp == 4) {
    tc_fence_after();
    tmem_free(tmem, 256);
  }
}

// ----------------------------------------------------------- heads up to 128
constexpr int kTwoStages = 4;

struct TwoShared {
  uint64_t q_full, kv_full[kTwoStages], kv_empty[kTwoStages], s_full[2], p_ready[2], grown[2], o_full[2], sums[2];
  uint64_t tail, drained;
  uint32_t tmem;
  Tile tile;
  float scale[2][kTile];
  float sum[2][kTile];
};
constexpr int kTwoBytes = (2 + kTwoStages) * Layout<128>::kTileBytes + 1024;

// Warps 0-3 and 4-7: softmax of the two tiles; 8-11: scaling O and the output;
// 12: products; 13: loads.
template <class T>
__global__ void __launch_bounds__(512, 1)
    two_tile_kernel(const __grid_constant__ Args a, const __grid_constant__ CUtensorMap q_map,
                    const __grid_constant__ CUtensorMap k_map, const __grid_constant__ CUtensorMap v_map) {
  constexpr int DP = 128;
  using L = Layout<DP>;
  constexpr bool kBf16 = std::is_same<T, __nv_bfloat16>::value;
  extern __shared__ uint8_t raw[];
  __shared__ TwoShared s;
  uint8_t* sq = raw + (1024 - (smem_u32(raw) & 1023)) % 1024;
  uint8_t* skv = sq + 2 * L::kTileBytes;
  const int warp = __shfl_sync(0xffffffffu, (int)(threadIdx.x >> 5), 0), lane = threadIdx.x & 31;
  const int h = blockIdx.x % a.heads, m = h / (a.heads / a.kv_heads);

  if (warp == 0) {
    Tile t = find_tile<false>(a, 2 * kTile, blockIdx.x / a.heads);
    t.index *= 2;
    if (lane == 0) s.tile = t;
  } else if (warp == 1 && lane == 0) {
    bar_init(&s.q_full, 1);
    for (int i = 0; i < kTwoStages; ++i) {
      bar_init(&s.kv_full[i], 1);
      bar_init(&s.kv_empty[i], 1);
    }
    for (int i = 0; i < 2; ++i) {
      bar_init(&s.s_full[i], 1);
      bar_init(&s.p_ready[i], 8);  // a warp arrives once: 4 of softmax, 4 that scale O
      bar_init(&s.grown[i], 4);
      bar_init(&s.o_full[i], 1);
      bar_init(&s.sums[i], 4);
    }
    bar_init(&s.tail, 1);
    bar_init(&s.drained, 1);
    fence_bar_init();
  } else if (warp == 12) {
    tmem_alloc(&s.tmem, 512);
  } else if (warp == 13 && lane == 0) {
    tma_prefetch(&q_map);
    tma_prefetch(&k_map);
    tma_prefetch(&v_map);
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = s.tmem, to = tmem + 2 * kTile;  // S and P of the tiles, then O
  const Tile place = s.tile;
  const int lq = place.part < 0 ? 0 : place.lq, lk = place.lk, tile0 = place.index, shift = lk - lq;
  auto seen = [&](int i) { return a.causal ? max(0, min(lk, i + shift + 1)) : lk; };
  auto tiles_of = [&](int t) {
    const int first = (tile0 + t) * kTile;
    return place.part < 0 || first >= lq ? 0 : (seen(min(lq, first + kTile) - 1) + kTile - 1) / kTile;
  };
  const int n0 = tiles_of(0), n1 = tiles_of(1), n = max(n0, n1);

  if (warp < 8) {
    regs_grow<184>();
    const int t = warp >> 2, row = threadIdx.x & (kTile - 1), steps = t ? n1 : n0;
    const uint32_t ts = tmem + ((uint32_t)((warp & 3) * 32) << 16) + t * kTile;
    const int i = (tile0 + t) * kTile + row, sees = seen(i), warp_sees = seen(i - lane);
    const float c = exponent_factor(a.scale);
    float top = -INFINITY, sum = 0.f;
    for (int j = 0; j < steps; ++j) {
      if (!bar_wait_warp(&s.s_full[t], j & 1, &g_timeouts)) break;
      tc_fence_after();
      uint32_t x[kTile];
#pragma unroll
      for (int b = 0; b < 4; ++b) tmem_ld32(ts + 32 * b, x + 32 * b);
#pragma unroll
      for (int b = 0; b < 4; ++b) tmem_ld_wait32(x + 32 * b);
      if ((j + 1) * kTile > warp_sees) hide(x, sees - j * kTile);
      const float keep = move_top<T>(top, row_max(x) * c);
      s.scale[t][row] = keep;
      bar_arrive_warp(&s.grown[t]);
      sum = sum * keep + write_p<T>(x, c, top, ts);
      tmem_st_wait();
      tc_fence_before();
      bar_arrive_warp(&s.p_ready[t]);
    }
    s.sum[t][row] = sum;
    bar_arrive_warp(&s.sums[t]);
    if (i < lq && !BFB_BAD(place.q0 + i < a.total_q)) a.lse[(int64_t)h * a.total_q + place.q0 + i] = lse_of(top, sum);
  } else if (warp < 12) {
    regs_shrink<80>();
    const int row = threadIdx.x & (kTile - 1);
    const uint32_t lanes = (uint32_t)((warp & 3) * 32) << 16;
    bool ok = true;
    for (int j = 0; j < n && ok; ++j) {
      for (int t = 0; t < 2; ++t) {
        if (j >= (t ? n1 : n0)) continue;
        if (!(ok = bar_wait_warp(&s.grown[t], j & 1, &g_timeouts))) break;
        const float keep = s.scale[t][row];
        // O holds the keys before: the softmax has had this step's scores, which were issued behind their product
        if (j > 0 && __any_sync(0xffffffffu, keep != 1.f)) {
          tc_fence_after();
          scale_o<DP>(to + lanes + t * DP, keep);
          tc_fence_before();
        }
        bar_arrive_warp(&s.p_ready[t]);
      }
    }
    for (int t = 0; t < 2 && ok; ++t) {
      const int steps = t ? n1 : n0, i = (tile0 + t) * kTile + row;
      if (!(ok = bar_wait_warp(&s.sums[t], 0, &g_timeouts) &&
                 (steps == 0 || bar_wait_warp(&s.o_full[t], 0, &g_timeouts))))
        break;
      tc_fence_after();
      T* out = static_cast<T*>(a.out) + ((place.q0 + i) * a.heads + h) * a.dim;
      write_o<T, DP>(to + lanes + t * DP, s.sum[t][row], out, a.dim, steps > 0, i < lq && !BFB_BAD(place.q0 + i < a.total_q));
    }
  } else {
    regs_shrink<64>();
    if (warp == 12 && n > 0) {
      const uint32_t ds = mma_desc(kBf16, kTile, false) | (a.scale < 0.f ? kNegateA : 0u);
      const uint32_t kv_addr = smem_u32(skv), q_addr = smem_u32(sq);
      int stage = 0;
      uint32_t phase = 0;
      auto next = [&](int& at) {
        at = stage;
        if (!bar_wait_warp(&s.kv_full[stage], phase, &g_timeouts)) return false;
        if (++stage == kTwoStages) {
          stage = 0;
          phase ^= 1;
        }
        return true;
      };
      auto scores = [&](int t, int at) {
        score<DP>(tmem + t * kTile, q_addr + t * L::kTileBytes, kv_addr + at * L::kTileBytes, ds);
        if (elect_one()) mma_commit(&s.s_full[t]);
      };
      int vs = 0, ks = 0;
      bool ok = bar_wait_warp(&s.q_full, 0, &g_timeouts) && next(ks);
      if (ok) {
        tc_fence_after();
        if (n0 > 0) scores(0, 0);
        if (n1 > 0) scores(1, 0);
        if (elect_one()) mma_commit(&s.kv_empty[0]);
      }
      for (int j = 0; j < n && ok; ++j) {
        const bool more = j + 1 < n;
        if (!(ok = next(vs) && (!more || next(ks)))) break;
#pragma unroll
        for (int t = 0; t < 2; ++t) {
          const int steps = t ? n1 : n0;
          if (j >= steps) continue;
          if (!(ok = bar_wait_warp(&s.p_ready[t], j & 1, &g_timeouts))) break;
          tc_fence_after();
          output<DP, kBf16>(to + t * DP, tmem + t * kTile, kv_addr + vs * L::kTileBytes, j == 0);
          if (j + 1 < steps) scores(t, ks);
          else if (elect_one()) mma_commit(&s.o_full[t]);
        }
        if (!ok) break;
        if (elect_one()) {
          mma_commit(&s.kv_empty[vs]);
          if (more) mma_commit(&s.kv_empty[ks]);
        }
      }
      if (elect_one()) mma_commit(&s.drained);  // nothing leaves before its products are done
      bar_wait_warp(&s.drained, 0, &g_timeouts);
    } else if (warp == 13 && n > 0) {
      const int64_t q0 = place.q0 + (int64_t)tile0 * kTile;
      if (lane == 0) {
        const int tiles = (tile0 + 1) * kTile < lq ? 2 : 1;
        bar_expect(&s.q_full, tiles * L::kTileBytes);
        for (int t = 0; t < tiles; ++t)
          for (int c = 0; c < DP / 64; ++c)
            tma_load(sq + t * L::kTileBytes + c * L::kPanel, &q_map, 64 * c, h, (int)(q0 + t * kTile), &s.q_full);
      }
      int it = 0;
      for (; it < 2 * n; ++it) {  // k0 v0 k1 v1 ..
        const int stage = it % kTwoStages, j = it >> 1;
        bool ok = true;
        if (lane == 0) ok = bar_wait(&s.kv_empty[stage], ((it / kTwoStages) & 1) ^ 1, &g_timeouts);
        if (!__shfl_sync(0xffffffffu, ok, 0)) break;
        load_kv<DP>(skv + stage * L::kTileBytes, (it & 1) ? &v_map : &k_map, m, place.k0 + (int64_t)j * kTile,
                    lk - j * kTile, it & 1, &s.kv_full[stage], &s.tail);
      }
      if (lane == 0 && it < 2 * n) {  // nor before its loads have landed
        bar_wait(&s.q_full, 0, &g_timeouts);
        for (int i = max(0, it - kTwoStages); i < it; ++i)
          bar_wait(&s.kv_full[i % kTwoStages], (i / kTwoStages) & 1, &g_timeouts);
      }
    }
  }
  tc_fence_before();
  __syncthreads();
  if (warp == 12) {
    tc_fence_after();
    tmem_free(tmem, 512);
  }
}

template <class K>
int launch(K kernel, const Args& a, int dtype, int rows, int threads, int bytes, cudaStream_t stream) {
  // first: it makes the device's context current on this thread, which the tensor maps need
  BFB_CUDA(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes));
  CUtensorMap q, k, v;
  BFB_TRY(make_map(&q, a.q, dtype, a.total_q, a.heads, a.dim, a.q_row, a.q_head));
  // without keys nothing is loaded, but the maps need an address
  BFB_TRY(make_map(&k, a.total_k ? a.k : a.q, dtype, a.total_k, a.kv_heads, a.dim, a.k_row, a.k_head));
  BFB_TRY(make_map(&v, a.total_k ? a.v : a.q, dtype, a.total_k, a.kv_heads, a.dim, a.v_row, a.v_head));
  const int64_t blocks = tile_bound(a.total_q, a.seqs, rows) * a.heads;
  if (blocks > 0x7fffffff) return BFB_ERR_TOO_LARGE;
  kernel<<<(unsigned)blocks, threads, bytes, stream>>>(a, q, k, v);
  BFB_CHECK_LAUNCH();
  return BFB_OK;
}

}  // namespace

int forward_sm100(const Args& a, int dtype, cudaStream_t stream) {
  if (a.dim <= 64)
    return dtype == BFB_F16 ? launch(one_tile_kernel<__half>, a, dtype, kTile, 256, kOneBytes, stream)
                            : launch(one_tile_kernel<__nv_bfloat16>, a, dtype, kTile, 256, kOneBytes, stream);
  return dtype == BFB_F16 ? launch(two_tile_kernel<__half>, a, dtype, 2 * kTile, 512, kTwoBytes, stream)
                          : launch(two_tile_kernel<__nv_bfloat16>, a, dtype, 2 * kTile, 512, kTwoBytes, stream);
}

int timeouts_forward(uint64_t* count, int reset) {
  unsigned long long x = 0ull;
  BFB_CUDA(cudaMemcpyFromSymbol(&x, g_timeouts, sizeof(x)));
  if (reset) {
    const unsigned long long z = 0ull;
    BFB_CUDA(cudaMemcpyToSymbol(g_timeouts, &z, sizeof(z)));
  }
  *count += x;
  return BFB_OK;
}

// The driver's encoder is reached through the runtime, so the library needs no -lcuda.
int make_map(CUtensorMap* map, const void* base, int dtype, int64_t rows, int heads, int dim, int64_t row_stride,
             int64_t head_stride) {
  using Encode = CUresult (*)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*,
                              const cuuint64_t*, const cuuint32_t*, const cuuint32_t*, CUtensorMapInterleave,
                              CUtensorMapSwizzle, CUtensorMapL2promotion, CUtensorMapFloatOOBfill);
  // initialised once, whichever host thread comes first
  static const Encode encode = [] {
    void* f = nullptr;
    cudaDriverEntryPointQueryResult found;
    const cudaError_t err = cudaGetDriverEntryPointByVersion("cuTensorMapEncodeTiled", &f, 12000, cudaEnableDefault, &found);
    return err == cudaSuccess && found == cudaDriverEntryPointSuccess ? reinterpret_cast<Encode>(f) : nullptr;
  }();
  if (!encode) return BFB_ERR_CUDA;
  // a tensor without rows is described with one: no tile of it is ever loaded
  const cuuint64_t sizes[3] = {(cuuint64_t)dim, (cuuint64_t)heads, (cuuint64_t)(rows > 0 ? rows : 1)};
  const cuuint64_t strides[2] = {(cuuint64_t)head_stride * 2, (cuuint64_t)row_stride * 2};
  const cuuint32_t box[3] = {64, 1, kTile}, step[3] = {1, 1, 1};
  const CUresult r = encode(map, dtype == BFB_F16 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16,
                            3, const_cast<void*>(base), sizes, strides, box, step, CU_TENSOR_MAP_INTERLEAVE_NONE,
                            CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                            CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  return r == CUDA_SUCCESS ? BFB_OK : BFB_ERR_INVALID_ARG;
}

}  // namespace attn
}  // namespace bfb
