// Packed attention, backward, on the tensor cores.  With c = scale log2(e),
//   P = exp2(c S - lse2),  dS = P (scale dP - scale delta)
// one kernel owns key tiles and sums dK and dV over the query tiles and the
// query heads of its key head, another owns query tiles and sums dQ over the
// key tiles.  That computes S and dP twice (eight products, with the P K below, for
// the five that one kernel with dQ in atomics would need), but every sum has a fixed order,
// no fp32 copy of dQ goes through memory, and nothing has to be cleared first.
//
// Both keep their sums in tensor memory over the whole walk.  dS (and P for
// dV) are rounded to 16 bits and stay in tensor memory, over the scores they
// came from, as the next product's first operand (the rounding of dS is most
// of what dQ and dK lose: relative errors of 0.0024 in bf16 and 0.0003 in fp16
// against 64 bits, where fp32 inside has 0.0017 and 0.0002); each 128 x 128 step is
// worked by two warpgroups, one per 64 columns, with 64 values per thread.
//
// fp16 has few numbers below 2^-14, and dS = P (..) is small as soon as the keys
// are many or the incoming gradient is (a mean over tokens): rounded as it is it
// loses its bits there, most entries at last.  So each row of dS, a query's in
// the dQ kernel and a key's in the other, is taken times a power of two that
// brings its bound |scale| |dO| |v| + |delta| (norms; the largest of what the row
// meets) to 2^13, and the fp32 sum is divided by it; entries down to 2^-27 of the
// bound keep all bits.  P is taken times 2^15 in the same way.  Exact in fp32, and
// bf16, whose range is fp32's, needs none of it.
//
// delta is needed before the walk over the keys that could sum it.  Its first
// value comes from the rounded o, off by up to 2^-9 (bf16) of |dO| |o|, which
// all of a row's dS share: where the softmax is peaked (P near 1, dS near 0; the
// first rows of a causal prompt in any case) that would be most of dQ and dK.
// So the dQ kernel sums e = rowsum(P (dP - delta)) - dlse's share in fp32 on its
// walk, which is what delta lacks, keeps P K beside dS K, and subtracts e P K from
// dQ at the end; delta + e is left for the dK and dV kernel, which runs second.
// That costs the dQ kernel a fourth product.
//
// Measured, one sequence of 8192 tokens, full.  8/2 heads of 128, bf16: dQ 456 us
// (tensor pipe 61 % busy, special functions 36 %), dK and dV 440 us (63 and 37
// %); 8 heads of 64, fp16: 407 us (33 and 39 %) and 423 us (32 and 37 %).  The
// chain of a step bounds them, with one block to an SM.
#include <algorithm>
#include <cfloat>

#include "attention.cuh"

namespace bfb {

BFB_DEBUG_COUNTER();
BFB_DEBUG_READER(debug_violations_attention_bwd)

namespace attn {

namespace {

using namespace sm100;

__device__ unsigned long long g_timeouts = 0ull;

constexpr int kThreads = 384;  // warps 0-7 work on the scores, 8 issues products, 9 loads
constexpr int kHalf = kTile / 2;
constexpr float kLog2e = 1.4426950408889634f;
constexpr float kUp = 15.f, kDown = 1.f / 32768.f;  // fp16: log2 of P's factor, and its inverse
constexpr uint32_t kNone = 0xffffffffu;  // no place in tensor memory

// The eight warps that work on the scores meet; all of them come here.
__device__ __forceinline__ void warpgroups_sync() { asm volatile("bar.sync 1, 256;" ::: "memory"); }

template <int DP>
struct Layout {
  static constexpr int kTileBytes = kTile * DP * 2;
  static constexpr int kPanel = kTile * 128;
  // dV's product starts on the first half of P while the second is formed: with heads of 128, where a product takes
  // as long as that (causal, 0.7 - 4 k tokens, 16/4 heads: 295 -> 285 us; with 64 the arrivals cost more, 83 -> 85);
  // dQ's P K in the same way (forward and backward 825 -> 814)
  static constexpr bool kSplit = DP == 128;
  static constexpr int kTiles = 7;  // two resident tiles, three of the first ring, two of the second
};

// The walked tensors come through two rings: the first (queries or keys) is
// read by the scores and again by the last product of its step, so it needs a
// stage more than the second to be loaded in time.
constexpr int kFirst = 3, kSecond = 2;

struct Shared {
  uint64_t own_full, a_full[kFirst], a_empty[kFirst], b_full[kSecond], b_empty[kSecond];
  uint64_t s_full, dp_full, p_half, p_ready, ds_ready, done, tail;
  uint32_t tmem;
  Tile tile;
  float2 most[8];
  alignas(16) float lse2[kFirst][kTile];  // read four at a time
  alignas(16) float delta[kSecond][kTile];  // dQ: what delta lacks, a half row from each warpgroup
};

template <int DP>
constexpr size_t smem_bytes() { return (size_t)Layout<DP>::kTiles * Layout<DP>::kTileBytes + sizeof(Shared); }
static_assert(smem_bytes<128>() <= 227 * 1024, "a block's shared memory");

// K steps of 16 of a 16-bit operand that two warpgroups wrote as 2 x 64
// columns: the second half starts 64 columns of tensor memory later.
__device__ __forceinline__ constexpr uint32_t half_step(int c) { return (c >> 2) * kHalf + (c & 3) * 8; }

// Clears the rows [from, to) of a tile in shared memory, by one warp.  Rows
// behind a sequence, and queries that see no key, meet zeros of P and dS in the
// products, but 0 * NaN is not 0.
template <int DP>
__device__ __forceinline__ void clear_rows(uint8_t* tile, int from, int to) {
  for (int c = 0; c < DP / 64; ++c)
    for (int b = from * 8 + (threadIdx.x & 31); b < to * 8; b += 32)
      reinterpret_cast<uint4*>(tile + c * Layout<DP>::kPanel)[b] = make_uint4(0, 0, 0, 0);
}

template <int DP>
__device__ __forceinline__ void load_tile(uint8_t* dst, const CUtensorMap* map, int head, int64_t row, uint64_t* bar) {
#pragma unroll
  for (int c = 0; c < DP / 64; ++c) tma_load(dst + c * Layout<DP>::kPanel, map, 64 * c, head, (int)row, bar);
}

// dst += A B over 128 rows of B (A in tensor memory, B's rows along K).
template <int DP, bool kBf16>
__device__ __forceinline__ void product_rows(uint32_t dst, uint32_t a, uint32_t b, bool first) {
  const TileDesc bd(b, Layout<DP>::kPanel);
  if (elect_one()) {
#pragma unroll
    for (int c = 0; c < kTile / 16; ++c)
      mma_ts(dst, a + half_step(c), bd.at(c * 2048), mma_desc(kBf16, DP, true), !first || c > 0);
  }
}
// The half of its steps whose columns each warpgroup wrote first (c0 = 0) or last (2).
template <int DP, bool kBf16>
__device__ __forceinline__ void product_rows_half(uint32_t dst, uint32_t a, uint32_t b, bool first,
                                                  int c0) {
  const TileDesc bd(b, Layout<DP>::kPanel);
  if (elect_one()) {
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const int c = c0 + (e & 1) + (e >> 1) * 4;
      mma_ts(dst, a + half_step(c), bd.at(c * 2048), mma_desc(kBf16, DP, true), !first || e > 0);
    }
  }
}
// dst = A B^T over the columns of two tiles.
template <int DP, bool kBf16>
__device__ __forceinline__ void product_cols(uint32_t dst, uint32_t a, uint32_t b) {
  const TileDesc ad(a, 16), bd(b, 16);
  if (elect_one()) {
#pragma unroll
    for (int c = 0; c < DP / 16; ++c) {
      const uint32_t off = (c / 4) * Layout<DP>::kPanel + (c % 4) * 32;
      mma_ss(dst, ad.at(off), bd.at(off), mma_desc(kBf16, kTile, false), c > 0);
    }
  }
}

// Position in a ring of N stages.
template <int N>
struct Ring {
  int stage = 0;
  uint32_t phase = 0;
  __device__ __forceinline__ void step() {
    if (++stage == N) {
      stage = 0;
      phase ^= 1;
    }
  }
};

// `cols` fp32 columns of a 128-row sum from tensor memory, as 16-bit values
// [col0, col0 + cols) of a row of [rows, heads, dim], times `by`; less e times
// those at `less`, where that is given.
template <class T>
__device__ __forceinline__ void write_row(uint32_t from, T* out, int col0, int cols, int dim, bool live, bool zero,
                                          float by, uint32_t less = kNone, float e = 0.f) {
  for (int b = 0; b < cols; b += 32) {
    uint32_t o[32];
    tmem_ld32(from + b, o);
    tmem_ld_wait32(o);
    if (less != kNone) {
      uint32_t p[32];
      tmem_ld32(less + b, p);
      tmem_ld_wait32(p);
#pragma unroll
      for (int f = 0; f < 32; ++f) o[f] = __float_as_uint(fmaf(-e, __uint_as_float(p[f]), __uint_as_float(o[f])));
    }
#pragma unroll
    for (int g = 0; g < 4; ++g) {
      const int col = col0 + b + 8 * g;
      if (!live || col >= dim) continue;
      uint4 w = make_uint4(0, 0, 0, 0);
      uint32_t* ww = reinterpret_cast<uint32_t*>(&w);
      if (!zero) {
#pragma unroll
        for (int f = 0; f < 4; ++f)
          ww[f] = pack2<T>(__uint_as_float(o[8 * g + 2 * f]) * by, __uint_as_float(o[8 * g + 2 * f + 1]) * by);
      }
      *reinterpret_cast<uint4*>(out + col) = w;
    }
  }
}

// Finds the block's tile (of keys, or of queries) and its sequence, sets up
// the barriers; false if there is no such tile.
template <bool kKeys>
__device__ __forceinline__ bool setup(Shared& s, const Args& a, int64_t item) {
  if (threadIdx.x < 32) {
    const Tile t = find_tile<kKeys>(a, kTile, item);
    if (threadIdx.x == 0) {
      s.tile = t;
      bar_init(&s.own_full, 1);
      for (int i = 0; i < kFirst; ++i) {
        bar_init(&s.a_full[i], 2);
        bar_init(&s.a_empty[i], 1);
      }
      for (int i = 0; i < kSecond; ++i) {
        bar_init(&s.b_full[i], 2);
        bar_init(&s.b_empty[i], 1);
      }
      bar_init(&s.s_full, 1);
      bar_init(&s.dp_full, 1);
      bar_init(&s.p_half, 8);
      bar_init(&s.p_ready, 8);  // one arrival of each warp
      bar_init(&s.ds_ready, 8);
      bar_init(&s.done, 1);
      bar_init(&s.tail, 1);
      fence_bar_init();
    }
  }
  __syncthreads();
  return s.tile.part >= 0;
}

__device__ __forceinline__ uint32_t tmem_start(Shared& s, int warp) {
  if (warp == 8) tmem_alloc(&s.tmem, 512);
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  return s.tmem;
}
__device__ __forceinline__ void tmem_end(Shared& s, int warp) {
  tc_fence_before();
  __syncthreads();
  if (warp == 8) {
    tc_fence_after();
    tmem_free(s.tmem, 512);
  }
}

// The largest x and the largest y of all threads of the warps that work on the
// scores; once in a block.
__device__ __forceinline__ float2 largest(Shared& s, float x, float y) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, o));
    y = fmaxf(y, __shfl_xor_sync(0xffffffffu, y, o));
  }
  if ((threadIdx.x & 31) == 0) s.most[threadIdx.x >> 5] = make_float2(x, y);
  warpgroups_sync();
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    x = fmaxf(x, s.most[i].x);
    y = fmaxf(y, s.most[i].y);
  }
  return make_float2(x, y);
}

// The power of two that brings `bound` into [2^13, 2^14): sums stay below fp16's
// 65504 with room for roundings.  1 where there is no such bound.
__device__ __forceinline__ float lift(float bound) {
  if (!(bound >= FLT_MIN && bound <= FLT_MAX)) return 1.f;
  const int e = max((int)(__float_as_uint(bound) >> 23) - 127, -100);
  return __uint_as_float((uint32_t)(127 + 13 - e) << 23);
}

// One warp's load of a ring's stage: waits for the stage, fetches the rows by
// TMA with (src, not NULL) one value for each, negated, `add` added, `past` from
// row `valid` on, clears the rows from there on and those before `skip` (kClear),
// and signals `full` (two arrivals).  The values are fetched before the wait, all at once: one after
// another behind it, their latencies were most of a step.
template <int DP, bool kClear>
__device__ __forceinline__ bool load_stage(uint8_t* dst, const CUtensorMap* map, int head, int64_t row, int64_t rows, int skip, int valid,
                                           uint64_t* full, uint64_t* empty, uint32_t parity, uint64_t* tail,
                                           uint32_t& tails, const float* src = nullptr, float* values = nullptr,
                                           float past = 0.f, float add = 0.f) {
  const int lane = threadIdx.x & 31;
  bool ok = true;
  float x[4];
  if (src) {
#pragma unroll
    for (int e = 0; e < 4; ++e) x[e] = lane + 32 * e < valid && !BFB_BAD(row + lane + 32 * e < rows) ? add - src[lane + 32 * e] : past;
  }
  if (lane == 0) ok = bar_wait(empty, parity ^ 1, &g_timeouts);
  if (!__shfl_sync(0xffffffffu, ok, 0)) return false;
  const bool clear = kClear && (valid < kTile || skip > 0);
  if (lane == 0) {
    uint64_t* bar = clear ? tail : full;
    bar_expect(bar, Layout<DP>::kTileBytes);
    load_tile<DP>(dst, map, head, row, bar);
  }
  if (src) {
#pragma unroll
    for (int e = 0; e < 4; ++e) values[lane + 32 * e] = x[e];
  }
  if (clear) {
    ok = bar_wait_warp(tail, tails & 1, &g_timeouts);
    ++tails;
    if (!__all_sync(0xffffffffu, ok)) return false;
    clear_rows<DP>(dst, 0, skip);
    clear_rows<DP>(dst, valid, kTile);
    fence_async_smem();
  }
  __syncwarp();
  if (lane == 0) {
    bar_arrive(full);
    if (clear) bar_arrive(full);
  }
  return true;
}

// A loader that gave up leaves only when what it has asked for has landed:
// the resident tiles, the last loads of both rings (a_loads and b_loads
// issued), and one waiting to be cleared.
__device__ __forceinline__ void drain_loads(Shared& s, int a_loads, int b_loads, uint32_t tails) {
  bar_wait(&s.own_full, 0, &g_timeouts);
  for (int i = max(0, a_loads - kFirst); i < a_loads; ++i)
    bar_wait(&s.a_full[i % kFirst], (i / kFirst) & 1, &g_timeouts);
  for (int i = max(0, b_loads - kSecond); i < b_loads; ++i)
    bar_wait(&s.b_full[i % kSecond], (i / kSecond) & 1, &g_timeouts);
  if (tails > 0) bar_wait(&s.tail, (tails - 1) & 1, &g_timeouts);
}

// ------------------------------------------------------------------ dK and dV
// S^T = K Q^T, dP^T = V dO^T, dV += P^T dO, dK += dS^T Q: a thread owns one
// key row.  While the warpgroups form P the tensor core makes dP, while they
// form dS it adds to dV and makes the next S, and dK with the next dP after
// that: one buffer of each is enough, 128 + 128 + 2 DP columns.
template <class T, int DP>
__global__ void __launch_bounds__(kThreads, 1)
    dkv_kernel(const __grid_constant__ Args a, const __grid_constant__ CUtensorMap q_map,
               const __grid_constant__ CUtensorMap k_map, const __grid_constant__ CUtensorMap v_map,
               const __grid_constant__ CUtensorMap g_map) {
  using L = Layout<DP>;
  constexpr bool kBf16 = std::is_same<T, __nv_bfloat16>::value;
  extern __shared__ __align__(1024) uint8_t tiles[];
  Shared& s = *reinterpret_cast<Shared*>(tiles + L::kTiles * L::kTileBytes);
  uint8_t *sk = tiles, *sv = sk + L::kTileBytes, *sq = sv + L::kTileBytes, *sg = sq + kFirst * L::kTileBytes;
  const int warp = __shfl_sync(0xffffffffu, (int)(threadIdx.x >> 5), 0), lane = threadIdx.x & 31;
  const int m = blockIdx.x % a.kv_heads, group = a.heads / a.kv_heads;
  if (!setup<true>(s, a, blockIdx.x / a.kv_heads)) return;
  const uint32_t tmem = tmem_start(s, warp);
  const uint32_t ts = tmem, tdp = tmem + kTile, tdv = tmem + 2 * kTile, tdk = tdv + DP;
  const Tile place = s.tile;
  const int lq = place.lq, lk = place.lk, j0 = place.index * kTile, shift = lk - lq;
  // query tiles that see any of these keys: from the one with the first row i that has i + shift >= j0
  const int first = a.causal ? max(0, j0 - shift) / kTile : 0;
  const int per_head = j0 < lk ? max(0, (lq + kTile - 1) / kTile - first) : 0;
  const int n = per_head * group;

  if (warp < 8) {
    regs_grow<208>();
    const int wg = warp >> 2, row = threadIdx.x & (kTile - 1), j = j0 + row;
    const uint32_t lanes = (uint32_t)((warp & 3) * 32) << 16, mine = lanes + wg * kHalf;
    const float2 c2 = make_float2(a.scale * kLog2e, a.scale * kLog2e), scale2 = make_float2(a.scale, a.scale);
    float f = 1.f;
    if (!kBf16 && n > 0) {
      float g = 0.f, d = 0.f;
      for (int hh = 0; hh < group; ++hh) {  // the rows that see any of these keys
        const int64_t at = (int64_t)(m * group + hh) * a.total_q + place.q0;
#pragma unroll 4
        for (int i = (a.causal ? max(0, j0 - shift) : 0) + (int)threadIdx.x; i < lq; i += 256) {
          g = fmaxf(g, a.norm_g[at + i]);
          d = fmaxf(d, fabsf(a.delta[at + i]));
        }
      }
      const float2 most = largest(s, g, d);
      if (j < lk) f = lift(fabsf(a.scale) * most.x * a.norm_v[(int64_t)m * a.total_k + place.k0 + j] + most.y);
    }
    const float2 down2 = make_float2(f * kDown, f * kDown);
    bool ok = true;
    int tile = 0;
    for (int i = 0; i < n; ++i) {
      const int sa = i % kFirst, sb = i % kSecond;
      if (!(ok = bar_wait_warp(&s.a_full[sa], (i / kFirst) & 1, &g_timeouts) && bar_wait_warp(&s.s_full, i & 1, &g_timeouts)))
        break;
      tc_fence_after();
      uint32_t x[kHalf];
      tmem_ld32(ts + mine, x);
      tmem_ld32(ts + mine + 32, x + 32);
      // the half's first query, and the first of its columns from which key row j is seen
      const int q = (first + tile) * kTile + wg * kHalf;
      if (++tile == per_head) tile = 0;
      const int from = j - shift - q;
      const bool masked = a.causal && j0 + kTile - 1 - shift - q > 0;
      const float4* lse2 = reinterpret_cast<const float4*>(s.lse2[sa] + wg * kHalf);
      const float4* delta = reinterpret_cast<const float4*>(s.delta[sb] + wg * kHalf);
      tmem_ld_wait32(x);
      tmem_ld_wait32(x + 32);
      float p[kHalf];
#pragma unroll
      for (int e = 0; e < kHalf; e += 4) {
        const float4 l = lse2[e / 4];  // negative
        const float2 u = fma2(pair_of(x + e), c2, make_float2(l.x, l.y));
        const float2 v = fma2(pair_of(x + e + 2), c2, make_float2(l.z, l.w));
        p[e] = exp2_approx(u.x);
        p[e + 1] = exp2_approx(u.y);
        p[e + 2] = exp2_approx(v.x);
        p[e + 3] = exp2_approx(v.y);
        if (e % 32 == 28) {
          const int b = e / 32;
          if (masked) {
#pragma unroll
            for (int f = 32 * b; f < 32 * b + 32; ++f)
              if (f < from) p[f] = 0.f;
          }
          uint32_t w[16];
#pragma unroll
          for (int f = 0; f < 16; ++f) w[f] = pack2<T>(p[32 * b + 2 * f], p[32 * b + 2 * f + 1]);
          tmem_st16(ts + mine + 16 * b, w);
          if (b == 1 || L::kSplit) {
            tmem_st_wait();
            tc_fence_before();
            bar_arrive_warp(b ? &s.p_ready : &s.p_half);
          }
        }
      }
      if (!(ok = bar_wait_warp(&s.b_full[sb], (i / kSecond) & 1, &g_timeouts) && bar_wait_warp(&s.dp_full, i & 1, &g_timeouts)))
        break;
      tc_fence_after();
      tmem_ld32(tdp + mine, x);
      tmem_ld32(tdp + mine + 32, x + 32);
      tmem_ld_wait32(x);
      tmem_ld_wait32(x + 32);
#pragma unroll
      for (int b = 0; b < 2; ++b) {
        uint32_t w[16];
#pragma unroll
        for (int e = 0; e < 16; e += 2) {
          const int at = 32 * b + 2 * e;
          const float4 d = delta[at / 4];  // negative
          float2 u = mul2(make_float2(p[at], p[at + 1]), fma2(pair_of(x + at), scale2, make_float2(d.x, d.y)));
          float2 v = mul2(make_float2(p[at + 2], p[at + 3]), fma2(pair_of(x + at + 2), scale2, make_float2(d.z, d.w)));
          if (!kBf16) {
            u = mul2(u, down2);
            v = mul2(v, down2);
          }
          if (masked) {
            if (at < from) u.x = 0.f;
            if (at + 1 < from) u.y = 0.f;
            if (at + 2 < from) v.x = 0.f;
            if (at + 3 < from) v.y = 0.f;
          }
          w[e] = pack2<T>(u.x, u.y);
          w[e + 1] = pack2<T>(v.x, v.y);
        }
        tmem_st16(tdp + mine + 16 * b, w);
      }
      tmem_st_wait();
      tc_fence_before();
      bar_arrive_warp(&s.ds_ready);
    }
    if (ok && (n == 0 || bar_wait_warp(&s.done, 0, &g_timeouts))) {
      tc_fence_after();
      T* out = static_cast<T*>(wg ? a.dk : a.dv) + ((place.k0 + j) * a.kv_heads + m) * a.dim;
      write_row<T>((wg ? tdk : tdv) + lanes, out, 0, DP, a.dim, j < place.room && !BFB_BAD(place.k0 + j < a.total_k), n == 0 || j >= lk,
                   kBf16 ? 1.f : wg ? 1.f / f : kDown);
    }
  } else {
    regs_shrink<88>();
    if (warp == 8 && n > 0) {
      const uint32_t ka = smem_u32(sk), va = smem_u32(sv), q_addr = smem_u32(sq), g_addr = smem_u32(sg);
      Ring<kFirst> qr;  // of the next scores
      Ring<kSecond> gr;
      bool ok = bar_wait_warp(&s.own_full, 0, &g_timeouts) && bar_wait_warp(&s.a_full[0], 0, &g_timeouts) &&
                bar_wait_warp(&s.b_full[0], 0, &g_timeouts);
      if (ok) {
        tc_fence_after();
        product_cols<DP, kBf16>(ts, ka, q_addr);
        if (elect_one()) mma_commit(&s.s_full);
        product_cols<DP, kBf16>(tdp, va, g_addr);
        if (elect_one()) mma_commit(&s.dp_full);
      }
      for (int i = 0; i < n && ok; ++i) {
        const bool more = i + 1 < n;
        const int qs = qr.stage, gs = gr.stage;
        const uint32_t q_now = q_addr + qs * L::kTileBytes, g_now = g_addr + gs * L::kTileBytes;
        qr.step();
        gr.step();
        if (L::kSplit) {
          if (!(ok = bar_wait_warp(&s.p_half, i & 1, &g_timeouts))) break;
          tc_fence_after();
          product_rows_half<DP, kBf16>(tdv, ts, g_now, i == 0, 0);
          if (!(ok = bar_wait_warp(&s.p_ready, i & 1, &g_timeouts))) break;
          tc_fence_after();
          product_rows_half<DP, kBf16>(tdv, ts, g_now, false, 2);
        } else {
          if (!(ok = bar_wait_warp(&s.p_ready, i & 1, &g_timeouts))) break;
          tc_fence_after();
          product_rows<DP, kBf16>(tdv, ts, g_now, i == 0);
        }
        if (more) {
          if (!(ok = bar_wait_warp(&s.a_full[qr.stage], qr.phase, &g_timeouts))) break;
          product_cols<DP, kBf16>(ts, ka, q_addr + qr.stage * L::kTileBytes);
          if (elect_one()) mma_commit(&s.s_full);
        }
        if (!(ok = bar_wait_warp(&s.ds_ready, i & 1, &g_timeouts))) break;
        tc_fence_after();
        product_rows<DP, kBf16>(tdk, tdp, q_now, i == 0);
        if (elect_one()) {  // both: the threads are done with lse2 and delta, too
          mma_commit(&s.a_empty[qs]);
          mma_commit(&s.b_empty[gs]);
        }
        if (more) {
          if (!(ok = bar_wait_warp(&s.b_full[gr.stage], gr.phase, &g_timeouts))) break;
          product_cols<DP, kBf16>(tdp, va, g_addr + gr.stage * L::kTileBytes);
          if (elect_one()) mma_commit(&s.dp_full);
        }
      }
      if (elect_one()) mma_commit(&s.done);
      bar_wait_warp(&s.done, 0, &g_timeouts);  // nothing leaves before its products are done
    } else if (warp == 9 && n > 0) {
      if (lane == 0) {
        bar_expect(&s.own_full, 2 * L::kTileBytes);
        load_tile<DP>(sk, &k_map, m, place.k0 + j0, &s.own_full);
        load_tile<DP>(sv, &v_map, m, place.k0 + j0, &s.own_full);
      }
      uint32_t tails = 0;
      int i = 0, a_loads = 0, tile = 0, h = m * group;
      for (; i < n; ++i) {
        const int q = (first + tile) * kTile, valid = lq - q, sa = i % kFirst, sb = i % kSecond;
        const int64_t at = (int64_t)h * a.total_q + place.q0 + q;
        const int skip = a.causal ? max(0, -shift - q) : 0;  // queries that see no key
        // rows past the sequence: P = exp2(-inf) = 0
        if (!load_stage<DP, true>(sq + sa * L::kTileBytes, &q_map, h, place.q0 + q, a.total_q, skip, valid, &s.a_full[sa], &s.a_empty[sa],
                                  (i / kFirst) & 1, &s.tail, tails, a.lse2 + at, s.lse2[sa], -INFINITY, kBf16 ? 0.f : kUp))
          break;
        ++a_loads;
        if (!load_stage<DP, true>(sg + sb * L::kTileBytes, &g_map, h, place.q0 + q, a.total_q, skip, valid, &s.b_full[sb], &s.b_empty[sb],
                                  (i / kSecond) & 1, &s.tail, tails, a.delta + at, s.delta[sb], 0.f))
          break;
        if (++tile == per_head) {
          tile = 0;
          ++h;
        }
      }
      if (lane == 0 && i < n) drain_loads(s, a_loads, i, tails);
    }
  }
  tmem_end(s, warp);
}

// ------------------------------------------------------------------------- dQ
// S = Q K^T, dP = dO V^T, dQ += dS K, and P K beside it: a thread owns one query
// row.  The order of the steps is that of dK and dV: P K takes dV's place.
template <class T, int DP>
__global__ void __launch_bounds__(kThreads, 1)
    dq_kernel(const __grid_constant__ Args a, const __grid_constant__ CUtensorMap q_map,
              const __grid_constant__ CUtensorMap k_map, const __grid_constant__ CUtensorMap v_map,
              const __grid_constant__ CUtensorMap g_map) {
  using L = Layout<DP>;
  constexpr bool kBf16 = std::is_same<T, __nv_bfloat16>::value;
  extern __shared__ __align__(1024) uint8_t tiles[];
  Shared& s = *reinterpret_cast<Shared*>(tiles + L::kTiles * L::kTileBytes);
  uint8_t *sq = tiles, *sg = sq + L::kTileBytes, *sk = sg + L::kTileBytes, *sv = sk + kFirst * L::kTileBytes;
  const int warp = __shfl_sync(0xffffffffu, (int)(threadIdx.x >> 5), 0), lane = threadIdx.x & 31;
  const int h = blockIdx.x % a.heads, m = h / (a.heads / a.kv_heads);
  if (!setup<false>(s, a, blockIdx.x / a.heads)) return;
  const uint32_t tmem = tmem_start(s, warp);
  const uint32_t ts = tmem, tdp = tmem + kTile, tdq = tmem + 2 * kTile, tpk = tdq + DP;
  const Tile place = s.tile;
  const int lq = place.lq, lk = place.lk, i0 = place.index * kTile, shift = lk - lq;
  auto seen = [&](int i) { return a.causal ? max(0, min(lk, i + shift + 1)) : lk; };
  const int n = (seen(min(lq, i0 + kTile) - 1) + kTile - 1) / kTile;

  if (warp < 8) {
    regs_grow<208>();
    const int wg = warp >> 2, row = threadIdx.x & (kTile - 1), i = i0 + row;
    const uint32_t lanes = (uint32_t)((warp & 3) * 32) << 16, mine = lanes + wg * kHalf;
    const float2 c2 = make_float2(a.scale * kLog2e, a.scale * kLog2e);
    const int64_t at = (int64_t)h * a.total_q + place.q0 + i;
    const bool in_part = i < lq && !BFB_BAD(place.q0 + i < a.total_q);
    const float lse2 = in_part ? a.lse2[at] : INFINITY;
    const float delta = in_part ? a.delta[at] : 0.f;
    float f = 1.f;
    if (!kBf16 && n > 0) {
      float v = 0.f;
#pragma unroll 4
      for (int j = threadIdx.x; j < min(lk, n * kTile); j += 256) v = fmaxf(v, a.norm_v[(int64_t)m * a.total_k + place.k0 + j]);
      v = largest(s, v, 0.f).x;
      if (in_part) f = lift(fabsf(a.scale) * a.norm_g[at] * v + fabsf(delta));
    }
    const float down = kBf16 ? 1.f : f * kDown, off = (kBf16 ? 0.f : kUp) - lse2;
    const float2 off2 = make_float2(off, off), scale2 = make_float2(a.scale * down, a.scale * down),
                 delta2 = make_float2(-delta * down, -delta * down);
    float2 lacks = make_float2(0.f, 0.f);
    const int sees = seen(i), warp_sees = seen(i - lane);
    bool ok = true;
    for (int j = 0; j < n; ++j) {
      if (!(ok = bar_wait_warp(&s.s_full, j & 1, &g_timeouts))) break;
      tc_fence_after();
      uint32_t x[kHalf];
      tmem_ld32(ts + mine, x);
      tmem_ld32(ts + mine + 32, x + 32);
      tmem_ld_wait32(x);
      tmem_ld_wait32(x + 32);
      const int limit = sees - j * kTile - wg * kHalf;
      const bool masked = warp_sees < j * kTile + wg * kHalf + kHalf;
      float p[kHalf];
#pragma unroll
      for (int b = 0; b < 2; ++b) {
        uint32_t w[16];
#pragma unroll
        for (int e = 32 * b; e < 32 * b + 32; e += 2) {
          const float2 u = fma2(pair_of(x + e), c2, off2);
          p[e] = exp2_approx(u.x);
          p[e + 1] = exp2_approx(u.y);
          if (masked) {
            if (e >= limit) p[e] = 0.f;
            if (e + 1 >= limit) p[e + 1] = 0.f;
          }
          w[e / 2 - 16 * b] = pack2<T>(p[e], p[e + 1]);
        }
        tmem_st16(ts + mine + 16 * b, w);
        if (b == 1 || L::kSplit) {
          tmem_st_wait();
          tc_fence_before();
          bar_arrive_warp(b ? &s.p_ready : &s.p_half);
        }
      }
      if (!(ok = bar_wait_warp(&s.dp_full, j & 1, &g_timeouts))) break;
      tc_fence_after();
      tmem_ld32(tdp + mine, x);
      tmem_ld32(tdp + mine + 32, x + 32);
      tmem_ld_wait32(x);
      tmem_ld_wait32(x + 32);
#pragma unroll
      for (int b = 0; b < 2; ++b) {
        uint32_t w[16];
#pragma unroll
        for (int e = 0; e < 16; ++e) {
          const int col = 32 * b + 2 * e;
          float2 u = mul2(make_float2(p[col], p[col + 1]), fma2(pair_of(x + col), scale2, delta2));
          if (masked) {
            if (col >= limit) u.x = 0.f;
            if (col + 1 >= limit) u.y = 0.f;
          }
          lacks = add2(lacks, u);
          w[e] = pack2<T>(u.x, u.y);
        }
        tmem_st16(tdp + mine + 16 * b, w);
      }
      tmem_st_wait();
      tc_fence_before();
      bar_arrive_warp(&s.ds_ready);
    }
    s.delta[wg][row] = lacks.x + lacks.y;
    warpgroups_sync();
    // of a row that sees no key nothing is read
    const bool live = in_part && lse2 != INFINITY;
    const float e = live ? s.delta[0][row] + s.delta[1][row] - (a.dlse ? f * a.scale * a.dlse[at] : 0.f) : 0.f;
    if (ok && live && wg == 0) a.delta[at] = delta + e / f;
    if (ok && (n == 0 || bar_wait_warp(&s.done, 0, &g_timeouts))) {
      tc_fence_after();
      T* out = static_cast<T*>(a.dq) + ((place.q0 + i) * a.heads + h) * a.dim;
      const int col0 = wg * (DP / 2);
      write_row<T>(tdq + lanes + col0, out, col0, DP / 2, a.dim, in_part, n == 0, 1.f / f, tpk + lanes + col0,
                   kBf16 ? e : e * kDown);
    }
  } else {
    regs_shrink<88>();
    if (warp == 8 && n > 0) {
      const uint32_t qa = smem_u32(sq), ga = smem_u32(sg), k_addr = smem_u32(sk), v_addr = smem_u32(sv);
      Ring<kFirst> kr;  // of the next scores
      Ring<kSecond> vr;
      bool ok = bar_wait_warp(&s.own_full, 0, &g_timeouts) && bar_wait_warp(&s.a_full[0], 0, &g_timeouts) &&
                bar_wait_warp(&s.b_full[0], 0, &g_timeouts);
      if (ok) {
        tc_fence_after();
        product_cols<DP, kBf16>(ts, qa, k_addr);
        if (elect_one()) mma_commit(&s.s_full);
        product_cols<DP, kBf16>(tdp, ga, v_addr);
        if (elect_one()) {
          mma_commit(&s.dp_full);
          mma_commit(&s.b_empty[0]);
        }
      }
      for (int j = 0; j < n && ok; ++j) {
        const bool more = j + 1 < n;
        const int ks = kr.stage;
        const uint32_t k_now = k_addr + ks * L::kTileBytes;
        kr.step();
        vr.step();
        if (L::kSplit) {
          if (!(ok = bar_wait_warp(&s.p_half, j & 1, &g_timeouts))) break;
          tc_fence_after();
          product_rows_half<DP, kBf16>(tpk, ts, k_now, j == 0, 0);
          if (!(ok = bar_wait_warp(&s.p_ready, j & 1, &g_timeouts))) break;
          tc_fence_after();
          product_rows_half<DP, kBf16>(tpk, ts, k_now, false, 2);
        } else {
          if (!(ok = bar_wait_warp(&s.p_ready, j & 1, &g_timeouts))) break;
          tc_fence_after();
          product_rows<DP, kBf16>(tpk, ts, k_now, j == 0);
        }
        if (more) {
          if (!(ok = bar_wait_warp(&s.a_full[kr.stage], kr.phase, &g_timeouts))) break;
          product_cols<DP, kBf16>(ts, qa, k_addr + kr.stage * L::kTileBytes);
          if (elect_one()) mma_commit(&s.s_full);
        }
        if (!(ok = bar_wait_warp(&s.ds_ready, j & 1, &g_timeouts))) break;
        tc_fence_after();
        product_rows<DP, kBf16>(tdq, tdp, k_now, j == 0);
        if (elect_one()) mma_commit(&s.a_empty[ks]);
        if (more) {
          if (!(ok = bar_wait_warp(&s.b_full[vr.stage], vr.phase, &g_timeouts))) break;
          product_cols<DP, kBf16>(tdp, ga, v_addr + vr.stage * L::kTileBytes);
          if (elect_one()) {
            mma_commit(&s.dp_full);
            mma_commit(&s.b_empty[vr.stage]);
          }
        }
      }
      if (elect_one()) mma_commit(&s.done);
      bar_wait_warp(&s.done, 0, &g_timeouts);
    } else if (warp == 9 && n > 0) {
      if (lane == 0) {
        bar_expect(&s.own_full, 2 * L::kTileBytes);
        load_tile<DP>(sq, &q_map, h, place.q0 + i0, &s.own_full);
        load_tile<DP>(sg, &g_map, h, place.q0 + i0, &s.own_full);
      }
      uint32_t tails = 0;
      int j = 0, a_loads = 0;
      for (; j < n; ++j) {
        const int valid = lk - j * kTile, sa = j % kFirst, sb = j % kSecond;
        const int64_t k = place.k0 + (int64_t)j * kTile;
        if (!load_stage<DP, true>(sk + sa * L::kTileBytes, &k_map, m, k, a.total_k, 0, valid, &s.a_full[sa], &s.a_empty[sa],
                                  (j / kFirst) & 1, &s.tail, tails))
          break;
        ++a_loads;
        if (!load_stage<DP, false>(sv + sb * L::kTileBytes, &v_map, m, k, a.total_k, 0, valid, &s.b_full[sb], &s.b_empty[sb],
                                   (j / kSecond) & 1, &s.tail, tails))
          break;
      }
      if (lane == 0 && j < n) drain_loads(s, a_loads, j, tails);
    }
  }
  tmem_end(s, warp);
}

// What both kernels read for each query and head: lse2 = log2(e) lse, +inf
// where no key is seen (so that P = 0), and delta = scale (rowsum(dO o) - dlse);
// for fp16 the norms of dO's rows, too, and behind these units those of v's.
// A group of lanes takes a row, 16 bytes each.
template <class T>
__global__ void __launch_bounds__(256) rows_kernel(const __grid_constant__ Args a, int lanes) {
  constexpr bool kNorms = std::is_same<T, __half>::value;
  int64_t unit = ((int64_t)blockIdx.x * 256 + threadIdx.x) / lanes;  // row * heads + head
  const int lane = threadIdx.x & (lanes - 1);
  const bool of_v = kNorms && unit >= a.total_q * a.heads;
  if (of_v) unit -= a.total_q * a.heads;
  const int heads = of_v ? a.kv_heads : a.heads;
  const bool live = unit < (of_v ? a.total_k : a.total_q) * heads;
  const int64_t r = unit / heads, h = unit - r * heads;
  float d = 0.f, sq = 0.f;
  if (live && lane * 8 < a.dim) {
    const uint4 y = *reinterpret_cast<const uint4*>(
        (of_v ? static_cast<const T*>(a.v) + r * a.v_row + h * a.v_head : static_cast<const T*>(a.dout) + unit * a.dim) +
        lane * 8);
    const T* v = reinterpret_cast<const T*>(&y);
    if (!of_v) {
      const uint4 x = *reinterpret_cast<const uint4*>(static_cast<const T*>(a.out) + unit * a.dim + lane * 8);
      const T* u = reinterpret_cast<const T*>(&x);
#pragma unroll
      for (int e = 0; e < 8; ++e) d += to_f32<T>(u[e]) * to_f32<T>(v[e]);
    }
    if (kNorms) {
#pragma unroll
      for (int e = 0; e < 8; ++e) sq += to_f32<T>(v[e]) * to_f32<T>(v[e]);
    }
  }
  for (int o = lanes >> 1; o > 0; o >>= 1) {
    d += __shfl_xor_sync(0xffffffffu, d, o);
    if (kNorms) sq += __shfl_xor_sync(0xffffffffu, sq, o);
  }
  if (!live || lane > 0) return;
  const int64_t at = h * (of_v ? a.total_k : a.total_q) + r;
  if (kNorms) (of_v ? a.norm_v : a.norm_g)[at] = sqrtf(sq);
  if (of_v) return;
  const float lse = a.lse[at];
  a.lse2[at] = lse == -INFINITY ? INFINITY : lse * kLog2e;
  a.delta[at] = a.scale * (d - (a.dlse ? a.dlse[at] : 0.f));
}

template <class T, int DP>
int launch(const Args& a, int dtype, cudaStream_t stream) {
  constexpr int kBytes = (int)smem_bytes<DP>();
  // first: it makes the device's context current on this thread, which the tensor maps need
  BFB_CUDA(cudaFuncSetAttribute(dkv_kernel<T, DP>, cudaFuncAttributeMaxDynamicSharedMemorySize, kBytes));
  BFB_CUDA(cudaFuncSetAttribute(dq_kernel<T, DP>, cudaFuncAttributeMaxDynamicSharedMemorySize, kBytes));
  CUtensorMap q, k, v, g;
  const void* any = a.total_q ? a.q : a.k;  // an address for the maps of tensors without rows: never loaded
  BFB_TRY(make_map(&q, a.total_q ? a.q : any, dtype, a.total_q, a.heads, a.dim, a.q_row, a.q_head));
  BFB_TRY(make_map(&g, a.total_q ? a.dout : any, dtype, a.total_q, a.heads, a.dim, (int64_t)a.heads * a.dim, a.dim));
  BFB_TRY(make_map(&k, a.total_k ? a.k : any, dtype, a.total_k, a.kv_heads, a.dim, a.k_row, a.k_head));
  BFB_TRY(make_map(&v, a.total_k ? a.v : any, dtype, a.total_k, a.kv_heads, a.dim, a.v_row, a.v_head));
  const int64_t q_blocks = tile_bound(a.total_q, a.seqs, kTile) * a.heads;
  const int64_t k_blocks = tile_bound(a.total_k, a.seqs, kTile) * a.kv_heads;
  int lanes = 1;
  while (lanes * 8 < a.dim) lanes <<= 1;
  const int64_t norms = dtype == BFB_F16 ? a.total_k * a.kv_heads : 0;
  const int64_t row_blocks = ceil_div((a.total_q * a.heads + norms) * lanes, 256);
  if (std::max(std::max(q_blocks, k_blocks), row_blocks) > 0x7fffffff) return BFB_ERR_TOO_LARGE;
  if (a.total_q > 0) {
    rows_kernel<T><<<(unsigned)row_blocks, 256, 0, stream>>>(a, lanes);
    BFB_CHECK_LAUNCH();
  }
  if (a.total_q > 0) {
    dq_kernel<T, DP><<<(unsigned)q_blocks, kThreads, kBytes, stream>>>(a, q, k, v, g);
    BFB_CHECK_LAUNCH();
  }
  if (a.total_k > 0) {
    dkv_kernel<T, DP><<<(unsigned)k_blocks, kThreads, kBytes, stream>>>(a, q, k, v, g);
    BFB_CHECK_LAUNCH();
  }
  return BFB_OK;
}

}  // namespace

int backward_sm100(const Args& a, int dtype, cudaStream_t stream) {
  if (dtype == BFB_F16) return a.dim <= 64 ? launch<__half, 64>(a, dtype, stream) : launch<__half, 128>(a, dtype, stream);
  return a.dim <= 64 ? launch<__nv_bfloat16, 64>(a, dtype, stream) : launch<__nv_bfloat16, 128>(a, dtype, stream);
}

int timeouts_backward(uint64_t* count, int reset) {
  unsigned long long x = 0ull;
  BFB_CUDA(cudaMemcpyFromSymbol(&x, g_timeouts, sizeof(x)));
  if (reset) {
    const unsigned long long z = 0ull;
    BFB_CUDA(cudaMemcpyToSymbol(g_timeouts, &z, sizeof(z)));
  }
  *count += x;
  return BFB_OK;
}

}  // namespace attn
}  // namespace bfb
