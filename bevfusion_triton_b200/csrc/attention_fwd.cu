// Packed attention, forward, on the tensor cores.
//
// One block takes two tiles of 128 query rows of one head of one sequence and
// walks the keys in tiles of 128, with the running maximum and sum of the
// softmax:
//   S = q k^T        (tcgen05, both operands in shared memory, S in tensor memory)
//   P = exp2(c (S - m)),  c = scale log2(e): one thread per row, rounded to 16
//                    bits and written over S in tensor memory
//   O += P v         (tcgen05, P from tensor memory)
// O stays in tensor memory over all keys.  Where a row's maximum grows, O and
// the sum would have to be scaled down at every step; here the maximum in use
// is only moved when it grows by more than 2^8 (P stays below 2^8, far from
// fp16's range), so the scaling is rare and its result the same.
//
// Warps: 0-3 and 4-7 softmax of the two tiles, 8-11 scale O and write the
// output, 12 issues the products, 13 loads by TMA.  While one tile is in its
// softmax, the tensor core works on the other.
#include <cfloat>

#include "attention.cuh"

namespace bfb {
namespace attn {

namespace {

using namespace sm100;

__device__ unsigned long long g_timeouts = 0ull;

constexpr int kThreads = 512;
constexpr float kGrow = 8.f;  // log2 of the growth that moves the maximum

template <int DP>
struct Layout {
  static constexpr int kStages = DP == 128 ? 4 : 6;
  // With heads of up to 64 tensor memory has room for P beside S, and the next scores are made as soon as the
  // softmax has read the last ones.  With 128 P lies over S, and the next scores wait for the product with P.
  static constexpr bool kApart = DP == 64;
  static constexpr int kO = 2 * kTile;                              // first column of the outputs
  static constexpr int kP = kApart ? kO + 2 * DP : 0;               // of P of the first tile
  static constexpr int kPStep = kApart ? kTile / 2 : kTile;         // from one tile's P to the other's
  static constexpr int kTileBytes = kTile * DP * 2;
  static constexpr int kPanel = kTile * 128;  // 64 columns of a tile
  static constexpr int kBytes = (2 + kStages) * kTileBytes + 1024;
};

struct Shared {
  uint64_t q_full, kv_full[6], kv_empty[6], s_full[2], s_read[2], p_ready[2], pv_done[2], grown[2], turn[2], o_full[2], sums[2], tail, drained;
  uint32_t tmem;
  int64_t q0, k0;
  int lq, lk, tile, part;
  float scale[2][kTile];
  float sum[2][kTile];
};

template <class T, int DP>
__global__ void __launch_bounds__(kThreads, 1)
    forward_kernel(const __grid_constant__ Args a, const __grid_constant__ CUtensorMap q_map,
                   const __grid_constant__ CUtensorMap k_map, const __grid_constant__ CUtensorMap v_map) {
  using L = Layout<DP>;
  constexpr bool kBf16 = std::is_same<T, __nv_bfloat16>::value;
  extern __shared__ uint8_t raw[];
  __shared__ Shared s;
  uint8_t* base = raw + (1024 - (smem_u32(raw) & 1023)) % 1024;
  uint8_t* sq = base;
  uint8_t* skv = base + 2 * L::kTileBytes;
  const int warp = __shfl_sync(0xffffffffu, (int)(threadIdx.x >> 5), 0), lane = threadIdx.x & 31;
  const int h = blockIdx.x % a.heads, m = h / (a.heads / a.kv_heads);

  if (warp == 0) {
    const Tile t = find_tile(a.cu_q, a.seqs, a.total_q, 2 * kTile, blockIdx.x / a.heads);
    if (lane == 0) {
      s.part = t.part;
      if (t.part >= 0) {
        int64_t k0;
        int room;
        other_rows(a.cu_k, a.seqs, a.total_k, t.part, k0, room);
        s.q0 = t.start;
        s.lq = t.rows;
        // causal: the last tiles, which see the most keys, start first
        s.tile = 2 * ((t.rows + 2 * kTile - 1) / (2 * kTile) - 1 - t.index);
        s.k0 = k0;
        s.lk = used_keys(a.kv_lengths, t.part, room);
      }
      bar_init(&s.q_full, 1);
      for (int i = 0; i < L::kStages; ++i) {
        bar_init(&s.kv_full[i], 1);
        bar_init(&s.kv_empty[i], 1);
      }
      for (int i = 0; i < 2; ++i) {
        bar_init(&s.s_full[i], 1);
        bar_init(&s.s_read[i], 4);
        bar_init(&s.pv_done[i], 1);
        bar_init(&s.p_ready[i], 8);  // a warp arrives once: 4 of softmax, 4 that scale O
        bar_init(&s.grown[i], 4);
        bar_init(&s.turn[i], 4);
        bar_init(&s.o_full[i], 1);
        bar_init(&s.sums[i], 4);
      }
      bar_init(&s.tail, 1);
      bar_init(&s.drained, 1);
      fence_bar_init();
    }
  }
  __syncthreads();
  if (s.part < 0) return;
  if (warp == 12) tmem_alloc(&s.tmem, 512);
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = s.tmem;
  const int lq = s.lq, lk = s.lk, tile0 = s.tile, shift = lk - lq;

  // keys that query row i of the sequence sees
  auto seen = [&](int i) { return a.causal ? max(0, min(lk, i + shift + 1)) : lk; };
  auto tiles_of = [&](int t) {
    const int first = (tile0 + t) * kTile;
    if (first >= lq) return 0;
    return (seen(min(lq, first + kTile) - 1) + kTile - 1) / kTile;
  };
  const int n0 = tiles_of(0), n1 = tiles_of(1), n = max(n0, n1);

  if (warp < 8) {
    // ------------------------------------------------------------- softmax
    regs_grow<184>();
    const int t = warp >> 2, row = threadIdx.x & (kTile - 1), steps = t ? n1 : n0;
    const uint32_t lanes = tmem + ((uint32_t)((warp & 3) * 32) << 16);
    const uint32_t ts = lanes + t * kTile, tp = lanes + L::kP + t * L::kPStep;
    const int i = (tile0 + t) * kTile + row, sees = seen(i);
    const int warp_sees = seen(i - lane);  // of the warp's first row: the fewest
    // positive: a negative scale's sign goes into the product, and 0 is the smallest number (hidden scores stay
    // -inf, and every other exponent 0)
    const float c = fmaxf(fabsf(a.scale) * 1.4426950408889634f, FLT_MIN);
    float top = -INFINITY, sum = 0.f;
    bool ok = true;
    for (int j = 0; j < steps && ok; ++j) {
      if (!(ok = bar_wait(&s.s_full[t], j & 1, &g_timeouts))) break;
      tc_fence_after();
      uint32_t x[kTile];
#pragma unroll
      for (int b = 0; b < 4; ++b) tmem_ld32(ts + 32 * b, x + 32 * b);
#pragma unroll
      for (int b = 0; b < 4; ++b) tmem_ld_wait32(x + 32 * b);
      if (L::kApart) {
        tc_fence_before();
        bar_arrive_warp(&s.s_read[t]);
      }
      if ((j + 1) * kTile > warp_sees) {  // some keys are hidden: their scores, whatever they are, become -inf
        const int limit = sees - j * kTile;
#pragma unroll
        for (int b = 0; b < kTile; ++b)
          if (b >= limit) x[b] = 0xff800000u;
      }
      float best[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
      for (int b = 0; b < kTile; b += 8)
#pragma unroll
        for (int e = 0; e < 4; ++e)
          best[e] = fmaxf(best[e], fmaxf(__uint_as_float(x[b + 2 * e]), __uint_as_float(x[b + 2 * e + 1])));
      const float now = fmaxf(fmaxf(best[0], best[1]), fmaxf(best[2], best[3])) * c;
      float keep = 1.f;
      if (now > top + kGrow || top == -INFINITY) {
        keep = now == -INFINITY ? 1.f : exp2_approx(top - now);  // 0 at the first keys
        top = now;
      }
      s.scale[t][row] = keep;
      bar_arrive_warp(&s.grown[t]);
      const float off = top == -INFINITY ? 0.f : -top;
      const float2 c2 = make_float2(c, c), off2 = make_float2(off, off);
      float2 part[2] = {};
      if (L::kApart && j > 0) {  // P's columns are read
        if (!(ok = bar_wait(&s.pv_done[t], (j - 1) & 1, &g_timeouts))) break;
        tc_fence_after();
      }
      // Left alone the two tiles' warps fall into step, and the special-function pipe idles while both look for
      // their maxima: each lets the other begin its exponentials when its own are half done (bev map, 16200 cells,
      // 8 heads of 64: 818 -> 772 us; after a quarter or three quarters 777 and 819).
      if (L::kApart && j < min(n0, n1) && (t || j > 0)) {
        if (!(ok = bar_wait(&s.turn[t], (t ? j : j - 1) & 1, &g_timeouts))) break;
      }
#pragma unroll
      for (int b = 0; b < 4; ++b) {
        uint32_t p[16];
#pragma unroll
        for (int e = 0; e < 16; ++e) {
          const int at = 32 * b + 2 * e;
          float2 u = fma2(pair_of(x + at), c2, off2);
          u = make_float2(exp2_approx(u.x), exp2_approx(u.y));
          part[e & 1] = add2(part[e & 1], u);
          p[e] = pack2<T>(u.x, u.y);
        }
        tmem_st16(tp + 16 * b, p);
        if (L::kApart && b == 1) bar_arrive_warp(&s.turn[1 - t]);
      }
      part[0] = add2(part[0], part[1]);
      sum = sum * keep + (part[0].x + part[0].y);
      tmem_st_wait();
      tc_fence_before();
      bar_arrive_warp(&s.p_ready[t]);
    }
    s.sum[t][row] = sum;
    bar_arrive_warp(&s.sums[t]);
    if (i < lq)
      a.lse[(int64_t)h * a.total_q + s.q0 + i] = sum == 0.f ? -INFINITY : (top + log2f(sum)) * 0.6931471805599453f;
  } else if (warp < 12) {
    // ------------------------------------------------- scaling O, the output
    regs_shrink<80>();
    const int row = threadIdx.x & (kTile - 1);
    const uint32_t to = tmem + ((uint32_t)((warp & 3) * 32) << 16) + L::kO;
    bool ok = true;
    for (int j = 0; j < n && ok; ++j) {
      for (int t = 0; t < 2; ++t) {
        if (j >= (t ? n1 : n0)) continue;
        if (!(ok = bar_wait(&s.grown[t], j & 1, &g_timeouts))) break;
        const float keep = s.scale[t][row];
        if (j > 0 && __any_sync(0xffffffffu, keep != 1.f)) {
          // O holds the keys before.  Where P lies over S that is known: the softmax has had this step's scores,
          // which were issued behind their product.
          if (L::kApart && !(ok = bar_wait(&s.pv_done[t], (j - 1) & 1, &g_timeouts))) break;
          tc_fence_after();
#pragma unroll
          for (int b = 0; b < DP / 32; ++b) {
            uint32_t o[32];
            tmem_ld32(to + t * DP + 32 * b, o);
            tmem_ld_wait32(o);
#pragma unroll
            for (int e = 0; e < 32; ++e) o[e] = __float_as_uint(__uint_as_float(o[e]) * keep);
            tmem_st32(to + t * DP + 32 * b, o);
          }
          tmem_st_wait();
          tc_fence_before();
        }
        bar_arrive_warp(&s.p_ready[t]);
      }
    }
    for (int t = 0; t < 2 && ok; ++t) {
      const int steps = t ? n1 : n0, i = (tile0 + t) * kTile + row;
      float inv = 0.f;
      if (!(ok = bar_wait(&s.sums[t], 0, &g_timeouts))) break;
      if (steps > 0) {
        if (!(ok = bar_wait(&s.o_full[t], 0, &g_timeouts))) break;
        tc_fence_after();
        const float sum = s.sum[t][row];
        inv = sum == 0.f ? 0.f : 1.f / sum;
      }
      T* out = static_cast<T*>(a.out) + ((s.q0 + i) * a.heads + h) * a.dim;
#pragma unroll
      for (int b = 0; b < DP / 32; ++b) {
        uint32_t o[32];
        if (steps > 0) {
          tmem_ld32(to + t * DP + 32 * b, o);
          tmem_ld_wait32(o);
        }
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          if (i >= lq || 32 * b + 8 * e >= a.dim) continue;
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
  } else {
    regs_shrink<64>();
    if (warp == 12 && n > 0) {
      // ---------------------------------------------------------- products
      constexpr uint32_t dv = mma_desc(kBf16, DP, true);
      const uint32_t ds = mma_desc(kBf16, kTile, false) | (a.scale < 0.f ? kNegateA : 0u);
      const bool leader = elect_one();
      const uint32_t kv_addr = smem_u32(skv), q_addr = smem_u32(sq);
      auto score = [&](int t, int stage) {
        const TileDesc qd(q_addr + t * L::kTileBytes, 16), kd(kv_addr + stage * L::kTileBytes, 16);
        if (leader) {
#pragma unroll
          for (int c = 0; c < DP / 16; ++c) {
            const uint32_t off = (c / 4) * L::kPanel + (c % 4) * 32;
            mma_ss(tmem + t * kTile, qd.at(off), kd.at(off), ds, c > 0);
          }
          mma_commit(&s.s_full[t]);
        }
      };
      // the rings' next stage and phase
      int stage = 0;
      uint32_t phase = 0;
      auto full = [&](int st, uint32_t ph) { return bar_wait(&s.kv_full[st], ph, &g_timeouts); };
      auto step = [&] {
        if (++stage == L::kStages) {
          stage = 0;
          phase ^= 1;
        }
      };
      bool ok = bar_wait(&s.q_full, 0, &g_timeouts) && full(0, 0);
      if (ok) {
        tc_fence_after();
        if (n0 > 0) score(0, 0);
        if (n1 > 0) score(1, 0);
        if (leader) mma_commit(&s.kv_empty[0]);
      }
      step();
      auto output = [&](int t, int j, const TileDesc& vd, bool last) {
        if (leader) {
#pragma unroll
          for (int c = 0; c < kTile / 16; ++c)
            mma_ts(tmem + L::kO + t * DP, tmem + L::kP + t * L::kPStep + c * 8, vd.at(c * 2048), dv, j > 0 || c > 0);
          if (L::kApart) mma_commit(&s.pv_done[t]);
          if (last) mma_commit(&s.o_full[t]);
        }
      };
      for (int j = 0; j < n && ok; ++j) {
        const bool more = j + 1 < n;
        int ks = 0, vs = 0;
        if (L::kApart && more) {
          ks = stage;
          if (!(ok = full(stage, phase))) break;
          step();
#pragma unroll
          for (int t = 0; t < 2; ++t) {
            if (j + 1 >= (t ? n1 : n0)) continue;
            if (!(ok = bar_wait(&s.s_read[t], j & 1, &g_timeouts))) break;
            tc_fence_after();
            score(t, ks);
          }
          if (!ok) break;
          if (leader) mma_commit(&s.kv_empty[ks]);
        }
        vs = stage;
        if (!(ok = full(stage, phase))) break;
        step();
        if (!L::kApart && more) {
          ks = stage;
          if (!(ok = full(stage, phase))) break;
          step();
        }
        const TileDesc vd(kv_addr + vs * L::kTileBytes, L::kPanel);
#pragma unroll
        for (int t = 0; t < 2; ++t) {
          const int steps = t ? n1 : n0;
          if (j >= steps) continue;
          if (!(ok = bar_wait(&s.p_ready[t], j & 1, &g_timeouts))) break;
          tc_fence_after();
          output(t, j, vd, j + 1 == steps);
          if (!L::kApart && j + 1 < steps) score(t, ks);
        }
        if (!ok) break;
        if (leader) {
          mma_commit(&s.kv_empty[vs]);
          if (!L::kApart && more) mma_commit(&s.kv_empty[ks]);
        }
      }
      // nothing leaves before its products are done
      if (leader) mma_commit(&s.drained);
      bar_wait(&s.drained, 0, &g_timeouts);
    } else if (warp == 13 && n > 0) {
      // -------------------------------------------------------------- loads
      const int64_t q0 = s.q0 + (int64_t)tile0 * kTile, k0 = s.k0;
      if (lane == 0) {
        tma_prefetch(&q_map);
        tma_prefetch(&k_map);
        tma_prefetch(&v_map);
        const bool two = (tile0 + 1) * kTile < lq;
        bar_expect(&s.q_full, (two ? 2 : 1) * L::kTileBytes);
        for (int t = 0; t < (two ? 2 : 1); ++t)
          for (int c = 0; c < DP / 64; ++c)
            tma_load(sq + t * L::kTileBytes + c * L::kPanel, &q_map, 64 * c, h, (int)(q0 + t * kTile), &s.q_full);
      }
      bool ok = true;
      int it = 0;
      for (; it < 2 * n; ++it) {
        // in the order of their use: k0 v0 k1 v1 .., or k0 k1 v0 k2 v1 .. where the scores run ahead
        const bool is_v = L::kApart ? it > 0 && (it % 2 == 0 || it == 2 * n - 1) : it % 2 == 1;
        const int j = !L::kApart ? it >> 1 : it == 2 * n - 1 ? n - 1 : is_v ? it / 2 - 1 : (it + 1) / 2;
        const int stage = it % L::kStages, valid = lk - j * kTile;
        if (lane == 0) ok = bar_wait(&s.kv_empty[stage], ((it / L::kStages) & 1) ^ 1, &g_timeouts);
        if (!(ok = __shfl_sync(0xffffffffu, ok, 0))) break;
        uint8_t* dst = skv + stage * L::kTileBytes;
        // Rows of v behind the last key are other sequences' (or anything): P is 0 there, but 0 * NaN is
        // not, so the last tile's are cleared before the product may read them.  k needs none of this:
        // its scores are replaced.
        const bool clear = is_v && valid < kTile;
        uint64_t* bar = clear ? &s.tail : &s.kv_full[stage];
        if (lane == 0) {
          bar_expect(bar, L::kTileBytes);
          for (int c = 0; c < DP / 64; ++c)
            tma_load(dst + c * L::kPanel, is_v ? &v_map : &k_map, 64 * c, m, (int)(k0 + (int64_t)j * kTile), bar);
        }
        if (clear) {  // once: the last tile
          ok = bar_wait(&s.tail, 0, &g_timeouts);
          for (int c = 0; c < DP / 64; ++c)
            for (int b = valid * 8 + lane; b < kTile * 8; b += 32)
              reinterpret_cast<uint4*>(dst + c * L::kPanel)[b] = make_uint4(0, 0, 0, 0);
          fence_async_smem();
          __syncwarp();
          if (lane == 0) bar_arrive(&s.kv_full[stage]);
        }
      }
      // nor before its loads have landed
      if (lane == 0 && it < 2 * n) {
        bar_wait(&s.q_full, 0, &g_timeouts);
        for (int i = max(0, it - L::kStages); i < it; ++i)
          bar_wait(&s.kv_full[i % L::kStages], (i / L::kStages) & 1, &g_timeouts);
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

template <class T, int DP>
int launch(const Args& a, int dtype, cudaStream_t stream) {
  // first: it makes the device's context current on this thread, which the tensor maps need
  BFB_CUDA(cudaFuncSetAttribute(forward_kernel<T, DP>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                Layout<DP>::kBytes));
  CUtensorMap q, k, v;
  BFB_TRY(make_map(&q, a.q, dtype, a.total_q, a.heads, a.dim, a.q_row, a.q_head));
  // without keys nothing is loaded, but the maps need an address
  BFB_TRY(make_map(&k, a.total_k ? a.k : a.q, dtype, a.total_k, a.kv_heads, a.dim, a.k_row, a.k_head));
  BFB_TRY(make_map(&v, a.total_k ? a.v : a.q, dtype, a.total_k, a.kv_heads, a.dim, a.v_row, a.v_head));
  const int64_t blocks = tile_bound(a.total_q, a.seqs, 2 * kTile) * a.heads;
  if (blocks > 0x7fffffff) return BFB_ERR_TOO_LARGE;
  forward_kernel<T, DP><<<(unsigned)blocks, kThreads, Layout<DP>::kBytes, stream>>>(a, q, k, v);
  BFB_CHECK_LAUNCH();
  return BFB_OK;
}

}  // namespace

int forward_sm100(const Args& a, int dtype, cudaStream_t stream) {
  if (dtype == BFB_F16) return a.dim <= 64 ? launch<__half, 64>(a, dtype, stream) : launch<__half, 128>(a, dtype, stream);
  return a.dim <= 64 ? launch<__nv_bfloat16, 64>(a, dtype, stream) : launch<__nv_bfloat16, 128>(a, dtype, stream);
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
  static Encode encode = nullptr;
  if (!encode) {
    void* f = nullptr;
    cudaDriverEntryPointQueryResult found;
    BFB_CUDA(cudaGetDriverEntryPointByVersion("cuTensorMapEncodeTiled", &f, 12000, cudaEnableDefault, &found));
    if (!f || found != cudaDriverEntryPointSuccess) return BFB_ERR_CUDA;
    encode = reinterpret_cast<Encode>(f);
  }
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
