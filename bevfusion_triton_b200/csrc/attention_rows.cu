// Packed attention, forward, for few queries against long keys: the newest
// token of each stream against its cache.
//
// Each key and value is then read for a handful of rows, so HBM bounds it and
// the point is to keep enough loads in flight on every SM.  The work, tiles of
// 64 / kHeads keys for kHeads times 16 rows (queries x query heads of a key
// head), is laid out in one line, (sequence, key heads, row tile) by (sequence,
// ..) and key tile by key tile within, and cut into equal stretches, one per block, whatever the
// sequences' lengths are.  A block that covers all keys of a group of rows
// writes its output; of the groups that a cut goes through it writes a record
// (maximum, sum, unscaled output), and a second kernel joins those.  A block
// has at most two: at its start and at its end.
//
// A block's four warps take kHeads key heads at once (4, 2 or 1, what divides
// their number) by 16 keys each, so that what they ask for together lies in
// long runs (a token's heads are neighbours in memory).  Each has its own
// cp.async stages and its own running softmax, and the warps meet only at the
// end of a group.  The products are mma.sync m16n8k16: the rows fill a 16-row
// fragment at best, a tcgen05 tile of 128 rows would be mostly padding, and
// the tensor pipe is not what bounds this.
//
// 24 streams of one query, caches of up to 30 k keys, 32/8 heads of 128, bf16 (479 MB): 114 us, 4.2 TB/s; a plain
// sum over as many bytes reaches 5.0.  Three stages and two blocks to an SM: two stages 112, three blocks 123
// (registers spill), eight warps and key heads in one block 118, one key head at a time 118.
#include <algorithm>

#include "attention.cuh"

namespace bfb {

BFB_DEBUG_COUNTER();
BFB_DEBUG_READER(debug_violations_attention_rows)

namespace attn {

namespace {

using sm100::exp2_approx;
using sm100::pack2;
using sm100::smem_u32;

constexpr int kWarps = 4, kThreads = 32 * kWarps;
constexpr int kRows = 16;
constexpr int kWarpKeys = 16;
constexpr int kStages = 3;
constexpr int kLeastTiles = 4;  // a block's least stretch: below it the joining costs more than the split gives
constexpr float kLn2 = 0.6931471805599453f;

template <int DP>
__host__ __device__ constexpr int stage_bytes() { return 2 * kWarpKeys * DP * 2; }  // keys and values of one warp
template <int DP>
__host__ __device__ constexpr int record_floats() { return kRows * DP + 2 * kRows; }

struct Seq {
  int64_t q0, k0;
  int lq, lk;
  int row_tiles, tiles;
  int64_t work;  // of all its key heads
};

// What the line's functions need beside the arguments: key heads of a block.
template <int kHeads>
__device__ __forceinline__ Seq seq_at(const Args& a, int s) {
  Seq x;
  x.q0 = part_start(a.cu_q, a.seqs, a.total_q, s + 1);
  x.lq = (int)max(part_start(a.cu_q, a.seqs, a.total_q, s + 2) - x.q0, (int64_t)0);
  x.k0 = part_start(a.cu_k, a.seqs, a.total_k, s + 1);
  const int room = (int)max(part_start(a.cu_k, a.seqs, a.total_k, s + 2) - x.k0, (int64_t)0);
  x.lk = a.kv_lengths ? min(max(a.kv_lengths[s], 0), room) : room;
  x.row_tiles = (int)(((int64_t)x.lq * (a.heads / a.kv_heads) + kRows - 1) / kRows);
  constexpr int kKeys = kWarpKeys * kWarps / kHeads;
  x.tiles = (x.lk + kKeys - 1) / kKeys;
  x.work = (int64_t)x.row_tiles * x.tiles * (a.kv_heads / kHeads);
  return x;
}

// End of sequence `s` in the line (lane-parallel inclusive sums), for the 32
// sequences from `base` on.
template <int kHeads>
__device__ __forceinline__ int64_t line_ends(const Args& a, int base, int64_t before) {
  const int lane = threadIdx.x & 31, s = base + lane;
  int64_t upto = s < a.seqs ? seq_at<kHeads>(a, s).work : 0;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int64_t x = __shfl_up_sync(0xffffffffu, upto, o);
    if (lane >= o) upto += x;
  }
  return before + upto;
}

template <int kHeads>
__device__ __forceinline__ int64_t line_length(const Args& a) {
  int64_t total = 0;
  for (int base = 0; base < a.seqs; base += 32) total = __shfl_sync(0xffffffffu, line_ends<kHeads>(a, base, total), 31);
  return total;
}

__device__ __forceinline__ int64_t stretch(int64_t total, int blocks) {
  return max((total + blocks - 1) / blocks, (int64_t)kLeastTiles);
}

__device__ __forceinline__ void cp16(uint32_t dst, const void* src, bool there) {
  asm volatile("cp.async.cg.shared.global.L2::128B [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(there ? 16 : 0)
               : "memory");
}
__device__ __forceinline__ void ldm4(uint32_t addr, uint32_t (&r)[4]) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr)
               : "memory");
}
__device__ __forceinline__ void ldm4t(uint32_t addr, uint32_t (&r)[4]) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr)
               : "memory");
}
template <class T>
__device__ __forceinline__ void mma(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1);
template <>
__device__ __forceinline__ void mma<__half>(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
template <>
__device__ __forceinline__ void mma<__nv_bfloat16>(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

template <class T, int DP, int kHeads>
__global__ void __launch_bounds__(kThreads, 2)
    rows_kernel(const __grid_constant__ Args a, float* __restrict__ records) {
  extern __shared__ __align__(128) uint8_t smem[];
  __shared__ float top_s[kWarps][kRows], sum_s[kWarps][kRows];
  // exponentials are taken from 15 below the maximum in fp16: P up to 2^15, a long tail's keys no subnormal numbers
  constexpr float kBelow = std::is_same<T, __half>::value ? 15.f : 0.f;
  constexpr int kChunks = DP / 8;  // 16-byte chunks of a row; chunk c of row r sits at c ^ (r % 8)
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, quad = lane & 3, g = lane >> 2;
  const int group = a.heads / a.kv_heads;
  uint8_t* mine = smem + warp * kStages * stage_bytes<DP>();
  const uint32_t mine_u = smem_u32(mine);
  const float c = a.scale * 1.4426950408889634f;

  constexpr int kKeys = kWarpKeys * kWarps / kHeads;  // of a tile
  const int head = warp % kHeads, slice = warp / kHeads;
  asm volatile("griddepcontrol.launch_dependents;");  // the joining kernel may set itself up
  const int64_t total = line_length<kHeads>(a), per = stretch(total, gridDim.x);
  const int64_t begin = (int64_t)blockIdx.x * per, end = min(begin + per, total);
  if (begin >= end) return;
  // the sequence that `begin` falls into
  int s = 0;
  int64_t base = 0;
  for (int b = 0; b < a.seqs; b += 32) {
    const int64_t ends = line_ends<kHeads>(a, b, base);
    const unsigned hit = __ballot_sync(0xffffffffu, begin < ends);
    if (hit) {
      const int src = __ffs(hit) - 1;
      const int64_t prev = __shfl_up_sync(0xffffffffu, ends, 1);
      base = src ? __shfl_sync(0xffffffffu, prev, src) : base;
      s = b + src;
      break;
    }
    base = __shfl_sync(0xffffffffu, ends, 31);
  }
  Seq x = seq_at<kHeads>(a, s);

  for (int64_t pos = begin; pos < end;) {
    while (pos - base >= x.work) {
      base += x.work;
      x = seq_at<kHeads>(a, ++s);
    }
    const int64_t local = pos - base;
    const int unit = (int)(local / x.tiles), rt = unit % x.row_tiles;
    const int m0 = unit / x.row_tiles * kHeads, m = m0 + head;
    const int tile0 = (int)(local % x.tiles), tiles = (int)min((int64_t)(x.tiles - tile0), end - pos);

    // the rows of this thread's fragments: g and g + 8 of the tile
    const int64_t row0 = (int64_t)rt * kRows + g;
    const int64_t rows = (int64_t)x.lq * group;
    uint32_t qf[DP / 16][4];
    int limit[2];
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      const int64_t r = row0 + 8 * e;
      const bool live = r < rows;
      const int i = live ? (int)(r / group) : 0;
      const T* q = static_cast<const T*>(a.q) + (x.q0 + i) * a.q_row +
                   (int64_t)(m * group + (live ? (int)(r % group) : 0)) * a.q_head;
      limit[e] = !live ? 0 : a.causal ? max(0, min(x.lk, i + x.lk - x.lq + 1)) : x.lk;
#pragma unroll
      for (int k = 0; k < DP / 16; ++k)
#pragma unroll
        for (int f = 0; f < 2; ++f) {
          const int col = 16 * k + 8 * f + 2 * quad;
          qf[k][2 * f + e] = live && col < a.dim ? *reinterpret_cast<const uint32_t*>(q + col) : 0u;
        }
    }

    // A lane copies the same 16-byte column of every row of its parity class; its addresses move by whole tiles.
    constexpr int kRowsAtOnce = 32 / kChunks;  // rows of one instruction of the warp
    const int ch = lane % kChunks, r0 = lane / kChunks;
    const bool column = ch * 8 < a.dim;
    const int64_t first_key = (int64_t)tile0 * kKeys + slice * kWarpKeys + r0;
    const T* kp = static_cast<const T*>(a.k) + (x.k0 + first_key) * a.k_row + m * a.k_head + ch * 8;
    const T* vp = static_cast<const T*>(a.v) + (x.k0 + first_key) * a.v_row + m * a.v_head + ch * 8;
    int left = x.lk - (int)first_key;  // keys from this lane's first row on
    int to = 0;                        // stage to be filled
    auto load = [&](bool more) {
      if (more) {
        const uint32_t dst = mine_u + to * stage_bytes<DP>();
        // keys past the last read as zeros, never as what lies there
#pragma unroll
        for (int e = 0; e < kWarpKeys / kRowsAtOnce; ++e) {
          const int r = r0 + e * kRowsAtOnce;
          const bool there = column && e * kRowsAtOnce < left;
          const uint32_t off = (r * kChunks + (ch ^ (r & 7))) * 16;
          cp16(dst + off, there ? kp + (int64_t)e * kRowsAtOnce * a.k_row : a.k, there);
          cp16(dst + kWarpKeys * DP * 2 + off, there ? vp + (int64_t)e * kRowsAtOnce * a.v_row : a.v, there);
        }
        kp += kKeys * a.k_row;
        vp += kKeys * a.v_row;
        left -= kKeys;
        if (++to == kStages) to = 0;
      }
      asm volatile("cp.async.commit_group;" ::: "memory");
    };

    float o[DP / 8][4] = {};
    float top[2] = {-INFINITY, -INFINITY}, sum[2] = {0.f, 0.f};
#pragma unroll
    for (int t = 0; t < kStages - 1; ++t) load(t < tiles);
    int from = 0;  // stage to be read
    for (int t = tile0; t < tile0 + tiles; ++t) {
      __syncwarp();  // the stage to be filled has been read by all lanes
      load(t + kStages - 1 < tile0 + tiles);
      asm volatile("cp.async.wait_group %0;" ::"n"(kStages - 1) : "memory");
      __syncwarp();
      const uint32_t ks = mine_u + from * stage_bytes<DP>(), vs = ks + kWarpKeys * DP * 2;
      if (++from == kStages) from = 0;
      float sc[2][4] = {}, sd[2][4] = {};  // even and odd steps: half the chain of dependent products
#pragma unroll
      for (int k = 0; k < DP / 16; ++k) {
        // matrices: keys 0-7 and 8-15 (lane >> 4) by the two halves of 16 columns (lane >> 3 & 1)
        const int r = (lane & 7) + ((lane >> 4) << 3), ch = 2 * k + ((lane >> 3) & 1);
        uint32_t b[4];
        ldm4(ks + (r * kChunks + (ch ^ (r & 7))) * 16, b);
        mma<T>(k % 2 ? sd[0] : sc[0], qf[k], b[0], b[1]);
        mma<T>(k % 2 ? sd[1] : sc[1], qf[k], b[2], b[3]);
      }
#pragma unroll
      for (int n = 0; n < 2; ++n)
#pragma unroll
        for (int e = 0; e < 4; ++e) sc[n][e] += sd[n][e];
      const int key0 = t * kKeys + slice * kWarpKeys + 2 * quad;
      float now[2] = {-INFINITY, -INFINITY};
#pragma unroll
      for (int n = 0; n < 2; ++n)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          sc[n][e] = key0 + 8 * n + (e & 1) < limit[e >> 1] ? sc[n][e] * c : -INFINITY;
          now[e >> 1] = fmaxf(now[e >> 1], sc[n][e]);
        }
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        now[e] = fmaxf(now[e], __shfl_xor_sync(0xffffffffu, now[e], 1));
        now[e] = fmaxf(now[e], __shfl_xor_sync(0xffffffffu, now[e], 2)) - kBelow;
      }
      if (__any_sync(0xffffffffu, now[0] > top[0] || now[1] > top[1])) {
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          const float t2 = fmaxf(top[e], now[e]);
          const float keep = t2 == -INFINITY ? 1.f : exp2_approx(top[e] - t2);
          top[e] = t2;
          sum[e] *= keep;
#pragma unroll
          for (int n = 0; n < DP / 8; ++n) {
            o[n][2 * e] *= keep;
            o[n][2 * e + 1] *= keep;
          }
        }
      }
#pragma unroll
      for (int n = 0; n < 2; ++n)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const float off = top[e >> 1] == -INFINITY ? 0.f : top[e >> 1];
          sc[n][e] = exp2_approx(sc[n][e] - off);
          sum[e >> 1] += sc[n][e];
        }
      const uint32_t p[4] = {pack2<T>(sc[0][0], sc[0][1]), pack2<T>(sc[0][2], sc[0][3]), pack2<T>(sc[1][0], sc[1][1]),
                             pack2<T>(sc[1][2], sc[1][3])};
#pragma unroll
      for (int n = 0; n < DP / 16; ++n) {
        // transposed: keys 0-7 and 8-15 (lane >> 3 & 1) by two groups of 8 columns (lane >> 4)
        const int r = lane & 15, ch = 2 * n + (lane >> 4);
        uint32_t b[4];
        ldm4t(vs + (r * kChunks + (ch ^ (r & 7))) * 16, b);
        mma<T>(o[2 * n], p, b[0], b[1]);
        mma<T>(o[2 * n + 1], p, b[2], b[3]);
      }
    }
    asm volatile("cp.async.wait_group 0;" ::: "memory");
    __syncwarp();

    // the warps' shares meet in shared memory, each warp's in its own stages
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      sum[e] += __shfl_xor_sync(0xffffffffu, sum[e], 1);
      sum[e] += __shfl_xor_sync(0xffffffffu, sum[e], 2);
      if (quad == 0) {
        top_s[warp][g + 8 * e] = top[e];
        sum_s[warp][g + 8 * e] = sum[e];
      }
#pragma unroll
      for (int n = 0; n < DP / 8; ++n)
        *reinterpret_cast<float2*>(mine + ((g + 8 * e) * DP + 8 * n + 2 * quad) * 4) =
            make_float2(o[n][2 * e], o[n][2 * e + 1]);
    }
    __syncthreads();
#pragma unroll
    for (int hh = 0; hh < kHeads; ++hh) {
      constexpr int kShares = kWarps / kHeads;  // warps hh, hh + kHeads, ..
      const int r = threadIdx.x >> 3, col0 = (threadIdx.x & 7) * 4;
      const int64_t rr = (int64_t)rt * kRows + r;
      float all = -INFINITY, total_sum = 0.f, w[kShares];
#pragma unroll
      for (int i = 0; i < kShares; ++i) all = fmaxf(all, top_s[hh + i * kHeads][r]);
#pragma unroll
      for (int i = 0; i < kShares; ++i) {
        w[i] = all == -INFINITY ? 1.f : exp2_approx(top_s[hh + i * kHeads][r] - all);
        total_sum += w[i] * sum_s[hh + i * kHeads][r];
      }
      const bool whole = tiles == x.tiles;
      // a group that a cut goes through is the first of its block or its last, so that a block has two records at most
      if (BFB_BAD(whole || pos == begin || pos + tiles == end)) continue;
      float* rec = records + (((int64_t)2 * blockIdx.x + (pos == begin ? 0 : 1)) * kHeads + hh) * record_floats<DP>();
      const int h = (m0 + hh) * group + (int)(rr % group);
      const int64_t row = x.q0 + rr / group;
      const float inv = total_sum == 0.f ? 0.f : 1.f / total_sum;
#pragma unroll
      for (int col = col0; col < DP; col += 32) {
        float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
        for (int i = 0; i < kShares; ++i) {
          const float4 u = *reinterpret_cast<const float4*>(
              smem + (hh + i * kHeads) * kStages * stage_bytes<DP>() + (r * DP + col) * 4);
          v.x += w[i] * u.x;
          v.y += w[i] * u.y;
          v.z += w[i] * u.z;
          v.w += w[i] * u.w;
        }
        if (!whole) {
          *reinterpret_cast<float4*>(rec + r * DP + col) = v;
        } else if (rr < rows && col < a.dim && !BFB_BAD(row < a.total_q && h < a.heads)) {
          uint2 packed = make_uint2(0u, 0u);
          if (inv != 0.f) packed = make_uint2(pack2<T>(v.x * inv, v.y * inv), pack2<T>(v.z * inv, v.w * inv));
          *reinterpret_cast<uint2*>(static_cast<T*>(a.out) + (row * a.heads + h) * a.dim + col) = packed;
        }
      }
      if ((threadIdx.x & 7) == 0) {
        if (!whole) {
          rec[kRows * DP + r] = all;
          rec[kRows * DP + kRows + r] = total_sum;
        } else if (rr < rows) {
          a.lse[h * a.total_q + row] = total_sum == 0.f ? -INFINITY : (all + log2f(total_sum)) * kLn2;
        }
      }
    }
    __syncthreads();
    pos += tiles;
  }
}

// Joins the records of the groups that more than one block worked on, and
// writes the rows that no block did (of no sequence, or without keys).  One
// warp per (query row, head).  It finds its records while the first kernel is
// still running, and waits for that before it reads them; their maxima and
// sums are then read all at once, a lane each.
template <class T, int DP, int kHeads>
__global__ void __launch_bounds__(128) join_kernel(const __grid_constant__ Args a, const float* __restrict__ records,
                                                   int blocks) {
  const int64_t unit = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 5);
  if (unit >= a.total_q * a.heads) return;
  const int lane = threadIdx.x & 31, group = a.heads / a.kv_heads;
  const int64_t row = unit / a.heads;
  const int h = (int)(unit - row * a.heads), m = h / group;
  // the last sequence that starts at or before the row
  int lo = 0, hi = a.seqs;
  while (lo < hi) {
    const int mid = (lo + hi) >> 1;
    if (part_start(a.cu_q, a.seqs, a.total_q, mid + 2) <= row) lo = mid + 1; else hi = mid;
  }
  const int s = lo;
  Seq x = {};
  if (s < a.seqs) x = seq_at<kHeads>(a, s);
  const bool inside = s < a.seqs && row >= x.q0 && row < x.q0 + x.lq;
  constexpr int kPer = DP / 32;
  float o[kPer] = {}, all = -INFINITY, sum = 0.f;
  if (inside && x.tiles > 0) {
    int64_t total = 0, base = 0;
    for (int b = 0; b < a.seqs; b += 32) {
      const int64_t ends = line_ends<kHeads>(a, b, total);
      const int64_t prev = __shfl_up_sync(0xffffffffu, ends, 1);
      if (s >= b && s < b + 32) base = s > b ? __shfl_sync(0xffffffffu, prev, s - b) : total;
      total = __shfl_sync(0xffffffffu, ends, 31);
    }
    const int64_t per = stretch(total, blocks);
    const int64_t r = (row - x.q0) * group + h % group;
    const int64_t first = base + ((int64_t)(m / kHeads) * x.row_tiles + r / kRows) * x.tiles;
    const int64_t c0 = first / per, c1 = (first + x.tiles - 1) / per;
    asm volatile("griddepcontrol.wait;" ::: "memory");
    if (c0 == c1) return;  // written by its block
    if (BFB_BAD(c0 >= 0 && c1 < blocks)) return;
    for (int64_t c = c0; c <= c1; c += 32) {
      const int n = (int)min((int64_t)32, c1 + 1 - c);
      // at the end of a block's stretch where it began before the group, else at its start
      const int64_t mine = c + min(lane, n - 1);
      const float* rec = records + ((2 * mine + (mine * per < first ? 1 : 0)) * kHeads + m % kHeads) * record_floats<DP>();
      const float top = lane < n ? rec[kRows * DP + r % kRows] : -INFINITY;
      const float part = lane < n ? rec[kRows * DP + kRows + r % kRows] : 0.f;
      float t2 = top;
#pragma unroll
      for (int d = 16; d > 0; d >>= 1) t2 = fmaxf(t2, __shfl_xor_sync(0xffffffffu, t2, d));
      t2 = fmaxf(t2, all);
      const float keep = t2 == -INFINITY ? 1.f : exp2_approx(all - t2), w = t2 == -INFINITY ? 1.f : exp2_approx(top - t2);
      all = t2;
      float add = part * w;
#pragma unroll
      for (int d = 16; d > 0; d >>= 1) add += __shfl_xor_sync(0xffffffffu, add, d);
      sum = sum * keep + add;
#pragma unroll
      for (int i = 0; i < kPer; ++i) o[i] *= keep;
#pragma unroll 4
      for (int e = 0; e < n; ++e) {
        const float we = __shfl_sync(0xffffffffu, w, e);
        const int64_t which = c + e;
        const float* from = records + ((2 * which + (which * per < first ? 1 : 0)) * kHeads + m % kHeads) * record_floats<DP>() +
                            (r % kRows) * DP + lane * kPer;
        float v[kPer];
        if (kPer == 4) *reinterpret_cast<float4*>(v) = *reinterpret_cast<const float4*>(from);
        else *reinterpret_cast<float2*>(v) = *reinterpret_cast<const float2*>(from);
#pragma unroll
        for (int i = 0; i < kPer; ++i) o[i] += we * v[i];
      }
    }
  }
  // every block waits, so that this kernel cannot end, and the next one start, before the first has
  asm volatile("griddepcontrol.wait;" ::: "memory");
  const float inv = sum == 0.f ? 0.f : 1.f / sum;
#pragma unroll
  for (int i = 0; i < kPer; ++i) {
    const int col = lane * kPer + i;
    if (col < a.dim) static_cast<T*>(a.out)[unit * a.dim + col] = from_f32<T>(inv == 0.f ? 0.f : o[i] * inv);
  }
  if (lane == 0) a.lse[h * a.total_q + row] = sum == 0.f ? -INFINITY : (all + log2f(sum)) * kLn2;
}

template <class T, int DP, int kHeads>
int launch(const Args& a, float* records, cudaStream_t stream) {
  constexpr int kBytes = kWarps * kStages * stage_bytes<DP>();
  BFB_CUDA(cudaFuncSetAttribute(rows_kernel<T, DP, kHeads>, cudaFuncAttributeMaxDynamicSharedMemorySize, kBytes));
  const int64_t joins = ceil_div(a.total_q * a.heads, 4);
  if (joins > 0x7fffffff) return BFB_ERR_TOO_LARGE;
  cudaLaunchAttribute early = {};
  early.id = cudaLaunchAttributeProgrammaticStreamSerialization;
  early.val.programmaticStreamSerializationAllowed = 1;
  cudaLaunchConfig_t config = {};
  config.gridDim = dim3((unsigned)joins);
  config.blockDim = dim3(128);
  config.stream = stream;
  config.attrs = &early;
  if (a.total_k > 0 && a.seqs > 0) {
    rows_kernel<T, DP, kHeads><<<kRowsBlocks, kThreads, kBytes, stream>>>(a, records);
    BFB_CHECK_LAUNCH();
    config.numAttrs = 1;
  }
  BFB_CUDA(cudaLaunchKernelEx(&config, join_kernel<T, DP, kHeads>, a, (const float*)records, (int)kRowsBlocks));
  BFB_CHECK_LAUNCH();
  return BFB_OK;
}

template <class T, int DP>
int launch_heads(const Args& a, float* records, cudaStream_t stream) {
  if (a.kv_heads % 4 == 0) return launch<T, DP, 4>(a, records, stream);
  if (a.kv_heads % 2 == 0) return launch<T, DP, 2>(a, records, stream);
  return launch<T, DP, 1>(a, records, stream);
}

}  // namespace

size_t rows_record_floats(int dim) {
  return (size_t)2 * kRowsBlocks * kWarps * (dim <= 64 ? record_floats<64>() : record_floats<128>());
}

int forward_rows(const Args& a, int dtype, float* records, cudaStream_t stream) {
  if (dtype == BFB_F16)
    return a.dim <= 64 ? launch_heads<__half, 64>(a, records, stream) : launch_heads<__half, 128>(a, records, stream);
  return a.dim <= 64 ? launch_heads<__nv_bfloat16, 64>(a, records, stream)
                       : launch_heads<__nv_bfloat16, 128>(a, records, stream);
}

}  // namespace attn
}  // namespace bfb
