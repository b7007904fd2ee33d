// What the attention kernels share: the arguments of a call, the packed
// sequences' rows, tensor maps.
#pragma once

#include "sm100.cuh"

namespace bfb {
namespace attn {

struct Args {
  const void *q, *k, *v;
  int64_t q_row, q_head, k_row, k_head, v_row, v_head;
  int64_t total_q, total_k;
  int heads, kv_heads, dim, seqs;
  const int32_t *cu_q, *cu_k, *kv_lengths;
  int causal;
  float scale;
  void* out;
  float* lse;
  // backward
  const void* dout;
  const float* dlse;     // may be NULL
  float *lse2, *delta, *norm_g;  // workspace, [heads, total_q] each; norms of the rows of dout
  float* norm_v;                 // workspace, [kv_heads, total_k]; fp16 alone needs the norms
  void *dq, *dk, *dv;
};

constexpr int kTile = 128;  // rows of a tensor-core tile

// Tiles of `rows` rows over packed sequences: the rows before the first and
// after the last sequence count as two more, without keys, so that every row
// of a tensor belongs to exactly one tile.  No more than this many tiles.
inline int64_t tile_bound(int64_t total, int64_t seqs, int rows) { return total / rows + seqs + 2; }

// Start of part i: part 0 holds the rows before sequence 0, part s + 1
// sequence s, part seqs + 1 the rows behind the last.  Clamped to the tensor,
// so offsets that are wrong cannot reach outside it.
__device__ __forceinline__ int64_t part_start(const int32_t* cu, int seqs, int64_t total, int i) {
  if (i == 0) return 0;
  if (i > seqs + 1) return total;
  return cu ? min(max((int64_t)cu[i - 1], (int64_t)0), total) : 0;
}

// A tile of one part's queries (or keys), and the part's rows in both tensors.
struct Tile {
  int part;        // -1: no such tile
  int index, tiles;  // the tile within the part, and how many it has
  int64_t q0, k0;  // first rows
  int lq, lk;      // queries, keys
  int room;        // key rows, of which lk hold keys
};

// The rows of part `part`, in a Tile.
__device__ __forceinline__ Tile part_rows(const Args& a, int part) {
  Tile t = {};
  t.part = part;
  if (part >= a.seqs + 2) return t;
  const bool seq = part >= 1 && part <= a.seqs;  // all loads at once: one latency
  const int used = seq && a.kv_lengths ? a.kv_lengths[part - 1] : 0x7fffffff;
  t.q0 = part_start(a.cu_q, a.seqs, a.total_q, part);
  t.k0 = part_start(a.cu_k, a.seqs, a.total_k, part);
  const int64_t q1 = part_start(a.cu_q, a.seqs, a.total_q, part + 1);
  const int64_t k1 = part_start(a.cu_k, a.seqs, a.total_k, part + 1);
  t.lq = (int)max(q1 - t.q0, (int64_t)0);
  t.room = (int)max(k1 - t.k0, (int64_t)0);
  t.lk = seq ? min(max(used, 0), t.room) : 0;
  return t;
}

// The item-th tile of `rows` rows of the queries (or keys), found by one warp:
// all lanes take part and all get it.  Up to 30 sequences' tiles come heaviest
// first, whichever sequence they are in: causal, in the order of their distance
// from the light end of a sequence (its first queries, its last keys), otherwise
// in the order of the sequences' lengths in the other tensor (backward, causal
// prompts of 2.8, 1.6, 4.1 and 3.0 k, 16/4 heads of 128: dK and dV 285 -> 249 us;
// full, 0.3 to 2.5 k, 8 heads of 64, against an order that mixes them: dQ 71 -> 62,
// dK and dV 92 -> 82).  More come sequence by sequence, heavy end first.  An item
// past the last tile gets part -1, no rows.
template <bool kKeys>
__device__ __forceinline__ Tile find_tile(const Args& a, int rows, int64_t item) {
  const int lane = threadIdx.x & 31;
  int64_t before = 0;
  Tile mine;
  int src = -1, index = 0;
  for (int base = 0; base < a.seqs + 2; base += 32) {
    mine = part_rows(a, base + lane);
    mine.tiles = ((kKeys ? mine.room : mine.lq) + rows - 1) / rows;
    if (a.seqs + 2 <= 32) {
      if (item >= __reduce_add_sync(0xffffffffu, mine.tiles)) break;
      if (a.causal) {
        // least r with no more than `item` tiles at a distance of r or more (distances from 0)
        int lo = 0, hi = __reduce_max_sync(0xffffffffu, mine.tiles);
        while (lo < hi) {
          const int r = (lo + hi) >> 1;
          if (__reduce_add_sync(0xffffffffu, max(mine.tiles - r, 0)) <= (int)item) hi = r; else lo = r + 1;
        }
        // so the tile's distance is r - 1; among those of this distance in the order of the sequences
        const int nth = (int)item - __reduce_add_sync(0xffffffffu, max(mine.tiles - lo, 0));
        src = __fns(__ballot_sync(0xffffffffu, mine.tiles >= lo), 0, nth + 1);
        const int tiles = __shfl_sync(0xffffffffu, mine.tiles, src);
        index = kKeys ? tiles - lo : lo - 1;
      } else {
        const int work = kKeys ? mine.lq : mine.lk;
        int start = 0;  // tiles of the sequences with more work, or as much and further left
        for (int o = 0; o < 32; ++o) {
          const int w = __shfl_sync(0xffffffffu, work, o), n = __shfl_sync(0xffffffffu, mine.tiles, o);
          if (w > work || (w == work && o < lane)) start += n;
        }
        src = __ffs(__ballot_sync(0xffffffffu, item >= start && item < start + mine.tiles)) - 1;
        index = (int)item - __shfl_sync(0xffffffffu, start, src);
      }
      break;
    }
    int64_t upto = mine.tiles;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int64_t x = __shfl_up_sync(0xffffffffu, upto, o);
      if (lane >= o) upto += x;
    }
    const unsigned hit = __ballot_sync(0xffffffffu, item < before + upto);
    if (hit) {
      src = __ffs(hit) - 1;
      const int left = (int)(before + __shfl_sync(0xffffffffu, upto, src) - item);  // tiles from this one on
      const int tiles = __shfl_sync(0xffffffffu, mine.tiles, src);
      index = kKeys ? tiles - left : left - 1;
      break;
    }
    before += __shfl_sync(0xffffffffu, upto, 31);
  }
  Tile t = {};
  t.part = -1;
  if (src < 0) return t;
  t.part = __shfl_sync(0xffffffffu, mine.part, src);
  t.index = index;
  t.q0 = __shfl_sync(0xffffffffu, mine.q0, src);
  t.k0 = __shfl_sync(0xffffffffu, mine.k0, src);
  t.lq = __shfl_sync(0xffffffffu, mine.lq, src);
  t.lk = __shfl_sync(0xffffffffu, mine.lk, src);
  t.room = __shfl_sync(0xffffffffu, mine.room, src);
  // the rows of no sequence have nothing in the other tensor
  if (kKeys && (t.part < 1 || t.part > a.seqs)) t.lq = 0;
  return t;
}

// Tensor map of [rows, heads, dim] 16-bit values whose box is 128 rows of 64
// values of one head, in the 128-byte swizzle; values past dim and rows past
// the tensor read as zeros.
int make_map(CUtensorMap* map, const void* base, int dtype, int64_t rows, int heads, int dim, int64_t row_stride,
             int64_t head_stride);

int forward_sm100(const Args& a, int dtype, cudaStream_t stream);
int backward_sm100(const Args& a, int dtype, cudaStream_t stream);
// Few queries against long keys, split over the keys; `records`: its workspace.
constexpr int kRowsBlocks = 148 * 2;  // two blocks fit an SM
size_t rows_record_floats(int dim);
int forward_rows(const Args& a, int dtype, float* records, cudaStream_t stream);
int timeouts_forward(uint64_t* count, int reset);
int timeouts_backward(uint64_t* count, int reset);

}  // namespace attn
}  // namespace bfb
