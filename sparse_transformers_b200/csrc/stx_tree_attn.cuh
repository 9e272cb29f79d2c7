// How stx_tree_attention's work is shared out (host and both kernels).
//
// A unit is (sequence, cache head, row tile): rows = tokens x query heads of the cache head, ROWS at most, token major.  Its
// keys are cut into tiles of KT slots.  All tiles of all units stand in one line, and each of G CTAs takes an equal stretch of it:
// the same number of tiles (off by one at most) whatever the lengths, which only the device knows.  A CTA's first and last unit may be shared with its neighbours; their partial sums (accumulator, maximum, sum
// of exponentials) go to slots 2 c and 2 c + 1 of the workspace and a second launch adds them in CTA order, so that the result does not depend on
// timing.  What lies between is finished by the CTA itself.
#pragma once

#include "stx_kv.cuh"

namespace stx {

constexpr int TREE_MAX_SEQ = 1024;

struct TreeArgs {
  const void* q;
  void* out;
  int64_t q_seq, q_tok, q_head, o_seq, o_tok, o_head;
  const int64_t *length, *counts, *masks;
  int64_t mask_stride;
  int64_t max_len;
  float scale_log2;  // scale * log2(e): soft-max in powers of two
  int n_seq, n_tok, nkv, group, hd;
  int tile_tok, row_tiles;  // tokens of a row tile, row tiles of a (sequence, cache head)
  int grid;                 // CTAs of the first launch, one or two an SM
  int sms;
  int cut, join, join_one;  // what splitting units costs, in tiles of this kernel (tree_line): a second segment in a CTA and the join, or the
                            // join alone; and the join of a single unit
  uint32_t copies;          // tiles of keys that a CTA of the tensor-core kernel requests at most
  float* part;              // [2 grid][hd / 4][ROWS][4], then [2 grid][2][ROWS]
};

struct TreeSeq {
  int len, cnt, keys;  // prefix, nodes, slots looked at
};
__device__ __forceinline__ TreeSeq tree_seq(const TreeArgs& a, int b) {
  TreeSeq s;
  s.len = static_cast<int>(min(static_cast<long long>(a.max_len), max(0ll, static_cast<long long>(a.length[b]))));
  s.cnt = a.counts ? static_cast<int>(min(static_cast<long long>(a.n_tok), max(0ll, static_cast<long long>(a.counts[b])))) : a.n_tok;
  s.keys = s.cnt > 0 ? s.len + min(s.cnt, static_cast<int>(a.max_len) - s.len) : 0;
  return s;
}
// A sequence without keys still has a tile: its rows are written (as zeros) by somebody.
__device__ __forceinline__ int tree_tiles(int keys, int kt) { return keys > 0 ? (keys + kt - 1) / kt : 1; }

constexpr int TREE_PRE = TREE_MAX_SEQ + 2;
// pre[b] = tiles of a row tile of one cache head, summed over the sequences before b; pre[n_seq] the sum; pre[n_seq + 1] is 1 where
// all have the same number.  By warp 0; the caller synchronises.  The host has made sure that the whole line has less than 2^31 tiles.
__device__ __forceinline__ void tree_prefix(const TreeArgs& a, int kt, int* pre) {
  if (threadIdx.x >= 32) return;
  int base = 0, most = 0, least = 0x7fffffff;
  for (int b0 = 0; b0 < a.n_seq; b0 += 32) {
    const int b = b0 + static_cast<int>(threadIdx.x);
    const int own = b < a.n_seq ? tree_tiles(tree_seq(a, b).keys, kt) : 0;
    int sum = own;
    if (b < a.n_seq) most = max(most, own), least = min(least, own);
#pragma unroll
    for (int off = 1; off < 32; off <<= 1) {
      const int o = __shfl_up_sync(0xffffffffu, sum, off);
      if (static_cast<int>(threadIdx.x) >= off) sum += o;
    }
    if (b < a.n_seq) pre[b] = base + sum - own;
    base += __shfl_sync(0xffffffffu, sum, 31);
  }
  most = __reduce_max_sync(0xffffffffu, most);
  least = __reduce_min_sync(0xffffffffu, least);
  if (threadIdx.x == 0) {
    pre[a.n_seq] = base;
    pre[a.n_seq + 1] = most == least;
  }
}

struct TreeLine {
  int total, ctas;  // W, G
  int each, more;   // W / G; the first W mod G CTAs have one tile more
  int per;          // units of a sequence
};
// Equal shares of two tiles or more, or a CTA for each unit.  Units of one length are better left whole where a share would end inside a unit and
// begin the next (two segments), or where the tiles saved take less than the join: nt tiles against those of a share, max(2, ceil(nt units / CTAs)),
// and the cost in tiles.  Where lengths differ, a CTA's stretch ends inside units either way, and shares are shorter.  (Comparisons only: divisions
// here took 1 us of both launches.)  us, whole units / shares of two, one sequence (in parentheses 16; 4 of 50 to 400 slots):
//   tiles                                     3             4             7             8
//   5 tokens x 24 heads on 8, 128 values
//     16-bit cache                       10.7 / 17.8   10.8 / 12.7   12.7 / 17.5   12.9 / 12.5   (16.4 / 25.2; 32.5 / 19.0)
//     int8 cache                         12.0 / 19.2   13.1 / 13.9   16.1 / 19.1   17.2 / 13.9   (19.0 / 27.7; 36.3 / 20.9)
//     fp32, general kernel               39.4 / 32.4   50.4 / 29.3   77.9 / 29.4   93.7 / 29.4   (134 / 133; 63.7 / 34.9)
//   the same of 3 heads on 1, int8       12.0 / 12.2   13.0 / 12.7   16.0 / 12.7   17.2 / 12.9   (17.9 / 14.5; 21.9 / 19.9)
//   the same of 256 values, 16-bit       17.4 / 27.6   18.6 / 17.9   22.2 / 27.7   23.4 / 18.1   (27.9 / 42.9; 57.8 / 32.2)
__device__ __forceinline__ TreeLine tree_line(const TreeArgs& a, const int* pre) {
  TreeLine l;
  l.per = a.nkv * a.row_tiles;
  l.total = pre[a.n_seq] * l.per;
  const int units = a.n_seq * l.per, nt = pre[1];
  l.ctas = max(1, min(a.grid, l.total >> 1));
  if (units < a.grid && nt < 4096 && pre[a.n_seq + 1] == 1) {
    const int cost = units == 1 ? a.join_one : (nt & 1) == 0 && l.total <= 2 * a.grid ? a.join : a.cut;
    const int share = a.grid > a.sms && l.total > 2 * a.sms ? 4 : 2;  // two CTAs an SM take twice as long
    if (nt <= share + cost || (nt - cost - 1) * a.sms < nt * units) l.ctas = units;
  }
  l.each = l.total / l.ctas;
  l.more = l.total - l.each * l.ctas;
  return l;
}
__device__ __forceinline__ int tree_begin(const TreeLine& l, int c) { return l.each * c + min(c, l.more); }
__device__ __forceinline__ int tree_owner(const TreeLine& l, int x) {
  const int cut = l.more * (l.each + 1);
  return x < cut ? x / (l.each + 1) : l.more + (x - cut) / l.each;
}

// The unit at position x of the line, and the part of [x, end) that lies in it.
struct TreeSeg {
  int b, head, rt;
  int t0, t1, nt;  // tiles of this segment, tiles of the unit
  int first;       // position of the unit's first tile
};
__device__ __forceinline__ TreeSeg tree_seg(const TreeArgs& a, const TreeLine& l, const int* pre, int x, int end) {
  int lo = 0, hi = a.n_seq - 1;
  while (lo < hi) {
    const int mid = (lo + hi + 1) >> 1;
    if (pre[mid] * l.per <= x) lo = mid;
    else hi = mid - 1;
  }
  TreeSeg s;
  s.b = lo;
  s.nt = pre[lo + 1] - pre[lo];
  const int in = x - pre[lo] * l.per, u = in / s.nt;
  s.t0 = in - u * s.nt;
  s.t1 = min(s.nt, s.t0 + end - x);
  s.first = x - s.t0;
  s.head = u / a.row_tiles;
  s.rt = u - s.head * a.row_tiles;
  return s;
}

// Bits of 32 slots from s0 on that a node sees: slots below len, nodes by `bits` (already cut to the nodes in use).
__device__ __forceinline__ uint32_t tree_visible(int s0, int len, unsigned long long bits) {
  const int rel = s0 - len;
  if (rel >= 64) return 0u;
  if (rel >= 0) return static_cast<uint32_t>(bits >> rel);
  if (rel <= -32) return 0xffffffffu;
  return static_cast<uint32_t>(bits << -rel) | ((1u << -rel) - 1u);
}
// Nodes that row token t sees (0 for a token that is not in use), without those behind the cache's end.
__device__ __forceinline__ unsigned long long tree_bits(const TreeArgs& a, const TreeSeq& s, int b, int t) {
  if (t >= s.cnt) return 0ull;
  const unsigned long long m = a.masks ? static_cast<unsigned long long>(a.masks[b * a.mask_stride + t]) : ~0ull >> (63 - t);
  const int nodes = s.keys - s.len;
  return nodes <= 0 ? 0ull : m & (~0ull >> (64 - nodes));
}

__host__ __device__ constexpr size_t tree_part_floats(int grid, int rows, int hd) {
  return static_cast<size_t>(2 * grid) * rows * (static_cast<size_t>((hd + 3) / 4) * 4 + 2);
}
__device__ __forceinline__ float* tree_part_o(const TreeArgs& a, int rows, int slot) {
  return a.part + static_cast<size_t>(slot) * rows * (((a.hd + 3) / 4) * 4);
}
__device__ __forceinline__ float* tree_part_ml(const TreeArgs& a, int rows, int slot) {
  return a.part + static_cast<size_t>(2 * a.grid) * rows * (((a.hd + 3) / 4) * 4) + static_cast<size_t>(slot) * 2 * rows;
}

// Adds the partial results of shared units; ROWS as in the first launch.
int launch_tree_join(const TreeArgs& a, int rows, int kt, int dtype, cudaStream_t s);

// The tensor-core kernel (stx_tree_attn_mma.cu): 16-bit models, caches that a tensor map can describe.
bool tree_mma_wanted(const stx_kv* cache);
int tree_mma(TreeArgs a, const stx_kv* cache, cudaStream_t s);
int tree_status(int* out, cudaStream_t s);

}  // namespace stx
