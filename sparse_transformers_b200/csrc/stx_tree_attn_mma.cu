// stx_tree_attention on the 5th-generation tensor cores: fp16 and bf16 models, caches of 16 or 8 bits.
//
// A CTA per SM walks its segments (stx_tree_attn.cuh): up to 128 rows (tokens x query heads of a cache head) against tiles of KT = 64
// slots.  Per tile
//   S = Q K^T      tcgen05.mma, 128 x KT, both operands in shared memory (128-byte swizzle), S in tensor memory
//   P = 2^(S c - m)  soft-max warps; P goes back to tensor memory in the model's type: one rounding of a weight, half a step (the general kernel
//                  holds weights in fp32, so this one's error against 64 bits is about a third larger on long contexts: 2.25e-3 for 1.65e-3 in bf16).
//                  fp16: the base is 7 lower, so that P fills the type up to 2^15 and is subnormal only below 2^-21 of the largest weight, not 2^-14
//                  (a slot that draws e^12 times the weight of the others and holds zeros is common, and they are all that the result consists of)
//   O += P V       tcgen05.mma, P from tensor memory, V as it lies in the cache ([slots][head_dim] is an MN-major operand)
// With heads of up to 128 two streams of tiles (even and odd ones of the segment) with S, O, m and l of their own share the CTA:
// while one's soft-max runs, the other one's products do, and neither waits for the other before the segment's end, where
// O = sum 2^(m_i - M) O_i.  A stream has two S buffers, so that its next S is there before its P is done.  O is rescaled only where a row's
// maximum has grown by more than 2^8: weights up to 256 are as exact in a floating type as those up to 1 (a published refinement of the one-pass
// soft-max, as is the conversion of int8 codes by way of an exponent's last places below).
// P lies over the first half of the S that it was made from, so the S after next is issued when its P V has completed.
//
// Two forms.  REP = 1 (33 to 128 rows): two warps share a row's tile.  REP = 4 (up to 32 rows): the rows stand in all four lane groups, each of
// which takes a quarter of the slots, because 2^x of a warp's lanes costs the same however few of them are in use.
//
// What bounds it, at 8 cache heads of 128 values and 32768 slots, one sequence (both launches, one after the other, caches larger than the L2):
//   8 tokens x 32 heads, bf16   39.0 us.  A tile in steady state takes 0.6 us, which is HBM's rate (32 KB x 148 CTAs).  The other 22 us
//                               are fixed: start and Q 5, first tile 3, end of the segment 3, join 4, two launches.
//   64 tokens x 32 heads, bf16  66.1 us (520 TFLOP/s).  The soft-max: 0.9 us a tile, of which a third is 2^x at the MUFU pipe's rate; its
//                               phases follow one another in a warp, and four warps a scheduler do not fill the gaps.
//   8 tokens, int8 / e4m3       49 / 58 us (64 tokens 132 / 133): 1.2 us a tile for the conversion and the waits around it, where HBM would need 0.35.
// Tiles of 128 slots with one S buffer a stream took 149 us for the 64 tokens above (nothing to do for a stream between its P and its next S).
// Measured and not kept: streams that start half a tile apart and longer sleeps in the waits (no difference); converting warps for each stream
// and one warp for all scales (8 tokens, int8: 50 -> 54 us; warps without an instruction were then the most frequent stall, so the loops of the
// roles are kept short).
//
// 8-bit caches: TMA brings the codes, eight warps turn them into 16-bit operands (exactly: int8 and e4m3 codes are numbers of
// both 16-bit types), and the scales of the rows go where they cost nothing: x = S (k_scale c) + log2 v_scale in one fused multiply-add, so that
// P is the weight times v_scale, bounded by the same running maximum, and l = sum P / v_scale in another.  The maximum is of weight times scale, what a
// row adds to O at most.  A row of zeros (scale 0) adds nothing to O: it takes the stand-in TM_ZERO_SCALE, below every scale of a row that fp16 results
// can show (its largest value is 448 scales at most, and 2^-40 * 448 is under half of fp16's smallest number), so that it does not push the others'
// P down, and its weight still enters l.  (Limits, bf16 only: a weight's part of l underflows next to a scale 2^100 times its row's, 2^60 for a row of
// zeros, and l overflows where every scale is below 2^-110.)
//
// Warps: 4 HF NS soft-max (warp w reads the tensor memory lanes 32 (w mod 4) ..), two TMA producers, one that issues the products of each
// stream, and for 8-bit caches eight that convert.  Every wait is bounded; when one expires all roles stop waiting, the rows become NaN, copies
// and products on their way are waited for, tensor memory is freed, and stx_tree_attention_status reports it.
#include "stx_tma.cuh"
#include "stx_tree_attn.cuh"

#include <cuda.h>

#include <algorithm>
#include <cstdlib>

namespace stx {

constexpr int TM_ROWS = 128;
constexpr float TM_SLACK = 8.f;  // in powers of two
constexpr float TM_ZERO_SCALE = 9.094947017729282e-13f;  // 2^-40, exact in log2 and inverse
constexpr uint32_t TM_WAIT_LIMIT = 1u << 17;  // polls of up to 4 us: half a second

__device__ int tree_expired;  // DEV_TIMEOUT once a wait of a call on this device has expired

template <int STORE, int HD, int REP> struct TmShape {
  static constexpr bool CODED = STORE != STX_STORE_SAME;
  static constexpr int KT = 64;                     // slots of a tile
  static constexpr int NS = HD == 256 ? 1 : 2;      // streams: two O of 256 columns do not fit next to S
  static constexpr int NB = 2 * NS;                 // S buffers, two for each stream
  static constexpr int BOXES = HD / 64;             // 128-byte wide parts of an operand row
  static constexpr uint32_t BOX = KT * 128;         // bytes of such a part of a K or V tile
  static constexpr uint32_t TILE = BOXES * BOX;
  static constexpr uint32_t QBOX = TM_ROWS * 128, Q = BOXES * QBOX;
  // Tiles in shared memory (16-bit), in a ring for each stream: whoever waits for a slot then knows its ring's earlier phases to be over, and
  // a phase's parity is not taken for another's.  What an SM has to have on its way is 45 KB (0.3 KB/ns of HBM x 148 SMs at 1 us).
  static constexpr int DK = HD == 64 ? (CODED ? 3 : 4) : 2;
  static constexpr int DV = HD == 64 ? (CODED ? 2 : 4) : HD == 128 ? (CODED ? 2 : 3) : CODED ? 1 : 2;
  static constexpr int RAW = CODED ? (HD == 64 ? 6 : HD == 128 ? 3 : 1) : 0;  // tiles of codes of K, and as many of V
  static constexpr uint32_t RAW_TILE = KT * HD;
  // Tiles of a stream whose scales are kept: those of tile c are overwritten with K of tile c + SCALES, which waits for S of tile c + 2, formed
  // in the place of P of tile c.
  static constexpr int SCALES = DK + 2;
  static constexpr int ISSUERS = NS;                // warps that issue products, one for each stream
  static constexpr int HF = REP == 1 ? 2 : 1;       // threads that share a row's part of a tile
  static constexpr int SW = 4 * HF * NS;            // warps of the soft-max
  static constexpr int CONV = CODED ? 8 : 0;        // warps that convert, half of them K
  static constexpr int WARPS = SW + 2 + ISSUERS + CONV;
  static constexpr int THREADS = 32 * WARPS;
  static constexpr uint32_t O_COL = 256;
  static constexpr uint32_t QX = Q < 32768 ? 32768 : Q;  // Q, later the exchange of a segment's end
  static constexpr uint32_t SMEM_TILES = QX + NS * (DK + DV) * TILE + 2 * RAW * RAW_TILE;
  static constexpr uint32_t SMEM_SCALES = CODED ? NS * SCALES * 3 * KT * 4 : 0;
  static constexpr uint32_t SMEM_ML = 2 * HF * NS * TM_ROWS * 4;  // m of a tile, two in turn; at a segment's end its m and l
  static constexpr uint32_t BARS = 2 * NS * (DK + DV) + 2 * NB + 4 * NS + 4 * RAW + (CODED ? NS * SCALES : 0);
  static constexpr uint32_t SMEM = 1024 + SMEM_TILES + SMEM_SCALES + SMEM_ML + BARS * 8 + 64;
  static_assert(SMEM + 4 * (TREE_PRE + TM_ROWS) + 64 <= 227 * 1024, "shared memory of a CTA");
};

__device__ __forceinline__ bool tm_wait(uint64_t* bar, uint32_t parity, volatile int* dead) {
  for (uint32_t it = 0; it < TM_WAIT_LIMIT; ++it) {
    if (mbar_try_wait(bar, parity)) return true;
    if ((it & 63) == 63 && *dead) return false;
    if (it > 4096) __nanosleep(64);
  }
  *dead = 1;
  return false;
}
__device__ __forceinline__ void tm_arrive(uint64_t* bar) {
  asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(smem_u32(bar)) : "memory");
}
// One lane of a converged warp.  The roles that issue products and copies run as whole warps and only the issuing is left to this lane: in code
// that a branch on the lane number has split off, descriptors cannot be taken for uniform, and each product cost twice its time.
__device__ __forceinline__ bool tm_elect() {
  uint32_t one;
  asm volatile("{\n\t.reg .pred p;\n\telect.sync _|p, 0xffffffff;\n\tselp.u32 %0, 1, 0, p;\n\t}" : "=r"(one));
  return one != 0;
}
__device__ __forceinline__ void tm_commit(uint64_t* bar) {
  asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(smem_u32(bar)) : "memory");
}
__device__ __forceinline__ void tm_fence_before() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void tm_fence_after() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void tm_fence_async() { asm volatile("fence.proxy.async.shared::cta;" ::: "memory"); }

// 128-byte swizzle.  K-major: rows of 64 elements, groups of 8 rows 1024 bytes apart.  MN-major: [16 k][64 mn] boxes, groups of 8 k
// 1024 bytes apart, the next 64 mn `lbo` bytes further.
__device__ __forceinline__ uint64_t tm_desc(uint32_t addr, uint32_t lbo) {
  uint64_t d = 0;
  d |= static_cast<uint64_t>((addr & 0x3ffffu) >> 4);
  d |= static_cast<uint64_t>(lbo >> 4) << 16;
  d |= static_cast<uint64_t>(1024 >> 4) << 32;
  d |= static_cast<uint64_t>(1) << 46;  // descriptor version
  d |= static_cast<uint64_t>(2) << 61;  // SWIZZLE_128B
  return d;
}
__device__ __forceinline__ void tm_mma_ss(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, bool accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}" ::"r"(d),
      "l"(a), "l"(b), "r"(idesc), "r"(static_cast<uint32_t>(accumulate))
      : "memory");
}
__device__ __forceinline__ void tm_mma_ts(uint32_t d, uint32_t a, uint64_t b, uint32_t idesc, bool accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}" ::"r"(d),
      "r"(a), "l"(b), "r"(idesc), "r"(static_cast<uint32_t>(accumulate))
      : "memory");
}
// Columns of the warp's 32 lanes.  The wait is part of the statement: between the two the compiler could move registers that are not
// there yet (it does where it has to spill).
__device__ __forceinline__ void tm_ld(uint32_t taddr, uint32_t (&r)[16]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x16.b32 "
      "{%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15}, [%16];\n\t"
      "tcgen05.wait::ld.sync.aligned;"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]),
        "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
      : "r"(taddr)
      : "memory");
}
__device__ __forceinline__ void tm_ld(uint32_t taddr, uint32_t (&r)[32]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x32.b32 "
      "{%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, "
      "%16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31}, [%32];\n\t"
      "tcgen05.wait::ld.sync.aligned;"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]),
        "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]),
        "=r"(r[16]), "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]),
        "=r"(r[24]), "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
      : "r"(taddr)
      : "memory");
}
__device__ __forceinline__ void tm_st(uint32_t taddr, const uint32_t (&r)[8]) {
  asm volatile("tcgen05.st.sync.aligned.32x32b.x8.b32 [%8], {%0, %1, %2, %3, %4, %5, %6, %7};" ::"r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]),
               "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(taddr)
               : "memory");
}
__device__ __forceinline__ void tm_st(uint32_t taddr, const uint32_t (&r)[16]) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x16.b32 [%16], {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15};" ::"r"(r[0]),
      "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]), "r"(r[10]), "r"(r[11]), "r"(r[12]),
      "r"(r[13]), "r"(r[14]), "r"(r[15]), "r"(taddr)
      : "memory");
}
__device__ __forceinline__ void tm_st_wait() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }

__device__ __forceinline__ float tm_exp2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
template <typename T>
__device__ __forceinline__ uint32_t tm_pack(float lo, float hi) {
  uint32_t r;
  if constexpr (DT<T>::id == STX_F16) asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
  else asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
  return r;
}
// Exponent bits of the two 16-bit values of a word that are not finite, as a mask of whole values.
template <typename T>
__device__ __forceinline__ uint32_t tm_not_finite(uint32_t w) {
  constexpr uint32_t E = DT<T>::id == STX_F16 ? 0x7c00u : 0x7f80u;
  return ((w & E) == E ? 0x0000ffffu : 0u) | ((w >> 16 & E) == E ? 0xffff0000u : 0u);
}

// Eight 16-bit values, in one load where they are aligned.
template <typename T>
__device__ __forceinline__ uint4 tm_load8(const T* p, int vec) {
  if (vec) return ld_cached16(p);
  const unsigned short* u = reinterpret_cast<const unsigned short*>(p);
  return make_uint4(u[0] | static_cast<uint32_t>(u[1]) << 16, u[2] | static_cast<uint32_t>(u[3]) << 16, u[4] | static_cast<uint32_t>(u[5]) << 16,
                    u[6] | static_cast<uint32_t>(u[7]) << 16);
}

// N values of a row (N: 2, 4, 8 or 16), `left` of them inside the head.
template <typename T, int N>
__device__ __forceinline__ void tm_store(T* p, int vec, const float (&o)[N], int left) {
#pragma unroll
  for (int j = 0; j < N; j += 8) {
    if (j >= left) break;
    constexpr int M = N < 8 ? N : 8;
    uint32_t w[M / 2];
#pragma unroll
    for (int i = 0; i < M / 2; ++i) w[i] = tm_pack<T>(o[j + 2 * i], o[j + 2 * i + 1]);
    if (vec) {
      if constexpr (M == 8) st16(p + j, make_uint4(w[0], w[1], w[2], w[3]));
      else if constexpr (M == 4) *reinterpret_cast<uint2*>(p) = make_uint2(w[0], w[1]);
      else *reinterpret_cast<uint32_t*>(p) = w[0];
    } else {
      unsigned short* u = reinterpret_cast<unsigned short*>(p + j);
#pragma unroll
      for (int i = 0; i < M; ++i) u[i] = static_cast<unsigned short>(w[i / 2] >> (16 * (i & 1)));
    }
  }
}
// Adds the values of the nodes in `nodes` that are not finite (they were left out of the products) to n results that this thread has just
// written: a row's values (rows 1, p at column `col`), or fp32 values four columns apart by `rows` (p at column 0).
template <typename T, int STORE, typename P>
__device__ __noinline__ void tm_add_bad(P* p, int rows, unsigned long long nodes, KvPtr<typename Held<T, STORE>::C> vc, int b, int head, int len, int col, int n) {
  for (; nodes; nodes &= nodes - 1) {
    const auto* vr = vc.row(b, head, len + __ffsll(static_cast<long long>(nodes)) - 1) + col;
    for (int j = 0; j < n; ++j) {
      const float v = held_value<T, STORE>(vr[j], 1.f);
      P* at = rows == 1 ? p + j : p + static_cast<size_t>((col + j) / 4) * rows * 4 + (col + j) % 4;
      if (!isfinite(v)) *at = DT<P>::from_f(DT<P>::to_f(*at) + v);
    }
  }
}

// Two 16-bit operands from two codes.  int8: the byte is put under the exponent of a number whose last place is 1, and that number
// taken off again.  e4m3: the bits are moved to the 16-bit type's places, which scales every number, subnormal ones too, by the same power of two.
// w: four codes; h: 0 or 1, which pair.
template <typename T, int STORE>
__device__ __forceinline__ uint32_t tm_operand(uint32_t w, int h) {
  uint32_t r;
  if constexpr (STORE == STX_STORE_INT8) {
    const uint32_t pick = h ? 0x4342u : 0x4140u;  // bytes {code, constant, code, constant}
    if constexpr (DT<T>::id == STX_F16) {  // 1024 + 128 + x  -  1152
      const uint32_t u = __byte_perm(w ^ 0x80808080u, 0x64646464u, pick);
      asm("sub.rn.f16x2 %0, %1, %2;" : "=r"(r) : "r"(u), "r"(0x64806480u));
    } else {  // (128 + low seven bits) - (128 or, for negative x, 256)
      const uint32_t u = __byte_perm(w & 0x7f7f7f7fu, 0x43434343u, pick), v = __byte_perm(w & 0x80808080u, 0x43434343u, pick);
      asm("{\n\t.reg .b32 one;\n\tmov.b32 one, 0xbf80bf80;\n\tfma.rn.bf16x2 %0, %1, one, %2;\n\t}" : "=r"(r) : "r"(v), "r"(u));
    }
  } else {
    const uint32_t t = __byte_perm(w, 0u, h ? 0x3424u : 0x1404u);  // {0, b0, 0, b1}: a code in the high byte of each half
    if constexpr (DT<T>::id == STX_F16) {
      const uint32_t u = (t & 0x80008000u) | ((t >> 1) & 0x3f803f80u);
      asm("mul.rn.f16x2 %0, %1, %2;" : "=r"(r) : "r"(u), "r"(0x5c005c00u));  // 2^8
    } else {
      const uint32_t u = (t & 0x80008000u) | ((t >> 4) & 0x07f007f0u);
      asm("{\n\t.reg .b32 z;\n\tmov.b32 z, 0x80008000;\n\tfma.rn.bf16x2 %0, %1, %2, z;\n\t}" : "=r"(r) : "r"(u), "r"(0x7b807b80u));  // 2^120
    }
  }
  return r;
}
// Whether one of four e4m3 codes is NaN (0x7f or 0xff).
__device__ __forceinline__ bool tm_code_nan(uint32_t w) { return (((w & 0x7f7f7f7fu) + 0x01010101u) & 0x80808080u) != 0; }

// The tiles of a CTA, one after the other.
struct TmWalk {
  int x, end;
  TreeSeg sg;
  TreeSeq sq;
  int t;
  bool begun;
};
__device__ __forceinline__ bool tm_next_segment(const TreeArgs& a, const TreeLine& l, const int* pre, TmWalk& w) {
  if (w.begun) w.x += w.sg.t1 - w.sg.t0;
  w.begun = true;
  if (w.x >= w.end) return false;
  w.sg = tree_seg(a, l, pre, w.x, w.end);
  w.sq = tree_seq(a, w.sg.b);
  w.t = w.sg.t0;
  return true;
}

struct TmMaps {
  CUtensorMap k, v;
  int order;  // which coordinate (1, 2, 3) is the slot, the head and the sequence: two bits each
};
__device__ __forceinline__ void tm_load(void* dst, const CUtensorMap* m, int order, int c0, int slot, int head, int seq, uint64_t* bar) {
  const int ps = order & 3, ph = (order >> 2) & 3;
  const int c1 = ps == 1 ? slot : ph == 1 ? head : seq;
  const int c2 = ps == 2 ? slot : ph == 2 ? head : seq;
  const int c3 = ps == 3 ? slot : ph == 3 ? head : seq;
  asm volatile(
      "cp.async.bulk.tensor.4d.shared::cta.global.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4, %5, %6}], [%2];" ::"r"(smem_u32(dst)),
      "l"(m), "r"(smem_u32(bar)), "r"(c0), "r"(c1), "r"(c2), "r"(c3)
      : "memory");
}

// x of N slots from their S (16-bit caches: S itself), what the row does not see as -infinity, and the largest of them.  TAIL: there are
// slots that the row may not see; `cut` is 0 for rows that are not in use.  The two forms are apart so that the common one has no masks in it.
template <int STORE, int KT, bool TAIL, int N>
__device__ __forceinline__ float tm_row_max(uint32_t (&r)[N], const float* sc, int s0, int len, unsigned long long bits, uint32_t cut) {
  float mx[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
  const uint32_t v = TAIL ? tree_visible(s0, len, bits) & cut : ~0u;
#pragma unroll
  for (int j = 0; j < N; j += 4) {
    float x[4];
#pragma unroll
    for (int e = 0; e < 4; ++e) x[e] = __uint_as_float(r[j + e]);
    if constexpr (STORE != STX_STORE_SAME) {
      const float4 kk = *reinterpret_cast<const float4*>(sc + j), lv = *reinterpret_cast<const float4*>(sc + KT + j);
      x[0] = fmaf(x[0], kk.x, lv.x), x[1] = fmaf(x[1], kk.y, lv.y), x[2] = fmaf(x[2], kk.z, lv.z), x[3] = fmaf(x[3], kk.w, lv.w);
    }
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      if (TAIL) x[e] = (v >> (j + e)) & 1u ? x[e] : -INFINITY;
      mx[e] = fmaxf(mx[e], x[e]);
      r[j + e] = __float_as_uint(x[e]);
    }
  }
  return fmaxf(fmaxf(mx[0], mx[1]), fmaxf(mx[2], mx[3]));
}
// P = 2^(x - base), packed in pairs, to N / 2 columns from p_addr on; returns the sum of the weights.
template <typename T, int STORE, int KT, bool TAIL, int N>
__device__ __forceinline__ float tm_row_weights(const uint32_t (&r)[N], uint32_t p_addr, const float* sc, float c, float base) {
  float l[4] = {0.f, 0.f, 0.f, 0.f};
  uint32_t p16[N / 2];
  if constexpr (DT<T>::id == STX_F16) base -= 7.f;  // P up to 2^15 (TM_SLACK + 7); O and l carry the same factor
#pragma unroll
  for (int j = 0; j < N; j += 4) {
    float p[4], iv[4] = {1.f, 1.f, 1.f, 1.f};
    if constexpr (STORE != STX_STORE_SAME) {
      const float4 ii = *reinterpret_cast<const float4*>(sc + 2 * KT + j);
      iv[0] = ii.x, iv[1] = ii.y, iv[2] = ii.z, iv[3] = ii.w;
    }
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const float x = __uint_as_float(r[j + e]);
      p[e] = tm_exp2(STORE != STX_STORE_SAME ? x - base : fmaf(x, c, -base));
      if (TAIL && x == -INFINITY) p[e] = iv[e] = 0.f;  // not seen: c may be 0, 1 / v_scale infinite or NaN
      l[e] = STORE != STX_STORE_SAME ? fmaf(p[e], iv[e], l[e]) : l[e] + p[e];
    }
    p16[j / 2] = tm_pack<T>(p[0], p[1]);
    p16[j / 2 + 1] = tm_pack<T>(p[2], p[3]);
  }
  tm_st(p_addr, p16);
  return (l[0] + l[1]) + (l[2] + l[3]);
}
// Whether any of the 64 threads of two warps says so; also a barrier of theirs.
__device__ __forceinline__ bool tm_any64(int bar, bool mine) {
  int r;
  asm volatile(
      "{\n\t.reg .pred a, b;\n\tsetp.ne.s32 a, %1, 0;\n\tbarrier.cta.red.or.pred b, %2, 64, a;\n\tselp.s32 %0, 1, 0, b;\n\t}"
      : "=r"(r)
      : "r"(static_cast<int>(mine)), "r"(bar)
      : "memory");
  return r != 0;
}

template <typename T, int STORE, int HD, int REP>
__global__ void __launch_bounds__(TmShape<STORE, HD, REP>::THREADS, 1)
k_tree_attn_mma(const TreeArgs a, const __grid_constant__ TmMaps maps, const KvPtr<typename Held<T, STORE>::C> kc,
                const KvPtr<typename Held<T, STORE>::C> vc, int vec) {
  typedef TmShape<STORE, HD, REP> Z;
  constexpr int KT = Z::KT, NS = Z::NS, HF = Z::HF, NB = Z::NB, DK = Z::DK, DV = Z::DV;
  extern __shared__ unsigned char tm_raw[];
  __shared__ int pre[TREE_PRE];
  __shared__ unsigned long long bad_s;  // nodes of the segment with a value that is not finite
  __shared__ uint32_t tmem_s;
  __shared__ float inv_s[TM_ROWS];
  __shared__ int dead_s;
  unsigned char* smem = reinterpret_cast<unsigned char*>((reinterpret_cast<uintptr_t>(tm_raw) + 1023) & ~static_cast<uintptr_t>(1023));
  unsigned char* q_t = smem;
  unsigned char* k_t = q_t + Z::QX;
  unsigned char* v_t = k_t + NS * DK * Z::TILE;
  unsigned char* raw_t = v_t + NS * DV * Z::TILE;
  float* sc_s = reinterpret_cast<float*>(raw_t + 2 * Z::RAW * Z::RAW_TILE);  // [SCALES][3][KT]
  float* ml_s = sc_s + Z::SMEM_SCALES / 4;  // [2][HF NS][TM_ROWS]
  uint64_t* bars = reinterpret_cast<uint64_t*>(ml_s + Z::SMEM_ML / 4);
  uint64_t *k_full = bars, *k_empty = k_full + NS * DK, *v_full = k_empty + NS * DK, *v_empty = v_full + NS * DV, *s_full = v_empty + NS * DV;
  uint64_t *p_full = s_full + NB, *pv_done = p_full + NB, *o_full = pv_done + NS, *q_full = o_full + NS, *drain = q_full + NS, *raw_full = drain + NS;
  uint64_t *raw_empty = raw_full + 2 * Z::RAW, *sc_full = raw_empty + 2 * Z::RAW;  // K's, then V's
  volatile int* dead = &dead_s;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;

  if (tid == 0) {
    for (int i = 0; i < NS * DK; ++i) {
      mbar_init(&k_full[i], Z::CODED ? Z::CONV / 2 : 1);
      mbar_init(&k_empty[i], 1);
    }
    for (int i = 0; i < NS * DV; ++i) {
      mbar_init(&v_full[i], Z::CODED ? Z::CONV / 2 : 1);
      mbar_init(&v_empty[i], 1);
    }
    for (int i = 0; i < NB; ++i) {
      mbar_init(&s_full[i], 1);
      mbar_init(&p_full[i], 4 * HF);
    }
    for (int i = 0; i < NS; ++i) {
      mbar_init(&pv_done[i], 1);
      mbar_init(&o_full[i], 1);
      mbar_init(&drain[i], 1);
      mbar_init(&q_full[i], Z::SW);
    }
    for (int i = 0; i < 2 * Z::RAW; ++i) {
      mbar_init(&raw_full[i], 1);
      mbar_init(&raw_empty[i], Z::CONV / 2);
    }
    if (Z::CODED)
      for (int i = 0; i < NS * Z::SCALES; ++i) mbar_init(&sc_full[i], 2);
    dead_s = 0;
    bad_s = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  pdl_wait();
  pdl_launch_dependents();
  tree_prefix(a, KT, pre);
  __syncthreads();
  const TreeLine line = tree_line(a, pre);
  const int cta = blockIdx.x;
  if (cta >= line.ctas) return;
  if (warp == Z::SW + 2) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], 512;" ::"r"(smem_u32(&tmem_s)) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
  }
  tm_fence_before();
  __syncthreads();
  tm_fence_after();
  const uint32_t tmem = tmem_s;
  const int begin = tree_begin(line, cta);
  TmWalk w;
  w.x = begin;
  w.end = tree_begin(line, cta + 1);
  w.begun = false;
  uint32_t issued[2] = {0, 0};  // copies that a producer has requested, by ring

  if (warp < Z::SW) {
    // ------------------------------------------------------------------ softmax: a thread has a row's half of the tile
    // REP = 4 (up to 32 rows): the rows stand in all four lane groups, and each group takes a quarter of a tile's slots, with m, l and O of its
    // own that are added at the end: as the powers of a warp's lanes cost the same however few of them are in use, this is a quarter of the work.
    constexpr int RR = TM_ROWS / REP, CW = KT / REP / HF;  // rows; slots of a thread
    const int st = warp / (4 * HF), hf = (warp >> 2) % HF, lg = warp & 3, tl = lg * 32 + lane, who = HF * st + hf;
    const int row = tl % RR, rep = tl / RR, cs = rep * (KT / REP) + hf * CW;  // cs: the first slot of this thread
    const int pair_bar = 2 + 4 * st + lg;  // of two warps that share rows
    const uint32_t lane_base = tmem + (static_cast<uint32_t>(lg * 32) << 16);
    const uint32_t s_base = lane_base + st * 2 * KT, o_addr = lane_base + Z::O_COL + st * HD;
    const float c = fabsf(a.scale_log2);
    uint32_t uses[2] = {0, 0};  // of the stream's two S buffers
    uint32_t n_o = 0;           // segments in which the stream had a tile
    uint32_t n_x = 0;           // exchanges of maxima with the other warp
    while (tm_next_segment(a, line, pre, w)) {
      const TreeSeg& sg = w.sg;
      const TreeSeq& sq = w.sq;
      const int tok0 = sg.rt * a.tile_tok, rows = min(a.tile_tok, a.n_tok - tok0) * a.group;
      const int tok = tok0 + row / a.group, head = sg.head * a.group + row % a.group;
      const bool mine = row < rows;
      const bool used = mine && tok < sq.cnt;
      const unsigned long long bits = used ? tree_bits(a, sq, sg.b, tok) : 0ull;
      const uint32_t cut = used ? 0xffffffffu : 0u;
      const bool warp_used = __any_sync(0xffffffffu, used);
      const int nt = sg.t1 - sg.t0;
      // ---- Q: a row's threads bring its pieces
      {
        const T* src = static_cast<const T*>(a.q) + sg.b * a.q_seq + tok * a.q_tok + head * a.q_head;
        const uint32_t flip = a.scale_log2 < 0.f ? 0x80008000u : 0u;  // a negative scale goes with Q
        constexpr int MINE = HD / 8 / (HF * NS), BATCH = MINE < 8 ? MINE : 8;  // 16-byte pieces of a row, requested together
#pragma unroll 1
        for (int c0 = 0; c0 < MINE; c0 += BATCH) {
          uint4 v[BATCH];
#pragma unroll
          for (int i = 0; i < BATCH; ++i) {
            const int ch = (c0 + i) * HF * NS + who;
            v[i] = used && ch * 8 < a.hd ? tm_load8(src + ch * 8, vec) : make_uint4(0, 0, 0, 0);  // hd is a multiple of 8
          }
#pragma unroll
          for (int i = 0; i < BATCH; ++i) {
            const int ch = (c0 + i) * HF * NS + who;
            const uint4 f = make_uint4(v[i].x ^ flip, v[i].y ^ flip, v[i].z ^ flip, v[i].w ^ flip);
            *reinterpret_cast<uint4*>(q_t + (ch >> 3) * Z::QBOX + tl * 128 + (((ch & 7) ^ (tl & 7)) << 4)) = f;
          }
        }
        tm_fence_async();
        __syncwarp();
        if (lane == 0) {  // a stream without a tile is not told: its phases are those of segments that cannot end without it
          tm_arrive(&q_full[0]);
          if (NS == 2 && nt > 1) tm_arrive(&q_full[1]);
        }
      }
      float m = -INFINITY, l = 0.f;
      for (int i = st; i < nt; i += NS) {
        const int s0 = (sg.t0 + i) * KT, buf = (i / NS) & 1;
        const bool tail = s0 + KT > sq.len;
        const uint32_t n = uses[0] + uses[1];  // tiles of this stream before this one
        const uint32_t s_addr = s_base + buf * KT;
        const uint32_t ss = Z::CODED ? st * Z::SCALES + n % Z::SCALES : 0;
        const float* sc = sc_s + ss * 3 * KT + cs;
        const uint32_t use = buf ? uses[1]++ : uses[0]++;
        bool ok = tm_wait(&s_full[2 * st + buf], use & 1, dead);
        if (Z::CODED) ok = tm_wait(&sc_full[ss], (n / Z::SCALES) & 1, dead) && ok;
        if (tail) {
          // slots behind the keys become zeros, and what is not finite in a node's value: 0 * NaN must not reach a row that
          // does not see the node (those that do get it back at the end)
          if (DV < 2 && i >= NS) ok = tm_wait(&pv_done[st], (n - 1) & 1, dead) && ok;  // else the slot's phase before may still be open
          ok = tm_wait(&v_full[st * DV + n % DV], (n / DV) & 1, dead) && ok;
          const int r = tid & (KT - 1), part = (tid % (128 * HF)) / KT, slot = s0 + r;
          if (ok && slot >= sq.len) {
            unsigned char* vr = v_t + (st * DV + n % DV) * Z::TILE + r * 128;
            bool bad = false;
#pragma unroll 1
            for (int ch = part; ch < HD / 8; ch += 2 * HF) {
              uint4* at = reinterpret_cast<uint4*>(vr + (ch >> 3) * Z::BOX + (((ch + lane) & 7) << 4));
              if (slot >= sq.keys) {
                *at = make_uint4(0, 0, 0, 0);
              } else {
                uint4 v = *at;
                const uint32_t e0 = tm_not_finite<T>(v.x), e1 = tm_not_finite<T>(v.y), e2 = tm_not_finite<T>(v.z), e3 = tm_not_finite<T>(v.w);
                if (e0 | e1 | e2 | e3) {
                  bad = true;
                  v.x &= ~e0, v.y &= ~e1, v.z &= ~e2, v.w &= ~e3;
                  *at = v;
                }
              }
            }
            if (bad) atomicOr(&bad_s, 1ull << (slot - sq.len));
            tm_fence_async();
          }
        }
        ok = __all_sync(0xffffffffu, ok);
        if (warp_used) {  // both warps of the rows say the same here; what they do together depends on nothing that only one of them knows
          uint32_t r[CW];
          float mx = -INFINITY;
          if (ok) {
            tm_fence_after();
            tm_ld(s_addr + cs, r);
            mx = tail ? tm_row_max<STORE, KT, true>(r, sc, s0 + cs, sq.len, bits, cut) : tm_row_max<STORE, KT, false>(r, sc, s0 + cs, sq.len, bits, cut);
            if (!Z::CODED && mx != -INFINITY) mx *= c;
            tm_fence_before();
          }
          // P lies over the first half of S: two warps that share a row have read theirs now.
          if (HF == 2 ? tm_any64(pair_bar, mx > m + TM_SLACK) : __any_sync(0xffffffffu, mx > m + TM_SLACK)) {
            if (HF == 2) {
              float* mx_s = ml_s + (n_x++ & 1) * HF * NS * TM_ROWS;
              mx_s[who * TM_ROWS + tl] = mx;
              tm_any64(pair_bar, false);
              mx = fmaxf(mx, mx_s[(who ^ 1) * TM_ROWS + tl]);
            }
            const float up = mx > m + TM_SLACK ? mx : m;
            const float f = up == m ? 1.f : exp2f(m - up);
            m = up;
            l *= f;
            if (i >= NS) {  // O holds something: the stream's last product has to be in it
              // Phase by parity: the one before it is over since S of this tile was formed, the one behind it waits for this tile's P.
              ok = __all_sync(0xffffffffu, tm_wait(&pv_done[st], (n - 1) & 1, dead)) && ok;
              tm_fence_after();
#pragma unroll 1
              for (int c0 = hf * (HD / HF); c0 < (hf + 1) * (HD / HF); c0 += 16) {
                uint32_t o[16];
                tm_ld(o_addr + c0, o);
#pragma unroll
                for (int j = 0; j < 16; ++j) o[j] = __float_as_uint(__uint_as_float(o[j]) * f);
                tm_st(o_addr + c0, o);
              }
            }
          }
          if (ok) {
            tm_fence_after();
            const float base = m == -INFINITY ? 0.f : m;
            l += tail ? tm_row_weights<T, STORE, KT, true>(r, s_addr + cs / 2, sc, c, base) : tm_row_weights<T, STORE, KT, false>(r, s_addr + cs / 2, sc, c, base);
#pragma unroll
            for (int k = 1; k < REP; ++k) {  // the slots of the other lane groups weigh nothing here
              const uint32_t zero[CW / 2] = {};
              tm_st(s_addr + ((rep + k) % REP) * (KT / REP / 2) + hf * (CW / 2), zero);
            }
          }
          tm_st_wait();
          tm_fence_before();
        }
        __syncwarp();
        if (lane == 0) tm_arrive(&p_full[2 * st + buf]);
      }
      // ---- the segment's end
      const bool have = nt > st;
      bool ok = true;
      if (have) ok = tm_wait(&o_full[st], n_o++ & 1, dead);  // (pv_done may be one phase or two behind or ahead here: its parity says nothing)
      ok = __all_sync(0xffffffffu, ok);
      tm_fence_after();
      if (!used) {  // whatever a row that is not in use has gathered next to others
        m = -INFINITY;
        l = 0.f;
      }
      asm volatile("bar.sync 1, %0;" ::"n"(32 * Z::SW) : "memory");  // bad_s of all warps; every product of the segment is done, every maximum read
      ml_s[who * TM_ROWS + tl] = m;
      ml_s[(HF * NS + who) * TM_ROWS + tl] = l;
      tm_fence_before();
      asm volatile("bar.sync 1, %0;" ::"n"(32 * Z::SW) : "memory");
      tm_fence_after();
      // The row's results, NS streams x REP lane groups: M, each one's factor 2^(m - M), and the sum, in the same order everywhere.
      float big = -INFINITY, sum = 0.f, f[NS];
#pragma unroll
      for (int k = 0; k < NS * REP; ++k) big = fmaxf(big, ml_s[HF * (k / REP) * TM_ROWS + (k % REP) * RR + row]);
#pragma unroll
      for (int k = 0; k < NS * REP; ++k) {
        const int at = HF * (k / REP) * TM_ROWS + (k % REP) * RR + row;
        const float mk = ml_s[at];
        float lk = ml_s[HF * NS * TM_ROWS + at];
        if (HF == 2) lk += ml_s[(HF * NS + 1) * TM_ROWS + at];
        sum += lk * (mk == big ? 1.f : exp2f(mk - big));
      }
#pragma unroll
      for (int k = 0; k < NS; ++k) {
        const float mk = ml_s[HF * k * TM_ROWS + tl];
        f[k] = mk == big ? 1.f : exp2f(mk - big);
      }
      const bool gone = !ok || *dead;
      const bool whole = sg.t0 == 0 && sg.t1 == sg.nt;
      const int slot = 2 * cta + (w.x == begin ? 0 : 1);
      float* po = tree_part_o(a, TM_ROWS, slot);
      // 1 / l; 0 where nothing was seen (what weights of zero met does not count), NaN where a wait has expired
      const float inv_row = gone ? __int_as_float(0x7fc00000) : big == -INFINITY && sum == 0.f ? 0.f : whole ? 1.f / sum : 1.f;
      if (who == 0 && rep == 0) {
        inv_s[row] = inv_row;
        if (!whole) {
          float* ml = tree_part_ml(a, TM_ROWS, slot);
          ml[row] = big;
          ml[TM_ROWS + row] = gone ? inv_row : sum;  // NaN: a part of which nothing was seen would count as one that has nothing to see
        }
      }
      const unsigned long long bad = bad_s;
      const uint32_t o_row = lane_base + Z::O_COL;
      // N columns of the thread's row, added over the streams
      auto gather = [&](int col, auto& o) {
        constexpr int N = sizeof(o) / sizeof(float);
        if (warp_used) {
          uint32_t r[N];
          tm_ld(o_row + col, r);
#pragma unroll
          for (int k = 0; k < N; ++k) o[k] = used ? __uint_as_float(r[k]) * f[0] : 0.f;
          if (NS == 2 && nt > 1) {
            tm_ld(o_row + HD + col, r);
#pragma unroll
            for (int k = 0; k < N; ++k) o[k] += used ? __uint_as_float(r[k]) * f[NS - 1] : 0.f;
          }
        } else {
#pragma unroll
          for (int k = 0; k < N; ++k) o[k] = 0.f;
        }
        __syncwarp();
      };
      // and N finished ones to their place
      auto put = [&](int orow, int col, auto& o, float inv) {
        constexpr int N = sizeof(o) / sizeof(float);
        if (orow >= rows || col >= a.hd) return;  // hd is a multiple of 8
        const int otok = tok0 + orow / a.group;
#pragma unroll
        for (int k = 0; k < N; ++k) o[k] = inv == 0.f ? 0.f : o[k] * inv;
        if (whole) {
          T* dst = static_cast<T*>(a.out) + sg.b * a.o_seq + otok * a.o_tok + (sg.head * a.group + orow % a.group) * a.o_head + col;
          tm_store<T, N>(dst, vec, o, a.hd - col);
          if (bad) tm_add_bad<T, STORE>(dst, 1, bad & tree_bits(a, sq, sg.b, otok), vc, sg.b, sg.head, sq.len, col, min(N, a.hd - col));
        } else {
#pragma unroll
          for (int k = 0; k < N; k += 4)
            if (col + k < a.hd) *reinterpret_cast<float4*>(po + (static_cast<size_t>((col + k) / 4) * TM_ROWS + orow) * 4) = make_float4(o[k], o[k + 1], o[k + 2], o[k + 3]);
          if (bad) tm_add_bad<T, STORE>(po + static_cast<size_t>(orow) * 4, TM_ROWS, bad & tree_bits(a, sq, sg.b, otok), vc, sg.b, sg.head, sq.len, col, min(N, a.hd - col));
        }
      };
      if constexpr (REP == 1) {  // a row's threads have a part of its columns each
        constexpr int CS = HD / (HF * NS);
#pragma unroll 1
        for (int c0 = who * CS; c0 < (who + 1) * CS; c0 += 16) {
          float o[16];
          gather(c0, o);
          put(row, c0, o, inv_row);
          __syncwarp();
        }
      } else {
        // The lane groups' sums meet in shared memory, [lane group][column][row]: over Q, which no product reads any more, as many columns as
        // fit, or, behind the CTA's last segment, all of them over the tiles.  A warp takes eight columns of all rows at a time from there.
        constexpr int FIT = Z::QX / (TM_ROWS * 4) < HD ? Z::QX / (TM_ROWS * 4) : HD;
        constexpr bool WIDE = NS * (DK + DV) * Z::TILE >= TM_ROWS * HD * 4;
        const bool last = WIDE && w.x + nt >= w.end;
        const int cw = last ? HD : FIT;  // columns at a time
        float* xch = reinterpret_cast<float*>(last ? k_t : q_t);
#pragma unroll 1
        for (int c0 = 0; c0 < HD; c0 += cw) {
#pragma unroll 1
          for (int c1 = who * (cw / NS); c1 < (who + 1) * (cw / NS); c1 += 32) {
            float o[32];
            gather(c0 + c1, o);
            float* to = xch + (rep * cw + c1) * RR + row;
#pragma unroll
            for (int k = 0; k < 32; ++k) to[k * RR] = o[k];
          }
          asm volatile("bar.sync 1, %0;" ::"n"(32 * Z::SW) : "memory");
#pragma unroll 1
          for (int c1 = 8 * warp; c1 < cw; c1 += 8 * Z::SW) {
            float o[8];
#pragma unroll
            for (int k = 0; k < 8; ++k) {
              const float* from = xch + (c1 + k) * RR + lane;
              o[k] = (from[0] + from[cw * RR]) + (from[2 * cw * RR] + from[3 * cw * RR]);
            }
            put(lane, c0 + c1, o, inv_s[lane]);
            __syncwarp();
          }
          if (c0 + cw < HD) asm volatile("bar.sync 1, %0;" ::"n"(32 * Z::SW) : "memory");
        }
      }
      tm_fence_before();
      __syncwarp();
      asm volatile("bar.sync 1, %0;" ::"n"(32 * Z::SW) : "memory");  // Q, m, l and bad_s are free
      if (tid == 0) bad_s = 0;
    }
  } else if (warp < Z::SW + 2) {
    // ------------------------------------------------------------------ TMA producers: one for K, one for V (a warp issues a box in about 150 ns)
    const int half = warp - Z::SW;
    const CUtensorMap* map = half ? &maps.v : &maps.k;
    constexpr uint32_t BYTES = Z::CODED ? Z::RAW_TILE : Z::TILE;
    const uint32_t d = Z::CODED ? Z::RAW : half ? DV : DK;
    uint64_t* full = Z::CODED ? raw_full + half * Z::RAW : half ? v_full : k_full;
    uint64_t* empty = Z::CODED ? raw_empty + half * Z::RAW : half ? v_empty : k_empty;
    unsigned char* base = Z::CODED ? raw_t + half * Z::RAW * Z::RAW_TILE : half ? v_t : k_t;
    uint32_t n[2] = {0, 0};  // tiles of each ring so far (codes: one ring for both streams)
    bool ok = true;
    while (ok && tm_next_segment(a, line, pre, w)) {
      for (int t = w.sg.t0; t < w.sg.t1 && ok; ++t) {
        const uint32_t st = Z::CODED || NS == 1 ? 0 : (t - w.sg.t0) & 1;
        if (half == 0 && n[0] + n[1] == a.copies) ok = false;  // for tests: no more keys, and the waits for them run out
        if (!ok) break;
        const uint32_t m = st ? n[1]++ : n[0]++, use = m / d, s = st * d + m % d;
        if (use) ok = __all_sync(0xffffffffu, tm_wait(&empty[s], (use - 1) & 1, dead));
        if (!ok) break;
        if (tm_elect()) {
          mbar_expect_tx(&full[s], BYTES);
#pragma unroll
          for (int i = 0; i < (Z::CODED ? 1 : Z::BOXES); ++i)
            tm_load(base + s * BYTES + i * Z::BOX, map, maps.order, 64 * i, t * KT, w.sg.head, w.sg.b, &full[s]);
        }
        __syncwarp();
        issued[0] = n[0], issued[1] = n[1];
      }
    }
  } else if (warp < Z::SW + 2 + Z::ISSUERS) {
    // ------------------------------------------------------------------ a stream's products
    {
      constexpr uint32_t fmt = DT<T>::id == STX_BF16 ? 1u : 0u;
      constexpr uint32_t common = (1u << 4) | (fmt << 7) | (fmt << 10) | (static_cast<uint32_t>(TM_ROWS >> 4) << 24);
      constexpr uint32_t idesc_s = common | (static_cast<uint32_t>(KT >> 3) << 17);
      constexpr uint32_t idesc_o = common | (1u << 16) | (static_cast<uint32_t>(HD >> 3) << 17);  // V is MN-major
      const int st = warp - (Z::SW + 2);
      uint32_t segs = 0, taken[2] = {0, 0};  // segments with a tile of the stream; uses of the stream's two P buffers
      uint32_t ns = 0, np = 0;               // S and P V of the stream so far
      bool ok = true;
      const uint64_t dq = tm_desc(smem_u32(q_t), 16);
      auto issue_s = [&](int i) {
        const uint32_t s = st * DK + ns % DK, b = 2 * st + ((i / NS) & 1);
        if (!__all_sync(0xffffffffu, tm_wait(&k_full[s], (ns / DK) & 1, dead))) return false;
        ++ns;
        tm_fence_after();
        const uint64_t dk = tm_desc(smem_u32(k_t) + s * Z::TILE, 16);
        if (tm_elect()) {
#pragma unroll
          for (int k = 0; k < HD / 16; ++k)  // values behind head_dim are zeros.  (Skipped by a branch here, all steps came out with the first one's A.)
            tm_mma_ss(tmem + b * KT, dq + ((k >> 2) * Z::QBOX + (k & 3) * 32) / 16, dk + ((k >> 2) * Z::BOX + (k & 3) * 32) / 16, idesc_s, k != 0);
          tm_commit(&k_empty[s]);
          tm_commit(&s_full[b]);
        }
        __syncwarp();
        return true;
      };
      while (ok && tm_next_segment(a, line, pre, w)) {
        const int nt = w.sg.t1 - w.sg.t0;
        if (nt <= st) continue;
        ok = __all_sync(0xffffffffu, tm_wait(&q_full[st], segs & 1, dead));
        ++segs;
        tm_fence_after();
        for (int i = st; i < min(NB, nt) && ok; i += NS) ok = issue_s(i);
        for (int i = st; i < nt && ok; i += NS) {
          const uint32_t s = st * DV + np % DV, half = (i / NS) & 1, b = 2 * st + half;
          const uint32_t use = half ? taken[1]++ : taken[0]++;
          ok = tm_wait(&p_full[b], use & 1, dead) && tm_wait(&v_full[s], (np / DV) & 1, dead);
          ok = __all_sync(0xffffffffu, ok);
          if (!ok) break;
          tm_fence_after();
          const uint64_t dv = tm_desc(smem_u32(v_t) + s * Z::TILE, Z::BOX);
          if (tm_elect()) {
#pragma unroll
            for (int k = 0; k < KT / 16; ++k)
              tm_mma_ts(tmem + Z::O_COL + st * HD, tmem + b * KT + k * 8, dv + k * 2048 / 16, idesc_o, i >= NS || k != 0);
            tm_commit(&v_empty[s]);
            tm_commit(&pv_done[st]);
            if (i + NS >= nt) tm_commit(&o_full[st]);
          }
          __syncwarp();
          // the next S of this buffer goes over the P just taken; the soft-max works on the other buffer meanwhile
          if (i + NB < nt) ok = __all_sync(0xffffffffu, tm_wait(&pv_done[st], np & 1, dead)) && issue_s(i + NB);
          ++np;
        }
      }
    }
  } else if constexpr (Z::CODED) {
    // ------------------------------------------------------------------ codes become operands: half of the warps for K (and the scales), half for V
    constexpr int CT = 16 * Z::CONV;  // threads of a half
    const int half = (tid - 32 * (Z::SW + 2 + Z::ISSUERS)) / CT, ct = (tid - 32 * (Z::SW + 2 + Z::ISSUERS)) % CT;
    const uint32_t d = half ? DV : DK;
    uint64_t *full = half ? v_full : k_full, *empty = half ? v_empty : k_empty;
    uint64_t *r_full = raw_full + half * Z::RAW, *r_empty = raw_empty + half * Z::RAW;
    const unsigned char* raw = raw_t + half * Z::RAW * Z::RAW_TILE;
    unsigned char* tiles_t = half ? v_t : k_t;
    const float c = fabsf(a.scale_log2);
    uint32_t n[2] = {0, 0}, rs = 0, ruse = 0;  // tiles of each stream so far; place in the ring of codes
    bool ok = true;
    // the scales of a tile are requested a tile ahead
    TmWalk ahead = w;
    bool more = half == 0 && ct < KT && tm_next_segment(a, line, pre, ahead);
    float ks = 0.f, vs = 0.f;
    auto request = [&]() {
      ks = 0.f;
      vs = 1.f;
      if (!more) return;
      const int slot = ahead.t * KT + ct;
      if (slot < ahead.sq.keys) {
        ks = kc.srow(ahead.sg.b, ahead.sg.head)[slot];
        vs = vc.srow(ahead.sg.b, ahead.sg.head)[slot];
      }
      if (++ahead.t == ahead.sg.t1) more = tm_next_segment(a, line, pre, ahead);
    };
    request();
    while (ok && tm_next_segment(a, line, pre, w)) {
      for (int t = w.sg.t0; t < w.sg.t1 && ok; ++t) {
        const uint32_t st = NS == 1 ? 0 : (t - w.sg.t0) & 1;
        const uint32_t m = st ? n[1]++ : n[0]++, use = m / d, s = st * d + m % d;
        if (use) ok = tm_wait(&empty[s], (use - 1) & 1, dead);
        ok = ok && tm_wait(&r_full[rs], ruse & 1, dead);
        ok = __all_sync(0xffffffffu, ok);
        if (!ok) break;
        constexpr int PER = HD / 16, EACH = KT * PER / CT, BATCH = EACH < 2 ? EACH : 2;  // 16-byte pieces of a row of codes, of a thread
        const unsigned char* src = raw + rs * Z::RAW_TILE;
        unsigned char* dst = tiles_t + s * Z::TILE;
#pragma unroll 1
        for (int i0 = 0; i0 < EACH; i0 += BATCH) {
          uint4 w4[BATCH];
#pragma unroll
          for (int i = 0; i < BATCH; ++i) w4[i] = *reinterpret_cast<const uint4*>(src + (ct + CT * (i0 + i)) * 16);
#pragma unroll
          for (int i = 0; i < BATCH; ++i) {
            const int at = ct + CT * (i0 + i), r = at / PER, piece = at % PER;
            // Eight lanes store at a time, of a row's two parts that lie in the same banks: those of the second part their upper half first.
            const int up = (piece >> 2) & 1;
            const uint32_t q4[4] = {up ? w4[i].z : w4[i].x, up ? w4[i].w : w4[i].y, up ? w4[i].x : w4[i].z, up ? w4[i].y : w4[i].w};
            uint32_t e[8];
#pragma unroll
            for (int k = 0; k < 8; ++k) e[k] = tm_operand<T, STORE>(q4[k / 2], k & 1);
            if constexpr (STORE == STX_STORE_E4M3) {
              if (tm_code_nan(q4[0]) || tm_code_nan(q4[1]) || tm_code_nan(q4[2]) || tm_code_nan(q4[3])) {
#pragma unroll
                for (int k = 0; k < 16; ++k)
                  if (((q4[k / 4] >> (8 * (k % 4))) & 0x7fu) == 0x7fu) e[k / 2] |= k & 1 ? 0x7fff0000u : 0x00007fffu;
              }
            }
            unsigned char* to = dst + (piece >> 2) * Z::BOX + r * 128;
            const int ch = (piece & 3) * 2 + up;
            *reinterpret_cast<uint4*>(to + ((ch ^ (r & 7)) << 4)) = make_uint4(e[0], e[1], e[2], e[3]);
            *reinterpret_cast<uint4*>(to + ((ch ^ 1 ^ (r & 7)) << 4)) = make_uint4(e[4], e[5], e[6], e[7]);
          }
        }
        tm_fence_async();
        __syncwarp();
        if (lane == 0) {
          tm_arrive(&r_empty[rs]);
          tm_arrive(&full[s]);
        }
        if (half == 0 && ct < KT) {
          const float v = vs == 0.f ? TM_ZERO_SCALE : vs;
          const uint32_t ss = st * Z::SCALES + m % Z::SCALES;
          float* sc = sc_s + ss * 3 * KT;
          sc[ct] = ks * c;
          sc[KT + ct] = log2f(v);
          sc[2 * KT + ct] = 1.f / v;
          __syncwarp();
          if (lane == 0) tm_arrive(&sc_full[ss]);
          request();
        }
        if (++rs == Z::RAW) {
          rs = 0;
          ++ruse;
        }
      }
    }
  }
  __syncwarp();
  tm_fence_before();
  __syncthreads();
  if (*dead) {  // a wait has expired: no copy and no product may still be on its way when the CTA leaves
    if (tid == 0) atomicOr(&tree_expired, DEV_TIMEOUT);
    if (warp >= Z::SW && warp < Z::SW + 2) {
      const int half = warp - Z::SW;
      const uint32_t d = Z::CODED ? Z::RAW : half ? DV : DK;
      uint64_t* full = Z::CODED ? raw_full + half * Z::RAW : half ? v_full : k_full;
      for (uint32_t st = 0; st < 2; ++st)
        for (uint32_t i = 0; i < d; ++i)
          if (issued[st] > i) mbar_wait_bounded(&full[st * d + i], ((issued[st] - 1 - i) / d) & 1);
    } else if (warp >= Z::SW + 2 && warp < Z::SW + 2 + Z::ISSUERS) {
      const int st = warp - (Z::SW + 2);
      if (tm_elect()) tm_commit(&drain[st]);
      __syncwarp();
      mbar_wait_bounded(&drain[st], 0);
    }
    __syncthreads();
  }
  if (warp == Z::SW + 2) {
    tm_fence_after();
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, 512;" ::"r"(tmem) : "memory");
  }
}

// ---------------------------------------------------------------------------------- host
typedef CUresult (*PFN_tmEncode)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*, const cuuint64_t*, const cuuint32_t*,
                                 const cuuint32_t*, CUtensorMapInterleave, CUtensorMapSwizzle, CUtensorMapL2promotion, CUtensorMapFloatOOBfill);
static PFN_tmEncode tm_encode() {
  static PFN_tmEncode fn = nullptr;
  if (!fn) {
    void* p = nullptr;
    cudaDriverEntryPointQueryResult q;
    if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &p, cudaEnableDefault, &q) == cudaSuccess && q == cudaDriverEntryPointSuccess)
      fn = reinterpret_cast<PFN_tmEncode>(p);
  }
  return fn;
}

// The order of the cache's dimensions by stride, as a tensor map wants them: each stride a multiple of the one before it, and
// no dimension reaching into the next.  False where the cache has none (overlapping or unaligned strides).
struct TmOrder {
  cuuint64_t dims[4], strides[3];
  int pos[3];  // coordinate of slot, head, sequence
};
static bool tm_order(const stx_kv* c, TmOrder* o) {
  const int64_t es = static_cast<int64_t>(store_size(c->store, c->dtype));
  struct D {
    int64_t n, stride;
    int id;
  } d[3] = {{c->max_len, c->slot_stride * es, 0}, {c->n_kv_heads, c->head_stride * es, 1}, {c->n_seq, c->seq_stride * es, 2}};
  if ((reinterpret_cast<uintptr_t>(c->k) | reinterpret_cast<uintptr_t>(c->v)) & 15) return false;
  // a dimension of one has no stride of its own: it goes last, behind all others
  std::stable_sort(d, d + 3, [](const D& x, const D& y) { return (x.n > 1) != (y.n > 1) ? x.n > 1 : x.n > 1 && x.stride < y.stride; });
  int64_t reach = c->head_dim * es, step = 16;
  o->dims[0] = static_cast<cuuint64_t>(c->head_dim);
  for (int i = 0; i < 3; ++i) {
    int64_t s = d[i].stride;
    if (d[i].n <= 1) s = (reach + step - 1) / step * step;
    if (s % step || s < reach || s >= (1ll << 40) || d[i].n > (1ll << 62) / s) return false;
    o->dims[i + 1] = static_cast<cuuint64_t>(d[i].n);
    o->strides[i] = static_cast<cuuint64_t>(s);
    o->pos[d[i].id] = i + 1;
    reach = s * d[i].n;
    step = s;
  }
  return true;
}

static int tm_map(CUtensorMap* m, const void* base, const stx_kv* c, const TmOrder& o, int box_cols, int box_slots) {
  PFN_tmEncode enc = tm_encode();
  if (!enc) {
    set_error("stx_tree_attention: cuTensorMapEncodeTiled is not available from this driver");
    return STX_ERR_CUDA;
  }
  const bool coded = c->store != STX_STORE_SAME;
  cuuint32_t box[4] = {static_cast<cuuint32_t>(box_cols), 1, 1, 1};
  box[o.pos[0]] = static_cast<cuuint32_t>(box_slots);
  const cuuint32_t estr[4] = {1, 1, 1, 1};
  const CUresult r = enc(m, coded ? CU_TENSOR_MAP_DATA_TYPE_UINT8 : c->dtype == STX_BF16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16,
                         4, const_cast<void*>(base), o.dims, o.strides, box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE,
                         coded ? CU_TENSOR_MAP_SWIZZLE_NONE : CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                         CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  if (r != CUDA_SUCCESS) {
    set_error("stx_tree_attention: cuTensorMapEncodeTiled failed with %d", static_cast<int>(r));
    return STX_ERR_CUDA;
  }
  return STX_OK;
}

template <typename T, int STORE, int HD, int REP>
static int launch_mma(TreeArgs a, const stx_kv* cache, const TmOrder& o, int vec, cudaStream_t s) {
  typedef TmShape<STORE, HD, REP> Z;
  typedef typename Held<T, STORE>::C C;
  TmMaps maps;
  int rc = tm_map(&maps.k, cache->k, cache, o, Z::CODED ? HD : 64, Z::KT);
  if (rc == STX_OK) rc = tm_map(&maps.v, cache->v, cache, o, Z::CODED ? HD : 64, Z::KT);
  if (rc != STX_OK) return rc;
  maps.order = o.pos[0] | (o.pos[1] << 2) | (o.pos[2] << 4);
  static bool attr_set[64] = {};
  int dev = 0;
  STX_CUDA(cudaGetDevice(&dev));
  if (dev < 0 || dev >= 64 || !attr_set[dev]) {
    STX_CUDA(cudaFuncSetAttribute(k_tree_attn_mma<T, STORE, HD, REP>, cudaFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(Z::SMEM)));
    if (dev >= 0 && dev < 64) attr_set[dev] = true;
  }
  STX_CUDA(launch_pdl(k_tree_attn_mma<T, STORE, HD, REP>, dim3(static_cast<unsigned>(a.grid)), dim3(Z::THREADS), Z::SMEM, s, a, maps, kv_ptr<C>(cache, false),
                      kv_ptr<C>(cache, true), vec));
  return launch_tree_join(a, TM_ROWS, Z::KT, cache->dtype, s);
}

// False: the general kernel has to do it.  a.tile_tok and the like are set here.
bool tree_mma_wanted(const stx_kv* cache) {
  TmOrder o;
  return cache->dtype != STX_F32 && tm_order(cache, &o);
}
int tree_mma(TreeArgs a, const stx_kv* cache, cudaStream_t s) {
  TmOrder o;
  if (!tm_order(cache, &o)) return STX_ERR_UNSUPPORTED;
  a.tile_tok = std::min(a.n_tok, TM_ROWS / a.group);
  a.row_tiles = (a.n_tok + a.tile_tok - 1) / a.tile_tok;
  a.grid = a.sms = num_sms();
  a.copies = 0xffffffffu;
  if (const char* e = getenv("STX_TREE_COPIES")) a.copies = static_cast<uint32_t>(strtoul(e, nullptr, 10));
  auto ok = [](const void* p, int64_t x, int64_t y, int64_t z) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0 && x % 8 == 0 && y % 8 == 0 && z % 8 == 0; };
  const int vec = ok(a.q, a.q_seq, a.q_tok, a.q_head) && ok(a.out, a.o_seq, a.o_tok, a.o_head);
  const bool few = a.tile_tok * a.group <= TM_ROWS / 4;
  // For tree_line, in ns and from runs over 2 to 8 tiles: a tile, a second segment in a CTA, the join.
  const bool coded = cache->store != STX_STORE_SAME;
  const int tile = (a.hd <= 64 ? (coded ? 900 : 400) : a.hd <= 128 ? (coded ? 1100 : 500) : coded ? 1500 : 1200) + (few ? 0 : 200);
  const int cut = a.hd <= 64 ? 3500 : a.hd <= 128 ? 5000 : 9000;
  const int join = few ? (a.hd <= 64 ? 2200 : a.hd <= 128 ? 2600 : 2000) : a.hd <= 64 ? 4000 : a.hd <= 128 ? 4500 : 8500;
  a.cut = (cut + join) / tile;
  a.join = join / tile;
  a.join_one = join / (2 * tile);
  auto by_heads = [&](auto t, auto st) -> int {
    typedef decltype(t) T;
    constexpr int S = decltype(st)::value;
    if (a.hd <= 64) return few ? launch_mma<T, S, 64, 4>(a, cache, o, vec, s) : launch_mma<T, S, 64, 1>(a, cache, o, vec, s);
    if (a.hd <= 128) return few ? launch_mma<T, S, 128, 4>(a, cache, o, vec, s) : launch_mma<T, S, 128, 1>(a, cache, o, vec, s);
    return few ? launch_mma<T, S, 256, 4>(a, cache, o, vec, s) : launch_mma<T, S, 256, 1>(a, cache, o, vec, s);
  };
  return by_store(cache->store, [&](auto st) -> int { return cache->dtype == STX_F16 ? by_heads(__half(), st) : by_heads(__nv_bfloat16(), st); });
}

int tree_status(int* out, cudaStream_t s) {
  int v = 0;
  STX_CUDA(cudaMemcpyFromSymbolAsync(&v, tree_expired, sizeof(int), 0, cudaMemcpyDeviceToHost, s));
  STX_CUDA(cudaStreamSynchronize(s));
  *out = v & DEV_TIMEOUT ? STX_ERR_TIMEOUT : STX_OK;
  if (v) {
    v = 0;
    STX_CUDA(cudaMemcpyToSymbolAsync(tree_expired, &v, sizeof(int), 0, cudaMemcpyHostToDevice, s));
    STX_CUDA(cudaStreamSynchronize(s));
  }
  return STX_OK;
}

}  // namespace stx
