// stx_tree_attention on the 5th-generation tensor cores: fp16 and bf16 models, caches of 16 or 8 bits.
//
// A CTA per SM walks its segments (stx_tree_attn.cuh): up to 128 rows (tokens x query heads of a cache head) against tiles of KT
// slots.  Per tile
//   S = Q K^T      tcgen05.mma, 128 x KT, both operands in shared memory (128-byte swizzle), S in tensor memory
//   P = 2^(S c - m)  softmax warps: a thread has a row; P goes back to tensor memory in the model's type
//   O += P V       tcgen05.mma, P from tensor memory, V as it lies in the cache ([slots][head_dim] is an MN-major operand)
// With heads of up to 128 two streams of tiles (even and odd ones of the segment) with S, O, m and l of their own share the CTA:
// while one's soft-max runs, the other one's products do, and neither waits for the other before the segment's end, where
// O = sum 2^(m_i - M) O_i.  O is rescaled only where a row's maximum has grown by more than 2^8: weights up to 256 are as exact in
// a floating type as those up to 1.
// P overwrites the S that it was made from, so the next S of a stream is issued when its P V has completed.
//
// What bounds it: a tile of 16-bit keys and values of 128 heads' values is 64 KB, 1.45 us of an SM's share of 6.5 TB/s (2700 clocks); the products
// take 1024 clocks of the tensor pipe, the 16384 powers 1024 of the MUFU pipe.  So HBM up to 128 rows, all three
// alike at 256.
//
// 8-bit caches: TMA brings the codes, four warps turn them into 16-bit operands (exactly: int8 and e4m3 codes are numbers of
// both 16-bit types), and the scales of the rows go where they cost nothing: x = S (k_scale c) + log2 v_scale in one fused multiply-add, so that
// P is the weight times v_scale, bounded by the same running maximum, and l = sum P / v_scale in another.
//
// Warps: 4 NS softmax (warp w reads the tensor memory lanes 32 (w mod 4) ..), then the TMA producer, the MMA issuer, and for 8-bit caches
// four that convert.  Every wait is bounded; when one expires all roles stop waiting, the rows become NaN and tensor memory is freed.
#include "stx_tma.cuh"
#include "stx_tree_attn.cuh"

#include <cuda.h>

#include <algorithm>

namespace stx {

constexpr int TM_ROWS = 128;
constexpr float TM_SLACK = 8.f;  // in powers of two
constexpr uint32_t TM_WAIT_LIMIT = 1u << 21;

template <int STORE, int HD> struct TmShape {
  static constexpr bool CODED = STORE != STX_STORE_SAME;
  static constexpr int KT = HD == 256 ? 64 : 128;   // slots of a tile
  static constexpr int NS = HD == 256 ? 1 : 2;      // streams: two O of 256 columns do not fit next to S
  static constexpr int BOXES = HD / 64;             // 128-byte wide parts of an operand row
  static constexpr uint32_t BOX = KT * 128;         // bytes of such a part of a K or V tile
  static constexpr uint32_t TILE = BOXES * BOX;
  static constexpr uint32_t QBOX = TM_ROWS * 128, Q = BOXES * QBOX;
  // Tiles in shared memory (16-bit): what an SM has to have on its way is 45 KB (0.3 KB/ns of HBM x 148 SMs at 1 us); the rest of 227 KB
  // is Q, the codes and what belongs to the sequences.
  static constexpr int DK = HD == 64 ? 4 : CODED ? 2 : HD == 128 ? 3 : 2;
  static constexpr int DV = HD == 64 ? 4 : CODED && HD == 256 ? 1 : 2;
  static constexpr int RAW = CODED ? (HD == 64 ? 6 : 3) : 0;  // tiles of codes, K and V in turn
  static constexpr uint32_t RAW_TILE = KT * HD;
  // Tiles whose scales are kept: those of tile n are overwritten with K of tile n + SCALES, which waits for S of tile n + SCALES - DK,
  // which waited for the soft-max of tile n + SCALES - DK - NS.
  static constexpr int SCALES = DK + NS;
  static constexpr int WARPS = 4 * NS + 2 + (CODED ? 4 : 0);
  static constexpr int THREADS = 32 * WARPS;
  static constexpr uint32_t O_COL = 256, S_COLS = KT;
  static constexpr uint32_t SMEM_TILES = Q + DK * TILE + DV * TILE + RAW * RAW_TILE;
  static constexpr uint32_t SMEM_SCALES = CODED ? SCALES * 3 * KT * 4 : 0;
  static constexpr uint32_t BARS = 2 * DK + 2 * DV + 6 + 2 + 2 * RAW + SCALES;
  static constexpr uint32_t SMEM = 1024 + SMEM_TILES + SMEM_SCALES + 2 * 2 * TM_ROWS * 4 + BARS * 8 + 64;
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
// 32 columns of the warp's 32 lanes; the values are there after tm_ld_wait().
__device__ __forceinline__ void tm_ld32(uint32_t taddr, uint32_t (&r)[32]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x32.b32 "
      "{%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, "
      "%16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31}, [%32];"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]),
        "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]), "=r"(r[16]),
        "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]), "=r"(r[24]),
        "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
      : "r"(taddr)
      : "memory");
}
__device__ __forceinline__ void tm_ld_wait() { asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory"); }
__device__ __forceinline__ void tm_st16(uint32_t taddr, const uint32_t (&r)[16]) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x16.b32 [%16], {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15};" ::"r"(r[0]),
      "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]), "r"(r[10]), "r"(r[11]), "r"(r[12]),
      "r"(r[13]), "r"(r[14]), "r"(r[15]), "r"(taddr)
      : "memory");
}
__device__ __forceinline__ void tm_st32(uint32_t taddr, const uint32_t (&r)[32]) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x32.b32 [%32], "
      "{%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, "
      "%16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31};" ::"r"(r[0]),
      "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]), "r"(r[10]), "r"(r[11]), "r"(r[12]),
      "r"(r[13]), "r"(r[14]), "r"(r[15]), "r"(r[16]), "r"(r[17]), "r"(r[18]), "r"(r[19]), "r"(r[20]), "r"(r[21]), "r"(r[22]), "r"(r[23]),
      "r"(r[24]), "r"(r[25]), "r"(r[26]), "r"(r[27]), "r"(r[28]), "r"(r[29]), "r"(r[30]), "r"(r[31]), "r"(taddr)
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
  long long x, end;
  TreeSeg sg;
  TreeSeq sq;
  int t;
  bool begun;
};
__device__ __forceinline__ bool tm_next_segment(const TreeArgs& a, const TreeLine& l, const long long* pre, TmWalk& w) {
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

template <typename T, int STORE, int HD>
__global__ void __launch_bounds__(TmShape<STORE, HD>::THREADS, 1)
k_tree_attn_mma(const TreeArgs a, const __grid_constant__ TmMaps maps, const KvPtr<typename Held<T, STORE>::C> kc,
                const KvPtr<typename Held<T, STORE>::C> vc, int vec) {
  typedef TmShape<STORE, HD> Z;
  constexpr int KT = Z::KT, NS = Z::NS, DK = Z::DK, DV = Z::DV;
  extern __shared__ unsigned char tm_raw[];
  __shared__ long long pre[TREE_MAX_SEQ + 1];
  __shared__ unsigned long long bad_s;  // nodes of the segment with a value that is not finite
  __shared__ uint32_t tmem_s;
  __shared__ int dead_s;
  unsigned char* smem = reinterpret_cast<unsigned char*>((reinterpret_cast<uintptr_t>(tm_raw) + 1023) & ~static_cast<uintptr_t>(1023));
  unsigned char* q_t = smem;
  unsigned char* k_t = q_t + Z::Q;
  unsigned char* v_t = k_t + DK * Z::TILE;
  unsigned char* raw_t = v_t + DV * Z::TILE;
  float* sc_s = reinterpret_cast<float*>(raw_t + Z::RAW * Z::RAW_TILE);  // [SCALES][3][KT]
  float* ml_s = sc_s + Z::SMEM_SCALES / 4;                               // [2][2][TM_ROWS]
  uint64_t* bars = reinterpret_cast<uint64_t*>(ml_s + 2 * 2 * TM_ROWS);
  uint64_t *k_full = bars, *k_empty = k_full + DK, *v_full = k_empty + DK, *v_empty = v_full + DV, *s_full = v_empty + DV;
  uint64_t *p_full = s_full + 2, *o_full = p_full + 2, *q_full = o_full + 2, *drain = q_full + 1, *raw_full = drain + 1;
  uint64_t *raw_empty = raw_full + Z::RAW, *sc_full = raw_empty + Z::RAW;
  volatile int* dead = &dead_s;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;

  if (tid == 0) {
    for (int i = 0; i < DK; ++i) {
      mbar_init(&k_full[i], Z::CODED ? 4 : 1);
      mbar_init(&k_empty[i], 1);
    }
    for (int i = 0; i < DV; ++i) {
      mbar_init(&v_full[i], Z::CODED ? 4 : 1);
      mbar_init(&v_empty[i], 1);
    }
    for (int i = 0; i < 2; ++i) {
      mbar_init(&s_full[i], 1);
      mbar_init(&p_full[i], 4);
      mbar_init(&o_full[i], 1);
    }
    mbar_init(q_full, 4 * NS);
    mbar_init(drain, 1);
    for (int i = 0; i < Z::RAW; ++i) {
      mbar_init(&raw_full[i], 1);
      mbar_init(&raw_empty[i], 4);
    }
    for (int i = 0; i < Z::SCALES; ++i) mbar_init(&sc_full[i], 4);
    dead_s = 0;
    bad_s = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  pdl_wait();
  pdl_launch_dependents();
  tree_prefix(a, KT, pre);
  __syncthreads();
  const TreeLine line = tree_line(a, pre);
  const long long cta = blockIdx.x;
  if (cta >= line.ctas) return;
  if (warp == 4 * NS + 1) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], 512;" ::"r"(smem_u32(&tmem_s)) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
  }
  tm_fence_before();
  __syncthreads();
  tm_fence_after();
  const uint32_t tmem = tmem_s;
  const long long begin = tree_begin(line, cta);
  TmWalk w;
  w.x = begin;
  w.end = tree_begin(line, cta + 1);
  w.begun = false;

  if (warp < 4 * NS) {
    // ------------------------------------------------------------------ softmax: a thread has a row
    const int st = warp >> 2, lg = warp & 3, row = lg * 32 + lane;
    const uint32_t lane_base = tmem + (static_cast<uint32_t>(lg * 32) << 16);
    const uint32_t s_addr = lane_base + st * Z::S_COLS, o_addr = lane_base + Z::O_COL + st * HD;
    const float c = fabsf(a.scale_log2);
    uint32_t n_s = 0, n_o = 0;  // tiles and segments of this stream so far
    uint32_t tiles = 0;         // tiles of the CTA before this segment
    while (tm_next_segment(a, line, pre, w)) {
      const TreeSeg& sg = w.sg;
      const TreeSeq& sq = w.sq;
      const int tok0 = sg.rt * a.tile_tok, rows = min(a.tile_tok, a.n_tok - tok0) * a.group;
      const int tok = tok0 + row / a.group, head = sg.head * a.group + row % a.group;
      const bool mine = row < rows;
      const bool used = mine && tok < sq.cnt;
      const unsigned long long bits = used ? tree_bits(a, sq, sg.b, tok) : 0ull;
      const bool warp_used = __any_sync(0xffffffffu, used);
      // ---- Q: each of the NS warps of a lane group brings a part of the rows' boxes
      {
        const T* src = static_cast<const T*>(a.q) + sg.b * a.q_seq + tok * a.q_tok + head * a.q_head;
        const uint32_t flip = a.scale_log2 < 0.f ? 0x80008000u : 0u;  // a negative scale goes with Q
        for (int ch = st; ch < HD / 8; ch += NS) {
          uint4 v = make_uint4(0, 0, 0, 0);
          if (used && ch * 8 < a.hd) {  // hd is a multiple of 8
            if (vec) {
              v = ld_cached16(src + ch * 8);
            } else {
              T e[8];
#pragma unroll
              for (int i = 0; i < 8; ++i) e[i] = src[ch * 8 + i];
              v = *reinterpret_cast<const uint4*>(e);
            }
            v.x ^= flip, v.y ^= flip, v.z ^= flip, v.w ^= flip;
          }
          *reinterpret_cast<uint4*>(q_t + (ch >> 3) * Z::QBOX + row * 128 + (((ch & 7) ^ (row & 7)) << 4)) = v;
        }
        tm_fence_async();
        __syncwarp();
        if (lane == 0) tm_arrive(q_full);
      }
      float m = -INFINITY, l = 0.f;
      const int nt = sg.t1 - sg.t0;
      for (int i = st; i < nt; i += NS) {
        const int s0 = (sg.t0 + i) * KT;
        const bool tail = s0 + KT > sq.len;
        const uint32_t n = tiles + i;
        const float* sc = sc_s + (Z::CODED ? (n % Z::SCALES) * 3 * KT : 0);
        bool ok = tm_wait(&s_full[st], n_s & 1, dead);
        if (Z::CODED) ok = tm_wait(&sc_full[n % Z::SCALES], (n / Z::SCALES) & 1, dead) && ok;
        if (tail) {
          // slots behind the keys become zeros, and what is not finite in a node's value: 0 * NaN must not reach a row that
          // does not see the node (those that do get it back at the end)
          ok = tm_wait(&v_full[n % DV], (n / DV) & 1, dead) && ok;
          const int r = tid & 127, slot = s0 + r;
          if (ok && r < KT && slot >= sq.len) {
            unsigned char* vr = v_t + (n % DV) * Z::TILE + r * 128;
            bool bad = false;
#pragma unroll 1
            for (int ch = 0; ch < HD / 8; ++ch) {
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
        ++n_s;
        if (ok && warp_used) {
          tm_fence_after();
          // ---- the row's largest x of this tile
          float mx = -INFINITY;
#pragma unroll
          for (int c0 = 0; c0 < KT; c0 += 64) {
            uint32_t r0[32], r1[32];
            tm_ld32(s_addr + c0, r0);
            tm_ld32(s_addr + c0 + 32, r1);
            tm_ld_wait();
            const uint32_t v0 = !tail ? 0xffffffffu : used ? tree_visible(s0 + c0, sq.len, bits) : 0u;
            const uint32_t v1 = !tail ? 0xffffffffu : used ? tree_visible(s0 + c0 + 32, sq.len, bits) : 0u;
            if constexpr (Z::CODED) {
#pragma unroll
              for (int j = 0; j < 64; j += 4) {
                const float4 kk = *reinterpret_cast<const float4*>(sc + c0 + j), lv = *reinterpret_cast<const float4*>(sc + KT + c0 + j);
                const float kx[4] = {kk.x, kk.y, kk.z, kk.w}, lx[4] = {lv.x, lv.y, lv.z, lv.w};
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                  const int jj = j + e;
                  const float s = __uint_as_float(jj < 32 ? r0[jj & 31] : r1[jj & 31]);
                  const float x = fmaf(s, kx[e], lx[e]);
                  if (!tail || (((jj < 32 ? v0 : v1) >> (jj & 31)) & 1u)) mx = fmaxf(mx, x);
                }
              }
            } else {
#pragma unroll
              for (int j = 0; j < 32; ++j) {
                if (!tail || ((v0 >> j) & 1u)) mx = fmaxf(mx, __uint_as_float(r0[j]));
                if (!tail || ((v1 >> j) & 1u)) mx = fmaxf(mx, __uint_as_float(r1[j]));
              }
            }
          }
          if (!Z::CODED && mx != -INFINITY) mx *= c;
          if (__any_sync(0xffffffffu, mx > m + TM_SLACK)) {
            const float up = mx > m + TM_SLACK ? mx : m;
            const float f = up == m ? 1.f : exp2f(m - up);
            m = up;
            l *= f;
            if (i >= NS) {  // O holds something; this stream's products have completed
#pragma unroll 1
              for (int c0 = 0; c0 < HD; c0 += 32) {
                uint32_t r[32];
                tm_ld32(o_addr + c0, r);
                tm_ld_wait();
#pragma unroll
                for (int j = 0; j < 32; ++j) r[j] = __float_as_uint(__uint_as_float(r[j]) * f);
                tm_st32(o_addr + c0, r);
              }
            }
          }
          // ---- P and its sum
          const float base = m == -INFINITY ? 0.f : m;
          float l0 = 0.f, l1 = 0.f;
#pragma unroll
          for (int c0 = 0; c0 < KT; c0 += 64) {
            uint32_t r0[32], r1[32];
            tm_ld32(s_addr + c0, r0);
            tm_ld32(s_addr + c0 + 32, r1);
            tm_ld_wait();
            const uint32_t v0 = !tail ? 0xffffffffu : used ? tree_visible(s0 + c0, sq.len, bits) : 0u;
            const uint32_t v1 = !tail ? 0xffffffffu : used ? tree_visible(s0 + c0 + 32, sq.len, bits) : 0u;
#pragma unroll
            for (int h = 0; h < 2; ++h) {
              uint32_t p16[16];
#pragma unroll
              for (int j = 0; j < 32; j += 4) {
                float p[4];
                if constexpr (Z::CODED) {
                  const int at = c0 + 32 * h + j;
                  const float4 kk = *reinterpret_cast<const float4*>(sc + at), lv = *reinterpret_cast<const float4*>(sc + KT + at),
                               iv = *reinterpret_cast<const float4*>(sc + 2 * KT + at);
                  const float kx[4] = {kk.x, kk.y, kk.z, kk.w}, lx[4] = {lv.x, lv.y, lv.z, lv.w}, ix[4] = {iv.x, iv.y, iv.z, iv.w};
#pragma unroll
                  for (int e = 0; e < 4; ++e) {
                    const float s = __uint_as_float(h ? r1[j + e] : r0[j + e]);
                    p[e] = tm_exp2(fmaf(s, kx[e], lx[e]) - base);
                    if (tail && !(((h ? v1 : v0) >> (j + e)) & 1u)) p[e] = 0.f;
                    if (tail && p[e] == 0.f) continue;  // 1 / v_scale may be infinite where it is not seen
                    (e & 1 ? l1 : l0) = fmaf(p[e], ix[e], e & 1 ? l1 : l0);
                  }
                } else {
#pragma unroll
                  for (int e = 0; e < 4; ++e) {
                    p[e] = tm_exp2(fmaf(__uint_as_float(h ? r1[j + e] : r0[j + e]), c, -base));
                    if (tail && !(((h ? v1 : v0) >> (j + e)) & 1u)) p[e] = 0.f;
                    (e & 1 ? l1 : l0) += p[e];
                  }
                }
                p16[j / 2] = tm_pack<T>(p[0], p[1]);
                p16[j / 2 + 1] = tm_pack<T>(p[2], p[3]);
              }
              tm_st16(s_addr + (c0 + 32 * h) / 2, p16);
            }
          }
          l += l0 + l1;
          tm_st_wait();
          tm_fence_before();
        }
        __syncwarp();
        if (lane == 0) tm_arrive(&p_full[st]);
      }
      // ---- the segment's end
      const bool have = nt > st;
      bool ok = true;
      if (have) {
        ok = tm_wait(&o_full[st], n_o & 1, dead);
        ++n_o;
      }
      ok = __all_sync(0xffffffffu, ok);
      tm_fence_after();
      if (!used) {  // whatever a row that is not in use has gathered next to others
        m = -INFINITY;
        l = 0.f;
      }
      float f = 1.f, big = m;
      if (NS == 2) {
        ml_s[st * 2 * TM_ROWS + row] = m;
        ml_s[(st * 2 + 1) * TM_ROWS + row] = l;
      }
      asm volatile("bar.sync 1, %0;" ::"n"(128 * NS) : "memory");  // m, l and bad_s of all warps; every product of the segment is done
      if (NS == 2) {
        const float mo = ml_s[(st ^ 1) * 2 * TM_ROWS + row], lo = ml_s[((st ^ 1) * 2 + 1) * TM_ROWS + row];
        big = fmaxf(m, mo);
        f = m == big ? 1.f : exp2f(m - big);
        const float fo = mo == big ? 1.f : exp2f(mo - big);
        l = l * f + lo * fo;
      }
      const bool gone = !ok || *dead;
      const bool both = NS == 2 && nt > 1;
      const bool whole = sg.t0 == 0 && sg.t1 == sg.nt;
      const long long slot = 2 * cta + (w.x == begin ? 0 : 1);
      float* po = tree_part_o(a, TM_ROWS, slot);
      float* xch = reinterpret_cast<float*>(q_t);  // [columns][rows]: no product reads Q any more
      const unsigned long long bad = bad_s & bits;
      T* dst = static_cast<T*>(a.out) + sg.b * a.o_seq + tok * a.o_tok + head * a.o_head;
      const float inv = big == -INFINITY && l == 0.f ? 0.f : 1.f / l;
      constexpr int HALF = HD / 2;
#pragma unroll 1
      for (int part = 0; part < 2; ++part) {
        if (both && st == 1) {
#pragma unroll 1
          for (int c0 = 0; c0 < HALF; c0 += 32) {
            uint32_t r[32];
            tm_ld32(o_addr + part * HALF + c0, r);
            tm_ld_wait();
#pragma unroll
            for (int j = 0; j < 32; ++j) xch[(c0 + j) * TM_ROWS + row] = __uint_as_float(r[j]) * f;
          }
        }
        if (both) asm volatile("bar.sync 1, %0;" ::"n"(128 * NS) : "memory");
        if (st == 0 && warp_used) {
#pragma unroll 1
          for (int c0 = 0; c0 < HALF; c0 += 32) {
            const int col = part * HALF + c0;
            uint32_t r[32];
            tm_ld32(o_addr + col, r);
            tm_ld_wait();
            float o[32];
#pragma unroll
            for (int j = 0; j < 32; ++j) {
              o[j] = __uint_as_float(r[j]) * f;
              if (both) o[j] += xch[(c0 + j) * TM_ROWS + row];
              if (big == -INFINITY && l == 0.f) o[j] = 0.f;  // nothing seen: what the weights of zero met does not count
            }
            if (bad) {  // values that are not finite, for the rows that see them
              for (unsigned long long left = bad; left; left &= left - 1) {
                const int node = __ffsll(static_cast<long long>(left)) - 1;
                const auto* vr = vc.row(sg.b, sg.head, sq.len + node);
#pragma unroll 1
                for (int j = 0; j < 32; ++j)
                  if (col + j < a.hd) {
                    const float v = held_value<T, STORE>(vr[col + j], 1.f);
                    if (!isfinite(v)) {
#pragma unroll
                      for (int k = 0; k < 32; ++k)
                        if (k == j) o[k] += v;
                    }
                  }
              }
            }
            if (gone) {
#pragma unroll
              for (int j = 0; j < 32; ++j) o[j] = __int_as_float(0x7fc00000);
            }
            if (whole) {
              if (mine) {
#pragma unroll
                for (int j = 0; j < 32; j += 8) {
                  if (col + j < a.hd) {
                    uint4 v;
                    v.x = tm_pack<T>(o[j] * inv, o[j + 1] * inv), v.y = tm_pack<T>(o[j + 2] * inv, o[j + 3] * inv);
                    v.z = tm_pack<T>(o[j + 4] * inv, o[j + 5] * inv), v.w = tm_pack<T>(o[j + 6] * inv, o[j + 7] * inv);
                    if (vec) {
                      st16(dst + col + j, v);
                    } else {
                      const T* e = reinterpret_cast<const T*>(&v);
#pragma unroll
                      for (int k = 0; k < 8; ++k) dst[col + j + k] = e[k];
                    }
                  }
                }
              }
            } else {
#pragma unroll
              for (int j = 0; j < 32; j += 4)
                if (col + j < a.hd)
                  *reinterpret_cast<float4*>(po + (static_cast<size_t>((col + j) / 4) * TM_ROWS + row) * 4) = make_float4(o[j], o[j + 1], o[j + 2], o[j + 3]);
            }
            __syncwarp();
          }
        } else if (st == 0 && whole && mine) {  // a warp of rows that are not in use: zeros
          for (int j = part * HALF; j < min(a.hd, (part + 1) * HALF); ++j) dst[j] = DT<T>::from_f(0.f);
        }
        __syncwarp();
        if (both) asm volatile("bar.sync 1, %0;" ::"n"(128 * NS) : "memory");
      }
      if (st == 0 && !whole) {
        float* ml = tree_part_ml(a, TM_ROWS, slot);
        ml[row] = big;
        ml[TM_ROWS + row] = l;
      }
      tm_fence_before();
      __syncwarp();
      asm volatile("bar.sync 1, %0;" ::"n"(128 * NS) : "memory");  // Q and bad_s are free
      if (tid == 0) bad_s = 0;
      tiles += nt;
    }
  } else if (warp == 4 * NS) {
    // ------------------------------------------------------------------ TMA producer
    if (lane == 0) {
      uint32_t nk = 0;  // 16-bit: tiles; codes: K and V tiles in turn
      bool ok = true;
      while (ok && tm_next_segment(a, line, pre, w)) {
        for (int t = w.sg.t0; t < w.sg.t1 && ok; ++t) {
          const int s0 = t * KT;
          if constexpr (!Z::CODED) {
            for (int half = 0; half < 2 && ok; ++half) {
              const uint32_t d = half ? DV : DK, s = nk % d, use = nk / d;
              uint64_t *full = half ? &v_full[s] : &k_full[s], *empty = half ? &v_empty[s] : &k_empty[s];
              if (use) ok = tm_wait(empty, (use - 1) & 1, dead);
              if (!ok) break;
              mbar_expect_tx(full, Z::TILE);
              unsigned char* dst = (half ? v_t : k_t) + s * Z::TILE;
#pragma unroll
              for (int i = 0; i < Z::BOXES; ++i)
                tm_load(dst + i * Z::BOX, half ? &maps.v : &maps.k, maps.order, 64 * i, s0, w.sg.head, w.sg.b, full);
            }
            if (ok) ++nk;
          } else {
            for (int half = 0; half < 2 && ok; ++half) {
              const uint32_t s = nk % Z::RAW, use = nk / Z::RAW;
              if (use) ok = tm_wait(&raw_empty[s], (use - 1) & 1, dead);
              if (!ok) break;
              mbar_expect_tx(&raw_full[s], Z::RAW_TILE);
              tm_load(raw_t + s * Z::RAW_TILE, half ? &maps.v : &maps.k, maps.order, 0, s0, w.sg.head, w.sg.b, &raw_full[s]);
              ++nk;
            }
          }
        }
      }
      if (*dead) {  // no copy may still be on its way when the CTA leaves
        if constexpr (!Z::CODED) {
          for (uint32_t s = 0; s < DK; ++s)
            if (nk > s) mbar_wait_bounded(&k_full[s], ((nk - 1 - s) / DK) & 1);
          for (uint32_t s = 0; s < DV; ++s)
            if (nk > s) mbar_wait_bounded(&v_full[s], ((nk - 1 - s) / DV) & 1);
        } else {
          for (uint32_t s = 0; s < Z::RAW; ++s)
            if (nk > s) mbar_wait_bounded(&raw_full[s], ((nk - 1 - s) / Z::RAW) & 1);
        }
      }
    }
  } else if (warp == 4 * NS + 1) {
    // ------------------------------------------------------------------ MMA issuer
    if (lane == 0) {
      constexpr uint32_t fmt = DT<T>::id == STX_BF16 ? 1u : 0u;
      constexpr uint32_t common = (1u << 4) | (fmt << 7) | (fmt << 10) | (static_cast<uint32_t>(TM_ROWS >> 4) << 24);
      constexpr uint32_t idesc_s = common | (static_cast<uint32_t>(KT >> 3) << 17);
      constexpr uint32_t idesc_o = common | (1u << 16) | (static_cast<uint32_t>(HD >> 3) << 17);  // V is MN-major
      const int ksteps = (a.hd + 15) / 16;  // values of a head behind hd are zeros
      uint32_t segs = 0, np[2] = {0, 0};
      uint32_t tiles = 0;
      bool ok = true;
      auto issue_s = [&](int i) {
        const uint32_t n = tiles + i;
        const int s = static_cast<int>(n % DK), st = i % NS;
        if (!tm_wait(&k_full[s], (n / DK) & 1, dead)) return false;
        tm_fence_after();
        for (int k = 0; k < ksteps; ++k) {
          const uint32_t qa = smem_u32(q_t) + (k >> 2) * Z::QBOX + (k & 3) * 32, ka = smem_u32(k_t) + s * Z::TILE + (k >> 2) * Z::BOX + (k & 3) * 32;
          tm_mma_ss(tmem + st * Z::S_COLS, tm_desc(qa, 16), tm_desc(ka, 16), idesc_s, k != 0);
        }
        tm_commit(&k_empty[s]);
        tm_commit(&s_full[st]);
        return true;
      };
      while (ok && tm_next_segment(a, line, pre, w)) {
        const int nt = w.sg.t1 - w.sg.t0;
        ok = tm_wait(q_full, segs & 1, dead);
        ++segs;
        tm_fence_after();
        for (int i = 0; i < min(NS, nt) && ok; ++i) ok = issue_s(i);
        for (int i = 0; i < nt && ok; ++i) {
          const uint32_t n = tiles + i;
          const int s = static_cast<int>(n % DV), st = i % NS;
          ok = tm_wait(&p_full[st], np[st] & 1, dead) && tm_wait(&v_full[s], (n / DV) & 1, dead);
          if (!ok) break;
          ++np[st];
          tm_fence_after();
          const uint32_t va = smem_u32(v_t) + s * Z::TILE;
#pragma unroll
          for (int k = 0; k < KT / 16; ++k)
            tm_mma_ts(tmem + Z::O_COL + st * HD, tmem + st * Z::S_COLS + k * 8, tm_desc(va + k * 2048, Z::BOX), idesc_o, i >= NS || k != 0);
          tm_commit(&v_empty[s]);
          if (i + NS >= nt) tm_commit(&o_full[st]);
          if (i + NS < nt) {
            ok = tm_wait(&v_empty[s], (n / DV) & 1, dead);  // P is read: S may overwrite it
            if (ok) ok = issue_s(i + NS);
          }
        }
        tiles += nt;
      }
      if (*dead) {  // no product may still be running when tensor memory is freed
        tm_commit(drain);
        mbar_wait_bounded(drain, 0);
      }
    }
  } else if constexpr (Z::CODED) {
    // ------------------------------------------------------------------ codes become operands
    const int ct = tid - 32 * (4 * NS + 2);  // 0 .. 127
    const float c = fabsf(a.scale_log2);
    uint32_t nr = 0;  // K and V tiles in turn
    uint32_t n = 0;
    bool ok = true;
    // the scales of a tile are requested a tile ahead
    TmWalk ahead = w;
    bool more = tm_next_segment(a, line, pre, ahead);
    float ks = 0.f, vs = 0.f;
    auto request = [&]() {
      ks = 0.f;
      vs = 1.f;
      if (!more) return;
      const int slot = ahead.t * KT + ct;
      if (ct < KT && slot < ahead.sq.keys) {
        ks = kc.srow(ahead.sg.b, ahead.sg.head)[slot];
        vs = vc.srow(ahead.sg.b, ahead.sg.head)[slot];
      }
      if (++ahead.t == ahead.sg.t1) more = tm_next_segment(a, line, pre, ahead);
    };
    request();
    while (ok && tm_next_segment(a, line, pre, w)) {
      for (int t = w.sg.t0; t < w.sg.t1 && ok; ++t, ++n) {
        const float ks0 = ks, vs0 = vs == 0.f ? 1.f : vs;  // a row of zeros: any scale
        request();
#pragma unroll 1
        for (int half = 0; half < 2 && ok; ++half, ++nr) {
          const uint32_t rs = nr % Z::RAW;
          const uint32_t d = half ? DV : DK, s = n % d;
          const uint32_t use = n / d;
          if (use) ok = tm_wait(half ? &v_empty[s] : &k_empty[s], (use - 1) & 1, dead);
          ok = ok && tm_wait(&raw_full[rs], (nr / Z::RAW) & 1, dead);
          ok = __all_sync(0xffffffffu, ok);
          if (!ok) break;
          if (half == 0) {
            float* sc = sc_s + (n % Z::SCALES) * 3 * KT;
            if (ct < KT) {
              sc[ct] = ks0 * c;
              sc[KT + ct] = log2f(vs0);
              sc[2 * KT + ct] = 1.f / vs0;
            }
            __syncwarp();
            if (lane == 0) tm_arrive(&sc_full[n % Z::SCALES]);
          }
          const unsigned char* src = raw_t + rs * Z::RAW_TILE;
          unsigned char* dst = (half ? v_t : k_t) + s * Z::TILE;
          constexpr int PER = HD / 16;  // 16-byte pieces of a row of codes
#pragma unroll 4
          for (int i = ct; i < KT * PER; i += 128) {
            const int r = i / PER, piece = i % PER;
            const uint4 raw = *reinterpret_cast<const uint4*>(src + i * 16);
            const uint32_t q4[4] = {raw.x, raw.y, raw.z, raw.w};
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
            unsigned char* at = dst + (piece >> 2) * Z::BOX + r * 128;
            const int ch = (piece & 3) * 2;
            *reinterpret_cast<uint4*>(at + ((ch ^ (r & 7)) << 4)) = make_uint4(e[0], e[1], e[2], e[3]);
            *reinterpret_cast<uint4*>(at + (((ch + 1) ^ (r & 7)) << 4)) = make_uint4(e[4], e[5], e[6], e[7]);
          }
          tm_fence_async();
          __syncwarp();
          if (lane == 0) {
            tm_arrive(&raw_empty[rs]);
            tm_arrive(half ? &v_full[s] : &k_full[s]);
          }
        }
      }
    }
  }
  __syncwarp();
  tm_fence_before();
  __syncthreads();
  if (warp == 4 * NS + 1) {
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

template <typename T, int STORE, int HD>
static int launch_mma(TreeArgs a, const stx_kv* cache, const TmOrder& o, int vec, cudaStream_t s) {
  typedef TmShape<STORE, HD> Z;
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
    STX_CUDA(cudaFuncSetAttribute(k_tree_attn_mma<T, STORE, HD>, cudaFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(Z::SMEM)));
    if (dev >= 0 && dev < 64) attr_set[dev] = true;
  }
  STX_CUDA(launch_pdl(k_tree_attn_mma<T, STORE, HD>, dim3(static_cast<unsigned>(a.grid)), dim3(Z::THREADS), Z::SMEM, s, a, maps, kv_ptr<C>(cache, false),
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
  a.min_tiles = 2;
  a.grid = num_sms();
  auto ok = [](const void* p, int64_t x, int64_t y, int64_t z) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0 && x % 8 == 0 && y % 8 == 0 && z % 8 == 0; };
  const int vec = ok(a.q, a.q_seq, a.q_tok, a.q_head) && ok(a.out, a.o_seq, a.o_tok, a.o_head);
  return by_store(cache->store, [&](auto st) -> int {
    constexpr int S = decltype(st)::value;
    if (cache->dtype == STX_F16)
      return a.hd <= 64 ? launch_mma<__half, S, 64>(a, cache, o, vec, s) : a.hd <= 128 ? launch_mma<__half, S, 128>(a, cache, o, vec, s) : launch_mma<__half, S, 256>(a, cache, o, vec, s);
    return a.hd <= 64 ? launch_mma<__nv_bfloat16, S, 64>(a, cache, o, vec, s)
                      : a.hd <= 128 ? launch_mma<__nv_bfloat16, S, 128>(a, cache, o, vec, s) : launch_mma<__nv_bfloat16, S, 256>(a, cache, o, vec, s);
  });
}

}  // namespace stx
