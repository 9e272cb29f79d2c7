// Rotary positions and the key/value cache of a decoder that checks drafted tokens (C ABI: stx_rope, stx_kv_append,
// stx_kv_read, stx_kv_keep, stx_draft_masks).
//
// Rotation of a pair by the angle a of its position:  y0 = f (x0 cos a - x1 sin a),  y1 = f (x1 cos a + x0 sin a).
// The angle, its sine and its cosine are formed in fp64 and rounded to fp32 once: an fp32 angle of position 10^6 would be off by
// 0.03, and an fp32 sine a few steps off moves a 16-bit rounding now and then.  A thread needs 8 of them for all heads of its
// token, about 20 fp64 operations each.
// Quantisation of a row (include/stx.h): scale = a / M, code = rn(x * (M / a)), both from the fp32 result of the rotation, so
// a cached key is rounded once.
//
//   k_rope_vec     16 values of a head a thread (two 16-byte vectors of 16-bit values), 8 pairs; a group of LPR lanes has a row.
//                  A thread keeps the sines of its pairs and walks the token's heads with them.
//   k_rope_any     a warp per row, any size, stride and alignment
//   k_kv_read_vec / k_kv_read_any, k_kv_keep, k_draft_masks
//
// What bounds them: HBM where there is much to move, else a launch.  8191 tokens x 40 heads of 128 values in bf16, 32 of them rotated: 38 us for
// 168 MB (4.4 TB/s); two prompts of 4096 tokens (32 + 8 + 8 heads) into an e4m3 cache and 16 x 4096 rows back: 64 us for 236 MB; 16 x 16384 rows of int8
// codes back to fp16: 40 us for 203 MB (5.1 TB/s).  Fewer heads a thread (more sines), more blocks an SM (spills) and requesting the next head
// ahead (registers: 54 us) were no faster.  Eight tokens: 7 us, which is an empty launch and one trip to memory.
#include "stx_kv.cuh"

#include <algorithm>

namespace stx {

int check_kv(const stx_kv* c, const char* who) {
  STX_CHECK_ARG(c && c->k && c->v, "%s: null cache", who);
  STX_CHECK_ARG(c->dtype == STX_F32 || c->dtype == STX_F16 || c->dtype == STX_BF16, "%s: bad dtype %d", who, c->dtype);
  STX_CHECK_ARG(c->store == STX_STORE_SAME || c->store == STX_STORE_INT8 || c->store == STX_STORE_E4M3, "%s: bad store %d", who, c->store);
  STX_CHECK_ARG(c->store == STX_STORE_SAME || (c->k_scale && c->v_scale), "%s: an 8-bit cache needs k_scale and v_scale", who);
  STX_CHECK_ARG(c->n_seq > 0 && c->n_kv_heads > 0 && c->max_len > 0, "%s: empty cache", who);
  STX_CHECK_ARG(c->max_len < (1ll << 30), "%s: max_len=%lld too large", who, static_cast<long long>(c->max_len));
  STX_CHECK_ARG(c->head_dim > 0 && c->head_dim <= 256, "%s: head_dim %d outside 1..256", who, c->head_dim);
  STX_CHECK_ARG(c->seq_stride >= 0 && c->head_stride >= 0 && c->slot_stride >= c->head_dim, "%s: bad cache strides", who);
  return STX_OK;
}
int check_heads(const stx_heads* h, const char* who, const char* name) {
  STX_CHECK_ARG(h && h->data, "%s: null %s", who, name);
  STX_CHECK_ARG(h->seq_stride >= 0 && h->token_stride >= 0 && h->head_stride >= 0, "%s: negative stride of %s", who, name);
  return STX_OK;
}

constexpr int ROPE_THREADS = 256;

// a / b of numbers that are not negative: a division of 64 bits costs about 100 instructions, as much as a row's other work.
__device__ __forceinline__ int64_t quick_div(int64_t a, int64_t b) {
  return ((a | b) >> 32) == 0 ? static_cast<int64_t>(static_cast<uint32_t>(a) / static_cast<uint32_t>(b)) : a / b;
}

// One launch of the rotation: q rows (heads 0 .. nh-1 of a token), then k and v rows where there is a cache.
template <typename T, int STORE> struct RopeArgs {
  typedef typename Held<T, STORE>::C C;
  const T *q, *k, *v;
  T* qo;
  int64_t q_seq, q_tok, q_head, qo_seq, qo_tok, qo_head, k_seq, k_tok, k_head, v_seq, v_tok, v_head;
  KvPtr<C> kc, vc;
  int64_t max_len;
  const int64_t *start, *counts, *positions;
  int64_t pos_stride;
  const double* turns;  // null: no rotation
  double factor, sign;  // sign -1: turned back
  int rot, interleaved;
  int64_t n_tok, tokens;  // tokens of a sequence, of all sequences
  int nh, nkv, hd, groups;  // groups: threads (rows of LPR lanes) that share a token's heads
};

// factor * cos and factor * sin of 2 pi pos turns, each rounded once.  The fraction of a turn is cut to r in [-1/8, 1/8] around a
// quarter n; the Taylor series of sin and cos up to a^11 and a^12 leave a^13 / 13! < 7e-12 at a = pi / 4, under a thousandth of an fp32 step.
__device__ __forceinline__ void pair_angle(double pos, double turns, double factor, double sign, float& c, float& s) {
  const double t = pos * turns, f = t - rint(t), n = rint(4.0 * f);
  const double a = 6.283185307179586 * fma(n, -0.25, f), z = a * a;
  const double sn = a * fma(z, fma(z, fma(z, fma(z, fma(z, -1.0 / 39916800, 1.0 / 362880), -1.0 / 5040), 1.0 / 120), -1.0 / 6), 1.0);
  const double cs = fma(z, fma(z, fma(z, fma(z, fma(z, fma(z, 1.0 / 479001600, -1.0 / 3628800), 1.0 / 40320), -1.0 / 720), 1.0 / 24), -0.5), 1.0);
  const int k = static_cast<int>(n);  // quarters turned, -2 .. 2
  const double c2 = k & 1 ? sn : cs, s2 = k & 1 ? cs : sn;
  c = static_cast<float>((k == 1 || k == 2 || k == -2 ? -c2 : c2) * factor);
  s = static_cast<float>((k == -1 || k == 2 || k == -2 ? -s2 : s2) * factor * sign);
}

// Two rounded products and a rounded sum, as in k_attn_decode, whatever kernel runs.
__device__ __forceinline__ float turned0(float x0, float x1, float c, float s) { return __fsub_rn(__fmul_rn(x0, c), __fmul_rn(x1, s)); }
__device__ __forceinline__ float turned1(float x0, float x1, float c, float s) { return __fadd_rn(__fmul_rn(x1, c), __fmul_rn(x0, s)); }

// Scale and inverse of a row from the bits of its largest magnitude (NaN and infinities sort above all finite values).
__device__ __forceinline__ void row_scale(uint32_t top_bits, float most, float& scale, float& inv) {
  const float top = __uint_as_float(top_bits);
  scale = top / most;
  inv = most / top;
  if (scale < 1.17549435e-38f) scale = inv = 0.f;  // below the normal numbers: held as zeros
  if (top_bits >= 0x7f800000u) {
    scale = __int_as_float(0x7fc00000);
    inv = 0.f;
  }
}
template <int STORE>
__device__ __forceinline__ uint32_t code4(float a, float b, float c, float d) {
  if constexpr (STORE == STX_STORE_INT8) {
    return (static_cast<uint32_t>(__float2int_rn(a)) & 255u) | ((static_cast<uint32_t>(__float2int_rn(b)) & 255u) << 8) |
           ((static_cast<uint32_t>(__float2int_rn(c)) & 255u) << 16) | (static_cast<uint32_t>(__float2int_rn(d)) << 24);
  } else {
    const uint32_t lo = __nv_cvt_float2_to_fp8x2(make_float2(a, b), __NV_SATFINITE, __NV_E4M3);
    const uint32_t hi = __nv_cvt_float2_to_fp8x2(make_float2(c, d), __NV_SATFINITE, __NV_E4M3);
    return lo | (hi << 16);
  }
}

// 8 consecutive values (fp32: two vectors of four).
template <typename T>
__device__ __forceinline__ void load8(const T* p, float (&f)[8]) {
  if constexpr (sizeof(T) == 2) {
    Unpack<T>::run(ld_cached16(p), f);
  } else {
    Unpack<T>::run(ld_cached16(p), f);
    Unpack<T>::run(ld_cached16(p + 4), f + 4);
  }
}
template <typename T>
__device__ __forceinline__ void store8(T* p, const float (&f)[8]) {
  if constexpr (sizeof(T) == 2) {
    T h[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) h[i] = DT<T>::from_f(f[i]);
    st16(p, *reinterpret_cast<const uint4*>(h));
  } else {
    st16(p, make_uint4(__float_as_uint(f[0]), __float_as_uint(f[1]), __float_as_uint(f[2]), __float_as_uint(f[3])));
    st16(p + 4, make_uint4(__float_as_uint(f[4]), __float_as_uint(f[5]), __float_as_uint(f[6]), __float_as_uint(f[7])));
  }
}

// hd a multiple of 16, rotary_dim too (or 0), everything 16-byte aligned.  Lane j of a row has two runs of 8 values: for
// j < rot / 16 the pairs 8 j .. 8 j + 7, behind them 16 values that are copied.
template <typename T, int STORE, int LPR>
__global__ void __launch_bounds__(ROPE_THREADS) k_rope_vec(const RopeArgs<T, STORE> a) {
  const int64_t id = static_cast<int64_t>(blockIdx.x) * ROPE_THREADS + threadIdx.x;
  const int j = threadIdx.x % LPR;
  const int64_t row = id / LPR;
  const int64_t tok = quick_div(row, a.groups);
  pdl_wait();
  pdl_launch_dependents();
  if (tok >= a.tokens) return;  // the lanes of a row leave together
  const int h0 = static_cast<int>(row - tok * a.groups);
  const int64_t b = quick_div(tok, a.n_tok), t = tok - b * a.n_tok;
  const bool used = !a.counts || t < a.counts[b];
  const bool act = 16 * j < a.hd;
  const bool turned = 16 * j < a.rot;
  const int64_t slot = a.start ? a.start[b] + t : t;
  const int first = turned && !a.interleaved ? 8 * j : 16 * j;
  const int second = turned && !a.interleaved ? a.rot / 2 + 8 * j : 16 * j + 8;
  float c[8], s[8];
  if (turned && used) {
    const double pos = static_cast<double>(a.positions ? a.positions[b * a.pos_stride + t] : slot);
#pragma unroll
    for (int i = 0; i < 8; ++i) pair_angle(pos, a.turns[8 * j + i], a.factor, a.sign, c[i], s[i]);
  }
  const bool there = used && slot >= 0 && slot < a.max_len;
  const int heads = a.nh + 2 * a.nkv;
  const uint32_t lanes = LPR == 32 ? 0xffffffffu : ((1u << LPR) - 1) << (threadIdx.x & 31 & ~(LPR - 1));
  for (int h = h0; h < heads; h += a.groups) {
    const bool is_q = h < a.nh, is_k = !is_q && h < a.nh + a.nkv;
    if (!is_q && !there) break;  // keys and values come last
    const int hh = is_q ? h : is_k ? h - a.nh : h - a.nh - a.nkv;
    const T* src = is_q ? a.q + b * a.q_seq + t * a.q_tok + hh * a.q_head
                        : is_k ? a.k + b * a.k_seq + t * a.k_tok + hh * a.k_head : a.v + b * a.v_seq + t * a.v_tok + hh * a.v_head;
    float x[8], y[8];
    if (act && used) {
      load8(src + first, x);
      load8(src + second, y);
    } else {
#pragma unroll
      for (int i = 0; i < 8; ++i) x[i] = y[i] = 0.f;
    }
    if (turned && used && (is_q || is_k)) {
      if (a.interleaved) {
#pragma unroll
        for (int i = 0; i < 8; i += 2) {  // x: pairs 0..3, y: pairs 4..7
          const float x0 = x[i], x1 = x[i + 1], y0 = y[i], y1 = y[i + 1];
          x[i] = turned0(x0, x1, c[i / 2], s[i / 2]);
          x[i + 1] = turned1(x0, x1, c[i / 2], s[i / 2]);
          y[i] = turned0(y0, y1, c[4 + i / 2], s[4 + i / 2]);
          y[i + 1] = turned1(y0, y1, c[4 + i / 2], s[4 + i / 2]);
        }
      } else {
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          const float x0 = x[i], x1 = y[i];
          x[i] = turned0(x0, x1, c[i], s[i]);
          y[i] = turned1(x0, x1, c[i], s[i]);
        }
      }
    }
    if (is_q) {
      if (act) {
        T* dst = a.qo + b * a.qo_seq + t * a.qo_tok + hh * a.qo_head;
        store8(dst + first, x);
        store8(dst + second, y);
      }
      continue;
    }
    const KvPtr<typename Held<T, STORE>::C>& cache = is_k ? a.kc : a.vc;
    auto* dst = cache.row(b, hh, slot);
    if constexpr (STORE == STX_STORE_SAME) {
      if (act) {
        store8(dst + first, x);
        store8(dst + second, y);
      }
    } else {
      uint32_t top = 0;
#pragma unroll
      for (int i = 0; i < 8; ++i) top = max(top, max(__float_as_uint(x[i]) & 0x7fffffffu, __float_as_uint(y[i]) & 0x7fffffffu));
#pragma unroll
      for (int off = LPR / 2; off > 0; off >>= 1) top = max(top, __shfl_xor_sync(lanes, top, off));
      float scale, inv;
      row_scale(top, Held<T, STORE>::MOST, scale, inv);
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        x[i] = inv == 0.f ? 0.f : x[i] * inv;  // no 0 * infinity
        y[i] = inv == 0.f ? 0.f : y[i] * inv;
      }
      if (act) {
        const uint2 cx = make_uint2(code4<STORE>(x[0], x[1], x[2], x[3]), code4<STORE>(x[4], x[5], x[6], x[7]));
        const uint2 cy = make_uint2(code4<STORE>(y[0], y[1], y[2], y[3]), code4<STORE>(y[4], y[5], y[6], y[7]));
        *reinterpret_cast<uint2*>(dst + first) = cx;
        *reinterpret_cast<uint2*>(dst + second) = cy;
      }
      if (j == 0) cache.srow(b, hh)[slot] = scale;
    }
  }
}

// A warp per (token, head).  Two passes over the row for the 8-bit stores; a pair's two values are formed by the thread of each.
template <typename T, int STORE>
__global__ void __launch_bounds__(ROPE_THREADS) k_rope_any(const RopeArgs<T, STORE> a) {
  const int lane = threadIdx.x & 31;
  const int64_t row = static_cast<int64_t>(blockIdx.x) * (ROPE_THREADS / 32) + (threadIdx.x >> 5);
  pdl_wait();
  pdl_launch_dependents();
  const int heads = a.nh + 2 * a.nkv;
  const int64_t tok = row / heads;
  if (tok >= a.tokens) return;
  const int h = static_cast<int>(row - tok * heads);
  const int64_t b = tok / a.n_tok, t = tok - b * a.n_tok;
  const bool used = !a.counts || t < a.counts[b];
  const bool is_q = h < a.nh, is_k = !is_q && h < a.nh + a.nkv;
  const int64_t slot = a.start ? a.start[b] + t : t;
  if (!is_q && !(used && slot >= 0 && slot < a.max_len)) return;
  const int hh = is_q ? h : is_k ? h - a.nh : h - a.nh - a.nkv;
  const T* src = is_q ? a.q + b * a.q_seq + t * a.q_tok + hh * a.q_head
                      : is_k ? a.k + b * a.k_seq + t * a.k_tok + hh * a.k_head : a.v + b * a.v_seq + t * a.v_tok + hh * a.v_head;
  const double pos = static_cast<double>(a.positions ? a.positions[b * a.pos_stride + t] : slot);
  const int half = a.rot / 2;
  auto value = [&](int i) -> float {
    if (!used) return 0.f;
    const float x = DT<T>::to_f(src[i]);
    if (i >= a.rot || !(is_q || is_k)) return x;
    const bool hi = a.interleaved ? (i & 1) : i >= half;
    const float o = DT<T>::to_f(src[a.interleaved ? i ^ 1 : hi ? i - half : i + half]);
    float c, s;
    pair_angle(pos, a.turns[a.interleaved ? i >> 1 : hi ? i - half : i], a.factor, a.sign, c, s);
    return hi ? turned1(o, x, c, s) : turned0(x, o, c, s);
  };
  if (is_q) {
    // q_out may be q: a value's partner is read before either is written (up to 1024 values: 32 a lane)
    T* dst = a.qo + b * a.qo_seq + t * a.qo_tok + hh * a.qo_head;
    float f[32];
#pragma unroll
    for (int k = 0; k < 32; ++k)
      if (lane + 32 * k < a.hd) f[k] = value(lane + 32 * k);
    __syncwarp();
#pragma unroll
    for (int k = 0; k < 32; ++k)
      if (lane + 32 * k < a.hd) dst[lane + 32 * k] = DT<T>::from_f(f[k]);
    return;
  }
  const KvPtr<typename Held<T, STORE>::C>& cache = is_k ? a.kc : a.vc;
  auto* dst = cache.row(b, hh, slot);
  if constexpr (STORE == STX_STORE_SAME) {
    for (int i = lane; i < a.hd; i += 32) dst[i] = DT<T>::from_f(value(i));
  } else {
    uint32_t top = 0;
    for (int i = lane; i < a.hd; i += 32) top = max(top, __float_as_uint(value(i)) & 0x7fffffffu);
    top = __reduce_max_sync(0xffffffffu, top);
    float scale, inv;
    row_scale(top, Held<T, STORE>::MOST, scale, inv);
    for (int i = lane; i < a.hd; i += 32)
      dst[i] = static_cast<typename Held<T, STORE>::C>(code4<STORE>(inv == 0.f ? 0.f : value(i) * inv, 0.f, 0.f, 0.f) & 255u);
    if (lane == 0) cache.srow(b, hh)[slot] = scale;
  }
}

static bool aligned16(const void* p, int64_t s0, int64_t s1, int64_t s2, size_t size) {
  return (reinterpret_cast<uintptr_t>(p) & 15) == 0 && (s0 * size) % 16 == 0 && (s1 * size) % 16 == 0 && (s2 * size) % 16 == 0;
}

template <typename T, int STORE>
static int launch_rope(RopeArgs<T, STORE> a, cudaStream_t s) {
  if (a.tokens == 0) return STX_OK;
  const int heads = a.nh + 2 * a.nkv;
  const size_t ts = sizeof(T), cs = sizeof(typename Held<T, STORE>::C);
  // The codes of a lane are two runs of 8 bytes, so an 8-bit cache needs no more than that; 16 keeps the rule one.
  bool vec = a.hd % 16 == 0 && a.rot % 16 == 0 && a.hd <= 256;
  if (a.nh) vec = vec && aligned16(a.q, a.q_seq, a.q_tok, a.q_head, ts) && aligned16(a.qo, a.qo_seq, a.qo_tok, a.qo_head, ts);
  if (a.nkv)
    vec = vec && aligned16(a.k, a.k_seq, a.k_tok, a.k_head, ts) && aligned16(a.v, a.v_seq, a.v_tok, a.v_head, ts) &&
          aligned16(a.kc.data, a.kc.seq, a.kc.head, a.kc.slot, cs) && aligned16(a.vc.data, a.vc.seq, a.vc.head, a.vc.slot, cs);
  if (!vec) {
    const int64_t warps = a.tokens * heads, blocks = (warps + ROPE_THREADS / 32 - 1) / (ROPE_THREADS / 32);
    STX_CHECK_ARG(blocks < (1ll << 31), "stx_rope / stx_kv_append: too many rows");
    STX_CUDA(launch_pdl(k_rope_any<T, STORE>, dim3(static_cast<unsigned>(blocks)), dim3(ROPE_THREADS), 0, s, a));
    return STX_OK;
  }
  const int need = a.hd / 16, lpr = need <= 4 ? 4 : need <= 8 ? 8 : 16;
  // Heads of a thread: as many as leave the chip about 1500 threads an SM, eight at most.
  const int64_t all = a.tokens * heads * lpr;
  const int64_t each = std::max<int64_t>(1, std::min<int64_t>(8, all / (static_cast<int64_t>(num_sms()) * 1536)));
  a.groups = static_cast<int>((heads + each - 1) / each);
  const int64_t blocks = (a.tokens * a.groups * lpr + ROPE_THREADS - 1) / ROPE_THREADS;
  STX_CHECK_ARG(blocks < (1ll << 31), "stx_rope / stx_kv_append: too many rows");
  const dim3 grid(static_cast<unsigned>(blocks)), block(ROPE_THREADS);
  if (lpr == 4) STX_CUDA(launch_pdl(k_rope_vec<T, STORE, 4>, grid, block, 0, s, a));
  else if (lpr == 8) STX_CUDA(launch_pdl(k_rope_vec<T, STORE, 8>, grid, block, 0, s, a));
  else STX_CUDA(launch_pdl(k_rope_vec<T, STORE, 16>, grid, block, 0, s, a));
  return STX_OK;
}

static int check_rotary(const stx_rotary* r, int head_dim, const char* who) {
  STX_CHECK_ARG(r->turns, "%s: null turns", who);
  STX_CHECK_ARG(r->rotary_dim > 0 && r->rotary_dim <= head_dim && r->rotary_dim % 2 == 0, "%s: rotary_dim %d of a head of %d", who,
                r->rotary_dim, head_dim);
  return STX_OK;
}
template <typename T, int STORE>
static void set_rotary(RopeArgs<T, STORE>& a, const stx_rotary* r, int inverse) {
  a.turns = r ? r->turns : nullptr;
  a.rot = r ? r->rotary_dim : 0;
  a.interleaved = r ? r->interleaved != 0 : 0;
  a.factor = r ? r->factor : 1.0;
  a.sign = inverse ? -1.0 : 1.0;
}

// ---------------------------------------------------------------------------------- reading back
// 16 values a thread: hd a multiple of 16, 16-byte aligned rows.
template <typename T, int STORE>
__global__ void __launch_bounds__(256) k_kv_read_vec(const KvPtr<typename Held<T, STORE>::C> kc, const KvPtr<typename Held<T, STORE>::C> vc,
                                                     const int64_t* __restrict__ start, int64_t n, int64_t max_len, int nkv, int hd,
                                                     int64_t items, T* __restrict__ k_out, T* __restrict__ v_out) {
  const int64_t id = static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x;
  pdl_wait();
  pdl_launch_dependents();
  if (id >= items) return;
  const int lpr = hd / 16;
  const int64_t row = quick_div(id, lpr), bh = quick_div(row, n), b = quick_div(bh, nkv);
  const int j = static_cast<int>(id - row * lpr), h = static_cast<int>(bh - b * nkv);
  const int64_t slot = (start ? start[b] : 0) + row - bh * n;
  const bool there = slot >= 0 && slot < max_len;
  const KvPtr<typename Held<T, STORE>::C>& c = blockIdx.y ? vc : kc;
  float f[2][8];
  if (!there) {
#pragma unroll
    for (int i = 0; i < 16; ++i) f[i / 8][i % 8] = 0.f;
  } else if constexpr (STORE == STX_STORE_SAME) {
    const T* src = c.row(b, h, slot) + 16 * j;
    load8(src, f[0]);
    load8(src + 8, f[1]);
  } else {
    const float scale = c.srow(b, h)[slot];
    const uint4 raw = ld_cached16(c.row(b, h, slot) + 16 * j);
    const uint32_t w[4] = {raw.x, raw.y, raw.z, raw.w};
#pragma unroll
    for (int i = 0; i < 16; ++i)
      f[i / 8][i % 8] = held_value<T, STORE>(static_cast<typename Held<T, STORE>::C>((w[i / 4] >> (8 * (i % 4))) & 255u), scale);
  }
  T* dst = (blockIdx.y ? v_out : k_out) + row * hd + 16 * j;
  store8(dst, f[0]);
  store8(dst + 8, f[1]);
}
template <typename T, int STORE>
__global__ void __launch_bounds__(256) k_kv_read_any(const KvPtr<typename Held<T, STORE>::C> kc, const KvPtr<typename Held<T, STORE>::C> vc,
                                                     const int64_t* __restrict__ start, int64_t n, int64_t max_len, int nkv, int hd,
                                                     int64_t items, T* __restrict__ k_out, T* __restrict__ v_out) {
  const int64_t id = static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x;
  pdl_wait();
  pdl_launch_dependents();
  if (id >= items) return;
  const int64_t row = quick_div(id, hd), bh = quick_div(row, n), b = quick_div(bh, nkv);
  const int d = static_cast<int>(id - row * hd), h = static_cast<int>(bh - b * nkv);
  const int64_t slot = (start ? start[b] : 0) + row - bh * n;
  const KvPtr<typename Held<T, STORE>::C>& c = blockIdx.y ? vc : kc;
  float f = 0.f;
  if (slot >= 0 && slot < max_len) f = held_value<T, STORE>(c.row(b, h, slot)[d], STORE == STX_STORE_SAME ? 1.f : c.srow(b, h)[slot]);
  (blockIdx.y ? v_out : k_out)[id] = DT<T>::from_f(f);
}

// ---------------------------------------------------------------------------------- the accepted rows move together
// A block per (head, k or v; sequence; layer): all rows of the path go to shared memory before the first is written.
__global__ void __launch_bounds__(256) k_kv_keep(unsigned char* k, unsigned char* v, float* ks, float* vs, int64_t layer, int64_t seq,
                                                 int64_t head, int64_t slot_b, int64_t slayer, int64_t sseq, int64_t shead, int row_bytes,
                                                 int64_t max_len, const int64_t* __restrict__ start, const int64_t* __restrict__ path,
                                                 int64_t path_stride, int n_path, const int64_t* __restrict__ counts) {
  extern __shared__ __align__(16) unsigned char rows_s[];
  __shared__ float scale_s[STX_DRAFT_MAX];
  const int h = blockIdx.x >> 1, b = blockIdx.y;
  const int64_t l = blockIdx.z;
  pdl_wait();
  pdl_launch_dependents();
  // Cut to 0 .. n_path in 64 bits: below, n is compared with unsigned thread numbers too.
  const int n = static_cast<int>(max(0ll, min(static_cast<long long>(n_path), static_cast<long long>(counts[b]))));
  const int64_t s0 = start[b];
  unsigned char* data = (blockIdx.x & 1 ? v : k) + l * layer + b * seq + h * head;
  float* scale = blockIdx.x & 1 ? vs : ks;
  if (scale) scale += l * slayer + b * sseq + h * shead;
  auto from = [&](int i) -> int64_t {  // -1: this pair is skipped
    const int64_t p = path[b * path_stride + i], src = s0 + p, dst = s0 + i;
    return src >= 0 && src < max_len && dst >= 0 && dst < max_len ? src : -1;
  };
  const bool wide = ((reinterpret_cast<uintptr_t>(data) | static_cast<uintptr_t>(slot_b) | static_cast<uintptr_t>(row_bytes)) & 15) == 0;
  const int unit = wide ? 16 : 1, per = row_bytes / unit;
  for (int i = threadIdx.x; i < n * per; i += blockDim.x) {
    const int r = i / per, o = (i - r * per) * unit;
    const int64_t src = from(r);
    if (src < 0) continue;
    if (wide) *reinterpret_cast<uint4*>(rows_s + r * row_bytes + o) = *reinterpret_cast<const uint4*>(data + src * slot_b + o);
    else rows_s[r * row_bytes + o] = data[src * slot_b + o];
  }
  if (scale && threadIdx.x < n && from(threadIdx.x) >= 0) scale_s[threadIdx.x] = scale[from(threadIdx.x)];
  __syncthreads();
  for (int i = threadIdx.x; i < n * per; i += blockDim.x) {
    const int r = i / per, o = (i - r * per) * unit;
    if (from(r) < 0) continue;
    if (wide) *reinterpret_cast<uint4*>(data + (s0 + r) * slot_b + o) = *reinterpret_cast<const uint4*>(rows_s + r * row_bytes + o);
    else data[(s0 + r) * slot_b + o] = rows_s[r * row_bytes + o];
  }
  if (scale && threadIdx.x < n && from(threadIdx.x) >= 0) scale[s0 + threadIdx.x] = scale_s[threadIdx.x];
}

// A warp per sequence; node i's bits follow from its parent's, which stand in shared memory.
__global__ void __launch_bounds__(32) k_draft_masks(const int64_t* __restrict__ parents, int n_tok, int64_t* __restrict__ masks,
                                                    int64_t* __restrict__ depth) {
  __shared__ unsigned long long m_s[STX_DRAFT_MAX];
  __shared__ int64_t p_s[STX_DRAFT_MAX];
  const int64_t at = static_cast<int64_t>(blockIdx.x) * n_tok;
  pdl_wait();
  pdl_launch_dependents();
  for (int i = threadIdx.x; i < n_tok; i += 32) p_s[i] = parents[at + i];
  __syncwarp();
  if (threadIdx.x == 0)
    for (int i = 0; i < n_tok; ++i) m_s[i] = (1ull << i) | (p_s[i] >= 0 && p_s[i] < i ? m_s[p_s[i]] : 0ull);
  __syncwarp();
  for (int i = threadIdx.x; i < n_tok; i += 32) {
    masks[at + i] = static_cast<int64_t>(m_s[i]);
    if (depth) depth[at + i] = __popcll(m_s[i]) - 1;
  }
}

}  // namespace stx

using namespace stx;

extern "C" {

int stx_rope(const stx_heads* x, const stx_heads* out, int64_t n_seq, int64_t n_tokens, int heads, int head_dim,
             const int64_t* positions, int64_t position_stride, const stx_rotary* rotary, int inverse, int dtype, void* stream) {
  int rc = check_heads(x, "stx_rope", "x");
  if (rc == STX_OK) rc = check_heads(out, "stx_rope", "out");
  if (rc != STX_OK) return rc;
  STX_CHECK_ARG(positions && rotary, "stx_rope: null pointer");
  STX_CHECK_ARG(dtype == STX_F32 || dtype == STX_F16 || dtype == STX_BF16, "stx_rope: bad dtype %d", dtype);
  STX_CHECK_ARG(n_seq >= 0 && n_tokens >= 0 && heads > 0 && head_dim > 0 && head_dim <= 1024 && position_stride >= 0, "stx_rope: bad shape");
  if ((rc = check_rotary(rotary, head_dim, "stx_rope")) != STX_OK) return rc;
  STX_CHECK_ARG(n_seq == 0 || n_tokens < (1ll << 40) / n_seq, "stx_rope: too many tokens");
  return by_dtype(dtype, [&](auto tag) -> int {
    typedef decltype(tag) T;
    RopeArgs<T, STX_STORE_SAME> a{};
    a.q = static_cast<const T*>(x->data);
    a.qo = static_cast<T*>(out->data);
    a.q_seq = x->seq_stride, a.q_tok = x->token_stride, a.q_head = x->head_stride;
    a.qo_seq = out->seq_stride, a.qo_tok = out->token_stride, a.qo_head = out->head_stride;
    a.positions = positions;
    a.pos_stride = position_stride;
    set_rotary(a, rotary, inverse);
    a.n_tok = n_tokens;
    a.tokens = n_seq * n_tokens;
    a.nh = heads;
    a.hd = head_dim;
    return launch_rope(a, static_cast<cudaStream_t>(stream));
  });
}

int stx_kv_append(const stx_kv* cache, const stx_heads* k, const stx_heads* v, int64_t n_tokens, const int64_t* start,
                  const int64_t* counts, const stx_rotary* rotary, const int64_t* positions, int64_t position_stride,
                  const stx_heads* q, const stx_heads* q_out, int n_heads, void* stream) {
  int rc = check_kv(cache, "stx_kv_append");
  if (rc == STX_OK) rc = check_heads(k, "stx_kv_append", "k");
  if (rc == STX_OK) rc = check_heads(v, "stx_kv_append", "v");
  if (rc == STX_OK && rotary) rc = check_rotary(rotary, cache->head_dim, "stx_kv_append");
  const bool has_q = q && q->data;
  if (rc == STX_OK && has_q) rc = check_heads(q, "stx_kv_append", "q");
  if (rc == STX_OK && has_q) rc = check_heads(q_out, "stx_kv_append", "q_out");
  if (rc != STX_OK) return rc;
  STX_CHECK_ARG(start, "stx_kv_append: null start");
  STX_CHECK_ARG(n_tokens >= 0 && position_stride >= 0 && n_tokens < (1ll << 40) / cache->n_seq, "stx_kv_append: bad shape");
  STX_CHECK_ARG(!has_q || n_heads > 0, "stx_kv_append: q needs n_heads");
  return by_dtype(cache->dtype, [&](auto tag) -> int {
    typedef decltype(tag) T;
    return by_store(cache->store, [&](auto st) -> int {
      RopeArgs<T, decltype(st)::value> a{};
      if (has_q) {
        a.q = static_cast<const T*>(q->data);
        a.qo = static_cast<T*>(q_out->data);
        a.q_seq = q->seq_stride, a.q_tok = q->token_stride, a.q_head = q->head_stride;
        a.qo_seq = q_out->seq_stride, a.qo_tok = q_out->token_stride, a.qo_head = q_out->head_stride;
      }
      a.k = static_cast<const T*>(k->data);
      a.v = static_cast<const T*>(v->data);
      a.k_seq = k->seq_stride, a.k_tok = k->token_stride, a.k_head = k->head_stride;
      a.v_seq = v->seq_stride, a.v_tok = v->token_stride, a.v_head = v->head_stride;
      a.kc = kv_ptr<typename Held<T, decltype(st)::value>::C>(cache, false);
      a.vc = kv_ptr<typename Held<T, decltype(st)::value>::C>(cache, true);
      a.max_len = cache->max_len;
      a.start = start;
      a.counts = counts;
      a.positions = positions;
      a.pos_stride = position_stride;
      set_rotary(a, rotary, 0);
      a.n_tok = n_tokens;
      a.tokens = cache->n_seq * n_tokens;
      a.nh = has_q ? n_heads : 0;
      a.nkv = cache->n_kv_heads;
      a.hd = cache->head_dim;
      return launch_rope(a, static_cast<cudaStream_t>(stream));
    });
  });
}

int stx_kv_read(const stx_kv* cache, const int64_t* start, int64_t n, void* k_out, void* v_out, void* stream) {
  int rc = check_kv(cache, "stx_kv_read");
  if (rc != STX_OK) return rc;
  STX_CHECK_ARG(n >= 0 && n < (1ll << 31), "stx_kv_read: n=%lld out of range", static_cast<long long>(n));
  if (n == 0) return STX_OK;
  STX_CHECK_ARG(k_out && v_out, "stx_kv_read: null output");
  return by_dtype(cache->dtype, [&](auto tag) -> int {
    typedef decltype(tag) T;
    return by_store(cache->store, [&](auto st) -> int {
      constexpr int S = decltype(st)::value;
      typedef typename Held<T, S>::C C;
      const KvPtr<C> kc = kv_ptr<C>(cache, false), vc = kv_ptr<C>(cache, true);
      const bool vec = cache->head_dim % 16 == 0 && aligned16(kc.data, kc.seq, kc.head, kc.slot, sizeof(C)) &&
                       aligned16(vc.data, vc.seq, vc.head, vc.slot, sizeof(C)) && aligned16(k_out, 0, 0, 0, 1) && aligned16(v_out, 0, 0, 0, 1);
      const int64_t items = static_cast<int64_t>(cache->n_seq) * cache->n_kv_heads * n * cache->head_dim / (vec ? 16 : 1);
      const int64_t blocks = (items + 255) / 256;
      STX_CHECK_ARG(blocks < (1ll << 31), "stx_kv_read: too many rows");
      const dim3 grid(static_cast<unsigned>(blocks), 2);
      STX_CUDA(launch_pdl(vec ? k_kv_read_vec<T, S> : k_kv_read_any<T, S>, grid, dim3(256), 0, static_cast<cudaStream_t>(stream), kc, vc, start, n,
                          cache->max_len, cache->n_kv_heads, cache->head_dim, items, static_cast<T*>(k_out), static_cast<T*>(v_out)));
      return STX_OK;
    });
  });
}

int stx_kv_keep(const stx_kv* cache, int64_t layers, int64_t layer_stride, int64_t scale_layer_stride, const int64_t* start,
                const int64_t* path, int64_t path_stride, int64_t n_path, const int64_t* counts, void* stream) {
  int rc = check_kv(cache, "stx_kv_keep");
  if (rc != STX_OK) return rc;
  STX_CHECK_ARG(start && path && counts, "stx_kv_keep: null pointer");
  STX_CHECK_ARG(n_path >= 0 && n_path <= STX_DRAFT_MAX, "stx_kv_keep: a path of %lld nodes is longer than %d", static_cast<long long>(n_path), STX_DRAFT_MAX);
  STX_CHECK_ARG(layers > 0 && layers < 65536 && layer_stride >= 0 && scale_layer_stride >= 0 && path_stride >= 0, "stx_kv_keep: bad layers or strides");
  STX_CHECK_ARG(cache->n_seq < 65536, "stx_kv_keep: more than 65535 sequences");
  if (n_path == 0) return STX_OK;
  const int64_t es = static_cast<int64_t>(store_size(cache->store, cache->dtype));
  const int row_bytes = static_cast<int>(cache->head_dim * es);
  const size_t smem = static_cast<size_t>(n_path) * row_bytes;
  if (smem > 48 * 1024) {
    static bool attr_set[64] = {};
    int dev = 0;
    STX_CUDA(cudaGetDevice(&dev));
    if (dev < 0 || dev >= 64 || !attr_set[dev]) {
      STX_CUDA(cudaFuncSetAttribute(k_kv_keep, cudaFuncAttributeMaxDynamicSharedMemorySize, STX_DRAFT_MAX * 256 * 4));
      if (dev >= 0 && dev < 64) attr_set[dev] = true;
    }
  }
  const bool scaled = cache->store != STX_STORE_SAME;
  STX_CUDA(launch_pdl(k_kv_keep, dim3(2u * static_cast<unsigned>(cache->n_kv_heads), static_cast<unsigned>(cache->n_seq), static_cast<unsigned>(layers)),
                      dim3(256), smem, static_cast<cudaStream_t>(stream), static_cast<unsigned char*>(cache->k), static_cast<unsigned char*>(cache->v),
                      scaled ? cache->k_scale : nullptr, scaled ? cache->v_scale : nullptr, layer_stride * es, cache->seq_stride * es,
                      cache->head_stride * es, cache->slot_stride * es, scale_layer_stride, cache->scale_seq_stride, cache->scale_head_stride,
                      row_bytes, cache->max_len, start, path, path_stride, static_cast<int>(n_path), counts));
  return STX_OK;
}

int stx_draft_masks(const int64_t* parents, int64_t n_seq, int64_t n_tokens, int64_t* masks, int64_t* depth, void* stream) {
  STX_CHECK_ARG(parents && masks, "stx_draft_masks: null pointer");
  STX_CHECK_ARG(n_seq >= 0 && n_seq < (1ll << 31), "stx_draft_masks: bad n_seq");
  STX_CHECK_ARG(n_tokens > 0 && n_tokens <= STX_DRAFT_MAX, "stx_draft_masks: a draft of %lld nodes is outside 1..%d", static_cast<long long>(n_tokens), STX_DRAFT_MAX);
  if (n_seq == 0) return STX_OK;
  STX_CUDA(launch_pdl(k_draft_masks, dim3(static_cast<unsigned>(n_seq)), dim3(32), 0, static_cast<cudaStream_t>(stream), parents,
                      static_cast<int>(n_tokens), masks, depth));
  return STX_OK;
}

}  // extern "C"
