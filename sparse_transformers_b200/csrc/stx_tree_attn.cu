// Attention of drafted tokens over a cache (C ABI: stx_tree_attention): entry points, the kernel for any type, size and
// alignment, and the launch that adds partial results.  include/stx.h has the definition, stx_tree_attn.cuh how the work is
// shared out.
//
// One pass over the keys with the running maximum m and sum l of the soft-max:
//   x_j = scale log2(e) q . k_j,  m' = max(m, max_j x_j),  p_j = 2^(x_j - m'),  l' = 2^(m - m') l + sum p_j,  o' = 2^(m - m') o + sum p_j v_j
#include "stx_tree_attn.cuh"

#include <algorithm>
#include <cmath>

namespace stx {

constexpr int TG_THREADS = 256;
constexpr int TG_KT = 64;

// Any type, store, head_dim and alignment, fp32 arithmetic on the FMA pipe.  Keys and values are turned into fp32 in
// shared memory; a thread has four rows x one key of the scores and TASKS x (four rows x four values) of the output.
// A weight of zero never touches the value's bits, so what a masked slot holds does not matter.
// Shared memory (floats): q [ROWS][hdp] | k [KT][hdp + 4] | v [KT][hdp] | p [ROWS][KT + 4] | m, l, corr [ROWS] ; hdp = hd rounded up to 4
template <typename T, int STORE, int ROWS, int TASKS>
__global__ void __launch_bounds__(TG_THREADS, 1) k_tree_attn_any(const TreeArgs a, const KvPtr<typename Held<T, STORE>::C> kc,
                                                               const KvPtr<typename Held<T, STORE>::C> vc, int vec) {
  typedef typename Held<T, STORE>::C C;
  extern __shared__ __align__(16) float tg[];
  __shared__ int pre[TREE_PRE];
  __shared__ unsigned long long bits_s[ROWS];
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int hdp = (a.hd + 3) / 4 * 4, d4n = hdp / 4;
  float* q_s = tg;
  float* k_s = q_s + ROWS * hdp;
  float* v_s = k_s + TG_KT * (hdp + 4);
  float* p_s = v_s + TG_KT * hdp;
  float* m_s = p_s + ROWS * (TG_KT + 4);
  float* l_s = m_s + ROWS;
  float* c_s = l_s + ROWS;
  pdl_wait();
  pdl_launch_dependents();
  tree_prefix(a, TG_KT, pre);
  __syncthreads();
  const TreeLine line = tree_line(a, pre);
  const int cta = blockIdx.x;
  if (cta >= line.ctas) return;
  const int end = tree_begin(line, cta + 1), begin = tree_begin(line, cta);
  for (int x = begin; x < end;) {
    const TreeSeg sg = tree_seg(a, line, pre, x, end);
    const TreeSeq sq = tree_seq(a, sg.b);
    const int tok0 = sg.rt * a.tile_tok, rows = min(a.tile_tok, a.n_tok - tok0) * a.group;
    __syncthreads();  // the segment before is written
    for (int i = tid; i < ROWS * hdp; i += TG_THREADS) {
      const int r = i / hdp, d = i - r * hdp;
      float f = 0.f;
      if (r < rows && d < a.hd) {
        const T* row = static_cast<const T*>(a.q) + sg.b * a.q_seq + (tok0 + r / a.group) * a.q_tok + (sg.head * a.group + r % a.group) * a.q_head;
        f = DT<T>::to_f(row[d]) * a.scale_log2;
      }
      q_s[i] = f;
    }
    for (int r = tid; r < ROWS; r += TG_THREADS) {
      m_s[r] = -INFINITY;
      l_s[r] = 0.f;
      bits_s[r] = r < rows ? tree_bits(a, sq, sg.b, tok0 + r / a.group) : 0ull;
    }
    float acc[TASKS][4][4];
#pragma unroll
    for (int k = 0; k < TASKS; ++k)
#pragma unroll
      for (int i = 0; i < 16; ++i) acc[k][i / 4][i % 4] = 0.f;
    for (int t = sg.t0; t < sg.t1; ++t) {
      const int s0 = t * TG_KT, n = min(TG_KT, sq.keys - s0);  // n <= 0: a sequence without keys
      __syncthreads();
      constexpr int CV = 16 / static_cast<int>(sizeof(C));
      for (int i = tid; i < 2 * TG_KT * (vec ? hdp / CV : hdp); i += TG_THREADS) {
        const int per = vec ? hdp / CV : hdp;
        const int half = i / (TG_KT * per), j = (i / per) % TG_KT, o = i % per;
        const KvPtr<C>& c = half ? vc : kc;
        float* dst = half ? v_s + j * hdp : k_s + j * (hdp + 4);
        const float scale = STORE == STX_STORE_SAME || j >= n ? 1.f : c.srow(sg.b, sg.head)[s0 + j];
        if (vec) {  // hd is a multiple of CV
          uint4 w = make_uint4(0, 0, 0, 0);
          if (j < n) w = ld_cached16(c.row(sg.b, sg.head, s0 + j) + o * CV);
          const C* e = reinterpret_cast<const C*>(&w);
#pragma unroll
          for (int u = 0; u < CV; ++u) dst[o * CV + u] = held_value<T, STORE>(e[u], scale);
        } else {
          dst[o] = j < n && o < a.hd ? held_value<T, STORE>(c.row(sg.b, sg.head, s0 + j)[o], scale) : 0.f;
        }
      }
      __syncthreads();
      for (int task = tid; task < TG_KT * (ROWS / 4); task += TG_THREADS) {
        const int j = task % TG_KT, r0 = task / TG_KT * 4;
        float s[4] = {0.f, 0.f, 0.f, 0.f};
        for (int d = 0; d < hdp; d += 4) {
          const float4 k = *reinterpret_cast<const float4*>(k_s + j * (hdp + 4) + d);
#pragma unroll
          for (int r = 0; r < 4; ++r) {
            const float4 q = *reinterpret_cast<const float4*>(q_s + (r0 + r) * hdp + d);
            s[r] = fmaf(q.x, k.x, fmaf(q.y, k.y, fmaf(q.z, k.z, fmaf(q.w, k.w, s[r]))));
          }
        }
#pragma unroll
        for (int r = 0; r < 4; ++r) p_s[(r0 + r) * (TG_KT + 4) + j] = s[r];
      }
      __syncthreads();
      for (int r = warp; r < ROWS; r += TG_THREADS / 32) {
        const unsigned long long bits = bits_s[r];
        const bool row_used = r < rows && tok0 + r / a.group < sq.cnt;
        const bool see0 = row_used && lane < n && ((tree_visible(s0, sq.len, bits) >> lane) & 1u);
        const bool see1 = row_used && lane + 32 < n && ((tree_visible(s0 + 32, sq.len, bits) >> lane) & 1u);
        const float x0 = see0 ? p_s[r * (TG_KT + 4) + lane] : -INFINITY, x1 = see1 ? p_s[r * (TG_KT + 4) + lane + 32] : -INFINITY;
        const float old = m_s[r];
        float mx = fmaxf(old, fmaxf(x0, x1));
#pragma unroll
        for (int off = 16; off > 0; off >>= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, off));
        const float p0 = see0 ? exp2f(x0 - mx) : 0.f, p1 = see1 ? exp2f(x1 - mx) : 0.f;
        const float sum = warp_sum_xor(p0 + p1);
        p_s[r * (TG_KT + 4) + lane] = p0;
        p_s[r * (TG_KT + 4) + lane + 32] = p1;
        if (lane == 0) {
          const float f = old == mx ? 1.f : exp2f(old - mx);  // also where nothing has been seen yet
          m_s[r] = mx;
          l_s[r] = fmaf(l_s[r], f, sum);
          c_s[r] = f;
        }
      }
      __syncthreads();
#pragma unroll
      for (int k = 0; k < TASKS; ++k) {
        const int task = tid + k * TG_THREADS, d4 = task % d4n, r0 = task / d4n * 4;
        if (r0 >= ROWS) continue;
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          const float f = c_s[r0 + r];
#pragma unroll
          for (int e = 0; e < 4; ++e) acc[k][r][e] *= f;
        }
        for (int j = 0; j < n; ++j) {
          const float4 v = *reinterpret_cast<const float4*>(v_s + j * hdp + 4 * d4);
#pragma unroll
          for (int r = 0; r < 4; ++r) {
            const float p = p_s[(r0 + r) * (TG_KT + 4) + j];
            if (p != 0.f) {
              acc[k][r][0] = fmaf(p, v.x, acc[k][r][0]);
              acc[k][r][1] = fmaf(p, v.y, acc[k][r][1]);
              acc[k][r][2] = fmaf(p, v.z, acc[k][r][2]);
              acc[k][r][3] = fmaf(p, v.w, acc[k][r][3]);
            }
          }
        }
      }
    }
    const bool whole = sg.t0 == 0 && sg.t1 == sg.nt;
    const int slot = 2 * cta + (x == begin ? 0 : 1);
    float* po = tree_part_o(a, ROWS, slot);
#pragma unroll
    for (int k = 0; k < TASKS; ++k) {
      const int task = tid + k * TG_THREADS, d4 = task % d4n, r0 = task / d4n * 4;
      if (r0 >= ROWS) continue;
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        const int row = r0 + r;
        if (whole) {
          if (row >= rows) continue;
          const float l = l_s[row];
          T* dst = static_cast<T*>(a.out) + sg.b * a.o_seq + (tok0 + row / a.group) * a.o_tok + (sg.head * a.group + row % a.group) * a.o_head;
#pragma unroll
          for (int e = 0; e < 4; ++e)
            if (4 * d4 + e < a.hd) dst[4 * d4 + e] = DT<T>::from_f(m_s[row] == -INFINITY && l == 0.f ? 0.f : acc[k][r][e] / l);
        } else {
          *reinterpret_cast<float4*>(po + (static_cast<size_t>(d4) * ROWS + row) * 4) = make_float4(acc[k][r][0], acc[k][r][1], acc[k][r][2], acc[k][r][3]);
        }
      }
    }
    if (!whole) {
      float* ml = tree_part_ml(a, ROWS, slot);
      for (int r = tid; r < ROWS; r += TG_THREADS) {
        ml[r] = m_s[r];
        ml[ROWS + r] = l_s[r];
      }
    }
    x += sg.t1 - sg.t0;
  }
}

constexpr int TJ_THREADS = 256;

// Blocks (x, y): unit x, or, where there are more units than CTAs, the one that begins in CTA x's tiles and ends behind them.
//   o = sum_i 2^(m_i - M) o_i / sum_i 2^(m_i - M) l_i over the CTAs i = c, c + 1, .. that have a part of it
// An item is four values of a row; P threads (2, 4 or 8, as there are parts) take every P-th part of it, four loads in flight each, and their
// sums are added in thread order.  Lengths and counts are inputs of the launch before, which has waited for whoever wrote them, so the unit is found
// while that launch still runs; a block without one leaves at once, all but one, so that this launch does not end before the one before it.
// Bound by trips to memory (unit, then m and l, then the parts): about 4 us; the parts lie in the L2.
template <typename T, int ROWS>
__global__ void __launch_bounds__(TJ_THREADS) k_tree_join(const TreeArgs a, int kt, int by_unit) {
  __shared__ int pre[TREE_PRE];
  __shared__ float m_s[TJ_THREADS], l_s[TJ_THREADS];
  __shared__ float4 o_s[TJ_THREADS];
  tree_prefix(a, kt, pre);
  __syncthreads();
  const TreeLine line = tree_line(a, pre);
  int at = 0;  // a position of the line in the unit
  bool mine = true;
  if (by_unit) {
    const int b = blockIdx.x / line.per;
    at = pre[b] * line.per + (blockIdx.x - b * line.per) * (pre[b + 1] - pre[b]);
  } else {
    mine = static_cast<int>(blockIdx.x) + 1 < line.ctas;
    at = mine ? tree_begin(line, blockIdx.x + 1) - 1 : 0;
  }
  const TreeSeg sg = tree_seg(a, line, pre, at, at + 1);
  const int cta = tree_owner(line, sg.first), begin = tree_begin(line, cta), parts = tree_owner(line, sg.first + sg.nt - 1) - cta + 1;
  mine = mine && parts > 1 && (by_unit || cta == static_cast<int>(blockIdx.x));
  if (!mine && (blockIdx.x | blockIdx.y)) return;
  pdl_wait();
  pdl_launch_dependents();
  if (!mine) return;
  const int rows = min(a.tile_tok, a.n_tok - sg.rt * a.tile_tok) * a.group, items = rows * ((a.hd + 3) / 4);
  // CTA c ends with this unit: its first slot when the unit is all it has, else its second; those behind begin with it
  const int slot0 = 2 * cta + (sg.first == begin ? 0 : 1);
  const int P = parts <= 2 ? 2 : parts <= 4 ? 4 : 8, N = TJ_THREADS / P;
  const int x = threadIdx.x & (N - 1), y = threadIdx.x / N;
  for (int i0 = blockIdx.y * N; i0 < items; i0 += gridDim.y * N) {
    const int item = i0 + x, d4 = item / rows, row = item - d4 * rows;
    float M = -INFINITY, l = 0.f;
    float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
    if (item < items) {
      for (int p0 = y; p0 < parts; p0 += 4 * P) {
        float m[4], li[4];
        float4 v[4];
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          const int part = p0 + k * P, slot = part == 0 ? slot0 : 2 * (cta + part);
          m[k] = -INFINITY;
          li[k] = 0.f;
          v[k] = make_float4(0.f, 0.f, 0.f, 0.f);
          if (part < parts) {
            const float* ml = tree_part_ml(a, ROWS, slot);
            m[k] = __ldcg(ml + row);
            li[k] = __ldcg(ml + ROWS + row);
            v[k] = __ldcg(reinterpret_cast<const float4*>(tree_part_o(a, ROWS, slot) + (static_cast<size_t>(d4) * ROWS + row) * 4));
          }
        }
        const float up = fmaxf(M, fmaxf(fmaxf(m[0], m[1]), fmaxf(m[2], m[3])));
        const float f0 = M == up ? 1.f : exp2f(M - up);
        M = up;
        l *= f0, o.x *= f0, o.y *= f0, o.z *= f0, o.w *= f0;
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          const float f = m[k] == -INFINITY && li[k] == 0.f ? 0.f : exp2f(m[k] - M);  // a part that has seen nothing
          l = fmaf(li[k], f, l), o.x = fmaf(v[k].x, f, o.x), o.y = fmaf(v[k].y, f, o.y), o.z = fmaf(v[k].z, f, o.z), o.w = fmaf(v[k].w, f, o.w);
        }
      }
    }
    m_s[threadIdx.x] = M;
    l_s[threadIdx.x] = l;
    o_s[threadIdx.x] = o;
    __syncthreads();
    if (y == 0 && item < items) {
      float all = -INFINITY, sum = 0.f, r[4] = {0.f, 0.f, 0.f, 0.f};
      for (int k = 0; k < P; ++k) all = fmaxf(all, m_s[k * N + x]);
      for (int k = 0; k < P; ++k) {
        const float m = m_s[k * N + x], li = l_s[k * N + x], f = m == -INFINITY && li == 0.f ? 0.f : exp2f(m - all);
        const float4 v = o_s[k * N + x];
        sum = fmaf(li, f, sum);
        r[0] = fmaf(v.x, f, r[0]), r[1] = fmaf(v.y, f, r[1]), r[2] = fmaf(v.z, f, r[2]), r[3] = fmaf(v.w, f, r[3]);
      }
      const int tok = sg.rt * a.tile_tok + row / a.group;
      T* dst = static_cast<T*>(a.out) + sg.b * a.o_seq + tok * a.o_tok + (sg.head * a.group + row % a.group) * a.o_head + 4 * d4;
#pragma unroll
      for (int e = 0; e < 4; ++e)
        if (4 * d4 + e < a.hd) dst[e] = DT<T>::from_f(all == -INFINITY && sum == 0.f ? 0.f : r[e] / sum);
    }
    __syncthreads();
  }
}

int launch_tree_join(const TreeArgs& a, int rows, int kt, int dtype, cudaStream_t s) {
  const int64_t units = static_cast<int64_t>(a.n_seq) * a.nkv * a.row_tiles;
  const int by_unit = units <= a.grid;
  const int x = by_unit ? static_cast<int>(units) : a.grid;
  // about four blocks an SM in all, and none without an item
  const int items = a.tile_tok * a.group * ((a.hd + 3) / 4);
  const dim3 grid(static_cast<unsigned>(x), static_cast<unsigned>(std::max(1, std::min((items + 31) / 32, 4 * num_sms() / x))));
  return by_dtype(dtype, [&](auto tag) -> int {
    typedef decltype(tag) T;
    if (rows == 16) STX_CUDA(launch_pdl(k_tree_join<T, 16>, grid, dim3(TJ_THREADS), 0, s, a, kt, by_unit));
    else if (rows == 64) STX_CUDA(launch_pdl(k_tree_join<T, 64>, grid, dim3(TJ_THREADS), 0, s, a, kt, by_unit));
    else STX_CUDA(launch_pdl(k_tree_join<T, 128>, grid, dim3(TJ_THREADS), 0, s, a, kt, by_unit));
    return STX_OK;
  });
}

template <typename T, int STORE, int ROWS, int TASKS>
static int launch_any(TreeArgs a, const stx_kv* c, cudaStream_t s) {
  typedef typename Held<T, STORE>::C C;
  const KvPtr<C> kc = kv_ptr<C>(c, false), vc = kv_ptr<C>(c, true);
  constexpr int CV = 16 / static_cast<int>(sizeof(C));
  auto ok = [&](const KvPtr<C>& p) {
    return (reinterpret_cast<uintptr_t>(p.data) & 15) == 0 && p.seq % CV == 0 && p.head % CV == 0 && p.slot % CV == 0;
  };
  const int vec = a.hd % CV == 0 && ok(kc) && ok(vc);
  const int hdp = (a.hd + 3) / 4 * 4;
  const size_t smem = sizeof(float) * (ROWS * hdp + TG_KT * (hdp + 4) + TG_KT * hdp + ROWS * (TG_KT + 4) + 3 * ROWS);
  static bool attr_set[64] = {};
  int dev = 0;
  STX_CUDA(cudaGetDevice(&dev));
  if (dev < 0 || dev >= 64 || !attr_set[dev]) {
    const int most = static_cast<int>(sizeof(float) * (ROWS * 256 + TG_KT * 260 + TG_KT * 256 + ROWS * (TG_KT + 4) + 3 * ROWS));
    STX_CUDA(cudaFuncSetAttribute(k_tree_attn_any<T, STORE, ROWS, TASKS>, cudaFuncAttributeMaxDynamicSharedMemorySize, most));
    if (dev >= 0 && dev < 64) attr_set[dev] = true;
  }
  STX_CUDA(launch_pdl(k_tree_attn_any<T, STORE, ROWS, TASKS>, dim3(static_cast<unsigned>(a.grid)), dim3(TG_THREADS), smem, s, a, kc, vc, vec));
  return launch_tree_join(a, ROWS, TG_KT, c->dtype, s);
}

}  // namespace stx

using namespace stx;

static int check_tree(int64_t n_tokens, int n_heads, int n_kv_heads, int head_dim) {
  STX_CHECK_ARG(n_tokens > 0 && n_tokens <= STX_DRAFT_MAX, "stx_tree_attention: a draft of %lld nodes is outside 1..%d",
                static_cast<long long>(n_tokens), STX_DRAFT_MAX);
  STX_CHECK_ARG(n_heads > 0 && n_kv_heads > 0 && n_heads % n_kv_heads == 0, "stx_tree_attention: %d query heads do not divide into %d key/value heads",
                n_heads, n_kv_heads);
  STX_CHECK_ARG(n_heads / n_kv_heads <= 64, "stx_tree_attention: %d query heads to a cache head, 64 at most", n_heads / n_kv_heads);
  STX_CHECK_ARG(head_dim > 0 && head_dim <= 256 && head_dim % 8 == 0, "stx_tree_attention: head_dim %d is not a multiple of 8 in 8..256", head_dim);
  return STX_OK;
}

extern "C" {

// Room for whichever kernel runs: 2 CTAs an SM of 64 rows or one of 128.
int stx_tree_attention_workspace_bytes(int64_t n_tokens, int n_heads, int n_kv_heads, int head_dim, int dtype, size_t* bytes_out) {
  STX_CHECK_ARG(bytes_out, "stx_tree_attention_workspace_bytes: null pointer");
  const int rc = check_tree(n_tokens, n_heads, n_kv_heads, head_dim);
  if (rc != STX_OK) return rc;
  STX_CHECK_ARG(dtype == STX_F32 || dtype == STX_F16 || dtype == STX_BF16, "stx_tree_attention_workspace_bytes: bad dtype %d", dtype);
  *bytes_out = sizeof(float) * tree_part_floats(num_sms(), 128, head_dim);
  return STX_OK;
}

int stx_tree_attention(const stx_kv* cache, const stx_heads* q, const stx_heads* out, int64_t n_tokens, int n_heads, float scale,
                       const int64_t* length, const int64_t* counts, const int64_t* masks, int64_t mask_stride, void* workspace,
                       void* stream) {
  int rc = check_kv(cache, "stx_tree_attention");
  if (rc == STX_OK) rc = check_heads(q, "stx_tree_attention", "q");
  if (rc == STX_OK) rc = check_heads(out, "stx_tree_attention", "out");
  if (rc != STX_OK) return rc;
  STX_CHECK_ARG(length && workspace, "stx_tree_attention: null pointer");
  STX_CHECK_ARG((reinterpret_cast<uintptr_t>(workspace) & 15) == 0, "stx_tree_attention: workspace must be 16-byte aligned");
  if ((rc = check_tree(n_tokens, n_heads, cache->n_kv_heads, cache->head_dim)) != STX_OK) return rc;
  const int group = n_heads / cache->n_kv_heads;
  STX_CHECK_ARG(cache->n_seq <= TREE_MAX_SEQ, "stx_tree_attention: %d sequences, %d at most", cache->n_seq, TREE_MAX_SEQ);
  STX_CHECK_ARG(cache->store == STX_STORE_SAME || cache->head_dim % 16 == 0, "stx_tree_attention: head_dim %d of an 8-bit cache is not a multiple of 16",
                cache->head_dim);
  STX_CHECK_ARG(std::isfinite(scale) && mask_stride >= 0, "stx_tree_attention: bad scale or mask stride");
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  TreeArgs a{};
  a.q = q->data;
  a.out = out->data;
  a.q_seq = q->seq_stride, a.q_tok = q->token_stride, a.q_head = q->head_stride;
  a.o_seq = out->seq_stride, a.o_tok = out->token_stride, a.o_head = out->head_stride;
  a.length = length;
  a.counts = counts;
  a.masks = masks;
  a.mask_stride = mask_stride;
  a.max_len = cache->max_len;
  a.scale_log2 = scale * 1.4426950408889634f;
  a.n_seq = cache->n_seq;
  a.n_tok = static_cast<int>(n_tokens);
  a.nkv = cache->n_kv_heads;
  a.group = group;
  a.hd = cache->head_dim;
  a.part = static_cast<float*>(workspace);
  // the line of tiles is counted in 32 bits; a cache that fits a device is far below
  STX_CHECK_ARG(static_cast<double>(cache->n_seq) * cache->n_kv_heads * n_tokens * (static_cast<double>(cache->max_len) / 64 + 1) < 2147483648.0,
                "stx_tree_attention: n_seq * n_kv_heads * n_tokens * max_len is too large");
  if (tree_mma_wanted(cache)) return tree_mma(a, cache, s);
  const int rows = group * a.n_tok > 16 ? 64 : 16;  // 64 rows read a key four times less often, 16 leave fewer of them empty
  a.tile_tok = std::min(a.n_tok, rows / group);
  a.row_tiles = (a.n_tok + a.tile_tok - 1) / a.tile_tok;
  a.sms = num_sms();
  a.grid = a.sms * (rows == 16 ? 2 : 1);
  a.cut = a.join = a.join_one = 0;  // a tile (11 or 22 us at 128 values) takes longer than any of them
  return by_dtype(cache->dtype, [&](auto tag) -> int {
    typedef decltype(tag) T;
    return by_store(cache->store, [&](auto st) -> int {
      constexpr int S = decltype(st)::value;
      return rows == 16 ? launch_any<T, S, 16, 1>(a, cache, s) : launch_any<T, S, 64, 4>(a, cache, s);
    });
  });
}

int stx_tree_attention_status(int* status_out, void* stream) {
  STX_CHECK_ARG(status_out, "stx_tree_attention_status: null pointer");
  return tree_status(status_out, static_cast<cudaStream_t>(stream));
}

}  // extern "C"
