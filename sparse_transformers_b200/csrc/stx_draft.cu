// Verification of drafted tokens (C ABI: stx_verify_draft; include/stx.h has the rules).
//
// Speculative sampling keeps the target's distribution p: a token x drawn from q is accepted with probability min(1, p(x) / q(x)),
// a refused one replaced by a draw from max(p - q, 0) / sum.  For fixed candidates it is enough to draw from p and to see
// whether a candidate was drawn.
//
//   k_verify_walk   a cluster per sequence: the walk is a chain of draws, each one row of V floats (a drawn token's successor is
//                   known only when it is drawn), so what counts is how fast one row goes through.
//   k_verify_tokens a warp per sequence, where the target's tokens are given
//
// 32 chains of 6 nodes over 128256 tokens: 13.1 us for 33 MB (5 us at HBM's rate; the rest is the trip for tokens and thresholds, the row's sum,
// two cluster barriers and the search in one stretch).  With one block an SM the 256 blocks took two waves and 24 us.  A tree of 32 nodes, one
// sequence over 32000 tokens: 8.2 us, 2 us for each node of the path.
#include "stx_common.cuh"

#include <algorithm>

namespace stx {

constexpr int VF_THREADS = 512;
constexpr int VF_WARPS = VF_THREADS / 32;
constexpr int VF_CLUSTER = 8;
constexpr int VF_SEGS = VF_WARPS * VF_CLUSTER;  // warps of a cluster, each with a stretch of the row
constexpr int VF_ALONE_V = 8192;                // vocabularies up to this: one CTA, no cluster

__device__ __forceinline__ uint32_t vf_map(const void* p, uint32_t rank) {
  uint32_t a;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(a) : "r"(static_cast<uint32_t>(__cvta_generic_to_shared(p))), "r"(rank));
  return a;
}
__device__ __forceinline__ void vf_store_f64(uint32_t at, double v) { asm volatile("st.shared::cluster.f64 [%0], %1;" ::"r"(at), "d"(v) : "memory"); }
__device__ __forceinline__ void vf_store_s32(uint32_t at, int v) { asm volatile("st.shared::cluster.s32 [%0], %1;" ::"r"(at), "r"(v) : "memory"); }
__device__ __forceinline__ void vf_sync() {
  asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}

struct VerifyArgs {
  const int64_t *tokens, *parents, *counts;
  const float *p, *q, *u;
  int64_t n_tok, V;
  int64_t *path, *count, *next;
};

// What p has more than q; NaN stays NaN.
__device__ __forceinline__ double vf_more(float p, float q) {
  const double d = static_cast<double>(p) - static_cast<double>(q);
  return d < 0.0 ? 0.0 : d;
}

// A row's entries [lo, hi) of a warp, 128 at a time: f(w) with lane l's four weights (entries 4 l .. 4 l + 3 of the 128; zeros
// behind hi).  Returns early when f says so.
template <int AHEAD, typename F>
__device__ __forceinline__ void vf_walk(const float* p, const float* q, int64_t lo, int64_t hi, bool vec, int lane, F f) {
  for (int64_t j0 = lo; j0 < hi; j0 += 128 * AHEAD) {
    float x[AHEAD][4], y[AHEAD][4];
#pragma unroll
    for (int k = 0; k < AHEAD; ++k) {
      const int64_t j = j0 + 128 * k + 4 * lane;
#pragma unroll
      for (int e = 0; e < 4; ++e) x[k][e] = y[k][e] = 0.f;
      if (vec && j + 4 <= hi) {
        const float4 v = *reinterpret_cast<const float4*>(p + j);
        x[k][0] = v.x, x[k][1] = v.y, x[k][2] = v.z, x[k][3] = v.w;
        if (q) {
          const float4 z = *reinterpret_cast<const float4*>(q + j);
          y[k][0] = z.x, y[k][1] = z.y, y[k][2] = z.z, y[k][3] = z.w;
        }
      } else {
#pragma unroll
        for (int e = 0; e < 4; ++e)
          if (j + e < hi) {
            x[k][e] = p[j + e];
            if (q) y[k][e] = q[j + e];
          }
      }
    }
#pragma unroll
    for (int k = 0; k < AHEAD; ++k) {
      double w[4];
#pragma unroll
      for (int e = 0; e < 4; ++e) w[e] = q ? vf_more(x[k][e], y[k][e]) : static_cast<double>(x[k][e]);
      if (j0 + 128 * k < hi && f(j0 + 128 * k, w)) return;
    }
  }
}

__global__ void __launch_bounds__(VF_THREADS, 2) k_verify_walk(const VerifyArgs a, int seg, int vec) {
  __shared__ double tot_s[2][VF_SEGS];  // sums of the cluster's stretches, two draws in turn
  __shared__ int tok_s[2];
  __shared__ int64_t x_s[STX_DRAFT_MAX], par_s[STX_DRAFT_MAX];
  __shared__ int taken_s[STX_DRAFT_MAX];
  uint32_t rank, ranks;
  asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(rank));
  asm volatile("mov.u32 %0, %%cluster_nctarank;" : "=r"(ranks));
  const int64_t b = blockIdx.x / ranks;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  pdl_wait();
  pdl_launch_dependents();
  const int n = static_cast<int>(a.counts ? max(0ll, min(static_cast<long long>(a.n_tok), static_cast<long long>(a.counts[b]))) : a.n_tok);
  const int64_t at = b * a.n_tok;
  for (int i = tid; i < a.n_tok; i += VF_THREADS) {
    x_s[i] = a.tokens[at + i];
    par_s[i] = a.parents ? a.parents[at + i] : i - 1;
    int ok = 0;
    if (a.q && i > 0 && i < n && x_s[i] >= 0 && x_s[i] < a.V) {
      const int64_t row = b * (a.n_tok - 1) + i - 1;
      ok = static_cast<double>(a.u[at + i]) * static_cast<double>(a.q[row * a.V + x_s[i]]) < static_cast<double>(a.p[(at + i - 1) * a.V + x_s[i]]);
    }
    taken_s[i] = ok;
  }
  for (int i = tid; i < 2 * VF_SEGS; i += VF_THREADS) (&tot_s[0][0])[i] = 0.0;
  __syncthreads();
  vf_sync();  // every CTA's sums are zero before the first of them arrives
  int len = n > 0 ? 1 : 0, v = 0;  // nodes taken, the last of them
  uint64_t nodes = 1;                         // the nodes taken, as bits
  if (a.q && n > 0) {
    while (v + 1 < n && taken_s[v + 1]) ++v;
    len = v + 1;
    nodes = ~0ull >> (63 - v);
  }
  int64_t next = -1;
  if (n > 0) {
    bool less = a.q && v + 1 < n;  // draw from what the target has more than the draft
    const int64_t lo = static_cast<int64_t>(rank * VF_WARPS + warp) * seg, hi = min(static_cast<long long>(a.V), static_cast<long long>(lo + seg));
    for (int turn = 0;; ++turn) {
      const float* p = a.p + (at + v) * a.V;
      const float* q = less ? a.q + (b * (a.n_tok - 1) + v) * a.V : nullptr;
      double own = 0.0;
      vf_walk<4>(p, q, lo, hi, vec, lane, [&](int64_t, const double(&w)[4]) {
        own += (w[0] + w[1]) + (w[2] + w[3]);
        return false;
      });
#pragma unroll
      for (int off = 16; off > 0; off >>= 1) own += __shfl_xor_sync(0xffffffffu, own, off);
      double* tot = tot_s[turn & 1];
      if (lane < static_cast<int>(ranks)) vf_store_f64(vf_map(&tot[rank * VF_WARPS + warp], lane), own);
      vf_sync();
      // every warp finds the stretch for itself: lane l has stretches 4 l .. 4 l + 3
      double t[4], sum = 0.0;
#pragma unroll
      for (int e = 0; e < 4; ++e) sum += t[e] = tot[4 * lane + e];
      double run = sum;
#pragma unroll
      for (int off = 1; off < 32; off <<= 1) {
        const double o = __shfl_up_sync(0xffffffffu, run, off);
        if (lane >= off) run += o;
      }
      const double whole = __shfl_sync(0xffffffffu, run, 31);
      if (!(whole > 0.0) || isinf(whole)) {
        if (less && whole == 0.0) {  // target and draft are the same: draw from the target
          less = false;
          continue;
        }
        next = -1;
        break;
      }
      const double aim = static_cast<double>(a.u[at + (a.q ? 0 : v)]) * whole;
      double before = run - sum, first = 0.0;
      int mine = -1, some = -1;  // the stretch whose running sum passes the aim; the last one of any weight
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        if (mine < 0 && before + t[e] > aim) {
          mine = 4 * lane + e;
          first = before;
        }
        if (t[e] > 0.0) some = 4 * lane + e;
        before += t[e];
      }
      const uint32_t has = __ballot_sync(0xffffffffu, mine >= 0);
      int stretch;
      if (has) {
        const int who = __ffs(has) - 1;
        stretch = __shfl_sync(0xffffffffu, mine, who);
        first = __shfl_sync(0xffffffffu, first, who);
      } else {
        stretch = __reduce_max_sync(0xffffffffu, some);
        first = aim;  // nothing passes it any more: the stretch's last entry of any weight
      }
      if (stretch == static_cast<int>(rank) * VF_WARPS + warp) {
        int found = -1, last = -1;
        double base = first;
        vf_walk<4>(p, q, lo, hi, vec, lane, [&](int64_t j0, const double(&w)[4]) {
          const double s4 = (w[0] + w[1]) + (w[2] + w[3]);
          double r = s4;
#pragma unroll
          for (int off = 1; off < 32; off <<= 1) {
            const double o = __shfl_up_sync(0xffffffffu, r, off);
            if (lane >= off) r += o;
          }
          double run4 = base + (r - s4);
          int hit = -1, any = -1;
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            run4 += w[e];
            if (hit < 0 && w[e] > 0.0 && run4 > aim) hit = static_cast<int>(j0) + 4 * lane + e;
            if (w[e] > 0.0) any = static_cast<int>(j0) + 4 * lane + e;
          }
          const uint32_t hits = __ballot_sync(0xffffffffu, hit >= 0);
          last = max(last, __reduce_max_sync(0xffffffffu, any));
          if (has && hits) {
            found = __shfl_sync(0xffffffffu, hit, __ffs(hits) - 1);
            return true;
          }
          base += __shfl_sync(0xffffffffu, r, 31);
          return false;
        });
        if (found < 0) found = last;
        if (lane < static_cast<int>(ranks)) vf_store_s32(vf_map(&tok_s[turn & 1], lane), found);
      }
      vf_sync();
      next = tok_s[turn & 1];
      if (a.q) break;
      // the child that carries the token, the lowest of equal ones
      uint32_t hit0 = __ballot_sync(0xffffffffu, lane > v && lane < n && par_s[lane < n ? lane : 0] == v && x_s[lane < n ? lane : 0] == next);
      uint32_t hit1 = __ballot_sync(0xffffffffu, lane + 32 > v && lane + 32 < n && par_s[lane + 32 < n ? lane + 32 : 0] == v && x_s[lane + 32 < n ? lane + 32 : 0] == next);
      const int child = hit0 ? __ffs(hit0) - 1 : hit1 ? 31 + __ffs(hit1) : -1;
      if (child < 0) break;
      v = child;
      nodes |= 1ull << v;
      ++len;
    }
  }
  vf_sync();  // no CTA leaves while another still writes to it
  if (rank == 0 && warp == 0) {
    for (int i = lane; i < a.n_tok; i += 32) a.path[at + i] = -1;
    __syncwarp();
    if (n > 0)
      for (int i = lane; i < 64; i += 32)
        if ((nodes >> i) & 1) a.path[at + __popcll(nodes & ((1ull << i) - 1))] = i;
    if (lane == 0) {
      a.count[b] = len;
      a.next[b] = next;
    }
  }
}

__global__ void __launch_bounds__(32) k_verify_tokens(const VerifyArgs a, const int64_t* __restrict__ target) {
  __shared__ int64_t x_s[STX_DRAFT_MAX], par_s[STX_DRAFT_MAX], t_s[STX_DRAFT_MAX];
  const int64_t b = blockIdx.x, at = b * a.n_tok;
  const int lane = threadIdx.x;
  pdl_wait();
  pdl_launch_dependents();
  const int n = static_cast<int>(a.counts ? max(0ll, min(static_cast<long long>(a.n_tok), static_cast<long long>(a.counts[b]))) : a.n_tok);
  for (int i = lane; i < a.n_tok; i += 32) {
    x_s[i] = a.tokens[at + i];
    par_s[i] = a.parents ? a.parents[at + i] : i - 1;
    t_s[i] = target[at + i];
  }
  __syncwarp();
  int v = 0, len = 0;
  int64_t next = -1;
  uint64_t nodes = 0;
  if (n > 0) {
    for (;;) {
      nodes |= 1ull << v;
      ++len;
      next = t_s[v];
      const uint32_t hit0 = __ballot_sync(0xffffffffu, lane > v && lane < n && par_s[lane] == v && x_s[lane] == next);
      const uint32_t hit1 = __ballot_sync(0xffffffffu, lane + 32 > v && lane + 32 < n && par_s[lane + 32] == v && x_s[lane + 32] == next);
      const int child = hit0 ? __ffs(hit0) - 1 : hit1 ? 31 + __ffs(hit1) : -1;
      if (child < 0) break;
      v = child;
    }
  }
  for (int i = lane; i < a.n_tok; i += 32) a.path[at + i] = -1;
  __syncwarp();
  for (int i = lane; i < 64; i += 32)
    if ((nodes >> i) & 1) a.path[at + __popcll(nodes & ((1ull << i) - 1))] = i;
  if (lane == 0) {
    a.count[b] = len;
    a.next[b] = next;
  }
}

}  // namespace stx

using namespace stx;

extern "C" {

int stx_verify_draft(const int64_t* tokens, const int64_t* parents, const float* target_probs, const int64_t* target_tokens,
                     const float* draft_probs, const float* uniform, const int64_t* counts, int64_t n_seq, int64_t n_tokens,
                     int64_t V, int64_t* path, int64_t* count, int64_t* next, void* stream) {
  STX_CHECK_ARG(tokens && path && count && next, "stx_verify_draft: null pointer");
  STX_CHECK_ARG((target_probs != nullptr) != (target_tokens != nullptr), "stx_verify_draft: give target_probs or target_tokens, one of them");
  STX_CHECK_ARG(n_tokens > 0 && n_tokens <= STX_DRAFT_MAX, "stx_verify_draft: a draft of %lld nodes is outside 1..%d", static_cast<long long>(n_tokens), STX_DRAFT_MAX);
  STX_CHECK_ARG(n_seq >= 0 && n_seq < (1ll << 27), "stx_verify_draft: bad n_seq");
  VerifyArgs a{};
  a.tokens = tokens;
  a.parents = parents;
  a.counts = counts;
  a.p = target_probs;
  a.q = n_tokens > 1 ? draft_probs : nullptr;  // a lone root has no draft row; its draw is the same
  a.u = uniform;
  a.n_tok = n_tokens;
  a.V = V;
  a.path = path;
  a.count = count;
  a.next = next;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  if (target_tokens) {
    STX_CHECK_ARG(!draft_probs && !uniform, "stx_verify_draft: target_tokens take neither draft_probs nor uniform");
    if (n_seq == 0) return STX_OK;
    STX_CUDA(launch_pdl(k_verify_tokens, dim3(static_cast<unsigned>(n_seq)), dim3(32), 0, s, a, target_tokens));
    return STX_OK;
  }
  STX_CHECK_ARG(uniform, "stx_verify_draft: target_probs need uniform");
  STX_CHECK_ARG(V > 0 && V <= STX_VERIFY_MAX_VOCAB, "stx_verify_draft: V=%lld outside 1..%d", static_cast<long long>(V), STX_VERIFY_MAX_VOCAB);
  STX_CHECK_ARG(!draft_probs || !parents, "stx_verify_draft: draft_probs belong to a chain: parents must be null");
  if (n_seq == 0) return STX_OK;
  const int ranks = V <= VF_ALONE_V ? 1 : VF_CLUSTER;
  const int64_t segs = static_cast<int64_t>(ranks) * VF_WARPS;
  const int seg = static_cast<int>(((V + segs - 1) / segs + 127) / 128 * 128);
  const int vec = V % 4 == 0 && ((reinterpret_cast<uintptr_t>(target_probs) | reinterpret_cast<uintptr_t>(draft_probs)) & 15) == 0;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(static_cast<unsigned>(n_seq * ranks));
  cfg.blockDim = dim3(VF_THREADS);
  cfg.stream = s;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  attr[1].id = cudaLaunchAttributeClusterDimension;
  attr[1].val.clusterDim.x = static_cast<unsigned>(ranks);
  attr[1].val.clusterDim.y = attr[1].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 2;
  STX_CUDA(cudaLaunchKernelEx(&cfg, k_verify_walk, a, seg, vec));
  return STX_OK;
}

}  // extern "C"
