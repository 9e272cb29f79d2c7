// PyTorch face of the operators for decoding from drafted tokens (include/stx.h: stx_rope .. stx_verify_draft).  Checks
// shapes, types, devices and strides, allocates results and workspaces from torch's allocator on the current stream (so that
// two streams or two captured graphs never share a workspace) and forwards to the C ABI.  No CPU implementation.
#include <torch/script.h>

#include <ATen/MemoryOverlap.h>
#include <ATen/cuda/CUDAContext.h>
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>

#include <optional>
#include <tuple>

#include "stx.h"

namespace stxb {

using torch::Tensor;
typedef std::optional<Tensor> MaybeTensor;

static void ok(int rc, const char* where) {
  if (rc == STX_OK) return;
  const char* msg = stx_last_error();
  TORCH_CHECK(false, (msg && *msg) ? msg : stx_status_string(rc), " [", where, "]");
}
static int dtype_of(const Tensor& t, const char* who) {
  switch (t.scalar_type()) {
    case c10::kFloat: return STX_F32;
    case c10::kHalf: return STX_F16;
    case c10::kBFloat16: return STX_BF16;
    default: TORCH_CHECK(false, who, ": unsupported dtype ", t.scalar_type(), " (float32, float16, bfloat16)");
  }
  return -1;
}
static void* stream_of(const c10::Device& d) { return static_cast<void*>(c10::cuda::getCurrentCUDAStream(d.index()).stream()); }

static void on_cuda(const Tensor& t, const char* who, const char* name) {
  TORCH_CHECK(t.is_cuda(), who, ": this build runs on CUDA only (", name, " is on ", t.device(), ")");
}
static void on(const c10::Device& d, const Tensor& t, const char* who, const char* name) {
  on_cuda(t, who, name);
  TORCH_CHECK(t.device() == d, who, ": ", name, " is on ", t.device(), ", not on ", d);
}
// These operators have no gradient; silently detaching a tensor that wants one would be worse than refusing it.
static void no_grad(const Tensor& t, const char* who, const char* name) {
  TORCH_CHECK(!(at::GradMode::is_enabled() && t.requires_grad()), who, ": has no gradient, but ", name,
              " requires one (call it under torch.no_grad())");
}
// Where it can be told: memory that a call writes may not be other memory that it reads or writes.  (Views with gaps, as the parts
// of a projection's block are, cannot be told apart but by their first element.)
static void apart(const Tensor& a, const Tensor& b, const char* who, const char* what) {
  if (a.numel() == 0 || b.numel() == 0) return;
  const auto lap = at::get_overlap_status(a, b);
  TORCH_CHECK(lap != at::MemOverlapStatus::Full && lap != at::MemOverlapStatus::Partial && a.data_ptr() != b.data_ptr(), who, ": ", what, " overlap");
}
// The caller's tensor has been written: what autograd saved of it is stale.
static void written(const Tensor& t) {
  if (!t.is_inference()) t.unsafeGetTensorImpl()->bump_version();
}
static void written(const MaybeTensor& t) {
  if (t) written(*t);
}
// int64 of exactly this shape, rows contiguous; returns the row stride (0 for a single row or an expanded one).
static int64_t index_rows(const c10::Device& d, const Tensor& t, at::IntArrayRef shape, const char* who, const char* name) {
  on(d, t, who, name);
  TORCH_CHECK(t.scalar_type() == c10::kLong, who, ": ", name, " must be int64");
  TORCH_CHECK(t.sizes() == shape, who, ": ", name, " must have the shape ", shape, ", not ", t.sizes());
  TORCH_CHECK(t.size(-1) <= 1 || t.stride(-1) == 1, who, ": the last dimension of ", name, " must be contiguous");
  return t.dim() < 2 || t.size(0) <= 1 ? 0 : t.stride(0);
}
static const int64_t* index_of(const c10::Device& d, const Tensor& t, int64_t n, const char* who, const char* name) {
  index_rows(d, t, {n}, who, name);
  return t.data_ptr<int64_t>();
}
static const int64_t* maybe_index(const c10::Device& d, const MaybeTensor& t, int64_t n, const char* who, const char* name) {
  return t ? index_of(d, *t, n, who, name) : nullptr;
}
static stx_heads heads_of(const Tensor& t, const char* who, const char* name) {
  TORCH_CHECK(t.dim() == 4, who, ": ", name, " must be [n_seq, n_tokens, heads, head_dim]");
  TORCH_CHECK(t.size(3) <= 1 || t.stride(3) == 1, who, ": the last dimension of ", name, " must be contiguous");
  return {t.data_ptr(), t.stride(0), t.stride(1), t.stride(2)};
}

static stx_kv kv_of(const Tensor& k, const Tensor& v, const MaybeTensor& ks, const MaybeTensor& vs, int dtype, bool written, const char* who) {
  on_cuda(k, who, "the cache");
  const auto d = k.device();
  on(d, v, who, "the cache's v");
  TORCH_CHECK(k.dim() == 4 && k.sizes() == v.sizes() && k.scalar_type() == v.scalar_type(), who,
              ": k and v of the cache must be [n_seq, n_kv_heads, max_len, head_dim] of one type");
  no_grad(k, who, "the cache");
  no_grad(v, who, "the cache");
  stx_kv c{};
  c.dtype = dtype;
  if (k.scalar_type() == c10::kChar) c.store = STX_STORE_INT8;
  else if (k.scalar_type() == c10::kFloat8_e4m3fn) c.store = STX_STORE_E4M3;
  else {
    TORCH_CHECK(dtype_of(k, who) == dtype, who, ": the cache holds ", k.scalar_type(), ", the other tensors do not");
    c.store = STX_STORE_SAME;
  }
  for (int i = 0; i < 4; ++i) TORCH_CHECK(k.size(i) <= 1 || k.stride(i) == v.stride(i), who, ": k and v of the cache must have the same strides");
  TORCH_CHECK(k.size(3) <= 1 || k.stride(3) == 1, who, ": head_dim of the cache must be contiguous");
  if (written) {
    at::assert_no_internal_overlap(k);
    at::assert_no_internal_overlap(v);
    apart(k, v, who, "k and v of the cache");
  }
  c.k = k.data_ptr();
  c.v = v.data_ptr();
  c.n_seq = static_cast<int>(k.size(0));
  c.n_kv_heads = static_cast<int>(k.size(1));
  c.max_len = k.size(2);
  c.head_dim = static_cast<int>(k.size(3));
  c.seq_stride = c.n_seq > 1 ? k.stride(0) : 0;
  c.head_stride = c.n_kv_heads > 1 ? k.stride(1) : 0;
  c.slot_stride = c.max_len > 1 ? k.stride(2) : c.head_dim;
  TORCH_CHECK((c.store != STX_STORE_SAME) == ks.has_value() && ks.has_value() == vs.has_value(), who,
              ": an 8-bit cache has k_scale and v_scale, another one has none");
  if (ks) {
    for (const Tensor* t : {&*ks, &*vs}) {
      on(d, *t, who, "a scale");
      no_grad(*t, who, "a scale");
      TORCH_CHECK(t->scalar_type() == c10::kFloat && t->dim() == 3 && t->sizes() == k.sizes().slice(0, 3) &&
                      (t->size(2) <= 1 || t->stride(2) == 1),
                  who, ": scales must be float32 [n_seq, n_kv_heads, max_len] with contiguous slots");
    }
    for (int i = 0; i < 2; ++i) TORCH_CHECK(ks->size(i) <= 1 || ks->stride(i) == vs->stride(i), who, ": k_scale and v_scale must have the same strides");
    if (written) {
      at::assert_no_internal_overlap(*ks);
      at::assert_no_internal_overlap(*vs);
      apart(*ks, *vs, who, "k_scale and v_scale");
    }
    c.k_scale = ks->data_ptr<float>();
    c.v_scale = vs->data_ptr<float>();
    c.scale_seq_stride = c.n_seq > 1 ? ks->stride(0) : 0;
    c.scale_head_stride = c.n_kv_heads > 1 ? ks->stride(1) : 0;
  }
  return c;
}

static stx_rotary rotary_of(const c10::Device& d, const Tensor& turns, bool interleaved, double factor, const char* who) {
  on(d, turns, who, "the rotary plan");
  TORCH_CHECK(turns.scalar_type() == c10::kDouble && turns.dim() == 1 && turns.is_contiguous(), who, ": turns must be float64 [rotary_dim / 2]");
  return {turns.data_ptr<double>(), static_cast<int>(2 * turns.size(0)), interleaved, factor};
}

// x [n, heads, hd] or [b, t, heads, hd], positions x.shape[:-2]
static Tensor rope(const Tensor& x, const Tensor& positions, const Tensor& turns, bool interleaved, double factor, bool inverse, const MaybeTensor& out) {
  constexpr const char* who = "rope";
  on_cuda(x, who, "x");
  no_grad(x, who, "x");
  TORCH_CHECK(x.dim() == 3 || x.dim() == 4, who, ": x must be [n, heads, head_dim] or [n_seq, n_tokens, heads, head_dim]");
  const int dt = dtype_of(x, who);
  c10::cuda::CUDAGuard guard(x.device());
  const int64_t pstride = index_rows(x.device(), positions, x.sizes().slice(0, x.dim() - 2), who, "positions");
  const stx_rotary rot = rotary_of(x.device(), turns, interleaved, factor, who);
  Tensor y = out ? *out : torch::empty(x.sizes(), x.options().requires_grad(false));
  if (out) {
    on(x.device(), y, who, "out");
    no_grad(y, who, "out");
    TORCH_CHECK(y.scalar_type() == x.scalar_type() && y.sizes() == x.sizes(), who, ": out must have x's shape and dtype");
    at::assert_no_internal_overlap(y);
    at::assert_no_partial_overlap(y, x);
    TORCH_CHECK(y.data_ptr() != x.data_ptr() || y.strides() == x.strides(), who, ": out may be x, not x in another order");
  }
  const Tensor x4 = x.dim() == 4 ? x : x.unsqueeze(0), y4 = x.dim() == 4 ? y : y.unsqueeze(0);
  const stx_heads hx = heads_of(x4, who, "x"), hy = heads_of(y4, who, "out");
  if (x.numel() == 0) return y;
  ok(stx_rope(&hx, &hy, x4.size(0), x4.size(1), static_cast<int>(x4.size(2)), static_cast<int>(x4.size(3)), positions.data_ptr<int64_t>(), pstride,
              &rot, inverse, dt, stream_of(x.device())),
     who);
  if (out) written(*out);
  return y;
}
static Tensor rope_new(const Tensor& x, const Tensor& positions, const Tensor& turns, bool interleaved, double factor, bool inverse) {
  return rope(x, positions, turns, interleaved, factor, inverse, MaybeTensor());
}
static Tensor rope_out(const Tensor& x, const Tensor& positions, const Tensor& turns, bool interleaved, double factor, bool inverse, const Tensor& out) {
  return rope(x, positions, turns, interleaved, factor, inverse, out);
}

static MaybeTensor kv_append(const Tensor& kc, const Tensor& vc, const MaybeTensor& ks, const MaybeTensor& vs, const Tensor& k, const Tensor& v,
                      const Tensor& start, const MaybeTensor& counts, const MaybeTensor& turns, bool interleaved, double factor,
                      const MaybeTensor& positions, const MaybeTensor& q, const MaybeTensor& q_out) {
  constexpr const char* who = "kv_append";
  on_cuda(k, who, "k");
  const auto d = k.device();
  const stx_kv c = kv_of(kc, vc, ks, vs, dtype_of(k, who), true, who);
  on(d, kc, who, "the cache");
  on(d, v, who, "v");
  no_grad(k, who, "k");
  no_grad(v, who, "v");
  TORCH_CHECK(v.scalar_type() == k.scalar_type() && k.sizes() == v.sizes() && k.dim() == 4, who, ": k and v must be [n_seq, n_tokens, n_kv_heads, head_dim] of one type");
  TORCH_CHECK(k.size(0) == c.n_seq && k.size(2) == c.n_kv_heads && k.size(3) == c.head_dim, who, ": k and v do not fit the cache");
  for (const Tensor* t : {&k, &v}) {
    apart(kc, *t, who, "the cache and the rows to be written");
    apart(vc, *t, who, "the cache and the rows to be written");
  }
  if (q) {
    apart(kc, *q, who, "the cache and q");
    apart(vc, *q, who, "the cache and q");
  }
  c10::cuda::CUDAGuard guard(d);
  const int64_t B = k.size(0), T = k.size(1);
  const stx_heads hk = heads_of(k, who, "k"), hv = heads_of(v, who, "v");
  stx_heads hq{}, ho{};
  MaybeTensor y;
  int nh = 0;
  if (q) {
    on(d, *q, who, "q");
    no_grad(*q, who, "q");
    TORCH_CHECK(q->scalar_type() == k.scalar_type() && q->dim() == 4 && q->size(0) == B && q->size(1) == T && q->size(3) == c.head_dim, who,
                ": q must be [n_seq, n_tokens, heads, head_dim] of k's type");
    nh = static_cast<int>(q->size(2));
    TORCH_CHECK(nh > 0, who, ": q has no heads");
    y = q_out ? *q_out : torch::empty(q->sizes(), q->options().requires_grad(false));
    if (q_out) {
      on(d, *y, who, "q_out");
      no_grad(*y, who, "q_out");
      for (const Tensor* t : {&k, &v, &kc, &vc}) apart(*y, *t, who, "q_out and what else the call reads or writes");
      TORCH_CHECK(y->scalar_type() == q->scalar_type() && y->sizes() == q->sizes(), who, ": q_out must have q's shape and dtype");
      at::assert_no_internal_overlap(*y);
      at::assert_no_partial_overlap(*y, *q);
      TORCH_CHECK(y->data_ptr() != q->data_ptr() || y->strides() == q->strides(), who, ": q_out may be q, not q in another order");
    }
    hq = heads_of(*q, who, "q");
    ho = heads_of(*y, who, "q_out");
  } else {
    TORCH_CHECK(!q_out, who, ": q_out without q");
  }
  stx_rotary rot{};
  if (turns) rot = rotary_of(d, *turns, interleaved, factor, who);
  const int64_t pstride = positions ? index_rows(d, *positions, {B, T}, who, "positions") : 0;
  const int64_t* st = index_of(d, start, B, who, "start");
  const int64_t* cn = maybe_index(d, counts, B, who, "counts");
  if (T == 0) return y;
  ok(stx_kv_append(&c, &hk, &hv, T, st, cn, turns ? &rot : nullptr, positions ? positions->data_ptr<int64_t>() : nullptr, pstride,
                   q ? &hq : nullptr, q ? &ho : nullptr, nh, stream_of(d)),
     who);
  written(kc), written(vc), written(ks), written(vs), written(q_out);
  return y;
}
static MaybeTensor kv_append_new(const Tensor& kc, const Tensor& vc, const MaybeTensor& ks, const MaybeTensor& vs, const Tensor& k, const Tensor& v,
                                 const Tensor& start, const MaybeTensor& counts, const MaybeTensor& turns, bool interleaved, double factor,
                                 const MaybeTensor& positions, const MaybeTensor& q) {
  return kv_append(kc, vc, ks, vs, k, v, start, counts, turns, interleaved, factor, positions, q, MaybeTensor());
}
static Tensor kv_append_out(const Tensor& kc, const Tensor& vc, const MaybeTensor& ks, const MaybeTensor& vs, const Tensor& k, const Tensor& v,
                            const Tensor& start, const MaybeTensor& counts, const MaybeTensor& turns, bool interleaved, double factor,
                            const MaybeTensor& positions, const MaybeTensor& q, const Tensor& q_out) {
  return *kv_append(kc, vc, ks, vs, k, v, start, counts, turns, interleaved, factor, positions, q, q_out);
}

// dtype: stx_dtype of the values
std::tuple<Tensor, Tensor> kv_read(const Tensor& kc, const Tensor& vc, const MaybeTensor& ks, const MaybeTensor& vs, int64_t dtype, const MaybeTensor& start, int64_t n) {
  constexpr const char* who = "kv_read";
  const stx_kv c = kv_of(kc, vc, ks, vs, static_cast<int>(dtype), false, who);
  TORCH_CHECK(n >= 0, who, ": n must not be negative");
  c10::cuda::CUDAGuard guard(kc.device());
  const auto o = torch::TensorOptions().device(kc.device()).dtype(dtype == STX_F32 ? c10::kFloat : dtype == STX_F16 ? c10::kHalf : c10::kBFloat16);
  Tensor k = torch::empty({c.n_seq, c.n_kv_heads, n, c.head_dim}, o), v = torch::empty(k.sizes(), o);
  ok(stx_kv_read(&c, maybe_index(kc.device(), start, c.n_seq, who, "start"), n, k.data_ptr(), v.data_ptr(), stream_of(kc.device())), who);
  return std::make_tuple(k, v);
}

// kc, vc [layers, n_seq, n_kv_heads, max_len, head_dim], scales [layers, n_seq, n_kv_heads, max_len]
void kv_keep(const Tensor& kc, const Tensor& vc, const MaybeTensor& ks, const MaybeTensor& vs, int64_t dtype, const Tensor& start, const Tensor& path, const Tensor& counts) {
  constexpr const char* who = "kv_keep";
  TORCH_CHECK(kc.dim() == 5 && kc.sizes() == vc.sizes() && kc.size(0) > 0, who, ": the cache must be [layers, n_seq, n_kv_heads, max_len, head_dim]");
  at::assert_no_internal_overlap(kc);
  at::assert_no_internal_overlap(vc);
  apart(kc, vc, who, "k and v of the cache");
  if (ks) at::assert_no_internal_overlap(*ks);
  if (vs) at::assert_no_internal_overlap(*vs);
  const stx_kv c = kv_of(kc[0], vc[0], ks ? MaybeTensor((*ks)[0]) : MaybeTensor(), vs ? MaybeTensor((*vs)[0]) : MaybeTensor(), static_cast<int>(dtype), true, who);
  TORCH_CHECK(kc.size(0) == 1 || kc.stride(0) == vc.stride(0), who, ": k and v of the cache must have the same strides");
  if (ks)
    TORCH_CHECK(ks->dim() == 4 && ks->size(0) == kc.size(0) && vs->sizes() == ks->sizes() && (kc.size(0) == 1 || ks->stride(0) == vs->stride(0)), who,
                ": scales must be [layers, n_seq, n_kv_heads, max_len]");
  const auto d = kc.device();
  c10::cuda::CUDAGuard guard(d);
  TORCH_CHECK(path.dim() == 2, who, ": path must be [n_seq, nodes]");
  const int64_t pstride = index_rows(d, path, {c.n_seq, path.size(1)}, who, "path");
  ok(stx_kv_keep(&c, kc.size(0), kc.size(0) > 1 ? kc.stride(0) : 0, ks && kc.size(0) > 1 ? ks->stride(0) : 0, index_of(d, start, c.n_seq, who, "start"),
                 path.data_ptr<int64_t>(), pstride, path.size(1), index_of(d, counts, c.n_seq, who, "counts"), stream_of(d)),
     who);
  written(kc), written(vc), written(ks), written(vs);
}

std::tuple<Tensor, Tensor> draft_masks(const Tensor& parents) {
  constexpr const char* who = "draft_masks";
  on_cuda(parents, who, "parents");
  TORCH_CHECK(parents.scalar_type() == c10::kLong && parents.dim() == 2, who, ": parents must be int64 [n_seq, nodes]");
  c10::cuda::CUDAGuard guard(parents.device());
  const Tensor p = parents.contiguous();
  Tensor masks = torch::empty_like(p), depth = torch::empty_like(p);
  ok(stx_draft_masks(p.data_ptr<int64_t>(), p.size(0), p.size(1), masks.data_ptr<int64_t>(), depth.data_ptr<int64_t>(), stream_of(p.device())), who);
  return std::make_tuple(masks, depth);
}

// masks [n_tokens] or [n_seq or 1, n_tokens]
static Tensor tree_attention(const Tensor& q, const Tensor& kc, const Tensor& vc, const MaybeTensor& ks, const MaybeTensor& vs, const Tensor& length,
                      const MaybeTensor& masks, const MaybeTensor& counts, std::optional<double> scale, const MaybeTensor& out) {
  constexpr const char* who = "tree_attention";
  on_cuda(q, who, "q");
  no_grad(q, who, "q");
  const auto d = q.device();
  const int dt = dtype_of(q, who);
  const stx_kv c = kv_of(kc, vc, ks, vs, dt, false, who);
  on(d, kc, who, "the cache");
  TORCH_CHECK(q.dim() == 4 && q.size(0) == c.n_seq && q.size(3) == c.head_dim, who, ": q must be [n_seq, n_tokens, heads, head_dim] and fit the cache");
  c10::cuda::CUDAGuard guard(d);
  const int64_t B = q.size(0), T = q.size(1);
  const int nh = static_cast<int>(q.size(2));
  Tensor y = out ? *out : torch::empty(q.sizes(), q.options().requires_grad(false));
  if (out) {
    on(d, y, who, "out");
    no_grad(y, who, "out");
    apart(y, kc, who, "out and the cache");
    apart(y, vc, who, "out and the cache");
    TORCH_CHECK(y.scalar_type() == q.scalar_type() && y.sizes() == q.sizes(), who, ": out must have q's shape and dtype");
    at::assert_no_internal_overlap(y);
    at::assert_no_overlap(y, q);
  }
  int64_t mstride = 0;
  if (masks) {
    TORCH_CHECK(masks->dim() >= 1 && masks->dim() <= 2, who, ": masks must be [nodes] or [n_seq, nodes]");
    const int64_t rows = masks->dim() == 2 ? masks->size(0) : 1;
    TORCH_CHECK(rows == 1 || rows == B, who, ": masks must have one row or one for each sequence");
    mstride = masks->dim() == 2 ? index_rows(d, *masks, {rows, T}, who, "masks") : index_rows(d, *masks, {T}, who, "masks");
  }
  const stx_heads hq = heads_of(q, who, "q"), ho = heads_of(y, who, "out");
  const int64_t* ln = index_of(d, length, B, who, "length");
  const int64_t* cn = maybe_index(d, counts, B, who, "counts");
  size_t bytes = 0;
  ok(stx_tree_attention_workspace_bytes(T, nh, c.n_kv_heads, c.head_dim, dt, &bytes), who);
  const Tensor ws = torch::empty({static_cast<int64_t>(bytes)}, torch::TensorOptions().dtype(torch::kUInt8).device(d));
  ok(stx_tree_attention(&c, &hq, &ho, T, nh, static_cast<float>(scale ? *scale : 1.0 / std::sqrt(static_cast<double>(c.head_dim))), ln, cn,
                        masks ? masks->data_ptr<int64_t>() : nullptr, mstride, ws.data_ptr(), stream_of(d)),
     who);
  written(out);
  return y;
}
static Tensor tree_attention_new(const Tensor& q, const Tensor& kc, const Tensor& vc, const MaybeTensor& ks, const MaybeTensor& vs,
                                 const Tensor& length, const MaybeTensor& masks, const MaybeTensor& counts, std::optional<double> scale) {
  return tree_attention(q, kc, vc, ks, vs, length, masks, counts, scale, MaybeTensor());
}
static Tensor tree_attention_out(const Tensor& q, const Tensor& kc, const Tensor& vc, const MaybeTensor& ks, const MaybeTensor& vs,
                                 const Tensor& length, const MaybeTensor& masks, const MaybeTensor& counts, std::optional<double> scale,
                                 const Tensor& out) {
  return tree_attention(q, kc, vc, ks, vs, length, masks, counts, scale, out);
}

std::tuple<Tensor, Tensor, Tensor> verify_draft(const Tensor& tokens, const Tensor& target, const MaybeTensor& uniform, const MaybeTensor& parents,
                                                const MaybeTensor& draft, const MaybeTensor& counts) {
  constexpr const char* who = "verify_draft";
  on_cuda(tokens, who, "tokens");
  const auto d = tokens.device();
  TORCH_CHECK(tokens.scalar_type() == c10::kLong && tokens.dim() == 2, who, ": tokens must be int64 [n_seq, nodes]");
  c10::cuda::CUDAGuard guard(d);
  const int64_t B = tokens.size(0), T = tokens.size(1);
  const bool given = target.scalar_type() == c10::kLong;
  on(d, target, who, "target");
  int64_t V = 0;
  if (given) {
    TORCH_CHECK(target.dim() == 2 && target.size(0) == B && target.size(1) == T && target.is_contiguous(), who, ": target tokens must be a contiguous [n_seq, nodes]");
    TORCH_CHECK(!uniform && !draft, who, ": target tokens take neither uniform nor draft");
  } else {
    TORCH_CHECK(target.scalar_type() == c10::kFloat && target.dim() == 3 && target.size(0) == B && target.size(1) == T && target.is_contiguous(), who,
                ": target must be contiguous float32 probabilities [n_seq, nodes, vocabulary] or int64 tokens [n_seq, nodes]");
    no_grad(target, who, "target");
    V = target.size(2);
    TORCH_CHECK(uniform, who, ": target probabilities need uniform random numbers");
    on(d, *uniform, who, "uniform");
    TORCH_CHECK(uniform->scalar_type() == c10::kFloat && uniform->dim() == 2 && uniform->size(0) == B && uniform->size(1) == T && uniform->is_contiguous(), who,
                ": uniform must be contiguous float32 [n_seq, nodes]");
  }
  if (draft) {
    on(d, *draft, who, "draft");
    no_grad(*draft, who, "draft");
    TORCH_CHECK(draft->scalar_type() == c10::kFloat && draft->dim() == 3 && draft->size(0) == B && draft->size(1) == T - 1 && draft->size(2) == V && draft->is_contiguous(),
                who, ": draft must be contiguous float32 [n_seq, nodes - 1, vocabulary]");
    TORCH_CHECK(!parents, who, ": draft probabilities belong to a chain: give no parents");
  }
  const Tensor x = tokens.contiguous();
  Tensor par;
  if (parents) {
    index_rows(d, *parents, {B, T}, who, "parents");
    par = parents->contiguous();
  }
  const auto o = tokens.options();
  Tensor path = torch::empty({B, T}, o), count = torch::empty({B}, o), next = torch::empty({B}, o);
  ok(stx_verify_draft(x.data_ptr<int64_t>(), parents ? par.data_ptr<int64_t>() : nullptr, given ? nullptr : target.data_ptr<float>(),
                      given ? target.data_ptr<int64_t>() : nullptr, draft ? draft->data_ptr<float>() : nullptr,
                      uniform ? uniform->data_ptr<float>() : nullptr, maybe_index(d, counts, B, who, "counts"), B, T, V, path.data_ptr<int64_t>(),
                      count.data_ptr<int64_t>(), next.data_ptr<int64_t>(), stream_of(d)),
     who);
  return std::make_tuple(path, count, next);
}

}  // namespace stxb

// The schemas name what is written, so that nobody who looks at a program by them drops or reorders these calls.
#define STX_CACHE "Tensor(a!) k_cache, Tensor(b!) v_cache, Tensor(c!)? k_scale, Tensor(d!)? v_scale, "
#define STX_ROPE "Tensor x, Tensor positions, Tensor turns, bool interleaved, float factor, bool inverse"
#define STX_APPEND STX_CACHE "Tensor k, Tensor v, Tensor start, Tensor? counts, Tensor? turns, bool interleaved, float factor, Tensor? positions, Tensor? q"
#define STX_ATTEND "Tensor q, Tensor k_cache, Tensor v_cache, Tensor? k_scale, Tensor? v_scale, Tensor length, Tensor? masks, Tensor? counts, float? scale"
TORCH_LIBRARY_FRAGMENT(sparse_mlp, m) {
  m.def("rope(" STX_ROPE ") -> Tensor", stxb::rope_new);
  m.def("rope.out(" STX_ROPE ", *, Tensor(a!) out) -> Tensor(a!)", stxb::rope_out);
  m.def("kv_append(" STX_APPEND ") -> Tensor?", stxb::kv_append_new);
  m.def("kv_append.out(" STX_APPEND ", *, Tensor(e!) q_out) -> Tensor(e!)", stxb::kv_append_out);
  m.def("kv_read", stxb::kv_read);
  m.def("kv_keep(" STX_CACHE "int dtype, Tensor start, Tensor path, Tensor counts) -> ()", stxb::kv_keep);
  m.def("draft_masks", stxb::draft_masks);
  m.def("tree_attention(" STX_ATTEND ") -> Tensor", stxb::tree_attention_new);
  m.def("tree_attention.out(" STX_ATTEND ", *, Tensor(a!) out) -> Tensor(a!)", stxb::tree_attention_out);
  m.def("verify_draft", stxb::verify_draft);
}
