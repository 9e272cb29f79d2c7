// Shared by the kernels that write, read and attend over a key/value cache (stx_kv).
#pragma once

#include <cuda_fp8.h>

#include "stx_common.cuh"

namespace stx {

// How a stored row becomes values.  C: type of a stored element.
template <typename T, int STORE> struct Held;
template <typename T> struct Held<T, STX_STORE_SAME> { typedef T C; };
template <typename T> struct Held<T, STX_STORE_INT8> {
  typedef int8_t C;
  static constexpr float MOST = 127.f;
};
template <typename T> struct Held<T, STX_STORE_E4M3> {
  typedef __nv_fp8_storage_t C;
  static constexpr float MOST = 448.f;
};

__device__ __forceinline__ float e4m3_to_f(__nv_fp8_storage_t c) { return __half2float(__half(__nv_cvt_fp8_to_halfraw(c, __NV_E4M3))); }

// Value of one stored element (scale 1 and ignored where the store has none).
template <typename T, int STORE>
__device__ __forceinline__ float held_value(typename Held<T, STORE>::C c, float scale) {
  if constexpr (STORE == STX_STORE_SAME) return DT<T>::to_f(c);
  else if constexpr (STORE == STX_STORE_INT8) return static_cast<float>(c) * scale;
  else return e4m3_to_f(c) * scale;
}

inline size_t store_size(int store, int dtype) { return store == STX_STORE_SAME ? dtype_size(dtype) : 1; }

// Checks of the fields that every entry relies on.
int check_kv(const stx_kv* c, const char* who);
int check_heads(const stx_heads* h, const char* who, const char* name);

// (layer, sequence, head) offsets are formed in 64 bits: a cache may have more than 2^32 elements.
template <typename C> struct KvPtr {
  C* data;
  float* scale;
  int64_t seq, head, slot, sseq, shead;
  __device__ __forceinline__ C* row(int64_t b, int64_t h, int64_t s) const { return data + b * seq + h * head + s * slot; }
  __device__ __forceinline__ float* srow(int64_t b, int64_t h) const { return scale + b * sseq + h * shead; }
};
template <typename C>
inline KvPtr<C> kv_ptr(const stx_kv* c, bool values) {
  return {static_cast<C*>(values ? c->v : c->k), values ? c->v_scale : c->k_scale, c->seq_stride, c->head_stride, c->slot_stride, c->scale_seq_stride, c->scale_head_stride};
}

// f(T tag) / f(T tag, integral_constant store) for the run-time type and store.
template <typename F>
inline int by_dtype(int dtype, F f) {
  switch (dtype) {
    case STX_F32: return f(float());
    case STX_F16: return f(__half());
    default: return f(__nv_bfloat16());
  }
}
template <int S> struct StoreTag { static constexpr int value = S; };
template <typename F>
inline int by_store(int store, F f) {
  switch (store) {
    case STX_STORE_INT8: return f(StoreTag<STX_STORE_INT8>());
    case STX_STORE_E4M3: return f(StoreTag<STX_STORE_E4M3>());
    default: return f(StoreTag<STX_STORE_SAME>());
  }
}

}  // namespace stx
