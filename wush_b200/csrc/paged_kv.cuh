// What the kernels of the paged key-value cache share: argument checks, element access, page lookup.
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_fp8.h>
#include <cuda_runtime.h>

#include <cstdint>
#include <type_traits>

#include "common.cuh"

namespace wush {
namespace kv {

constexpr int MAX_DIM = 256;
constexpr int64_t MAX_TOKENS = INT32_MAX - (1 << 16);
constexpr int STATUS_INDEX = 2;   // an index outside its table; a timeout (1) already in the word stays

__device__ __forceinline__ void report_index(int* status) {
  if (status) atomicCAS(status, 0, STATUS_INDEX);
}

inline int element_bytes(int type) { return type == WUSH_TYPE_E4M3 ? 1 : 2; }

inline bool aligned16(const void* p) { return ((uintptr_t)p & 15) == 0; }

inline int check_heads(const wush_heads* t, int esize) {
  if (!t || !t->data) return WUSH_ERR_NULL_POINTER;
  if (!aligned16(t->data) || (t->row * esize) % 16 || (t->head * esize) % 16) return WUSH_ERR_BAD_ALIGNMENT;
  if (t->row < 0 || t->head < 0) return WUSH_ERR_BAD_SHAPE;
  return WUSH_OK;
}

// The pool and the table themselves; `type` is the element type of the queries of the call.
inline int check_pages(const wush_kv_pages* kv, const wush_kv_table* t, int type) {
  if (!kv || !t || !kv->k || !kv->v) return WUSH_ERR_NULL_POINTER;
  if (type != WUSH_TYPE_BF16 && type != WUSH_TYPE_FP16) return WUSH_ERR_BAD_FLAG;
  if (kv->type != WUSH_TYPE_E4M3 && kv->type != type) return WUSH_ERR_BAD_FLAG;
  const int e = element_bytes(kv->type);
  if (kv->num_pages <= 0 || kv->num_pages > INT32_MAX || kv->page_size <= 0 || kv->heads <= 0 || kv->heads > 65535)
    return WUSH_ERR_BAD_SHAPE;
  if (kv->dim <= 0 || kv->dim > MAX_DIM || (kv->dim * e) % 16) return WUSH_ERR_BAD_SHAPE;
  const int64_t strides[6] = {kv->k_page, kv->k_row, kv->k_head, kv->v_page, kv->v_row, kv->v_head};
  for (int64_t s : strides) {
    if (s < 0) return WUSH_ERR_BAD_SHAPE;
    if ((s * e) % 16) return WUSH_ERR_BAD_ALIGNMENT;
  }
  if (!aligned16(kv->k) || !aligned16(kv->v)) return WUSH_ERR_BAD_ALIGNMENT;
  if ((kv->type == WUSH_TYPE_E4M3) != (kv->k_scale != nullptr) || (kv->type == WUSH_TYPE_E4M3) != (kv->v_scale != nullptr))
    return WUSH_ERR_NULL_POINTER;
  if (kv->bounds) {
    if (kv->bounds_type != WUSH_TYPE_BF16 && kv->bounds_type != WUSH_TYPE_FP16) return WUSH_ERR_BAD_FLAG;
    if (!aligned16(kv->bounds)) return WUSH_ERR_BAD_ALIGNMENT;
  }
  if (t->seqs < 0 || t->width <= 0 || t->stride < 0 || (t->seqs > 0 && !t->block_table)) return WUSH_ERR_BAD_SHAPE;
  // positions and lengths are 32-bit, and kernels look some tiles ahead
  if (t->seqs > INT32_MAX || t->width > INT32_MAX || t->width * kv->page_size > MAX_TOKENS) return WUSH_ERR_TOO_LARGE;
  return WUSH_OK;
}

// Launch of a kernel that may start while the one before it in the stream still runs.  Such a kernel executes
// griddepcontrol.wait in every thread before it touches global memory, and before any of its blocks ends.
struct EarlyLaunch {
  cudaLaunchAttribute attribute;
  cudaLaunchConfig_t cfg;
  explicit EarlyLaunch(cudaStream_t stream) : attribute{}, cfg{} {
    attribute.id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attribute.val.programmaticStreamSerializationAllowed = 1;
    cfg.stream = stream;
    cfg.attrs = &attribute;
    cfg.numAttrs = 1;
  }
  const cudaLaunchConfig_t* config(dim3 grid, int threads, size_t smem) {
    cfg.gridDim = grid;
    cfg.blockDim = dim3(threads);
    cfg.dynamicSmemBytes = smem;
    return &cfg;
  }
};

// ---- element types -----------------------------------------------------------------------------------------------
template <typename T>
__device__ __forceinline__ float2 to_float2(uint32_t two);
template <>
__device__ __forceinline__ float2 to_float2<__nv_bfloat16>(uint32_t two) {
  return __bfloat1622float2(*reinterpret_cast<const __nv_bfloat162*>(&two));
}
template <>
__device__ __forceinline__ float2 to_float2<__half>(uint32_t two) {
  return __half22float2(*reinterpret_cast<const __half2*>(&two));
}

template <typename T>
__device__ __forceinline__ uint32_t pack2(float lo, float hi);
template <>
__device__ __forceinline__ uint32_t pack2<__nv_bfloat16>(float lo, float hi) {
  const __nv_bfloat162 p = __floats2bfloat162_rn(lo, hi);
  return *reinterpret_cast<const uint32_t*>(&p);
}
template <>
__device__ __forceinline__ uint32_t pack2<__half>(float lo, float hi) {
  const __half2 p = __floats2half2_rn(lo, hi);
  return *reinterpret_cast<const uint32_t*>(&p);
}

// four E4M3 bytes as two pairs of fp16 (exact; NaN stays NaN)
__device__ __forceinline__ void e4m3x4_to_f16x4(uint32_t four_bytes, uint32_t& lo, uint32_t& hi) {
  asm("{\n.reg .b16 l, h;\nmov.b32 {l, h}, %2;\ncvt.rn.f16x2.e4m3x2 %0, l;\ncvt.rn.f16x2.e4m3x2 %1, h;\n}\n"
      : "=r"(lo), "=r"(hi)
      : "r"(four_bytes));
}
// two numbers as E4M3 bytes, low byte first; NaN stays NaN, the rest saturates at +-448
__device__ __forceinline__ uint32_t pack2_e4m3(float lo, float hi) {
  uint16_t h;
  asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;\n" : "=h"(h) : "f"(hi), "f"(lo));
  return h;
}

// 8 channels of a row of 16-bit numbers as fp32; `p` points at the first of them
template <typename T>
__device__ __forceinline__ void load8(const T* p, float (&x)[8]) {
  const uint4 v = *reinterpret_cast<const uint4*>(p);
  const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float2 f = to_float2<T>(w[i]);
    x[2 * i] = f.x;
    x[2 * i + 1] = f.y;
  }
}
template <typename T>
__device__ __forceinline__ void store8(T* p, const float (&x)[8]) {
  *reinterpret_cast<uint4*>(p) = make_uint4(pack2<T>(x[0], x[1]), pack2<T>(x[2], x[3]), pack2<T>(x[4], x[5]), pack2<T>(x[6], x[7]));
}
template <>
__device__ __forceinline__ void store8<__nv_fp8_e4m3>(__nv_fp8_e4m3* p, const float (&x)[8]) {
  *reinterpret_cast<uint2*>(p) = make_uint2(pack2_e4m3(x[0], x[1]) | (pack2_e4m3(x[2], x[3]) << 16),
                                            pack2_e4m3(x[4], x[5]) | (pack2_e4m3(x[6], x[7]) << 16));
}

// ---- products ------------------------------------------------------------------------------------------------------
// d [16 x 8] += a [16 x 16] . b [16 x 8] of fp16 (M is __half) or bf16 numbers
template <typename M>
__device__ __forceinline__ void mma(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
  if (std::is_same<M, __half>::value)
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};\n"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
  else
    asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};\n"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

// tokens of a sequence that its table can hold (or pages that a list can); more than that is reported
__device__ __forceinline__ int clamp_length(int len, int64_t capacity, int* status) {
  if (len > capacity) {
    report_index(status);
    return (int)capacity;
  }
  return len < 0 ? 0 : len;
}

// (the sum passes 2^31 where pages are that large, not 2^32)
__device__ __forceinline__ int pages_of_length(int len, int page_size) {
  return (int)(((uint32_t)len + (uint32_t)page_size - 1) / (uint32_t)page_size);
}

// physical page of logical page lp (0 <= lp < width), or -1 and a report when the entry is outside the pool
__device__ __forceinline__ int lookup_page(const wush_kv_table& t, int64_t seq, int lp, int64_t num_pages, int* status) {
  const int page = t.block_table[seq * t.stride + lp];
  if ((uint32_t)page >= (uint64_t)num_pages) {
    report_index(status);
    return -1;
  }
  return page;
}

}  // namespace kv
}  // namespace wush
