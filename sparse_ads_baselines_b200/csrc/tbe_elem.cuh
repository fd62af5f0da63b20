// Element types and row vectors of the expert-routing and gradient-clipping kernels.
//
// These kernels move rows of any width and alignment: a row is cut into vectors of VB bytes, VB the
// largest of 16, 8, 4 and 2 that divides every address and stride of the call.  They also take
// bfloat16, which the table kernels do not.
#pragma once

#include <cuda_bf16.h>
#include <string.h>

#include <atomic>

#include "tbe_common.cuh"

namespace tbe {

// The knob "row_threads": most threads per launch of dispatch / combine (0: as many as 32-bit indices allow).
extern std::atomic<int> g_row_threads;

template <>
struct Raw<4> {
  uint32_t w[1];
};
template <>
struct Raw<2> {
  uint16_t w[1];
};

template <>
__device__ __forceinline__ Raw<4> ld_stream<4>(const void* p) {
  Raw<4> r;
  asm volatile("ld.global.nc.L1::no_allocate.u32 %0, [%1];" : "=r"(r.w[0]) : "l"(p));
  return r;
}
template <>
__device__ __forceinline__ Raw<2> ld_stream<2>(const void* p) {
  Raw<2> r;
  asm volatile("ld.global.nc.L1::no_allocate.u16 %0, [%1];" : "=h"(r.w[0]) : "l"(p));
  return r;
}
template <>
__device__ __forceinline__ void st_row<4>(void* p, const Raw<4>& r) {
  asm volatile("st.global.u32 [%0], %1;" : : "l"(p), "r"(r.w[0]) : "memory");
}
template <>
__device__ __forceinline__ void st_row<2>(void* p, const Raw<2>& r) {
  asm volatile("st.global.u16 [%0], %1;" : : "l"(p), "h"(r.w[0]) : "memory");
}

template <int VB>
__device__ __forceinline__ Raw<VB> raw_none() {
  Raw<VB> r;
#pragma unroll
  for (int i = 0; i < static_cast<int>(sizeof(r.w) / sizeof(r.w[0])); ++i) r.w[i] = 0;
  return r;
}

template <typename T>
__device__ __forceinline__ typename Acc<T>::type to_acc(T v);
template <>
__device__ __forceinline__ float to_acc<float>(float v) {
  return v;
}
template <>
__device__ __forceinline__ double to_acc<double>(double v) {
  return v;
}
template <>
__device__ __forceinline__ float to_acc<__half>(__half v) {
  return __half2float(v);
}
template <>
__device__ __forceinline__ float to_acc<__nv_bfloat16>(__nv_bfloat16 v) {
  return __bfloat162float(v);
}

template <typename T>
__device__ __forceinline__ T from_acc(typename Acc<T>::type v);
template <>
__device__ __forceinline__ float from_acc<float>(float v) {
  return v;
}
template <>
__device__ __forceinline__ double from_acc<double>(double v) {
  return v;
}
template <>
__device__ __forceinline__ __half from_acc<__half>(float v) {
  return __float2half_rn(v);
}
template <>
__device__ __forceinline__ __nv_bfloat16 from_acc<__nv_bfloat16>(float v) {
  return __float2bfloat16_rn(v);
}

// A vector's elements in the accumulator type, and back with one rounding to nearest even.
template <typename T, int VB>
__device__ __forceinline__ void expand(const Raw<VB>& r, typename Acc<T>::type* out) {
  constexpr int N = VB / sizeof(T);
  T e[N];
  memcpy(e, &r, VB);
#pragma unroll
  for (int i = 0; i < N; ++i) out[i] = to_acc<T>(e[i]);
}
template <typename T, int VB>
__device__ __forceinline__ Raw<VB> narrow(const typename Acc<T>::type* in) {
  constexpr int N = VB / sizeof(T);
  T e[N];
#pragma unroll
  for (int i = 0; i < N; ++i) e[i] = from_acc<T>(in[i]);
  Raw<VB> r;
  memcpy(&r, e, VB);
  return r;
}

// Bytes of an element, and of a weight or a sum beside it.
inline int any_elem_size(int dtype) { return dtype == TBE_BF16 ? 2 : elem_size(dtype); }
inline int acc_size(int dtype) { return dtype == TBE_F64 ? 8 : 4; }
inline bool known_dtype(int dtype) {
  return dtype == TBE_F32 || dtype == TBE_F16 || dtype == TBE_F64 || dtype == TBE_BF16;
}

// Largest vector (16, 8, 4 or 2 bytes) that divides all of `bits`, the OR of addresses and strides in bytes.
inline int vector_bytes_of(uint64_t bits) { return bits % 16 == 0 ? 16 : bits % 8 == 0 ? 8 : bits % 4 == 0 ? 4 : 2; }

inline uint64_t addr_bits(const void* p) { return static_cast<uint64_t>(reinterpret_cast<uintptr_t>(p)); }

// Whether every address is a multiple of `size` (null is).  The entry points refuse what would fault on the GPU.
template <typename... P>
bool aligned_to(uint64_t size, P... p) {
  return ((addr_bits(p) | ...) & (size - 1)) == 0;
}

}  // namespace tbe
