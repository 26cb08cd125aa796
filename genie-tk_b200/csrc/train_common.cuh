// Shared pieces of the training operators (layernorm_train.cu, grad_clip.cu, embedding.cu):
// element types and vectors, the launch helper, warp and block sums.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <stdint.h>

#include <string>

#include "gtk_host.h"

namespace gtk {

template <typename T>
struct Elem;
template <>
struct Elem<float> {
  static __device__ __forceinline__ float load(float v) { return v; }
  static __device__ __forceinline__ float store(float v) { return v; }
};
template <>
struct Elem<__nv_bfloat16> {
  static __device__ __forceinline__ float load(__nv_bfloat16 v) { return __bfloat162float(v); }
  static __device__ __forceinline__ __nv_bfloat16 store(float v) { return __float2bfloat16_rn(v); }
};
template <>
struct Elem<__half> {
  static __device__ __forceinline__ float load(__half v) { return __half2float(v); }
  static __device__ __forceinline__ __half store(float v) { return __float2half_rn(v); }
};

template <typename T, int V>
struct alignas(sizeof(T) * V) Vec {
  T v[V];
};

template <typename T, int V>
__device__ __forceinline__ Vec<T, V> ld_vec(const T* p) {
  return *reinterpret_cast<const Vec<T, V>*>(p);
}
template <typename T, int V>
__device__ __forceinline__ void st_vec(T* p, const Vec<T, V>& v) {
  *reinterpret_cast<Vec<T, V>*>(p) = v;
}

// Waits until the kernel before this one on the stream has finished and its writes are
// visible; at once when the launch carried no programmatic dependency.
__device__ __forceinline__ void wait_previous_kernel() { asm volatile("griddepcontrol.wait;" ::: "memory"); }
// Lets the next kernel of the stream be scheduled; it still waits for this one's end in
// wait_previous_kernel().
__device__ __forceinline__ void allow_next_kernel() { asm volatile("griddepcontrol.launch_dependents;" ::: "memory"); }

// Launch on `st`; `after_previous`: the kernel may be set up while its predecessor on the
// stream still runs. It must call wait_previous_kernel() before it touches memory.
template <typename... KArgs, typename... Args>
int launch(const char* what, void (*kernel)(KArgs...), int64_t blocks, int threads, int smem, cudaStream_t st,
           bool after_previous, Args... args) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(static_cast<unsigned>(blocks));
  cfg.blockDim = dim3(static_cast<unsigned>(threads));
  cfg.dynamicSmemBytes = static_cast<size_t>(smem);
  cfg.stream = st;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = after_previous ? 1 : 0;
  cudaError_t e = cudaLaunchKernelEx(&cfg, kernel, static_cast<KArgs>(args)...);
  if (e != cudaSuccess) {
    cudaGetLastError();
    return fail(GTK_ERR_CUDA, std::string(what) + ": " + cudaGetErrorString(e));
  }
  return GTK_OK;
}

// Resident blocks of `kernel` on the whole device.
template <typename F>
int64_t resident_blocks(F kernel, int threads, int smem) {
  int per_sm = 0;
  if (cudaOccupancyMaxActiveBlocksPerMultiprocessor(&per_sm, kernel, threads, static_cast<size_t>(smem)) !=
          cudaSuccess ||
      per_sm < 1) {
    cudaGetLastError();
    per_sm = 1;
  }
  return static_cast<int64_t>(per_sm) * num_sms();
}

inline bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15u) == 0; }

inline size_t dtype_bytes(int dtype) { return dtype == GTK_F32 ? 4 : 2; }
inline bool dtype_ok(int dtype) { return dtype == GTK_F32 || dtype == GTK_BF16 || dtype == GTK_F16; }

}  // namespace gtk
