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

// V elements of a vector load or store, kept as the words they come in (arrays of 16-bit classes
// under predicates end up in local memory).
template <int kBytes>
struct Words;
template <>
struct Words<16> {
  using type = uint4;
  static __device__ __forceinline__ uint32_t get(const uint4& r, int i) {
    return i == 0 ? r.x : i == 1 ? r.y : i == 2 ? r.z : r.w;
  }
  static __device__ __forceinline__ uint4 make(const uint32_t (&w)[4]) { return make_uint4(w[0], w[1], w[2], w[3]); }
};
template <>
struct Words<8> {
  using type = uint2;
  static __device__ __forceinline__ uint32_t get(const uint2& r, int i) { return i == 0 ? r.x : r.y; }
  static __device__ __forceinline__ uint2 make(const uint32_t (&w)[2]) { return make_uint2(w[0], w[1]); }
};
template <>
struct Words<4> {
  using type = uint32_t;
  static __device__ __forceinline__ uint32_t get(uint32_t r, int) { return r; }
  static __device__ __forceinline__ uint32_t make(const uint32_t (&w)[1]) { return w[0]; }
};
template <>
struct Words<2> {
  using type = unsigned short;
  static __device__ __forceinline__ uint32_t get(unsigned short r, int) { return r; }
  static __device__ __forceinline__ unsigned short make(const uint32_t (&w)[1]) {
    return static_cast<unsigned short>(w[0]);
  }
};

// Two 16-bit elements of a word.
template <typename T>
struct Pair;
template <>
struct Pair<__nv_bfloat16> {
  static __device__ __forceinline__ float lo(uint32_t w) { return __uint_as_float(w << 16); }
  static __device__ __forceinline__ float hi(uint32_t w) { return __uint_as_float(w & 0xffff0000u); }
  static __device__ __forceinline__ uint32_t make(float a, float b) {
    const __nv_bfloat162 h = __floats2bfloat162_rn(a, b);
    return *reinterpret_cast<const uint32_t*>(&h);
  }
};
template <>
struct Pair<__half> {
  static __device__ __forceinline__ float lo(uint32_t w) {
    return __half2float(__ushort_as_half(static_cast<unsigned short>(w & 0xffffu)));
  }
  static __device__ __forceinline__ float hi(uint32_t w) {
    return __half2float(__ushort_as_half(static_cast<unsigned short>(w >> 16)));
  }
  static __device__ __forceinline__ uint32_t make(float a, float b) {
    const __half2 h = __floats2half2_rn(a, b);
    return *reinterpret_cast<const uint32_t*>(&h);
  }
};

template <typename T, int V>
struct Vec {
  using W = Words<static_cast<int>(sizeof(T)) * V>;
  typename W::type r;
  // Element j as fp32 (j is a constant wherever loops are unrolled).
  __device__ __forceinline__ float get(int j) const {
    if constexpr (sizeof(T) == 4)
      return __uint_as_float(W::get(r, j));
    else
      return (j & 1) ? Pair<T>::hi(W::get(r, j >> 1)) : Pair<T>::lo(W::get(r, j >> 1));
  }
  // Rounded from fp32.
  static __device__ __forceinline__ Vec of(const float (&f)[V]) {
    constexpr int kWords = (static_cast<int>(sizeof(T)) * V + 3) / 4;
    uint32_t w[kWords];
#pragma unroll
    for (int i = 0; i < kWords; ++i) {
      if constexpr (sizeof(T) == 4)
        w[i] = __float_as_uint(f[i]);
      else
        w[i] = Pair<T>::make(f[(2 * i) % V], V > 1 ? f[(2 * i + 1) % V] : 0.f);
    }
    Vec v;
    v.r = W::make(w);
    return v;
  }
  static __device__ __forceinline__ Vec zero() {
    const float f[V] = {};
    return of(f);
  }
};

// fp32 arithmetic on pairs: one instruction for two elements.
__device__ __forceinline__ unsigned long long pair_bits(float2 a) { return *reinterpret_cast<unsigned long long*>(&a); }
__device__ __forceinline__ float2 pair_of(unsigned long long b) { return *reinterpret_cast<float2*>(&b); }
__device__ __forceinline__ float2 add2(float2 a, float2 b) {
  unsigned long long r;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(pair_bits(a)), "l"(pair_bits(b)));
  return pair_of(r);
}
__device__ __forceinline__ float2 mul2(float2 a, float2 b) {
  unsigned long long r;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(pair_bits(a)), "l"(pair_bits(b)));
  return pair_of(r);
}
__device__ __forceinline__ float2 fma2(float2 a, float2 b, float2 c) {
  unsigned long long r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(pair_bits(a)), "l"(pair_bits(b)), "l"(pair_bits(c)));
  return pair_of(r);
}
// A product that is rounded before anything is added to it (the assembler fuses mul.rn.f32x2, and
// even a product with -0 added, with an add that follows).
__device__ __forceinline__ float2 rounded_mul2(float2 a, float2 b) {
  return make_float2(__fmul_rn(a.x, b.x), __fmul_rn(a.y, b.y));
}
__device__ __forceinline__ float2 both(float v) { return make_float2(v, v); }

template <typename T, int V>
__device__ __forceinline__ Vec<T, V> ld_vec(const T* p) {
  Vec<T, V> v;
  v.r = *reinterpret_cast<const typename Vec<T, V>::W::type*>(p);
  return v;
}
template <typename T, int V>
__device__ __forceinline__ void st_vec(T* p, const Vec<T, V>& v) {
  *reinterpret_cast<typename Vec<T, V>::W::type*>(p) = v.r;
}

// The same, marked as not to be kept in the L2 cache: for outputs larger than it.
template <typename T, int V>
__device__ __forceinline__ void st_vec_streaming(T* p, const Vec<T, V>& v) {
  if constexpr (sizeof(T) * V >= 4)
    __stcs(reinterpret_cast<typename Vec<T, V>::W::type*>(p), v.r);
  else
    st_vec<T, V>(p, v);
}

// Division of n < 2^31 by a constant of the launch.
struct Divisor {
  uint32_t d, m, shift;
  __device__ __forceinline__ uint32_t quotient(uint32_t n) const { return d == 1 ? n : __umulhi(n, m) >> shift; }
};

// With l = ceil(log2 d) and m = floor(2^(31 + l) / d) + 1, floor(n m / 2^(31 + l)) is n / d for
// n < 2^31 (m d exceeds 2^(31 + l) by e <= d <= 2^l, and n e < 2^(31 + l)).
inline Divisor divisor(uint32_t d) {
  uint32_t l = 0;
  while ((uint64_t(1) << l) < d) ++l;
  if (d <= 1) return Divisor{1, 0, 0};
  return Divisor{d, static_cast<uint32_t>((uint64_t(1) << (31 + l)) / d + 1), l - 1};
}

// Waits until the kernel before this one on the stream has finished and its writes are
// visible; at once when the launch carried no programmatic dependency.
__device__ __forceinline__ void wait_previous_kernel() { asm volatile("griddepcontrol.wait;" ::: "memory"); }
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

// The same in clusters of `cluster` blocks (a divisor of `blocks`).
template <typename... KArgs, typename... Args>
int launch_clusters(const char* what, void (*kernel)(KArgs...), int64_t blocks, int threads, int smem, int cluster,
                    cudaStream_t st, Args... args) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(static_cast<unsigned>(blocks));
  cfg.blockDim = dim3(static_cast<unsigned>(threads));
  cfg.dynamicSmemBytes = static_cast<size_t>(smem);
  cfg.stream = st;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = static_cast<unsigned>(cluster);
  attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  cudaError_t e = cudaLaunchKernelEx(&cfg, kernel, static_cast<KArgs>(args)...);
  if (e == cudaSuccess) return GTK_OK;
  cudaGetLastError();
  return fail(GTK_ERR_CUDA, std::string(what) + ": " + cudaGetErrorString(e));
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
