// LayerNorm over the last axis for training: the forward that keeps its statistics and the
// backward with the parameters' gradients.
//
//   mean_r = sum_c x_rc / D      rstd_r = (sum_c (x_rc - mean_r)^2 / D + eps)^-1/2
//   y_rc   = xh_rc w_c + b_c,    xh_rc  = (x_rc - mean_r) rstd_r
//   g_rc   = dy_rc w_c           dx_rc  = rstd_r (g_rc - mean_c(g) - xh_rc mean_c(g xh))
//   dw_c   = sum_r dy_rc xh_rc   db_c   = sum_r dy_rc
//
// x, y, dy, dx are fp32, bf16 or fp16; w, b and their gradients are fp32 or x's type. All
// arithmetic is fp32, the statistics are stored in fp32, and each 16-bit result is rounded
// once, at its store. The variance is the sum of squared deviations from the finished mean
// (not E[x^2] - mean^2, which cancels), so a row is held in registers and reduced twice.
//
// g is rounded to fp32 before it enters dx as it is before it enters its mean (__fmul_rn keeps
// the compiler from fusing the product into g - mean(g)), so that what cancels in the formula
// cancels here: rows of one element have dx = 0.
//
// What bounds it: HBM. The forward reads x and writes y once, the backward reads x and dy and
// writes dx once. A group of G threads owns a row and keeps 16 (D <= 8192) or 32 (D <= 16384)
// of its elements per thread in registers: up to 32 threads the reductions are shuffles,
// beyond that the group is the block and they go through shared memory. 16 elements per
// thread make few shuffle steps per element (D = 128: 8 threads, 3 steps). Wider rows take
// the loop kernels, which read a row again for each reduction.
//
// dw and db: a thread meets the same columns in every row of its group, so it sums them in
// registers over all the group's rows; the block's groups are then joined in shared memory,
// the block writes one partial row, and a second kernel adds the partials in a fixed order.
// No atomics: the same inputs give the same bits.
#include <atomic>

#include "train_common.cuh"

namespace gtk {
namespace ln {

constexpr int kMaxWidth = 1 << 20;
constexpr int kGroupThreads = 256;  // block of the kernels whose groups are at most a warp
constexpr int kMaxBlockGroup = 512;
constexpr int kJoinCols = 32;
constexpr int kJoinThreads = 1024;

// Where row r of a tensor with up to three leading axes begins: r = (a n1 + b) n2 + c lies
// at a s0 + b s1 + c s2 (element strides); n1 = n2 = 0: rows follow one another, s2 apart.
struct RowMap {
  int64_t s0, s1, s2;
  uint32_t n1, n2;
};

__device__ __forceinline__ int64_t row_offset(const RowMap& m, uint32_t r) {
  if (m.n2 == 0) return static_cast<int64_t>(r) * m.s2;
  const uint32_t t = r / m.n2, c = r - t * m.n2;
  const uint32_t a = t / m.n1, b = t - a * m.n1;
  return a * m.s0 + b * m.s1 + c * m.s2;
}

// Sum over the group: G <= 32 lanes of a warp.
__device__ __forceinline__ float group_sum(float v, int G) {
  for (int o = G >> 1; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}

// Sums of two values over the block (at most 16 warps); `buf` alternates between two halves,
// so that one barrier per reduction is enough.
__device__ __forceinline__ float2 block_sum2(float a, float b, float2* buf, int& half) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    a += __shfl_xor_sync(0xffffffffu, a, o);
    b += __shfl_xor_sync(0xffffffffu, b, o);
  }
  float2* s = buf + 16 * half;
  half ^= 1;
  if ((threadIdx.x & 31) == 0) s[threadIdx.x >> 5] = make_float2(a, b);
  __syncthreads();
  const int nw = blockDim.x >> 5;
  float2 t = s[0];
  for (int i = 1; i < nw; ++i) {
    t.x += s[i].x;
    t.y += s[i].y;
  }
  return t;
}

template <typename T, int V, int K>
struct Row {
  Vec<T, V> e[K];
  __device__ __forceinline__ void load(const T* p, int lane, int G, int nv, bool valid) {
#pragma unroll
    for (int k = 0; k < K; ++k) {
      const int i = lane + G * k;
      if (valid && i < nv)
        e[k] = ld_vec<T, V>(p + static_cast<int64_t>(i) * V);
      else
        e[k] = Vec<T, V>::zero();
    }
  }
};

// Parameters of the thread's columns as floats; `other` where there is none.
template <typename W, int V, int K>
__device__ __forceinline__ void load_columns(float (&out)[K * V], const W* w, int lane, int G, int D, float other) {
#pragma unroll
  for (int k = 0; k < K; ++k)
#pragma unroll
    for (int j = 0; j < V; ++j) {
      const int c = (lane + G * k) * V + j;
      out[k * V + j] = (w && c < D) ? Elem<W>::load(w[c]) : other;
    }
}

// Forward. kBlock: the block is one group of blockDim.x threads; else groups of G <= 32.
template <typename T, typename W, int V, int K, bool kBlock>
__global__ void __launch_bounds__(kBlock ? kMaxBlockGroup : kGroupThreads)
    forward_kernel(const T* __restrict__ x, RowMap xm, const W* __restrict__ w, const W* __restrict__ b,
                   T* __restrict__ y, float* __restrict__ mean_out, float* __restrict__ rstd_out, uint32_t rows,
                   int D, int G, float eps) {
  __shared__ float2 red[32];
  int half = 0;
  const int lane = kBlock ? threadIdx.x : (threadIdx.x & (G - 1));
  const uint32_t per_block = kBlock ? 1u : static_cast<uint32_t>(blockDim.x / G);
  const uint32_t first = kBlock ? blockIdx.x : blockIdx.x * per_block + threadIdx.x / G;
  const uint32_t step = gridDim.x * per_block;
  const int nv = D / V;
  const float inv_d = 1.0f / static_cast<float>(D);
  float wf[K * V], bf[K * V];
  load_columns<W, V, K>(wf, w, lane, G, D, 1.f);
  load_columns<W, V, K>(bf, b, lane, G, D, 0.f);
  Row<T, V, K> next;
  next.load(x + (first < rows ? row_offset(xm, first) : 0), lane, G, nv, first < rows);
  // every group of the block makes the same number of turns, so that shuffles and barriers meet
  const uint32_t block_first = kBlock ? first : blockIdx.x * per_block;
  for (uint64_t base = block_first, r64 = first; base < rows; base += step, r64 += step) {
    const bool valid = r64 < rows;
    Row<T, V, K> cur = next;
    const bool more = r64 + step < rows;
    next.load(x + (more ? row_offset(xm, static_cast<uint32_t>(r64 + step)) : 0), lane, G, nv, more);
    float s = 0.f;
#pragma unroll
    for (int k = 0; k < K; ++k)
#pragma unroll
      for (int j = 0; j < V; ++j) s += cur.e[k].get(j);
    const float mean = (kBlock ? block_sum2(s, 0.f, red, half).x : group_sum(s, G)) * inv_d;
    float q = 0.f;
#pragma unroll
    for (int k = 0; k < K; ++k)
      if (lane + G * k < nv)
#pragma unroll
        for (int j = 0; j < V; ++j) {
          const float d = cur.e[k].get(j) - mean;
          q = fmaf(d, d, q);
        }
    const float var = (kBlock ? block_sum2(q, 0.f, red, half).x : group_sum(q, G)) * inv_d;
    const float rstd = 1.0f / sqrtf(var + eps);
    if (!valid) continue;
    T* yr = y + static_cast<int64_t>(r64) * D;
#pragma unroll
    for (int k = 0; k < K; ++k) {
      const int i = lane + G * k;
      if (i >= nv) continue;
      float o[V];
#pragma unroll
      for (int j = 0; j < V; ++j) o[j] = fmaf((cur.e[k].get(j) - mean) * rstd, wf[k * V + j], bf[k * V + j]);
      st_vec<T, V>(yr + static_cast<int64_t>(i) * V, Vec<T, V>::of(o));
    }
    if (lane == 0) {
      mean_out[r64] = mean;
      rstd_out[r64] = rstd;
    }
  }
}

// Backward: dx and, per block, one partial row [dw | db] of 2 D floats.
template <typename T, typename W, int V, int K, bool kBlock>
__global__ void __launch_bounds__(kBlock ? kMaxBlockGroup : kGroupThreads)
    backward_kernel(const T* __restrict__ dy, RowMap dm, const T* __restrict__ x, RowMap xm,
                    const W* __restrict__ w, const float* __restrict__ mean_in, const float* __restrict__ rstd_in,
                    T* __restrict__ dx, float* __restrict__ partial, uint32_t rows, int D, int G) {
  extern __shared__ float cols[];  // groups of a warp or less: [2][D]
  __shared__ float2 red[32];
  int half = 0;
  const int lane = kBlock ? threadIdx.x : (threadIdx.x & (G - 1));
  const uint32_t per_block = kBlock ? 1u : static_cast<uint32_t>(blockDim.x / G);
  const uint32_t first = kBlock ? blockIdx.x : blockIdx.x * per_block + threadIdx.x / G;
  const uint32_t step = gridDim.x * per_block;
  const int nv = D / V;
  const float inv_d = 1.0f / static_cast<float>(D);
  float wf[K * V], aw[K * V], ab[K * V];
  load_columns<W, V, K>(wf, w, lane, G, D, 1.f);
#pragma unroll
  for (int i = 0; i < K * V; ++i) aw[i] = ab[i] = 0.f;
  const uint32_t block_first = kBlock ? first : blockIdx.x * per_block;
  for (uint64_t base = block_first, r64 = first; base < rows; base += step, r64 += step) {
    const bool valid = r64 < rows;
    const uint32_t r = valid ? static_cast<uint32_t>(r64) : 0u;
    Row<T, V, K> xr, gr;
    xr.load(x + row_offset(xm, r), lane, G, nv, valid);
    gr.load(dy + row_offset(dm, r), lane, G, nv, valid);
    const float mean = valid ? __ldg(mean_in + r) : 0.f;
    const float rstd = valid ? __ldg(rstd_in + r) : 0.f;
    float c1 = 0.f, c2 = 0.f;
#pragma unroll
    for (int k = 0; k < K; ++k)
      if (valid && lane + G * k < nv)
#pragma unroll
        for (int j = 0; j < V; ++j) {
          const float d = gr.e[k].get(j);
          const float xh = (xr.e[k].get(j) - mean) * rstd;
          const float g = __fmul_rn(d, wf[k * V + j]);
          aw[k * V + j] = fmaf(d, xh, aw[k * V + j]);
          ab[k * V + j] += d;
          c1 += g;
          c2 = fmaf(g, xh, c2);
        }
    if (kBlock) {
      const float2 t = block_sum2(c1, c2, red, half);
      c1 = t.x * inv_d;
      c2 = t.y * inv_d;
    } else {
      c1 = group_sum(c1, G) * inv_d;
      c2 = group_sum(c2, G) * inv_d;
    }
    if (!valid) continue;
    T* dr = dx + static_cast<int64_t>(r64) * D;
#pragma unroll
    for (int k = 0; k < K; ++k) {
      const int i = lane + G * k;
      if (i >= nv) continue;
      float o[V];
#pragma unroll
      for (int j = 0; j < V; ++j) {
        const float xh = (xr.e[k].get(j) - mean) * rstd;
        const float g = __fmul_rn(gr.e[k].get(j), wf[k * V + j]);
        o[j] = rstd * ((g - c1) - xh * c2);
      }
      st_vec<T, V>(dr + static_cast<int64_t>(i) * V, Vec<T, V>::of(o));
    }
  }
  if (!partial) return;
  float* pw = partial + static_cast<int64_t>(blockIdx.x) * 2 * D;
  float* pb = pw + D;
  if (kBlock) {
#pragma unroll
    for (int k = 0; k < K; ++k)
      if (lane + G * k < nv)
#pragma unroll
        for (int j = 0; j < V; ++j) {
          const int c = (lane + G * k) * V + j;
          pw[c] = aw[k * V + j];
          pb[c] = ab[k * V + j];
        }
    return;
  }
  // the warp's groups by shuffles, then the warps one after another in shared memory
#pragma unroll
  for (int i = 0; i < K * V; ++i)
    for (int o = G; o < 32; o <<= 1) {
      aw[i] += __shfl_xor_sync(0xffffffffu, aw[i], o);
      ab[i] += __shfl_xor_sync(0xffffffffu, ab[i], o);
    }
  const int warp = threadIdx.x >> 5, nw = blockDim.x >> 5;
  for (int t = 0; t < nw; ++t) {
    if (warp == t && (threadIdx.x & 31) < G)
#pragma unroll
      for (int k = 0; k < K; ++k)
        if (lane + G * k < nv)
#pragma unroll
          for (int j = 0; j < V; ++j) {
            const int c = (lane + G * k) * V + j;
            cols[c] = (t ? cols[c] : 0.f) + aw[k * V + j];
            cols[D + c] = (t ? cols[D + c] : 0.f) + ab[k * V + j];
          }
    __syncthreads();
  }
  for (int c = threadIdx.x; c < 2 * D; c += blockDim.x) pw[c] = cols[c];
}

// dw, db: the sum of `n` partial rows of 2 D floats, in a fixed order (64 bits across warps).
template <typename W>
__global__ void __launch_bounds__(kJoinThreads)
    join_kernel(const float* __restrict__ partial, int n, int D, W* __restrict__ dw, W* __restrict__ db) {
  wait_previous_kernel();
  __shared__ double part[kJoinThreads / 32][kJoinCols + 1];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int c = blockIdx.x * kJoinCols + lane;
  double s = 0.0;
  if (c < 2 * D) {
    const float* p = partial + c;
    const int64_t ld = 2 * static_cast<int64_t>(D);
#pragma unroll 8
    for (int i = warp; i < n; i += kJoinThreads / 32) s += static_cast<double>(p[i * ld]);
  }
  part[warp][lane] = s;
  __syncthreads();
  if (warp) return;
  for (int i = 1; i < kJoinThreads / 32; ++i) s += part[i][lane];
  if (c < D) {
    if (dw) dw[c] = Elem<W>::store(static_cast<float>(s));
  } else if (c < 2 * D) {
    if (db) db[c - D] = Elem<W>::store(static_cast<float>(s));
  }
}

// ---- Rows of more than 16384 elements -----------------------------------------------------

template <typename T, typename W>
__global__ void __launch_bounds__(kMaxBlockGroup)
    forward_wide_kernel(const T* __restrict__ x, RowMap xm, const W* __restrict__ w, const W* __restrict__ b,
                        T* __restrict__ y, float* __restrict__ mean_out, float* __restrict__ rstd_out, uint32_t rows,
                        int D, float eps) {
  __shared__ float2 red[32];
  int half = 0;
  const float inv_d = 1.0f / static_cast<float>(D);
  for (uint64_t r = blockIdx.x; r < rows; r += gridDim.x) {
    const T* xr = x + row_offset(xm, static_cast<uint32_t>(r));
    float s = 0.f, q = 0.f;
    for (int c = threadIdx.x; c < D; c += blockDim.x) s += Elem<T>::load(xr[c]);
    const float mean = block_sum2(s, 0.f, red, half).x * inv_d;
    for (int c = threadIdx.x; c < D; c += blockDim.x) {
      const float d = Elem<T>::load(xr[c]) - mean;
      q = fmaf(d, d, q);
    }
    const float rstd = 1.0f / sqrtf(block_sum2(q, 0.f, red, half).x * inv_d + eps);
    T* yr = y + static_cast<int64_t>(r) * D;
    for (int c = threadIdx.x; c < D; c += blockDim.x)
      yr[c] = Elem<T>::store(fmaf((Elem<T>::load(xr[c]) - mean) * rstd, w ? Elem<W>::load(w[c]) : 1.f,
                                  b ? Elem<W>::load(b[c]) : 0.f));
    if (threadIdx.x == 0) {
      mean_out[r] = mean;
      rstd_out[r] = rstd;
    }
  }
}

template <typename T, typename W>
__global__ void __launch_bounds__(kMaxBlockGroup)
    backward_wide_kernel(const T* __restrict__ dy, RowMap dm, const T* __restrict__ x, RowMap xm,
                         const W* __restrict__ w, const float* __restrict__ mean_in,
                         const float* __restrict__ rstd_in, T* __restrict__ dx, uint32_t rows, int D) {
  __shared__ float2 red[32];
  int half = 0;
  const float inv_d = 1.0f / static_cast<float>(D);
  for (uint64_t r = blockIdx.x; r < rows; r += gridDim.x) {
    const T* xr = x + row_offset(xm, static_cast<uint32_t>(r));
    const T* gr = dy + row_offset(dm, static_cast<uint32_t>(r));
    const float mean = mean_in[r], rstd = rstd_in[r];
    float c1 = 0.f, c2 = 0.f;
    for (int c = threadIdx.x; c < D; c += blockDim.x) {
      const float g = __fmul_rn(Elem<T>::load(gr[c]), w ? Elem<W>::load(w[c]) : 1.f);
      c1 += g;
      c2 = fmaf(g, (Elem<T>::load(xr[c]) - mean) * rstd, c2);
    }
    const float2 t = block_sum2(c1, c2, red, half);
    T* dr = dx + static_cast<int64_t>(r) * D;
    for (int c = threadIdx.x; c < D; c += blockDim.x) {
      const float g = __fmul_rn(Elem<T>::load(gr[c]), w ? Elem<W>::load(w[c]) : 1.f);
      const float xh = (Elem<T>::load(xr[c]) - mean) * rstd;
      dr[c] = Elem<T>::store(rstd * ((g - t.x * inv_d) - xh * (t.y * inv_d)));
    }
  }
}

// Partial [dw | db] of the rows [y * per, (y + 1) * per), one column per thread.
template <typename T>
__global__ void __launch_bounds__(256)
    columns_wide_kernel(const T* __restrict__ dy, RowMap dm, const T* __restrict__ x, RowMap xm,
                        const float* __restrict__ mean_in, const float* __restrict__ rstd_in,
                        float* __restrict__ partial, uint32_t rows, uint32_t per, int D, int col_blocks) {
  const int c = (blockIdx.x % col_blocks) * 256 + threadIdx.x;
  const uint32_t slab = blockIdx.x / col_blocks;
  if (c >= D) return;
  const uint64_t r0 = static_cast<uint64_t>(slab) * per;
  const uint64_t r1 = r0 + per < rows ? r0 + per : rows;
  float sw = 0.f, sb = 0.f;
  for (uint64_t r = r0; r < r1; ++r) {
    const float d = Elem<T>::load(dy[row_offset(dm, static_cast<uint32_t>(r)) + c]);
    const float v = Elem<T>::load(x[row_offset(xm, static_cast<uint32_t>(r)) + c]);
    sw = fmaf(d, (v - mean_in[r]) * rstd_in[r], sw);
    sb += d;
  }
  float* p = partial + static_cast<int64_t>(slab) * 2 * D;
  p[c] = sw;
  p[D + c] = sb;
}

// ---- Host ---------------------------------------------------------------------------------

constexpr int64_t kWideSlabs = 64;

struct Shape {
  int V, G;
  bool block, thirty_two, wide;
};

// Elements per thread and threads per row (see the file comment). 16-byte vectors when every
// row of every tensor begins on a 16-byte boundary, else single elements.
Shape choose(int64_t D, bool vec, int elem_bytes) {
  Shape s = {};
  s.V = vec ? 16 / elem_bytes : 1;
  s.wide = D > 16384;
  s.thirty_two = D > 8192;
  const int64_t per = s.thirty_two ? 32 : 16;
  int G = 1;
  while (static_cast<int64_t>(G) * per < D) G <<= 1;
  if (s.thirty_two && G < 64) G = 64;
  s.G = G;
  s.block = G > 32;
  return s;
}

// Partial rows that the workspace holds: as many as the backward has blocks, which are at most
// 1024 threads' worth per SM (16 blocks) on the 148 SMs of this family, and no more than rows.
int64_t max_partials(int64_t rows, int64_t D) {
  if (D > 16384) return rows < kWideSlabs ? rows : kWideSlabs;
  const Shape s = choose(D, false, 4);
  const int threads = s.block ? s.G : kGroupThreads;
  int64_t cap = 1024 / threads;
  cap = 148 * (cap > 16 ? 16 : cap);
  return rows < cap ? rows : cap;
}

struct Args {
  const void *x, *dy, *w, *b;
  RowMap xm, dm;
  void *y, *dx, *dw, *db;
  float *mean, *rstd, *partial;
  int64_t rows;
  int D;
  float eps;
  cudaStream_t st;
};

// Resident blocks of a kernel by block size (64, 128, 256, 512 threads), asked for once.
constexpr int kBlockSizes = 4;
template <typename F>
int64_t cached_residency(std::atomic<int64_t>* cache, F kernel, int threads, int smem) {
  std::atomic<int64_t>& c = cache[threads >= 512 ? 3 : threads >= 256 ? 2 : threads >= 128 ? 1 : 0];
  int64_t v = c.load(std::memory_order_relaxed);
  if (!v) c.store(v = resident_blocks(kernel, threads, smem), std::memory_order_relaxed);
  return v;
}

template <typename T, typename W, int V, int K, bool kBlock>
int run_forward(const Args& a, const Shape& s) {
  auto kernel = forward_kernel<T, W, V, K, kBlock>;
  const int threads = kBlock ? s.G : kGroupThreads;
  static std::atomic<int64_t> cache[kBlockSizes];
  const int64_t cap = cached_residency(cache, kernel, threads, 0);
  const int64_t per = kBlock ? 1 : kGroupThreads / s.G;
  int64_t blocks = (a.rows + per - 1) / per;
  if (blocks > cap) blocks = cap;
  return launch("layernorm forward", kernel, blocks, threads, 0, a.st, false, static_cast<const T*>(a.x), a.xm,
                static_cast<const W*>(a.w), static_cast<const W*>(a.b), static_cast<T*>(a.y), a.mean, a.rstd,
                static_cast<uint32_t>(a.rows), a.D, s.G, a.eps);
}

template <typename W>
int run_join(const Args& a, int64_t n) {
  return launch("layernorm gradient join", join_kernel<W>, (2 * static_cast<int64_t>(a.D) + kJoinCols - 1) / kJoinCols,
                kJoinThreads, 0, a.st, true, static_cast<const float*>(a.partial), static_cast<int>(n), a.D,
                static_cast<W*>(a.dw), static_cast<W*>(a.db));
}

template <typename T, typename W, int V, int K, bool kBlock>
int run_backward(const Args& a, const Shape& s) {
  auto kernel = backward_kernel<T, W, V, K, kBlock>;
  const int threads = kBlock ? s.G : kGroupThreads;
  const int smem = kBlock ? 0 : 2 * a.D * static_cast<int>(sizeof(float));
  static std::atomic<int64_t> cache[kBlockSizes];
  const int64_t cap = cached_residency(cache, kernel, threads, kBlock ? 0 : 4096);
  const int64_t per = kBlock ? 1 : kGroupThreads / s.G;
  int64_t blocks = (a.rows + per - 1) / per;
  if (blocks > cap) blocks = cap;
  const int64_t most = max_partials(a.rows, a.D);
  if (blocks > most) blocks = most;
  if (int e = launch("layernorm backward", kernel, blocks, threads, smem, a.st, false, static_cast<const T*>(a.dy),
                     a.dm, static_cast<const T*>(a.x), a.xm, static_cast<const W*>(a.w),
                     static_cast<const float*>(a.mean), static_cast<const float*>(a.rstd), static_cast<T*>(a.dx),
                     a.partial, static_cast<uint32_t>(a.rows), a.D, s.G))
    return e;
  return a.partial ? run_join<W>(a, blocks) : GTK_OK;
}

template <typename T, typename W>
int run_wide(const Args& a, bool backward) {
  int64_t blocks = static_cast<int64_t>(num_sms()) * 4;
  if (blocks > a.rows) blocks = a.rows;
  const uint32_t rows = static_cast<uint32_t>(a.rows);
  if (!backward)
    return launch("layernorm forward", forward_wide_kernel<T, W>, blocks, kMaxBlockGroup, 0, a.st, false,
                  static_cast<const T*>(a.x), a.xm, static_cast<const W*>(a.w), static_cast<const W*>(a.b),
                  static_cast<T*>(a.y), a.mean, a.rstd, rows, a.D, a.eps);
  if (int e = launch("layernorm backward", backward_wide_kernel<T, W>, blocks, kMaxBlockGroup, 0, a.st, false,
                     static_cast<const T*>(a.dy), a.dm, static_cast<const T*>(a.x), a.xm,
                     static_cast<const W*>(a.w), static_cast<const float*>(a.mean),
                     static_cast<const float*>(a.rstd), static_cast<T*>(a.dx), rows, a.D))
    return e;
  if (!a.partial) return GTK_OK;
  const int64_t slabs_max = max_partials(a.rows, a.D);
  const uint32_t per = static_cast<uint32_t>((a.rows + slabs_max - 1) / slabs_max);
  const int64_t slabs = (a.rows + per - 1) / per;
  const int col_blocks = (a.D + 255) / 256;
  if (int e = launch("layernorm weight gradient", columns_wide_kernel<T>, slabs * col_blocks, 256, 0, a.st, false,
                     static_cast<const T*>(a.dy), a.dm, static_cast<const T*>(a.x), a.xm,
                     static_cast<const float*>(a.mean), static_cast<const float*>(a.rstd), a.partial, rows, per, a.D,
                     col_blocks))
    return e;
  return run_join<W>(a, slabs);
}

template <typename T, typename W, int V, int K, bool kBlock>
int run_one(const Args& a, const Shape& s, bool backward) {
  return backward ? run_backward<T, W, V, K, kBlock>(a, s) : run_forward<T, W, V, K, kBlock>(a, s);
}

template <typename T, typename W>
int run_typed(const Args& a, bool vec, bool backward) {
  constexpr int VX = 16 / static_cast<int>(sizeof(T));
  const Shape s = choose(a.D, vec, sizeof(T));
  if (s.wide) return run_wide<T, W>(a, backward);
  if (s.V > 1) {
    if (s.thirty_two) return run_one<T, W, VX, 32 / VX, true>(a, s, backward);
    if (s.block) return run_one<T, W, VX, 16 / VX, true>(a, s, backward);
    return run_one<T, W, VX, 16 / VX, false>(a, s, backward);
  }
  if (s.thirty_two) return run_one<T, W, 1, 32, true>(a, s, backward);
  if (s.block) return run_one<T, W, 1, 16, true>(a, s, backward);
  return run_one<T, W, 1, 16, false>(a, s, backward);
}

int run(const Args& a, int xt, int wt, bool vec, bool backward) {
  if (xt == GTK_F32) return run_typed<float, float>(a, vec, backward);
  if (xt == GTK_BF16)
    return wt == GTK_F32 ? run_typed<__nv_bfloat16, float>(a, vec, backward)
                         : run_typed<__nv_bfloat16, __nv_bfloat16>(a, vec, backward);
  return wt == GTK_F32 ? run_typed<__half, float>(a, vec, backward) : run_typed<__half, __half>(a, vec, backward);
}

// Checks a tensor's leading axes and fills its RowMap; `vec` is cleared when some row does not
// begin on a 16-byte boundary.
int row_map(const gtk_rows* v, const void* base, int64_t rows, int64_t D, size_t bytes, const char* what, RowMap* out,
            bool* vec) {
  if ((D * bytes) % 16 || !aligned16(base)) *vec = false;
  if (!v) {
    *out = RowMap{0, 0, D, 0, 0};
    return GTK_OK;
  }
  for (int i = 0; i < 3; ++i) {
    if (v->size[i] < 1 || v->size[i] > rows)
      return fail(GTK_ERR_INVALID_ARG, std::string("layernorm: bad leading sizes of ") + what);
    if (v->stride[i] < 0) return fail(GTK_ERR_INVALID_ARG, std::string("layernorm: negative stride of ") + what);
    if (v->size[i] > 1 && (v->stride[i] * static_cast<int64_t>(bytes)) % 16) *vec = false;
  }
  if (v->size[0] * v->size[1] > rows || v->size[0] * v->size[1] * v->size[2] != rows)
    return fail(GTK_ERR_INVALID_ARG, std::string("layernorm: the leading sizes of ") + what + " do not make up rows");
  *out = RowMap{v->stride[0], v->stride[1], v->stride[2], static_cast<uint32_t>(v->size[1]),
                static_cast<uint32_t>(v->size[2])};
  return GTK_OK;
}

int check_common(int64_t rows, int64_t D, int x_dtype, int w_dtype) {
  if (!dims_ok(rows, (int64_t(1) << 31) - 1)) return fail(GTK_ERR_INVALID_ARG, "layernorm: rows must be 1..2^31-1");
  if (!dims_ok(D, kMaxWidth)) return fail(GTK_ERR_INVALID_ARG, "layernorm: D must be 1..2^20");
  if (!dtype_ok(x_dtype) || !(w_dtype == GTK_F32 || w_dtype == x_dtype))
    return fail(GTK_ERR_UNSUPPORTED, "layernorm: x is fp32, bf16 or fp16, the parameters fp32 or x's type");
  return GTK_OK;
}

int check_elem_ptr(const void* p, const char* name, int dtype) { return check_ptr(p, name, dtype_bytes(dtype)); }

}  // namespace ln
}  // namespace gtk

using namespace gtk;

extern "C" {

size_t gtk_layernorm_backward_workspace_bytes(int64_t rows, int64_t D) {
  if (!dims_ok(rows, (int64_t(1) << 31) - 1) || !dims_ok(D, ln::kMaxWidth)) return 0;
  return static_cast<size_t>(ln::max_partials(rows, D)) * 2 * D * sizeof(float);
}

int gtk_layernorm_forward(const void* x, const gtk_rows* x_rows, int x_dtype, const void* weight, const void* bias,
                          int w_dtype, void* y, float* mean, float* rstd, int64_t rows, int64_t D, float eps,
                          void* stream) {
  if (int e = ln::check_common(rows, D, x_dtype, w_dtype)) return e;
  if (!(eps >= 0.f)) return fail(GTK_ERR_INVALID_ARG, "layernorm: eps must be >= 0");
  if (int e = ln::check_elem_ptr(x, "x", x_dtype)) return e;
  if (int e = ln::check_elem_ptr(y, "y", x_dtype)) return e;
  if (weight)
    if (int e = ln::check_elem_ptr(weight, "weight", w_dtype)) return e;
  if (bias)
    if (int e = ln::check_elem_ptr(bias, "bias", w_dtype)) return e;
  if (int e = check_ptr(mean, "mean", 4)) return e;
  if (int e = check_ptr(rstd, "rstd", 4)) return e;
  ln::Args a = {};
  bool vec = aligned16(y);
  if (int e = ln::row_map(x_rows, x, rows, D, dtype_bytes(x_dtype), "x", &a.xm, &vec)) return e;
  if (int e = check_device()) return e;
  a.x = x, a.w = weight, a.b = bias, a.y = y, a.mean = mean, a.rstd = rstd;
  a.rows = rows, a.D = static_cast<int>(D), a.eps = eps, a.st = static_cast<cudaStream_t>(stream);
  return ln::run(a, x_dtype, w_dtype, vec, false);
}

int gtk_layernorm_backward(const void* dy, const gtk_rows* dy_rows, const void* x, const gtk_rows* x_rows,
                           int x_dtype, const void* weight, int w_dtype, const float* mean, const float* rstd,
                           void* dx, void* dweight, void* dbias, void* workspace, size_t workspace_bytes,
                           int64_t rows, int64_t D, void* stream) {
  if (int e = ln::check_common(rows, D, x_dtype, w_dtype)) return e;
  const bool params = dweight || dbias;
  if (params && workspace_bytes < gtk_layernorm_backward_workspace_bytes(rows, D))
    return fail(GTK_ERR_WORKSPACE, "layernorm: workspace too small");
  if (int e = ln::check_elem_ptr(dy, "dy", x_dtype)) return e;
  if (int e = ln::check_elem_ptr(x, "x", x_dtype)) return e;
  if (int e = ln::check_elem_ptr(dx, "dx", x_dtype)) return e;
  if (weight)
    if (int e = ln::check_elem_ptr(weight, "weight", w_dtype)) return e;
  if (dweight)
    if (int e = ln::check_elem_ptr(dweight, "dweight", w_dtype)) return e;
  if (dbias)
    if (int e = ln::check_elem_ptr(dbias, "dbias", w_dtype)) return e;
  if (int e = check_ptr(mean, "mean", 4)) return e;
  if (int e = check_ptr(rstd, "rstd", 4)) return e;
  if (params)
    if (int e = check_ptr(workspace, "workspace")) return e;
  ln::Args a = {};
  bool vec = aligned16(dx);
  if (int e = ln::row_map(x_rows, x, rows, D, dtype_bytes(x_dtype), "x", &a.xm, &vec)) return e;
  if (int e = ln::row_map(dy_rows, dy, rows, D, dtype_bytes(x_dtype), "dy", &a.dm, &vec)) return e;
  if (int e = check_device()) return e;
  a.x = x, a.dy = dy, a.w = weight, a.dx = dx, a.dw = dweight, a.db = dbias;
  a.mean = const_cast<float*>(mean), a.rstd = const_cast<float*>(rstd);
  a.partial = params ? static_cast<float*>(workspace) : nullptr;
  a.rows = rows, a.D = static_cast<int>(D), a.st = static_cast<cudaStream_t>(stream);
  return ln::run(a, x_dtype, w_dtype, vec, true);
}

}  // extern "C"
