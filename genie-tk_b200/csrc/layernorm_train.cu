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
// g is rounded to fp32 before it enters dx as it is before it enters its mean (a product fused
// into g - mean(g) is not), so that what cancels in the formula cancels here: rows of one
// element have dx = 0.
//
// What bounds it: HBM for fp32 rows. For 16-bit rows, half as many bytes, the chains of dependent
// instructions in the 8 to 16 warps of an SM (4096 x 4096 bf16: issue slots half busy, DRAM 26% in the
// forward and 38% in the backward of their peak); elements are therefore taken in pairs where fp32
// allows (add2, mul2, fma2). The forward reads x and writes y once, the backward reads x and dy and writes dx once. A group of G threads owns a row,
// 16 of its elements per thread (32 from D = 8193 on, up to 16384): up to 32 threads the reductions
// are shuffles, beyond that the group is the block, they go through shared memory, and two rows
// share each barrier. 16 elements per thread make few shuffle steps per element (D = 128: 8 threads,
// 3 steps). The rows that follow are on their way meanwhile: every thread copies its own elements
// of the next rows to a ring in shared memory (cp.async), which takes no registers and, as nobody
// else reads them, no barriers. Wider rows take the loop kernels, which read a row again for
// each reduction.
//
// Widths that no 16-byte vector divides: rows then begin at different places of a vector, but all
// rows of one group at the same place, because the groups step by a multiple of eight rows. The
// group's vectors are laid over its rows from the boundary before them (`lead` elements earlier),
// and only the first and the last vector of a row are looked at by element. That goes for contiguous
// rows on a 16-byte boundary. Strided rows of such widths, and rows behind a base off a boundary, are
// read by element and without a ring (512 x 512 x 129 fp32 with swapped axes: forward 86 us, backward
// 118; with contiguous copies made first 168 and 302).
//
// Rows of a transposed pair tensor lie far apart in one axis and next to one another in the other.
// They are visited in tiles of 8 x 4, which reads runs of eight rows and writes runs of four
// (in plain order, the backward of 512 x 512 x 128 fp32 takes 75 us instead of 73).
//
// dw and db: a thread meets the same columns in every row of its group, so it sums them in
// registers over all the group's rows; the block's groups are then joined in shared memory,
// the block writes one partial row, and a second kernel adds the partials in a fixed order, in fp32
// trees (512 x 512 x 128: 1.7e-7 of the norm from the 64-bit sums). A grid of up to eight blocks is launched as one cluster and adds them itself, through distributed shared
// memory (37 rows of 384: 4.2 us instead of 5.0 from a graph, 8.5 instead of 10.7 from Python).
// No atomics: the same inputs give the same bits.
#include <cooperative_groups.h>

#include <atomic>

#include "train_common.cuh"

namespace gtk {
namespace ln {

constexpr int kMaxWidth = 1 << 20;
constexpr int kGroupThreads = 256;  // block of the kernels whose groups are at most a warp
constexpr int kMaxBlockGroup = 512;
constexpr int kJoinThreads = 512;
constexpr int kMaxStages = 2;             // turns in the ring: this one and the next
constexpr int kRingBytes = 200 * 1024;    // most of an SM
constexpr int kMaxCluster = 8;

// Where row r of a tensor with up to three leading axes begins: r = (a n1 + b) n2 + c lies
// at a s0 + b s1 + c s2 (element strides); `plain`: rows follow one another, s2 apart.
struct RowMap {
  int64_t s0, s1, s2;
  Divisor n1, n2;
  bool plain;
};

// The order in which rows are visited: as they come, or (`tiled`) the n1 x n2 planes of rows in
// tiles of 8 x 4, t1 x t2 of them (the last ones in part outside). `visits` counts places.
struct Order {
  Divisor t1, t2;
  uint32_t n1, n2;
  uint32_t visits;  // below 2^31
  bool tiled;
};
constexpr uint32_t kNoRow = 0xffffffffu;

// A row and, with tiles, its coordinates.
struct Place {
  uint32_t r, a, b, c;
};

__device__ __forceinline__ Place place_at(const Order& o, uint32_t v) {
  Place p = {kNoRow, 0, 0, 0};
  if (v >= o.visits) return p;
  if (!o.tiled) {
    p.r = v;
    return p;
  }
  const uint32_t tile = v >> 5, t = o.t2.quotient(tile);
  p.a = o.t1.quotient(t);
  p.b = (t - p.a * o.t1.d) * 8 + (v & 7u);
  p.c = (tile - t * o.t2.d) * 4 + (v >> 3 & 3u);
  if (p.b < o.n1 && p.c < o.n2) p.r = (p.a * o.n1 + p.b) * o.n2 + p.c;
  return p;
}

__device__ __forceinline__ int64_t row_offset(const RowMap& m, uint32_t r) {
  if (m.plain) return static_cast<int64_t>(r) * m.s2;
  const uint32_t t = m.n2.quotient(r), c = r - t * m.n2.d;
  const uint32_t a = m.n1.quotient(t), b = t - a * m.n1.d;
  return a * m.s0 + b * m.s1 + c * m.s2;
}

__device__ __forceinline__ int64_t row_offset(const RowMap& m, const Order& o, const Place& p) {
  if (o.tiled && !m.plain && m.n1.d == o.n1 && m.n2.d == o.n2) return p.a * m.s0 + p.b * m.s1 + p.c * m.s2;
  return row_offset(m, p.r);
}

// Sums over a group of G <= 32 lanes of a warp.
template <int n>
__device__ __forceinline__ void group_sum(float (&v)[n], int G) {
  for (int o = G >> 1; o > 0; o >>= 1)
#pragma unroll
    for (int i = 0; i < n; ++i) v[i] += __shfl_xor_sync(0xffffffffu, v[i], o);
}

// Sums of n = 1, 2 or 4 values over the block (at most 16 warps). The values are spread over the
// lanes as they are added up, so that all of them take 5 or 6 shuffles in the warp and, behind the
// barrier, 4 or 5 over the warps and n to hand them out. `buf` (two halves of 64 floats, zeros at
// first) alternates, so that one barrier per reduction is enough.
template <int n>
__device__ __forceinline__ void block_sum(float (&v)[n], float* buf, int& half) {
  const int lane = threadIdx.x & 31;
  float x;
  if constexpr (n == 4) {
    const bool hi = lane & 16;
    const float a = (hi ? v[2] : v[0]) + __shfl_xor_sync(0xffffffffu, hi ? v[0] : v[2], 16);
    const float b = (hi ? v[3] : v[1]) + __shfl_xor_sync(0xffffffffu, hi ? v[1] : v[3], 16);
    const bool up = lane & 8;
    x = (up ? b : a) + __shfl_xor_sync(0xffffffffu, up ? a : b, 8);
  } else if constexpr (n == 2) {
    const bool hi = lane & 16;
    x = (hi ? v[1] : v[0]) + __shfl_xor_sync(0xffffffffu, hi ? v[0] : v[1], 16);
    x += __shfl_xor_sync(0xffffffffu, x, 8);
  } else {
    x = v[0] + __shfl_xor_sync(0xffffffffu, v[0], 16);
    x += __shfl_xor_sync(0xffffffffu, x, 8);
  }
#pragma unroll
  for (int o = 4; o > 0; o >>= 1) x += __shfl_xor_sync(0xffffffffu, x, o);
  float* s = buf + 64 * half;
  half ^= 1;
  constexpr int kEach = 32 / n;  // lanes that hold one value
  if (lane % kEach == 0) s[(threadIdx.x >> 5) * n + lane / kEach] = x;
  __syncthreads();
  // lane = (warp, value), values fastest
  x = s[n == 1 ? (lane & 15) : lane];
  if constexpr (n == 4) x += s[32 + lane];
#pragma unroll
  for (int o = n == 4 ? 16 : n == 2 ? 16 : 8; o >= n; o >>= 1) x += __shfl_xor_sync(0xffffffffu, x, o);
#pragma unroll
  for (int i = 0; i < n; ++i) v[i] = n == 1 ? x : __shfl_sync(0xffffffffu, x, i);
}

// Zeros in the buffers of block_sum.
__device__ __forceinline__ void block_sum_init(float* buf) {
  for (int i = threadIdx.x; i < 128; i += blockDim.x) buf[i] = 0.f;
  __syncthreads();
}

// How a group's vectors lie over its rows: vector i covers the columns i V - lead .. + V - 1. kEdge:
// the width is no multiple of V, so that rows begin and end inside a vector.
template <bool kEdge>
struct Lay {
  int lane, G, nv, lead_, D;
  __device__ __forceinline__ int lead() const { return kEdge ? lead_ : 0; }
};

// A thread's elements of a row: K vectors of V at vector indices lane + G k < nv. Vectors come
// through a ring slot in shared memory ([k][thread], 16 bytes each; slots of vectors that do not
// exist hold zeros from the start); single elements (V = 1: rows that begin anywhere) through
// registers, without a row ahead.
template <typename T, int V, int K, bool kEdge>
struct Row {
  using L = Lay<kEdge>;
  static constexpr bool kAsync = V > 1;
  static constexpr int kBytes = 16;
  Vec<T, V> e[kAsync ? 1 : K];
  const char* slot;
  int pitch;

  // `from`: where the thread's first vector begins in the row. The last vector reads no further than
  // the row; the first one begins with up to V - 1 elements of the row before.
  static __device__ __forceinline__ void request(uint32_t to, int pitch, const T* from, const L& l) {
    if constexpr (kAsync) {
#pragma unroll
      for (int k = 0; k < K; ++k) {
        const int i = l.lane + l.G * k;
        if (i >= l.nv) continue;
        const T* src = from + l.G * k * V;
        if constexpr (kEdge) {
          const int left = (l.lead() + l.D - i * V) * static_cast<int>(sizeof(T));
          asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(to + k * pitch), "l"(src),
                       "r"(left < 16 ? left : 16)
                       : "memory");
        } else {
          asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(to + k * pitch), "l"(src) : "memory");
        }
      }
    }
  }
  // What was requested (kAsync), or now.
  __device__ __forceinline__ void open(const char* s, int pt, const T* p, const L& l) {
    if constexpr (kAsync) {
      slot = s;
      pitch = pt;
    } else {
#pragma unroll
      for (int k = 0; k < K; ++k) {
        const int i = l.lane + l.G * k;
        e[k] = i < l.nv ? ld_vec<T, V>(p + i) : Vec<T, V>::zero();
      }
    }
  }
  // Vector k; elements before the row are zeros.
  __device__ __forceinline__ Vec<T, V> vec(int k, const L& l) const {
    if constexpr (!kAsync) return e[k];
    Vec<T, V> v = ld_vec<T, V>(reinterpret_cast<const T*>(slot + k * pitch));
    if (kEdge && k == 0 && l.lead() > l.lane * V) {
      float f[V];
#pragma unroll
      for (int j = 0; j < V; ++j) f[j] = j < l.lead() ? 0.f : v.get(j);
      v = Vec<T, V>::of(f);
    }
    return v;
  }
  // The thread's elements in pairs: 2 p and 2 p + 1.
  __device__ __forceinline__ void pairs(float2 (&out)[K * V / 2], const L& l) const {
    if constexpr (V == 1) {
#pragma unroll
      for (int p = 0; p < K / 2; ++p) out[p] = make_float2(e[2 * p].get(0), e[2 * p + 1].get(0));
    } else {
#pragma unroll
      for (int k = 0; k < K; ++k) {
        const Vec<T, V> v = vec(k, l);
#pragma unroll
        for (int j = 0; j < V / 2; ++j) out[k * (V / 2) + j] = make_float2(v.get(2 * j), v.get(2 * j + 1));
      }
    }
  }
};

// Stores the thread's elements of a row, `from` where its first vector begins; the row's first and last
// vector by element where the row begins or ends inside.
template <typename T, int V, int K, bool kEdge>
__device__ __forceinline__ void store_row(T* from, const float2 (&f)[K * V / 2], const Lay<kEdge>& l) {
  if constexpr (V == 1) {
#pragma unroll
    for (int k = 0; k < K; ++k)
      if (l.lane + l.G * k < l.D) from[l.G * k] = Elem<T>::store(k & 1 ? f[k / 2].y : f[k / 2].x);
  } else {
#pragma unroll
    for (int k = 0; k < K; ++k) {
      const int i = l.lane + l.G * k, c = i * V - l.lead();
      if (i >= l.nv) continue;
      T* p = from + l.G * k * V;
      float o[V];
#pragma unroll
      for (int j = 0; j < V / 2; ++j) o[2 * j] = f[k * (V / 2) + j].x, o[2 * j + 1] = f[k * (V / 2) + j].y;
      if (!kEdge || (c >= 0 && c + V <= l.D)) {
        st_vec<T, V>(p, Vec<T, V>::of(o));
      } else {
#pragma unroll
        for (int j = 0; j < V; ++j)
          if (c + j >= 0 && c + j < l.D) p[j] = Elem<T>::store(o[j]);
      }
    }
  }
}

// The column of the thread's element e (0 .. K V - 1); negative or >= D where there is none.
template <int V, bool kEdge>
__device__ __forceinline__ int column_of(int e, const Lay<kEdge>& l) {
  return (l.lane + l.G * (e / V)) * V - l.lead() + e % V;
}

// Floats of dw (and of db) in a partial row: the columns, and room for a lead.
__host__ __device__ __forceinline__ int partial_pitch(int D) { return D % 8 ? (D + 14) / 8 * 8 : D; }

__device__ __forceinline__ void commit_copies() { asm volatile("cp.async.commit_group;" ::: "memory"); }
// Until all but the newest `stages` - 1 groups of this thread's copies have arrived.
__device__ __forceinline__ void wait_copies(int stages) {
  if (stages >= 2)
    asm volatile("cp.async.wait_group 1;" ::: "memory");
  else
    asm volatile("cp.async.wait_group 0;" ::: "memory");
}

// The thread's columns of a parameter in pairs: kept in registers with 16 elements per thread,
// read again for every row (from the L1 cache) with 32.
template <typename W, int V, int K, bool kEdge>
struct Columns {
  using L = Lay<kEdge>;
  static constexpr bool kKeep = V * K <= 16;
  float2 f[kKeep ? V * K / 2 : 1];
  const W* w;
  float other;
  __device__ __forceinline__ float element(int e, const L& l) const {
    const int c = column_of<V, kEdge>(e, l);
    return w && c >= 0 && c < l.D ? Elem<W>::load(w[c]) : other;
  }
  __device__ __forceinline__ Columns(const W* p, float absent, const L& l) : w(p), other(absent) {
    if constexpr (kKeep) {
#pragma unroll
      for (int i = 0; i < V * K / 2; ++i) f[i] = make_float2(element(2 * i, l), element(2 * i + 1, l));
    }
  }
  __device__ __forceinline__ float2 get(int i, const L& l) const {
    if constexpr (kKeep) return f[i];
    return make_float2(element(2 * i, l), element(2 * i + 1, l));
  }
};

// Zeros in the thread's slots of vectors that do not exist, in `rows` rows of the ring.
template <typename T, int V, int K, bool kEdge>
__device__ __forceinline__ void zero_missing(char* mine, int pitch, int rows, const Lay<kEdge>& l) {
  if constexpr (V > 1) {
    if (l.nv >= l.G * K) return;
    for (int r = 0; r < rows; ++r)
#pragma unroll
      for (int k = 0; k < K; ++k)
        if (l.lane + l.G * k >= l.nv) *reinterpret_cast<uint4*>(mine + (r * K + k) * pitch) = make_uint4(0, 0, 0, 0);
  }
}

// The rows of a tensor in visiting order, for one thread: addresses of its first vector. kPlain: one
// row follows the other, so the address moves by a fixed step; else it is computed for each row.
template <typename T, int V, bool kPlain, bool kEdge>
struct Rows {
  T* at;         // kPlain: of the next visit asked for
  int64_t step;  // elements from a visit of the group to its next
  __device__ __forceinline__ Rows(T* base, const RowMap& m, uint32_t first, uint32_t visits_apart,
                                  const Lay<kEdge>& l) {
    at = base + (kPlain ? static_cast<int64_t>(first) * l.D : 0) - l.lead() + l.lane * V;
    step = static_cast<int64_t>(visits_apart) * l.D;
  }
  __device__ __forceinline__ T* row(int q, const RowMap& m, const Order& o, const Place& p) const {
    return at + (kPlain ? q * step : row_offset(m, o, p));
  }
  __device__ __forceinline__ void advance(int n) {
    if (kPlain) at += n * step;
  }
};

template <bool kPlain>
__device__ __forceinline__ Place visit(const Order& o, uint32_t v) {
  if constexpr (kPlain) return Place{v < o.visits ? v : kNoRow, 0, 0, 0};
  return place_at(o, v);
}

// Forward. kBlock: the block is one group of blockDim.x threads; else groups of G <= 32. A turn of
// the loop takes N rows of each group.
template <typename T, typename W, int V, int K, bool kBlock, int N, bool kPlain, bool kEdge>
__global__ void __launch_bounds__(kBlock ? kMaxBlockGroup : kGroupThreads)
    forward_kernel(const T* __restrict__ x, RowMap xm, Order order, const W* __restrict__ w,
                   const W* __restrict__ b, T* __restrict__ y, float* __restrict__ mean_out,
                   float* __restrict__ rstd_out, int D, int G, int stages, float eps) {
  extern __shared__ __align__(16) char ring[];
  __shared__ float red[128];
  using R = Row<T, V, K, kEdge>;
  using L = Lay<kEdge>;
  constexpr int P = K * V / 2;
  int half = 0;
  const uint32_t per_block = kBlock ? 1u : blockDim.x / G;
  const uint32_t block_first = blockIdx.x * per_block;
  const uint32_t first = kBlock ? block_first : block_first + threadIdx.x / G;
  const uint32_t step = gridDim.x * per_block;
  const int lead = kEdge ? static_cast<int>(first * static_cast<uint32_t>(D) & (V - 1)) : 0;
  const L l = {static_cast<int>(kBlock ? threadIdx.x : (threadIdx.x & (G - 1))),
               kBlock ? static_cast<int>(blockDim.x) : G,
               (lead + D + V - 1) / V, lead, D};
  const bool full = l.nv >= l.G * K;  // every vector of the thread exists
  const int pitch = blockDim.x * R::kBytes, row_bytes = K * pitch, stage_bytes = N * row_bytes;
  char* mine = ring + threadIdx.x * R::kBytes;
  const uint32_t mine_at = static_cast<uint32_t>(__cvta_generic_to_shared(mine));
  const float inv_d = 1.0f / static_cast<float>(D);
  const RowMap ym = {0, 0, D, {}, {}, true};
  Rows<const T, V, kPlain, kEdge> from(x, xm, first, step, l);
  Rows<T, V, true, kEdge> to(y, ym, kPlain ? first : 0, step, l);
  zero_missing<T, V, K>(mine, pitch, stages * N, l);
  auto request = [&](int slot, uint32_t v) {
#pragma unroll
    for (int q = 0; q < N; ++q) {
      const Place at = visit<kPlain>(order, v + q * step);
      if (at.r != kNoRow) R::request(mine_at + slot + q * row_bytes, pitch, from.row(q, xm, order, at), l);
    }
    from.advance(N);
    commit_copies();
  };
  const int last_slot = (stages - 1) * stage_bytes;
  if constexpr (R::kAsync)
    for (int s = 0; s + 1 < stages; ++s) request(s * stage_bytes, first + s * (N * step));
  const Columns<W, V, K, kEdge> wc(w, 1.f, l), bc(b, 0.f, l);
  if constexpr (kBlock) block_sum_init(red);
  int now = 0;  // the slot of this turn, in bytes
  // every group of the block makes the same number of turns, so that shuffles and barriers meet
  for (uint32_t base = block_first, v0 = first; base < order.visits; base += N * step, v0 += N * step) {
    if constexpr (R::kAsync) {
      request(now ? now - stage_bytes : last_slot, v0 + (stages - 1) * (N * step));
      wait_copies(stages);
    }
    uint32_t r[N];
    float2 v[N][P];
    float s[N], sq[N];
#pragma unroll
    for (int q = 0; q < N; ++q) {
      const Place at = visit<kPlain>(order, v0 + q * step);
      r[q] = at.r;
      R row;
      if constexpr (R::kAsync) {
        row.open(mine + now + q * row_bytes, pitch, nullptr, l);
      } else {
        L lq = l;
        if (r[q] == kNoRow) lq.nv = 0;
        row.open(nullptr, 0, r[q] == kNoRow ? x : x + row_offset(xm, order, at), lq);
      }
      row.pairs(v[q], l);
      float2 t = make_float2(0.f, 0.f);
#pragma unroll
      for (int p = 0; p < P; ++p) t = add2(t, v[q][p]);
      s[q] = t.x + t.y;
    }
    now = now == last_slot ? 0 : now + stage_bytes;
    if constexpr (kBlock)
      block_sum<N>(s, red, half);
    else
      group_sum<N>(s, G);
#pragma unroll
    for (int q = 0; q < N; ++q) {
      s[q] *= inv_d;
#pragma unroll
      for (int p = 0; p < P; ++p) v[q][p] = add2(v[q][p], both(-s[q]));
      if (kEdge || !full) {  // elements that do not exist have no deviation
#pragma unroll
        for (int p = 0; p < P; ++p) {
          const int c = column_of<V, kEdge>(2 * p, l), c2 = column_of<V, kEdge>(2 * p + 1, l);
          if (c < 0 || c >= D) v[q][p].x = 0.f;
          if (c2 < 0 || c2 >= D) v[q][p].y = 0.f;
        }
      }
      float2 t = make_float2(0.f, 0.f);
#pragma unroll
      for (int p = 0; p < P; ++p) t = fma2(v[q][p], v[q][p], t);
      sq[q] = t.x + t.y;
    }
    if constexpr (kBlock)
      block_sum<N>(sq, red, half);
    else
      group_sum<N>(sq, G);
#pragma unroll
    for (int q = 0; q < N; ++q) {
      if (r[q] == kNoRow) continue;
      const float rstd = 1.0f / sqrtf(sq[q] * inv_d + eps);
#pragma unroll
      for (int p = 0; p < P; ++p) v[q][p] = fma2(mul2(v[q][p], both(rstd)), wc.get(p, l), bc.get(p, l));
      store_row<T, V, K, kEdge>(kPlain ? to.at + q * to.step : to.at + static_cast<int64_t>(r[q]) * D, v[q], l);
      if (l.lane == 0) {
        mean_out[r[q]] = s[q];
        rstd_out[r[q]] = rstd;
      }
    }
    if (kPlain) to.advance(N);
  }
}

// Backward: dx and, per block, one partial row [dw | db] of 2 D floats. The ring's stage holds N
// x rows, N dy rows and, for each warp (group, where that is smaller), their mean and rstd.
template <typename T, typename W, int V, int K, bool kBlock, int N, bool kPlain, bool kEdge>
__global__ void __launch_bounds__(kBlock ? kMaxBlockGroup : kGroupThreads, kBlock ? 1 : 2)
    backward_kernel(const T* __restrict__ dy, RowMap dm, const T* __restrict__ x, RowMap xm, Order order,
                    const W* __restrict__ w, const float* __restrict__ mean_in, const float* __restrict__ rstd_in,
                    T* __restrict__ dx, float* __restrict__ partial, W* __restrict__ dw, W* __restrict__ db, int D,
                    int G, int stages) {
  extern __shared__ __align__(16) char ring[];
  __shared__ float red[128];
  using R = Row<T, V, K, kEdge>;
  using L = Lay<kEdge>;
  constexpr int P = K * V / 2;
  int half = 0;
  const uint32_t per_block = kBlock ? 1u : blockDim.x / G;
  const uint32_t block_first = blockIdx.x * per_block;
  const uint32_t first = kBlock ? block_first : block_first + threadIdx.x / G;
  const uint32_t step = gridDim.x * per_block;
  const int lead = kEdge ? static_cast<int>(first * static_cast<uint32_t>(D) & (V - 1)) : 0;
  const L l = {static_cast<int>(kBlock ? threadIdx.x : (threadIdx.x & (G - 1))),
               kBlock ? static_cast<int>(blockDim.x) : G,
               (lead + D + V - 1) / V, lead, D};
  const int pitch = blockDim.x * R::kBytes, row_bytes = K * pitch;
  const int share = kBlock ? 32 : G;  // threads that share a copy of the statistics
  const int stats_stage = blockDim.x / share * 2 * N * 4;  // bytes
  const int stage_bytes = 2 * N * row_bytes;
  char* mine = ring + threadIdx.x * R::kBytes;
  const uint32_t mine_at = static_cast<uint32_t>(__cvta_generic_to_shared(mine));
  char* stats = ring + stages * stage_bytes + threadIdx.x / share * (2 * N * 4);
  const uint32_t stats_at = static_cast<uint32_t>(__cvta_generic_to_shared(stats));
  const bool leader = threadIdx.x % share == 0;
  const float inv_d = 1.0f / static_cast<float>(D);
  const RowMap om = {0, 0, D, {}, {}, true};
  Rows<const T, V, kPlain, kEdge> xs(x, xm, first, step, l), gs(dy, dm, first, step, l);
  Rows<T, V, true, kEdge> to(dx, om, kPlain ? first : 0, step, l);
  zero_missing<T, V, K>(mine, pitch, stages * 2 * N, l);
  float2 aw[P], ab[P];
#pragma unroll
  for (int p = 0; p < P; ++p) aw[p] = ab[p] = make_float2(0.f, 0.f);
  auto request = [&](int slot, int stat, uint32_t v) {
#pragma unroll
    for (int q = 0; q < N; ++q) {
      const Place at = visit<kPlain>(order, v + q * step);
      if (at.r == kNoRow) continue;
      R::request(mine_at + slot + 2 * q * row_bytes, pitch, xs.row(q, xm, order, at), l);
      R::request(mine_at + slot + (2 * q + 1) * row_bytes, pitch, gs.row(q, dm, order, at), l);
      if (leader) {
        const uint32_t st = stats_at + stat + 8 * q;
        asm volatile("cp.async.ca.shared.global [%0], [%1], 4;" ::"r"(st), "l"(mean_in + at.r) : "memory");
        asm volatile("cp.async.ca.shared.global [%0], [%1], 4;" ::"r"(st + 4), "l"(rstd_in + at.r) : "memory");
      }
    }
    xs.advance(N);
    gs.advance(N);
    commit_copies();
  };
  const int last_slot = (stages - 1) * stage_bytes, last_stat = (stages - 1) * stats_stage;
  if constexpr (R::kAsync)
    for (int s = 0; s + 1 < stages; ++s) request(s * stage_bytes, s * stats_stage, first + s * (N * step));
  const Columns<W, V, K, kEdge> wc(w, 1.f, l);
  if constexpr (kBlock) block_sum_init(red);
  int now = 0, stat = 0;  // the slots of this turn, in bytes
  for (uint32_t base = block_first, v0 = first; base < order.visits; base += N * step, v0 += N * step) {
    if constexpr (R::kAsync) {
      request(now ? now - stage_bytes : last_slot, now ? stat - stats_stage : last_stat,
              v0 + (stages - 1) * (N * step));
      wait_copies(stages);
      __syncwarp();  // the statistics come from the first lane's copies
    }
    uint32_t r[N];
    R xr[N], gr[N];
    float mean[N], rstd[N], c[2 * N];
#pragma unroll
    for (int q = 0; q < N; ++q) {
      const Place at = visit<kPlain>(order, v0 + q * step);
      r[q] = at.r;
      const bool valid = r[q] != kNoRow;
      mean[q] = rstd[q] = 0.f;
      if constexpr (R::kAsync) {
        const float2 st = *reinterpret_cast<const float2*>(stats + stat + 8 * q);
        if (valid) mean[q] = st.x, rstd[q] = st.y;
        xr[q].open(mine + now + 2 * q * row_bytes, pitch, nullptr, l);
        gr[q].open(mine + now + (2 * q + 1) * row_bytes, pitch, nullptr, l);
      } else {
        L lq = l;
        if (!valid) lq.nv = 0;
        if (valid) {
          mean[q] = __ldg(mean_in + r[q]);
          rstd[q] = __ldg(rstd_in + r[q]);
        }
        xr[q].open(nullptr, 0, valid ? x + row_offset(xm, order, at) : x, lq);
        gr[q].open(nullptr, 0, valid ? dy + row_offset(dm, order, at) : dy, lq);
      }
      c[2 * q] = c[2 * q + 1] = 0.f;
      if (!valid) continue;
      float2 xp[P], gp[P], c1 = make_float2(0.f, 0.f), c2 = c1;
      xr[q].pairs(xp, l);
      gr[q].pairs(gp, l);
#pragma unroll
      for (int p = 0; p < P; ++p) {
        const float2 xh = mul2(add2(xp[p], both(-mean[q])), both(rstd[q]));
        const float2 g = mul2(gp[p], wc.get(p, l));
        aw[p] = fma2(gp[p], xh, aw[p]);
        ab[p] = add2(ab[p], gp[p]);
        c1 = add2(c1, g);
        c2 = fma2(g, xh, c2);
      }
      c[2 * q] = c1.x + c1.y;
      c[2 * q + 1] = c2.x + c2.y;
    }
    if constexpr (kBlock)
      block_sum<2 * N>(c, red, half);
    else
      group_sum<2 * N>(c, G);
#pragma unroll
    for (int q = 0; q < N; ++q) {
      if (r[q] == kNoRow) continue;
      const float c1 = c[2 * q] * inv_d, c2 = c[2 * q + 1] * inv_d;
      float2 xp[P], gp[P];
      xr[q].pairs(xp, l);
      gr[q].pairs(gp, l);
#pragma unroll
      for (int p = 0; p < P; ++p) {
        const float2 xh = mul2(add2(xp[p], both(-mean[q])), both(rstd[q]));
        const float2 g = rounded_mul2(gp[p], wc.get(p, l));
        xp[p] = mul2(both(rstd[q]), fma2(xh, both(-c2), add2(g, both(-c1))));
      }
      store_row<T, V, K, kEdge>(kPlain ? to.at + q * to.step : to.at + static_cast<int64_t>(r[q]) * D, xp, l);
    }
    if (kPlain) to.advance(N);
    now = now == last_slot ? 0 : now + stage_bytes;
    stat = now ? stat + stats_stage : 0;
  }
  const bool direct = dw || db;  // the grid is one cluster, which joins its blocks' sums itself
  if (!partial && !direct) return;
  const int ld = partial_pitch(D);
  float* pw = partial + static_cast<int64_t>(blockIdx.x) * 2 * ld;
  if (kBlock && !direct) {
    // as the vectors lie: column c at c + lead
#pragma unroll
    for (int k = 0; k < K; ++k) {
      const int i = l.lane + l.G * k;
      if (i >= l.nv) continue;
      if constexpr (V == 1) {
        pw[i] = k & 1 ? aw[k / 2].y : aw[k / 2].x;
        pw[ld + i] = k & 1 ? ab[k / 2].y : ab[k / 2].x;
      } else {
#pragma unroll
        for (int j = 0; j < V / 2; j += 2) {
          const int p = k * (V / 2) + j;
          *reinterpret_cast<float4*>(pw + i * V + 2 * j) = make_float4(aw[p].x, aw[p].y, aw[p + 1].x, aw[p + 1].y);
          *reinterpret_cast<float4*>(pw + ld + i * V + 2 * j) = make_float4(ab[p].x, ab[p].y, ab[p + 1].x, ab[p + 1].y);
        }
      }
    }
    return;
  }
  // every warp adds its groups in the ring's memory, then the block the warps. Groups that lie
  // alike are added by shuffles (with a lead, the groups of a warp lie differently); a block that
  // is one group has its sums in its threads.
  wait_copies(1);
  __syncthreads();
  const int warp = threadIdx.x >> 5, parts = kBlock ? 1 : blockDim.x >> 5;
  float* cols = reinterpret_cast<float*>(ring) + (kBlock ? 0 : warp * 2 * D);
  if (!kBlock && !kEdge) {
#pragma unroll
    for (int p = 0; p < P; ++p)
      for (int o = G; o < 32; o <<= 1) {
        aw[p].x += __shfl_xor_sync(0xffffffffu, aw[p].x, o);
        aw[p].y += __shfl_xor_sync(0xffffffffu, aw[p].y, o);
        ab[p].x += __shfl_xor_sync(0xffffffffu, ab[p].x, o);
        ab[p].y += __shfl_xor_sync(0xffffffffu, ab[p].y, o);
      }
  } else if (!kBlock) {
    for (int i = threadIdx.x & 31; i < 2 * D; i += 32) cols[i] = 0.f;
    __syncwarp();
  }
  for (int t = 0; t < (!kBlock && kEdge ? 32 / G : 1); ++t) {
    if (kBlock || static_cast<int>(threadIdx.x & 31) / G == t)
#pragma unroll
      for (int e = 0; e < K * V; ++e) {
        const int col = column_of<V, kEdge>(e, l);
        if (col < 0 || col >= D) continue;
        const bool more = !kBlock && kEdge;
        cols[col] = (more ? cols[col] : 0.f) + (e & 1 ? aw[e / 2].y : aw[e / 2].x);
        cols[D + col] = (more ? cols[D + col] : 0.f) + (e & 1 ? ab[e / 2].y : ab[e / 2].x);
      }
    __syncwarp();
  }
  __syncthreads();
  cols = reinterpret_cast<float*>(ring);
  for (int i = threadIdx.x; i < 2 * D && (parts > 1 || !direct); i += blockDim.x) {
    float t = 0.f;
    for (int q = 0; q < parts; ++q) t += cols[q * 2 * D + i];
    if (direct)
      cols[i] = t;
    else
      pw[i < D ? i : i - D + ld] = t;
  }
  if (!direct) return;
  namespace cg = cooperative_groups;
  cg::cluster_group cluster = cg::this_cluster();
  const int blocks = static_cast<int>(cluster.num_blocks());
  cluster.sync();
  for (int i = cluster.block_rank() * blockDim.x + threadIdx.x; i < 2 * D; i += blocks * blockDim.x) {
    float v[kMaxCluster], t = 0.f;  // all on their way together
#pragma unroll
    for (int r = 0; r < kMaxCluster; ++r) v[r] = r < blocks ? cluster.map_shared_rank(cols, r)[i] : 0.f;
#pragma unroll
    for (int r = 0; r < kMaxCluster; ++r) t += v[r];
    if (i < D) {
      if (dw) dw[i] = Elem<W>::store(t);
    } else if (db) {
      db[i - D] = Elem<W>::store(t);
    }
  }
  cluster.sync();  // nobody leaves while others read its memory
}

// dw, db: the sum of `n` partial rows of two times `ld` floats, in a fixed order, as a tree. Partial
// row i holds column c at c + (i D mod V) (shift: V - 1, or 0). A warp covers kCols columns of
// 32 / kCols rows at a time; blocks of dw come first, then those of db.
template <typename W, int kCols>
__global__ void __launch_bounds__(kJoinThreads)
    join_kernel(const float* __restrict__ partial, int n, int D, int ld, uint32_t shift, W* __restrict__ dw,
                W* __restrict__ db) {
  wait_previous_kernel();
  constexpr int kWarps = kJoinThreads / 32, kRows = 32 / kCols;
  __shared__ float part[kWarps][kCols];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int half = (D + kCols - 1) / kCols;  // blocks
  const bool second = static_cast<int>(blockIdx.x) >= half;
  const int c0 = (static_cast<int>(blockIdx.x) - (second ? half : 0)) * kCols;
  W* out = second ? db : dw;
  if (!out) return;
  const int c = c0 + (lane & (kCols - 1));
  float s = 0.f;
  if (c < D) {
    constexpr int kStep = kWarps * kRows;  // a multiple of V: all rows of a thread lie alike
    int i = warp * kRows + lane / kCols;
    const int64_t row = 2 * static_cast<int64_t>(ld), apart = kStep * row;
    const float* p =
        partial + c + (second ? ld : 0) + i * row + (static_cast<uint32_t>(i) * static_cast<uint32_t>(D) & shift);
    for (; i + 3 * kStep < n; i += 4 * kStep, p += 4 * apart) s += (p[0] + p[apart]) + (p[2 * apart] + p[3 * apart]);
    for (; i < n; i += kStep, p += apart) s += *p;
  }
#pragma unroll
  for (int o = kCols; o < 32; o <<= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
  if (lane < kCols) part[warp][lane] = s;
  __syncthreads();
  // warp k adds column k over the warps
  for (int k = warp; k < kCols; k += kWarps) {
    float t = lane < kWarps ? part[lane][k] : 0.f;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) t += __shfl_xor_sync(0xffffffffu, t, o);
    if (lane == 0 && c0 + k < D) out[c0 + k] = Elem<W>::store(t);
  }
}

// ---- Rows of more than 16384 elements (a vector less where none divides the width) -----------------
// By element, a row read again for each of its sums: far from HBM's rate. 4096 x 65536 bf16: forward
// 1170 us, backward 1410 (164 and 245 at the copy's rate); 64 x 65536: 63 and 103; 64 x 2^20 fp32:
// 2810 and 2730 (82 and 123).

template <typename T, typename W>
__global__ void __launch_bounds__(kMaxBlockGroup)
    forward_wide_kernel(const T* __restrict__ x, RowMap xm, const W* __restrict__ w, const W* __restrict__ b,
                        T* __restrict__ y, float* __restrict__ mean_out, float* __restrict__ rstd_out, uint32_t rows,
                        int D, float eps) {
  __shared__ float red[128];
  block_sum_init(red);
  int half = 0;
  const float inv_d = 1.0f / static_cast<float>(D);
  for (uint64_t r = blockIdx.x; r < rows; r += gridDim.x) {
    const T* xr = x + row_offset(xm, static_cast<uint32_t>(r));
    float s[1] = {0.f}, q[1] = {0.f};
    for (int c = threadIdx.x; c < D; c += blockDim.x) s[0] += Elem<T>::load(xr[c]);
    block_sum<1>(s, red, half);
    const float mean = s[0] * inv_d;
    for (int c = threadIdx.x; c < D; c += blockDim.x) {
      const float d = Elem<T>::load(xr[c]) - mean;
      q[0] = fmaf(d, d, q[0]);
    }
    block_sum<1>(q, red, half);
    const float rstd = 1.0f / sqrtf(q[0] * inv_d + eps);
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
  __shared__ float red[128];
  block_sum_init(red);
  int half = 0;
  const float inv_d = 1.0f / static_cast<float>(D);
  for (uint64_t r = blockIdx.x; r < rows; r += gridDim.x) {
    const T* xr = x + row_offset(xm, static_cast<uint32_t>(r));
    const T* gr = dy + row_offset(dm, static_cast<uint32_t>(r));
    const float mean = mean_in[r], rstd = rstd_in[r];
    float t[2] = {0.f, 0.f};
    for (int c = threadIdx.x; c < D; c += blockDim.x) {
      const float g = __fmul_rn(Elem<T>::load(gr[c]), w ? Elem<W>::load(w[c]) : 1.f);
      t[0] += g;
      t[1] = fmaf(g, (Elem<T>::load(xr[c]) - mean) * rstd, t[1]);
    }
    block_sum<2>(t, red, half);
    T* dr = dx + static_cast<int64_t>(r) * D;
    for (int c = threadIdx.x; c < D; c += blockDim.x) {
      const float g = __fmul_rn(Elem<T>::load(gr[c]), w ? Elem<W>::load(w[c]) : 1.f);
      const float xh = (Elem<T>::load(xr[c]) - mean) * rstd;
      dr[c] = Elem<T>::store(rstd * ((g - t[0] * inv_d) - xh * (t[1] * inv_d)));
    }
  }
}

// A sum in fp32 with what its additions rounded off beside it (Knuth's two-sum).
struct LongSum {
  float hi = 0.f, lo = 0.f;
  __device__ __forceinline__ void add(float v) {
    const float s = hi + v, back = s - hi;
    lo += (hi - (s - back)) + (v - back);
    hi = s;
  }
  __device__ __forceinline__ float value() const { return hi + lo; }
};

// Partial [dw | db] of the rows [y * per, (y + 1) * per), one column per thread. `per` grows with the
// rows: from 16 rows on (kLong) sixteen are added one on another, and the sixteens in a LongSum. That
// costs nothing (4096 x 65536 bf16, the whole backward: 1410 us, 1412 with one chain); sums in 64 bits
// cost 4%, and so would the registers of the long form for few rows (64 x 2^20 fp32: 2723 us, not 2840).
constexpr uint32_t kChain = 16;

template <typename T, bool kLong>
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
  if constexpr (kLong) {
    LongSum tw, tb;
    uint64_t r = r0;
    while (r1 - r >= kChain) {
#pragma unroll 16
      for (uint32_t u = 0; u < kChain; ++u, ++r) {
        const float d = Elem<T>::load(dy[row_offset(dm, static_cast<uint32_t>(r)) + c]);
        const float v = Elem<T>::load(x[row_offset(xm, static_cast<uint32_t>(r)) + c]);
        sw = fmaf(d, (v - mean_in[r]) * rstd_in[r], sw);
        sb += d;
      }
      tw.add(sw);
      tb.add(sb);
      sw = sb = 0.f;
    }
#pragma unroll 4
    for (; r < r1; ++r) {
      const float d = Elem<T>::load(dy[row_offset(dm, static_cast<uint32_t>(r)) + c]);
      const float v = Elem<T>::load(x[row_offset(xm, static_cast<uint32_t>(r)) + c]);
      sw = fmaf(d, (v - mean_in[r]) * rstd_in[r], sw);
      sb += d;
    }
    tw.add(sw);
    tb.add(sb);
    sw = tw.value();
    sb = tb.value();
  } else {
    for (uint64_t r = r0; r < r1; ++r) {
      const float d = Elem<T>::load(dy[row_offset(dm, static_cast<uint32_t>(r)) + c]);
      const float v = Elem<T>::load(x[row_offset(xm, static_cast<uint32_t>(r)) + c]);
      sw = fmaf(d, (v - mean_in[r]) * rstd_in[r], sw);
      sb += d;
    }
  }
  const int ld = partial_pitch(D);
  float* p = partial + static_cast<int64_t>(slab) * 2 * ld;
  p[c] = sw;
  p[ld + c] = sb;
}

// ---- Host ---------------------------------------------------------------------------------

constexpr int64_t kWideSlabs = 64;

struct Shape {
  int G;
  bool block, thirty_two, wide;
};

// Threads per row and elements per thread (see the file comment). A row whose width no vector
// divides takes up to a vector more.
Shape choose(int64_t D) {
  Shape s = {};
  const int64_t cover = D + (D % 8 ? 7 : 0);
  s.wide = cover > 16384;
  s.thirty_two = cover > 8192;
  const int64_t per = s.thirty_two ? 32 : 16;
  const int64_t need = (cover + per - 1) / per;  // threads
  s.block = need > 32;
  if (s.block)
    s.G = static_cast<int>((need + 31) / 32 * 32);
  else
    for (s.G = 1; s.G < need;) s.G <<= 1;
  return s;
}

// Partial rows that the workspace holds: as many as the backward has blocks, which are at most
// 1024 threads' worth per SM (16 blocks) on the 148 SMs of this family, and no more than rows.
int64_t max_partials(int64_t rows, int64_t D) {
  const Shape s = choose(D);
  if (s.wide) return rows < kWideSlabs ? rows : kWideSlabs;
  const int threads = s.block ? s.G : kGroupThreads;
  int64_t cap = 1024 / threads;
  cap = 148 * (cap > 16 ? 16 : cap);
  return rows < cap ? rows : cap;
}

struct Args {
  const void *x, *dy, *w, *b;
  RowMap xm, dm;
  Order order;
  void *y, *dx, *dw, *db;
  float *mean, *rstd, *partial;
  int64_t rows;
  int D;
  float eps;
  cudaStream_t st;
};

// The ring: stages, bytes, and the blocks of an SM. What is on its way should be about what HBM
// needs for its latency, 64 KB an SM; 16-bit rows take what there is, as their arithmetic takes longer.
// More costs in fp32: reads far ahead of the writes leave the DRAM pages that the writes need (512 x
// 512 x 128, backward: 66 us with 64 KB an SM, 70 with 200 KB; 4096 x 4096 bf16: 28.8 with 128 KB,
// 26.8 with 200 KB).
struct Ring {
  int stages, bytes, blocks;
};
template <typename R>
Ring ring_for(int threads, int K, int tensors, int most_blocks, int extra, size_t elem_bytes) {
  Ring r = {1, 0, most_blocks < 1 ? 1 : most_blocks};
  const int stage = tensors * K * threads * R::kBytes + extra;
  if (R::kAsync) {
    const int want = (elem_bytes == 4 ? 64 : 200) * 1024 / (kMaxStages * stage);
    if (r.blocks > want) r.blocks = want < 1 ? 1 : want;
    r.stages = kRingBytes / r.blocks / stage;
    r.stages = r.stages < 1 ? 1 : r.stages > kMaxStages ? kMaxStages : r.stages;
    r.bytes = r.stages * stage;
  }
  return r;
}

// Resident blocks of a kernel by block size (multiples of 32), asked for once.
constexpr int kBlockSizes = kMaxBlockGroup / 32 + 1;
template <typename F>
int64_t cached_residency(std::atomic<int64_t>* cache, F kernel, int threads, int smem) {
  std::atomic<int64_t>& c = cache[threads / 32];
  int64_t v = c.load(std::memory_order_relaxed);
  if (!v) c.store(v = resident_blocks(kernel, threads, smem), std::memory_order_relaxed);
  return v;
}

// Blocks for `visits` rows in turns of N per group: all that fit the device at once. `edge`: rows
// begin inside vectors, so a group's rows have to lie a multiple of eight apart: either the
// groups of all blocks together are one, or no group has a second row.
int64_t grid_for(int64_t visits, int64_t per, int N, int64_t cap, bool edge) {
  const int64_t turn = per * N;
  int64_t blocks = (visits + turn - 1) / turn;
  if (blocks > cap) blocks = cap;
  if (!edge || per % 8 == 0) return blocks;
  return blocks >= 8 ? blocks & ~int64_t(7) : visits;
}

template <typename T, typename W, int V, int K, bool kBlock, int N, bool kPlain, bool kEdge>
int run_forward(const Args& a, const Shape& s) {
  auto kernel = forward_kernel<T, W, V, K, kBlock, N, kPlain, kEdge>;
  using R = Row<T, V, K, kEdge>;
  const int threads = kBlock ? s.G : kGroupThreads;
  const Ring ring = ring_for<R>(threads, K, N, 1024 / threads, 0, sizeof(T));
  if (int e = ensure_smem(reinterpret_cast<const void*>(kernel), kRingBytes)) return e;
  static std::atomic<int64_t> cache[kBlockSizes];
  int64_t cap = cached_residency(cache, kernel, threads, ring.bytes);
  const int64_t in_flight = static_cast<int64_t>(num_sms()) * ring.blocks;
  if (R::kAsync && cap > in_flight) cap = in_flight;
  const int64_t blocks = grid_for(a.order.visits, kBlock ? 1 : kGroupThreads / s.G, N, cap, kEdge);
  return launch("layernorm forward", kernel, blocks, threads, ring.bytes, a.st, false, static_cast<const T*>(a.x),
                a.xm, a.order, static_cast<const W*>(a.w), static_cast<const W*>(a.b), static_cast<T*>(a.y), a.mean,
                a.rstd, a.D, s.G, ring.stages, a.eps);
}

template <typename W>
int run_join(const Args& a, int64_t n, int shift) {
  // eight columns a block until that makes more blocks than the device takes at once
  const bool narrow = a.D <= 8 * 148;
  const int cols = narrow ? 8 : 32;
  return launch("layernorm gradient join", narrow ? join_kernel<W, 8> : join_kernel<W, 32>,
                2 * ((static_cast<int64_t>(a.D) + cols - 1) / cols), kJoinThreads, 0, a.st, true,
                static_cast<const float*>(a.partial), static_cast<int>(n), a.D, partial_pitch(a.D),
                static_cast<uint32_t>(shift), static_cast<W*>(a.dw), static_cast<W*>(a.db));
}

template <typename T, typename W, int V, int K, bool kBlock, int N, bool kPlain, bool kEdge>
int run_backward(const Args& a, const Shape& s) {
  auto kernel = backward_kernel<T, W, V, K, kBlock, N, kPlain, kEdge>;
  using R = Row<T, V, K, kEdge>;
  const int threads = kBlock ? s.G : kGroupThreads;
  // a stage's statistics: 8 bytes a row for each warp or smaller group; the ring also joins the groups
  Ring ring = ring_for<R>(threads, K, 2 * N, 512 / threads, threads / (kBlock ? 32 : s.G) * 8 * N, sizeof(T));
  const int join_bytes = kGroupThreads / 32 * 2 * a.D * 4;
  if (!kBlock && ring.bytes < join_bytes) ring.bytes = join_bytes;
  if (kBlock && ring.bytes < 2 * a.D * 4) ring.bytes = 2 * a.D * 4;
  if (int e = ensure_smem(reinterpret_cast<const void*>(kernel), kRingBytes)) return e;
  static std::atomic<int64_t> cache[kBlockSizes];
  int64_t cap = cached_residency(cache, kernel, threads, ring.bytes);
  const int64_t in_flight = static_cast<int64_t>(num_sms()) * ring.blocks;
  if (R::kAsync && cap > in_flight) cap = in_flight;
  const int64_t most = max_partials(a.rows, a.D);
  if (cap > most) cap = most;
  const int64_t blocks = grid_for(a.order.visits, kBlock ? 1 : kGroupThreads / s.G, N, cap, kEdge);
  // Up to eight blocks are one cluster, which needs neither a second launch nor partial rows.
  if (a.partial && blocks <= kMaxCluster)
    return launch_clusters("layernorm backward", kernel, blocks, threads, ring.bytes, static_cast<int>(blocks), a.st,
                           static_cast<const T*>(a.dy), a.dm, static_cast<const T*>(a.x), a.xm, a.order,
                           static_cast<const W*>(a.w), static_cast<const float*>(a.mean),
                           static_cast<const float*>(a.rstd), static_cast<T*>(a.dx), static_cast<float*>(nullptr),
                           static_cast<W*>(a.dw), static_cast<W*>(a.db), a.D, s.G, ring.stages);
  if (int e = launch("layernorm backward", kernel, blocks, threads, ring.bytes, a.st, false,
                     static_cast<const T*>(a.dy), a.dm, static_cast<const T*>(a.x), a.xm, a.order,
                     static_cast<const W*>(a.w), static_cast<const float*>(a.mean),
                     static_cast<const float*>(a.rstd), static_cast<T*>(a.dx), a.partial, static_cast<W*>(nullptr),
                     static_cast<W*>(nullptr), a.D, s.G, ring.stages))
    return e;
  return a.partial ? run_join<W>(a, blocks, kBlock && kEdge ? V - 1 : 0) : GTK_OK;
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
  auto columns = per >= kChain ? columns_wide_kernel<T, true> : columns_wide_kernel<T, false>;
  if (int e = launch("layernorm weight gradient", columns, slabs * col_blocks, 256, 0, a.st, false,
                     static_cast<const T*>(a.dy), a.dm, static_cast<const T*>(a.x), a.xm,
                     static_cast<const float*>(a.mean), static_cast<const float*>(a.rstd), a.partial, rows, per, a.D,
                     col_blocks))
    return e;
  return run_join<W>(a, slabs, 0);
}

template <typename T, typename W, int V, int K, bool kBlock, int N, bool kPlain, bool kEdge>
int run_one(const Args& a, const Shape& s, bool backward) {
  return backward ? run_backward<T, W, V, K, kBlock, N, kPlain, kEdge>(a, s)
                  : run_forward<T, W, V, K, kBlock, N, kPlain, kEdge>(a, s);
}

// Vectors of 16 bytes.
template <typename T, typename W, bool kPlain, bool kEdge>
int run_vectors(const Args& a, const Shape& s, bool backward) {
  constexpr int V = 16 / static_cast<int>(sizeof(T));
  if (s.thirty_two) return run_one<T, W, V, 32 / V, true, 1, kPlain, kEdge>(a, s, backward);
  if (!s.block) return run_one<T, W, V, 16 / V, false, 1, kPlain, kEdge>(a, s, backward);
  // two rows a turn, once there are more rows than blocks and where two turns of them fit the ring
  if (2 * 2 * (backward ? 2 : 1) * (16 / V) * s.G * 16 > kRingBytes - 4096 ||
      a.rows <= static_cast<int64_t>(num_sms()) * (512 / s.G))
    return run_one<T, W, V, 16 / V, true, 1, kPlain, kEdge>(a, s, backward);
  return run_one<T, W, V, 16 / V, true, 2, kPlain, kEdge>(a, s, backward);
}

template <typename T, typename W>
int run_typed(const Args& a, bool vec, bool backward) {
  const Shape s = choose(a.D);
  if (s.wide) return run_wide<T, W>(a, backward);
  if (vec) {
    const bool plain = a.xm.plain && (!backward || a.dm.plain);
    if (a.D % (16 / static_cast<int>(sizeof(T)))) return run_vectors<T, W, true, true>(a, s, backward);
    return plain ? run_vectors<T, W, true, false>(a, s, backward) : run_vectors<T, W, false, false>(a, s, backward);
  }
  if (s.thirty_two) return run_one<T, W, 1, 32, true, 1, false, false>(a, s, backward);
  if (s.block) return run_one<T, W, 1, 16, true, 1, false, false>(a, s, backward);
  return run_one<T, W, 1, 16, false, 1, false, false>(a, s, backward);
}

int run(const Args& a, int xt, int wt, bool vec, bool backward) {
  if (xt == GTK_F32) return run_typed<float, float>(a, vec, backward);
  if (xt == GTK_BF16)
    return wt == GTK_F32 ? run_typed<__nv_bfloat16, float>(a, vec, backward)
                         : run_typed<__nv_bfloat16, __nv_bfloat16>(a, vec, backward);
  return wt == GTK_F32 ? run_typed<__half, float>(a, vec, backward) : run_typed<__half, __half>(a, vec, backward);
}

// Checks a tensor's leading axes and fills its RowMap; `vec` is cleared when its rows cannot be
// read in aligned 16-byte vectors: they begin anywhere, or strided rows do not all begin on a
// boundary.
int row_map(const gtk_rows* v, const void* base, int64_t rows, int64_t D, size_t bytes, const char* what, RowMap* out,
            bool* vec) {
  if (!aligned16(base)) *vec = false;
  if (!v) {
    *out = RowMap{0, 0, D, divisor(1), divisor(1), true};
    return GTK_OK;
  }
  if ((D * bytes) % 16) *vec = false;
  for (int i = 0; i < 3; ++i) {
    if (v->size[i] < 1 || v->size[i] > rows)
      return fail(GTK_ERR_INVALID_ARG, std::string("layernorm: bad leading sizes of ") + what);
    if (v->stride[i] < 0) return fail(GTK_ERR_INVALID_ARG, std::string("layernorm: negative stride of ") + what);
    if (v->size[i] > 1 && (v->stride[i] * static_cast<int64_t>(bytes)) % 16) *vec = false;
  }
  if (v->size[0] * v->size[1] > rows || v->size[0] * v->size[1] * v->size[2] != rows)
    return fail(GTK_ERR_INVALID_ARG, std::string("layernorm: the leading sizes of ") + what + " do not make up rows");
  *out = RowMap{v->stride[0], v->stride[1], v->stride[2], divisor(static_cast<uint32_t>(v->size[1])),
                divisor(static_cast<uint32_t>(v->size[2])), false};
  return GTK_OK;
}

// Tiles where a tensor's rows lie closer along its second axis than along its third.
Order order_for(int64_t rows, const RowMap& a, const RowMap* b) {
  Order o = {divisor(1), divisor(1), 0, 0, static_cast<uint32_t>(rows), false};
  for (const RowMap* m : {&a, b}) {
    if (!m || m->plain || m->n2.d < 4 || m->n1.d < 8 || m->s1 >= m->s2) continue;
    const uint64_t t1 = (m->n1.d + 7) / 8, t2 = (m->n2.d + 3) / 4;
    const uint64_t planes = rows / (static_cast<uint64_t>(m->n1.d) * m->n2.d);
    if (planes * t1 * t2 * 32 >= (uint64_t(1) << 31)) continue;
    return Order{divisor(static_cast<uint32_t>(t1)), divisor(static_cast<uint32_t>(t2)), m->n1.d, m->n2.d,
                 static_cast<uint32_t>(planes * t1 * t2 * 32), true};
  }
  return o;
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
  return static_cast<size_t>(ln::max_partials(rows, D)) * 2 * ln::partial_pitch(static_cast<int>(D)) * sizeof(float);
}

int gtk_layernorm_forward(const void* x, const gtk_rows* x_rows, int x_dtype, const void* weight, const void* bias,
                          int w_dtype, void* y, float* mean, float* rstd, int64_t rows, int64_t D, float eps,
                          void* stream) try {
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
  a.order = ln::order_for(rows, a.xm, nullptr);
  if (int e = check_device()) return e;
  a.x = x, a.w = weight, a.b = bias, a.y = y, a.mean = mean, a.rstd = rstd;
  a.rows = rows, a.D = static_cast<int>(D), a.eps = eps, a.st = static_cast<cudaStream_t>(stream);
  return ln::run(a, x_dtype, w_dtype, vec, false);
} catch (...) {
  return fail_no_memory();
}

int gtk_layernorm_backward(const void* dy, const gtk_rows* dy_rows, const void* x, const gtk_rows* x_rows,
                           int x_dtype, const void* weight, int w_dtype, const float* mean, const float* rstd,
                           void* dx, void* dweight, void* dbias, void* workspace, size_t workspace_bytes,
                           int64_t rows, int64_t D, void* stream) try {
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
  // vectors are laid over the rows of all tensors at once: with a strided tensor, rows that all
  // begin on a boundary
  if ((x_rows || dy_rows) && (D * dtype_bytes(x_dtype)) % 16) vec = false;
  a.order = ln::order_for(rows, a.xm, &a.dm);
  if (int e = check_device()) return e;
  a.x = x, a.dy = dy, a.w = weight, a.dx = dx, a.dw = dweight, a.db = dbias;
  a.mean = const_cast<float*>(mean), a.rstd = const_cast<float*>(rstd);
  a.partial = params ? static_cast<float*>(workspace) : nullptr;
  a.rows = rows, a.D = static_cast<int>(D), a.st = static_cast<cudaStream_t>(stream);
  return ln::run(a, x_dtype, w_dtype, vec, true);
} catch (...) {
  return fail_no_memory();
}

}  // extern "C"
