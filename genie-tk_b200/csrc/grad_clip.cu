// The global norm of many gradients, and clipping by it:
//
//   norm = (sum over all elements g^2)^1/2   (or max |g|)
//   k    = min(1, max_norm / (norm + 1e-6))
//   out  = k g                               (in place, or to other tensors of g's type or fp32)
//
// k is NaN when the norm is (every output becomes NaN) and 0 when the norm is infinite, the
// same as torch.nn.utils.clip_grad_norm_.
//
// What bounds it: HBM, and for the gradients of a small model the host and the launches. Two
// launches: clip_norm_kernel reads the gradients once and leaves one partial per block;
// clip_scale_kernel adds the partials (every block the same sum, in the same order) and scales.
// The list of tensors travels in the first kernel's parameters (24 bytes a tensor, up to 1000
// tensors a launch), which writes it to the workspace for the second: there is no table to copy
// to the device and nothing to keep alive behind the call.
//
// The tensors are cut into chunks, which the blocks take in turn, each with a search of the table:
// the device then reads one stretch of memory at a time. The second kernel walks the chunks
// backwards: what the first one read last is still in the L2 cache then (24 Mi fp32 elements into another
// tensor, from a graph: 43.6 us instead of 51.6; 2^27 bf16 ones into fp32 182 instead of 187). In place
// and with k = 1 it has nothing to do and returns. In place and with k < 1 the gradients of a
// small model take 6.3 us (58 tensors, from a graph), 2^25 fp32 elements in 256 tensors 58 us.
//
// Squares are summed 16 at a time in fp32 and from there on in 64 bits. Where such a sum is not
// a plain number (it overflowed, or is so small that its squares may have underflowed) the 16
// are squared in 64 bits, so the norm holds for gradients of any magnitude.
#include <algorithm>
#include <vector>

#include "train_common.cuh"

namespace gtk {
namespace clip {

constexpr int kThreads = 256;
// Elements per thread and chunk. Few elements in all are cut finely, to spread them over the
// device; many coarsely, so that a thread has 128 bytes in flight (see `coarse` below).
constexpr int kFine = 16, kCoarse = 64;  // chunks of 2^12 and 2^14 elements
constexpr int kFineBlocks = 8, kCoarseBlocks = 4;  // per SM
constexpr int kBlocksPerSm = kFineBlocks;
constexpr int kMaxBlocks = 148 * kBlocksPerSm;  // partials per launch
constexpr int kMaxTensors = 1000;             // of one launch (24,000 of the 32,764 parameter bytes)
constexpr float kEps = 1e-6f;

struct Tensor {
  const void* in;
  void* out;
  uint32_t first_chunk;  // of the tensor, counted over the launch
  uint16_t last_len;     // elements of its last chunk, from 1 on
  uint8_t in_type, out_type;
};
static_assert(sizeof(Tensor) == 24, "the parameter table's size");

// Chunks begin on 16-byte boundaries of the gradient: they are counted from the boundary at or
// before its first element, `lead` elements earlier, and the first chunk is that much shorter.
__host__ __device__ __forceinline__ int lead_of(const void* in, int type) {
  return static_cast<int>((reinterpret_cast<uintptr_t>(in) & 15u) / (type == GTK_F32 ? 4 : 2));
}

struct Span {
  int64_t off;  // of the chunk's first element in the tensor
  int n;
};
// Chunk i (of `size` elements) of a tensor; `last`: its last one.
__device__ __forceinline__ Span span_of(const Tensor& e, uint32_t i, bool last, int size) {
  const int lead = lead_of(e.in, e.in_type);
  Span s;
  s.off = i ? static_cast<int64_t>(i) * size - lead : 0;
  s.n = last ? e.last_len : i ? size : size - lead;
  return s;
}

template <int N>
struct Table {
  Tensor t[N];
  int n;
  uint32_t chunks;  // of all tensors
};

// What the second kernel needs of a launch's table, in the workspace.
struct Shadow {
  Tensor t[kMaxTensors];
};

// The tensor that holds chunk c: first(i) is ascending in i < n.
template <typename F>
__device__ __forceinline__ int find(F first, int n, uint32_t c) {
  int lo = 0, hi = n - 1;
  while (lo < hi) {
    const int mid = (lo + hi + 1) >> 1;
    if (first(mid) <= c)
      lo = mid;
    else
      hi = mid - 1;
  }
  return lo;
}

// |v| as an ordered integer, in which NaN is above infinity.
__device__ __forceinline__ uint32_t magnitude(float v) { return __float_as_uint(v) & 0x7fffffffu; }

__device__ __forceinline__ double join(double a, double b, bool inf_norm) {
  if (!inf_norm) return a + b;
  return __longlong_as_double(max(__double_as_longlong(a), __double_as_longlong(b)));
}

// The sum of squares of n loaded vectors, or the largest magnitude (as ordered bits in a double).
template <typename T, int V, int K>
__device__ __forceinline__ double reduce(const Vec<T, V> (&e)[K], bool inf_norm) {
  if (inf_norm) {
    uint32_t m = 0;
#pragma unroll
    for (int k = 0; k < K; ++k)
#pragma unroll
      for (int j = 0; j < V; ++j) m = max(m, magnitude(e[k].get(j)));
    return __longlong_as_double(static_cast<long long>(m));
  }
  float s = 0.f;
#pragma unroll
  for (int k = 0; k < K; ++k)
#pragma unroll
    for (int j = 0; j < V; ++j) {
      const float v = e[k].get(j);
      s = fmaf(v, v, s);
    }
  if (s > 1e-20f && s < 1e37f) return static_cast<double>(s);
  double d = 0.0;
#pragma unroll
  for (int k = 0; k < K; ++k)
#pragma unroll
    for (int j = 0; j < V; ++j) {
      const double v = static_cast<double>(e[k].get(j));
      d = fma(v, v, d);
    }
  return d;
}

// Elements before the first 16-byte boundary (of `bytes` each), at most n.
template <typename T>
__device__ __forceinline__ int head_of(const T* p, int n) {
  const int head = static_cast<int>(((16u - (reinterpret_cast<uintptr_t>(p) & 15u)) & 15u) / sizeof(T));
  return head < n ? head : n;
}

// Vectors of V elements that a thread loads at once: 128 bytes, or the fine chunk's share.
template <typename T, int V, int kPer>
constexpr int vectors() {
  const int all = kPer / V, most = 128 / (V * static_cast<int>(sizeof(T)));
  return all < most ? all : most;
}

template <typename T, int kPer>
__device__ __forceinline__ void norm_chunk(const T* p, int n, bool inf_norm, double& acc) {
  constexpr int V = 16 / sizeof(T);
  constexpr int K = vectors<T, V, kPer>();
  // elements before the first 16-byte boundary, then vectors, then the rest
  const int head = head_of(p, n), nv = (n - head) / V;
  const T* src = p + head + threadIdx.x * V;
  constexpr int kStep = 16 / V;  // sixteen squares to a sum
  int left = nv - static_cast<int>(threadIdx.x);
#pragma unroll 1
  for (; left > (K - 1) * kThreads; left -= K * kThreads, src += K * kThreads * V) {
    Vec<T, V> e[K / kStep][kStep];
#pragma unroll
    for (int k = 0; k < K; ++k) e[k / kStep][k % kStep] = ld_vec<T, V>(src + k * kThreads * V);
#pragma unroll
    for (int k = 0; k < K / kStep; ++k) acc = join(acc, reduce(e[k], inf_norm), inf_norm);
  }
  constexpr int R = kStep;  // what is left, a sum at once
#pragma unroll 1
  for (; left > 0; left -= R * kThreads, src += R * kThreads * V) {
    Vec<T, V> e[R];
#pragma unroll
    for (int k = 0; k < R; ++k)
      e[k] = left > k * kThreads ? ld_vec<T, V>(src + k * kThreads * V) : Vec<T, V>::zero();
    acc = join(acc, reduce(e, inf_norm), inf_norm);
  }
  const int loose = n - nv * V, x = threadIdx.x;
  if (x < loose) {
    const Vec<T, 1> w[1] = {ld_vec<T, 1>(p + (x < head ? x : x + nv * V))};
    acc = join(acc, reduce(w, inf_norm), inf_norm);
  }
}

// The block's total in every thread.
__device__ __forceinline__ double block_total(double v, bool inf_norm) {
  __shared__ double s[kThreads / 32];
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v = join(v, __shfl_xor_sync(0xffffffffu, v, o), inf_norm);
  if ((threadIdx.x & 31) == 0) s[threadIdx.x >> 5] = v;
  __syncthreads();
  double t = s[0];
#pragma unroll
  for (int i = 1; i < kThreads / 32; ++i) t = join(t, s[i], inf_norm);
  return t;
}

template <int N, int kPer>
__global__ void __launch_bounds__(kThreads, kPer == kFine ? kFineBlocks : kCoarseBlocks)
    clip_norm_kernel(const __grid_constant__ Table<N> tab, double* __restrict__ partial, Shadow* __restrict__ shadow,
                     bool inf_norm) {
  if (shadow)
    for (int i = blockIdx.x * kThreads + threadIdx.x; i < tab.n; i += gridDim.x * kThreads) shadow->t[i] = tab.t[i];
  constexpr int kChunk = kThreads * kPer;
  double acc = 0.0;
  for (uint32_t c = blockIdx.x; c < tab.chunks; c += gridDim.x) {
    const int t = find([&](int i) { return tab.t[i].first_chunk; }, tab.n, c);
    const uint32_t next = t + 1 < tab.n ? tab.t[t + 1].first_chunk : tab.chunks;
    const Tensor& e = tab.t[t];
    const Span sp = span_of(e, c - e.first_chunk, c + 1 == next, kChunk);
    const int64_t off = sp.off;
    const int n = sp.n;
    if (e.in_type == GTK_F32)
      norm_chunk<float, kPer>(static_cast<const float*>(e.in) + off, n, inf_norm, acc);
    else if (e.in_type == GTK_BF16)
      norm_chunk<__nv_bfloat16, kPer>(static_cast<const __nv_bfloat16*>(e.in) + off, n, inf_norm, acc);
    else
      norm_chunk<__half, kPer>(static_cast<const __half*>(e.in) + off, n, inf_norm, acc);
  }
  const double total = block_total(acc, inf_norm);
  if (threadIdx.x == 0) partial[blockIdx.x] = total;
}

// The norm from all blocks' partials, the same in every block.
__device__ __forceinline__ double total_norm(const double* partial, int n, bool inf_norm) {
  constexpr int kAtOnce = (kMaxBlocks + kThreads - 1) / kThreads;  // all of one launch
  double v = 0.0;
  for (int i0 = threadIdx.x; i0 < n; i0 += kThreads * kAtOnce) {
    double t[kAtOnce];
#pragma unroll
    for (int u = 0; u < kAtOnce; ++u) t[u] = i0 + u * kThreads < n ? partial[i0 + u * kThreads] : 0.0;
#pragma unroll
    for (int u = 0; u < kAtOnce; ++u) v = join(v, t[u], inf_norm);
  }
  v = block_total(v, inf_norm);
  return inf_norm ? static_cast<double>(__uint_as_float(static_cast<uint32_t>(__double_as_longlong(v)))) : sqrt(v);
}

template <typename T, typename O, int V>
__device__ __forceinline__ Vec<O, V> scaled(const Vec<T, V>& e, float k) {
  float f[V];
#pragma unroll
  for (int j = 0; j < V; ++j) f[j] = e.get(j) * k;
  return Vec<O, V>::of(f);
}

// o = k p over one chunk. Vectors of V elements: 16 bytes of the output each, so that a warp's
// stores are contiguous (16-bit gradients to fp32: 8-byte loads, 16-byte stores).
template <typename T, typename O, int kPer>
__device__ __forceinline__ void scale_chunk(const void* in, void* out, int64_t off, int n, float k) {
  const T* p = static_cast<const T*>(in) + off;
  O* o = static_cast<O*>(out) + off;
  constexpr int V = 16 / sizeof(O);
  constexpr int K = vectors<T, V, kPer>();
  const int head = head_of(p, n), nv = (n - head) / V;
  if ((reinterpret_cast<uintptr_t>(o + head) & 15u) != 0) {  // gradient and output lie differently
#pragma unroll 4
    for (int i = threadIdx.x; i < n; i += kThreads) o[i] = Elem<O>::store(Elem<T>::load(p[i]) * k);
    return;
  }
  const T* src = p + head + threadIdx.x * V;
  O* dst = o + head + threadIdx.x * V;
  int left = nv - static_cast<int>(threadIdx.x);
#pragma unroll 1
  for (; left > (K - 1) * kThreads; left -= K * kThreads, src += K * kThreads * V, dst += K * kThreads * V) {
    Vec<T, V> e[K];
#pragma unroll
    for (int q = 0; q < K; ++q) e[q] = ld_vec<T, V>(src + q * kThreads * V);
#pragma unroll
    for (int q = 0; q < K; ++q) st_vec<O, V>(dst + q * kThreads * V, scaled<T, O, V>(e[q], k));
  }
  constexpr int R = K < 4 ? K : 4;  // what is left, a few vectors at once
#pragma unroll 1
  for (; left > 0; left -= R * kThreads, src += R * kThreads * V, dst += R * kThreads * V) {
    Vec<T, V> e[R];
#pragma unroll
    for (int q = 0; q < R; ++q)
      e[q] = left > q * kThreads ? ld_vec<T, V>(src + q * kThreads * V) : Vec<T, V>::zero();
#pragma unroll
    for (int q = 0; q < R; ++q)
      if (left > q * kThreads) st_vec<O, V>(dst + q * kThreads * V, scaled<T, O, V>(e[q], k));
  }
  const int loose = n - nv * V, x = threadIdx.x;
  if (x < loose) {
    const int i = x < head ? x : x + nv * V;
    o[i] = Elem<O>::store(Elem<T>::load(p[i]) * k);
  }
}

// The same by element in 64 bits, for factors that fp32 has few bits of or none (below 2^-126, where
// the norm is near fp32's largest or above it).
template <typename T, typename O>
__device__ __forceinline__ void scale_wide(const void* in, void* out, int64_t off, int n, double q) {
  const T* p = static_cast<const T*>(in) + off;
  O* o = static_cast<O*>(out) + off;
#pragma unroll 1
  for (int i = threadIdx.x; i < n; i += kThreads)
    o[i] = Elem<O>::store(static_cast<float>(static_cast<double>(Elem<T>::load(p[i])) * q));
}

template <int kPer>
__global__ void __launch_bounds__(kThreads, kPer == kFine ? kFineBlocks : kCoarseBlocks)
    clip_scale_kernel(const Shadow* __restrict__ shadow, int tensors, uint32_t chunks,
                      const double* __restrict__ partial, int partials, bool inf_norm, double max_norm, bool in_place,
                      float* __restrict__ norm_out) {
  wait_previous_kernel();
  __shared__ uint32_t first[kMaxTensors + 1];
  for (int i = threadIdx.x; i < tensors; i += kThreads) first[i] = shadow->t[i].first_chunk;
  if (threadIdx.x == 0) first[tensors] = chunks;
  const double norm = total_norm(partial, partials, inf_norm);  // its barrier covers `first` too
  if (norm_out && blockIdx.x == 0 && threadIdx.x == 0) *norm_out = static_cast<float>(norm);
  const double q = max_norm / (norm + static_cast<double>(kEps));
  const float k = static_cast<float>(q < 1.0 || isnan(q) ? q : 1.0);
  if (in_place && k == 1.f) return;
  constexpr int kChunk = kThreads * kPer;
  if (q > 0.0 && q < 0x1p-126) {
#pragma unroll 1
    for (uint32_t c = blockIdx.x; c < chunks; c += gridDim.x) {
      const int t = find([&](int i) { return first[i]; }, tensors, c);
      const Tensor e = shadow->t[t];
      const Span sp = span_of(e, c - first[t], c + 1 == first[t + 1], kChunk);
      if (e.in_type == GTK_F32)
        scale_wide<float, float>(e.in, e.out, sp.off, sp.n, q);
      else if (e.in_type == GTK_BF16 && e.out_type == GTK_BF16)
        scale_wide<__nv_bfloat16, __nv_bfloat16>(e.in, e.out, sp.off, sp.n, q);
      else if (e.in_type == GTK_BF16)
        scale_wide<__nv_bfloat16, float>(e.in, e.out, sp.off, sp.n, q);
      else if (e.out_type == GTK_F16)
        scale_wide<__half, __half>(e.in, e.out, sp.off, sp.n, q);
      else
        scale_wide<__half, float>(e.in, e.out, sp.off, sp.n, q);
    }
    return;
  }
#pragma unroll 1
  for (uint32_t back = blockIdx.x; back < chunks; back += gridDim.x) {
    const uint32_t c = chunks - 1 - back;
    const int t = find([&](int i) { return first[i]; }, tensors, c);
    const Tensor e = shadow->t[t];
    const Span sp = span_of(e, c - first[t], c + 1 == first[t + 1], kChunk);
    const int64_t off = sp.off;
    const int n = sp.n;
    if (e.in_type == GTK_F32)
      scale_chunk<float, float, kPer>(e.in, e.out, off, n, k);
    else if (e.in_type == GTK_BF16 && e.out_type == GTK_BF16)
      scale_chunk<__nv_bfloat16, __nv_bfloat16, kPer>(e.in, e.out, off, n, k);
    else if (e.in_type == GTK_BF16)
      scale_chunk<__nv_bfloat16, float, kPer>(e.in, e.out, off, n, k);
    else if (e.out_type == GTK_F16)
      scale_chunk<__half, __half, kPer>(e.in, e.out, off, n, k);
    else
      scale_chunk<__half, float, kPer>(e.in, e.out, off, n, k);
  }
}

__global__ void __launch_bounds__(kThreads)
    norm_only_kernel(const double* __restrict__ partial, int partials, bool inf_norm, float* __restrict__ norm_out) {
  wait_previous_kernel();
  const double norm = total_norm(partial, partials, inf_norm);
  if (threadIdx.x == 0) *norm_out = static_cast<float>(norm);
}

struct Request {
  std::vector<Tensor> t;       // without the empty ones; first_chunk and last_len not set
  std::vector<int64_t> numel;
  int64_t elements;
  bool inf_norm, in_place, scale;
  double max_norm;
  float* norm;
  char* ws;
  cudaStream_t st;
};

// The workspace: kMaxBlocks partials and one shadow table per launch.
size_t launches_for(int64_t n) {
  return static_cast<size_t>(n <= kMaxTensors ? 1 : (n + kMaxTensors - 1) / kMaxTensors);
}
size_t partial_bytes(int64_t n) { return round_up(sizeof(double) * kMaxBlocks * launches_for(n), 256); }
size_t workspace_bytes(int64_t n) {
  const size_t launches = launches_for(n);
  const size_t last = sizeof(Tensor) * static_cast<size_t>(n - (launches - 1) * kMaxTensors);
  return partial_bytes(n) + (launches - 1) * sizeof(Shadow) + round_up(last, 256);
}

struct Part {
  int tensors, blocks;
  uint32_t chunks;
  Shadow* shadow;
};

// Coarse chunks from 2 M elements on (one tensor into another, from a graph, fine and coarse: 2 Mi fp32
// elements 6.9 and 6.5 us, 16 Mi 29.3 and 27.7, 2^27 bf16 ones into fp32 196 and 182; 1 Mi: 5.5 and 6.2).
bool coarse(int64_t elements) { return elements >= 2 * 1000 * 1000; }

// The first kernel over the tensors [first, first + n).
template <int N>
int norm_part(const Request& r, size_t first, size_t n, int partials, Part* part) {
  Table<N> tab;
  const bool big = coarse(r.elements);
  const int shift = big ? 14 : 12;
  static_assert(kThreads * kCoarse == 1 << 14 && kThreads * kFine == 1 << 12, "chunk sizes");
  uint32_t chunks = 0;
  for (size_t i = 0; i < n; ++i) {
    tab.t[i] = r.t[first + i];
    const int64_t lead = lead_of(tab.t[i].in, tab.t[i].in_type), numel = r.numel[first + i];
    const int64_t m = (numel + lead + (int64_t(1) << shift) - 1) >> shift;
    tab.t[i].first_chunk = chunks;
    tab.t[i].last_len = static_cast<uint16_t>(m == 1 ? numel : numel + lead - ((m - 1) << shift));
    chunks += static_cast<uint32_t>(m);
  }
  const int64_t cap = std::min<int64_t>(static_cast<int64_t>(num_sms()) * (big ? kCoarseBlocks : kFineBlocks),
                                        kMaxBlocks);
  const uint32_t blocks = chunks < cap ? chunks : static_cast<uint32_t>(cap);
  tab.n = part->tensors = static_cast<int>(n);
  tab.chunks = part->chunks = chunks;
  part->blocks = static_cast<int>(blocks);
  return launch("gradient norm", big ? clip_norm_kernel<N, kCoarse> : clip_norm_kernel<N, kFine>, part->blocks,
                kThreads, 0, r.st, false, tab, reinterpret_cast<double*>(r.ws) + partials,
                r.scale ? part->shadow : nullptr, r.inf_norm);
}

int run(const Request& r, int64_t n_given) {
  const double* partial = reinterpret_cast<const double*>(r.ws);
  Shadow* shadow = reinterpret_cast<Shadow*>(r.ws + partial_bytes(n_given));
  const size_t launches = (r.t.size() + kMaxTensors - 1) / kMaxTensors;
  std::vector<Part> parts(launches);
  int partials = 0;
  for (size_t i = 0; i < launches; ++i) {
    const size_t first = i * kMaxTensors, n = std::min<size_t>(kMaxTensors, r.t.size() - first);
    parts[i].shadow = shadow + i;
    // the launch copies its whole table, 1.5 to 24 KB: it takes the smallest that holds the tensors
    const int e = n <= 64    ? norm_part<64>(r, first, n, partials, &parts[i])
                  : n <= 256 ? norm_part<256>(r, first, n, partials, &parts[i])
                  : n <= 512 ? norm_part<512>(r, first, n, partials, &parts[i])
                             : norm_part<kMaxTensors>(r, first, n, partials, &parts[i]);
    if (e) return e;
    partials += parts[i].blocks;
  }
  if (!r.scale || r.t.empty())
    return launch("gradient norm", norm_only_kernel, 1, kThreads, 0, r.st, !r.t.empty(), partial, partials,
                  r.inf_norm, r.norm);
  auto scale = coarse(r.elements) ? clip_scale_kernel<kCoarse> : clip_scale_kernel<kFine>;
  for (size_t i = 0; i < launches; ++i)
    if (int e = launch("gradient clipping", scale, parts[i].blocks, kThreads, 0, r.st, i == 0,
                       static_cast<const Shadow*>(parts[i].shadow), parts[i].tensors, parts[i].chunks,
                       partial, partials, r.inf_norm, r.max_norm, r.in_place,
                       i == 0 ? r.norm : static_cast<float*>(nullptr)))
      return e;
  return GTK_OK;
}

struct Range {
  uintptr_t begin, end;
  int64_t id;
};

bool overlap_within(const std::vector<Range>& v) {
  for (size_t i = 1; i < v.size(); ++i)
    if (v[i].begin < v[i - 1].end) return true;
  return false;
}

// Sorted by address (mostly it is already).
void order(std::vector<Range>* v) {
  auto less = [](const Range& a, const Range& b) { return a.begin < b.begin; };
  if (!std::is_sorted(v->begin(), v->end(), less)) std::sort(v->begin(), v->end(), less);
}

// Outputs may not overlap one another, nor any input but their own at exactly its place.
bool outputs_clash(std::vector<Range> in, std::vector<Range> out, bool in_place) {
  order(&out);
  if (overlap_within(out)) return true;
  if (in_place) return false;
  order(&in);
  // inputs may overlap one another, so their ends are not in order: compare with the furthest
  size_t o = 0;
  for (const Range& a : in) {
    while (o < out.size() && out[o].end <= a.begin) ++o;
    for (size_t k = o; k < out.size() && out[k].begin < a.end; ++k)
      if (!(out[k].begin == a.begin && out[k].end == a.end && out[k].id == a.id)) return true;
  }
  return false;
}

int gather(const void* const* grads, void* const* outs, const int64_t* numel, const int* dtypes,
           const int* out_dtypes, int64_t n, Request* r) {
  if (n < 0 || (n > 0 && (!grads || !numel || !dtypes)))
    return fail(GTK_ERR_INVALID_ARG, "gradient norm: bad tensor list");
  r->t.reserve(n);
  r->numel.reserve(n);
  // what is read and what is written, as far as one look at each tensor tells
  uintptr_t in_low = ~uintptr_t(0), in_high = 0, out_low = ~uintptr_t(0), out_high = 0;
  bool ascending = true;  // every output begins behind the end of the one before
  for (int64_t i = 0; i < n; ++i) {
    const int64_t m = numel[i];
    if (m < 0 || m > (int64_t(1) << 40))
      return fail(GTK_ERR_INVALID_ARG, "gradient norm: bad size of tensor " + std::to_string(i));
    const int it = dtypes[i], ot = (outs && out_dtypes) ? out_dtypes[i] : it;
    if (!dtype_ok(it) || !(ot == it || ot == GTK_F32))
      return fail(GTK_ERR_UNSUPPORTED,
                  "gradient norm: gradients are fp32, bf16 or fp16, outputs fp32 or the gradient's type");
    if (!m) continue;
    void* o = outs ? outs[i] : const_cast<void*>(grads[i]);
    if (!grads[i] || !o) return fail(GTK_ERR_INVALID_ARG, "gradient norm: NULL tensor " + std::to_string(i));
    const uintptr_t a = reinterpret_cast<uintptr_t>(grads[i]), b = reinterpret_cast<uintptr_t>(o);
    if ((a & (dtype_bytes(it) - 1)) || (b & (dtype_bytes(ot) - 1)))
      return fail(GTK_ERR_ALIGNMENT, "gradient norm: tensor " + std::to_string(i) + " is misaligned");
    r->t.push_back(Tensor{grads[i], o, 0, 0, static_cast<uint8_t>(it), static_cast<uint8_t>(ot)});
    r->numel.push_back(m);
    r->elements += m;
    in_low = std::min(in_low, a);
    in_high = std::max(in_high, a + m * dtype_bytes(it));
    ascending = ascending && b >= out_high;
    out_low = std::min(out_low, b);
    out_high = std::max(out_high, b + m * dtype_bytes(ot));
  }
  if (r->elements > (int64_t(1) << 42)) return fail(GTK_ERR_UNSUPPORTED, "gradient norm: too many elements");
  const bool apart = !outs || in_high <= out_low || out_high <= in_low;
  if (!r->scale || (ascending && apart)) return GTK_OK;
  std::vector<Range> in, out;
  out.reserve(r->t.size());
  if (outs) in.reserve(r->t.size());
  for (size_t i = 0; i < r->t.size(); ++i) {
    const Tensor& t = r->t[i];
    const uintptr_t a = reinterpret_cast<uintptr_t>(t.in), b = reinterpret_cast<uintptr_t>(t.out);
    out.push_back(Range{b, b + r->numel[i] * dtype_bytes(t.out_type), static_cast<int64_t>(i)});
    if (outs) in.push_back(Range{a, a + r->numel[i] * dtype_bytes(t.in_type), static_cast<int64_t>(i)});
  }
  if (outputs_clash(std::move(in), std::move(out), !outs))
    return fail(GTK_ERR_INVALID_ARG,
                outs ? "gradient clipping: outputs overlap one another or other gradients"
                     : "gradient clipping: the gradients overlap one another (the same tensor twice?)");
  return GTK_OK;
}

int start(const void* const* grads, void* const* outs, const int64_t* numel, const int* dtypes, const int* out_dtypes,
          int64_t n, int norm_kind, float* norm, void* workspace, size_t workspace_bytes_given, void* stream,
          Request* r) {
  if (norm_kind != GTK_NORM_2 && norm_kind != GTK_NORM_INF)
    return fail(GTK_ERR_UNSUPPORTED, "gradient norm: the norm is GTK_NORM_2 or GTK_NORM_INF");
  if (int e = gather(grads, outs, numel, dtypes, out_dtypes, n, r)) return e;
  if (int e = check_ptr(norm, "norm", 4)) return e;
  if (workspace_bytes_given < workspace_bytes(n)) return fail(GTK_ERR_WORKSPACE, "gradient norm: workspace too small");
  if (int e = check_ptr(workspace, "workspace", 256)) return e;
  if (int e = check_device()) return e;
  r->inf_norm = norm_kind == GTK_NORM_INF;
  r->in_place = !outs;
  r->norm = norm;
  r->ws = static_cast<char*>(workspace);
  r->st = static_cast<cudaStream_t>(stream);
  return run(*r, n);
}

}  // namespace clip
}  // namespace gtk

using namespace gtk;

extern "C" {

size_t gtk_grad_norm_workspace_bytes(int64_t n_tensors) {
  return n_tensors < 0 ? 0 : clip::workspace_bytes(n_tensors);
}

int gtk_grad_norm(const void* const* grads, const int64_t* numel, const int* dtypes, int64_t n_tensors, int norm_kind,
                  float* norm, void* workspace, size_t workspace_bytes, void* stream) try {
  clip::Request r = {};
  return clip::start(grads, nullptr, numel, dtypes, nullptr, n_tensors, norm_kind, norm, workspace, workspace_bytes,
                     stream, &r);
} catch (...) {
  return fail_no_memory();
}

int gtk_clip_grad_norm(const void* const* grads, void* const* outs, const int64_t* numel, const int* dtypes,
                       const int* out_dtypes, int64_t n_tensors, int norm_kind, double max_norm, float* norm,
                       void* workspace, size_t workspace_bytes, void* stream) try {
  if (!(max_norm >= 0.0)) return fail(GTK_ERR_INVALID_ARG, "gradient clipping: max_norm must be >= 0");
  clip::Request r = {};
  r.scale = true;
  r.max_norm = max_norm;
  return clip::start(grads, outs, numel, dtypes, out_dtypes, n_tensors, norm_kind, norm, workspace, workspace_bytes,
                     stream, &r);
} catch (...) {
  return fail_no_memory();
}

}  // extern "C"
