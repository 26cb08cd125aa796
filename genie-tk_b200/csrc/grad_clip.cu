// The global norm of many gradients, and clipping by it:
//
//   norm = (sum over all elements g^2)^1/2   (or max |g|)
//   k    = min(1, max_norm / (norm + 1e-6))
//   out  = k g                               (in place, or to other tensors of g's type or fp32)
//
// k is NaN when the norm is (every output becomes NaN) and 0 when the norm is infinite, the
// same as torch.nn.utils.clip_grad_norm_.
//
// What bounds it: HBM, and for the gradients of a small model the launches. Two launches:
// clip_norm_kernel reads the gradients once and leaves one partial per block; clip_scale_kernel
// adds the partials (every block the same sum, in the same order) and scales. The tensors
// reach the kernels as a table in the kernel's own parameters (up to 1000 tensors a launch), so
// there is no table to copy to the device and nothing to keep alive behind the call.
//
// The tensors are cut into chunks of 8192 elements, and every block owns a run of consecutive
// chunks. The second kernel walks its run backwards: what the first one read last is still in
// the L2 cache then. In place and with k = 1 it has nothing to do and returns.
//
// Squares are summed 16 at a time in fp32 and from there on in 64 bits. Where such a sum is not
// a plain number (it overflowed, or is so small that its squares may have underflowed) the 16
// are squared in 64 bits, so the norm holds for gradients of any magnitude.
#include <algorithm>
#include <vector>

#include "train_common.cuh"

namespace gtk {
namespace clip {

constexpr int kThreads = 512;
constexpr int kPer = 16;                      // elements per thread and chunk
constexpr int kChunk = kThreads * kPer;       // 8192
constexpr int kBlocksPerSm = 2;
constexpr int kMaxBlocks = 148 * kBlocksPerSm;  // partials per launch
constexpr int kMaxTensors = 1000;             // of one launch (32,000 of the 32,764 parameter bytes)
constexpr float kEps = 1e-6f;

struct Tensor {
  const void* in;
  void* out;
  int64_t numel;
  uint32_t first_chunk;
  uint8_t in_type, out_type;
};

template <int N>
struct Table {
  Tensor t[N];
  int n;
  uint32_t chunks;  // of all tensors
  uint32_t per;     // chunks of one block
};

// The tensor that holds chunk c (t.first_chunk is ascending).
template <int N>
__device__ __forceinline__ int find(const Table<N>& tab, uint32_t c) {
  int lo = 0, hi = tab.n - 1;
  while (lo < hi) {
    const int mid = (lo + hi + 1) >> 1;
    if (tab.t[mid].first_chunk <= c)
      lo = mid;
    else
      hi = mid - 1;
  }
  return lo;
}

__device__ __forceinline__ float square_or_max(float acc, float v, bool inf_norm) {
  // |v| as an ordered integer, in which NaN is above infinity
  if (inf_norm) return __uint_as_float(max(__float_as_uint(acc), __float_as_uint(v) & 0x7fffffffu));
  return fmaf(v, v, acc);
}

// acc += the squares of n values whose fp32 sum is s (or the maximum, as ordered bits).
template <int n>
__device__ __forceinline__ void add_sum(double& acc, float s, const float (&v)[n], bool inf_norm) {
  if (inf_norm) {
    acc = __longlong_as_double(max(__double_as_longlong(acc), static_cast<long long>(__float_as_uint(s))));
    return;
  }
  if (s > 1e-20f && s < 1e37f) {
    acc += static_cast<double>(s);
    return;
  }
  for (int i = 0; i < n; ++i) acc = fma(static_cast<double>(v[i]), static_cast<double>(v[i]), acc);
}

template <typename T>
__device__ __forceinline__ void norm_chunk(const T* p, int n, bool inf_norm, double& acc) {
  constexpr int V = 16 / sizeof(T);
  constexpr int K = kPer / V;
  // elements before the first 16-byte boundary, then vectors, then the rest
  int head = static_cast<int>(((16u - (reinterpret_cast<uintptr_t>(p) & 15u)) & 15u) / sizeof(T));
  head = head < n ? head : n;
  const int nv = (n - head) / V;
  Vec<T, V> e[K];
#pragma unroll
  for (int k = 0; k < K; ++k) {
    const int i = threadIdx.x + k * kThreads;
    if (i < nv)
      e[k] = ld_vec<T, V>(p + head + i * V);
    else
#pragma unroll
      for (int j = 0; j < V; ++j) e[k].v[j] = Elem<T>::store(0.f);
  }
  float v[kPer], s = 0.f;
#pragma unroll
  for (int k = 0; k < K; ++k)
#pragma unroll
    for (int j = 0; j < V; ++j) {
      v[k * V + j] = Elem<T>::load(e[k].v[j]);
      s = square_or_max(s, v[k * V + j], inf_norm);
    }
  if (s != 0.f || threadIdx.x < nv) add_sum(acc, s, v, inf_norm);
  const int loose = n - nv * V;
  if (threadIdx.x < loose) {
    const int i = threadIdx.x < head ? threadIdx.x : threadIdx.x + nv * V;
    float w[1] = {Elem<T>::load(p[i])};
    add_sum(acc, square_or_max(0.f, w[0], inf_norm), w, inf_norm);
  }
}

__device__ __forceinline__ double join(double a, double b, bool inf_norm) {
  if (!inf_norm) return a + b;
  return __longlong_as_double(max(__double_as_longlong(a), __double_as_longlong(b)));
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

template <int N>
__global__ void __launch_bounds__(kThreads)
    clip_norm_kernel(const __grid_constant__ Table<N> tab, double* __restrict__ partial, bool inf_norm) {
  double acc = 0.0;
  const uint32_t c0 = blockIdx.x * tab.per;
  const uint32_t c1 = min(c0 + tab.per, tab.chunks);
  int t = c0 < c1 ? find(tab, c0) : 0;
  for (uint32_t c = c0; c < c1; ++c) {
    while (t + 1 < tab.n && tab.t[t + 1].first_chunk <= c) ++t;
    const Tensor& e = tab.t[t];
    const int64_t off = static_cast<int64_t>(c - e.first_chunk) * kChunk;
    const int n = static_cast<int>(min(static_cast<int64_t>(kChunk), e.numel - off));
    if (e.in_type == GTK_F32)
      norm_chunk(static_cast<const float*>(e.in) + off, n, inf_norm, acc);
    else if (e.in_type == GTK_BF16)
      norm_chunk(static_cast<const __nv_bfloat16*>(e.in) + off, n, inf_norm, acc);
    else
      norm_chunk(static_cast<const __half*>(e.in) + off, n, inf_norm, acc);
  }
  const double total = block_total(acc, inf_norm);
  if (threadIdx.x == 0) partial[blockIdx.x] = total;
}

// The norm from all blocks' partials, the same in every block.
__device__ __forceinline__ double total_norm(const double* partial, int n, bool inf_norm) {
  double v = 0.0;
  for (int i = threadIdx.x; i < n; i += kThreads) v = join(v, partial[i], inf_norm);
  v = block_total(v, inf_norm);
  return inf_norm ? static_cast<double>(__uint_as_float(static_cast<uint32_t>(__double_as_longlong(v)))) : sqrt(v);
}

template <typename T, typename O>
__device__ __forceinline__ void scale_chunk(const T* p, O* o, int n, float k) {
  constexpr int V = 16 / sizeof(T);
  constexpr int K = kPer / V;
  int head = static_cast<int>(((16u - (reinterpret_cast<uintptr_t>(p) & 15u)) & 15u) / sizeof(T));
  head = head < n ? head : n;
  const int nv = (n - head) / V;
  constexpr int kOutAlign = sizeof(O) * V < 16 ? sizeof(O) * V : 16;
  const bool vec = (reinterpret_cast<uintptr_t>(o + head) % kOutAlign) == 0;
  Vec<T, V> e[K];
#pragma unroll
  for (int q = 0; q < K; ++q) {
    const int i = threadIdx.x + q * kThreads;
    if (i < nv) e[q] = ld_vec<T, V>(p + head + i * V);
  }
#pragma unroll
  for (int q = 0; q < K; ++q) {
    const int i = threadIdx.x + q * kThreads;
    if (i >= nv) continue;
    O* d = o + head + i * V;
    constexpr int VO = kOutAlign / sizeof(O);
#pragma unroll
    for (int a = 0; a < V; a += VO) {
      Vec<O, VO> w;
#pragma unroll
      for (int j = 0; j < VO; ++j) w.v[j] = Elem<O>::store(Elem<T>::load(e[q].v[a + j]) * k);
      if (vec)
        st_vec<O, VO>(d + a, w);
      else
#pragma unroll
        for (int j = 0; j < VO; ++j) d[a + j] = w.v[j];
    }
  }
  const int loose = n - nv * V;
  if (threadIdx.x < loose) {
    const int i = threadIdx.x < head ? threadIdx.x : threadIdx.x + nv * V;
    o[i] = Elem<O>::store(Elem<T>::load(p[i]) * k);
  }
}

template <int N>
__global__ void __launch_bounds__(kThreads)
    clip_scale_kernel(const __grid_constant__ Table<N> tab, const double* __restrict__ partial, int partials,
                      bool inf_norm, double max_norm, bool in_place, float* __restrict__ norm_out) {
  wait_previous_kernel();
  const double norm = total_norm(partial, partials, inf_norm);
  if (norm_out && blockIdx.x == 0 && threadIdx.x == 0) *norm_out = static_cast<float>(norm);
  const double q = max_norm / (norm + static_cast<double>(kEps));
  const float k = static_cast<float>(q < 1.0 || isnan(q) ? q : 1.0);
  if (in_place && k == 1.f) return;
  const uint32_t c0 = blockIdx.x * tab.per;
  const uint32_t c1 = min(c0 + tab.per, tab.chunks);
  if (c0 >= c1) return;
  int t = find(tab, c1 - 1);
  for (uint32_t c = c1; c-- > c0;) {
    while (tab.t[t].first_chunk > c) --t;
    const Tensor& e = tab.t[t];
    const int64_t off = static_cast<int64_t>(c - e.first_chunk) * kChunk;
    const int n = static_cast<int>(min(static_cast<int64_t>(kChunk), e.numel - off));
    if (e.in_type == GTK_F32)
      scale_chunk(static_cast<const float*>(e.in) + off, static_cast<float*>(e.out) + off, n, k);
    else if (e.in_type == GTK_BF16 && e.out_type == GTK_BF16)
      scale_chunk(static_cast<const __nv_bfloat16*>(e.in) + off, static_cast<__nv_bfloat16*>(e.out) + off, n, k);
    else if (e.in_type == GTK_BF16)
      scale_chunk(static_cast<const __nv_bfloat16*>(e.in) + off, static_cast<float*>(e.out) + off, n, k);
    else if (e.out_type == GTK_F16)
      scale_chunk(static_cast<const __half*>(e.in) + off, static_cast<__half*>(e.out) + off, n, k);
    else
      scale_chunk(static_cast<const __half*>(e.in) + off, static_cast<float*>(e.out) + off, n, k);
  }
}

__global__ void __launch_bounds__(kThreads)
    norm_only_kernel(const double* __restrict__ partial, int partials, bool inf_norm, float* __restrict__ norm_out) {
  wait_previous_kernel();
  const double norm = total_norm(partial, partials, inf_norm);
  if (threadIdx.x == 0) *norm_out = static_cast<float>(norm);
}

struct Request {
  std::vector<Tensor> t;  // without the empty ones
  bool inf_norm, in_place, scale;
  double max_norm;
  float* norm;
  double* partial;
  cudaStream_t st;
};

int blocks_for(uint32_t chunks) {
  const int cap = num_sms() * kBlocksPerSm < kMaxBlocks ? num_sms() * kBlocksPerSm : kMaxBlocks;
  return static_cast<int>(chunks < static_cast<uint32_t>(cap) ? chunks : static_cast<uint32_t>(cap));
}

template <int N>
void fill(Table<N>* tab, const Request& r, size_t first, size_t n) {
  uint32_t chunks = 0;
  for (size_t i = 0; i < n; ++i) {
    tab->t[i] = r.t[first + i];
    tab->t[i].first_chunk = chunks;
    chunks += static_cast<uint32_t>((r.t[first + i].numel + kChunk - 1) / kChunk);
  }
  tab->n = static_cast<int>(n);
  tab->chunks = chunks;
  const uint32_t blocks = static_cast<uint32_t>(blocks_for(chunks));
  tab->per = (chunks + blocks - 1) / blocks;
}

// One launch over the tensors [first, first + n). `scale`: the second kernel, else the first.
template <int N>
int run_part(const Request& r, size_t first, size_t n, bool scale, bool write_norm, int* partials) {
  Table<N> tab;
  fill(&tab, r, first, n);
  const int blocks = static_cast<int>((tab.chunks + tab.per - 1) / tab.per);
  if (!scale) {
    const int e = launch("gradient norm", clip_norm_kernel<N>, blocks, kThreads, 0, r.st, false, tab,
                         r.partial + *partials, r.inf_norm);
    *partials += blocks;
    return e;
  }
  return launch("gradient clipping", clip_scale_kernel<N>, blocks, kThreads, 0, r.st, write_norm, tab,
                static_cast<const double*>(r.partial), *partials, r.inf_norm, r.max_norm, r.in_place,
                write_norm ? r.norm : static_cast<float*>(nullptr));
}

int run(const Request& r) {
  int partials = 0;
  for (int phase = 0; phase < (r.scale ? 2 : 1); ++phase)
    for (size_t first = 0; first < r.t.size(); first += kMaxTensors) {
      const size_t n = std::min<size_t>(kMaxTensors, r.t.size() - first);
      // the table travels with every launch: 2, 8 or 32 KB of parameters, by the number of tensors
      const int e = n <= 64    ? run_part<64>(r, first, n, phase, first == 0, &partials)
                    : n <= 256 ? run_part<256>(r, first, n, phase, first == 0, &partials)
                               : run_part<kMaxTensors>(r, first, n, phase, first == 0, &partials);
      if (e) return e;
    }
  if (r.scale && !r.t.empty()) return GTK_OK;
  return launch("gradient norm", norm_only_kernel, 1, kThreads, 0, r.st, !r.t.empty(),
                static_cast<const double*>(r.partial), partials, r.inf_norm, r.norm);
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
  std::vector<Range> in, out;
  r->t.reserve(n);
  out.reserve(n);
  if (outs) in.reserve(n);
  for (int64_t i = 0; i < n; ++i) {
    if (numel[i] < 0 || numel[i] > (int64_t(1) << 40))
      return fail(GTK_ERR_INVALID_ARG, "gradient norm: bad size of tensor " + std::to_string(i));
    const int ot = (outs && out_dtypes) ? out_dtypes[i] : dtypes[i];
    if (!dtype_ok(dtypes[i]) || !(ot == dtypes[i] || ot == GTK_F32))
      return fail(GTK_ERR_UNSUPPORTED,
                  "gradient norm: gradients are fp32, bf16 or fp16, outputs fp32 or the gradient's type");
    if (!numel[i]) continue;
    void* o = outs ? outs[i] : const_cast<void*>(grads[i]);
    if (!grads[i] || !o) return fail(GTK_ERR_INVALID_ARG, "gradient norm: NULL tensor " + std::to_string(i));
    const uintptr_t a = reinterpret_cast<uintptr_t>(grads[i]), b = reinterpret_cast<uintptr_t>(o);
    if (a % dtype_bytes(dtypes[i]) || b % dtype_bytes(ot))
      return fail(GTK_ERR_ALIGNMENT, "gradient norm: tensor " + std::to_string(i) + " is misaligned");
    r->t.push_back(Tensor{grads[i], o, numel[i], 0, static_cast<uint8_t>(dtypes[i]), static_cast<uint8_t>(ot)});
    if (!r->scale) continue;
    out.push_back(Range{b, b + numel[i] * dtype_bytes(ot), i});
    if (outs) in.push_back(Range{a, a + numel[i] * dtype_bytes(dtypes[i]), i});
  }
  int64_t chunks = 0;
  for (const Tensor& t : r->t) chunks += (t.numel + kChunk - 1) / kChunk;
  if (chunks > (int64_t(1) << 31)) return fail(GTK_ERR_UNSUPPORTED, "gradient norm: too many elements");
  if (r->scale && outputs_clash(std::move(in), std::move(out), !outs))
    return fail(GTK_ERR_INVALID_ARG,
                outs ? "gradient clipping: outputs overlap one another or other gradients"
                     : "gradient clipping: the gradients overlap one another (the same tensor twice?)");
  return GTK_OK;
}

size_t workspace_bytes(int64_t n) {
  const int64_t launches = (n + kMaxTensors - 1) / kMaxTensors;
  return sizeof(double) * static_cast<size_t>(kMaxBlocks) * static_cast<size_t>(launches < 1 ? 1 : launches);
}

int start(const void* const* grads, void* const* outs, const int64_t* numel, const int* dtypes, const int* out_dtypes,
          int64_t n, int norm_kind, float* norm, void* workspace, size_t workspace_bytes_given, void* stream,
          Request* r) {
  if (norm_kind != GTK_NORM_2 && norm_kind != GTK_NORM_INF)
    return fail(GTK_ERR_UNSUPPORTED, "gradient norm: the norm is GTK_NORM_2 or GTK_NORM_INF");
  if (int e = gather(grads, outs, numel, dtypes, out_dtypes, n, r)) return e;
  if (int e = check_ptr(norm, "norm", 4)) return e;
  if (workspace_bytes_given < workspace_bytes(n)) return fail(GTK_ERR_WORKSPACE, "gradient norm: workspace too small");
  if (int e = check_ptr(workspace, "workspace")) return e;
  if (int e = check_device()) return e;
  r->inf_norm = norm_kind == GTK_NORM_INF;
  r->in_place = !outs;
  r->norm = norm;
  r->partial = static_cast<double*>(workspace);
  r->st = static_cast<cudaStream_t>(stream);
  return run(*r);
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
  return fail(GTK_ERR_INVALID_ARG, "gradient norm: out of host memory");
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
  return fail(GTK_ERR_INVALID_ARG, "gradient clipping: out of host memory");
}

}  // extern "C"
