// Embedding lookup with scaling, and its gradient by sorted tokens:
//
//   y_t  = s W[tok_t]                      (a gather; zeros for a token outside 0 .. V-1)
//   dW_v = s sum_{t : tok_t = v} dy_t      (zeros for a token that does not occur, and padding)
//
// Forward: HBM bound. It writes T rows and reads each row of W that occurs at least once. The output
// is written as one array, thread by thread in 16-byte vectors, whatever the width; the tokens and
// the table's elements behind them come through the caches, four vectors at a time per thread.
//
// Backward: HBM bound too -- it reads dy once and writes the whole of dW once -- if the rows
// of one token can be found together. So the tokens are sorted first (stable, least digit first,
// up to 8 bits a pass; four bytes of key and four of position per token, small beside dy; one
// cluster of blocks does it up to 8192 tokens), and the sorted list is cut into chunks of equal length,
// whatever the tokens' frequencies: a group of 4 to 32 lanes (as the row is wide) sums the dy rows of
// its chunk in registers, in list order, with the next twelve rows in flight, and writes a row of dW
// at each change of token. Runs
// that cross chunks are joined in the block, and those that cross blocks from a scratch buffer
// of at most two rows a block, by a last kernel and in order. Rows of tokens that do not occur are
// zeroed by further blocks of the same launch, which look them up in the sorted keys.
// No atomics on floating-point values: the same inputs give the same bits. Sums are fp32: a chunk's
// rows of one token by fours, one four after another (at most 256, and a few single rows at the run's
// ends), the chunks of a block one after another (8 to 64), and the blocks of a run over the 16 warps of
// the last kernel, which add eight at a time (one addition for each 128 blocks) and meet in a tree. dW
// is rounded once. (64-bit additions between the chunks took twice the time of the joining kernel.)
#include <cooperative_groups.h>

#include "train_common.cuh"

namespace gtk {
namespace emb {

constexpr int kSortThreads = 1024;
constexpr int kMaxCluster = 8;                    // sorting blocks that exchange through their shared memory
constexpr int64_t kClusterTokens = static_cast<int64_t>(kSortThreads) * kMaxCluster;
constexpr int kMaxPer = 8;                        // tokens per thread of the sort over many tiles
constexpr int kMaxBits = 8;                       // of a digit
constexpr int kBins = 1 << kMaxBits;
constexpr int kWarps = kSortThreads / 32;
constexpr int kSlices = kSortThreads / kBins;     // threads per bin
constexpr int kMaxWidth = 1 << 20;
constexpr int64_t kMaxSorted = int64_t(1) << 27;  // tokens of a backward call

// The key of token v: itself, or V (sorted last and then ignored) when it is out of range or padding.
__device__ __forceinline__ uint32_t key_of(int64_t v, uint32_t V, int64_t padding, bool* bad) {
  if (v < 0 || v >= static_cast<int64_t>(V)) {
    *bad = true;
    return V;
  }
  return v == padding ? V : static_cast<uint32_t>(v);
}

struct SortShared {
  uint16_t count[kWarps][kBins];
  uint32_t part[kSlices][kBins];
  uint32_t base[kBins];
  uint32_t scan[kBins / 32];
};

// Exclusive scan of one value per bin over the first kBins threads; all threads call it.
__device__ __forceinline__ uint32_t scan_bins(SortShared& s, uint32_t v) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  uint32_t x = v;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const uint32_t y = __shfl_up_sync(0xffffffffu, x, o);
    if (lane >= o) x += y;
  }
  if (threadIdx.x < kBins && lane == 31) s.scan[warp] = x;
  __syncthreads();
  uint32_t before = 0;
  if (threadIdx.x < kBins)
    for (int w = 0; w < warp; ++w) before += s.scan[w];
  return before + x - v;
}

// Stable rank of the tile's elements by a digit of `bits` bits: the thread's element i (index
// tile_index(i) of the tile) has digit[i], kBins where there is no element. After the call and a
// barrier, s.count[w][b] holds the number of elements of digit b in the warps before w; rank[i]
// is the element's rank among its warp's elements of that digit. The total of digit threadIdx.x
// is returned to the first kBins threads. Equal digits within a warp are found with one ballot
// per bit (__match_any_sync took 5 us where this takes 1).
template <int N>
__device__ __forceinline__ uint32_t rank_tile(SortShared& s, const uint32_t (&digit)[N], uint32_t (&rank)[N],
                                              int bits) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  for (int b = lane; b < kBins; b += 32) s.count[warp][b] = 0;
  __syncwarp();
#pragma unroll
  for (int i = 0; i < N; ++i) {
    const uint32_t d = digit[i];
    const bool valid = d < kBins;
    uint32_t peers = __ballot_sync(0xffffffffu, valid);
#pragma unroll
    for (int b = 0; b < kMaxBits; ++b)
      if (b < bits) {
        const bool one = (d >> b) & 1u;
        const uint32_t ones = __ballot_sync(0xffffffffu, one);
        peers &= one ? ones : ~ones;
      }
    const uint32_t before = valid ? s.count[warp][d] : 0;
    __syncwarp();
    rank[i] = before + __popc(peers & ((1u << lane) - 1u));
    if (valid && (peers >> lane) == 1u) s.count[warp][d] = static_cast<uint16_t>(rank[i] + 1);
    __syncwarp();
  }
  __syncthreads();
  // exclusive counts over the warps: kSlices threads per bin, each for consecutive warps
  constexpr int kRun = kWarps / kSlices;
  const int bin = threadIdx.x & (kBins - 1), slice = threadIdx.x / kBins;
  uint32_t n[kRun], total = 0;
#pragma unroll
  for (int w = 0; w < kRun; ++w) total += n[w] = s.count[slice * kRun + w][bin];
  s.part[slice][bin] = total;
  __syncthreads();
  uint32_t at = 0;
  total = 0;
#pragma unroll
  for (int i = 0; i < kSlices; ++i) {
    const uint32_t t = s.part[i][bin];
    at += i < slice ? t : 0;
    total += t;
  }
#pragma unroll
  for (int w = 0; w < kRun; ++w) {
    s.count[slice * kRun + w][bin] = static_cast<uint16_t>(at);
    at += n[w];
  }
  return total;
}

// Consecutive elements belong to a warp, so that ranks by warp keep the order.
template <int N>
__device__ __forceinline__ int tile_index(int i) {
  return (threadIdx.x >> 5) * 32 * N + i * 32 + (threadIdx.x & 31);
}

// The whole sort in one launch of one cluster: up to eight blocks of 1024 tokens, which read one
// another's digit counts and send every token to the block of its next place through distributed
// shared memory. (Four launches over tiles take 3 us longer for 8192 tokens in two passes. With more
// tokens per thread the cluster falls behind the tiles from 10,000 tokens on.)
// Further clusters, where `zero` is given, zero `zero_bytes` there meanwhile (16-byte multiples).
template <typename I>
__global__ void __launch_bounds__(kSortThreads)
    sort_cluster_kernel(const I* __restrict__ tokens, int T, uint32_t V, int64_t padding, int passes, int bits,
                        uint32_t* __restrict__ keys_out, uint32_t* __restrict__ pos_out, uint4* __restrict__ zero,
                        int64_t zero_bytes, uint32_t* status) {
  namespace cg = cooperative_groups;
  cg::cluster_group cluster = cg::this_cluster();
  if (blockIdx.x >= cluster.num_blocks()) {
    const int64_t step = static_cast<int64_t>(gridDim.x - cluster.num_blocks()) * kSortThreads;
    for (int64_t i = static_cast<int64_t>(blockIdx.x - cluster.num_blocks()) * kSortThreads + threadIdx.x;
         i < zero_bytes / 16; i += step)
      zero[i] = make_uint4(0, 0, 0, 0);
    return;
  }
  extern __shared__ uint32_t buf[];  // [2][1024]: keys, positions
  __shared__ SortShared s;
  __shared__ uint32_t totals[kBins];
  constexpr int kHere = kSortThreads, N = 1;  // tokens of a block, and of a thread
  const int blocks = static_cast<int>(cluster.num_blocks()), me = static_cast<int>(cluster.block_rank());
  bool bad = false;
  uint32_t key[N], pos[N];
#pragma unroll
  for (int i = 0; i < N; ++i) {
    const int t = me * kHere + tile_index<N>(i);
    pos[i] = static_cast<uint32_t>(t);
    key[i] = t < T ? key_of(static_cast<int64_t>(tokens[t]), V, padding, &bad) : 0u;
  }
  for (int p = 0; p < passes; ++p) {
    uint32_t digit[N], rank[N];
#pragma unroll
    for (int i = 0; i < N; ++i)
      digit[i] = me * kHere + tile_index<N>(i) < T ? (key[i] >> (bits * p)) & ((1u << bits) - 1u) : kBins;
    const uint32_t total = rank_tile<N>(s, digit, rank, bits);
    if (threadIdx.x < kBins) totals[threadIdx.x] = total;
    cluster.sync();
    uint32_t before = 0, all = 0;
    if (threadIdx.x < kBins) {
      uint32_t n[kMaxCluster];
#pragma unroll
      for (int r = 0; r < kMaxCluster; ++r) n[r] = r < blocks ? cluster.map_shared_rank(totals, r)[threadIdx.x] : 0u;
#pragma unroll
      for (int r = 0; r < kMaxCluster; ++r) {
        before += r < me ? n[r] : 0;
        all += n[r];
      }
    }
    const uint32_t base = scan_bins(s, all);
    if (threadIdx.x < kBins) s.base[threadIdx.x] = base + before;
    __syncthreads();
#pragma unroll
    for (int i = 0; i < N; ++i)
      if (digit[i] < kBins) {
        const uint32_t to = s.base[digit[i]] + s.count[threadIdx.x >> 5][digit[i]] + rank[i];
        uint32_t* there = cluster.map_shared_rank(buf, to / kHere);
        there[to % kHere] = key[i];
        there[kHere + to % kHere] = pos[i];
      }
    cluster.sync();  // the tokens have arrived, and nobody reads `totals` of this pass any more
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const int t = tile_index<N>(i);
      if (me * kHere + t < T) {
        key[i] = buf[t];
        pos[i] = buf[kHere + t];
      }
    }
  }
#pragma unroll
  for (int i = 0; i < N; ++i) {
    const int t = me * kHere + tile_index<N>(i);
    if (t < T) {
      keys_out[t] = key[i];
      pos_out[t] = pos[i];
    }
  }
  if (status && bad) atomicOr(status, GTK_STATUS_BAD_TOKEN);
}

// Pass `pass` of the sort over many tiles, first half: the tile's digit counts. The first pass
// reads the tokens, later ones the keys of the pass before. Warps count in four histograms; 32
// equal digits (frequent tokens, sorted data) are one addition.
template <typename I, int N>
__global__ void __launch_bounds__(kSortThreads)
    count_kernel(const I* __restrict__ tokens, const uint32_t* __restrict__ keys, int64_t T, uint32_t V,
                 int64_t padding, int pass, int bits, uint32_t* __restrict__ counts, uint32_t* status) {
  wait_previous_kernel();
  __shared__ uint32_t hist[4][kBins];
  (&hist[0][0])[threadIdx.x] = 0;
  __syncthreads();
  bool bad = false;
  uint32_t digit[N];
#pragma unroll
  for (int i = 0; i < N; ++i) {
    const int64_t t = static_cast<int64_t>(blockIdx.x) * (kSortThreads * N) + tile_index<N>(i);
    uint32_t k = 0;
    if (t < T) k = pass == 0 ? key_of(static_cast<int64_t>(tokens[t]), V, padding, &bad) : keys[t];
    digit[i] = t < T ? (k >> (bits * pass)) & ((1u << bits) - 1u) : kBins;
  }
  uint32_t* h = hist[(threadIdx.x >> 5) & 3];
#pragma unroll
  for (int i = 0; i < N; ++i) {
    const uint32_t first = __shfl_sync(0xffffffffu, digit[i], 0);
    if (__all_sync(0xffffffffu, digit[i] == first)) {
      if ((threadIdx.x & 31) == 0 && first < kBins) atomicAdd(h + first, 32u);
    } else if (digit[i] < kBins) {
      atomicAdd(h + digit[i], 1u);
    }
  }
  __syncthreads();
  if (threadIdx.x < kBins)
    counts[static_cast<int64_t>(blockIdx.x) * kBins + threadIdx.x] =
        hist[0][threadIdx.x] + hist[1][threadIdx.x] + hist[2][threadIdx.x] + hist[3][threadIdx.x];
  if (status && bad) atomicOr(status, GTK_STATUS_BAD_TOKEN);
}

// Second half: where the tile's elements go, from all tiles' counts.
template <typename I, int N>
__global__ void __launch_bounds__(kSortThreads)
    scatter_kernel(const I* __restrict__ tokens, const uint32_t* __restrict__ keys, const uint32_t* __restrict__ pos,
                   int64_t T, uint32_t V, int64_t padding, int pass, int bits, const uint32_t* __restrict__ counts,
                   int tiles, uint32_t* __restrict__ keys_out, uint32_t* __restrict__ pos_out) {
  wait_previous_kernel();
  __shared__ SortShared s;
  __shared__ uint32_t before_part[kSortThreads], total_part[kSortThreads];
  uint32_t key[N], p0[N], digit[N], rank[N];
  int64_t token[N];  // requested here, looked at after the counts, which are on their way meanwhile
#pragma unroll
  for (int i = 0; i < N; ++i) {
    const int64_t t = static_cast<int64_t>(blockIdx.x) * (kSortThreads * N) + tile_index<N>(i);
    p0[i] = static_cast<uint32_t>(t);
    token[i] = t >= T ? 0 : pass == 0 ? static_cast<int64_t>(tokens[t]) : static_cast<int64_t>(keys[t]);
    if (pass && t < T) p0[i] = pos[t];
  }
  // thread = (slice of the tiles, bin)
  const int bins = 1 << bits, slices = kSortThreads >> bits;
  const int bin = threadIdx.x & (bins - 1), slice = threadIdx.x >> bits;
  uint32_t before = 0, total = 0;
  constexpr int kAtOnce = 8;
  for (int t0 = slice; t0 < tiles; t0 += slices * kAtOnce) {
    uint32_t n[kAtOnce];
#pragma unroll
    for (int u = 0; u < kAtOnce; ++u) {
      const int t = t0 + u * slices;
      n[u] = t < tiles ? counts[static_cast<int64_t>(t) * kBins + bin] : 0u;
    }
#pragma unroll
    for (int u = 0; u < kAtOnce; ++u) {
      total += n[u];
      before += t0 + u * slices < static_cast<int>(blockIdx.x) ? n[u] : 0u;
    }
  }
  before_part[threadIdx.x] = before;
  total_part[threadIdx.x] = total;
  bool bad = false;
#pragma unroll
  for (int i = 0; i < N; ++i) {
    const int64_t t = static_cast<int64_t>(blockIdx.x) * (kSortThreads * N) + tile_index<N>(i);
    key[i] = pass == 0 ? key_of(token[i], V, padding, &bad) : static_cast<uint32_t>(token[i]);
    digit[i] = t < T ? (key[i] >> (bits * pass)) & ((1u << bits) - 1u) : kBins;
  }
  __syncthreads();
  before = total = 0;
  if (threadIdx.x < bins)
    for (int i = 0; i < slices; ++i) {
      before += before_part[(i << bits) + threadIdx.x];
      total += total_part[(i << bits) + threadIdx.x];
    }
  const uint32_t base = scan_bins(s, total);
  if (threadIdx.x < kBins) s.base[threadIdx.x] = base + before;
  rank_tile<N>(s, digit, rank, bits);
  __syncthreads();
#pragma unroll
  for (int i = 0; i < N; ++i)
    if (digit[i] < kBins) {
      const uint32_t to = s.base[digit[i]] + s.count[threadIdx.x >> 5][digit[i]] + rank[i];
      keys_out[to] = key[i];
      pos_out[to] = p0[i];
    }
}

// ---- Sums over the runs of equal tokens -----------------------------------------------------

constexpr int kSumThreads = 256;
constexpr int kBatch = 4;   // dy rows that a group requests and adds at once
constexpr int kAhead = 3;   // batches on their way

// A lane has V columns of a slab of S V: consecutive ones where V divides the width, else (kEdge) V
// that are S apart.
template <int V, int S, bool kEdge>
__device__ __forceinline__ int column(int lane, int j) {
  return kEdge ? lane + S * j : lane * V + j;
}

// The lane's columns of a row of dW; `row` is where the slab begins in it, `cols` the slab's columns.
template <typename W, int V, int S, bool kEdge>
__device__ __forceinline__ void write_row(W* row, const float (&acc)[V], float scale, int lane, int cols) {
  if constexpr (!kEdge) {
    float f[V];
#pragma unroll
    for (int j = 0; j < V; ++j) f[j] = acc[j] * scale;
    constexpr int kMost = 16 / static_cast<int>(sizeof(W));  // elements of a store
    constexpr int kEach = V < kMost ? V : kMost;
#pragma unroll
    for (int j = 0; j < V; j += kEach)
      st_vec<W, kEach>(row + lane * V + j, Vec<W, kEach>::of(reinterpret_cast<const float(&)[kEach]>(f[j])));
  } else {
#pragma unroll
    for (int j = 0; j < V; ++j)
      if (lane + S * j < cols) row[lane + S * j] = Elem<W>::store(acc[j] * scale);
  }
}

// The dy rows of a group's chunk, requested three batches ahead of their use: 16-byte vectors to a ring
// in shared memory with cp.async, which takes no registers. Where V divides the width, a lane reads
// only what it requested itself, and its own wait is enough. Else the rows begin anywhere: the group
// copies the vectors that hold its slab of the row, from the boundary at or before it on (dy begins
// on one, so that this is never outside of it), and its lanes meet before they read their elements.
template <typename T, int V, int S, bool kEdge>
struct Rows {
  static constexpr int kSlots = kAhead + 1;
  static constexpr int kRowBytes = S * 16 + (kEdge ? 16 : 0);
  static constexpr int kGroupBytes = kSlots * kBatch * kRowBytes;
  static constexpr int kRingBytes = kSumThreads / S * kGroupBytes;
  const T* dy;  // where the slab begins in the first row
  const int D, cols, lane;
  const bool mine;  // the lane has columns
  const uint32_t vocab, mask;
  char* ring;
  uint32_t lead[kEdge ? kSlots : 1];  // elements from the boundary to the slab, four bits for each row

  __device__ __forceinline__ Rows(const T* d, int width, int slab, int ln, uint32_t v, char* r)
      : dy(d + slab * S * V),
        D(width),
        cols(width - slab * S * V < S * V ? width - slab * S * V : S * V),
        lane(ln),
        mine((kEdge ? ln : ln * V) < cols),
        vocab(v),
        mask(S == 32 ? 0xffffffffu : ((1u << (S & 31)) - 1u) << (threadIdx.x & 31 & ~(S - 1))),
        ring(r + threadIdx.x / S * kGroupBytes) {}

  __device__ __forceinline__ void request(int slot, const uint32_t (&k)[kBatch], const uint32_t (&p)[kBatch]) {
    if constexpr (kEdge) {
      __syncwarp(mask);  // the slot's last rows have been read
      lead[slot] = 0;
    }
#pragma unroll
    for (int u = 0; u < kBatch; ++u) {
      if (k[u] >= vocab) continue;
      const T* row = dy + static_cast<int64_t>(p[u]) * D;
      uint32_t to = static_cast<uint32_t>(__cvta_generic_to_shared(ring + (slot * kBatch + u) * kRowBytes));
      if constexpr (!kEdge) {
        if (mine)
          asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(to + lane * 16), "l"(row + lane * V)
                       : "memory");
      } else {
        const uint32_t before = static_cast<uint32_t>(reinterpret_cast<uintptr_t>(row) & 15u);
        const char* from = reinterpret_cast<const char*>(row) - before;
        const int bytes = static_cast<int>(before) + cols * static_cast<int>(sizeof(T));
        lead[slot] |= (before / static_cast<uint32_t>(sizeof(T))) << (4 * u);
        for (int i = lane * 16; i < bytes; i += S * 16)
          asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(to + i), "l"(from + i),
                       "r"(bytes - i < 16 ? bytes - i : 16)
                       : "memory");
      }
    }
    asm volatile("cp.async.commit_group;" ::: "memory");
  }

  // The batch requested kAhead batches ago.
  __device__ __forceinline__ void arrived() {
    asm volatile("cp.async.wait_group %0;" ::"n"(kAhead) : "memory");
    if constexpr (kEdge) __syncwarp(mask);
  }
  __device__ __forceinline__ void take(int slot, int u, float (&f)[V]) const {
    const char* row = ring + (slot * kBatch + u) * kRowBytes;
    if constexpr (!kEdge) {
      const Vec<T, V> v = ld_vec<T, V>(reinterpret_cast<const T*>(row + lane * 16));
#pragma unroll
      for (int j = 0; j < V; ++j) f[j] = v.get(j);
    } else {
      const T* first = reinterpret_cast<const T*>(row) + (lead[slot] >> (4 * u) & 15u) + lane;
#pragma unroll
      for (int j = 0; j < V; ++j) f[j] = lane + S * j < cols ? Elem<T>::load(first[S * j]) : 0.f;
    }
  }
  __device__ __forceinline__ void drain() { asm volatile("cp.async.wait_group 0;" ::: "memory"); }
};

// How a group's chunk meets its neighbours. kHead: its first run began before it; kHeadOn: and
// that run goes on behind it (the chunk is one run). kTail: its last run begins in it and goes on.
constexpr uint32_t kHead = 1, kHeadOn = 2, kTail = 4;

// A group of S lanes sums the sorted entries [c L, (c + 1) L) over a slab of columns (S = 32, or
// fewer where the row is that narrow: one slab). A block is one slab of 256 / S consecutive chunks
// (a unit), joined in shared memory, so that at most two partial rows a unit go to memory:
// partial[2 u] for the run that began before it, partial[2 u + 1] for the one that begins in it
// and goes on. Groups of a warp take their own ways; what lanes exchange, they exchange in the group.
template <typename T, typename W, int V, int S, bool kEdge>
__device__ __forceinline__ void sum_unit(const T* __restrict__ dy, const uint32_t* __restrict__ keys,
                                         const uint32_t* __restrict__ pos, W* __restrict__ dw,
                                         float* __restrict__ partial, int64_t n, uint32_t vocab, int D, int L,
                                         int64_t unit, int slab, float scale, float (*edge)[2][S * V], uint32_t* how,
                                         uint32_t* run_key, char* ring) {
  constexpr int kGroups = kSumThreads / S, kRing = kAhead + 1;
  const int lane = threadIdx.x % S, group = threadIdx.x / S;
  const int64_t i0 = (unit * kGroups + group) * L;
  if (lane == 0) how[group] = 0;
  if (i0 < n) {
    const int m = static_cast<int>(i0 + L < n ? L : n - i0);
    const int batches = (m + kBatch - 1) / kBatch;
    const uint32_t left = i0 > 0 ? keys[i0 - 1] : 0xffffffffu;
    const uint32_t right = i0 + m < n ? keys[i0 + m] : 0xffffffffu;
    Rows<T, V, S, kEdge> rows(dy, D, slab, lane, vocab, ring);
    W* dw_slab = dw + slab * S * V;
    // The keys and positions of S batches, one batch per lane, and those of the next S. Chunks begin
    // on 16-byte boundaries of both arrays, whose ends are padded; places that hold no entry get a
    // key above all.
    uint4 k_now = {}, p_now = {}, k_next = {}, p_next = {};
    auto window = [&](int b, uint4& k, uint4& p) {
      k = make_uint4(0xffffffffu, 0xffffffffu, 0xffffffffu, 0xffffffffu);
      p = make_uint4(0, 0, 0, 0);
      const int left_over = m - (b + lane) * kBatch;
      if (left_over <= 0) return;
      const uint4 a = *reinterpret_cast<const uint4*>(keys + i0 + (b + lane) * kBatch);
      p = *reinterpret_cast<const uint4*>(pos + i0 + (b + lane) * kBatch);
      k.x = a.x;
      if (left_over > 1) k.y = a.y;
      if (left_over > 2) k.z = a.z;
      if (left_over > 3) k.w = a.w;
    };
    uint32_t key[kRing][kBatch];
    auto request = [&](int slot, int b) {  // b: of the window
      uint32_t p[kBatch];
      key[slot][0] = __shfl_sync(rows.mask, k_now.x, b, S);
      key[slot][1] = __shfl_sync(rows.mask, k_now.y, b, S);
      key[slot][2] = __shfl_sync(rows.mask, k_now.z, b, S);
      key[slot][3] = __shfl_sync(rows.mask, k_now.w, b, S);
      p[0] = __shfl_sync(rows.mask, p_now.x, b, S);
      p[1] = __shfl_sync(rows.mask, p_now.y, b, S);
      p[2] = __shfl_sync(rows.mask, p_now.z, b, S);
      p[3] = __shfl_sync(rows.mask, p_now.w, b, S);
      rows.request(slot, key[slot], p);
    };
    window(0, k_now, p_now);
    window(S, k_next, p_next);
#pragma unroll
    for (int b = 0; b < kAhead; ++b) request(b, b);
    float acc[V];
#pragma unroll
    for (int j = 0; j < V; ++j) acc[j] = 0.f;
    uint32_t cur = key[0][0];
    bool continued = cur == left;  // the current run began in an earlier chunk
    uint32_t flags = continued && cur < vocab ? kHead : 0u;
    if (lane == 0) run_key[group] = cur;
    for (int b0 = 0; b0 < batches; b0 += kRing) {
#pragma unroll
      for (int g = 0; g < kRing; ++g) {
        if (b0 + g >= batches) break;
        // a later batch is on its way while this one is added up; the first of a window is
        // always requested at g = 1
        const int ahead = b0 + g + kAhead;
        if (g == 1 && ahead % S == 0) {
          k_now = k_next;
          p_now = p_next;
          window(ahead + S, k_next, p_next);
        }
        request((g + kAhead) % kRing, ahead % S);
        rows.arrived();
        const uint32_t(&k)[kBatch] = key[g];
        float f[kBatch][V];
#pragma unroll
        for (int u = 0; u < kBatch; ++u) rows.take(g, u, f[u]);
        if (k[0] == cur && k[kBatch - 1] == cur && cur < vocab) {  // all of the current run: a tree
#pragma unroll
          for (int j = 0; j < V; ++j) acc[j] += (f[0][j] + f[1][j]) + (f[2][j] + f[3][j]);
          continue;
        }
#pragma unroll
        for (int u = 0; u < kBatch; ++u) {
          if (k[u] >= vocab) continue;  // none, or sorted last: nothing follows but more of them
          if (k[u] != cur) {
            if (rows.mine) {
              if (continued)
#pragma unroll
                for (int j = 0; j < V; ++j) edge[group][0][column<V, S, kEdge>(lane, j)] = acc[j];
              else
                write_row<W, V, S, kEdge>(dw_slab + static_cast<int64_t>(cur) * D, acc, scale, lane, rows.cols);
            }
            cur = k[u];
            continued = false;
#pragma unroll
            for (int j = 0; j < V; ++j) acc[j] = 0.f;
          }
#pragma unroll
          for (int j = 0; j < V; ++j) acc[j] += f[u][j];
        }
      }
    }
    rows.drain();
    if (cur < vocab) {
      const bool goes_on = cur == right;
      if (!goes_on && !continued) {
        if (rows.mine) write_row<W, V, S, kEdge>(dw_slab + static_cast<int64_t>(cur) * D, acc, scale, lane, rows.cols);
      } else {
        flags |= continued ? (goes_on ? kHeadOn : 0u) : kTail;
        if (rows.mine)
#pragma unroll
          for (int j = 0; j < V; ++j) edge[group][continued ? 0 : 1][column<V, S, kEdge>(lane, j)] = acc[j];
      }
    }
    if (lane == 0) how[group] = flags;
  }
  __syncthreads();
  // the unit's chunks in order, one column per thread
  for (int x = threadIdx.x; x < S * V; x += kSumThreads) {
    const int c = slab * S * V + x;
    if (c >= D) continue;
    float acc = 0.f;
    bool carrying = false, began_here = false;
    for (int w = 0; w < kGroups; ++w) {
      const uint32_t f = how[w];
      if (f & kHead) {
        acc += edge[w][0][x];
        carrying = true;
        if (!(f & kHeadOn)) {
          if (began_here)
            dw[static_cast<int64_t>(run_key[w]) * D + c] = Elem<W>::store(acc * scale);
          else
            partial[unit * 2 * D + c] = acc;
          acc = 0.f;
          carrying = began_here = false;
        }
      }
      if (f & kTail) {
        acc = edge[w][1][x];
        carrying = began_here = true;
      }
    }
    if (carrying) partial[(unit * 2 + (began_here ? 1 : 0)) * D + c] = acc;
  }
}

// Blocks [0, units * slabs) sum; those behind them zero the rows of the tokens that do not occur:
// 32 rows and zero_cols columns per warp, a binary search of the sorted keys for each row.
template <typename T, typename W, int V, int S, bool kEdge>
__global__ void __launch_bounds__(kSumThreads, 2)
    run_sums_kernel(const T* __restrict__ dy, const uint32_t* __restrict__ keys, const uint32_t* __restrict__ pos,
                    W* __restrict__ dw, float* __restrict__ partial, int64_t n, uint32_t vocab, int D, int L,
                    int slabs, int64_t sum_blocks, int zero_cols, int zero_slabs, float scale) {
  wait_previous_kernel();
  extern __shared__ __align__(16) char ring[];
  constexpr int kGroups = kSumThreads / S;
  __shared__ float edge[kGroups][2][S * V];
  __shared__ uint32_t how[kGroups], run_key[kGroups];
  if (blockIdx.x < sum_blocks) {
    const int64_t unit = blockIdx.x / static_cast<uint32_t>(slabs);
    sum_unit<T, W, V, S, kEdge>(dy, keys, pos, dw, partial, n, vocab, D, L, unit,
                                static_cast<int>(blockIdx.x - unit * slabs), scale, edge, how, run_key, ring);
    return;
  }
  const int lane = threadIdx.x & 31;
  const int64_t item = (blockIdx.x - sum_blocks) * (kSumThreads / 32) + (threadIdx.x >> 5);
  const int64_t row0 = item / zero_slabs * 32;
  if (row0 >= vocab) return;
  const uint32_t v = static_cast<uint32_t>(row0) + lane;
  int64_t lo = 0, hi = n;  // the first entry with keys >= v
  while (lo < hi) {
    const int64_t mid = (lo + hi) >> 1;
    if (keys[mid] < v)
      lo = mid + 1;
    else
      hi = mid;
  }
  uint32_t absent = __ballot_sync(0xffffffffu, v < vocab && !(lo < n && keys[lo] == v));
  const int c0 = static_cast<int>(item % zero_slabs) * zero_cols;
  const int c1 = c0 + zero_cols < D ? c0 + zero_cols : D;
  constexpr int Z = kEdge ? 1 : 16 / static_cast<int>(sizeof(W));
  for (; absent; absent &= absent - 1) {
    W* row = dw + (row0 + __ffs(absent) - 1) * D;
    for (int c = c0 + lane * Z; c < c1; c += 32 * Z) st_vec<W, Z>(row + c, Vec<W, Z>::zero());
  }
}

// The runs that cross units: the block of the unit in which one begins adds its tail and the heads
// of the units after it, 128 columns at a time.
constexpr int kJoinCols = 128;
constexpr int kJoinThreads = 512;
constexpr int kJoinWarps = kJoinThreads / 32;

template <typename W>
__global__ void __launch_bounds__(kJoinThreads)
    join_runs_kernel(const uint32_t* __restrict__ keys, const float* __restrict__ partial, W* __restrict__ dw,
                     int64_t n, uint32_t vocab, int D, int64_t unit_len, int slabs, float scale) {
  wait_previous_kernel();
  __shared__ float part[kJoinWarps][kJoinCols];
  const int64_t u = blockIdx.x / static_cast<uint32_t>(slabs);
  const int col0 = static_cast<int>(blockIdx.x - u * slabs) * kJoinCols;
  const int64_t i0 = u * unit_len, i1 = i0 + unit_len;
  if (i1 >= n) return;  // the last unit starts no run that goes on
  const uint32_t k = keys[i1 - 1];
  if (k >= vocab || keys[i1] != k) return;
  if (i0 > 0 && keys[i0] == k && keys[i0 - 1] == k) return;  // it began earlier
  // the units behind it whose first entry belongs to the run
  int64_t heads = 0;
  for (int count = kJoinThreads; count == kJoinThreads; heads += count) {
    const int64_t j = (u + 1 + heads + threadIdx.x) * unit_len;
    count = __syncthreads_count(j < n && keys[j] == k);
  }
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  float s[kJoinCols / 32] = {};
  constexpr int kAtOnce = 8;
  for (int64_t j0 = warp; j0 <= heads; j0 += kJoinWarps * kAtOnce) {  // 0: the tail, then the heads
    float t[kAtOnce][kJoinCols / 32];
#pragma unroll
    for (int v = 0; v < kAtOnce; ++v) {
      const int64_t j = j0 + v * kJoinWarps;
      const float* p = partial + (j == 0 ? u * 2 + 1 : (u + j) * 2) * D + col0 + lane;
#pragma unroll
      for (int i = 0; i < kJoinCols / 32; ++i) t[v][i] = j <= heads && col0 + lane + 32 * i < D ? p[32 * i] : 0.f;
    }
#pragma unroll
    for (int i = 0; i < kJoinCols / 32; ++i)
      s[i] += ((t[0][i] + t[1][i]) + (t[2][i] + t[3][i])) + ((t[4][i] + t[5][i]) + (t[6][i] + t[7][i]));
  }
#pragma unroll
  for (int i = 0; i < kJoinCols / 32; ++i) part[warp][lane + 32 * i] = s[i];
  __syncthreads();
  const int c = col0 + threadIdx.x;
  if (threadIdx.x >= kJoinCols || c >= D) return;
  float t[kJoinWarps];
#pragma unroll
  for (int w = 0; w < kJoinWarps; ++w) t[w] = part[w][threadIdx.x];
#pragma unroll
  for (int o = kJoinWarps / 2; o > 0; o >>= 1)
#pragma unroll
    for (int w = 0; w < o; ++w) t[w] += t[w + o];
  dw[static_cast<int64_t>(k) * D + c] = Elem<W>::store(t[0] * scale);
}

// ---- Forward ----------------------------------------------------------------------------------

constexpr int kAtOnce = 4;  // vectors of a thread on their way

// y = scale W[tokens], as one array in vectors of V elements: thread by thread along tiles of
// `tile_rows` rows (which begin on 16-byte boundaries), so that narrow rows and those that no vector
// divides (kEdge) are written in whole vectors as well. by_row divides by the row's vectors, or
// with kEdge by its elements.
template <typename T, typename I, int V, bool kEdge>
__global__ void __launch_bounds__(256)
    lookup_kernel(const I* __restrict__ tokens, const T* __restrict__ w, T* __restrict__ y, int64_t n, int64_t vocab,
                  int D, Divisor by_row, int tile_rows, float scale, bool streaming, uint32_t* status) {
  bool bad = false;
  const int64_t tiles = (n + tile_rows - 1) / tile_rows;
  for (int64_t tile = blockIdx.x; tile < tiles; tile += gridDim.x) {
    const int64_t row0 = tile * tile_rows;
    const int rows = static_cast<int>(n - row0 < tile_rows ? n - row0 : tile_rows);
    const uint32_t elements = static_cast<uint32_t>(rows) * static_cast<uint32_t>(D);
    const uint32_t vectors = (elements + V - 1) / V;
    const I* tok = tokens + row0;
    T* out = y + row0 * D;
    auto token = [&](uint32_t r) {
      const int64_t t = static_cast<int64_t>(tok[r]);
      const bool ok = t >= 0 && t < vocab;
      if (!ok) bad = true;
      return ok ? t : int64_t(-1);
    };
    for (uint32_t v0 = threadIdx.x; v0 < vectors; v0 += blockDim.x * kAtOnce) {
      Vec<T, V> e[kAtOnce];
      if constexpr (!kEdge) {
        int64_t at[kAtOnce];
#pragma unroll
        for (int q = 0; q < kAtOnce; ++q) {
          const uint32_t v = v0 + q * blockDim.x;
          at[q] = -1;
          if (v >= vectors) continue;
          const uint32_t r = by_row.quotient(v);
          const int64_t t = token(r);
          if (t >= 0) at[q] = t * D + static_cast<int64_t>(v - r * by_row.d) * V;
        }
#pragma unroll
        for (int q = 0; q < kAtOnce; ++q) e[q] = at[q] >= 0 ? ld_vec<T, V>(w + at[q]) : Vec<T, V>::zero();
      } else {
#pragma unroll
        for (int q = 0; q < kAtOnce; ++q) {
          const uint32_t v = v0 + q * blockDim.x;
          float f[V] = {};
          if (v < vectors) {
            uint32_t r = by_row.quotient(v * V), c = v * V - r * D;
            int64_t t = token(r);
            if (c + V <= static_cast<uint32_t>(D)) {  // inside one row
              const T* from = w + (t >= 0 ? t * D + c : 0);
#pragma unroll
              for (int j = 0; j < V; ++j) f[j] = t >= 0 ? Elem<T>::load(from[j]) : 0.f;
            } else {
#pragma unroll
              for (int j = 0; j < V; ++j) {
                if (v * V + j >= elements) break;
                if (c == static_cast<uint32_t>(D)) {
                  c = 0;
                  t = token(++r);
                }
                if (t >= 0) f[j] = Elem<T>::load(w[t * D + c]);
                ++c;
              }
            }
          }
          e[q] = Vec<T, V>::of(f);
        }
      }
#pragma unroll
      for (int q = 0; q < kAtOnce; ++q) {
        const uint32_t v = v0 + q * blockDim.x;
        if (v >= vectors) continue;
        float o[V];
#pragma unroll
        for (int j = 0; j < V; ++j) o[j] = e[q].get(j) * scale;
        T* to = out + static_cast<int64_t>(v) * V;
        if (kEdge && v * V + V > elements) {  // the last vector of the array
#pragma unroll
          for (int j = 0; j < V; ++j)
            if (v * V + j < elements) to[j] = Elem<T>::store(o[j]);
        } else if (streaming) {
          st_vec_streaming<T, V>(to, Vec<T, V>::of(o));
        } else {
          st_vec<T, V>(to, Vec<T, V>::of(o));
        }
      }
    }
  }
  if (status && bad) atomicOr(status, GTK_STATUS_BAD_TOKEN);
}

// ---- Host ---------------------------------------------------------------------------------------

int check_sizes(int64_t T, int64_t vocab, int64_t D) {
  if (!dims_ok(T, (int64_t(1) << 31) - 1)) return fail(GTK_ERR_INVALID_ARG, "embedding: tokens must be 1..2^31-1");
  if (!dims_ok(vocab, (int64_t(1) << 31) - 1))
    return fail(GTK_ERR_INVALID_ARG, "embedding: vocabulary must be 1..2^31-1");
  if (!dims_ok(D, kMaxWidth)) return fail(GTK_ERR_INVALID_ARG, "embedding: width must be 1..2^20");
  return GTK_OK;
}

// The backward's plan: what the workspace holds and how the sorted list is cut.
struct Plan {
  int passes, bits;  // of the sort, for keys 0 .. vocab
  int per;           // tokens per thread, of the sort over tiles
  int64_t tiles;
  bool zero_first;   // all of dW is zeroed beside the sort
  int lanes;                                   // of a group: 4 to 32, as many as have columns
  int64_t L, units;                            // entries of a group's chunk; units of 256 / lanes chunks
  size_t keys, pos, counts, partial, total;    // byte offsets (keys, pos: two buffers each)
};

Plan plan_for(int64_t T, int64_t vocab, int64_t D, int dy_dtype, int w_dtype) {
  Plan p = {};
  int bits = 1;
  while (vocab >> bits) ++bits;
  p.passes = (bits + kMaxBits - 1) / kMaxBits;
  p.bits = (bits + p.passes - 1) / p.passes;
  // up to 128 tiles: a tile's places come from all tiles' counts, but its scattered stores (the longest
  // part, 19 us with 8192 tokens a tile) take the shorter the fewer they are
  p.per = 1;
  while (p.per < kMaxPer && T > int64_t(128) * kSortThreads * p.per) p.per <<= 1;
  p.tiles = (T + kSortThreads * p.per - 1) / (kSortThreads * p.per);
  // The sort of a short list leaves most of the device idle for some 8 us, in which it can zero
  // all of dW. The rows that do occur are then written twice, which costs less than that time
  // as long as they are at most 32 MB (8192 tokens, 32000 x 1024 bf16: the whole gradient takes
  // 26.7 us, against 28.8 when the absent rows are looked up and zeroed after the sort).
  p.zero_first = T <= kClusterTokens &&
                 (T < vocab ? T : vocab) * D * static_cast<int64_t>(dtype_bytes(w_dtype)) <= (32 << 20);
  const int each = 16 / static_cast<int>(dtype_bytes(dy_dtype));  // columns of a lane
  p.lanes = 4;
  while (p.lanes < 32 && static_cast<int64_t>(p.lanes) * each < D) p.lanes <<= 1;
  // About 8 warps per SM, in whole batches (24: 5 to 15% slower, more runs cross chunks); 16 where rows
  // are taken apart by element, which takes longer per byte. Up to 512 tokens make one unit: the
  // launch that joins units costs more than the longer chunks.
  const int64_t slabs = (D + p.lanes * each - 1) / (p.lanes * each), groups = kSumThreads / p.lanes;
  const int64_t per_device = 148 * (D % each ? 2 : 1) * groups;
  int64_t L = T <= 512 ? (T + groups - 1) / groups : (T * slabs + per_device - 1) / per_device;
  L = (L + kBatch - 1) / kBatch * kBatch;
  p.L = L > 1024 ? 1024 : L;
  p.units = (T + p.L * groups - 1) / (p.L * groups);
  size_t at = 0;
  auto take = [&](size_t bytes) {
    const size_t o = at;
    at += round_up(bytes, 256);
    return o;
  };
  const bool tiled = T > kClusterTokens, two = tiled && p.passes > 1;
  p.keys = take((two ? 2 : 1) * round_up(4 * T, 256));
  p.pos = take((two ? 2 : 1) * round_up(4 * T, 256));
  p.counts = take(tiled ? 4 * kBins * p.tiles : 0);
  p.partial = take(p.units > 1 ? static_cast<size_t>(p.units) * 2 * D * sizeof(float) : 0);
  p.total = at;
  return p;
}

struct Args {
  const void *tokens, *dy;
  void* dw;
  char* ws;
  int64_t T, vocab, D, padding, dw_bytes;
  float scale;
  uint32_t* status;
  cudaStream_t st;
};

template <typename I>
int sort_cluster(const Args& a, const Plan& p, uint32_t* keys, uint32_t* pos) {
  auto kernel = sort_cluster_kernel<I>;
  const int smem = 2 * kSortThreads * 4;
  if (int e = ensure_smem(reinterpret_cast<const void*>(kernel), smem)) return e;
  int blocks = 1;
  while (static_cast<int64_t>(blocks) * kSortThreads < a.T) blocks <<= 1;
  const int64_t zero_bytes = p.zero_first ? a.dw_bytes : 0;
  // two blocks per SM, in whole clusters, but no more than there are 64 KB pieces
  int64_t zero_blocks = (zero_bytes + 65535) / 65536;
  if (zero_blocks > 2 * num_sms()) zero_blocks = 2 * num_sms();
  zero_blocks = (zero_blocks + blocks - 1) / blocks * blocks;
  return launch_clusters("embedding token sort", kernel, blocks + zero_blocks, kSortThreads, smem, blocks, a.st,
                         static_cast<const I*>(a.tokens), static_cast<int>(a.T), static_cast<uint32_t>(a.vocab),
                         a.padding, p.passes, p.bits, keys, pos, static_cast<uint4*>(a.dw), zero_bytes, a.status);
}

// Two launches a pass; keys and positions alternate between two buffers.
template <typename I, int N>
int sort_tiles(const Args& a, const Plan& p, uint32_t* const (&k)[2], uint32_t* const (&q)[2], const uint32_t** keys,
               const uint32_t** pos) {
  const I* tokens = static_cast<const I*>(a.tokens);
  const uint32_t V = static_cast<uint32_t>(a.vocab);
  uint32_t* counts = reinterpret_cast<uint32_t*>(a.ws + p.counts);
  const uint32_t *ki = nullptr, *qi = nullptr;
  for (int pass = 0; pass < p.passes; ++pass) {
    uint32_t *ko = k[pass & 1], *qo = q[pass & 1];
    if (int e = launch("embedding token count", count_kernel<I, N>, p.tiles, kSortThreads, 0, a.st, pass > 0, tokens,
                       ki, a.T, V, a.padding, pass, p.bits, counts, a.status))
      return e;
    if (int e = launch("embedding token scatter", scatter_kernel<I, N>, p.tiles, kSortThreads, 0, a.st, true, tokens,
                       ki, qi, a.T, V, a.padding, pass, p.bits, static_cast<const uint32_t*>(counts),
                       static_cast<int>(p.tiles), ko, qo))
      return e;
    ki = ko;
    qi = qo;
  }
  *keys = ki;
  *pos = qi;
  return GTK_OK;
}

template <typename I>
int sort(const Args& a, const Plan& p, const uint32_t** keys, const uint32_t** pos) {
  const size_t half = round_up(4 * a.T, 256);
  uint32_t* k[2] = {reinterpret_cast<uint32_t*>(a.ws + p.keys), reinterpret_cast<uint32_t*>(a.ws + p.keys + half)};
  uint32_t* q[2] = {reinterpret_cast<uint32_t*>(a.ws + p.pos), reinterpret_cast<uint32_t*>(a.ws + p.pos + half)};
  if (a.T <= kClusterTokens) {
    *keys = k[0];
    *pos = q[0];
    return sort_cluster<I>(a, p, k[0], q[0]);
  }
  switch (p.per) {
    case 1:
      return sort_tiles<I, 1>(a, p, k, q, keys, pos);
    case 2:
      return sort_tiles<I, 2>(a, p, k, q, keys, pos);
    case 4:
      return sort_tiles<I, 4>(a, p, k, q, keys, pos);
    default:
      return sort_tiles<I, kMaxPer>(a, p, k, q, keys, pos);
  }
}

template <typename T, typename W, int S, bool kEdge>
int sums(const Args& a, const Plan& p, const uint32_t* keys, const uint32_t* pos) {
  constexpr int V = 16 / static_cast<int>(sizeof(T)), kCols = S * V;
  const int slabs = static_cast<int>((a.D + kCols - 1) / kCols);
  const int64_t sum_blocks = p.units * slabs;
  constexpr int kPerBlock = kSumThreads / 32;
  const int zero_cols = 1024;
  const int zero_slabs = static_cast<int>((a.D + zero_cols - 1) / zero_cols);
  const int64_t zero_blocks =
      p.zero_first ? 0 : ((a.vocab + 31) / 32 * zero_slabs + kPerBlock - 1) / kPerBlock;
  const int join_slabs = static_cast<int>((a.D + kJoinCols - 1) / kJoinCols);
  if (sum_blocks + zero_blocks > (int64_t(1) << 31) - 1 || p.units * join_slabs > (int64_t(1) << 31) - 1)
    return fail(GTK_ERR_UNSUPPORTED, "embedding: tokens or vocabulary times width too large");
  float* partial = reinterpret_cast<float*>(a.ws + p.partial);
  const uint32_t V32 = static_cast<uint32_t>(a.vocab);
  auto kernel = run_sums_kernel<T, W, V, S, kEdge>;
  constexpr int kSmem = Rows<T, V, S, kEdge>::kRingBytes;
  if (int e = ensure_smem(reinterpret_cast<const void*>(kernel), kSmem)) return e;
  if (int e = launch("embedding run sums", kernel, sum_blocks + zero_blocks, kSumThreads, kSmem, a.st, true,
                     static_cast<const T*>(a.dy), keys, pos, static_cast<W*>(a.dw), partial, a.T, V32,
                     static_cast<int>(a.D), static_cast<int>(p.L), slabs, sum_blocks, zero_cols, zero_slabs, a.scale))
    return e;
  if (p.units == 1) return GTK_OK;
  return launch("embedding run join", join_runs_kernel<W>, (p.units - 1) * join_slabs, kJoinThreads, 0, a.st, true,
                keys, static_cast<const float*>(partial), static_cast<W*>(a.dw), a.T, V32, static_cast<int>(a.D),
                p.L * (kSumThreads / S), join_slabs, a.scale);
}

template <typename T, typename W, bool kEdge>
int sums_by_lanes(const Args& a, const Plan& p, const uint32_t* keys, const uint32_t* pos) {
  switch (p.lanes) {
    case 4:
      return sums<T, W, 4, kEdge>(a, p, keys, pos);
    case 8:
      return sums<T, W, 8, kEdge>(a, p, keys, pos);
    case 16:
      return sums<T, W, 16, kEdge>(a, p, keys, pos);
    default:
      return sums<T, W, 32, kEdge>(a, p, keys, pos);
  }
}

template <typename T, typename W>
int backward_typed(const Args& a, const Plan& p, const uint32_t* keys, const uint32_t* pos) {
  return a.D % (16 / static_cast<int>(sizeof(T))) ? sums_by_lanes<T, W, true>(a, p, keys, pos)
                                                  : sums_by_lanes<T, W, false>(a, p, keys, pos);
}

template <typename T, typename I>
int forward_typed(const Args& a, const void* w, void* y) {
  constexpr int VX = 16 / static_cast<int>(sizeof(T));
  const bool edge = a.D % VX != 0 || !aligned16(w);  // rows of the table by element
  const bool vec = aligned16(y);                     // else the output too
  auto kernel = !vec   ? lookup_kernel<T, I, 1, false>
                : edge ? lookup_kernel<T, I, VX, true>
                       : lookup_kernel<T, I, VX, false>;
  // Tiles of about 8192 elements, smaller where that leaves the device idle, in whole vectors.
  int64_t rows = 8192 / a.D, few = (a.T + 4 * num_sms() - 1) / (4 * num_sms());
  if (rows > few) rows = few;
  rows = rows < 8 ? (edge ? 8 : rows < 1 ? 1 : rows) : rows / 8 * 8;
  const int64_t tiles = (a.T + rows - 1) / rows, cap = int64_t(1) << 30;
  // An output that the L2 cache cannot hold anyway is written past it (512 x 512 pairs of 128 fp32
  // channels: 24.7 us instead of 30.9); a small one stays there for its reader.
  const bool streaming = a.T * a.D * static_cast<int64_t>(sizeof(T)) > (int64_t(64) << 20);
  const Divisor by_row = divisor(static_cast<uint32_t>(vec && !edge ? a.D / VX : a.D));
  return launch("embedding lookup", kernel, tiles < cap ? tiles : cap, 256, 0, a.st, false,
                static_cast<const I*>(a.tokens), static_cast<const T*>(w), static_cast<T*>(y), a.T, a.vocab,
                static_cast<int>(a.D), by_row, static_cast<int>(rows), a.scale, streaming, a.status);
}

template <typename I>
int forward_by_type(const Args& a, const void* w, void* y, int dtype) {
  if (dtype == GTK_F32) return forward_typed<float, I>(a, w, y);
  if (dtype == GTK_BF16) return forward_typed<__nv_bfloat16, I>(a, w, y);
  return forward_typed<__half, I>(a, w, y);
}

int check_tokens(const void* tokens, int index_bits) {
  if (index_bits != 32 && index_bits != 64)
    return fail(GTK_ERR_UNSUPPORTED, "embedding: tokens are int32 or int64");
  return check_ptr(tokens, "tokens", index_bits / 8);
}

}  // namespace emb
}  // namespace gtk

using namespace gtk;

extern "C" {

int gtk_embedding_forward(const void* tokens, int index_bits, const void* weight, int dtype, void* y, int64_t n_tokens,
                          int64_t vocab, int64_t D, float scale, uint32_t* status, void* stream) try {
  if (int e = emb::check_sizes(n_tokens, vocab, D)) return e;
  if (!dtype_ok(dtype)) return fail(GTK_ERR_UNSUPPORTED, "embedding: the table is fp32, bf16 or fp16");
  if (int e = emb::check_tokens(tokens, index_bits)) return e;
  if (int e = check_ptr(weight, "weight", dtype_bytes(dtype))) return e;
  if (int e = check_ptr(y, "y", dtype_bytes(dtype))) return e;
  if (int e = check_device()) return e;
  emb::Args a = {};
  a.tokens = tokens, a.T = n_tokens, a.vocab = vocab, a.D = D, a.scale = scale, a.status = status;
  a.st = static_cast<cudaStream_t>(stream);
  return index_bits == 64 ? emb::forward_by_type<int64_t>(a, weight, y, dtype)
                          : emb::forward_by_type<int32_t>(a, weight, y, dtype);
} catch (...) {
  return fail_no_memory();
}

size_t gtk_embedding_backward_workspace_bytes(int64_t n_tokens, int64_t vocab, int64_t D, int dy_dtype) {
  if (!dims_ok(n_tokens) || !dims_ok(vocab) || !dims_ok(D, emb::kMaxWidth) || !dtype_ok(dy_dtype)) return 0;
  return emb::plan_for(n_tokens, vocab, D, dy_dtype, dy_dtype).total;
}

int gtk_embedding_backward(const void* dy, int dy_dtype, const void* tokens, int index_bits, void* dweight,
                           int w_dtype, int64_t n_tokens, int64_t vocab, int64_t D, float scale, int64_t padding,
                           void* workspace, size_t workspace_bytes, uint32_t* status, void* stream) try {
  if (int e = emb::check_sizes(n_tokens, vocab, D)) return e;
  // every tile of the sort reads all tiles' counts: beyond this it would take longer than it is worth
  if (n_tokens > emb::kMaxSorted) return fail(GTK_ERR_UNSUPPORTED, "embedding: the gradient takes up to 2^27 tokens");
  if (!dtype_ok(dy_dtype) || !(w_dtype == dy_dtype || w_dtype == GTK_F32))
    return fail(GTK_ERR_UNSUPPORTED, "embedding: dy is fp32, bf16 or fp16, the table's gradient fp32 or dy's type");
  if (padding >= vocab) return fail(GTK_ERR_INVALID_ARG, "embedding: the padding token must be below the vocabulary");
  emb::Plan p = emb::plan_for(n_tokens, vocab, D, dy_dtype, w_dtype);
  if (workspace_bytes < p.total) return fail(GTK_ERR_WORKSPACE, "embedding: workspace too small");
  if (int e = emb::check_tokens(tokens, index_bits)) return e;
  if (int e = check_ptr(dy, "dy")) return e;
  if (int e = check_ptr(dweight, "dweight")) return e;
  if (int e = check_ptr(workspace, "workspace", 256)) return e;
  if (int e = check_device()) return e;
  emb::Args a = {};
  a.tokens = tokens, a.dy = dy, a.dw = dweight, a.ws = static_cast<char*>(workspace), a.T = n_tokens;
  a.vocab = vocab, a.D = D, a.padding = padding, a.scale = scale, a.status = status;
  a.dw_bytes = vocab * D * static_cast<int64_t>(dtype_bytes(w_dtype));
  p.zero_first = p.zero_first && a.dw_bytes % 16 == 0;
  a.st = static_cast<cudaStream_t>(stream);
  const uint32_t *keys = nullptr, *pos = nullptr;
  if (int e = index_bits == 64 ? emb::sort<int64_t>(a, p, &keys, &pos) : emb::sort<int32_t>(a, p, &keys, &pos))
    return e;
  if (dy_dtype == GTK_F32) return emb::backward_typed<float, float>(a, p, keys, pos);
  if (dy_dtype == GTK_BF16)
    return w_dtype == GTK_F32 ? emb::backward_typed<__nv_bfloat16, float>(a, p, keys, pos)
                              : emb::backward_typed<__nv_bfloat16, __nv_bfloat16>(a, p, keys, pos);
  return w_dtype == GTK_F32 ? emb::backward_typed<__half, float>(a, p, keys, pos)
                            : emb::backward_typed<__half, __half>(a, p, keys, pos);
} catch (...) {
  return fail_no_memory();
}

}  // extern "C"
