// Embedding lookup with scaling, and its gradient by sorted tokens:
//
//   y_t  = s W[tok_t]                      (a gather; zeros for a token outside 0 .. V-1)
//   dW_v = s sum_{t : tok_t = v} dy_t      (zeros for a token that does not occur, and padding)
//
// Forward: HBM bound. It writes T rows and reads each row of W that occurs at least once; a
// warp copies rows in 16-byte vectors, several rows at a time so that the loads of the tokens
// and of the rows behind them overlap.
//
// Backward: HBM bound too -- it reads dy once and writes the whole of dW once -- if the rows
// of one token can be found together. So the tokens are sorted first (stable, least digit
// first, in at most four passes of 8 bits; four bytes of key and four of position per token, small
// beside dy), and the sorted list is cut into chunks of equal length, whatever the tokens'
// frequencies: a warp sums the dy rows of its chunk in registers, in list order, and writes a
// row of dW at each change of token. A token whose run crosses chunks gets its partial sums
// from a scratch buffer: each chunk writes at most one for the run it continues ("head") and
// one for the run it starts and does not finish ("tail"); a last kernel adds them in order.
// Rows of tokens that do not occur are zeroed by further warps from a bitmap of the tokens.
// No atomics on floating-point values: the same inputs give the same bits. Sums are fp32 in a
// chunk and 64-bit between chunks; dW is rounded once.
#include <vector>

#include "train_common.cuh"

namespace gtk {
namespace emb {

constexpr int kSortThreads = 1024;
constexpr int kSortPer = 8;
constexpr int kTile = kSortThreads * kSortPer;  // tokens of one sorting block
constexpr int kBins = 256;
constexpr int kWarps = kSortThreads / 32;
constexpr int kMaxWidth = 1 << 20;

// The key of token t: itself, or V (sorted last and then ignored) when it is out of range or padding.
template <typename I>
__device__ __forceinline__ uint32_t key_of(const I* tokens, int64_t t, uint32_t V, int64_t padding, bool* bad) {
  const int64_t v = static_cast<int64_t>(tokens[t]);
  if (v < 0 || v >= static_cast<int64_t>(V)) {
    *bad = true;
    return V;
  }
  return v == padding ? V : static_cast<uint32_t>(v);
}

// Peers of this lane with the same digit, among the active lanes.
__device__ __forceinline__ uint32_t same_digit(uint32_t active, uint32_t d) { return __match_any_sync(active, d); }

struct SortShared {
  uint16_t count[kWarps][kBins];
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
  __syncthreads();
  return before + x - v;
}

// Stable rank of the tile's elements by digit: thread's element i (tile index
// warp * 32 * kSortPer + i * 32 + lane) has `digit[i]`, kBins where there is no element. After
// the call s.count[w][b] holds the number of elements of digit b in the warps before w, and
// rank[i] the element's rank among its warp's elements of that digit; the total of digit
// threadIdx.x is returned to the first kBins threads.
__device__ __forceinline__ uint32_t rank_tile(SortShared& s, const uint32_t (&digit)[kSortPer],
                                              uint32_t (&rank)[kSortPer]) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  for (int b = lane; b < kBins; b += 32) s.count[warp][b] = 0;
  __syncwarp();
#pragma unroll
  for (int i = 0; i < kSortPer; ++i) {
    const uint32_t d = digit[i];
    const uint32_t peers = same_digit(0xffffffffu, d);
    const uint32_t before = d < kBins ? s.count[warp][d] : 0;
    __syncwarp();
    rank[i] = before + __popc(peers & ((1u << lane) - 1u));
    if (d < kBins && (peers >> lane) == 1u) s.count[warp][d] = static_cast<uint16_t>(rank[i] + 1);
    __syncwarp();
  }
  __syncthreads();
  uint32_t total = 0;
  if (threadIdx.x < kBins)
    for (int w = 0; w < kWarps; ++w) {
      const uint32_t n = s.count[w][threadIdx.x];
      s.count[w][threadIdx.x] = static_cast<uint16_t>(total);
      total += n;
    }
  return total;
}

__device__ __forceinline__ int tile_index(int i) {
  return (threadIdx.x >> 5) * 32 * kSortPer + i * 32 + (threadIdx.x & 31);
}

// Marks `key` in the bitmap of occurring tokens.
__device__ __forceinline__ void mark(uint32_t* present, uint32_t key) {
  const uint32_t bit = 1u << (key & 31);
  if (!(__ldcg(present + (key >> 5)) & bit)) atomicOr(present + (key >> 5), bit);
}

// All of the sort in one block: T <= kTile. Keys and positions stay in registers between the
// passes and cross through shared memory.
template <typename I>
__global__ void __launch_bounds__(kSortThreads)
    sort_small_kernel(const I* __restrict__ tokens, int T, uint32_t V, int64_t padding, int passes,
                      uint32_t* __restrict__ keys_out, uint32_t* __restrict__ pos_out, uint32_t* __restrict__ present,
                      uint32_t* status) {
  extern __shared__ uint32_t buf[];  // [2][kTile]: keys, positions
  __shared__ SortShared s;
  uint32_t* bk = buf;
  uint32_t* bp = buf + kTile;
  for (uint32_t w = threadIdx.x; w < (V + 31) / 32; w += kSortThreads) present[w] = 0;
  __syncthreads();
  bool bad = false;
  uint32_t key[kSortPer], pos[kSortPer];
#pragma unroll
  for (int i = 0; i < kSortPer; ++i) {
    const int t = tile_index(i);
    pos[i] = static_cast<uint32_t>(t);
    key[i] = t < T ? key_of(tokens, t, V, padding, &bad) : 0xffffffffu;
    if (key[i] < V) mark(present, key[i]);
  }
  for (int p = 0; p < passes; ++p) {
    uint32_t digit[kSortPer], rank[kSortPer];
#pragma unroll
    for (int i = 0; i < kSortPer; ++i) digit[i] = tile_index(i) < T ? (key[i] >> (8 * p)) & 255u : kBins;
    const uint32_t total = rank_tile(s, digit, rank);
    const uint32_t base = scan_bins(s, threadIdx.x < kBins ? total : 0);
    if (threadIdx.x < kBins) s.base[threadIdx.x] = base;
    __syncthreads();
#pragma unroll
    for (int i = 0; i < kSortPer; ++i)
      if (digit[i] < kBins) {
        const uint32_t to = s.base[digit[i]] + s.count[threadIdx.x >> 5][digit[i]] + rank[i];
        bk[to] = key[i];
        bp[to] = pos[i];
      }
    __syncthreads();
#pragma unroll
    for (int i = 0; i < kSortPer; ++i) {
      const int t = tile_index(i);
      if (t < T) {
        key[i] = bk[t];
        pos[i] = bp[t];
      }
    }
    __syncthreads();
  }
#pragma unroll
  for (int i = 0; i < kSortPer; ++i) {
    const int t = tile_index(i);
    if (t < T) {
      keys_out[t] = key[i];
      pos_out[t] = pos[i];
    }
  }
  if (status && bad) atomicOr(status, GTK_STATUS_BAD_TOKEN);
}

// Pass `p` of the sort over many tiles, first half: the tile's digit counts. The first pass
// reads the tokens, later ones the keys of the pass before.
template <typename I>
__global__ void __launch_bounds__(kSortThreads)
    count_kernel(const I* __restrict__ tokens, const uint32_t* __restrict__ keys, int64_t T, uint32_t V,
                 int64_t padding, int pass, uint32_t* __restrict__ counts, uint32_t* __restrict__ present,
                 uint32_t* status) {
  wait_previous_kernel();
  __shared__ SortShared s;
  if (pass == 0)
    for (int64_t w = static_cast<int64_t>(blockIdx.x) * kSortThreads + threadIdx.x; w < (V + 31) / 32;
         w += static_cast<int64_t>(gridDim.x) * kSortThreads)
      present[w] = 0;
  bool bad = false;
  uint32_t digit[kSortPer], rank[kSortPer];
#pragma unroll
  for (int i = 0; i < kSortPer; ++i) {
    const int64_t t = static_cast<int64_t>(blockIdx.x) * kTile + tile_index(i);
    uint32_t k = 0;
    if (t < T) k = pass == 0 ? key_of(tokens, t, V, padding, &bad) : keys[t];
    digit[i] = t < T ? (k >> (8 * pass)) & 255u : kBins;
  }
  const uint32_t total = rank_tile(s, digit, rank);
  if (threadIdx.x < kBins) counts[static_cast<int64_t>(blockIdx.x) * kBins + threadIdx.x] = total;
  if (status && bad) atomicOr(status, GTK_STATUS_BAD_TOKEN);
}

// Second half: where the tile's elements go, from all tiles' counts.
template <typename I>
__global__ void __launch_bounds__(kSortThreads)
    scatter_kernel(const I* __restrict__ tokens, const uint32_t* __restrict__ keys, const uint32_t* __restrict__ pos,
                   int64_t T, uint32_t V, int64_t padding, int pass, const uint32_t* __restrict__ counts, int tiles,
                   uint32_t* __restrict__ keys_out, uint32_t* __restrict__ pos_out, uint32_t* __restrict__ present) {
  wait_previous_kernel();
  __shared__ SortShared s;
  __shared__ uint32_t before_part[kSortThreads / kBins][kBins], total_part[kSortThreads / kBins][kBins];
  uint32_t key[kSortPer], p0[kSortPer], digit[kSortPer], rank[kSortPer];
  bool bad = false;
#pragma unroll
  for (int i = 0; i < kSortPer; ++i) {
    const int64_t t = static_cast<int64_t>(blockIdx.x) * kTile + tile_index(i);
    key[i] = 0;
    p0[i] = static_cast<uint32_t>(t);
    if (t < T) {
      if (pass == 0) {
        key[i] = key_of(tokens, t, V, padding, &bad);
        if (key[i] < V) mark(present, key[i]);
      } else {
        key[i] = keys[t];
        p0[i] = pos[t];
      }
    }
    digit[i] = t < T ? (key[i] >> (8 * pass)) & 255u : kBins;
  }
  // thread = (slice of the tiles, bin)
  const int bin = threadIdx.x & (kBins - 1), slice = threadIdx.x / kBins;
  uint32_t before = 0, total = 0;
#pragma unroll 8
  for (int t = slice; t < tiles; t += kSortThreads / kBins) {
    const uint32_t n = counts[static_cast<int64_t>(t) * kBins + bin];
    total += n;
    before += t < static_cast<int>(blockIdx.x) ? n : 0;
  }
  before_part[slice][bin] = before;
  total_part[slice][bin] = total;
  __syncthreads();
  before = total = 0;
  if (threadIdx.x < kBins)
    for (int i = 0; i < kSortThreads / kBins; ++i) {
      before += before_part[i][threadIdx.x];
      total += total_part[i][threadIdx.x];
    }
  const uint32_t base = scan_bins(s, total);
  if (threadIdx.x < kBins) s.base[threadIdx.x] = base + before;
  rank_tile(s, digit, rank);
  __syncthreads();
#pragma unroll
  for (int i = 0; i < kSortPer; ++i)
    if (digit[i] < kBins) {
      const uint32_t to = s.base[digit[i]] + s.count[threadIdx.x >> 5][digit[i]] + rank[i];
      keys_out[to] = key[i];
      pos_out[to] = p0[i];
    }
}

// ---- Sums over the runs of equal tokens -----------------------------------------------------

constexpr int kSumThreads = 256;
constexpr int kBatch = 8;  // dy rows in flight per warp

template <typename W, int V>
__device__ __forceinline__ void write_row(W* dst, const float (&acc)[V], float scale) {
  Vec<W, V> o;
#pragma unroll
  for (int j = 0; j < V; ++j) o.v[j] = Elem<W>::store(acc[j] * scale);
  st_vec<W, V>(dst, o);
}

// Chunk c covers the sorted entries [c L, (c + 1) L); a slab is 32 V columns. Warps
// [0, chunks * slabs) sum, the blocks after them zero the rows of absent tokens, 32 rows and one
// slab per warp.
template <typename T, typename W, int V>
__global__ void __launch_bounds__(kSumThreads)
    run_sums_kernel(const T* __restrict__ dy, const uint32_t* __restrict__ keys, const uint32_t* __restrict__ pos,
                    const uint32_t* __restrict__ present, W* __restrict__ dw, float* __restrict__ partial, int64_t n,
                    uint32_t vocab, int D, int L, int64_t chunks, int slabs, int64_t sum_blocks, float scale) {
  wait_previous_kernel();
  const int lane = threadIdx.x & 31;
  const int64_t warp = (static_cast<int64_t>(blockIdx.x) * kSumThreads + threadIdx.x) >> 5;
  if (blockIdx.x >= sum_blocks) {
    const int64_t item = warp - sum_blocks * (kSumThreads / 32);
    const int64_t word = item / slabs;
    const int col = (static_cast<int>(item % slabs) * 32 + lane) * V;
    if (word >= (static_cast<int64_t>(vocab) + 31) / 32 || col >= D) return;
    const uint32_t bits = present[word];
    const float zero[V] = {};
    for (int r = 0; r < 32; ++r) {
      const int64_t row = word * 32 + r;
      if (row < vocab && !(bits >> r & 1u)) write_row<W, V>(dw + row * D + col, zero, 0.f);
    }
    return;
  }
  if (warp >= chunks * slabs) return;
  const int64_t c = warp / slabs;
  const int col = (static_cast<int>(warp % slabs) * 32 + lane) * V;
  const bool mine = col < D;
  const int64_t i0 = c * L, i1 = i0 + L < n ? i0 + L : n;
  const uint32_t left = i0 > 0 ? keys[i0 - 1] : 0xffffffffu;
  const uint32_t right = i1 < n ? keys[i1] : 0xffffffffu;
  float acc[V];
#pragma unroll
  for (int j = 0; j < V; ++j) acc[j] = 0.f;
  uint32_t cur = keys[i0];
  bool continued = cur == left;  // the current run began in an earlier chunk
  float* head = partial + (c * 2) * static_cast<int64_t>(D) + col;
  for (int64_t b = i0; b < i1; b += 32) {
    const int64_t e = b + lane;
    const uint32_t my_key = e < i1 ? keys[e] : 0xffffffffu;
    const uint32_t my_pos = e < i1 ? pos[e] : 0u;
    const int m = static_cast<int>(i1 - b < 32 ? i1 - b : 32);
    for (int q = 0; q < m; q += kBatch) {
      Vec<T, V> row[kBatch];
#pragma unroll
      for (int u = 0; u < kBatch; ++u) {
        const uint32_t k = __shfl_sync(0xffffffffu, my_key, q + u);
        const uint32_t p = __shfl_sync(0xffffffffu, my_pos, q + u);
        if (mine && k < vocab) row[u] = ld_vec<T, V>(dy + static_cast<int64_t>(p) * D + col);
      }
#pragma unroll
      for (int u = 0; u < kBatch; ++u) {
        if (q + u >= m) break;
        const uint32_t k = __shfl_sync(0xffffffffu, my_key, q + u);
        if (k >= vocab) continue;  // sorted last: nothing follows but more of them
        if (k != cur) {
          if (mine) {
            if (continued)
#pragma unroll
              for (int j = 0; j < V; ++j) head[j] = acc[j];
            else
              write_row<W, V>(dw + static_cast<int64_t>(cur) * D + col, acc, scale);
          }
          cur = k;
          continued = false;
#pragma unroll
          for (int j = 0; j < V; ++j) acc[j] = 0.f;
        }
        if (mine)
#pragma unroll
          for (int j = 0; j < V; ++j) acc[j] += Elem<T>::load(row[u].v[j]);
      }
    }
  }
  if (!mine || cur >= vocab) return;
  const bool goes_on = cur == right;
  if (!goes_on && !continued) {
    write_row<W, V>(dw + static_cast<int64_t>(cur) * D + col, acc, scale);
    return;
  }
  float* to = continued ? head : head + D;
#pragma unroll
  for (int j = 0; j < V; ++j) to[j] = acc[j];
}

// The runs that cross chunks: the block of the chunk in which one begins adds its tail and the
// heads of the chunks after it.
constexpr int kJoinThreads = 512;
constexpr int kJoinCols = 32;

template <typename W>
__global__ void __launch_bounds__(kJoinThreads)
    join_runs_kernel(const uint32_t* __restrict__ keys, const float* __restrict__ partial, W* __restrict__ dw,
                     int64_t n, uint32_t vocab, int D, int L, int64_t chunks, float scale) {
  wait_previous_kernel();
  __shared__ double part[kJoinThreads / 32][kJoinCols];
  const int64_t c = blockIdx.x;
  const int64_t i0 = c * L, i1 = i0 + L;
  if (i1 >= n) return;  // the last chunk starts no run that goes on
  const uint32_t k = keys[i1 - 1];
  if (k >= vocab || keys[i1] != k) return;
  if (i0 > 0 && keys[i0] == k && keys[i0 - 1] == k) return;  // it began earlier
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  for (int c0 = 0; c0 < D; c0 += kJoinCols) {
    const int col = c0 + lane;
    double s = 0.0;
    if (col < D) {
      if (warp == 0) s = partial[(c * 2 + 1) * static_cast<int64_t>(D) + col];
      for (int64_t j = c + 1 + warp; j < chunks && keys[j * L] == k; j += kJoinThreads / 32)
        s += partial[(j * 2) * static_cast<int64_t>(D) + col];
    }
    part[warp][lane] = s;
    __syncthreads();
    if (warp == 0 && col < D) {
      for (int w = 1; w < kJoinThreads / 32; ++w) s += part[w][lane];
      dw[static_cast<int64_t>(k) * D + col] = Elem<W>::store(static_cast<float>(s * scale));
    }
    __syncthreads();
  }
}

// ---- Forward ----------------------------------------------------------------------------------

constexpr int kRowsAtOnce = 4;

// y = scale W[tokens]; rows of nv vectors of V elements. One warp takes kRowsAtOnce rows.
template <typename T, typename I, int V>
__global__ void __launch_bounds__(256)
    lookup_kernel(const I* __restrict__ tokens, const T* __restrict__ w, T* __restrict__ y, int64_t n, int64_t vocab,
                  int D, float scale, uint32_t* status) {
  const int lane = threadIdx.x & 31;
  const int64_t warps = (static_cast<int64_t>(gridDim.x) * blockDim.x) >> 5;
  const int nv = D / V;
  bool bad = false;
  for (int64_t r = ((static_cast<int64_t>(blockIdx.x) * blockDim.x + threadIdx.x) >> 5) * kRowsAtOnce; r < n;
       r += warps * kRowsAtOnce) {
    int64_t tok[kRowsAtOnce];
#pragma unroll
    for (int q = 0; q < kRowsAtOnce; ++q) tok[q] = r + q < n ? static_cast<int64_t>(tokens[r + q]) : 0;
    for (int i = lane; i < nv; i += 32) {
      Vec<T, V> e[kRowsAtOnce];
#pragma unroll
      for (int q = 0; q < kRowsAtOnce; ++q) {
        const bool ok = tok[q] >= 0 && tok[q] < vocab;
        if (ok)
          e[q] = ld_vec<T, V>(w + tok[q] * D + static_cast<int64_t>(i) * V);
        else {
          bad = true;
#pragma unroll
          for (int j = 0; j < V; ++j) e[q].v[j] = Elem<T>::store(0.f);
        }
      }
#pragma unroll
      for (int q = 0; q < kRowsAtOnce; ++q) {
        if (r + q >= n) continue;
        Vec<T, V> o;
#pragma unroll
        for (int j = 0; j < V; ++j) o.v[j] = Elem<T>::store(Elem<T>::load(e[q].v[j]) * scale);
        st_vec<T, V>(y + (r + q) * D + static_cast<int64_t>(i) * V, o);
      }
    }
  }
  if (status && bad) atomicOr(status, GTK_STATUS_BAD_TOKEN);
}

// ---- Host ---------------------------------------------------------------------------------------

int check_sizes(int64_t T, int64_t vocab, int64_t D) {
  if (!dims_ok(T, (int64_t(1) << 31) - 1)) return fail(GTK_ERR_INVALID_ARG, "embedding: tokens must be 1..2^31-1");
  if (!dims_ok(vocab, (int64_t(1) << 31) - 1)) return fail(GTK_ERR_INVALID_ARG, "embedding: vocabulary must be 1..2^31-1");
  if (!dims_ok(D, kMaxWidth)) return fail(GTK_ERR_INVALID_ARG, "embedding: width must be 1..2^20");
  return GTK_OK;
}

int vec_width(int64_t D, size_t bytes, bool aligned) {
  return aligned && (D * bytes) % 16 == 0 ? static_cast<int>(16 / bytes) : 1;
}

// The backward's plan: what the workspace holds and how the sorted list is cut.
struct Plan {
  int passes;        // of 8 bits, for keys 0 .. vocab
  int64_t tiles;
  int64_t L, chunks;
  size_t keys, pos, counts, present, partial, total;  // byte offsets (keys, pos: two buffers each)
};

Plan plan_for(int64_t T, int64_t vocab, int64_t D) {
  Plan p = {};
  p.passes = 1;
  while (p.passes < 4 && (vocab >> (8 * p.passes)) != 0) ++p.passes;
  p.tiles = (T + kTile - 1) / kTile;
  // long enough that about 16 warps per SM have a chunk (of the narrowest slab, 32 columns: the
  // workspace covers every type), at least 32 entries
  const int64_t slabs = (D + 127) / 128;
  int64_t L = (T * slabs + 148 * 16 - 1) / (148 * 16);
  L = (L + 31) / 32 * 32;
  p.L = L < 32 ? 32 : (L > 1024 ? 1024 : L);
  p.chunks = (T + p.L - 1) / p.L;
  size_t at = 0;
  auto take = [&](size_t bytes) {
    const size_t o = at;
    at += round_up(bytes, 256);
    return o;
  };
  p.keys = take(2 * round_up(4 * T, 256));
  p.pos = take(2 * round_up(4 * T, 256));
  p.counts = take(p.tiles > 1 ? 4 * kBins * p.tiles : 0);
  p.present = take((vocab + 31) / 32 * 4);
  p.partial = take(p.chunks > 1 ? static_cast<size_t>(p.chunks) * 2 * D * sizeof(float) : 0);
  p.total = at;
  return p;
}

struct Args {
  const void *tokens, *dy;
  void* dw;
  char* ws;
  int64_t T, vocab, D, padding;
  float scale;
  uint32_t* status;
  cudaStream_t st;
};

template <typename I>
int sort(const Args& a, const Plan& p, const uint32_t** keys, const uint32_t** pos) {
  const size_t half = round_up(4 * a.T, 256);
  uint32_t* k[2] = {reinterpret_cast<uint32_t*>(a.ws + p.keys), reinterpret_cast<uint32_t*>(a.ws + p.keys + half)};
  uint32_t* q[2] = {reinterpret_cast<uint32_t*>(a.ws + p.pos), reinterpret_cast<uint32_t*>(a.ws + p.pos + half)};
  uint32_t* present = reinterpret_cast<uint32_t*>(a.ws + p.present);
  const I* tokens = static_cast<const I*>(a.tokens);
  const uint32_t V = static_cast<uint32_t>(a.vocab);
  if (p.tiles == 1) {
    const int smem = 2 * kTile * 4;
    if (int e = ensure_smem(reinterpret_cast<const void*>(sort_small_kernel<I>), smem)) return e;
    *keys = k[0];
    *pos = q[0];
    return launch("embedding token sort", sort_small_kernel<I>, 1, kSortThreads, smem, a.st, false, tokens,
                  static_cast<int>(a.T), V, a.padding, p.passes, k[0], q[0], present, a.status);
  }
  uint32_t* counts = reinterpret_cast<uint32_t*>(a.ws + p.counts);
  const uint32_t *ki = nullptr, *qi = nullptr;
  for (int pass = 0; pass < p.passes; ++pass) {
    uint32_t *ko = k[pass & 1], *qo = q[pass & 1];
    if (int e = launch("embedding token count", count_kernel<I>, p.tiles, kSortThreads, 0, a.st, pass > 0, tokens, ki,
                       a.T, V, a.padding, pass, counts, present, a.status))
      return e;
    if (int e = launch("embedding token scatter", scatter_kernel<I>, p.tiles, kSortThreads, 0, a.st, true, tokens, ki,
                       qi, a.T, V, a.padding, pass, static_cast<const uint32_t*>(counts), static_cast<int>(p.tiles),
                       ko, qo, present))
      return e;
    ki = ko;
    qi = qo;
  }
  *keys = ki;
  *pos = qi;
  return GTK_OK;
}

template <typename T, typename W, int V>
int sums(const Args& a, const Plan& p, const uint32_t* keys, const uint32_t* pos) {
  const int slabs = static_cast<int>((a.D + 32 * V - 1) / (32 * V));
  constexpr int kPerBlock = kSumThreads / 32;
  const int64_t sum_blocks = (p.chunks * slabs + kPerBlock - 1) / kPerBlock;
  const int64_t zero_blocks = ((a.vocab + 31) / 32 * slabs + kPerBlock - 1) / kPerBlock;
  if (sum_blocks + zero_blocks > (int64_t(1) << 31) - 1)
    return fail(GTK_ERR_UNSUPPORTED, "embedding: vocabulary times width is too large");
  float* partial = reinterpret_cast<float*>(a.ws + p.partial);
  const uint32_t V32 = static_cast<uint32_t>(a.vocab);
  if (int e = launch("embedding run sums", run_sums_kernel<T, W, V>, sum_blocks + zero_blocks, kSumThreads, 0, a.st,
                     true, static_cast<const T*>(a.dy), keys, pos,
                     reinterpret_cast<const uint32_t*>(a.ws + p.present), static_cast<W*>(a.dw), partial, a.T, V32,
                     static_cast<int>(a.D), static_cast<int>(p.L), p.chunks, slabs, sum_blocks, a.scale))
    return e;
  if (p.chunks == 1) return GTK_OK;
  return launch("embedding run join", join_runs_kernel<W>, p.chunks, kJoinThreads, 0, a.st, true, keys,
                static_cast<const float*>(partial), static_cast<W*>(a.dw), a.T, V32, static_cast<int>(a.D),
                static_cast<int>(p.L), p.chunks, a.scale);
}

template <typename T, typename W>
int backward_typed(const Args& a, const Plan& p, const uint32_t* keys, const uint32_t* pos) {
  constexpr int VX = 16 / static_cast<int>(sizeof(T));
  const bool vec = vec_width(a.D, sizeof(T), aligned16(a.dy)) > 1 && a.D * sizeof(W) % 16 == 0 &&
                   reinterpret_cast<uintptr_t>(a.dw) % (sizeof(W) * VX) == 0;
  return vec ? sums<T, W, VX>(a, p, keys, pos) : sums<T, W, 1>(a, p, keys, pos);
}

template <typename T, typename I>
int forward_typed(const Args& a, const void* w, void* y) {
  constexpr int VX = 16 / static_cast<int>(sizeof(T));
  const bool vec = vec_width(a.D, sizeof(T), aligned16(w) && aligned16(y)) > 1;
  auto kernel = vec ? lookup_kernel<T, I, VX> : lookup_kernel<T, I, 1>;
  int64_t blocks = (a.T + kRowsAtOnce * 8 - 1) / (kRowsAtOnce * 8);
  const int64_t cap = static_cast<int64_t>(num_sms()) * 8;
  if (blocks > cap) blocks = cap;
  return launch("embedding lookup", kernel, blocks, 256, 0, a.st, false, static_cast<const I*>(a.tokens),
                static_cast<const T*>(w), static_cast<T*>(y), a.T, a.vocab, static_cast<int>(a.D), a.scale, a.status);
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
                          int64_t vocab, int64_t D, float scale, uint32_t* status, void* stream) {
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
}

size_t gtk_embedding_backward_workspace_bytes(int64_t n_tokens, int64_t vocab, int64_t D) {
  if (!dims_ok(n_tokens) || !dims_ok(vocab) || !dims_ok(D, emb::kMaxWidth)) return 0;
  return emb::plan_for(n_tokens, vocab, D).total;
}

int gtk_embedding_backward(const void* dy, int dy_dtype, const void* tokens, int index_bits, void* dweight,
                           int w_dtype, int64_t n_tokens, int64_t vocab, int64_t D, float scale, int64_t padding,
                           void* workspace, size_t workspace_bytes, uint32_t* status, void* stream) {
  if (int e = emb::check_sizes(n_tokens, vocab, D)) return e;
  if (!dtype_ok(dy_dtype) || !(w_dtype == dy_dtype || w_dtype == GTK_F32))
    return fail(GTK_ERR_UNSUPPORTED, "embedding: dy is fp32, bf16 or fp16, the table's gradient fp32 or dy's type");
  if (padding >= vocab) return fail(GTK_ERR_INVALID_ARG, "embedding: the padding token must be below the vocabulary");
  const emb::Plan p = emb::plan_for(n_tokens, vocab, D);
  if (workspace_bytes < p.total) return fail(GTK_ERR_WORKSPACE, "embedding: workspace too small");
  if (int e = emb::check_tokens(tokens, index_bits)) return e;
  if (int e = check_ptr(dy, "dy", dtype_bytes(dy_dtype))) return e;
  if (int e = check_ptr(dweight, "dweight", dtype_bytes(w_dtype))) return e;
  if (int e = check_ptr(workspace, "workspace", 256)) return e;
  if (int e = check_device()) return e;
  emb::Args a = {};
  a.tokens = tokens, a.dy = dy, a.dw = dweight, a.ws = static_cast<char*>(workspace), a.T = n_tokens;
  a.vocab = vocab, a.D = D, a.padding = padding, a.scale = scale, a.status = status;
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
}

}  // extern "C"
