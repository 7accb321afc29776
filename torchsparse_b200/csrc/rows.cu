// Rows grouped by an index, and the operators made of that: a stable counting sort of row keys, the embedding lookup
// with its gradient summed token by token, and rows sorted by expert and back.
//
// Every sum over the rows of a group runs over the grouped order in fixed pieces, so results do not depend on the
// order in which thread blocks run: there is no floating-point atomic in this file.
#include "rows.cuh"

namespace tsb {
namespace {

// ------------------------------------------------------------------------------------------------ grouping
// A least-significant-digit radix sort of (key, row) with digits of up to 8 bits.  A tile of 4096 keys is ranked by one
// block: warp w owns 256 consecutive keys and counts them 32 at a time with __match_any_sync, so equal keys keep
// their order; a scan over the warps of a tile and one over the tiles of a digit make the ranks global.
constexpr int kSortThreads = 512;
constexpr int kSortWarps = kSortThreads / 32;
constexpr int kSortItems = 8;
constexpr int kSortTile = kSortThreads * kSortItems;
constexpr int kMaxDigits = 256;

struct KeySource {
  const void* keys;      // int32 or int64, `stride` elements apart
  int64_t stride;
  int is64;
  unsigned n_groups;     // a key outside [0, n_groups) becomes n_groups and sorts last
  int64_t skip;          // one more key that counts as outside (-1: none)
};

__device__ __forceinline__ unsigned read_key(const KeySource& s, int64_t i) {
  const int64_t k = s.is64 ? __ldg(reinterpret_cast<const long long*>(s.keys) + i * s.stride)
                           : (int64_t)__ldg(reinterpret_cast<const int*>(s.keys) + i * s.stride);
  return (k < 0 || k >= (int64_t)s.n_groups || k == s.skip) ? s.n_groups : (unsigned)k;
}

// Ranks of the keys of a tile among equal digits of the same warp; whist[w][d] ends as the exclusive sum over the
// warps before w and total[d] as the tile's count.  Item `it` of lane l is key w * 256 + it * 32 + l of the tile.
__device__ __forceinline__ void rank_tile(const unsigned (&digit)[kSortItems], const bool (&on)[kSortItems],
                                          unsigned (&rank)[kSortItems], unsigned short (*whist)[kMaxDigits],
                                          unsigned* total, int n_digits) {
  const int w = threadIdx.x >> 5, lane = threadIdx.x & 31;
  for (int d = lane; d < n_digits; d += 32) whist[w][d] = 0;
  __syncwarp();
#pragma unroll
  for (int it = 0; it < kSortItems; ++it) {
    const unsigned d = on[it] ? digit[it] : (unsigned)kMaxDigits;      // keys beyond the end match only one another
    const unsigned same = __match_any_sync(0xffffffffu, d);
    const unsigned before = on[it] ? whist[w][d] : 0u;
    rank[it] = before + __popc(same & ((1u << lane) - 1));
    __syncwarp();
    if (on[it] && lane == __ffs(same) - 1) whist[w][d] = (unsigned short)(before + __popc(same));
    __syncwarp();
  }
  __syncthreads();
  for (int d = threadIdx.x; d < n_digits; d += kSortThreads) {
    unsigned sum = 0;
    for (int i = 0; i < kSortWarps; ++i) {
      const unsigned v = whist[i][d];
      whist[i][d] = (unsigned short)sum;
      sum += v;
    }
    total[d] = sum;
  }
  __syncthreads();
}

// in place: total[0..n_digits) -> exclusive sums, by the first warp
__device__ __forceinline__ void scan_digits(unsigned* total, int n_digits) {
  if (threadIdx.x < 32) {
    unsigned carry = 0;
    for (int d0 = 0; d0 < n_digits; d0 += 32) {
      const int d = d0 + threadIdx.x;
      const unsigned v = d < n_digits ? total[d] : 0u;
      unsigned inc = v;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const unsigned up = __shfl_up_sync(0xffffffffu, inc, o);
        if ((int)threadIdx.x >= o) inc += up;
      }
      if (d < n_digits) total[d] = carry + inc - v;
      carry += __shfl_sync(0xffffffffu, inc, 31);
    }
  }
  __syncthreads();
}

struct SortOut {
  int* order;        // [n] row at a sorted position
  int* inverse;      // [n] sorted position of a row, or null
  unsigned* keys;    // [n] key at a sorted position, or null
};

// n <= kSortTile: every pass in one block, through shared memory
__global__ void __launch_bounds__(kSortThreads) sort_one_tile_kernel(KeySource src, int n, int passes, int bits, SortOut out,
                                                                     int* __restrict__ offsets) {
  __shared__ unsigned short whist[kSortWarps][kMaxDigits];
  __shared__ unsigned total[kMaxDigits];
  __shared__ unsigned skey[kSortTile];
  __shared__ unsigned short srow[kSortTile];
  const int w = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int base = w * 32 * kSortItems + lane;
  unsigned key[kSortItems], row[kSortItems], digit[kSortItems], rank[kSortItems];
  bool on[kSortItems];
#pragma unroll
  for (int it = 0; it < kSortItems; ++it) {
    row[it] = (unsigned)(base + it * 32);
    on[it] = (int)row[it] < n;
    key[it] = on[it] ? read_key(src, row[it]) : 0u;
  }
  for (int p = 0; p < passes; ++p) {
#pragma unroll
    for (int it = 0; it < kSortItems; ++it) digit[it] = (key[it] >> (p * bits)) & ((1u << bits) - 1);
    rank_tile(digit, on, rank, whist, total, 1 << bits);
    scan_digits(total, 1 << bits);
#pragma unroll
    for (int it = 0; it < kSortItems; ++it) {
      if (!on[it]) continue;
      const unsigned pos = total[digit[it]] + whist[w][digit[it]] + rank[it];
      skey[pos] = key[it];
      srow[pos] = (unsigned short)row[it];
    }
    __syncthreads();
#pragma unroll
    for (int it = 0; it < kSortItems; ++it) {
      if (!on[it]) continue;
      key[it] = skey[base + it * 32];
      row[it] = srow[base + it * 32];
    }
    __syncthreads();
  }
#pragma unroll
  for (int it = 0; it < kSortItems; ++it) {
    if (!on[it]) continue;
    const int pos = base + it * 32;
    out.order[pos] = (int)row[it];
    if (out.inverse) out.inverse[row[it]] = pos;
    if (out.keys) out.keys[pos] = key[it];
  }
  if (offsets) {       // first position whose key is not below the group
    for (unsigned g = threadIdx.x; g <= src.n_groups; g += kSortThreads) {
      int lo = 0, hi = n;
      while (lo < hi) {
        const int mid = (lo + hi) >> 1;
        if (skey[mid] < g) lo = mid + 1; else hi = mid;
      }
      offsets[g] = lo;
    }
  }
}

// keys and rows of one pass: the caller's keys in the first, the previous pass's pairs afterwards
struct PassIn {
  KeySource src;
  const unsigned* keys;      // null: the first pass
  const int* rows;
};

__device__ __forceinline__ void load_tile(const PassIn& in, int64_t n, unsigned (&key)[kSortItems], bool (&on)[kSortItems],
                                          int64_t first) {
#pragma unroll
  for (int it = 0; it < kSortItems; ++it) {
    const int64_t i = first + it * 32;
    on[it] = i < n;
    key[it] = on[it] ? (in.keys ? __ldg(in.keys + i) : read_key(in.src, i)) : 0u;
  }
}

__global__ void __launch_bounds__(kSortThreads) sort_count_kernel(PassIn in, int64_t n, int shift, int bits, int64_t tiles,
                                                                  unsigned* __restrict__ counts) {
  __shared__ unsigned short whist[kSortWarps][kMaxDigits];
  __shared__ unsigned total[kMaxDigits];
  const int64_t first = (int64_t)blockIdx.x * kSortTile + (threadIdx.x >> 5) * 32 * kSortItems + (threadIdx.x & 31);
  unsigned key[kSortItems], digit[kSortItems], rank[kSortItems];
  bool on[kSortItems];
  load_tile(in, n, key, on, first);
#pragma unroll
  for (int it = 0; it < kSortItems; ++it) digit[it] = (key[it] >> shift) & ((1u << bits) - 1);
  rank_tile(digit, on, rank, whist, total, 1 << bits);
  for (int d = threadIdx.x; d < (1 << bits); d += kSortThreads) counts[d * tiles + blockIdx.x] = total[d];
}

// one block per digit: exclusive sums over the tiles in place, the digit's count behind them
__global__ void __launch_bounds__(256) sort_scan_kernel(unsigned* __restrict__ counts, int64_t tiles, int n_digits) {
  __shared__ unsigned wsum[8];
  unsigned* row = counts + (int64_t)blockIdx.x * tiles;
  unsigned carry = 0;
  const int lane = threadIdx.x & 31, w = threadIdx.x >> 5;
  for (int64_t t0 = 0; t0 < tiles; t0 += 256) {
    const int64_t t = t0 + threadIdx.x;
    const unsigned v = t < tiles ? row[t] : 0u;
    unsigned inc = v;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const unsigned up = __shfl_up_sync(0xffffffffu, inc, o);
      if (lane >= o) inc += up;
    }
    if (lane == 31) wsum[w] = inc;
    __syncthreads();
    unsigned before = carry, all = 0;
    for (int i = 0; i < 8; ++i) {
      if (i < w) before += wsum[i];
      all += wsum[i];
    }
    if (t < tiles) row[t] = before + inc - v;
    carry += all;
    __syncthreads();
  }
  if (threadIdx.x == 0) counts[(int64_t)n_digits * tiles + blockIdx.x] = carry;
}

__global__ void __launch_bounds__(kSortThreads) sort_scatter_kernel(PassIn in, int64_t n, int shift, int bits, int64_t tiles,
                                                                    const unsigned* __restrict__ counts, SortOut out) {
  __shared__ unsigned short whist[kSortWarps][kMaxDigits];
  __shared__ unsigned total[kMaxDigits];
  __shared__ unsigned start[kMaxDigits];
  const int w = threadIdx.x >> 5;
  const int64_t first = (int64_t)blockIdx.x * kSortTile + w * 32 * kSortItems + (threadIdx.x & 31);
  unsigned key[kSortItems], digit[kSortItems], rank[kSortItems];
  bool on[kSortItems];
  load_tile(in, n, key, on, first);
  for (int d = threadIdx.x; d < (1 << bits); d += kSortThreads) start[d] = counts[(int64_t)(1 << bits) * tiles + d];
#pragma unroll
  for (int it = 0; it < kSortItems; ++it) digit[it] = (key[it] >> shift) & ((1u << bits) - 1);
  rank_tile(digit, on, rank, whist, total, 1 << bits);      // its barriers also publish start[]
  scan_digits(start, 1 << bits);
#pragma unroll
  for (int it = 0; it < kSortItems; ++it) {
    if (!on[it]) continue;
    const unsigned d = digit[it];
    const int64_t pos = (int64_t)start[d] + counts[d * tiles + blockIdx.x] + whist[w][d] + rank[it];
    const int64_t i = first + it * 32;
    const int row = in.keys ? __ldg(in.rows + i) : (int)i;
    out.order[pos] = row;
    if (out.keys) out.keys[pos] = key[it];
    if (out.inverse) out.inverse[row] = (int)pos;
  }
}

__device__ __forceinline__ int64_t lower_bound(const unsigned* __restrict__ keys, int64_t n, unsigned g) {
  int64_t lo = 0, hi = n;
  while (lo < hi) {
    const int64_t mid = (lo + hi) >> 1;
    if (__ldg(keys + mid) < g) lo = mid + 1; else hi = mid;
  }
  return lo;
}

__global__ void group_offsets_kernel(const unsigned* __restrict__ keys, int64_t n, int64_t n_groups, int* __restrict__ offsets) {
  for (int64_t g = blockIdx.x * (int64_t)blockDim.x + threadIdx.x; g <= n_groups; g += (int64_t)gridDim.x * blockDim.x)
    offsets[g] = (int)lower_bound(keys, n, (unsigned)g);
}

struct SortPlan {
  int passes, bits;
  int64_t tiles;
  size_t counts, pairs, bytes;      // sizes of the parts of the workspace
};

SortPlan sort_plan(int64_t n, int64_t n_groups) {
  SortPlan p;
  int total = 1;
  while ((n_groups >> total) != 0) ++total;
  p.passes = (total + 7) / 8;
  p.bits = (total + p.passes - 1) / p.passes;
  p.tiles = cdiv(n, kSortTile);
  p.counts = align_up(((size_t)(p.tiles + 1) << p.bits) * sizeof(unsigned), 256);
  p.pairs = align_up((size_t)n * 4, 256);
  p.bytes = n <= kSortTile ? 256 : p.counts + 5 * p.pairs;      // two sets of (key, row), the sorted keys
  return p;
}

// order / inverse / keys / offsets of n keys; `sorted` (never null) receives the sorted keys when n > one tile
int run_sort(const KeySource& src, int64_t n, SortOut out, int* offsets, void* workspace, cudaStream_t st) {
  const SortPlan p = sort_plan(n, src.n_groups);
  if (n <= kSortTile) {
    sort_one_tile_kernel<<<1, kSortThreads, 0, st>>>(src, (int)n, p.passes, p.bits, out, offsets);
    TSB_LAUNCH_CHECK();
    return TSB_OK;
  }
  char* ws = static_cast<char*>(workspace);
  unsigned* counts = reinterpret_cast<unsigned*>(ws);
  unsigned* keys[2];
  int* rows[2];
  for (int i = 0; i < 2; ++i) {
    keys[i] = reinterpret_cast<unsigned*>(ws + p.counts + 2 * i * p.pairs);
    rows[i] = reinterpret_cast<int*>(ws + p.counts + (2 * i + 1) * p.pairs);
  }
  unsigned* last = out.keys ? out.keys : reinterpret_cast<unsigned*>(ws + p.counts + 4 * p.pairs);
  PassIn in{src, nullptr, nullptr};
  for (int i = 0; i < p.passes; ++i) {
    const bool end = i + 1 == p.passes;
    const SortOut to = end ? SortOut{out.order, out.inverse, last} : SortOut{rows[i & 1], nullptr, keys[i & 1]};
    sort_count_kernel<<<(unsigned)p.tiles, kSortThreads, 0, st>>>(in, n, i * p.bits, p.bits, p.tiles, counts);
    TSB_LAUNCH_CHECK();
    sort_scan_kernel<<<1 << p.bits, 256, 0, st>>>(counts, p.tiles, 1 << p.bits);
    TSB_LAUNCH_CHECK();
    sort_scatter_kernel<<<(unsigned)p.tiles, kSortThreads, 0, st>>>(in, n, i * p.bits, p.bits, p.tiles, counts, to);
    TSB_LAUNCH_CHECK();
    in.keys = to.keys;
    in.rows = to.order;
  }
  if (offsets) {
    group_offsets_kernel<<<grid_for((int64_t)src.n_groups + 1, 256), 256, 0, st>>>(last, n, src.n_groups, offsets);
    TSB_LAUNCH_CHECK();
  }
  return TSB_OK;
}

// ------------------------------------------------------------------------------------------------ embedding
// y[i] = scale * table[token[i]], zeros where the token is no row of the table: one vector of a row per thread.
template <typename T, int VEC>
__global__ void __launch_bounds__(256) embed_kernel(const T* __restrict__ table, KeySource src, int64_t n, int64_t c, float scale,
                                                    T* __restrict__ out) {
  const int64_t cols = c / VEC, total = n * cols;
  for (int64_t t = blockIdx.x * (int64_t)blockDim.x + threadIdx.x; t < total; t += (int64_t)gridDim.x * blockDim.x) {
    const int64_t i = t / cols, j = (t - i * cols) * VEC;
    const unsigned row = read_key(src, i);
    Pack<T, VEC> p;
    if (row < src.n_groups) {
      p.load(table + (int64_t)row * c + j);
      float v[VEC];
      p.get(v);
#pragma unroll
      for (int e = 0; e < VEC; ++e) v[e] *= scale;
      p.set(v);
    } else {
      p.clear();
    }
    p.store(out + i * c + j);
  }
}

// The gradient of the table: dtable[v] = scale * sum of grad[i] over the rows i whose token is v.
//
// The rows are walked in sorted order by workers of `cols` threads (one thread per vector of a row), each over `len`
// positions.  A token whose positions lie inside one worker is summed and written there; one that crosses workers
// leaves a 32-bit partial sum per worker, `tail` where it begins and `head` where it goes on, which embed_join_kernel
// adds up in order.  The blocks behind the workers write the zeros of the tokens that do not occur.
struct EmbedGrad {
  const unsigned* keys;      // sorted; n_rows marks rows without a token
  const int* order;
  int64_t n, n_rows, c;
  int len;                   // positions of a worker
  int64_t workers;
  int cols, per_block;       // threads of a worker, workers of a block
  float scale;
  float* head;               // [workers, c]
  float* tail;
};

template <typename T, int VEC>
__global__ void __launch_bounds__(256) embed_grad_kernel(EmbedGrad a, const T* __restrict__ grad, T* __restrict__ dtable,
                                                         int64_t worker_blocks, int zero_rows) {
  if (blockIdx.x >= worker_blocks) {
    __shared__ unsigned char absent[256];
    const int64_t v0 = (blockIdx.x - worker_blocks) * (int64_t)zero_rows;
    if ((int)threadIdx.x < zero_rows) {
      const int64_t v = v0 + threadIdx.x;
      bool none = false;
      if (v < a.n_rows) {
        const int64_t at = lower_bound(a.keys, a.n, (unsigned)v);
        none = at >= a.n || __ldg(a.keys + at) != (unsigned)v;
      }
      absent[threadIdx.x] = none;
    }
    __syncthreads();
    const int cols = (int)(a.c / VEC);
    Pack<T, VEC> zero;
    zero.clear();
    for (int t = threadIdx.x; t < zero_rows * cols; t += blockDim.x) {
      const int r = t / cols;
      if (absent[r]) zero.store(dtable + (v0 + r) * a.c + (int64_t)(t - r * cols) * VEC);
    }
    return;
  }
  const int slot = threadIdx.x / a.cols;
  const int64_t w = blockIdx.x * (int64_t)a.per_block + slot;
  if (slot >= a.per_block || w >= a.workers) return;
  const int64_t p0 = w * a.len, p1 = min(p0 + a.len, a.n);
  const unsigned none = (unsigned)a.n_rows;
  for (int64_t j = (int64_t)(threadIdx.x - slot * a.cols) * VEC; j < a.c; j += (int64_t)a.cols * VEC) {
    float acc[VEC];
#pragma unroll
    for (int e = 0; e < VEC; ++e) acc[e] = 0.f;
    unsigned cur = __ldg(a.keys + p0);
    bool goes_on = p0 > 0 && __ldg(a.keys + p0 - 1) == cur;      // the run began in an earlier worker
    for (int64_t p = p0; p < p1 && cur != none;) {
      constexpr int U = 4;
      Pack<T, VEC> v[U];
      unsigned key[U];
#pragma unroll
      for (int u = 0; u < U; ++u) {
        key[u] = p + u < p1 ? __ldg(a.keys + p + u) : none;
        if (key[u] != none) v[u].load(grad + (int64_t)__ldg(a.order + p + u) * a.c + j);
      }
#pragma unroll
      for (int u = 0; u < U; ++u) {
        if (p + u >= p1 || cur == none) continue;
        if (key[u] != cur) {      // the run of `cur` ended inside this worker
          if (goes_on) {
#pragma unroll
            for (int e = 0; e < VEC; ++e) a.head[w * a.c + j + e] = acc[e];
          } else {
            Pack<T, VEC> o;
#pragma unroll
            for (int e = 0; e < VEC; ++e) acc[e] *= a.scale;
            o.set(acc);
            o.store(dtable + (int64_t)cur * a.c + j);
          }
#pragma unroll
          for (int e = 0; e < VEC; ++e) acc[e] = 0.f;
          cur = key[u];
          goes_on = false;
          if (cur == none) continue;
        }
        float g[VEC];
        v[u].get(g);
#pragma unroll
        for (int e = 0; e < VEC; ++e) acc[e] += g[e];
      }
      p += U;
    }
    if (cur == none) continue;
    const bool on = p1 < a.n && __ldg(a.keys + p1) == cur;      // the run goes on in the next worker
    if (goes_on || on) {
      float* to = goes_on ? a.head : a.tail;
#pragma unroll
      for (int e = 0; e < VEC; ++e) to[w * a.c + j + e] = acc[e];
    } else {
      Pack<T, VEC> o;
#pragma unroll
      for (int e = 0; e < VEC; ++e) acc[e] *= a.scale;
      o.set(acc);
      o.store(dtable + (int64_t)cur * a.c + j);
    }
  }
}

// One block per worker in which a run begins that goes on: tail + the heads of the workers that follow.
template <typename T>
__global__ void __launch_bounds__(256) embed_join_kernel(EmbedGrad a, T* __restrict__ dtable) {
  __shared__ float part[256];
  for (int64_t w = blockIdx.x; w < a.workers; w += gridDim.x) {
    const int64_t p0 = w * a.len, p1 = p0 + a.len;
    if (p1 >= a.n) continue;
    const unsigned key = __ldg(a.keys + p1 - 1);
    if (key == (unsigned)a.n_rows || __ldg(a.keys + p1) != key) continue;
    if (__ldg(a.keys + p0) == key && p0 > 0 && __ldg(a.keys + p0 - 1) == key) continue;      // it began before
    const int64_t last = (lower_bound(a.keys, a.n, key + 1) - 1) / a.len;      // the worker in which it ends
    // 256 threads = columns x slices of the workers w + 1 .. last
    const int cols = a.c < 256 ? (int)a.c : 256, slices = 256 / cols;
    const int slice = threadIdx.x / cols;
    for (int64_t j0 = 0; j0 < a.c; j0 += cols) {
      const int64_t j = j0 + (threadIdx.x - slice * cols);
      float s = 0.f;
      if (slice < slices && j < a.c) {
#pragma unroll 4
        for (int64_t k = w + 1 + slice; k <= last; k += slices) s += a.head[k * a.c + j];
      }
      part[threadIdx.x] = s;
      __syncthreads();
      if (slice == 0 && j < a.c) {
        float all = a.tail[w * a.c + j];
        for (int i = 0; i < slices; ++i) all += part[i * cols + threadIdx.x];
        dtable[(int64_t)key * a.c + j] = from_f32<T>(all * a.scale);
      }
      __syncthreads();
    }
  }
}

EmbedGrad embed_plan(int64_t n, int64_t n_rows, int64_t c, int dtype, int vec) {
  EmbedGrad a{};
  a.n = n;
  a.n_rows = n_rows;
  a.c = c;
  const int64_t vecs = c / vec;
  a.cols = (int)(vecs < 256 ? vecs : 256);
  a.per_block = 256 / a.cols;
  int64_t len = cdiv(n * a.cols, (int64_t)kSmCount * 2048);
  len = len < 8 ? 8 : len > 64 ? 64 : len;
  a.len = (int)len;
  a.workers = cdiv(n, len);
  return a;
}

// ------------------------------------------------------------------------------------------------ experts
// Position p of the sorted rows belongs to choice order[p] of the n * k choices; positions at and behind offsets[E]
// belong to choices of no expert.

// xs[inverse[i][j]] = x[i], zeros behind the kept rows: one vector of a (row, choice) per thread, so the k reads of a
// row meet in the L1 cache.
template <typename T, int VEC>
__global__ void __launch_bounds__(256) dispatch_kernel(const T* __restrict__ x, const int* __restrict__ inverse,
                                                       const int* __restrict__ kept, int64_t pairs, int k, int64_t c,
                                                       T* __restrict__ xs) {
  const int64_t cols = c / VEC, total = pairs * cols, n_kept = __ldg(kept);
  for (int64_t t = blockIdx.x * (int64_t)blockDim.x + threadIdx.x; t < total; t += (int64_t)gridDim.x * blockDim.x) {
    const int64_t q = t / cols, j = (t - q * cols) * VEC;
    const int64_t pos = __ldg(inverse + q);
    if (pos < 0 || pos >= pairs) continue;
    Pack<T, VEC> p;
    if (pos < n_kept) p.load(x + q / k * c + j); else p.clear();
    p.store(xs + pos * c + j);
  }
}

// out[i] = sum over j of w[i][j] * rows[inverse[i][j]] (w null: 1), in the order of j
template <typename T, int VEC>
__global__ void __launch_bounds__(256) combine_kernel(const T* __restrict__ rows, const void* __restrict__ w, int w_dtype,
                                                      const int* __restrict__ inverse, const int* __restrict__ kept, int64_t n,
                                                      int k, int64_t c, T* __restrict__ out) {
  const int64_t cols = c / VEC, total = n * cols, pairs = n * k;
  const int64_t n_kept = min((int64_t)__ldg(kept), pairs);
  for (int64_t t = blockIdx.x * (int64_t)blockDim.x + threadIdx.x; t < total; t += (int64_t)gridDim.x * blockDim.x) {
    const int64_t i = t / cols, j = (t - i * cols) * VEC;
    float acc[VEC];
#pragma unroll
    for (int e = 0; e < VEC; ++e) acc[e] = 0.f;
#pragma unroll 4
    for (int q = 0; q < k; ++q) {
      const int64_t pos = __ldg(inverse + i * k + q);
      if (pos < 0 || pos >= n_kept) continue;
      Pack<T, VEC> p;
      p.load(rows + pos * c + j);
      const float f = w ? load_any(w, w_dtype, i * k + q) : 1.f;
      float v[VEC];
      p.get(v);
#pragma unroll
      for (int e = 0; e < VEC; ++e) acc[e] = fmaf(f, v[e], acc[e]);
    }
    Pack<T, VEC> o;
    o.set(acc);
    o.store(out + i * c + j);
  }
}

// One warp per choice: drows[pos] = w * dout[i] and dw = <dout[i], rows[pos]>, both zero for a choice of no expert.
template <typename T, int VEC>
__global__ void __launch_bounds__(256) combine_grad_kernel(const T* __restrict__ dout, const T* __restrict__ rows,
                                                           const void* __restrict__ w, int w_dtype,
                                                           const int* __restrict__ inverse, const int* __restrict__ kept,
                                                           int64_t n, int k, int64_t c, T* __restrict__ drows,
                                                           void* __restrict__ dw) {
  const int64_t pairs = n * k, cols = c / VEC;
  const int64_t n_kept = __ldg(kept);
  const int lane = threadIdx.x & 31;
  for (int64_t q = (blockIdx.x * (int64_t)blockDim.x + threadIdx.x) >> 5; q < pairs; q += ((int64_t)gridDim.x * blockDim.x) >> 5) {
    const int64_t pos = __ldg(inverse + q), i = q / k;
    const bool there = pos >= 0 && pos < pairs, used = there && pos < n_kept;
    const float f = used ? load_any(w, w_dtype, q) : 0.f;
    float dot = 0.f;
    for (int64_t v = lane; v < cols; v += 32) {
      Pack<T, VEC> g, r;
      if (used) {
        g.load(dout + i * c + v * VEC);
        r.load(rows + pos * c + v * VEC);
        float a[VEC], b[VEC];
        g.get(a);
        r.get(b);
#pragma unroll
        for (int e = 0; e < VEC; ++e) {
          dot = fmaf(a[e], b[e], dot);
          a[e] *= f;
        }
        g.set(a);
      } else {
        g.clear();
      }
      if (there) g.store(drows + pos * c + v * VEC);
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) dot += __shfl_down_sync(0xffffffffu, dot, o);
    if (lane == 0) store_any(dw, w_dtype, q, dot);
  }
}

bool good_dtype(int dtype) { return dtype == TSB_F32 || dtype == TSB_F16 || dtype == TSB_BF16; }
constexpr int64_t kMaxRows = 0x7fffffff;      // positions and rows are 32-bit integers

}  // namespace
}  // namespace tsb

using namespace tsb;

extern "C" {

size_t tsb_group_rows_workspace_bytes(int64_t n, int64_t n_groups) {
  if (n < 0 || n_groups < 1 || n > kMaxRows || n_groups > kMaxRows) return 0;
  return sort_plan(n, n_groups).bytes;
}

int tsb_group_rows(const void* keys, int32_t keys_are_i64, int64_t stride, int64_t n, int64_t n_groups, int32_t* order,
                   int32_t* inverse, int32_t* offsets, void* workspace, size_t workspace_bytes, tsb_stream_t stream) {
  if (n < 0 || n_groups < 1 || stride < 0 || (n && (!keys || !order)) || !offsets) return TSB_ERR_BAD_ARG;
  if (n > kMaxRows || n_groups > kMaxRows) return TSB_ERR_LIMIT;
  cudaStream_t st = as_stream(stream);
  if (n == 0) {
    TSB_CUDA_TRY(cudaMemsetAsync(offsets, 0, (size_t)(n_groups + 1) * sizeof(int32_t), st));
    return TSB_OK;
  }
  if (!workspace || workspace_bytes < sort_plan(n, n_groups).bytes) return TSB_ERR_WORKSPACE;
  const KeySource src{keys, stride, keys_are_i64, (unsigned)n_groups, -1};
  return run_sort(src, n, SortOut{order, inverse, nullptr}, offsets, workspace, st);
}

int tsb_embedding_fwd(const void* table, const void* tokens, int32_t tokens_are_i64, int64_t n, int64_t n_rows, int64_t c,
                      float scale, int32_t dtype, void* out, tsb_stream_t stream) {
  if (n < 0 || n_rows < 0 || c < 1 || (n && (!tokens || !out)) || (n && n_rows && !table)) return TSB_ERR_BAD_ARG;
  if (!good_dtype(dtype)) return TSB_ERR_UNSUPPORTED;
  if (n_rows > kMaxRows) return TSB_ERR_LIMIT;
  if (n == 0) return TSB_OK;
  const KeySource src{tokens, 1, tokens_are_i64, (unsigned)n_rows, -1};
  const int vec = vector_width(dtype, c, (uintptr_t)table | (uintptr_t)out);
  return dispatch_pack(dtype, vec, [&](auto tag) -> int {
    using T = typename decltype(tag)::T;
    constexpr int VEC = decltype(tag)::VEC;
    embed_kernel<T, VEC><<<grid_for(n * (c / VEC), 256, 32), 256, 0, as_stream(stream)>>>((const T*)table, src, n, c, scale, (T*)out);
    TSB_LAUNCH_CHECK();
    return TSB_OK;
  });
}

size_t tsb_embedding_bwd_workspace_bytes(int64_t n, int64_t n_rows, int64_t c, int32_t dtype) {
  if (n < 1 || n_rows < 1 || c < 1 || n > kMaxRows || n_rows > kMaxRows || !good_dtype(dtype)) return 256;
  // the widest vector has the fewest threads per worker and with them the shortest, most numerous workers
  size_t partials = 0;
  for (int vec = 1; vec <= 16 / (int)dtype_size(dtype); vec *= 2) {
    if (c % vec) continue;
    const size_t b = align_up((size_t)embed_plan(n, n_rows, c, dtype, vec).workers * c * sizeof(float), 256);
    if (b > partials) partials = b;
  }
  return align_up(sort_plan(n, n_rows).bytes, 256) + 2 * align_up((size_t)n * 4, 256) + 2 * partials;
}

int tsb_embedding_bwd(const void* grad, const void* tokens, int32_t tokens_are_i64, int64_t n, int64_t n_rows, int64_t c,
                      float scale, int64_t padding_row, int32_t dtype, void* dtable, void* workspace, size_t workspace_bytes,
                      tsb_stream_t stream) {
  if (n < 0 || n_rows < 0 || c < 1 || (n && (!tokens || !grad)) || (n_rows && !dtable)) return TSB_ERR_BAD_ARG;
  if (!good_dtype(dtype)) return TSB_ERR_UNSUPPORTED;
  if (n > kMaxRows || n_rows > kMaxRows) return TSB_ERR_LIMIT;
  cudaStream_t st = as_stream(stream);
  if (n_rows == 0) return TSB_OK;
  if (n == 0) {
    TSB_CUDA_TRY(cudaMemsetAsync(dtable, 0, (size_t)n_rows * c * dtype_size(dtype), st));
    return TSB_OK;
  }
  if (!workspace || workspace_bytes < tsb_embedding_bwd_workspace_bytes(n, n_rows, c, dtype)) return TSB_ERR_WORKSPACE;
  const int vec = vector_width(dtype, c, (uintptr_t)grad | (uintptr_t)dtable);
  EmbedGrad a = embed_plan(n, n_rows, c, dtype, vec);
  a.scale = scale;
  char* ws = static_cast<char*>(workspace) + align_up(sort_plan(n, n_rows).bytes, 256);
  unsigned* keys = reinterpret_cast<unsigned*>(ws);
  ws += align_up((size_t)n * 4, 256);
  int* order = reinterpret_cast<int*>(ws);
  ws += align_up((size_t)n * 4, 256);
  const size_t partials = align_up((size_t)a.workers * c * sizeof(float), 256);
  a.keys = keys;
  a.order = order;
  a.head = reinterpret_cast<float*>(ws);
  a.tail = reinterpret_cast<float*>(ws + partials);
  const KeySource src{tokens, 1, tokens_are_i64, (unsigned)n_rows, padding_row};
  const int rc = run_sort(src, n, SortOut{order, nullptr, keys}, nullptr, workspace, st);
  if (rc != TSB_OK) return rc;
  return dispatch_pack(dtype, vec, [&](auto tag) -> int {
    using T = typename decltype(tag)::T;
    constexpr int VEC = decltype(tag)::VEC;
    const int64_t worker_blocks = cdiv(a.workers, a.per_block);
    const int zero_rows = c >= 256 ? 16 : 256;      // rows that a block looks up and clears
    const int64_t blocks = worker_blocks + cdiv(n_rows, zero_rows);
    if (blocks > 0x7fffffff) return TSB_ERR_LIMIT;
    embed_grad_kernel<T, VEC><<<(unsigned)blocks, 256, 0, st>>>(a, (const T*)grad, (T*)dtable, worker_blocks, zero_rows);
    TSB_LAUNCH_CHECK();
    if (a.workers > 1) {
      embed_join_kernel<T><<<grid_for(a.workers, 1, 8), 256, 0, st>>>(a, (T*)dtable);
      TSB_LAUNCH_CHECK();
    }
    return TSB_OK;
  });
}

int tsb_expert_dispatch(const void* x, const int32_t* inverse, const int32_t* kept, int64_t n, int32_t k, int64_t c,
                        int32_t dtype, void* xs, tsb_stream_t stream) {
  if (n < 0 || k < 1 || c < 1 || (n && (!x || !inverse || !kept || !xs))) return TSB_ERR_BAD_ARG;
  if (!good_dtype(dtype)) return TSB_ERR_UNSUPPORTED;
  if (n > kMaxRows / k) return TSB_ERR_LIMIT;
  if (n == 0) return TSB_OK;
  const int vec = vector_width(dtype, c, (uintptr_t)x | (uintptr_t)xs);
  return dispatch_pack(dtype, vec, [&](auto tag) -> int {
    using T = typename decltype(tag)::T;
    constexpr int VEC = decltype(tag)::VEC;
    dispatch_kernel<T, VEC><<<grid_for(n * k * (c / VEC), 256, 32), 256, 0, as_stream(stream)>>>((const T*)x, inverse, kept, n * k, k,
                                                                                                c, (T*)xs);
    TSB_LAUNCH_CHECK();
    return TSB_OK;
  });
}

int tsb_expert_combine(const void* rows, const void* weights, int32_t weights_dtype, const int32_t* inverse, const int32_t* kept,
                       int64_t n, int32_t k, int64_t c, int32_t dtype, void* out, tsb_stream_t stream) {
  if (n < 0 || k < 1 || c < 1 || (n && (!rows || !inverse || !kept || !out))) return TSB_ERR_BAD_ARG;
  if (!good_dtype(dtype) || (weights && !good_dtype(weights_dtype))) return TSB_ERR_UNSUPPORTED;
  if (n > kMaxRows / k) return TSB_ERR_LIMIT;
  if (n == 0) return TSB_OK;
  const int vec = vector_width(dtype, c, (uintptr_t)rows | (uintptr_t)out);
  return dispatch_pack(dtype, vec, [&](auto tag) -> int {
    using T = typename decltype(tag)::T;
    constexpr int VEC = decltype(tag)::VEC;
    combine_kernel<T, VEC><<<grid_for(n * (c / VEC), 256, 32), 256, 0, as_stream(stream)>>>((const T*)rows, weights, weights_dtype,
                                                                                          inverse, kept, n, k, c, (T*)out);
    TSB_LAUNCH_CHECK();
    return TSB_OK;
  });
}

int tsb_expert_combine_bwd(const void* dout, const void* rows, const void* weights, int32_t weights_dtype,
                           const int32_t* inverse, const int32_t* kept, int64_t n, int32_t k, int64_t c, int32_t dtype,
                           void* drows, void* dweights, tsb_stream_t stream) {
  if (n < 0 || k < 1 || c < 1 || (n && (!dout || !rows || !weights || !inverse || !kept || !drows || !dweights)))
    return TSB_ERR_BAD_ARG;
  if (!good_dtype(dtype) || !good_dtype(weights_dtype)) return TSB_ERR_UNSUPPORTED;
  if (n > kMaxRows / k) return TSB_ERR_LIMIT;
  if (n == 0) return TSB_OK;
  const int vec = vector_width(dtype, c, (uintptr_t)dout | (uintptr_t)rows | (uintptr_t)drows);
  return dispatch_pack(dtype, vec, [&](auto tag) -> int {
    using T = typename decltype(tag)::T;
    constexpr int VEC = decltype(tag)::VEC;
    combine_grad_kernel<T, VEC><<<grid_for(n * k * 32, 256, 32), 256, 0, as_stream(stream)>>>(
        (const T*)dout, (const T*)rows, weights, weights_dtype, inverse, kept, n, k, c, (T*)drows, dweights);
    TSB_LAUNCH_CHECK();
    return TSB_OK;
  });
}

}  // extern "C"
