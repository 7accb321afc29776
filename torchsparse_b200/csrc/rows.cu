// Rows grouped by an index, and the operators made of that: a stable counting sort of row keys, the embedding lookup
// with its gradient summed token by token, and rows sorted by expert and back.
//
// Every sum over the rows of a group runs over the grouped order in fixed pieces, so results do not depend on the
// order in which thread blocks run: there is no floating-point atomic in this file.  Sums are held in 32 bits and rounded
// to the type of the rows once, at the end.
#include <cooperative_groups.h>

#include <mutex>
#include <type_traits>

#include "rows.cuh"

namespace cg = cooperative_groups;

namespace tsb {
namespace {

// ------------------------------------------------------------------------------------------------ grouping
// A least-significant-digit radix sort of (key, row) with digits of up to 9 bits: 511 groups need one pass, 262143 two.
// Keys are ranked in tiles: warp w owns 256 consecutive keys and counts them 32 at a time, so equal keys keep their order;
// sums over the warps of a tile and over the tiles make the ranks global.  The only atomics count, on integers.
constexpr int kItems = 8;                        // keys of a thread
constexpr int kMaxDigits = 512;
static_assert(32 * kItems * sizeof(uint2) == kMaxDigits * sizeof(unsigned), "a warp's pairs and its masks share memory");
constexpr int kSortThreads = 256;                // of a tile of the sort of many keys
constexpr int kSortTile = kSortThreads * kItems;
constexpr int kClusterThreads = 1024;            // of a block of the sort of few keys, at most
constexpr int kClusterBlocks = 8;                // the largest cluster that every device guarantees
constexpr int kClusterKeys = kClusterBlocks * kClusterThreads * kItems;

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
// Which lanes of a warp have the same digit is found by setting their bits in a word per digit (masks, kMaxDigits words
// per warp; the same memory may serve scatter_tile): for 8192 keys in a block __match_any_sync took 12000 cycles, one
// vote per bit 9000, this 3600.
__device__ __forceinline__ void rank_tile(const unsigned (&digit)[kItems], const bool (&on)[kItems], unsigned (&rank)[kItems],
                                          unsigned short (*whist)[kMaxDigits], unsigned* masks, unsigned* total, int n_digits) {
  const int w = threadIdx.x >> 5, lane = threadIdx.x & 31, warps = blockDim.x >> 5;
  unsigned* mask = masks + w * kMaxDigits;
  for (int d = lane; d < n_digits; d += 32) {
    whist[w][d] = 0;
    mask[d] = 0;
  }
  __syncwarp();
#pragma unroll
  for (int it = 0; it < kItems; ++it) {
    if (on[it]) atomicOr(mask + digit[it], 1u << lane);
    __syncwarp();
    unsigned same = 0, before = 0;
    if (on[it]) {
      same = mask[digit[it]];
      before = whist[w][digit[it]];
    }
    rank[it] = before + __popc(same & ((1u << lane) - 1));
    __syncwarp();
    if (on[it] && lane == __ffs(same) - 1) {
      whist[w][digit[it]] = (unsigned short)(before + __popc(same));
      mask[digit[it]] = 0;
    }
    __syncwarp();
  }
  __syncthreads();
  for (int d = threadIdx.x; d < n_digits; d += blockDim.x) {
    unsigned sum = 0;
#pragma unroll 8
    for (int i = 0; i < warps; ++i) {
      const unsigned v = whist[i][d];
      whist[i][d] = (unsigned short)sum;
      sum += v;
    }
    total[d] = sum;
  }
  __syncthreads();
}

// In place: v[0..n) -> exclusive sums, by the whole block.  A word holds two 32-bit sums that are scanned at once.
// wsum: 33 words.
__device__ __forceinline__ void scan_digits(unsigned long long* v, int n, unsigned long long* wsum) {
  const int lane = threadIdx.x & 31, w = threadIdx.x >> 5, warps = blockDim.x >> 5;
  const auto inclusive = [&](unsigned long long x) {
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const unsigned long long up = __shfl_up_sync(0xffffffffu, x, o);
      if (lane >= o) x += up;
    }
    return x;
  };
  unsigned long long carry = 0;
  for (int d0 = 0; d0 < n; d0 += blockDim.x) {
    const int d = d0 + threadIdx.x;
    const unsigned long long own = d < n ? v[d] : 0ull, inc = inclusive(own);
    if (lane == 31) wsum[w] = inc;
    __syncthreads();
    if (w == 0) {
      const unsigned long long x = lane < warps ? wsum[lane] : 0ull, sum = inclusive(x);
      wsum[lane] = sum - x;
      if (lane == 31) wsum[32] = sum;
    }
    __syncthreads();
    if (d < n) v[d] = carry + wsum[w] + inc - own;
    carry += wsum[32];
    __syncthreads();
  }
}

// The keys of a tile leave it in the order of their digits: neighbours then go to neighbouring places, in runs instead of
// one by one.  both[d]: place of digit d in the tile (high) and, all tiles before it and `before[d]` keys of earlier tiles
// added, in the sorted rows (low).  put(position, key, row).
template <typename Put>
__device__ __forceinline__ void scatter_tile(const unsigned (&key)[kItems], const unsigned (&row)[kItems], const bool (&on)[kItems],
                                             const unsigned (&digit)[kItems], const unsigned (&rank)[kItems],
                                             const unsigned short (*whist)[kMaxDigits], unsigned long long* both,
                                             const unsigned* before, uint2* local, int count, int shift, int n_digits, Put&& put) {
  const int w = threadIdx.x >> 5;
#pragma unroll
  for (int it = 0; it < kItems; ++it)
    if (on[it]) local[(unsigned)(both[digit[it]] >> 32) + whist[w][digit[it]] + rank[it]] = make_uint2(key[it], row[it]);
  __syncthreads();
#pragma unroll 4
  for (int t = threadIdx.x; t < count; t += blockDim.x) {
    const uint2 v = local[t];
    const unsigned d = (v.x >> shift) & (n_digits - 1);
    const unsigned long long b = both[d];
    put((unsigned)b + before[d] + (unsigned)t - (unsigned)(b >> 32), v.x, v.y);
  }
}

struct SortOut {
  int* order;        // [n] row at a sorted position
  int* inverse;      // [n] sorted position of a row, or null
  unsigned* keys;    // [n] key at a sorted position, or null
  int* offsets;      // [n_groups + 1], or null; written where one digit holds the whole key
};

// n <= kClusterKeys: one cluster does every pass in one launch.  Block r holds the positions from r * tile on; its keys
// stay in registers, the counts and the sorted pairs cross through the blocks' shared memory, the last pass writes the
// result.  32768 keys below 100003, two passes: 21 us (three launches a pass as below took 32), of which the ranks take
// a fifth, the exchange of pairs nearly half.
size_t cluster_smem(int threads) {
  return (size_t)threads * kItems * 16 + (kMaxDigits + 33) * 8 + 2 * kMaxDigits * 4 + (size_t)(threads / 32) * kMaxDigits * 2;
}

__global__ void __launch_bounds__(kClusterThreads) sort_cluster_kernel(KeySource src, int n, int passes, int bits, SortOut out) {
  extern __shared__ __align__(16) unsigned char smem[];
  const int tile = blockDim.x * kItems;
  uint2* pairs = reinterpret_cast<uint2*>(smem);
  uint2* local = pairs + tile;
  unsigned long long* both = reinterpret_cast<unsigned long long*>(local + tile);
  unsigned long long* wsum = both + kMaxDigits;
  unsigned* total = reinterpret_cast<unsigned*>(wsum + 33);
  unsigned* before = total + kMaxDigits;
  auto whist = reinterpret_cast<unsigned short(*)[kMaxDigits]>(before + kMaxDigits);
  cg::cluster_group cluster = cg::this_cluster();
  const int w = threadIdx.x >> 5, blocks = (int)gridDim.x;
  const int at = w * 32 * kItems + (threadIdx.x & 31), base = (int)blockIdx.x * tile, count = min(tile, n - base);
  const unsigned per = 0xffffffffu / (unsigned)tile + 1;      // pos / tile = pos * per >> 32 for pos, tile <= 65536
  unsigned key[kItems], row[kItems], digit[kItems], rank[kItems];
  bool on[kItems];
#pragma unroll
  for (int it = 0; it < kItems; ++it) {
    row[it] = (unsigned)(base + at + it * 32);
    on[it] = at + it * 32 < count;
    key[it] = on[it] ? read_key(src, row[it]) : 0u;
  }
  const int n_digits = 1 << bits;
  for (int p = 0; p < passes; ++p) {
#pragma unroll
    for (int it = 0; it < kItems; ++it) digit[it] = (key[it] >> (p * bits)) & (n_digits - 1);
    rank_tile(digit, on, rank, whist, reinterpret_cast<unsigned*>(local), total, n_digits);
    if (blocks > 1) cluster.sync();      // every block's counts are there
    for (int d = threadIdx.x; d < n_digits; d += blockDim.x) {
      unsigned sum = 0, mine = 0;
#pragma unroll
      for (int q = 0; q < kClusterBlocks; ++q) {
        if (q >= blocks) break;
        if (q == (int)blockIdx.x) mine = sum;      // what earlier blocks have of this digit
        sum += *cluster.map_shared_rank(total + d, q);
      }
      both[d] = (unsigned long long)total[d] << 32 | sum;
      before[d] = mine;
    }
    __syncthreads();
    scan_digits(both, n_digits, wsum);
    if (out.offsets && blockIdx.x == 0)
      for (int d = threadIdx.x; d <= (int)src.n_groups; d += blockDim.x) out.offsets[d] = (int)(unsigned)both[d];
    if (p + 1 == passes) {
      scatter_tile(key, row, on, digit, rank, whist, both, before, local, count, p * bits, n_digits,
                   [&](unsigned pos, unsigned k, unsigned r) {
                     out.order[pos] = (int)r;
                     if (out.inverse) out.inverse[r] = (int)pos;
                     if (out.keys) out.keys[pos] = k;
                   });
      if (blocks > 1) cluster.sync();      // no block reads this one's counts any more
      break;
    }
    scatter_tile(key, row, on, digit, rank, whist, both, before, local, count, p * bits, n_digits,
                 [&](unsigned pos, unsigned k, unsigned r) {
                   const unsigned to = __umulhi(pos, per);
                   cluster.map_shared_rank(pairs, (int)to)[pos - to * tile] = make_uint2(k, r);
                 });
    if (blocks > 1) cluster.sync(); else __syncthreads();      // the pairs are there
#pragma unroll
    for (int it = 0; it < kItems; ++it) {
      if (!on[it]) continue;
      const uint2 v = pairs[at + it * 32];
      key[it] = v.x;
      row[it] = v.y;
    }
  }
}

// More keys: three launches a pass, tiles of 2048 keys.  500009 keys below 301, one pass: 18 us, all of it latency.
//
// keys and rows of one pass: the caller's keys in the first, the previous pass's pairs afterwards
struct PassIn {
  KeySource src;
  const unsigned* keys;      // null: the first pass
  const int* rows;
};

__device__ __forceinline__ void load_tile(const PassIn& in, int64_t n, unsigned (&key)[kItems], bool (&on)[kItems], int64_t first) {
#pragma unroll
  for (int it = 0; it < kItems; ++it) {
    const int64_t i = first + it * 32;
    on[it] = i < n;
    key[it] = on[it] ? (in.keys ? __ldg(in.keys + i) : read_key(in.src, i)) : 0u;
  }
}

__global__ void __launch_bounds__(kSortThreads) sort_count_kernel(PassIn in, int64_t n, int shift, int bits, int64_t tiles,
                                                                  unsigned* __restrict__ counts) {
  __shared__ unsigned total[kMaxDigits];
  const int n_digits = 1 << bits;
  unsigned key[kItems];
  bool on[kItems];
  load_tile(in, n, key, on, (int64_t)blockIdx.x * kSortTile + (threadIdx.x >> 5) * 32 * kItems + (threadIdx.x & 31));
  for (int d = threadIdx.x; d < n_digits; d += kSortThreads) total[d] = 0;
  __syncthreads();
#pragma unroll
  for (int it = 0; it < kItems; ++it)
    if (on[it]) atomicAdd(total + ((key[it] >> shift) & (n_digits - 1)), 1u);
  __syncthreads();
  for (int d = threadIdx.x; d < n_digits; d += kSortThreads) counts[d * tiles + blockIdx.x] = total[d];
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
  __shared__ unsigned short whist[kSortThreads / 32][kMaxDigits];
  __shared__ unsigned total[kMaxDigits], before[kMaxDigits];
  __shared__ unsigned long long both[kMaxDigits], wsum[33];
  __shared__ uint2 local[kSortTile];
  const int at = (threadIdx.x >> 5) * 32 * kItems + (threadIdx.x & 31), n_digits = 1 << bits;
  const int64_t base = (int64_t)blockIdx.x * kSortTile;
  unsigned key[kItems], row[kItems], digit[kItems], rank[kItems];
  bool on[kItems];
  load_tile(in, n, key, on, base + at);
#pragma unroll
  for (int it = 0; it < kItems; ++it) {
    const int64_t i = base + at + it * 32;
    row[it] = !on[it] ? 0u : in.keys ? (unsigned)__ldg(in.rows + i) : (unsigned)i;
    digit[it] = (key[it] >> shift) & (n_digits - 1);
  }
  rank_tile(digit, on, rank, whist, reinterpret_cast<unsigned*>(local), total, n_digits);
  for (int d = threadIdx.x; d < n_digits; d += kSortThreads) {
    both[d] = (unsigned long long)total[d] << 32 | counts[(int64_t)n_digits * tiles + d];
    before[d] = counts[d * tiles + blockIdx.x];
  }
  __syncthreads();
  scan_digits(both, n_digits, wsum);
  if (out.offsets && blockIdx.x == 0)
    for (int d = threadIdx.x; d <= (int)in.src.n_groups; d += kSortThreads) out.offsets[d] = (int)(unsigned)both[d];
  scatter_tile(key, row, on, digit, rank, whist, both, before, local, (int)min((int64_t)kSortTile, n - base), shift, n_digits,
               [&](unsigned pos, unsigned k, unsigned r) {
                 out.order[pos] = (int)r;
                 if (out.keys) out.keys[pos] = k;
                 if (out.inverse) out.inverse[r] = (int)pos;
               });
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
  while ((n_groups >> total) != 0) ++total;      // keys are 0 .. n_groups
  p.passes = (total + 8) / 9;
  p.bits = (total + p.passes - 1) / p.passes;
  p.tiles = cdiv(n, kSortTile);
  p.pairs = align_up((size_t)n * 4, 256);
  p.counts = n <= kClusterKeys ? 0 : align_up(((size_t)(p.tiles + 1) << p.bits) * sizeof(unsigned), 256);
  // the sorted keys where the offsets are searched in them; two sets of (key, row) beside the tiles' counts
  p.bytes = n <= kClusterKeys ? (p.passes > 1 ? p.pairs : 0) : p.counts + 5 * p.pairs;
  return p;
}

int allow_cluster_smem() {
  static std::mutex mu;
  static bool done[64] = {};
  int dev = 0;
  TSB_CUDA_TRY(cudaGetDevice(&dev));
  if (dev < 0 || dev >= 64) return TSB_ERR_LIMIT;
  std::lock_guard<std::mutex> lock(mu);
  if (!done[dev]) {
    TSB_CUDA_TRY(cudaFuncSetAttribute(sort_cluster_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                      (int)cluster_smem(kClusterThreads)));
    done[dev] = true;
  }
  return TSB_OK;
}

// order / inverse / keys / offsets of n >= 1 keys
int run_sort(const KeySource& src, int64_t n, SortOut out, void* workspace, cudaStream_t st) {
  const SortPlan p = sort_plan(n, src.n_groups);
  char* ws = static_cast<char*>(workspace);
  int* const offsets = out.offsets;
  const bool search = offsets && p.passes > 1;      // more than one digit: the offsets are searched in the sorted keys
  if (search && !out.keys) out.keys = reinterpret_cast<unsigned*>(ws);
  if (p.passes > 1) out.offsets = nullptr;
  if (n <= kClusterKeys) {
    const int rc = allow_cluster_smem();
    if (rc != TSB_OK) return rc;
    // 2048 keys fit a block of 8 warps; more of them are spread over the whole cluster
    const int64_t warps = cdiv(n, (n <= kSortTile ? 1 : kClusterBlocks) * 32 * kItems);
    const int threads = 32 * (int)(warps < 2 ? 2 : warps);
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)cdiv(n, (int64_t)threads * kItems));
    cfg.blockDim = dim3(threads);
    cfg.dynamicSmemBytes = cluster_smem(threads);
    cfg.stream = st;
    cudaLaunchAttribute at[1];
    at[0].id = cudaLaunchAttributeClusterDimension;
    at[0].val.clusterDim.x = cfg.gridDim.x;
    at[0].val.clusterDim.y = at[0].val.clusterDim.z = 1;
    cfg.attrs = at;
    cfg.numAttrs = 1;
    count_launch();
    TSB_CUDA_TRY(cudaLaunchKernelEx(&cfg, sort_cluster_kernel, src, (int)n, p.passes, p.bits, out));
  } else {
    unsigned* counts = reinterpret_cast<unsigned*>(ws + p.pairs);
    ws += p.pairs + p.counts;
    PassIn in{src, nullptr, nullptr};
    for (int i = 0; i < p.passes; ++i) {
      SortOut to = out;
      if (i + 1 < p.passes)
        to = SortOut{reinterpret_cast<int*>(ws + (2 * (i & 1) + 1) * p.pairs), nullptr,
                     reinterpret_cast<unsigned*>(ws + 2 * (i & 1) * p.pairs), nullptr};
      sort_count_kernel<<<(unsigned)p.tiles, kSortThreads, 0, st>>>(in, n, i * p.bits, p.bits, p.tiles, counts);
      TSB_LAUNCH_CHECK();
      sort_scan_kernel<<<1 << p.bits, 256, 0, st>>>(counts, p.tiles, 1 << p.bits);
      TSB_LAUNCH_CHECK();
      sort_scatter_kernel<<<(unsigned)p.tiles, kSortThreads, 0, st>>>(in, n, i * p.bits, p.bits, p.tiles, counts, to);
      TSB_LAUNCH_CHECK();
      in.keys = to.keys;
      in.rows = to.order;
    }
  }
  if (search) {
    group_offsets_kernel<<<grid_for((int64_t)src.n_groups + 1, 256), 256, 0, st>>>(out.keys, n, src.n_groups, offsets);
    TSB_LAUNCH_CHECK();
  }
  return TSB_OK;
}

// ------------------------------------------------------------------------------------------------ embedding
constexpr int kThreads = 256;
// y[i] = scale * table[token[i]], zeros where the token is no row of the table: a thread has U vectors of the result, and the
// blocks follow one another.  (A grid that stays and reads the tokens of its next vectors ahead took 27 us where this
// takes 20, for 500009 x 64 bf16: waiting blocks are replaced sooner than waiting loops go round.)
//
// A vector of the result (16 bytes wherever its rows lie, the result being one run of memory) is made of PARTS loads of VEC
// values, as wide as the rows of the table allow: a part lies in one row, a vector may lie in two or more.
// Row and part of a thread's first vector take one exact division, those of the next ones a step of whole rows and parts:
// with a division for each this kernel was bound by its arithmetic.
struct TokenStep {
  unsigned rows, parts;      // of the vectors of a block
};

template <typename T, int VEC, int PARTS>
__global__ void __launch_bounds__(kThreads) embed_kernel(const T* __restrict__ table, KeySource src, int64_t total, RowSplit split,
                                                         TokenStep step, float scale, T* __restrict__ out) {
  constexpr int U = PARTS > 4 ? 2 : 4;
  const int64_t t0 = blockIdx.x * (int64_t)(kThreads * U) + threadIdx.x;
  const unsigned cols = split.cols, c = cols * VEC;
  Pack<T, VEC> v[U][PARTS];
  int64_t first = split.row(t0 * PARTS);
  unsigned part = (unsigned)(t0 * PARTS - first * cols);
  int left = (int)min(total - t0 * PARTS, (int64_t)(kThreads * U * PARTS));      // parts of the result from t0 on
#pragma unroll
  for (int u = 0; u < U; ++u) {
    int64_t i = first;
    unsigned col = part, row = left > 0 ? read_key(src, i) : src.n_groups;
#pragma unroll
    for (int q = 0; q < PARTS; ++q) {
      v[u][q].clear();
      if (q < left && row < src.n_groups) v[u][q].load(table + (uint64_t)row * c + col * VEC);
      if (q + 1 < PARTS && ++col == cols) {
        col = 0;
        ++i;
        if (q + 1 < left) row = read_key(src, i);
      }
    }
    first += step.rows;
    part += step.parts;
    if (part >= cols) {
      part -= cols;
      ++first;
    }
    left -= kThreads * PARTS;
  }
#pragma unroll
  for (int u = 0; u < U; ++u) {
    const int64_t t = (t0 + u * kThreads) * PARTS;
    if (t >= total) break;
    Pack<T, VEC * PARTS> o;
    float f[VEC * PARTS];
#pragma unroll
    for (int q = 0; q < PARTS; ++q) {
      float g[VEC];
      v[u][q].get(g);
#pragma unroll
      for (int e = 0; e < VEC; ++e) f[q * VEC + e] = g[e] * scale;
    }
    o.set(f);
    if (PARTS == 1 || t + PARTS <= total) {
      o.store(out + t * VEC);
    } else {      // the end of the result
#pragma unroll
      for (int q = 0; q < PARTS; ++q) {
        if (t + q >= total) break;
#pragma unroll
        for (int e = 0; e < VEC; ++e) out[(t + q) * VEC + e] = from_f32<T>(f[q * VEC + e]);
      }
    }
  }
}

// The gradient of the table: dtable[v] = scale * sum of grad[i] over the rows i whose token is v.
//
// The rows are walked in sorted order by workers of `cols` threads (one thread per vector of a row), each over `len`
// positions; a block holds `per_block` workers of consecutive positions.  A token whose positions lie inside one
// worker is summed and written there.  One that crosses workers leaves 32-bit partial sums in shared memory, `tail`
// where it begins and `head` where it goes on, which the worker in which it begins adds up in order; one that crosses
// blocks leaves them in memory for embed_join_kernel.  The blocks behind the workers write the zeros of the tokens that
// do not occur, so every row of the table is written exactly once.
//
// 32768 x 2048 bf16 into 100003 rows: 88 us for 544 MB, 83 at the copy rate.  500009 x 64 bf16 into 301 rows: 19 us for
// 64 MB, bound by the latency of a worker's start and its last joins; 27 us before the rows came by cp.async.
struct EmbedGrad {
  const unsigned* keys;      // sorted; n_rows marks rows without a token
  const int* order;
  int64_t n, n_rows, c;
  int len;                   // positions of a worker
  int tile;                  // vectors of a row that a block takes (grid.y tiles)
  int per_block;             // workers of a block
  int64_t span, blocks;      // positions of a block, blocks
  float scale;
  float* head;               // [blocks, c]
  float* tail;
};

constexpr int kGradAhead = 2;      // batches on their way
template <typename T, int VEC>
constexpr int kGradRows = VEC * sizeof(T) == 16 ? 4 : 8;      // rows of a batch
template <typename T, int VEC>
constexpr int kGradBytes = kAsyncVector<T, VEC> ? (kGradAhead + 1) * kGradRows<T, VEC> * kThreads * VEC * (int)sizeof(T) : 0;

template <typename T, int VEC>
__device__ __forceinline__ void write_row(const EmbedGrad& a, float (&acc)[VEC], T* __restrict__ to) {
  Pack<T, VEC> o;
#pragma unroll
  for (int e = 0; e < VEC; ++e) acc[e] *= a.scale;
  o.set(acc);
  o.store(to);
}

template <typename T, int VEC>
__global__ void __launch_bounds__(kThreads, 3) embed_grad_kernel(EmbedGrad a, const T* __restrict__ grad, T* __restrict__ dtable,
                                                              int zero_rows) {
  extern __shared__ __align__(16) unsigned char pipe[];
  __shared__ float s_head[VEC][kThreads], s_tail[VEC][kThreads];
  __shared__ unsigned char s_flags[kThreads];      // of a worker: 1 = it has a tail, 2 = its head goes on behind it
  const int first = blockIdx.y * a.tile, width = min(a.tile, (int)(a.c / VEC) - first);
  if (blockIdx.x >= a.blocks) {
    const int64_t v0 = (blockIdx.x - a.blocks) * (int64_t)zero_rows;
    if ((int)threadIdx.x < zero_rows) {
      const int64_t v = v0 + threadIdx.x;
      bool none = false;
      if (v < a.n_rows) {
        const int64_t at = lower_bound(a.keys, a.n, (unsigned)v);
        none = at >= a.n || __ldg(a.keys + at) != (unsigned)v;
      }
      s_flags[threadIdx.x] = none;
    }
    __syncthreads();
    Pack<T, VEC> zero;
    zero.clear();
    for (int t = threadIdx.x; t < zero_rows * width; t += kThreads) {
      const int r = t / width;
      if (s_flags[r]) zero.store(dtable + (v0 + r) * a.c + (int64_t)(first + t - r * width) * VEC);
    }
    return;
  }
  const unsigned none = (unsigned)a.n_rows;
  const int slot = threadIdx.x / width, col = threadIdx.x - slot * width;
  const int64_t j = (int64_t)(first + col) * VEC;
  const int64_t p0 = blockIdx.x * a.span + (int64_t)slot * a.len, p1 = min(p0 + a.len, a.n);
  const bool live = slot < a.per_block && p0 < a.n;
  bool has_head = false, through = false, has_tail = false;
  unsigned cur = none;
  float acc[VEC];
#pragma unroll
  for (int e = 0; e < VEC; ++e) acc[e] = 0.f;
  if (live) {
    cur = __ldg(a.keys + p0);
    bool goes_on = cur != none && p0 > 0 && __ldg(a.keys + p0 - 1) == cur;      // the run began in an earlier worker
    has_head = goes_on;
    const auto take = [&](unsigned key, const Pack<T, VEC>& v) {
      if (cur == none) return;
      if (key != cur) {      // the run of `cur` ended inside this worker
        if (goes_on) {
#pragma unroll
          for (int e = 0; e < VEC; ++e) s_head[e][threadIdx.x] = acc[e];
        } else {
          write_row(a, acc, dtable + (int64_t)cur * a.c + j);
        }
#pragma unroll
        for (int e = 0; e < VEC; ++e) acc[e] = 0.f;
        cur = key;
        goes_on = false;
        if (cur == none) return;
      }
      float g[VEC];
      v.get(g);
#pragma unroll
      for (int e = 0; e < VEC; ++e) acc[e] += g[e];
    };
    const int count = (int)(p1 - p0);
    const unsigned* keys = a.keys + p0;
    const int* order = a.order + p0;
    constexpr int U = kGradRows<T, VEC>;
    if constexpr (kAsyncVector<T, VEC>) {
      // Rows come through shared memory by cp.async, kGradAhead batches ahead, in slots of this thread's own; the rows'
      // numbers are read one batch before they are needed, the keys one batch before they are compared.
      constexpr int D = kGradAhead + 1, kBytes = Pack<T, VEC>::kBytes;
      unsigned char* mine = pipe + threadIdx.x * kBytes;
      const auto slot = [&](int stage, int u) { return mine + (stage * U + u) * kThreads * kBytes; };
      int row[U];
      unsigned key[U], next[U];
      const auto rows_of = [&](int k) {
#pragma unroll
        for (int u = 0; u < U; ++u) row[u] = k + u < count ? __ldg(order + k + u) : -1;
      };
      const auto issue = [&](int stage) {
#pragma unroll
        for (int u = 0; u < U; ++u)
          if (row[u] >= 0) async_copy<kBytes>(slot(stage, u), grad + (int64_t)row[u] * a.c + j);
        async_commit();
      };
      rows_of(0);
#pragma unroll
      for (int d = 0; d < kGradAhead; ++d) {
        issue(d);
        rows_of((d + 1) * U);
      }
#pragma unroll
      for (int u = 0; u < U; ++u) key[u] = u < count ? __ldg(keys + u) : none;
      int stage = 0;
      for (int k = 0; k < count && cur != none; k += U) {
        issue(stage == 0 ? D - 1 : stage - 1);
        rows_of(k + D * U);
#pragma unroll
        for (int u = 0; u < U; ++u) next[u] = k + U + u < count ? __ldg(keys + k + U + u) : none;
        async_wait<kGradAhead>();
#pragma unroll
        for (int u = 0; u < U; ++u) {
          Pack<T, VEC> v;
          v.raw = *reinterpret_cast<const typename Pack<T, VEC>::Raw*>(slot(stage, u));
          if (k + u < count) take(key[u], v);
        }
#pragma unroll
        for (int u = 0; u < U; ++u) key[u] = next[u];
        stage = stage + 1 == D ? 0 : stage + 1;
      }
      async_wait<0>();
    } else {
      for (int k = 0; k < count && cur != none; k += U) {
        Pack<T, VEC> v[U];
        unsigned key[U];
#pragma unroll
        for (int u = 0; u < U; ++u) {
          key[u] = k + u < count ? __ldg(keys + k + u) : none;
          if (key[u] != none) v[u].load(grad + (int64_t)__ldg(order + k + u) * a.c + j);
        }
#pragma unroll
        for (int u = 0; u < U; ++u)
          if (k + u < count) take(key[u], v[u]);
      }
    }
    if (cur != none) {
      const bool on = p1 < a.n && __ldg(a.keys + p1) == cur;      // the run goes on in the next worker
      if (goes_on) {
        through = on;
#pragma unroll
        for (int e = 0; e < VEC; ++e) s_head[e][threadIdx.x] = acc[e];
      } else if (on) {
        has_tail = true;
#pragma unroll
        for (int e = 0; e < VEC; ++e) s_tail[e][threadIdx.x] = acc[e];
      } else {
        write_row(a, acc, dtable + (int64_t)cur * a.c + j);
      }
    }
    if (col == 0) s_flags[slot] = (has_tail ? 1 : 0) | (through ? 2 : 0);
  }
  __syncthreads();
  if (!live) return;
  // A run that began before this block: the first worker collects its heads.  One that began in a worker: that worker.
  const bool begins = slot == 0 && has_head;
  if (!begins && !has_tail) return;
  for (int which = begins ? 0 : 1; which < (has_tail ? 2 : 1); ++which) {
    int x = slot;
    bool more = which == 0 ? through : true;
#pragma unroll
    for (int e = 0; e < VEC; ++e) acc[e] = which == 0 ? s_head[e][threadIdx.x] : s_tail[e][threadIdx.x];
    while (more && x + 1 < a.per_block) {
      ++x;
#pragma unroll
      for (int e = 0; e < VEC; ++e) acc[e] += s_head[e][x * width + col];
      more = s_flags[x] & 2;
    }
    if (which == 0 || more) {
      float* to = (which == 0 ? a.head : a.tail) + blockIdx.x * a.c + j;
#pragma unroll
      for (int e = 0; e < VEC; ++e) to[e] = acc[e];
    } else {
      write_row(a, acc, dtable + (int64_t)cur * a.c + j);
    }
  }
}

// A block per block of embed_grad_kernel in which a run begins that goes on behind it, and per 128 JV channels: its tail and
// the heads of the blocks that follow (those whose first key is the same), threads = channels (JV a thread) x slices of
// those blocks.  Most find no run to join and leave at once: 5 us for 500009 tokens of 301 rows, 13 us for 32768 x 2048.
constexpr int kJoinThreads = 512, kJoinColumns = 128;
template <typename T, int JV>
__global__ void __launch_bounds__(kJoinThreads) embed_join_kernel(EmbedGrad a, T* __restrict__ dtable) {
  __shared__ float part[JV][kJoinThreads];
  const int64_t p0 = blockIdx.x * a.span, p1 = p0 + a.span;
  if (p1 >= a.n) return;
  const unsigned key = __ldg(a.keys + p1 - 1);
  if (key == (unsigned)a.n_rows || __ldg(a.keys + p1) != key) return;
  if (p0 > 0 && __ldg(a.keys + p0 - 1) == key) return;      // it began before (the keys are sorted)
  const int64_t j0 = (int64_t)blockIdx.y * kJoinColumns * JV;
  const int cols = (int)min((a.c - j0) / JV, (int64_t)kJoinColumns), slices = kJoinThreads / cols;
  const int slice = threadIdx.x / cols, q = threadIdx.x - slice * cols;
  const int64_t j = j0 + q * JV;
  float s[JV];
#pragma unroll
  for (int e = 0; e < JV; ++e) s[e] = 0.f;
  if (slice < slices) {
    constexpr int U = 4;
    bool more = true;
    for (int64_t k = blockIdx.x + 1 + slice; more; k += U * slices) {
      Pack<float, JV> v[U];
      bool on[U];
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const int64_t b = k + u * slices;
        on[u] = b < a.blocks && __ldg(a.keys + b * a.span) == key;
        v[u].clear();
        if (on[u]) v[u].load(a.head + b * a.c + j);
      }
#pragma unroll
      for (int u = 0; u < U; ++u) {
        float f[JV];
        v[u].get(f);
        if (on[u]) {
#pragma unroll
          for (int e = 0; e < JV; ++e) s[e] += f[e];
        }
      }
      more = on[U - 1];
    }
  }
#pragma unroll
  for (int e = 0; e < JV; ++e) part[e][threadIdx.x] = s[e];
  __syncthreads();
  if (slice != 0) return;
#pragma unroll
  for (int e = 0; e < JV; ++e) {
    float all = a.tail[blockIdx.x * a.c + j + e];
    for (int i = 0; i < slices; ++i) all += part[e][i * cols + q];
    dtable[(int64_t)key * a.c + j + e] = from_f32<T>(all * a.scale);
  }
}

EmbedGrad embed_plan(int64_t n, int64_t n_rows, int64_t c, int vec) {
  EmbedGrad a{};
  a.n = n;
  a.n_rows = n_rows;
  a.c = c;
  const int64_t vecs = c / vec;
  a.tile = (int)cdiv(vecs, cdiv(vecs, kThreads));
  a.per_block = kThreads / a.tile;
  // one wave of resident blocks where that leaves workers of 8 to 64 positions
  int64_t len = cdiv(n, cdiv(3 * kSmCount, cdiv(vecs, a.tile)) * a.per_block);
  len = len < 8 ? 8 : len > 64 ? 64 : len;
  a.len = (int)len;
  a.span = len * a.per_block;
  a.blocks = cdiv(n, a.span);
  return a;
}

// ------------------------------------------------------------------------------------------------ experts
// Position p of the sorted rows belongs to choice order[p] of the n * k choices; positions at and behind offsets[E]
// belong to choices of no expert.

// xs[inverse[i][j]] = x[i], zeros behind the kept rows: a vector of x is read once and written k times.  131072 x 2 of 512
// bf16: 60 us for 402 MB, the copy rate.
template <typename T, int VEC>
__global__ void __launch_bounds__(kThreads) dispatch_kernel(const T* __restrict__ x, const int* __restrict__ inverse,
                                                            const int* __restrict__ kept, int64_t total, int64_t pairs, int k,
                                                            RowSplit split, T* __restrict__ xs) {
  constexpr int U = 2;
  const int64_t t0 = blockIdx.x * (int64_t)(kThreads * U) + threadIdx.x;
  const int64_t c = (int64_t)split.cols * VEC, n_kept = __ldg(kept);
  Pack<T, VEC> v[U], zero;
  zero.clear();
#pragma unroll
  for (int u = 0; u < U; ++u)
    if (t0 + u * kThreads < total) v[u].load(x + (t0 + u * kThreads) * VEC);
#pragma unroll
  for (int u = 0; u < U; ++u) {
    const int64_t t = t0 + u * kThreads;
    if (t >= total) break;
    const int64_t i = split.row(t), j = (t - i * split.cols) * VEC;
    for (int q = 0; q < k; ++q) {
      const int64_t pos = __ldg(inverse + i * k + q);
      if (pos >= 0 && pos < pairs) (pos < n_kept ? v[u] : zero).store(xs + pos * c + j);
    }
  }
}

// The two kernels below give a row (a choice) to a group of `lanes` threads and let a grid that fits the machine walk over
// the rows.  A step is what a thread reads at once: two steps more are on their way through shared memory by cp.async, in slots of the
// thread's own, and the indices of the step behind them; single 16-bit values are loaded when they are needed, with the
// next step's indices on their way.  (131072 x 2 of 512 bf16: combined in 79 us with loads
// into registers, in 64 us so; the gradient in 132 and 104 us.)
constexpr int kStepAhead = 2;
constexpr int step_vectors(int bytes) { return bytes == 16 ? 4 : 8; }      // of a thread
constexpr int step_bytes(int bytes) { return bytes >= 4 ? (kStepAhead + 1) * step_vectors(bytes) * kThreads * bytes : 0; }
constexpr int row_blocks(int bytes) { return (bytes >= 8 ? 3 : 6) * kSmCount; }      // resident: 48 KB of slots each, or 24

// out[i] = sum over j of w[i][j] * rows[inverse[i][j]] (w null: 1), in the order of j.  A step: KU choices of a row, U vectors
// of each.
template <typename T, int VEC, int KU>
__global__ void __launch_bounds__(kThreads) combine_kernel(const T* __restrict__ rows, const void* __restrict__ w, int w_dtype,
                                                           const int* __restrict__ inverse, const int* __restrict__ kept,
                                                           int64_t n, int k, int64_t c, int lanes, T* __restrict__ out) {
  constexpr int kBytes = Pack<T, VEC>::kBytes, U = step_vectors(kBytes) / KU;
  constexpr bool kAsync = kAsyncVector<T, VEC>;
  constexpr int D = kAsync ? kStepAhead + 1 : 1;
  extern __shared__ __align__(16) unsigned char pipe[];
  const int cols = (int)(c / VEC), groups = kThreads / lanes, group = threadIdx.x / lanes, lane = threadIdx.x - group * lanes;
  const int64_t step = (int64_t)gridDim.x * groups;
  const unsigned n_kept = (unsigned)min((int64_t)max(__ldg(kept), 0), n * k);
  struct Place {      // row, first vector, first choice
    int64_t i;
    int v, q;
  };
  const auto advance = [&](Place& p) {
    p.q += KU;
    if (p.q < k) return;
    p.q = 0;
    p.v += lanes * U;
    if (p.v < cols) return;
    p.v = lane;
    p.i += step;
  };
  // positions (no expert: none) and weights of a step
  const unsigned none = 0xffffffffu;
  const auto fetch = [&](const Place& p, unsigned (&pos)[KU], float (&f)[KU]) {
#pragma unroll
    for (int u = 0; u < KU; ++u) {
      const bool in = p.i < n && p.q + u < k;
      pos[u] = in ? (unsigned)__ldg(inverse + p.i * k + p.q + u) : none;
      f[u] = in && w ? load_any(w, w_dtype, p.i * k + p.q + u) : 1.f;
    }
  };
  const auto slot = [&](int stage, int u, int x) { return pipe + (((stage * KU + u) * U + x) * kThreads + threadIdx.x) * kBytes; };
  const auto issue = [&](int stage, const Place& p, const unsigned (&pos)[KU]) {
#pragma unroll
    for (int u = 0; u < KU; ++u)
#pragma unroll
      for (int x = 0; x < U; ++x)
        if (pos[u] < n_kept && p.v + x * lanes < cols)
          async_copy<kBytes>(slot(stage, u, x), rows + (int64_t)pos[u] * c + (p.v + x * lanes) * VEC);
    async_commit();
  };
  Place now{blockIdx.x * (int64_t)groups + group, lane, 0}, ahead = now;
  if (group >= groups || lane >= cols) now.i = ahead.i = n;      // threads left over
  unsigned pos[D + 1][KU];      // of the steps from `now` on; the last is on its way
  float f[D + 1][KU];
  fetch(ahead, pos[0], f[0]);
#pragma unroll
  for (int d = 0; d < D - 1; ++d) {
    if constexpr (kAsync) issue(d, ahead, pos[d]);
    advance(ahead);
    fetch(ahead, pos[d + 1], f[d + 1]);
  }
  float acc[U][VEC];
  int stage = 0;
  while (now.i < n) {
    if constexpr (kAsync) issue(stage == 0 ? D - 1 : stage - 1, ahead, pos[D - 1]);
    advance(ahead);
    fetch(ahead, pos[D], f[D]);
    Pack<T, VEC> p[KU][U];
    if constexpr (kAsync) {
      async_wait<kStepAhead>();
    } else {
#pragma unroll
      for (int u = 0; u < KU; ++u)
#pragma unroll
        for (int x = 0; x < U; ++x)
          if (pos[0][u] < n_kept && now.v + x * lanes < cols) p[u][x].load(rows + (int64_t)pos[0][u] * c + (now.v + x * lanes) * VEC);
    }
    if (now.q == 0) {
#pragma unroll
      for (int x = 0; x < U; ++x)
#pragma unroll
        for (int e = 0; e < VEC; ++e) acc[x][e] = 0.f;
    }
#pragma unroll
    for (int u = 0; u < KU; ++u) {
      if (pos[0][u] >= n_kept) continue;
#pragma unroll
      for (int x = 0; x < U; ++x) {
        if (now.v + x * lanes >= cols) continue;
        if constexpr (kAsync) p[u][x].raw = *reinterpret_cast<const typename Pack<T, VEC>::Raw*>(slot(stage, u, x));
        float v[VEC];
        p[u][x].get(v);
#pragma unroll
        for (int e = 0; e < VEC; ++e) acc[x][e] = fmaf(f[0][u], v[e], acc[x][e]);
      }
    }
    if (now.q + KU >= k) {
#pragma unroll
      for (int x = 0; x < U; ++x) {
        if (now.v + x * lanes >= cols) continue;
        Pack<T, VEC> o;
        o.set(acc[x]);
        o.store(out + now.i * c + (now.v + x * lanes) * VEC);
      }
    }
    advance(now);
#pragma unroll
    for (int d = 0; d < D; ++d)
#pragma unroll
      for (int u = 0; u < KU; ++u) {
        pos[d][u] = pos[d + 1][u];
        f[d][u] = f[d + 1][u];
      }
    stage = stage + 1 == D ? 0 : stage + 1;
  }
  if constexpr (kAsync) async_wait<0>();
}

// drows[pos] = w * dout[i] and dw = <dout[i], rows[pos]> of a choice, both zero for a choice of no expert.  A step: two vectors
// of both rows; `lanes` is a power of two up to a warp.  Choices of one row share its dout through the caches.
template <typename T, int VEC>
__global__ void __launch_bounds__(kThreads) combine_grad_kernel(const T* __restrict__ dout, const T* __restrict__ rows,
                                                                const void* __restrict__ w, int w_dtype,
                                                                const int* __restrict__ inverse, const int* __restrict__ kept,
                                                                int64_t pairs, RowSplit by_k, int64_t c, int lanes,
                                                                T* __restrict__ drows, void* __restrict__ dw) {
  constexpr int kBytes = Pack<T, VEC>::kBytes, U = step_vectors(kBytes) / 2;
  constexpr bool kAsync = kAsyncVector<T, VEC>;
  constexpr int D = kAsync ? kStepAhead + 1 : 1;
  extern __shared__ __align__(16) unsigned char pipe[];
  const int cols = (int)(c / VEC), lane = threadIdx.x & (lanes - 1), groups = kThreads / lanes;
  const int64_t step = (int64_t)gridDim.x * groups;
  const unsigned n_kept = (unsigned)min((int64_t)max(__ldg(kept), 0), pairs);
  struct Place {      // choice, first vector
    int64_t q;
    int v;
  };
  const auto advance = [&](Place& p) {
    p.v += lanes * U;
    if (p.v - lane < cols) return;      // the same for all threads of a warp, which sum together
    p.v = lane;
    p.q += step;
  };
  const unsigned none = 0xffffffffu;
  const auto fetch = [&](const Place& p, unsigned& pos, float& f) {
    pos = p.q < pairs ? (unsigned)__ldg(inverse + p.q) : none;
    f = p.q < pairs ? load_any(w, w_dtype, p.q) : 0.f;
  };
  const auto slot = [&](int stage, int i, int u) { return pipe + (((stage * 2 + i) * U + u) * kThreads + threadIdx.x) * kBytes; };
  const auto issue = [&](int stage, const Place& p, unsigned pos) {
    if (pos < n_kept) {
      const T* g = dout + by_k.row(p.q) * c + p.v * VEC;
      const T* r = rows + (int64_t)pos * c + p.v * VEC;
#pragma unroll
      for (int u = 0; u < U; ++u) {
        if (p.v + u * lanes >= cols) continue;
        async_copy<kBytes>(slot(stage, 0, u), r + u * lanes * VEC);
        async_copy<kBytes>(slot(stage, 1, u), g + u * lanes * VEC);
      }
    }
    async_commit();
  };
  const int64_t warp_q = blockIdx.x * (int64_t)groups + (threadIdx.x / 32) * (32 / lanes);      // of the warp's first group
  const int64_t own = threadIdx.x / lanes - (threadIdx.x / 32) * (32 / lanes);
  Place now{warp_q + own, lane}, ahead = now;
  unsigned pos[D + 1];
  float f[D + 1];
  fetch(ahead, pos[0], f[0]);
#pragma unroll
  for (int d = 0; d < D - 1; ++d) {
    if constexpr (kAsync) issue(d, ahead, pos[d]);
    advance(ahead);
    fetch(ahead, pos[d + 1], f[d + 1]);
  }
  float dot = 0.f;
  int stage = 0;
  while (now.q - own < pairs) {      // the same for all threads of a warp
    if constexpr (kAsync) issue(stage == 0 ? D - 1 : stage - 1, ahead, pos[D - 1]);
    advance(ahead);
    fetch(ahead, pos[D], f[D]);
    const bool used = pos[0] < n_kept;
    T* d0 = drows + (int64_t)pos[0] * c;
    if constexpr (kAsync) async_wait<kStepAhead>();
    if (used) {
      Pack<T, VEC> r[U], g[U];
      if constexpr (!kAsync) {
#pragma unroll
        for (int u = 0; u < U; ++u) {
          if (now.v + u * lanes >= cols) continue;
          r[u].load(rows + (int64_t)pos[0] * c + (now.v + u * lanes) * VEC);
          g[u].load(dout + by_k.row(now.q) * c + (now.v + u * lanes) * VEC);
        }
      }
#pragma unroll
      for (int u = 0; u < U; ++u) {
        if (now.v + u * lanes >= cols) continue;
        if constexpr (kAsync) {
          r[u].raw = *reinterpret_cast<const typename Pack<T, VEC>::Raw*>(slot(stage, 0, u));
          g[u].raw = *reinterpret_cast<const typename Pack<T, VEC>::Raw*>(slot(stage, 1, u));
        }
        float a[VEC], b[VEC];
        g[u].get(a);
        r[u].get(b);
#pragma unroll
        for (int e = 0; e < VEC; ++e) {
          dot = fmaf(a[e], b[e], dot);
          a[e] *= f[0];
        }
        g[u].set(a);
        g[u].store(d0 + (now.v + u * lanes) * VEC);
      }
    } else if ((int64_t)pos[0] < pairs) {
      Pack<T, VEC> zero;
      zero.clear();
#pragma unroll
      for (int u = 0; u < U; ++u)
        if (now.v + u * lanes < cols) zero.store(d0 + (now.v + u * lanes) * VEC);
    }
    if (now.v - lane + lanes * U >= cols) {      // the choice's last step
      for (int o = lanes >> 1; o > 0; o >>= 1) dot += __shfl_down_sync(0xffffffffu, dot, o, lanes);
      if (lane == 0 && now.q < pairs) store_any(dw, w_dtype, now.q, dot);
      dot = 0.f;
    }
    advance(now);
#pragma unroll
    for (int d = 0; d < D; ++d) {
      pos[d] = pos[d + 1];
      f[d] = f[d + 1];
    }
    stage = stage + 1 == D ? 0 : stage + 1;
  }
  if constexpr (kAsync) async_wait<0>();
}

// threads of a row of `cols` vectors
int row_lanes(int64_t cols) {
  int lanes = 1;
  while (lanes < 32 && lanes < cols) lanes *= 2;
  return lanes;
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
  const size_t need = sort_plan(n, n_groups).bytes;
  if (workspace_bytes < need || (need && !workspace)) return TSB_ERR_WORKSPACE;
  const KeySource src{keys, stride, keys_are_i64, (unsigned)n_groups, -1};
  return run_sort(src, n, SortOut{order, inverse, nullptr, offsets}, workspace, st);
}

int tsb_embedding_fwd(const void* table, const void* tokens, int32_t tokens_are_i64, int64_t n, int64_t n_rows, int64_t c,
                      float scale, int32_t dtype, void* out, tsb_stream_t stream) {
  if (n < 0 || n_rows < 0 || c < 1 || (n && (!tokens || !out)) || (n && n_rows && !table)) return TSB_ERR_BAD_ARG;
  if (!good_dtype(dtype)) return TSB_ERR_UNSUPPORTED;
  if (n > kMaxRows || n_rows > kMaxRows || c > kMaxChannels) return TSB_ERR_LIMIT;
  if (n == 0) return TSB_OK;
  const KeySource src{tokens, 1, tokens_are_i64, (unsigned)n_rows, -1};
  const bool wide = (uintptr_t)out % 16 == 0;
  const int vec = vector_width(dtype, c, (uintptr_t)table | (wide ? 0 : (uintptr_t)out));
  const int64_t total = n * (c / vec);
  return dispatch_pack(dtype, vec, [&](auto tag) -> int {
    using T = typename decltype(tag)::T;
    constexpr int VEC = decltype(tag)::VEC, WIDE = 16 / (int)sizeof(T) / VEC;
    const auto run = [&](auto parts) -> int {
      constexpr int PARTS = decltype(parts)::value;
      const int64_t blocks = cdiv(cdiv(total, PARTS), kThreads * (PARTS > 4 ? 2 : 4));
      if (blocks > 0x7fffffff) return TSB_ERR_LIMIT;
      const unsigned cols = (unsigned)(c / VEC);
      embed_kernel<T, VEC, PARTS><<<(unsigned)blocks, kThreads, 0, as_stream(stream)>>>(
          (const T*)table, src, total, row_split(cols), TokenStep{kThreads * PARTS / cols, kThreads * PARTS % cols}, scale, (T*)out);
      TSB_LAUNCH_CHECK();
      return TSB_OK;
    };
    if (wide) return run(std::integral_constant<int, WIDE>());
    return run(std::integral_constant<int, 1>());
  });
}

size_t tsb_embedding_bwd_workspace_bytes(int64_t n, int64_t n_rows, int64_t c, int32_t dtype) {
  if (n < 1 || n_rows < 1 || c < 1 || n > kMaxRows || n_rows > kMaxRows || c > kMaxChannels || !good_dtype(dtype)) return 256;
  size_t partials = 0;      // of the vector width that leaves the most
  for (int vec = 1; vec <= 16 / (int)dtype_size(dtype); vec *= 2) {
    if (c % vec) continue;
    const size_t b = align_up((size_t)embed_plan(n, n_rows, c, vec).blocks * c * sizeof(float), 256);
    if (b > partials) partials = b;
  }
  return sort_plan(n, n_rows).bytes + 2 * align_up((size_t)n * 4, 256) + 2 * partials;
}

int tsb_embedding_bwd(const void* grad, const void* tokens, int32_t tokens_are_i64, int64_t n, int64_t n_rows, int64_t c,
                      float scale, int64_t padding_row, int32_t dtype, void* dtable, void* workspace, size_t workspace_bytes,
                      tsb_stream_t stream) {
  if (n < 0 || n_rows < 0 || c < 1 || (n && (!tokens || !grad)) || (n_rows && !dtable)) return TSB_ERR_BAD_ARG;
  if (!good_dtype(dtype)) return TSB_ERR_UNSUPPORTED;
  if (n > kMaxRows || n_rows > kMaxRows || c > kMaxChannels) return TSB_ERR_LIMIT;
  cudaStream_t st = as_stream(stream);
  if (n_rows == 0) return TSB_OK;
  if (n == 0) {
    TSB_CUDA_TRY(cudaMemsetAsync(dtable, 0, (size_t)n_rows * c * dtype_size(dtype), st));
    return TSB_OK;
  }
  if (!workspace || workspace_bytes < tsb_embedding_bwd_workspace_bytes(n, n_rows, c, dtype)) return TSB_ERR_WORKSPACE;
  const int vec = vector_width(dtype, c, (uintptr_t)grad | (uintptr_t)dtable);
  EmbedGrad a = embed_plan(n, n_rows, c, vec);
  const int zero_rows = c >= 256 ? 64 : 256;      // rows that a block looks up and clears
  const int64_t blocks = a.blocks + cdiv(n_rows, zero_rows);
  if (blocks > 0x7fffffff) return TSB_ERR_LIMIT;
  a.scale = scale;
  char* ws = static_cast<char*>(workspace) + sort_plan(n, n_rows).bytes;
  unsigned* keys = reinterpret_cast<unsigned*>(ws);
  ws += align_up((size_t)n * 4, 256);
  int* order = reinterpret_cast<int*>(ws);
  ws += align_up((size_t)n * 4, 256);
  a.keys = keys;
  a.order = order;
  a.head = reinterpret_cast<float*>(ws);
  a.tail = reinterpret_cast<float*>(ws + align_up((size_t)a.blocks * c * sizeof(float), 256));
  const KeySource src{tokens, 1, tokens_are_i64, (unsigned)n_rows, padding_row};
  const int sorted = run_sort(src, n, SortOut{order, nullptr, keys, nullptr}, workspace, st);
  if (sorted != TSB_OK) return sorted;
  return dispatch_pack(dtype, vec, [&](auto tag) -> int {
    using T = typename decltype(tag)::T;
    constexpr int VEC = decltype(tag)::VEC;
    const dim3 grid((unsigned)blocks, (unsigned)cdiv(c / VEC, a.tile));
    const int rc = launch_wide<embed_grad_kernel<T, VEC>, kGradBytes<T, VEC>>(grid, kThreads, st, a, (const T*)grad, (T*)dtable,
                                                                             zero_rows);
    if (rc != TSB_OK) return rc;
    if (a.blocks > 1) {
      const auto join = [&](int jv) { return dim3((unsigned)(a.blocks - 1), (unsigned)cdiv(c, kJoinColumns * jv)); };
      if (c % 4 == 0) embed_join_kernel<T, 4><<<join(4), kJoinThreads, 0, st>>>(a, (T*)dtable);
      else embed_join_kernel<T, 1><<<join(1), kJoinThreads, 0, st>>>(a, (T*)dtable);
      TSB_LAUNCH_CHECK();
    }
    return TSB_OK;
  });
}

int tsb_expert_dispatch(const void* x, const int32_t* inverse, const int32_t* kept, int64_t n, int32_t k, int64_t c,
                        int32_t dtype, void* xs, tsb_stream_t stream) {
  if (n < 0 || k < 1 || c < 1 || (n && (!x || !inverse || !kept || !xs))) return TSB_ERR_BAD_ARG;
  if (!good_dtype(dtype)) return TSB_ERR_UNSUPPORTED;
  if (n > kMaxRows / k || c > kMaxChannels) return TSB_ERR_LIMIT;
  if (n == 0) return TSB_OK;
  const int vec = vector_width(dtype, c, (uintptr_t)x | (uintptr_t)xs);
  const int64_t total = n * (c / vec), blocks = cdiv(total, kThreads * 2);
  if (blocks > 0x7fffffff) return TSB_ERR_LIMIT;
  return dispatch_pack(dtype, vec, [&](auto tag) -> int {
    using T = typename decltype(tag)::T;
    constexpr int VEC = decltype(tag)::VEC;
    dispatch_kernel<T, VEC><<<(unsigned)blocks, kThreads, 0, as_stream(stream)>>>((const T*)x, inverse, kept, total, n * k, k,
                                                                                  row_split(c / VEC), (T*)xs);
    TSB_LAUNCH_CHECK();
    return TSB_OK;
  });
}

int tsb_expert_combine(const void* rows, const void* weights, int32_t weights_dtype, const int32_t* inverse, const int32_t* kept,
                       int64_t n, int32_t k, int64_t c, int32_t dtype, void* out, tsb_stream_t stream) {
  if (n < 0 || k < 1 || c < 1 || (n && (!rows || !inverse || !kept || !out))) return TSB_ERR_BAD_ARG;
  if (!good_dtype(dtype) || (weights && !good_dtype(weights_dtype))) return TSB_ERR_UNSUPPORTED;
  if (n > kMaxRows / k || c > kMaxChannels) return TSB_ERR_LIMIT;
  if (n == 0) return TSB_OK;
  const int vec = vector_width(dtype, c, (uintptr_t)rows | (uintptr_t)out);
  // choices of a step: as few steps as four at once need, evenly filled; threads of a row: as many as its vectors need
  const int ku = (int)cdiv(k, cdiv(k, 4)), u = step_vectors(vec * (int)dtype_size(dtype)) / ku;
  const int64_t vecs = c / vec;
  const int lanes = (int)cdiv(vecs, u * cdiv(vecs, kThreads * u));
  const int64_t want = cdiv(n, kThreads / lanes);
  return dispatch_pack(dtype, vec, [&](auto tag) -> int {
    using T = typename decltype(tag)::T;
    constexpr int VEC = decltype(tag)::VEC, BYTES = step_bytes(Pack<T, VEC>::kBytes);
    const int64_t most = row_blocks(Pack<T, VEC>::kBytes);
    const dim3 grid((unsigned)(want < most ? want : most));
    const auto run = [&](auto choices) -> int {
      return launch_wide<combine_kernel<T, VEC, decltype(choices)::value>, BYTES>(grid, kThreads, as_stream(stream), (const T*)rows,
                                                                                 weights, weights_dtype, inverse, kept, n, k, c, lanes,
                                                                                 (T*)out);
    };
    switch (ku) {
      case 1: return run(std::integral_constant<int, 1>());
      case 2: return run(std::integral_constant<int, 2>());
      case 3: return run(std::integral_constant<int, 3>());
      default: return run(std::integral_constant<int, 4>());
    }
  });
}

int tsb_expert_combine_bwd(const void* dout, const void* rows, const void* weights, int32_t weights_dtype,
                           const int32_t* inverse, const int32_t* kept, int64_t n, int32_t k, int64_t c, int32_t dtype,
                           void* drows, void* dweights, tsb_stream_t stream) {
  if (n < 0 || k < 1 || c < 1 || (n && (!dout || !rows || !weights || !inverse || !kept || !drows || !dweights)))
    return TSB_ERR_BAD_ARG;
  if (!good_dtype(dtype) || !good_dtype(weights_dtype)) return TSB_ERR_UNSUPPORTED;
  if (n > kMaxRows / k || c > kMaxChannels) return TSB_ERR_LIMIT;
  if (n == 0) return TSB_OK;
  const int vec = vector_width(dtype, c, (uintptr_t)dout | (uintptr_t)rows | (uintptr_t)drows);
  const int lanes = row_lanes(c / vec);
  const int64_t want = cdiv(n * k * lanes, kThreads);
  return dispatch_pack(dtype, vec, [&](auto tag) -> int {
    using T = typename decltype(tag)::T;
    constexpr int VEC = decltype(tag)::VEC, BYTES = step_bytes(Pack<T, VEC>::kBytes);
    const int64_t most = row_blocks(Pack<T, VEC>::kBytes);
    return launch_wide<combine_grad_kernel<T, VEC>, BYTES>(dim3((unsigned)(want < most ? want : most)), kThreads, as_stream(stream),
                                                           (const T*)dout, (const T*)rows, weights, weights_dtype, inverse, kept,
                                                           n * k, row_split(k), c, lanes, (T*)drows, dweights);
  });
}

}  // extern "C"
