// Group normalisation with an activation over rows grouped by sample, channels last.
//
//   mean, var   over the rows of a sample and the d = c / g channels of a group
//   y = act(z), z = (x - mean) * rstd * w + b
//   dz = dy * act'(z);  db = sum dz;  dw = sum dz * xhat;  dx = rstd * (dz * w - m1 - xhat * m2) with m1 and m2 the
//   means of dz * w and dz * w * xhat over the sample and group
//
// Rows are walked in grouped order in `nblk` equal chunks, one block each.  Where a chunk meets sample s its partial
// sums go to slot (block + s): both only grow along the rows, so every meeting has a slot of its own, and there are
// nblk + samples of them however ragged the samples are.  A second kernel joins the slots of each sample in order,
// a third one walks the rows again.  No atomics: the sums do not depend on the order in which blocks run.
//
// Variances are joined from means and sums of squares about them, piece by piece, never as a difference of two large
// sums, in 32 bits; y and dx are rounded to the type of the features once.  Small inputs take one block per sample and
// group instead (norm_small).
#include <type_traits>

#include "rows.cuh"

namespace tsb {
namespace {

constexpr int kNormThreads = 256;
constexpr int kNormWarps = kNormThreads / 32;
constexpr int kNormBlocks = 3 * kSmCount;      // three blocks of 256 threads and up to 80 registers are resident on an SM
enum { kActNone = 0, kActRelu = 1, kActLeaky = 2, kActSilu = 3 };

struct Norm {
  int64_t n;             // rows
  int c, g, d;           // channels, groups, channels of a group
  int b;                 // samples
  int cols;              // vectors of a row
  int tile;              // vectors of a row that one block takes (grid.y tiles)
  int64_t chunk;         // rows of a block
  int nblk;
  const int* order;      // row at a grouped position, or null: the rows are grouped already
  const int* offsets;    // [b + 1]
  const void *w, *bias;  // [c] of p_dtype, or null
  int p_dtype;
  float eps, slope;
  int act;
};

__device__ __forceinline__ int64_t offset_of(const Norm& a, int s) {
  const int64_t v = __ldg(a.offsets + s);
  return v < 0 ? 0 : v > a.n ? a.n : v;
}

// chunk of a position: both are below 2^31
__device__ __forceinline__ int chunk_of(const Norm& a, int64_t p) { return (int)((unsigned)p / (unsigned)a.chunk); }

// First sample that ends behind position p (a.b: none).  The whole warp searches: up to 128 samples cost one round trip.
__device__ __forceinline__ int first_sample(const Norm& a, int64_t p) {
  const int lane = threadIdx.x & 31;
  int lo = 0, hi = a.b;      // samples before lo end at or before p; sample hi (if any) ends behind it
  while (hi - lo > 128) {
    const int step = (hi - lo + 31) / 32, at = lo + (lane + 1) * step - 1;
    const bool before = at < hi && offset_of(a, at + 1) <= p;
    const int k = __popc(__ballot_sync(0xffffffffu, before));
    hi = min(hi, lo + (k + 1) * step - 1);
    lo += k * step;
  }
  bool before[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) before[i] = lo + lane + 32 * i < hi && offset_of(a, lo + lane + 32 * i + 1) <= p;
  int k = 0;
#pragma unroll
  for (int i = 0; i < 4; ++i) k += __popc(__ballot_sync(0xffffffffu, before[i]));
  return lo + k;
}

// Row at a grouped position; -1 for an entry of a caller's order that is no row.
template <bool ORDERED>
__device__ __forceinline__ int64_t row_at(const Norm& a, int64_t p) {
  if constexpr (!ORDERED) return p;
  const int64_t r = __ldg(a.order + p);
  return r >= 0 && r < a.n ? r : -1;
}

// The `count` rows p, p + step, .. of a thread, U at a time: f(v, at, full) with v[i][u] the vector of array i in row u and
// at[u] the row's offset, which is -1 for a row that is not there unless `full` says that all are.
//
// Vectors of 4 bytes and more come through shared memory by cp.async, each thread filling and reading slots of its own: three
// batches are on their way without holding registers, nothing waits for another thread, and the order and the borders of
// the samples do not matter.  Single 16-bit values are loaded directly.
constexpr int kPipeDepth = 3;
template <typename T, int VEC>
constexpr int kBatch = VEC * sizeof(T) == 16 ? 4 : 8;      // vectors of a batch, of one array or two
template <typename T, int VEC>
constexpr int kPipeBytes = kAsyncVector<T, VEC> ? kPipeDepth * kBatch<T, VEC> * kNormThreads * VEC * (int)sizeof(T) : 0;

template <typename T, int VEC, int ARRAYS, int U, bool ORDERED, typename F>
__device__ __forceinline__ void for_rows(const Norm& a, const T* const (&src)[ARRAYS], int64_t p, int step, int count,
                                         unsigned char* pipe, F&& f) {
  const int64_t pitch = (int64_t)step * a.c;
  int64_t off = p * a.c;      // of row k where the rows lie in order
  const auto offset = [&](int k, int u, int64_t base) -> int64_t {
    if (k + u >= count) return -1;
    if constexpr (ORDERED) {
      const int64_t r = row_at<true>(a, p + (int64_t)(k + u) * step);
      return r < 0 ? -1 : r * a.c;
    }
    return base + u * pitch;
  };
  if constexpr (kAsyncVector<T, VEC>) {
    constexpr int kBytes = Pack<T, VEC>::kBytes, kStage = ARRAYS * U * kNormThreads * kBytes;
    unsigned char* mine = pipe + threadIdx.x * kBytes;
    const auto copy = [&](int stage, int u, int64_t at) {
#pragma unroll
      for (int i = 0; i < ARRAYS; ++i) async_copy<kBytes>(mine + stage * kStage + (u * ARRAYS + i) * kNormThreads * kBytes, src[i] + at);
    };
    const auto issue = [&](int stage, int k, int64_t base) {
      if (!ORDERED && k + U <= count) {
#pragma unroll
        for (int u = 0; u < U; ++u) copy(stage, u, base + u * pitch);
      } else {
#pragma unroll
        for (int u = 0; u < U; ++u) {
          const int64_t at = offset(k, u, base);
          if (at >= 0) copy(stage, u, at);
        }
      }
      async_commit();      // an empty group where nothing was left to read
    };
    constexpr int kAhead = (kPipeDepth - 1) * U;
#pragma unroll
    for (int d = 0; d < kPipeDepth - 1; ++d) issue(d, d * U, off + d * U * pitch);
    int stage = 0;
    for (int k = 0; k < count; k += U, off += U * pitch) {
      issue(stage == 0 ? kPipeDepth - 1 : stage - 1, k + kAhead, off + kAhead * pitch);
      async_wait<kPipeDepth - 1>();
      Pack<T, VEC> v[ARRAYS][U];
      int64_t at[U];
#pragma unroll
      for (int u = 0; u < U; ++u)
#pragma unroll
        for (int i = 0; i < ARRAYS; ++i)
          v[i][u].raw =
              *reinterpret_cast<const typename Pack<T, VEC>::Raw*>(mine + stage * kStage + (u * ARRAYS + i) * kNormThreads * kBytes);
      if (!ORDERED && k + U <= count) {
#pragma unroll
        for (int u = 0; u < U; ++u) at[u] = off + u * pitch;
        f(v, at, std::true_type());
      } else {
#pragma unroll
        for (int u = 0; u < U; ++u) at[u] = offset(k, u, off);
        f(v, at, std::false_type());
      }
      stage = stage + 1 == kPipeDepth ? 0 : stage + 1;
    }
    async_wait<0>();
  } else {
    for (int k = 0; k < count; k += U, off += U * pitch) {
      Pack<T, VEC> v[ARRAYS][U];
      int64_t at[U];
#pragma unroll
      for (int u = 0; u < U; ++u) {
        at[u] = offset(k, u, off);
#pragma unroll
        for (int i = 0; i < ARRAYS; ++i)
          if (at[u] >= 0) v[i][u].load(src[i] + at[u]);
      }
      f(v, at, std::false_type());
    }
  }
}

// Two values at once: the packed 32-bit instructions halve what the arithmetic takes of the issue slots.  Each rounds as
// its scalar form does.
__device__ __forceinline__ void fma2(float& x, float& y, float a, float b, float c, float d, float e, float f) {
  asm("{.reg .b64 p, q, r; mov.b64 p, {%2, %3}; mov.b64 q, {%4, %5}; mov.b64 r, {%6, %7}; fma.rn.f32x2 p, p, q, r; mov.b64 {%0, %1}, p;}"
      : "=f"(x), "=f"(y) : "f"(a), "f"(b), "f"(c), "f"(d), "f"(e), "f"(f));
}
__device__ __forceinline__ void add2(float& x, float& y, float a, float b, float c, float d) {
  asm("{.reg .b64 p, q; mov.b64 p, {%2, %3}; mov.b64 q, {%4, %5}; add.rn.f32x2 p, p, q; mov.b64 {%0, %1}, p;}"
      : "=f"(x), "=f"(y) : "f"(a), "f"(b), "f"(c), "f"(d));
}
__device__ __forceinline__ void mul2(float& x, float& y, float a, float b, float c, float d) {
  asm("{.reg .b64 p, q; mov.b64 p, {%2, %3}; mov.b64 q, {%4, %5}; mul.rn.f32x2 p, p, q; mov.b64 {%0, %1}, p;}"
      : "=f"(x), "=f"(y) : "f"(a), "f"(b), "f"(c), "f"(d));
}
// r[e] = x[e] * y[j(e)] + z[l(e)] and the like over VEC values; the indices let a group's value stand for several channels
template <int N, typename Y, typename Z>
__device__ __forceinline__ void fma_all(float (&r)[N], const float (&x)[N], Y&& y, Z&& z) {
  if constexpr (N == 1) {
    r[0] = fmaf(x[0], y(0), z(0));
  } else {
#pragma unroll
    for (int e = 0; e < N; e += 2) fma2(r[e], r[e + 1], x[e], x[e + 1], y(e), y(e + 1), z(e), z(e + 1));
  }
}
template <int N, typename Y>
__device__ __forceinline__ void add_all(float (&r)[N], const float (&x)[N], Y&& y) {
  if constexpr (N == 1) {
    r[0] = x[0] + y(0);
  } else {
#pragma unroll
    for (int e = 0; e < N; e += 2) add2(r[e], r[e + 1], x[e], x[e + 1], y(e), y(e + 1));
  }
}
template <int N, typename Y>
__device__ __forceinline__ void mul_all(float (&r)[N], const float (&x)[N], Y&& y) {
  if constexpr (N == 1) {
    r[0] = x[0] * y(0);
  } else {
#pragma unroll
    for (int e = 0; e < N; e += 2) mul2(r[e], r[e + 1], x[e], x[e + 1], y(e), y(e + 1));
  }
}

// 1 / (1 + 2^(-z log2 e)) with the hardware's exponential and reciprocal, each good to 2^-22: half the instructions of the
// library's forms, which also serve subnormal arguments (here 2^x below 2^-126 vanishes beside the 1, and beyond 2^126
// the quotient is below 2^-126 and becomes zero).
template <int N>
__device__ __forceinline__ void sigmoid(float (&p)[N], const float (&z)[N]) {
  mul_all(p, z, [](int) { return -1.4426950408889634f; });
#pragma unroll
  for (int e = 0; e < N; ++e) asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(p[e]) : "f"(p[e]));
  add_all(p, p, [](int) { return 1.f; });
#pragma unroll
  for (int e = 0; e < N; ++e) asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(p[e]) : "f"(p[e]));
}

template <int N>
__device__ __forceinline__ void activate(float (&z)[N], int act, float slope) {
  if (act == kActRelu) {
#pragma unroll
    for (int i = 0; i < N; ++i) z[i] = z[i] < 0.f ? 0.f : z[i];      // a NaN stays one
  } else if (act == kActLeaky) {
#pragma unroll
    for (int i = 0; i < N; ++i) z[i] = z[i] > 0.f ? z[i] : z[i] * slope;
  } else if (act == kActSilu) {
    float p[N];
    sigmoid(p, z);
    mul_all(z, z, [&](int i) { return p[i]; });
  }
}

// g *= act'(z)
template <int N>
__device__ __forceinline__ void activate_grad(const float (&z)[N], float (&g)[N], int act, float slope) {
  if (act == kActRelu) {
#pragma unroll
    for (int i = 0; i < N; ++i) g[i] = z[i] > 0.f ? g[i] : 0.f;
  } else if (act == kActLeaky) {
#pragma unroll
    for (int i = 0; i < N; ++i) g[i] = z[i] > 0.f ? g[i] : g[i] * slope;
  } else if (act == kActSilu) {
    float p[N], q[N], r[N];      // act' = z p (1 - p) + p
    sigmoid(p, z);
    mul_all(q, z, [&](int i) { return p[i]; });
    fma_all(r, p, [](int) { return -1.f; }, [](int) { return 1.f; });
    fma_all(q, q, [&](int i) { return r[i]; }, [&](int i) { return p[i]; });
    mul_all(g, g, [&](int i) { return q[i]; });
  }
}

// sum over `width` neighbouring lanes, a power of two
__device__ __forceinline__ float warp_sum(float v, int width = 32) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1)
    if (o < width) v += __shfl_down_sync(0xffffffffu, v, o, width);
  return __shfl_sync(0xffffffffu, v, 0, width);
}

// rows that lane l of `lanes` takes of `rows`; one division for all lanes
struct LaneRows {
  int each, more;
  __device__ __forceinline__ LaneRows(int64_t rows, int lanes) {
    each = (int)((unsigned)rows / (unsigned)lanes);      // a chunk has fewer than 2^31 rows
    more = (int)rows - each * lanes;
  }
  __device__ __forceinline__ int of(int l) const { return each + (l < more); }
};

// channels of group gr that column tile y holds
__device__ __forceinline__ int tile_channels(const Norm& a, int vec, int y, int gr) {
  const int lo = max(y * a.tile * vec, gr * a.d), hi = min(min((y + 1) * a.tile * vec, a.c), (gr + 1) * a.d);
  return max(hi - lo, 0);
}

// ------------------------------------------------------------------------------------------------ statistics
// The mean and the sum of squares about it of the values that a thread has seen: one pair where a vector lies in one
// group (A == 1), one pair per channel otherwise (A == VEC).
template <int VEC, int A>
struct Running {
  static constexpr int W = VEC / A;
  float n, mean[A], m2[A];
  __device__ __forceinline__ void clear() {
    n = 0.f;
#pragma unroll
    for (int i = 0; i < A; ++i) mean[i] = m2[i] = 0.f;
  }
  // U vectors at once: their own mean and squares are exact to rounding and are joined to the running pair
  template <typename T, int U>
  __device__ __forceinline__ void add(const Pack<T, VEC> (&v)[U]) {
    constexpr float kCount = (float)(U * W), kInv = 1.f / kCount;      // W values of a vector share a pair
    float f[U][VEC], chan[VEC], sum[A], sq[A];
#pragma unroll
    for (int u = 0; u < U; ++u) v[u].get(f[u]);
    const auto gather = [&](float (&to)[A]) {      // the channels of a pair
#pragma unroll
      for (int i = 0; i < A; ++i) {
        to[i] = chan[i * W];
#pragma unroll
        for (int e = 1; e < W; ++e) to[i] += chan[i * W + e];
      }
    };
#pragma unroll
    for (int e = 0; e < VEC; ++e) chan[e] = f[0][e];
#pragma unroll
    for (int u = 1; u < U; ++u) add_all(chan, chan, [&](int e) { return f[u][e]; });
    gather(sum);
#pragma unroll
    for (int i = 0; i < A; ++i) sum[i] *= kInv;
#pragma unroll
    for (int e = 0; e < VEC; ++e) chan[e] = 0.f;
#pragma unroll
    for (int u = 0; u < U; ++u) {
      add_all(f[u], f[u], [&](int e) { return -sum[e / W]; });
      fma_all(chan, f[u], [&](int e) { return f[u][e]; }, [&](int e) { return chan[e]; });
    }
    gather(sq);
    const float all = n + kCount, share = __fdividef(kCount, all), cross = n * share;
#pragma unroll
    for (int i = 0; i < A; ++i) {
      const float t = sum[i] - mean[i];
      mean[i] = fmaf(t, share, mean[i]);
      m2[i] += fmaf(t * t, cross, sq[i]);
    }
    n = all;
  }
};

// One read of x.  1M x 64 bf16: 33 us, 3.9 TB/s, where the copy rate takes 20; 61441 x 96 bf16, which the L2 cache holds: 9
// us.  Some 5 us are the start of a block (its samples, the first rows) and the join at its end: twice as many blocks of
// half the rows took 36 us, three times as many 41.  For the other 8 the counters name no one limit: memory is 52 % busy, 0.59
// instructions issue per cycle, and a warp's first stall is the wait for its rows.
template <typename T, int VEC, int A, bool ORDERED>
__global__ void __launch_bounds__(kNormThreads, 3) norm_stats_kernel(Norm a, const T* __restrict__ x, float2* __restrict__ slots) {
  extern __shared__ __align__(16) unsigned char pipe[];
  __shared__ float2 part[A * kNormThreads];
  const int first = blockIdx.y * a.tile, width = min(a.tile, a.cols - first);
  const int lane = threadIdx.x / width, col = threadIdx.x - lane * width;
  const int lanes = kNormThreads / width;
  const int64_t p0 = blockIdx.x * a.chunk, p1 = min(p0 + a.chunk, a.n);
  const T* xc = x + (int64_t)(first + col) * VEC;
  for (int s = first_sample(a, p0); s < a.b; ++s) {
    const int64_t begin = offset_of(a, s);
    if (begin >= p1) break;
    const int64_t lo = max(p0, begin), hi = min(p1, offset_of(a, s + 1));
    if (lo >= hi) continue;
    if (lane < lanes) {
      constexpr int U = kBatch<T, VEC>;
      Running<VEC, A> run;
      run.clear();
      const T* const src[1] = {xc};
      const int count = LaneRows(hi - lo, lanes).of(lane);
      int left = count;
      for_rows<T, VEC, 1, U, ORDERED>(a, src, lo + lane, lanes, count, pipe, [&](auto& v, const auto& at, auto) {
        if constexpr (ORDERED) {
#pragma unroll
          for (int u = 0; u < U; ++u)
            if (at[u] < 0) v[0][u].clear();      // an entry of the order that is no row
        }
        if (left >= U) {
          run.add(v[0]);
        } else {
#pragma unroll
          for (int u = 0; u < U; ++u) {
            const Pack<T, VEC> one[1] = {v[0][u]};
            if (u < left) run.add(one);
          }
        }
        left -= U;
      });
#pragma unroll
      for (int i = 0; i < A; ++i) part[i * kNormThreads + threadIdx.x] = make_float2(run.mean[i], run.m2[i]);
    }
    __syncthreads();
    // `sub` lanes per group of this column tile, a power of two up to a warp
    const int c_lo = first * VEC, c_hi = (first + width) * VEC;
    const int g_lo = c_lo / a.d, g_hi = (c_hi - 1) / a.d;
    const LaneRows rows(hi - lo, lanes);
    float2* slot = slots + ((int64_t)blockIdx.y * (a.nblk + a.b) + blockIdx.x + s) * a.g;
    const int most = lanes * (min(a.d, c_hi - c_lo) / (VEC / A)), lg = most >= 32 ? 5 : 32 - __clz(most - 1);
    const int sub = 1 << lg, side = 32 >> lg, in = threadIdx.x & (sub - 1);
    for (int g0 = g_lo + (threadIdx.x >> 5) * side; g0 <= g_hi; g0 += kNormWarps * side) {      // the same for a warp
      const int gr = g0 + ((threadIdx.x & 31) >> lg);
      const int k_lo = max(gr * a.d, c_lo), k_hi = min((gr + 1) * a.d, c_hi);
      const int per_lane = (k_hi - k_lo) / (VEC / A), entries = gr <= g_hi ? per_lane * lanes : 0;
      float w = 0.f, m = 0.f, q = 0.f;
      for (int pass = 0; pass < 2; ++pass) {      // the joint mean, then the squares about it
        float acc = 0.f;
        for (int t = in; t < entries; t += sub) {
          const int l = per_lane == 1 ? t : (int)((unsigned)t / (unsigned)per_lane);
          const int k = k_lo + (t - l * per_lane) * (VEC / A) - c_lo;
          const float cnt = (float)(rows.of(l) * (VEC / A));
          if (cnt == 0.f) continue;
          const float2 e = part[k % VEC / (VEC / A) * kNormThreads + l * width + k / VEC];
          if (pass == 0) {
            w += cnt;
            acc = fmaf(cnt, e.x, acc);
          } else {
            acc += fmaf(cnt * (e.x - m), e.x - m, e.y);
          }
        }
        acc = warp_sum(acc, sub);
        if (pass == 0) {
          w = warp_sum(w, sub);
          m = acc / w;
        } else {
          q = acc;
        }
      }
      if (in == 0 && gr <= g_hi) slot[gr] = make_float2(m, q);
    }
    __syncthreads();
  }
}

// One warp per sample and group: the slots of the sample, joined in the order of the rows.
__global__ void __launch_bounds__(128) norm_join_kernel(Norm a, int vec, int tiles, const float2* __restrict__ slots,
                                                        float* __restrict__ mean, float* __restrict__ rstd) {
  const int lane = threadIdx.x & 31;
  for (int64_t t = blockIdx.x * 4 + (threadIdx.x >> 5); t < (int64_t)a.b * a.g; t += (int64_t)gridDim.x * 4) {
    const int s = (int)((unsigned)t / (unsigned)a.g), gr = (int)t - s * a.g;
    const int64_t begin = offset_of(a, s), end = offset_of(a, s + 1);
    float w = 0.f, m = 0.f, q = 0.f;
    if (begin < end) {
      const int j0 = chunk_of(a, begin), j1 = chunk_of(a, end - 1);
      for (int pass = 0; pass < 2; ++pass) {
        float acc = 0.f;
        for (int y = 0; y < tiles; ++y) {
          const int width = tile_channels(a, vec, y, gr);
          if (width == 0) continue;
          const float2* at = slots + ((int64_t)y * (a.nblk + a.b) + s) * a.g + gr;
#pragma unroll 4
          for (int j = j0 + lane; j <= j1; j += 32) {
            const float cnt = (float)(min(end, (j + 1) * a.chunk) - max(begin, j * a.chunk)) * width;
            const float2 e = at[(int64_t)j * a.g];
            if (pass == 0) {
              w += cnt;
              acc = fmaf(cnt, e.x, acc);
            } else {
              acc += fmaf(cnt * (e.x - m), e.x - m, e.y);
            }
          }
        }
        acc = warp_sum(acc);
        if (pass == 0) {
          w = warp_sum(w);
          m = acc / w;
        } else {
          q = acc / w;
        }
      }
    }
    if (lane == 0) {
      mean[t] = m;
      rstd[t] = 1.f / sqrtf(q + a.eps);
    }
  }
}

// What a thread needs of its VEC channels within one sample: z = (x + away) * a + b with away = -mean, a = rstd * w.
template <int VEC, int A>
struct Channels {
  static constexpr int W = VEC / A;
  float away[A], a[VEC], b[VEC];
  __device__ __forceinline__ void load(const Norm& n, int s, int k0, const float* __restrict__ mean_, const float* __restrict__ rstd_) {
#pragma unroll
    for (int i = 0; i < A; ++i) away[i] = -__ldg(mean_ + (int64_t)s * n.g + (k0 + i * W) / n.d);
#pragma unroll
    for (int e = 0; e < VEC; ++e) {
      a[e] = __ldg(rstd_ + (int64_t)s * n.g + (k0 + e / W * W) / n.d) * (n.w ? load_any(n.w, n.p_dtype, k0 + e) : 1.f);
      b[e] = n.bias ? load_any(n.bias, n.p_dtype, k0 + e) : 0.f;
    }
  }
  __device__ __forceinline__ void center(float (&x)[VEC]) const {
    add_all(x, x, [&](int e) { return away[e / W]; });
  }
  __device__ __forceinline__ void affine(float (&z)[VEC], const float (&x)[VEC]) const {
    fma_all(z, x, [&](int e) { return a[e]; }, [&](int e) { return b[e]; });
  }
};

// Zeros in the rows of the block's chunk that belong to no sample.
template <typename T, int VEC, bool ORDERED>
__device__ __forceinline__ void clear_outside(const Norm& a, int64_t p0, int64_t p1, int lane, int lanes, T* __restrict__ out) {
  const int64_t begin = a.b ? offset_of(a, 0) : a.n, end = a.b ? offset_of(a, a.b) : a.n;
  if (begin <= p0 && end >= p1) return;
  Pack<T, VEC> zero;
  zero.clear();
  for (int64_t p = p0 + lane; p < p1; p += lanes) {
    if (p >= begin && p < end) continue;
    const int64_t r = row_at<ORDERED>(a, p);
    if (r >= 0) zero.store(out + r * a.c);
  }
}

// The rows are walked from the end of the chunk to its beginning: what the statistics read last is still in the L2 cache.  Of x
// 33 MB of 77 are read from memory a second time (400003 x 96 fp16), 85 of 128 (1M x 64 bf16).  The latter with SiLU: 42
// us, where 213 MB take 33 at the copy rate; shared loads and the special functions share a queue (MIO throttle).
template <typename T, int VEC, int A, bool ORDERED>
__global__ void __launch_bounds__(kNormThreads, 3) norm_apply_kernel(Norm a, const T* __restrict__ x, const float* __restrict__ mean,
                                                                     const float* __restrict__ rstd, T* __restrict__ y) {
  constexpr int U = kBatch<T, VEC>, W = VEC / A;
  extern __shared__ __align__(16) unsigned char pipe[];
  const int first = blockIdx.y * a.tile, width = min(a.tile, a.cols - first);
  const int lane = threadIdx.x / width, lanes = kNormThreads / width;
  const int k0 = (first + threadIdx.x - lane * width) * VEC;
  const int64_t p0 = blockIdx.x * a.chunk, p1 = min(p0 + a.chunk, a.n);
  const T* xc = x + k0;
  T* yc = y + k0;
  const int last = min(first_sample(a, p1 - 1), a.b - 1);
  if (lane >= lanes) return;
  clear_outside<T, VEC, ORDERED>(a, p0, p1, lane, lanes, yc);
  for (int s = last; s >= 0; --s) {
    const int64_t end = offset_of(a, s + 1);
    if (end <= p0) break;
    const int64_t lo = max(p0, offset_of(a, s)), hi = min(p1, end);
    if (lo >= hi) continue;
    Channels<VEC, A> ch;
    ch.load(a, s, k0, mean, rstd);
    const T* const src[1] = {xc};
    for_rows<T, VEC, 1, U, ORDERED>(a, src, hi - 1 - lane, -lanes, LaneRows(hi - lo, lanes).of(lane), pipe,
                                    [&](auto& v, const auto& at, auto full) {
#pragma unroll
      for (int u = 0; u < U; ++u) {
        if (!decltype(full)::value && at[u] < 0) continue;
        float z[VEC];
        v[0][u].get(z);
        ch.center(z);
        ch.affine(z, z);
        activate(z, a.act, a.slope);
        v[0][u].set(z);
        v[0][u].store(yc + at[u]);
      }
    });
  }
}

// ------------------------------------------------------------------------------------------------ gradient
// Per slot and channel: the sums of dz and of dz * xhat.  1M x 64 bf16 with SiLU: 58 us for 256 MB (39 at the copy rate):
// bound by the chain from x to the sums (exponential, reciprocal) in the 24 warps that the registers allow; two blocks of
// more registers took 55 us here and 34 instead of 33 for 150011 x 128 fp32.
template <typename T, int VEC, int A, bool ORDERED>
__global__ void __launch_bounds__(kNormThreads, 3) norm_grad_sums_kernel(Norm a, const T* __restrict__ x, const T* __restrict__ dy,
                                                                         const float* __restrict__ mean,
                                                                         const float* __restrict__ rstd, float2* __restrict__ slots) {
  constexpr int U = kBatch<T, VEC> / 2, W = VEC / A;
  extern __shared__ __align__(16) unsigned char pipe[];
  __shared__ float2 part[VEC * kNormThreads];
  const int first = blockIdx.y * a.tile, width = min(a.tile, a.cols - first);
  const int lane = threadIdx.x / width, lanes = kNormThreads / width, col = threadIdx.x - lane * width;
  const int k0 = (first + col) * VEC;
  const int64_t p0 = blockIdx.x * a.chunk, p1 = min(p0 + a.chunk, a.n);
  const T *xc = x + k0, *gc = dy + k0;
  for (int s = first_sample(a, p0); s < a.b; ++s) {
    const int64_t begin = offset_of(a, s);
    if (begin >= p1) break;
    const int64_t lo = max(p0, begin), hi = min(p1, offset_of(a, s + 1));
    if (lo >= hi) continue;
    if (lane < lanes) {
      float s1[VEC], s2[VEC];
#pragma unroll
      for (int e = 0; e < VEC; ++e) s1[e] = s2[e] = 0.f;
      Channels<VEC, A> ch;
      ch.load(a, s, k0, mean, rstd);
      const T* const src[2] = {xc, gc};
      for_rows<T, VEC, 2, U, ORDERED>(a, src, lo + lane, lanes, LaneRows(hi - lo, lanes).of(lane), pipe,
                                      [&](auto& v, const auto& at, auto full) {
#pragma unroll
        for (int u = 0; u < U; ++u) {
          if (!decltype(full)::value && at[u] < 0) continue;
          float h[VEC], z[VEC], g[VEC];
          v[0][u].get(h);
          v[1][u].get(g);
          ch.center(h);
          ch.affine(z, h);
          activate_grad(z, g, a.act, a.slope);
          add_all(s1, s1, [&](int e) { return g[e]; });
          fma_all(s2, g, [&](int e) { return h[e]; }, [&](int e) { return s2[e]; });
        }
      });
#pragma unroll
      for (int e = 0; e < VEC; ++e) part[e * kNormThreads + threadIdx.x] = make_float2(s1[e], s2[e]);
    }
    __syncthreads();
    float2* slot = slots + ((int64_t)blockIdx.x + s) * a.c;
    for (int t = threadIdx.x; t < width * VEC; t += kNormThreads) {
      const int e = t / width, q = t - e * width, k = (first + q) * VEC + e;
      const float scale = __ldg(rstd + (int64_t)s * a.g + k / a.d);
      float u = 0.f, v = 0.f;
#pragma unroll 8
      for (int l = 0; l < lanes; ++l) {
        const float2 f = part[e * kNormThreads + l * width + q];
        u += f.x;
        v += f.y;
      }
      slot[k] = make_float2(u, v * scale);
    }
    __syncthreads();
  }
}

// One block per sample and group: the sums of its channels over the slots, and the two means that dx needs.
// Where there are fewer blocks than SMs they are twice as large: 16 blocks over 222 slots of 12 channels took 6.7 us with
// 256 threads, 4.9 with 512; they wait for memory.
constexpr int kJoinThreads = 512;
__global__ void __launch_bounds__(kJoinThreads) norm_grad_join_kernel(Norm a, const float2* __restrict__ slots,
                                                                      float2* __restrict__ by_channel, float2* __restrict__ by_group) {
  __shared__ float2 part[kJoinThreads];
  const int width = min(a.d, (int)blockDim.x), lanes = blockDim.x / width;
  const int lane = threadIdx.x / width, q = threadIdx.x - lane * width;
  for (int64_t t = blockIdx.x; t < (int64_t)a.b * a.g; t += gridDim.x) {
    const int s = (int)((unsigned)t / (unsigned)a.g), gr = (int)t - s * a.g;
    const int64_t begin = offset_of(a, s), end = offset_of(a, s + 1);
    float m1 = 0.f, m2 = 0.f;
    for (int k = q; k - q < a.d; k += width) {
      const float w = a.w && k < a.d ? load_any(a.w, a.p_dtype, gr * a.d + k) : 1.f;
      float u = 0.f, v = 0.f;
      if (lane < lanes && k < a.d && begin < end) {
        const int j0 = chunk_of(a, begin), j1 = chunk_of(a, end - 1);
#pragma unroll 8
        for (int j = j0 + lane; j <= j1; j += lanes) {
          const float2 f = slots[((int64_t)j + s) * a.c + gr * a.d + k];
          u += f.x;
          v += f.y;
        }
      }
      part[threadIdx.x] = make_float2(u, v);
      __syncthreads();
      for (int half = lanes; half > 1;) {      // the upper half of the lanes onto the lower
        const int keep = (half + 1) / 2;
        if (lane + keep < half) {
          u += part[threadIdx.x + keep * width].x;
          v += part[threadIdx.x + keep * width].y;
          part[threadIdx.x] = make_float2(u, v);
        }
        half = keep;
        __syncthreads();
      }
      if (lane == 0 && k < a.d) {
        const int ch = gr * a.d + k;
        by_channel[(int64_t)s * a.c + ch] = make_float2(u, v);
        m1 = fmaf(w, u, m1);
        m2 = fmaf(w, v, m2);
      }
      __syncthreads();
    }
    part[threadIdx.x] = lane == 0 ? make_float2(m1, m2) : make_float2(0.f, 0.f);
    __syncthreads();
    if (threadIdx.x < 32) {
      float u = 0.f, v = 0.f;
      for (int i = threadIdx.x; i < width; i += 32) {
        u += part[i].x;
        v += part[i].y;
      }
      u = warp_sum(u);
      v = warp_sum(v);
      const float inv = begin < end ? 1.f / ((float)(end - begin) * a.d) : 0.f;
      if (threadIdx.x == 0) by_group[t] = make_float2(u * inv, v * inv);
    }
    __syncthreads();
  }
}

// dw and db of the 32 channels of this block: their sums over the samples, in order
__device__ __forceinline__ void sum_params(const Norm& a, const float2* __restrict__ by_channel, void* __restrict__ dw,
                                           void* __restrict__ db, float2* part) {
  const int k = blockIdx.x * 32 + (threadIdx.x & 31), lane = threadIdx.x >> 5;      // 32 channels x 8 slices of the samples
  float u = 0.f, v = 0.f;
  if (k < a.c)
    for (int s = lane; s < a.b; s += kNormWarps) {
      const float2 f = by_channel[(int64_t)s * a.c + k];
      u += f.x;
      v += f.y;
    }
  part[threadIdx.x] = make_float2(u, v);
  __syncthreads();
  if (lane == 0 && k < a.c) {
    for (int l = 1; l < kNormWarps; ++l) {
      u += part[l * 32 + threadIdx.x].x;
      v += part[l * 32 + threadIdx.x].y;
    }
    if (db) store_any(db, a.p_dtype, k, u);
    if (dw) store_any(dw, a.p_dtype, k, v);
  }
}

// dx = rstd * (dz * w - m1 - xhat * m2) = dz * a + (x - mean) * k2 + k1 with k1 = -rstd * m1, k2 = -rstd^2 * m2
// 1M x 64 bf16 with SiLU: 58 us for 384 MB, the copy rate; the rows are walked backwards as above.
template <typename T, int VEC, int A, bool ORDERED>
__global__ void __launch_bounds__(kNormThreads, 3) norm_grad_apply_kernel(Norm a, const T* __restrict__ x, const T* __restrict__ dy,
                                                                          const float* __restrict__ mean,
                                                                          const float* __restrict__ rstd,
                                                                          const float2* __restrict__ by_group,
                                                                          const float2* __restrict__ by_channel,
                                                                          T* __restrict__ dx, void* __restrict__ dw,
                                                                          void* __restrict__ db) {
  constexpr int U = kBatch<T, VEC> / 2, W = VEC / A;
  extern __shared__ __align__(16) unsigned char pipe[];
  if ((dw || db) && blockIdx.y == 0 && blockIdx.x * 32 < a.c) {      // the first blocks also write the parameters' gradients
    __shared__ float2 part[kNormThreads];
    sum_params(a, by_channel, dw, db, part);
  }
  const int first = blockIdx.y * a.tile, width = min(a.tile, a.cols - first);
  const int lane = threadIdx.x / width, lanes = kNormThreads / width;
  const int k0 = (first + threadIdx.x - lane * width) * VEC;
  const int64_t p0 = blockIdx.x * a.chunk, p1 = min(p0 + a.chunk, a.n);
  const T *xc = x + k0, *gc = dy + k0;
  T* dc = dx + k0;
  const int last = min(first_sample(a, p1 - 1), a.b - 1);
  if (lane >= lanes) return;
  clear_outside<T, VEC, ORDERED>(a, p0, p1, lane, lanes, dc);
  for (int s = last; s >= 0; --s) {
    const int64_t end = offset_of(a, s + 1);
    if (end <= p0) break;
    const int64_t lo = max(p0, offset_of(a, s)), hi = min(p1, end);
    if (lo >= hi) continue;
    Channels<VEC, A> ch;
    ch.load(a, s, k0, mean, rstd);
    float k1[A], k2[A];
#pragma unroll
    for (int i = 0; i < A; ++i) {
      const int64_t at = (int64_t)s * a.g + (k0 + i * W) / a.d;
      const float2 f = __ldg(by_group + at);
      const float r = __ldg(rstd + at);
      k1[i] = -r * f.x;
      k2[i] = -r * r * f.y;
    }
    const T* const src[2] = {xc, gc};
    for_rows<T, VEC, 2, U, ORDERED>(a, src, hi - 1 - lane, -lanes, LaneRows(hi - lo, lanes).of(lane), pipe,
                                    [&](auto& v, const auto& at, auto full) {
#pragma unroll
      for (int u = 0; u < U; ++u) {
        if (!decltype(full)::value && at[u] < 0) continue;
        float h[VEC], z[VEC], g[VEC];
        v[0][u].get(h);
        v[1][u].get(g);
        ch.center(h);
        ch.affine(z, h);
        activate_grad(z, g, a.act, a.slope);
        fma_all(h, h, [&](int e) { return k2[e / W]; }, [&](int e) { return k1[e / W]; });
        fma_all(g, g, [&](int e) { return ch.a[e]; }, [&](int e) { return h[e]; });
        v[1][u].set(g);
        v[1][u].store(dc + at[u]);
      }
    });
  }
}

__global__ void __launch_bounds__(kNormThreads) norm_grad_params_kernel(Norm a, const float2* __restrict__ by_channel,
                                                                        void* __restrict__ dw, void* __restrict__ db) {
  __shared__ float2 part[kNormThreads];
  sum_params(a, by_channel, dw, db, part);
}

// ------------------------------------------------------------------------------------------------ small samples
// One block per sample and group, with the group's values in registers between the sums and the result: one launch, one
// read.  What a long sample has beyond the registers is read again, so every size is served; norm_small() says when.
// 1217 x 256 fp16 in 32 groups: 7 us in place of 13, bound by the round trips to memory of a block.
constexpr int kSmallThreads = 512;
constexpr int kSmallVectors = 4096;      // vectors of a sample and group that a block holds at most in the backward pass

// sum over the block, the same bits in every thread; `part`: one float per warp
__device__ __forceinline__ float block_sum(float v, float* part) {
  v = warp_sum(v);
  __syncthreads();      // the last use of part is over
  if ((threadIdx.x & 31) == 0) part[threadIdx.x >> 5] = v;
  __syncthreads();
  v = 0.f;
  for (int i = 0; i < (int)(blockDim.x >> 5); ++i) v += part[i];
  return v;
}

template <typename T, int VEC, bool ORDERED>
__global__ void __launch_bounds__(kSmallThreads) norm_small_kernel(Norm a, const T* __restrict__ x, T* __restrict__ y,
                                                                   float* __restrict__ mean_, float* __restrict__ rstd_) {
  constexpr int R = 2 * kSmallVectors / kSmallThreads;
  __shared__ float part[kSmallThreads / 32];
  const int dv = a.d / VEC, gr = blockIdx.x, s = blockIdx.y;
  const int lanes = blockDim.x / dv, lane = threadIdx.x / dv, k0 = gr * a.d + (threadIdx.x - lane * dv) * VEC;
  const bool on = lane < lanes;
  const T* xc = x + k0;
  T* yc = y + k0;
  if (s == 0 && on) clear_outside<T, VEC, ORDERED>(a, 0, a.n, lane, lanes, yc);
  const int64_t lo = a.b ? offset_of(a, s) : 0, hi = a.b ? offset_of(a, s + 1) : 0, first = on ? lo + lane : hi;
  const int64_t rest = first + (int64_t)R * lanes;
  Pack<T, VEC> v[R];
  float sum = 0.f;
#pragma unroll
  for (int r = 0; r < R; ++r) {
    const int64_t p = first + r * lanes, row = p < hi ? row_at<ORDERED>(a, p) : -1;
    v[r].clear();
    if (row >= 0) v[r].load(xc + row * a.c);
  }
  auto each = [&](auto&& f) {      // the rows beyond the registers, four at a time
    for (int64_t p = rest; p < hi; p += 4 * lanes) {
      Pack<T, VEC> q[4];
      int64_t row[4];
#pragma unroll
      for (int u = 0; u < 4; ++u) {
        row[u] = p + u * lanes < hi ? row_at<ORDERED>(a, p + u * lanes) : -1;
        q[u].clear();
        if (row[u] >= 0) q[u].load(xc + row[u] * a.c);
      }
#pragma unroll
      for (int u = 0; u < 4; ++u)
        if (p + u * lanes < hi) f(q[u], row[u]);
    }
  };
  const auto add = [&](const Pack<T, VEC>& q) {
    float f[VEC];
    q.get(f);
#pragma unroll
    for (int e = 0; e < VEC; ++e) sum += f[e];
  };
#pragma unroll
  for (int r = 0; r < R; ++r) add(v[r]);      // zeros where there is no row
  each([&](const Pack<T, VEC>& q, int64_t) { add(q); });
  const float count = (float)max(hi - lo, (int64_t)1) * a.d;
  const float mean = block_sum(sum, part) / count;
  float sq = 0.f;
  const auto square = [&](const Pack<T, VEC>& q) {
    float f[VEC];
    q.get(f);
#pragma unroll
    for (int e = 0; e < VEC; ++e) sq = fmaf(f[e] - mean, f[e] - mean, sq);
  };
#pragma unroll
  for (int r = 0; r < R; ++r) {
    forget(v[r].raw);
    if (first + r * lanes < hi) square(v[r]);
  }
  each([&](const Pack<T, VEC>& q, int64_t) { square(q); });
  const float rstd = 1.f / sqrtf(block_sum(sq, part) / count + a.eps);
  if (threadIdx.x == 0 && mean_ && a.b) {
    mean_[(int64_t)s * a.g + gr] = mean;
    rstd_[(int64_t)s * a.g + gr] = rstd;
  }
  if (!on) return;
  float w[VEC], b[VEC];
#pragma unroll
  for (int e = 0; e < VEC; ++e) {
    w[e] = rstd * (a.w ? load_any(a.w, a.p_dtype, k0 + e) : 1.f);
    b[e] = a.bias ? load_any(a.bias, a.p_dtype, k0 + e) : 0.f;
  }
  const auto put = [&](Pack<T, VEC>& q, int64_t row) {
    if (row < 0) return;
    float z[VEC];
    q.get(z);
#pragma unroll
    for (int e = 0; e < VEC; ++e) z[e] = fmaf(z[e] - mean, w[e], b[e]);
    activate(z, a.act, a.slope);
    q.set(z);
    q.store(yc + row * a.c);
  };
#pragma unroll
  for (int r = 0; r < R; ++r) {
    forget(v[r].raw);
    if (first + r * lanes < hi) put(v[r], row_at<ORDERED>(a, first + r * lanes));
  }
  each([&](Pack<T, VEC>& q, int64_t row) { put(q, row); });
}

// by_channel[s][k] receives the sums of dz and dz * xhat where there are several samples; one writes dw and db itself
template <typename T, int VEC, bool ORDERED>
__global__ void __launch_bounds__(kSmallThreads) norm_small_grad_kernel(Norm a, const T* __restrict__ x, const T* __restrict__ dy,
                                                                        const float* __restrict__ mean_,
                                                                        const float* __restrict__ rstd_,
                                                                        float2* __restrict__ by_channel, T* __restrict__ dx,
                                                                        void* __restrict__ dw, void* __restrict__ db) {
  constexpr int R = kSmallVectors / kSmallThreads;
  __shared__ float part[kSmallThreads / 32];
  __shared__ float2 sums[VEC * kSmallThreads];
  const int dv = a.d / VEC, gr = blockIdx.x, s = blockIdx.y;
  const int lanes = blockDim.x / dv, lane = threadIdx.x / dv, col = threadIdx.x - lane * dv, k0 = gr * a.d + col * VEC;
  const bool on = lane < lanes;
  const T *xc = x + k0, *gc = dy + k0;
  T* dc = dx + k0;
  if (s == 0 && on) clear_outside<T, VEC, ORDERED>(a, 0, a.n, lane, lanes, dc);
  const int64_t lo = a.b ? offset_of(a, s) : 0, hi = a.b ? offset_of(a, s + 1) : 0, first = on ? lo + lane : hi;
  const int64_t rest = first + (int64_t)R * lanes;
  const float mean = a.b ? __ldg(mean_ + (int64_t)s * a.g + gr) : 0.f, rstd = a.b ? __ldg(rstd_ + (int64_t)s * a.g + gr) : 0.f;
  float w[VEC], b[VEC];
#pragma unroll
  for (int e = 0; e < VEC; ++e) {
    w[e] = rstd * (on && a.w ? load_any(a.w, a.p_dtype, k0 + e) : 1.f);
    b[e] = on && a.bias ? load_any(a.bias, a.p_dtype, k0 + e) : 0.f;
  }
  Pack<T, VEC> vx[R], vg[R];
#pragma unroll
  for (int r = 0; r < R; ++r) {
    const int64_t p = first + r * lanes, row = p < hi ? row_at<ORDERED>(a, p) : -1;
    vx[r].clear();
    vg[r].clear();
    if (row >= 0) {
      vx[r].load(xc + row * a.c);
      vg[r].load(gc + row * a.c);
    }
  }
  auto each = [&](auto&& f) {      // the rows beyond the registers, two at a time
    for (int64_t p = rest; p < hi; p += 2 * lanes) {
      Pack<T, VEC> qx[2], qg[2];
      int64_t row[2];
#pragma unroll
      for (int u = 0; u < 2; ++u) {
        row[u] = p + u * lanes < hi ? row_at<ORDERED>(a, p + u * lanes) : -1;
        if (row[u] < 0) continue;
        qx[u].load(xc + row[u] * a.c);
        qg[u].load(gc + row[u] * a.c);
      }
#pragma unroll
      for (int u = 0; u < 2; ++u)
        if (row[u] >= 0) f(qx[u], qg[u], row[u]);
    }
  };
  const auto terms = [&](const Pack<T, VEC>& qx, const Pack<T, VEC>& qg, float (&h)[VEC], float (&g)[VEC]) {
    float z[VEC];
    qx.get(h);
    qg.get(g);
#pragma unroll
    for (int e = 0; e < VEC; ++e) {
      h[e] -= mean;
      z[e] = fmaf(h[e], w[e], b[e]);
    }
    activate_grad(z, g, a.act, a.slope);
  };
  float s1[VEC], s2[VEC];
#pragma unroll
  for (int e = 0; e < VEC; ++e) s1[e] = s2[e] = 0.f;
  const auto add = [&](const Pack<T, VEC>& qx, const Pack<T, VEC>& qg) {
    float h[VEC], g[VEC];
    terms(qx, qg, h, g);
#pragma unroll
    for (int e = 0; e < VEC; ++e) {
      s1[e] += g[e];
      s2[e] = fmaf(g[e], h[e], s2[e]);
    }
  };
#pragma unroll
  for (int r = 0; r < R; ++r)
    if (first + r * lanes < hi) add(vx[r], vg[r]);
  each([&](const Pack<T, VEC>& qx, const Pack<T, VEC>& qg, int64_t) { add(qx, qg); });
#pragma unroll
  for (int e = 0; e < VEC; ++e) sums[e * kSmallThreads + threadIdx.x] = make_float2(s1[e], s2[e]);
  __syncthreads();
  // the lanes of a channel: slices of them by several threads, then the slices by one
  const int slices = max((int)blockDim.x / a.d, 1);
  float m1 = 0.f, m2 = 0.f;
  for (int k = threadIdx.x % a.d; k < a.d; k += blockDim.x) {
    const int slice = threadIdx.x / a.d;
    float u = 0.f, v = 0.f;
    if (slice < slices) {
      for (int l = slice; l < lanes; l += slices) {
        const float2 f = sums[k % VEC * kSmallThreads + l * dv + k / VEC];
        u += f.x;
        v += f.y;
      }
      // w of this channel times its sums, over the whole group: m1 and m2
      const float wk = a.w ? load_any(a.w, a.p_dtype, gr * a.d + k) : 1.f;
      m1 = fmaf(wk, u, m1);
      m2 = fmaf(wk * rstd, v, m2);
    }
    s1[0] = u;
    s2[0] = v;
  }
  m1 = block_sum(m1, part);      // its barriers also end the reads of sums[]
  m2 = block_sum(m2, part);
  const float count = (float)max(hi - lo, (int64_t)1) * a.d;
  const float k1 = rstd * (m1 / count), k2 = rstd * rstd * (m2 / count);
  if (slices > 1) {
    if ((int)threadIdx.x < slices * a.d) sums[threadIdx.x] = make_float2(s1[0], s2[0]);
    __syncthreads();
  }
  for (int k = threadIdx.x; k < a.d; k += blockDim.x) {
    float u = 0.f, v = 0.f;
    if (slices > 1) {
      for (int i = 0; i < slices; ++i) {
        u += sums[i * a.d + k].x;
        v += sums[i * a.d + k].y;
      }
    } else {      // one slice: all lanes of a channel that this thread summed above
      for (int l = 0; l < lanes; ++l) {
        const float2 f = sums[k % VEC * kSmallThreads + l * dv + k / VEC];
        u += f.x;
        v += f.y;
      }
    }
    v = hi > lo ? v * rstd : 0.f;      // an empty sample has no deviation: with eps = 0 its rstd is infinite
    const int ch = gr * a.d + k;
    if (a.b > 1) {
      by_channel[(int64_t)s * a.c + ch] = make_float2(u, v);
    } else {
      if (db) store_any(db, a.p_dtype, ch, u);
      if (dw) store_any(dw, a.p_dtype, ch, v);
    }
  }
  if (!on) return;
  const auto put = [&](const Pack<T, VEC>& qx, Pack<T, VEC>& qg, int64_t row) {
    if (row < 0) return;
    float h[VEC], g[VEC];
    terms(qx, qg, h, g);
#pragma unroll
    for (int e = 0; e < VEC; ++e) g[e] = fmaf(g[e], w[e], -fmaf(h[e], k2, k1));
    qg.set(g);
    qg.store(dc + row * a.c);
  };
#pragma unroll
  for (int r = 0; r < R; ++r) {
    forget(vx[r].raw);
    forget(vg[r].raw);
    if (first + r * lanes < hi) put(vx[r], vg[r], row_at<ORDERED>(a, first + r * lanes));
  }
  each([&](const Pack<T, VEC>& qx, Pack<T, VEC>& qg, int64_t row) { put(qx, qg, row); });
}

// ------------------------------------------------------------------------------------------------ host
bool good_dtype(int dtype) { return dtype == TSB_F32 || dtype == TSB_F16 || dtype == TSB_BF16; }

int check_norm(int64_t n, int64_t c, int64_t g, int64_t b, const void* offsets, int dtype, int p_dtype, int act) {
  if (n < 0 || c < 1 || g < 1 || c % g != 0 || b < 0 || (b && !offsets) || act < kActNone || act > kActSilu) return TSB_ERR_BAD_ARG;
  if (!good_dtype(dtype) || !good_dtype(p_dtype)) return TSB_ERR_UNSUPPORTED;
  if (n > 0x7fffffff || c > 65536 || b > 0x7fffffff / g) return TSB_ERR_LIMIT;
  return TSB_OK;
}

// f(PackTag<T, VEC>, A, ORDERED): A = 1 where a vector lies in one group, 2 where its halves do, else VEC
template <typename F>
int dispatch_norm(int dtype, int vec, int d, bool ordered, F&& f) {
  return dispatch_pack(dtype, vec, [&](auto tag) -> int {
    using T = typename decltype(tag)::T;
    constexpr int VEC = decltype(tag)::VEC;
    auto with = [&](auto each) -> int {
      return ordered ? f(tag, each, std::true_type()) : f(tag, each, std::false_type());
    };
    if constexpr (VEC == 8) {
      if (d % 8 != 0) return with(std::integral_constant<int, 2>());
    } else if constexpr (VEC * sizeof(T) < 16 && VEC > 1) {
      if (d % VEC != 0) return with(std::integral_constant<int, VEC>());
    }
    return with(std::integral_constant<int, 1>());
  });
}

Norm norm_shape(int64_t n, int64_t c, int64_t g, int64_t b, int vec) {
  Norm a{};
  a.n = n;
  a.c = (int)c;
  a.g = (int)g;
  a.d = (int)(c / g);
  a.b = (int)b;
  a.cols = (int)(c / vec);
  a.tile = (int)cdiv(a.cols, cdiv(a.cols, kNormThreads));
  const int64_t tiles = cdiv(a.cols, a.tile);
  int64_t blocks = cdiv(n, (int64_t)(kNormThreads / a.tile) * 4);      // four rows per lane at least
  if (blocks > cdiv(kNormBlocks, tiles)) blocks = cdiv(kNormBlocks, tiles);
  if (blocks < 1) blocks = 1;
  a.chunk = cdiv(n, blocks);
  if (a.chunk < 1) a.chunk = 1;
  a.nblk = (int)cdiv(n, a.chunk);
  return a;
}

// The widest vector, or half of it (8 bytes) where 16 bytes lie in more than two groups: with a mean and a deviation for
// each channel of the wide one the gradient kernels would spill.
int norm_vector(int dtype, int64_t c, int64_t g, uintptr_t bits) {
  const int vec = vector_width(dtype, c, bits);
  const int64_t d = c / g, part = vec == 8 ? 4 : vec;
  return vec * (int)dtype_size(dtype) == 16 && d % part != 0 ? vec / 2 : vec;
}

// One block per sample and group where a sample of mean length fits the block's registers, the whole input is small (a row of a
// group counts as 32 bytes at least, what a read of it moves) and one sample that had nearly all rows would fit four times
// the registers: the offsets are on the device, so the lengths are not known here.
// Forward and backward on the device against the streaming kernels, which take two or three launches more each way; first
// samples of equal lengths, then one of a third of the rows, then one of all among empty ones:
//   8000 rows of 64 channels bf16, 4 samples, 8 groups    8 + 15 / 14 + 17     9 + 17 / 14 + 17   15 + 35 / 12 + 14 us
//   16384 rows, 16 samples                                 8 + 13 / 11 + 14    12 + 27 / 15 + 18   37 + 65 / 11 + 14 us
//   30000 rows, 16 samples                                 9 + 15 / 16 + 19    20 + 43 / 16 + 19   72 + 113 / 14 + 16 us
//   60000 rows of 64 channels, 64 samples, 64 groups     120 + 167 / 29 + 33
bool norm_small(int64_t n, int64_t c, int64_t g, int64_t b, int dtype) {
  const int64_t d = c / g, dv = d / vector_width(dtype, d, 0), bytes = d * (int64_t)dtype_size(dtype);
  return b <= 65535 && dv <= 64 && cdiv(n, b > 1 ? b : 1) * dv <= kSmallVectors && n * dv <= 4 * kSmallVectors &&
         n * g * (bytes < 32 ? 32 : bytes) <= (8 << 20);
}

// threads of a block of the small kernels: two vectors each for a sample of mean length
int small_threads(int64_t n, int64_t b, int dv) {
  const int64_t want = cdiv(cdiv(n, b > 1 ? b : 1) * dv, 2 * 32) * 32;
  return (int)(want < 128 ? 128 : want > kSmallThreads ? kSmallThreads : want);
}

template <typename F>
int dispatch_small(int dtype, int vec, bool ordered, F&& f) {
  return dispatch_pack(dtype, vec, [&](auto tag) -> int { return ordered ? f(tag, std::true_type()) : f(tag, std::false_type()); });
}

// Parts of the workspaces, for the vector width that needs the most: which one a call takes is up to its addresses.
// f(shape) of every width that divides a row, the largest
template <typename F>
int64_t most_of_widths(int64_t n, int64_t c, int64_t g, int64_t b, int dtype, F&& f) {
  int64_t most = 0;
  for (int vec = 1; vec * (int)dtype_size(dtype) <= 16 && c % vec == 0; vec *= 2) {
    const int64_t need = f(norm_shape(n, c, g, b, vec));
    if (need > most) most = need;
  }
  return most;
}
size_t fwd_slot_bytes(int64_t n, int64_t c, int64_t g, int64_t b, int dtype) {
  const int64_t slots = most_of_widths(n, c, g, b, dtype, [&](const Norm& a) { return cdiv(a.cols, a.tile) * (a.nblk + b); });
  return align_up((size_t)slots * g * sizeof(float2), 256);
}
int64_t grad_slots(int64_t n, int64_t c, int64_t g, int64_t b, int dtype) {
  return most_of_widths(n, c, g, b, dtype, [&](const Norm& a) { return a.nblk + b; });
}
size_t stat_bytes(int64_t g, int64_t b) { return align_up((size_t)b * g * sizeof(float), 256); }
size_t channel_bytes(int64_t c, int64_t b) { return align_up((size_t)b * c * sizeof(float2), 256); }

Norm norm_args(Norm a, const int32_t* order, const int32_t* offsets, const void* weight, const void* bias, int param_dtype,
               float eps, int act, float slope) {
  a.order = order;
  a.offsets = offsets;
  a.w = weight;
  a.bias = bias;
  a.p_dtype = param_dtype;
  a.eps = eps;
  a.act = act;
  a.slope = slope;
  return a;
}

}  // namespace
}  // namespace tsb

using namespace tsb;

extern "C" {

size_t tsb_group_norm_fwd_workspace_bytes(int64_t n, int64_t c, int64_t g, int64_t b, int32_t dtype) {
  if (check_norm(n, c, g, 0, nullptr, dtype, 0, 0) != TSB_OK || b < 0 || norm_small(n, c, g, b, dtype)) return 0;
  return fwd_slot_bytes(n, c, g, b, dtype) + 2 * stat_bytes(g, b);
}

int tsb_group_norm_fwd(const void* x, const int32_t* order, const int32_t* offsets, const void* weight, const void* bias,
                       int64_t n, int64_t c, int64_t g, int64_t b, float eps, int32_t act, float slope, int32_t dtype,
                       int32_t param_dtype, void* y, float* mean, float* rstd, void* workspace, size_t workspace_bytes,
                       tsb_stream_t stream) {
  const int bad = check_norm(n, c, g, b, offsets, dtype, param_dtype, act);
  if (bad != TSB_OK) return bad;
  if ((n && (!x || !y)) || !mean != !rstd) return TSB_ERR_BAD_ARG;
  cudaStream_t st = as_stream(stream);
  const uintptr_t bits = (uintptr_t)x | (uintptr_t)y;
  if (norm_small(n, c, g, b, dtype)) {
    const int vec = vector_width(dtype, c / g, bits), dv = (int)(c / g) / vec;      // at most 512: 64 of the widest vectors
    const Norm a = norm_args(norm_shape(n, c, g, b, vec), order, offsets, weight, bias, param_dtype, eps, act, slope);
    const dim3 grid((unsigned)g, (unsigned)(b > 1 ? b : 1));
    const int threads = dv > 128 ? kSmallThreads : small_threads(n, b, dv);
    return dispatch_small(dtype, vec, order != nullptr, [&](auto tag, auto ordered) -> int {
      using T = typename decltype(tag)::T;
      norm_small_kernel<T, decltype(tag)::VEC, decltype(ordered)::value>
          <<<grid, threads, 0, st>>>(a, (const T*)x, (T*)y, mean, rstd);
      TSB_LAUNCH_CHECK();
      return TSB_OK;
    });
  }
  if (workspace_bytes < fwd_slot_bytes(n, c, g, b, dtype) + 2 * stat_bytes(g, b) || !workspace) return TSB_ERR_WORKSPACE;
  const int vec = norm_vector(dtype, c, g, bits);
  const Norm a = norm_args(norm_shape(n, c, g, b, vec), order, offsets, weight, bias, param_dtype, eps, act, slope);
  char* ws = static_cast<char*>(workspace);
  float2* slots = reinterpret_cast<float2*>(ws);
  if (!mean) {
    mean = reinterpret_cast<float*>(ws + fwd_slot_bytes(n, c, g, b, dtype));
    rstd = reinterpret_cast<float*>(ws + fwd_slot_bytes(n, c, g, b, dtype) + stat_bytes(g, b));
  }
  const int tiles = (int)cdiv(a.cols, a.tile);
  const dim3 grid((unsigned)a.nblk, (unsigned)tiles);
  return dispatch_norm(dtype, vec, a.d, order != nullptr, [&](auto tag, auto each, auto ordered) -> int {
    using T = typename decltype(tag)::T;
    constexpr int VEC = decltype(tag)::VEC, A = decltype(each)::value;
    constexpr bool ORDERED = decltype(ordered)::value;
    if (n && b) {
      const int rc = launch_wide<norm_stats_kernel<T, VEC, A, ORDERED>, kPipeBytes<T, VEC>>(grid, kNormThreads, st, a, (const T*)x,
                                                                                              slots);
      if (rc != TSB_OK) return rc;
    }
    if (b) {
      norm_join_kernel<<<grid_for((int64_t)a.b * a.g, 4), 128, 0, st>>>(a, VEC, tiles, slots, mean, rstd);
      TSB_LAUNCH_CHECK();
    }
    if (n) {
      const int rc = launch_wide<norm_apply_kernel<T, VEC, A, ORDERED>, kPipeBytes<T, VEC>>(grid, kNormThreads, st, a, (const T*)x, mean,
                                                            rstd, (T*)y);
      if (rc != TSB_OK) return rc;
    }
    return TSB_OK;
  });
}

size_t tsb_group_norm_bwd_workspace_bytes(int64_t n, int64_t c, int64_t g, int64_t b, int32_t dtype) {
  if (check_norm(n, c, g, 0, nullptr, dtype, 0, 0) != TSB_OK || b < 0) return 0;
  if (norm_small(n, c, g, b, dtype)) return b > 1 ? channel_bytes(c, b) : 0;
  return channel_bytes(c, grad_slots(n, c, g, b, dtype)) + channel_bytes(c, b) + channel_bytes(g, b);
}

int tsb_group_norm_bwd(const void* x, const void* dy, const int32_t* order, const int32_t* offsets, const void* weight,
                       const void* bias, const float* mean, const float* rstd, int64_t n, int64_t c, int64_t g, int64_t b,
                       int32_t act, float slope, int32_t dtype, int32_t param_dtype, void* dx, void* dweight, void* dbias,
                       void* workspace, size_t workspace_bytes, tsb_stream_t stream) {
  const int bad = check_norm(n, c, g, b, offsets, dtype, param_dtype, act);
  if (bad != TSB_OK) return bad;
  if ((n && (!x || !dy || !dx)) || (b && (!mean || !rstd))) return TSB_ERR_BAD_ARG;
  cudaStream_t st = as_stream(stream);
  const size_t need = tsb_group_norm_bwd_workspace_bytes(n, c, g, b, dtype);
  if (workspace_bytes < need || (need && !workspace)) return TSB_ERR_WORKSPACE;
  const uintptr_t bits = (uintptr_t)x | (uintptr_t)dy | (uintptr_t)dx;
  char* ws = static_cast<char*>(workspace);
  if (norm_small(n, c, g, b, dtype)) {
    const int vec = vector_width(dtype, c / g, bits), dv = (int)(c / g) / vec;      // at most 512: 64 of the widest vectors
    const Norm a = norm_args(norm_shape(n, c, g, b, vec), order, offsets, weight, bias, param_dtype, 0.f, act, slope);
    const dim3 grid((unsigned)g, (unsigned)(b > 1 ? b : 1));
    const int threads = dv > 128 ? kSmallThreads : small_threads(n, b, dv);
    float2* by_channel = reinterpret_cast<float2*>(ws);
    return dispatch_small(dtype, vec, order != nullptr, [&](auto tag, auto ordered) -> int {
      using T = typename decltype(tag)::T;
      norm_small_grad_kernel<T, decltype(tag)::VEC, decltype(ordered)::value>
          <<<grid, threads, 0, st>>>(a, (const T*)x, (const T*)dy, mean, rstd, by_channel, (T*)dx, dweight, dbias);
      TSB_LAUNCH_CHECK();
      if (b > 1 && (dweight || dbias)) {
        norm_grad_params_kernel<<<(unsigned)cdiv(a.c, 32), kNormThreads, 0, st>>>(a, by_channel, dweight, dbias);
        TSB_LAUNCH_CHECK();
      }
      return TSB_OK;
    });
  }
  const int vec = norm_vector(dtype, c, g, bits);
  const Norm a = norm_args(norm_shape(n, c, g, b, vec), order, offsets, weight, bias, param_dtype, 0.f, act, slope);
  float2* slots = reinterpret_cast<float2*>(ws);
  const size_t slot_bytes = channel_bytes(c, grad_slots(n, c, g, b, dtype));
  float2* by_channel = reinterpret_cast<float2*>(ws + slot_bytes);
  float2* by_group = reinterpret_cast<float2*>(ws + slot_bytes + channel_bytes(c, b));
  const dim3 grid((unsigned)a.nblk, (unsigned)cdiv(a.cols, a.tile));
  const bool fold = (int64_t)a.nblk * 32 >= c;      // enough blocks for the parameters: no launch of their own
  return dispatch_norm(dtype, vec, a.d, order != nullptr, [&](auto tag, auto each, auto ordered) -> int {
    using T = typename decltype(tag)::T;
    constexpr int VEC = decltype(tag)::VEC, A = decltype(each)::value;
    constexpr bool ORDERED = decltype(ordered)::value;
    if (n && b) {
      const int rc = launch_wide<norm_grad_sums_kernel<T, VEC, A, ORDERED>, kPipeBytes<T, VEC>>(grid, kNormThreads, st, a, (const T*)x,
                                                            (const T*)dy, mean, rstd, slots);
      if (rc != TSB_OK) return rc;
    }
    if (b) {
      const int64_t pairs = (int64_t)a.b * a.g;
      norm_grad_join_kernel<<<grid_for(pairs, 1), pairs <= kSmCount ? kJoinThreads : kJoinThreads / 2, 0, st>>>(a, slots, by_channel,
                                                                                                           by_group);
      TSB_LAUNCH_CHECK();
    }
    if (n) {
      const int rc = launch_wide<norm_grad_apply_kernel<T, VEC, A, ORDERED>, kPipeBytes<T, VEC>>(grid, kNormThreads, st, a, (const T*)x,
                                                            (const T*)dy, mean, rstd, by_group, by_channel, (T*)dx,
                                                            fold ? dweight : nullptr, fold ? dbias : nullptr);
      if (rc != TSB_OK) return rc;
    }
    if (!fold && (dweight || dbias)) {
      norm_grad_params_kernel<<<(unsigned)cdiv(a.c, 32), kNormThreads, 0, st>>>(a, by_channel, dweight, dbias);
      TSB_LAUNCH_CHECK();
    }
    return TSB_OK;
  });
}

}  // extern "C"
