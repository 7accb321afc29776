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
// sums, in 32 bits.
#include "rows.cuh"

namespace tsb {
namespace {

constexpr int kNormThreads = 512;
enum { kActNone = 0, kActRelu = 1, kActLeaky = 2, kActSilu = 3 };

struct Norm {
  int64_t n;             // rows
  int c, g, d;           // channels, groups, channels of a group
  int b;                 // samples
  int cols;              // vectors of a row
  int tile;              // vectors of a row that one block takes (grid.y tiles)
  int lanes;             // rows that a block takes at once
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

// first sample that ends behind position p (a.b: none)
__device__ __forceinline__ int first_sample(const Norm& a, int64_t p) {
  int lo = 0, hi = a.b;
  while (lo < hi) {
    const int mid = (lo + hi) >> 1;
    if (offset_of(a, mid + 1) <= p) lo = mid + 1; else hi = mid;
  }
  return lo;
}

// row at a grouped position, -1 for an entry of a caller's order that is no row
__device__ __forceinline__ int64_t row_at(const Norm& a, int64_t p) {
  if (!a.order) return p;
  const int64_t r = __ldg(a.order + p);
  return r >= 0 && r < a.n ? r : -1;
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
#pragma unroll
    for (int i = 0; i < N; ++i) z[i] = z[i] / (1.f + __expf(-z[i]));
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
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const float p = 1.f / (1.f + __expf(-z[i]));
      g[i] *= p * (1.f + z[i] * (1.f - p));
    }
  }
}

__device__ __forceinline__ float warp_sum(float v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_down_sync(0xffffffffu, v, o);
  return __shfl_sync(0xffffffffu, v, 0);
}

// rows that lane l of `lanes` takes of `rows`
__device__ __forceinline__ int64_t lane_rows(int64_t rows, int lanes, int l) { return l < rows ? (rows - l - 1) / lanes + 1 : 0; }

// channels of group gr that column tile y holds
__device__ __forceinline__ int tile_channels(const Norm& a, int vec, int y, int gr) {
  const int lo = max(y * a.tile * vec, gr * a.d), hi = min(min((y + 1) * a.tile * vec, a.c), (gr + 1) * a.d);
  return max(hi - lo, 0);
}

// ------------------------------------------------------------------------------------------------ statistics
// A thread holds the mean and the sum of squares about it of the values that it has seen: one pair where a vector lies in
// one group (A == 1), one pair per channel otherwise (A == VEC).  U rows are read together; their own mean and squares
// are exact to rounding and are joined to the running pair.
template <typename T, int VEC, int A>
__global__ void __launch_bounds__(kNormThreads) norm_stats_kernel(Norm a, const T* __restrict__ x, float2* __restrict__ slots) {
  __shared__ float2 part[A * kNormThreads];
  const int first = blockIdx.y * a.tile, width = min(a.tile, a.cols - first);
  const int lane = threadIdx.x / width, col = threadIdx.x - lane * width;
  const int lanes = kNormThreads / width;
  const int64_t p0 = blockIdx.x * a.chunk, p1 = min(p0 + a.chunk, a.n);
  for (int s = first_sample(a, p0); s < a.b; ++s) {
    const int64_t begin = offset_of(a, s);
    if (begin >= p1) break;
    const int64_t lo = max(p0, begin), hi = min(p1, offset_of(a, s + 1));
    if (lo >= hi) continue;
    float n = 0.f, mean[A], m2[A];
#pragma unroll
    for (int i = 0; i < A; ++i) mean[i] = m2[i] = 0.f;
    if (lane < lanes) {
      constexpr int U = 4;
      const int64_t at = (int64_t)(first + col) * VEC;
      for (int64_t p = lo + lane; p < hi; p += (int64_t)lanes * U) {
        Pack<T, VEC> v[U];
        int got = 0;
#pragma unroll
        for (int u = 0; u < U; ++u) {
          const int64_t q = p + (int64_t)u * lanes;
          v[u].clear();
          if (q < hi) {
            const int64_t r = row_at(a, q);
            if (r >= 0) v[u].load(x + r * a.c + at);
            ++got;
          }
        }
        constexpr int W = VEC / A;
        const float cnt = (float)(got * W), inv = 1.f / cnt, all = n + cnt, share = cnt / all;
        float sum[A], sq[A];
#pragma unroll
        for (int i = 0; i < A; ++i) sum[i] = sq[i] = 0.f;
#pragma unroll
        for (int u = 0; u < U; ++u) {
          float f[VEC];
          v[u].get(f);      // zeros beyond the end
#pragma unroll
          for (int e = 0; e < VEC; ++e) sum[e / W] += f[e];
        }
#pragma unroll
        for (int i = 0; i < A; ++i) sum[i] *= inv;
#pragma unroll
        for (int u = 0; u < U; ++u) {
          if (u >= got) continue;
          float f[VEC];
          v[u].get(f);
#pragma unroll
          for (int e = 0; e < VEC; ++e) {
            const float t = f[e] - sum[e / W];
            sq[e / W] = fmaf(t, t, sq[e / W]);
          }
        }
#pragma unroll
        for (int i = 0; i < A; ++i) {
          const float t = sum[i] - mean[i];
          mean[i] = fmaf(t, share, mean[i]);
          m2[i] += sq[i] + t * t * n * share;
        }
        n = all;
      }
#pragma unroll
      for (int i = 0; i < A; ++i) part[i * kNormThreads + threadIdx.x] = make_float2(mean[i], m2[i]);
    }
    __syncthreads();
    // one warp per group of this column tile
    const int c_lo = first * VEC, c_hi = (first + width) * VEC;
    const int g_lo = c_lo / a.d, g_hi = (c_hi - 1) / a.d;
    const int64_t rows = hi - lo;
    float2* slot = slots + ((int64_t)blockIdx.y * (a.nblk + a.b) + blockIdx.x + s) * a.g;
    for (int gr = g_lo + (threadIdx.x >> 5); gr <= g_hi; gr += kNormThreads / 32) {
      const int k_lo = max(gr * a.d, c_lo), k_hi = min((gr + 1) * a.d, c_hi);
      const int per_lane = (k_hi - k_lo) / (VEC / A), entries = per_lane * lanes;
      float w = 0.f, m = 0.f, q = 0.f;
      for (int pass = 0; pass < 2; ++pass) {      // the joint mean, then the squares about it
        float acc = 0.f;
        for (int t = threadIdx.x & 31; t < entries; t += 32) {
          const int l = t / per_lane, k = k_lo + (t - l * per_lane) * (VEC / A) - c_lo;
          const float cnt = (float)lane_rows(rows, lanes, l) * (VEC / A);
          if (cnt == 0.f) continue;
          const float2 e = part[(A == 1 ? 0 : k % VEC) * kNormThreads + l * width + k / VEC];
          if (pass == 0) {
            w += cnt;
            acc = fmaf(cnt, e.x, acc);
          } else {
            acc += fmaf(cnt * (e.x - m), e.x - m, e.y);
          }
        }
        acc = warp_sum(acc);
        if (pass == 0) {
          w = warp_sum(w);
          m = acc / w;
        } else {
          q = acc;
        }
      }
      if ((threadIdx.x & 31) == 0) slot[gr] = make_float2(m, q);
    }
    __syncthreads();
  }
}

// One warp per sample and group: the slots of the sample, joined in the order of the rows.
__global__ void __launch_bounds__(128) norm_join_kernel(Norm a, int vec, int tiles, const float2* __restrict__ slots,
                                                        float* __restrict__ mean, float* __restrict__ rstd) {
  const int lane = threadIdx.x & 31;
  for (int64_t t = blockIdx.x * 4 + (threadIdx.x >> 5); t < (int64_t)a.b * a.g; t += (int64_t)gridDim.x * 4) {
    const int s = (int)(t / a.g), gr = (int)(t - (int64_t)s * a.g);
    const int64_t begin = offset_of(a, s), end = offset_of(a, s + 1);
    float w = 0.f, m = 0.f, q = 0.f;
    if (begin < end) {
      const int j0 = (int)(begin / a.chunk), j1 = (int)((end - 1) / a.chunk);
      for (int pass = 0; pass < 2; ++pass) {
        float acc = 0.f;
        for (int y = 0; y < tiles; ++y) {
          const int width = tile_channels(a, vec, y, gr);
          if (width == 0) continue;
          for (int j = j0 + lane; j <= j1; j += 32) {
            const float cnt = (float)(min(end, (j + 1) * a.chunk) - max(begin, j * a.chunk)) * width;
            const float2 e = slots[((int64_t)y * (a.nblk + a.b) + j + s) * a.g + gr];
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

// What a thread needs of its VEC channels within one sample.
template <int VEC>
struct Channels {
  float mean[VEC], rstd[VEC], w[VEC], b[VEC];
  __device__ __forceinline__ void load(const Norm& a, int s, int k0, const float* __restrict__ mean_, const float* __restrict__ rstd_) {
#pragma unroll
    for (int e = 0; e < VEC; ++e) {
      const int64_t at = (int64_t)s * a.g + (k0 + e) / a.d;
      mean[e] = __ldg(mean_ + at);
      rstd[e] = __ldg(rstd_ + at);
      w[e] = a.w ? load_any(a.w, a.p_dtype, k0 + e) : 1.f;
      b[e] = a.bias ? load_any(a.bias, a.p_dtype, k0 + e) : 0.f;
    }
  }
};

// f(row, sample, sample changed) for every row of the block's chunk that belongs to this thread's lane; the rows come last
// chunk first, so that those read last by the pass before are still in the L2 cache.  Rows of no sample have sample -1.
template <typename T, int VEC, typename Begin, typename Row>
__device__ __forceinline__ void walk(const Norm& a, int lane, int lanes, Begin&& begin_sample, Row&& row) {
  const int64_t p0 = blockIdx.x * a.chunk, p1 = min(p0 + a.chunk, a.n);
  int64_t covered = p0;
  for (int s = first_sample(a, p0); s < a.b; ++s) {
    const int64_t begin = offset_of(a, s);
    if (begin >= p1) break;
    const int64_t lo = max(p0, begin), hi = min(p1, offset_of(a, s + 1));
    for (int64_t p = covered + lane; p < lo; p += lanes) row(p, false);
    if (lo >= hi) continue;
    begin_sample(s);
    for (int64_t p = lo + lane; p < hi; p += lanes) row(p, true);
    covered = max(covered, hi);
  }
  for (int64_t p = covered + lane; p < p1; p += lanes) row(p, false);
}

template <typename T, int VEC>
__global__ void __launch_bounds__(kNormThreads) norm_apply_kernel(Norm a, const T* __restrict__ x, const float* __restrict__ mean,
                                                                  const float* __restrict__ rstd, T* __restrict__ y) {
  const int first = blockIdx.y * a.tile, width = min(a.tile, a.cols - first);
  const int lane = threadIdx.x / width, lanes = kNormThreads / width;
  if (lane >= lanes) return;
  const int k0 = (first + threadIdx.x - lane * width) * VEC;
  Channels<VEC> ch;
  walk<T, VEC>(a, lane, lanes, [&](int s) { ch.load(a, s, k0, mean, rstd); }, [&](int64_t p, bool in) {
    const int64_t r = row_at(a, p);
    if (r < 0) return;
    Pack<T, VEC> v;
    if (in) {
      v.load(x + r * a.c + k0);
      float z[VEC];
      v.get(z);
#pragma unroll
      for (int e = 0; e < VEC; ++e) z[e] = fmaf((z[e] - ch.mean[e]) * ch.rstd[e], ch.w[e], ch.b[e]);
      activate(z, a.act, a.slope);
      v.set(z);
    } else {
      v.clear();
    }
    v.store(y + r * a.c + k0);
  });
}

// ------------------------------------------------------------------------------------------------ gradient
// Per slot and channel: the sums of dz and of dz * xhat.
template <typename T, int VEC>
__global__ void __launch_bounds__(kNormThreads) norm_grad_sums_kernel(Norm a, const T* __restrict__ x, const T* __restrict__ dy,
                                                                      const float* __restrict__ mean, const float* __restrict__ rstd,
                                                                      float2* __restrict__ slots) {
  __shared__ float2 part[VEC * kNormThreads];
  const int first = blockIdx.y * a.tile, width = min(a.tile, a.cols - first);
  const int lane = threadIdx.x / width, lanes = kNormThreads / width, col = threadIdx.x - lane * width;
  const int k0 = (first + col) * VEC;
  const int64_t p0 = blockIdx.x * a.chunk, p1 = min(p0 + a.chunk, a.n);
  for (int s = first_sample(a, p0); s < a.b; ++s) {
    const int64_t begin = offset_of(a, s);
    if (begin >= p1) break;
    const int64_t lo = max(p0, begin), hi = min(p1, offset_of(a, s + 1));
    if (lo >= hi) continue;
    float s1[VEC], s2[VEC];
#pragma unroll
    for (int e = 0; e < VEC; ++e) s1[e] = s2[e] = 0.f;
    if (lane < lanes) {
      Channels<VEC> ch;
      ch.load(a, s, k0, mean, rstd);
      for (int64_t p = lo + lane; p < hi; p += lanes) {
        const int64_t r = row_at(a, p);
        if (r < 0) continue;
        Pack<T, VEC> vx, vg;
        vx.load(x + r * a.c + k0);
        vg.load(dy + r * a.c + k0);
        float h[VEC], z[VEC], g[VEC];
        vx.get(h);
        vg.get(g);
#pragma unroll
        for (int e = 0; e < VEC; ++e) {
          h[e] = (h[e] - ch.mean[e]) * ch.rstd[e];
          z[e] = fmaf(h[e], ch.w[e], ch.b[e]);
        }
        activate_grad(z, g, a.act, a.slope);
#pragma unroll
        for (int e = 0; e < VEC; ++e) {
          s1[e] += g[e];
          s2[e] = fmaf(g[e], h[e], s2[e]);
        }
      }
#pragma unroll
      for (int e = 0; e < VEC; ++e) part[e * kNormThreads + threadIdx.x] = make_float2(s1[e], s2[e]);
    }
    __syncthreads();
    float2* slot = slots + ((int64_t)blockIdx.x + s) * a.c;
    for (int t = threadIdx.x; t < width * VEC; t += kNormThreads) {
      const int e = t / width, q = t - e * width;
      float u = 0.f, v = 0.f;
      for (int l = 0; l < lanes; ++l) {
        const float2 f = part[e * kNormThreads + l * width + q];
        u += f.x;
        v += f.y;
      }
      slot[(first + q) * VEC + e] = make_float2(u, v);
    }
    __syncthreads();
  }
}

// One block per sample and group: the sums of its channels over the slots, and the two means that dx needs.
constexpr int kJoinThreads = 256;
__global__ void __launch_bounds__(kJoinThreads) norm_grad_join_kernel(Norm a, const float2* __restrict__ slots,
                                                                      float2* __restrict__ by_channel, float2* __restrict__ by_group) {
  __shared__ float2 part[kJoinThreads];
  const int width = min(a.d, kJoinThreads), lanes = kJoinThreads / width;
  const int lane = threadIdx.x / width, q = threadIdx.x - lane * width;
  for (int64_t t = blockIdx.x; t < (int64_t)a.b * a.g; t += gridDim.x) {
    const int s = (int)(t / a.g), gr = (int)(t - (int64_t)s * a.g);
    const int64_t begin = offset_of(a, s), end = offset_of(a, s + 1);
    float m1 = 0.f, m2 = 0.f;
    for (int k = q; k - q < a.d; k += width) {
      float u = 0.f, v = 0.f;
      if (lane < lanes && k < a.d && begin < end) {
        const int j0 = (int)(begin / a.chunk), j1 = (int)((end - 1) / a.chunk);
        for (int j = j0 + lane; j <= j1; j += lanes) {
          const float2 f = slots[((int64_t)j + s) * a.c + gr * a.d + k];
          u += f.x;
          v += f.y;
        }
      }
      part[threadIdx.x] = make_float2(u, v);
      __syncthreads();
      if (lane == 0 && k < a.d) {
        for (int l = 1; l < lanes; ++l) {
          u += part[l * width + q].x;
          v += part[l * width + q].y;
        }
        const int ch = gr * a.d + k;
        by_channel[(int64_t)s * a.c + ch] = make_float2(u, v);
        const float w = a.w ? load_any(a.w, a.p_dtype, ch) : 1.f;
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

template <typename T, int VEC>
__global__ void __launch_bounds__(kNormThreads) norm_grad_apply_kernel(Norm a, const T* __restrict__ x, const T* __restrict__ dy,
                                                                       const float* __restrict__ mean, const float* __restrict__ rstd,
                                                                       const float2* __restrict__ by_group, T* __restrict__ dx) {
  const int first = blockIdx.y * a.tile, width = min(a.tile, a.cols - first);
  const int lane = threadIdx.x / width, lanes = kNormThreads / width;
  if (lane >= lanes) return;
  const int k0 = (first + threadIdx.x - lane * width) * VEC;
  Channels<VEC> ch;
  float m1[VEC], m2[VEC];
  walk<T, VEC>(a, lane, lanes,
               [&](int s) {
                 ch.load(a, s, k0, mean, rstd);
#pragma unroll
                 for (int e = 0; e < VEC; ++e) {
                   const float2 f = __ldg(by_group + (int64_t)s * a.g + (k0 + e) / a.d);
                   m1[e] = f.x;
                   m2[e] = f.y;
                 }
               },
               [&](int64_t p, bool in) {
                 const int64_t r = row_at(a, p);
                 if (r < 0) return;
                 Pack<T, VEC> vx, vg;
                 if (in) {
                   vx.load(x + r * a.c + k0);
                   vg.load(dy + r * a.c + k0);
                   float h[VEC], z[VEC], g[VEC];
                   vx.get(h);
                   vg.get(g);
#pragma unroll
                   for (int e = 0; e < VEC; ++e) {
                     h[e] = (h[e] - ch.mean[e]) * ch.rstd[e];
                     z[e] = fmaf(h[e], ch.w[e], ch.b[e]);
                   }
                   activate_grad(z, g, a.act, a.slope);
#pragma unroll
                   for (int e = 0; e < VEC; ++e) g[e] = ch.rstd[e] * (fmaf(g[e], ch.w[e], -m1[e]) - h[e] * m2[e]);
                   vg.set(g);
                 } else {
                   vg.clear();
                 }
                 vg.store(dx + r * a.c + k0);
               });
}

// dw and db: the channels' sums over the samples, in their order
__global__ void __launch_bounds__(256) norm_grad_params_kernel(Norm a, const float2* __restrict__ by_channel, void* __restrict__ dw,
                                                               void* __restrict__ db) {
  __shared__ float2 part[256];
  const int k = blockIdx.x * 32 + (threadIdx.x & 31), lane = threadIdx.x >> 5;      // 32 channels x 8 slices of the samples
  float u = 0.f, v = 0.f;
  if (k < a.c)
    for (int s = lane; s < a.b; s += 8) {
      const float2 f = by_channel[(int64_t)s * a.c + k];
      u += f.x;
      v += f.y;
    }
  part[threadIdx.x] = make_float2(u, v);
  __syncthreads();
  if (lane == 0 && k < a.c) {
    for (int l = 1; l < 8; ++l) {
      u += part[l * 32 + threadIdx.x].x;
      v += part[l * 32 + threadIdx.x].y;
    }
    if (db) store_any(db, a.p_dtype, k, u);
    if (dw) store_any(dw, a.p_dtype, k, v);
  }
}

// ------------------------------------------------------------------------------------------------ host
bool good_dtype(int dtype) { return dtype == TSB_F32 || dtype == TSB_F16 || dtype == TSB_BF16; }

int check_norm(int64_t n, int64_t c, int64_t g, int64_t b, const void* offsets, int dtype, int p_dtype, int act) {
  if (n < 0 || c < 1 || g < 1 || c % g != 0 || b < 0 || (b && !offsets) || act < kActNone || act > kActSilu) return TSB_ERR_BAD_ARG;
  if (!good_dtype(dtype) || !good_dtype(p_dtype)) return TSB_ERR_UNSUPPORTED;
  if (n > 0x7fffffff || b > 0x3fffffff || c > 65536) return TSB_ERR_LIMIT;
  return TSB_OK;
}

Norm norm_shape(int64_t n, int64_t c, int64_t g, int64_t b, int vec) {
  Norm a{};
  a.n = n;
  a.c = (int)c;
  a.g = (int)g;
  a.d = (int)(c / g);
  a.b = (int)b;
  a.cols = (int)(c / vec);
  a.tile = a.cols < kNormThreads ? a.cols : kNormThreads;
  a.lanes = kNormThreads / a.tile;
  int64_t blocks = cdiv(n, (int64_t)a.lanes * 4);      // four rows per lane at least
  if (blocks > 2 * kSmCount) blocks = 2 * kSmCount;
  if (blocks < 1) blocks = 1;
  a.chunk = cdiv(n, blocks);
  if (a.chunk < 1) a.chunk = 1;
  a.nblk = (int)cdiv(n, a.chunk);
  return a;
}

// slots of the forward statistics for the vector width that needs the most column tiles
size_t fwd_slot_bytes(int64_t n, int64_t c, int64_t g, int64_t b) {
  const int64_t tiles = cdiv(c, kNormThreads);
  return align_up((size_t)tiles * (2 * kSmCount + b) * g * sizeof(float2), 256);
}

}  // namespace
}  // namespace tsb

using namespace tsb;

extern "C" {

size_t tsb_group_norm_fwd_workspace_bytes(int64_t n, int64_t c, int64_t g, int64_t b) {
  if (check_norm(n, c, g, 0, nullptr, 0, 0, 0) != TSB_OK || b < 0) return 0;
  return fwd_slot_bytes(n, c, g, b);
}

int tsb_group_norm_fwd(const void* x, const int32_t* order, const int32_t* offsets, const void* weight, const void* bias,
                       int64_t n, int64_t c, int64_t g, int64_t b, float eps, int32_t act, float slope, int32_t dtype,
                       int32_t param_dtype, void* y, float* mean, float* rstd, void* workspace, size_t workspace_bytes,
                       tsb_stream_t stream) {
  const int bad = check_norm(n, c, g, b, offsets, dtype, param_dtype, act);
  if (bad != TSB_OK) return bad;
  if ((n && (!x || !y)) || (b && (!mean || !rstd))) return TSB_ERR_BAD_ARG;
  cudaStream_t st = as_stream(stream);
  if (workspace_bytes < fwd_slot_bytes(n, c, g, b) || !workspace) return TSB_ERR_WORKSPACE;
  const int vec = vector_width(dtype, c, (uintptr_t)x | (uintptr_t)y);
  Norm a = norm_shape(n, c, g, b, vec);
  a.order = order;
  a.offsets = offsets;
  a.w = weight;
  a.bias = bias;
  a.p_dtype = param_dtype;
  a.eps = eps;
  a.act = act;
  a.slope = slope;
  float2* slots = static_cast<float2*>(workspace);
  const int tiles = (int)cdiv(a.cols, a.tile);
  const dim3 grid((unsigned)a.nblk, (unsigned)tiles);
  return dispatch_pack(dtype, vec, [&](auto tag) -> int {
    using T = typename decltype(tag)::T;
    constexpr int VEC = decltype(tag)::VEC;
    if (n && b) {
      if (a.d % VEC == 0) norm_stats_kernel<T, VEC, 1><<<grid, kNormThreads, 0, st>>>(a, (const T*)x, slots);
      else norm_stats_kernel<T, VEC, VEC><<<grid, kNormThreads, 0, st>>>(a, (const T*)x, slots);
      TSB_LAUNCH_CHECK();
    }
    if (b) {
      norm_join_kernel<<<grid_for((int64_t)a.b * a.g, 4), 128, 0, st>>>(a, VEC, tiles, slots, mean, rstd);
      TSB_LAUNCH_CHECK();
    }
    if (n) {
      norm_apply_kernel<T, VEC><<<grid, kNormThreads, 0, st>>>(a, (const T*)x, mean, rstd, (T*)y);
      TSB_LAUNCH_CHECK();
    }
    return TSB_OK;
  });
}

size_t tsb_group_norm_bwd_workspace_bytes(int64_t n, int64_t c, int64_t g, int64_t b) {
  if (check_norm(n, c, g, 0, nullptr, 0, 0, 0) != TSB_OK || b < 0) return 0;
  return align_up((size_t)(2 * kSmCount + b) * c * sizeof(float2), 256) + align_up((size_t)b * c * sizeof(float2), 256) +
         align_up((size_t)b * g * sizeof(float2), 256) + 256;
}

int tsb_group_norm_bwd(const void* x, const void* dy, const int32_t* order, const int32_t* offsets, const void* weight,
                       const void* bias, const float* mean, const float* rstd, int64_t n, int64_t c, int64_t g, int64_t b,
                       int32_t act, float slope, int32_t dtype, int32_t param_dtype, void* dx, void* dweight, void* dbias,
                       void* workspace, size_t workspace_bytes, tsb_stream_t stream) {
  const int bad = check_norm(n, c, g, b, offsets, dtype, param_dtype, act);
  if (bad != TSB_OK) return bad;
  if ((n && (!x || !dy || !dx)) || (b && (!mean || !rstd))) return TSB_ERR_BAD_ARG;
  cudaStream_t st = as_stream(stream);
  if (workspace_bytes < tsb_group_norm_bwd_workspace_bytes(n, c, g, b) || !workspace) return TSB_ERR_WORKSPACE;
  const int vec = vector_width(dtype, c, (uintptr_t)x | (uintptr_t)dy | (uintptr_t)dx);
  Norm a = norm_shape(n, c, g, b, vec);
  a.order = order;
  a.offsets = offsets;
  a.w = weight;
  a.bias = bias;
  a.p_dtype = param_dtype;
  a.act = act;
  a.slope = slope;
  char* ws = static_cast<char*>(workspace);
  float2* slots = reinterpret_cast<float2*>(ws);
  ws += align_up((size_t)(2 * kSmCount + b) * c * sizeof(float2), 256);
  float2* by_channel = reinterpret_cast<float2*>(ws);
  float2* by_group = reinterpret_cast<float2*>(ws + align_up((size_t)b * c * sizeof(float2), 256));
  const dim3 grid((unsigned)a.nblk, (unsigned)cdiv(a.cols, a.tile));
  return dispatch_pack(dtype, vec, [&](auto tag) -> int {
    using T = typename decltype(tag)::T;
    constexpr int VEC = decltype(tag)::VEC;
    if (n && b) {
      norm_grad_sums_kernel<T, VEC><<<grid, kNormThreads, 0, st>>>(a, (const T*)x, (const T*)dy, mean, rstd, slots);
      TSB_LAUNCH_CHECK();
    }
    if (b) {
      norm_grad_join_kernel<<<grid_for((int64_t)a.b * a.g, 1), kJoinThreads, 0, st>>>(a, slots, by_channel, by_group);
      TSB_LAUNCH_CHECK();
    }
    if (n && dx) {
      norm_grad_apply_kernel<T, VEC><<<grid, kNormThreads, 0, st>>>(a, (const T*)x, (const T*)dy, mean, rstd, by_group, (T*)dx);
      TSB_LAUNCH_CHECK();
    }
    if (dweight || dbias) {
      norm_grad_params_kernel<<<(unsigned)cdiv(a.c, 32), 256, 0, st>>>(a, by_channel, dweight, dbias);
      TSB_LAUNCH_CHECK();
    }
    return TSB_OK;
  });
}

}  // extern "C"
