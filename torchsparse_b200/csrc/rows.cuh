// Shared by the operators over grouped rows (rows.cu, norm.cu): vector loads and stores of feature rows, the
// activations and the parameter loads whose type is only known at run time.
#pragma once

#include <atomic>

#include "common.cuh"

namespace tsb {

template <int BYTES>
struct RawOf;
template <>
struct RawOf<16> { using type = uint4; };
template <>
struct RawOf<8> { using type = uint2; };
template <>
struct RawOf<4> { using type = unsigned; };
template <>
struct RawOf<2> { using type = unsigned short; };

// The compiler forgets what it derived from a value: packed values that are read twice are unpacked twice, instead of being
// held unpacked in twice or four times the registers.
__device__ __forceinline__ void forget(uint4& v) { asm volatile("" : "+r"(v.x), "+r"(v.y), "+r"(v.z), "+r"(v.w)); }
__device__ __forceinline__ void forget(uint2& v) { asm volatile("" : "+r"(v.x), "+r"(v.y)); }
__device__ __forceinline__ void forget(unsigned& v) { asm volatile("" : "+r"(v)); }
__device__ __forceinline__ void forget(unsigned short& v) { asm volatile("" : "+h"(v)); }

// VEC neighbouring values of a row, moved as one load or store of VEC * sizeof(T) bytes
template <typename T, int VEC>
struct Pack {
  using Raw = typename RawOf<(int)sizeof(T) * VEC>::type;
  Raw raw;
  __device__ __forceinline__ void load(const T* p) { raw = __ldg(reinterpret_cast<const Raw*>(p)); }
  __device__ __forceinline__ void store(T* p) const { *reinterpret_cast<Raw*>(p) = raw; }
  static constexpr int kBytes = VEC * (int)sizeof(T);
  __device__ __forceinline__ void clear() { raw = Raw{}; }
  __device__ __forceinline__ void get(float (&v)[VEC]) const {
    const T* e = reinterpret_cast<const T*>(&raw);
#pragma unroll
    for (int i = 0; i < VEC; ++i) v[i] = to_f32(e[i]);
  }
  __device__ __forceinline__ void set(const float (&v)[VEC]) {
    T* e = reinterpret_cast<T*>(&raw);
#pragma unroll
    for (int i = 0; i < VEC; ++i) e[i] = from_f32<T>(v[i]);
  }
};

// Largest vector (in elements, up to 16 bytes) that divides a row of c elements and to which every base pointer is
// aligned; `bits` is the OR of the pointers.
inline int vector_width(int dtype, int64_t c, uintptr_t bits) {
  const int size = (int)dtype_size(dtype);
  for (int bytes = 16; bytes > size; bytes >>= 1)
    if (((c * size) % bytes == 0) && (bits % bytes == 0)) return bytes / size;
  return 1;
}

template <typename T_, int VEC_>
struct PackTag {
  using T = T_;
  static constexpr int VEC = VEC_;
};

// Vectors that cp.async can move: all but the single 16-bit value.
template <typename T, int VEC>
constexpr bool kAsyncVector = VEC * sizeof(T) >= 4;

// f(PackTag<T, VEC>()) for the type and vector width found at run time
template <typename F>
inline int dispatch_pack(int dtype, int vec, F&& f) {
  switch (dtype) {
    case TSB_F32:
      switch (vec) {
        case 4: return f(PackTag<float, 4>());
        case 2: return f(PackTag<float, 2>());
        default: return f(PackTag<float, 1>());
      }
    case TSB_F16:
      switch (vec) {
        case 8: return f(PackTag<__half, 8>());
        case 4: return f(PackTag<__half, 4>());
        case 2: return f(PackTag<__half, 2>());
        default: return f(PackTag<__half, 1>());
      }
    case TSB_BF16:
      switch (vec) {
        case 8: return f(PackTag<__nv_bfloat16, 8>());
        case 4: return f(PackTag<__nv_bfloat16, 4>());
        case 2: return f(PackTag<__nv_bfloat16, 2>());
        default: return f(PackTag<__nv_bfloat16, 1>());
      }
  }
  return TSB_ERR_UNSUPPORTED;
}

// Row and vector of a flat index over rows of `cols` vectors, without a 64-bit division: m = floor(2^64 / cols) + 1 gives the
// exact quotient while index * cols < 2^64.
struct RowSplit {
  uint64_t m;
  unsigned cols;
  __device__ __forceinline__ int64_t row(int64_t t) const { return m ? (int64_t)__umul64hi((uint64_t)t, m) : t; }
};
inline RowSplit row_split(int64_t cols) { return RowSplit{cols == 1 ? 0 : ~0ull / (uint64_t)cols + 1, (unsigned)cols}; }
// A launch has fewer than 2^31 blocks, which the entries check, and a block at most 4096 vectors of the result: a flat index
// is below 2^43 + 2^12, and with rows of at most 2^20 vectors index * cols stays below 2^64.
constexpr int64_t kMaxChannels = 1 << 20;

// One value of an array whose type is a run-time argument (parameters, router weights: few values, read once).
__device__ __forceinline__ float load_any(const void* p, int dtype, int64_t i) {
  if (dtype == TSB_F32) return __ldg(reinterpret_cast<const float*>(p) + i);
  if (dtype == TSB_F16) return to_f32(reinterpret_cast<const __half*>(p)[i]);
  return to_f32(reinterpret_cast<const __nv_bfloat16*>(p)[i]);
}
__device__ __forceinline__ void store_any(void* p, int dtype, int64_t i, float v) {
  if (dtype == TSB_F32) reinterpret_cast<float*>(p)[i] = v;
  else if (dtype == TSB_F16) reinterpret_cast<__half*>(p)[i] = from_f32<__half>(v);
  else reinterpret_cast<__nv_bfloat16*>(p)[i] = from_f32<__nv_bfloat16>(v);
}

// launches a kernel with BYTES of dynamic shared memory, which its device has to be told of once
template <auto KERNEL, int BYTES, typename... Q>
inline int launch_wide(dim3 grid, int threads, cudaStream_t st, Q... args) {
  if (BYTES > 0) {
    static std::atomic<bool> told[64];
    int dev = 0;
    TSB_CUDA_TRY(cudaGetDevice(&dev));
    if (dev >= 64 || !told[dev].load(std::memory_order_acquire)) {
      TSB_CUDA_TRY(cudaFuncSetAttribute(KERNEL, cudaFuncAttributeMaxDynamicSharedMemorySize, BYTES));
      if (dev < 64) told[dev].store(true, std::memory_order_release);
    }
  }
  KERNEL<<<grid, threads, BYTES, st>>>(args...);
  TSB_LAUNCH_CHECK();
  return TSB_OK;
}

// 4, 8 or 16 bytes into shared memory without passing through registers; commit closes a group, wait<N> leaves the N newest
// open
template <int BYTES>
__device__ __forceinline__ void async_copy(void* to, const void* from) {
  const unsigned at = (unsigned)__cvta_generic_to_shared(to);
  if constexpr (BYTES == 16) asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(at), "l"(from) : "memory");
  else asm volatile("cp.async.ca.shared.global [%0], [%1], %2;" ::"r"(at), "l"(from), "n"(BYTES) : "memory");
}
__device__ __forceinline__ void async_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void async_wait() {
  asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}

}  // namespace tsb
