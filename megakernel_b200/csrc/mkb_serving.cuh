// Shared by the batched-serving kernels: types, the packed batch's layout, and
// where a request's keys lie in the paged cache.
#pragma once

#include <cmath>
#include <cstdint>
#include <utility>
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include "../../include/mkb200.h"
#include "mkb_ptx.cuh"

namespace mkb {
namespace sv {

// ---- two values of a 16-bit type in one word, and back --------------------------
template <typename T>
struct Pair;
template <>
struct Pair<__nv_bfloat16> {
  static __device__ __forceinline__ float2 get(uint32_t u) { return make_float2(bf_lo(u), bf_hi(u)); }
  static __device__ __forceinline__ uint32_t put(float a, float b) { return pack_bf2(a, b); }
  static constexpr int kDtype = MKB_BF16;
};
template <>
struct Pair<__half> {
  static __device__ __forceinline__ float2 get(uint32_t u) { return __half22float2(*reinterpret_cast<const __half2*>(&u)); }
  static __device__ __forceinline__ uint32_t put(float a, float b) {
    const __half2 h = __floats2half2_rn(a, b);
    return *reinterpret_cast<const uint32_t*>(&h);
  }
  static constexpr int kDtype = MKB_FP16;
};

// eight consecutive values from 16 (or 32) aligned bytes
template <typename T>
__device__ __forceinline__ void load8(const T* p, float v[8]) {
  const uint4 u = *reinterpret_cast<const uint4*>(p);
  const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float2 f = Pair<T>::get(w[i]);
    v[2 * i] = f.x;
    v[2 * i + 1] = f.y;
  }
}
template <>
__device__ __forceinline__ void load8<float>(const float* p, float v[8]) {
  const float4 a = reinterpret_cast<const float4*>(p)[0], b = reinterpret_cast<const float4*>(p)[1];
  v[0] = a.x; v[1] = a.y; v[2] = a.z; v[3] = a.w;
  v[4] = b.x; v[5] = b.y; v[6] = b.z; v[7] = b.w;
}
template <typename T>
__device__ __forceinline__ uint4 pack8(const float v[8]) {
  return make_uint4(Pair<T>::put(v[0], v[1]), Pair<T>::put(v[2], v[3]), Pair<T>::put(v[4], v[5]),
                    Pair<T>::put(v[6], v[7]));
}

// ---- the packed batch ---------------------------------------------------------------

// The request of packed token `t` (every lane of a warp calls it, all with the same
// t): how many of cu[1 .. batch] are <= t. 32 probes at a time: one load deep up to
// 32 requests, two up to 1,024.
__device__ __forceinline__ int request_of(const int* cu, int batch, int t) {
  const int lane = threadIdx.x & 31;
  int lo = 0, n = batch;  // the answer lies in [lo, lo + n], cu[lo] <= t
  while (n > 0) {
    const int step = (n + 31) / 32;
    const int at = lo + (lane + 1) * step;  // probes cu[at], the last of its stretch
    const bool below = at <= lo + n && cu[at] <= t;
    const int full = __popc(__ballot_sync(0xffffffffu, below));
    lo += full * step;
    n = step == 1 ? 0 : min(step - 1, n - full * step);
  }
  return min(lo, batch - 1);
}

// Keys of a request at most: they are counted in 32 bits, with room for the tiles past the last.
constexpr int kMaxKeys = 1 << 30;

// Where packed token `t`'s request lies: its rows first .. first + n - 1, clamped to
// the batch so that no offsets of the caller's lead out of it.
struct Request {
  int b, first, n;
};
__device__ __forceinline__ Request request_rows(const int* cu, int b, int q_len, int tokens) {
  if (cu == nullptr) return {b, b * q_len, q_len};
  const int first = min(max(cu[b], 0), tokens);
  return {b, first, max(min(cu[b + 1], tokens) - first, 0)};
}
__device__ __forceinline__ Request request_at(const int* cu, int batch, int q_len, int tokens, int t) {
  return request_rows(cu, cu == nullptr ? t / q_len : request_of(cu, batch, t), q_len, tokens);
}

// ---- V that is not finite -------------------------------------------------------------
// A product over a whole tile would bring it into rows that do not see it (0 * inf = NaN),
// so it is cleared there and added to the rows that do.

// Whether one of these eight values is not finite: 0 * x + n is NaN then.
template <typename T>
__device__ __forceinline__ uint32_t odd8(const uint4& u, uint32_t n) {
  const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    if constexpr (Pair<T>::kDtype == MKB_BF16)
      asm("fma.rn.bf16x2 %0, %1, %2, %0;" : "+r"(n) : "r"(w[i]), "r"(0u));
    else
      asm("fma.rn.f16x2 %0, %1, %2, %0;" : "+r"(n) : "r"(w[i]), "r"(0u));
  }
  return n;
}
template <typename T>
__device__ __forceinline__ bool finite(uint16_t v) {
  constexpr uint32_t kExp = Pair<T>::kDtype == MKB_BF16 ? 0x7f80u : 0x7c00u;
  return (v & kExp) != kExp;
}

// Adds to z what of V's values at keys [begin, end) of request b is not finite. Warp-wide;
// the lane holds dims [lane * D / 32, + D / 32).
template <typename T, int D, bool kPaged>
__device__ __noinline__ void sum_odd(const mkb_attn_args& a, int b, int first, int hk, int begin, int end, float* z) {
  constexpr int kPer = D / 32;
  const int lane = threadIdx.x & 31;
#pragma unroll 4
  for (int j = begin; j < end; ++j) {
    int64_t vo = static_cast<int64_t>(first + j) * a.v_stride[0];
    if (kPaged) {
      const int64_t page = a.block_table[b * a.table_stride + j / a.page_size];
      if (page < 0 || page >= a.pages) continue;  // (reported by the loads)
      vo = page * a.v_stride[0] + j % a.page_size * a.v_stride[2];
    }
    const uint32_t* v = reinterpret_cast<const uint32_t*>(static_cast<const T*>(a.v) + vo + hk * a.v_stride[1]);
#pragma unroll
    for (int i = 0; i < kPer / 2; ++i) {
      const uint32_t u = v[lane * (kPer / 2) + i];
      const float2 f = Pair<T>::get(u);
      if (!finite<T>(u & 0xffffu)) z[2 * i] += f.x;
      if (!finite<T>(u >> 16)) z[2 * i + 1] += f.y;
    }
  }
}

// ---- early launch ----------------------------------------------------------------------
// A kernel of this family may be brought in while the one before it in the stream is
// still running its last blocks: it sets itself up, and waits (depend_wait) before it
// touches memory until all that came before has completed. What it reads may be written
// during its life, so its loads are plain ones: no path for read-only data, no pointer
// declared free of aliases, which would let the compiler take that path or move a load.
__device__ __forceinline__ void depend_launch() { asm volatile("griddepcontrol.launch_dependents;" ::: "memory"); }
__device__ __forceinline__ void depend_wait() { asm volatile("griddepcontrol.wait;" ::: "memory"); }

template <typename... P, typename... A>
cudaError_t launch_early(void (*kernel)(P...), int grid, int threads, size_t smem, cudaStream_t stream, A&&... args) {
  cudaLaunchConfig_t c = {};
  c.gridDim = dim3(grid);
  c.blockDim = dim3(threads);
  c.dynamicSmemBytes = smem;
  c.stream = stream;
  cudaLaunchAttribute at = {};
  at.id = cudaLaunchAttributeProgrammaticStreamSerialization;
  at.val.programmaticStreamSerializationAllowed = 1;
  c.attrs = &at;
  c.numAttrs = 1;
  return cudaLaunchKernelEx(&c, kernel, std::forward<A>(args)...);
}

// ---- testing -----------------------------------------------------------------------------
// CTA `cta` (-1: none, -2: each) loads its first `from` pieces and no more.
struct Withheld {
  int cta, from;
  __device__ __forceinline__ bool here() const { return cta != -1 && (cta == -2 || cta == static_cast<int>(blockIdx.x)); }
};
Withheld withheld();  // of a launch: mkb_attn.cu

// ---- host: what the entry points check ---------------------------------------------------
inline bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15u) == 0; }
inline bool strides_ok(const int64_t* s, int n, int unit = 8) {  // whole 16 bytes: 8 values of the 16-bit types
  for (int i = 0; i < n; ++i)
    if (s[i] < 0 || s[i] % unit) return false;
  return true;
}

// Records the first error of a launch.
__device__ __forceinline__ void report(uint32_t* status, uint32_t code) {
  if (status != nullptr) atomicCAS(status, 0u, code);
}

}  // namespace sv
}  // namespace mkb
