// paged_append: from the QKV projection of a packed batch to the attention's inputs.
//
//   q, k heads:  y = x / sqrt(mean(x^2) + eps) * w   (where the norm has a weight)
//                out[i] = y[i] cos[p, i] + rot(y)[i] sin[p, i],  rot(y) = (-y[D/2:], y[:D/2])
//   v heads:     out = x
// at the token's position p; q goes to q_out, k and v to slot p % page_size of page
// block_table[b, p / page_size] (k also to k_out where a prompt's attention follows).
//
// All FP32 inside, one rounding to the cache's type at the store (the attention's
// operands are 16-bit). The kernel moves bytes: each head is read once and written
// once. A row of D values is D / 16 lanes wide, a lane holding eight values of the
// low half and the eight of the high half that RoPE pairs with them, so the rotation
// needs no exchange, every access is 16 bytes, and the norm's sum is log2(D / 16)
// shuffles. One block per token: its heads share the request, the page and the
// cos / sin values. A block waits for one lookup after another (request, length, page,
// tables), so blocks in flight carry the bandwidth: six of an SM at 80 registers, where
// the compiler's own 111 left four. 16,000 tokens from FP32: 71 us, 5.7 TB/s of the 6.6
// that a copy reaches (four blocks: 84 us; eight, with spills: 75).

#include "mkb_serving.cuh"

namespace mkb {
namespace sv {

constexpr int kAppendThreads = 128;

// Eight values as they lie in memory.
template <typename S>
struct Raw8 {
  uint4 v[sizeof(S) / 2];
  __device__ __forceinline__ void load(const S* p) {
#pragma unroll
    for (int i = 0; i < static_cast<int>(sizeof(S)) / 2; ++i) v[i] = __ldcs(reinterpret_cast<const uint4*>(p) + i);
  }
  __device__ __forceinline__ void get(float x[8]) const {
    if constexpr (sizeof(S) == 4) {
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        x[4 * i] = __uint_as_float(v[i].x);
        x[4 * i + 1] = __uint_as_float(v[i].y);
        x[4 * i + 2] = __uint_as_float(v[i].z);
        x[4 * i + 3] = __uint_as_float(v[i].w);
      }
    } else {
      const uint32_t w[4] = {v[0].x, v[0].y, v[0].z, v[0].w};
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const float2 f = Pair<S>::get(w[i]);
        x[2 * i] = f.x;
        x[2 * i + 1] = f.y;
      }
    }
  }
};

template <typename S, typename T, int D>
__global__ void __launch_bounds__(kAppendThreads, 6) append_kernel(const mkb_append_args a) {
  constexpr int kLanes = D / 16;                    // lanes of a head
  constexpr int kRows = kAppendThreads / kLanes;    // heads of a block at a time
  const int t = blockIdx.x;
  const int part = threadIdx.x % kLanes;
  const int row0 = threadIdx.x / kLanes;
  const int d0 = 8 * part, d1 = D / 2 + 8 * part;
  const int rows = a.heads + 2 * a.kv_heads;

  depend_launch();
  depend_wait();
  Raw8<S> lo, hi;  // the next head's values, asked for before anything else is known
  auto fetch = [&](int row) {
    if (row >= rows) return;
    const S* src = static_cast<const S*>(a.qkv) + t * a.qkv_stride[0] + row * a.qkv_stride[1];
    lo.load(src + d0);
    hi.load(src + d1);
  };
  fetch(row0);
  const Request rq = request_at(a.cu_q, a.batch, a.q_len, a.tokens, t);
  const int b = rq.b, at = t - rq.first;
  const int pos = at >= 0 && at < rq.n ? max(a.kv_lens[b], 0) - rq.n + at : -1;
  int64_t page = -1;
  uint32_t bad = 0;
  if (pos >= 0) {
    const int entry = pos >> (31 - __clz(a.page_size));
    if (pos >= a.rope_rows) {
      bad = MKB_SERVE_BAD_POSITION;
    } else if (entry >= a.table_width) {
      bad = MKB_SERVE_BAD_LENGTH;
    } else {
      page = a.block_table[b * a.table_stride + entry];
      if (page < 0 || page >= a.pages) bad = MKB_SERVE_BAD_PAGE;
    }
  }
  if (bad != 0 && threadIdx.x == 0) report(a.status, bad);
  const bool store = pos >= 0 && bad == 0;
  const int64_t slot = pos & (a.page_size - 1);

  float cs[16], sn[16];
  if (store) {
    const size_t r = (size_t)pos * D;
    if (a.rope_fp32) {
      const float* c = static_cast<const float*>(a.cos_table) + r;
      const float* s = static_cast<const float*>(a.sin_table) + r;
      load8(c + d0, cs);
      load8(c + d1, cs + 8);
      load8(s + d0, sn);
      load8(s + d1, sn + 8);
    } else {
      const T* c = static_cast<const T*>(a.cos_table) + r;
      const T* s = static_cast<const T*>(a.sin_table) + r;
      load8(c + d0, cs);
      load8(c + d1, cs + 8);
      load8(s + d0, sn);
      load8(s + d1, sn + 8);
    }
  }
  // no such position: zeros, or NaN where that is an error, whatever the token holds
  const uint32_t none = bad != 0 ? 0x7fff7fffu : 0u;

  for (int r0 = 0; r0 < rows; r0 += kRows) {
    const int row = r0 + row0;
    const bool live = row < rows;
    float x[16];
    lo.get(x);
    hi.get(x + 8);
    fetch(row + kRows);
    const bool is_v = row >= a.heads + a.kv_heads;
    const void* weight = row < a.heads ? a.q_norm : a.k_norm;
    if (a.q_norm != nullptr || a.k_norm != nullptr) {  // uniform: every lane takes the shuffles
      float ss = 0.f;
#pragma unroll
      for (int i = 0; i < 16; ++i) ss += live ? x[i] * x[i] : 0.f;
#pragma unroll
      for (int o = kLanes / 2; o > 0; o /= 2) ss += __shfl_xor_sync(0xffffffffu, ss, o);
      if (live && !is_v && weight != nullptr) {
        const float rstd = rsqrtf(ss * (1.0f / D) + a.eps);
        float w[16];
        load8(static_cast<const T*>(weight) + d0, w);
        load8(static_cast<const T*>(weight) + d1, w + 8);
#pragma unroll
        for (int i = 0; i < 16; ++i) x[i] = x[i] * rstd * w[i];
      }
    }
    if (!live) continue;
    if (!is_v) {
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const float lo = x[i], hi = x[i + 8];
        x[i] = lo * cs[i] - hi * sn[i];
        x[i + 8] = hi * cs[i + 8] + lo * sn[i + 8];
      }
    }
    uint4 u0 = pack8<T>(x), u1 = pack8<T>(x + 8);
    if (!store) u0 = u1 = make_uint4(none, none, none, none);
    T* dst = nullptr;
    if (row < a.heads) {
      dst = static_cast<T*>(a.q_out) + ((size_t)t * a.heads + row) * D;
    } else if (store) {
      const int64_t h = row - a.heads - (is_v ? a.kv_heads : 0);
      const int64_t* st = is_v ? a.v_stride : a.k_stride;
      dst = static_cast<T*>(is_v ? a.v_cache : a.k_cache) + page * st[0] + h * st[1] + slot * st[2];
    }
    if (dst != nullptr) {
      *reinterpret_cast<uint4*>(dst + d0) = u0;
      *reinterpret_cast<uint4*>(dst + d1) = u1;
    }
    if (a.k_out != nullptr && row >= a.heads && !is_v) {
      T* k = static_cast<T*>(a.k_out) + ((size_t)t * a.kv_heads + row - a.heads) * D;
      *reinterpret_cast<uint4*>(k + d0) = u0;
      *reinterpret_cast<uint4*>(k + d1) = u1;
    }
  }
}

template <typename S, typename T>
cudaError_t append_dim(const mkb_append_args& a, cudaStream_t stream) {
  if (a.head_dim == 128) return launch_early(append_kernel<S, T, 128>, a.tokens, kAppendThreads, 0, stream, a);
  return launch_early(append_kernel<S, T, 64>, a.tokens, kAppendThreads, 0, stream, a);
}
template <typename T>
cudaError_t append_source(const mkb_append_args& a, cudaStream_t stream) {
  if (a.source_dtype == MKB_BF16) return append_dim<__nv_bfloat16, T>(a, stream);
  if (a.source_dtype == MKB_FP16) return append_dim<__half, T>(a, stream);
  return append_dim<float, T>(a, stream);
}

}  // namespace sv
}  // namespace mkb

extern "C" cudaError_t mkb_paged_append(const mkb_append_args* a, cudaStream_t stream) {
  using namespace mkb::sv;
  if (a == nullptr || a->tokens < 0 || a->batch < 0) return cudaErrorInvalidValue;
  if (a->tokens == 0 || a->batch == 0) return a->tokens == 0 ? cudaSuccess : cudaErrorInvalidValue;
  if ((a->dtype != MKB_BF16 && a->dtype != MKB_FP16) || a->source_dtype < MKB_BF16 || a->source_dtype > MKB_FP32)
    return cudaErrorInvalidValue;
  if ((a->head_dim != 64 && a->head_dim != 128) || a->heads < 1 || a->kv_heads < 1) return cudaErrorInvalidValue;
  if (a->cu_q == nullptr && (a->q_len < 1 || (int64_t)a->q_len * a->batch != a->tokens)) return cudaErrorInvalidValue;
  if (a->page_size < 16 || (a->page_size & (a->page_size - 1)) || a->pages < 0 || a->table_width < 0 || a->rope_rows < 0) return cudaErrorInvalidValue;
  if (!a->qkv || !a->q_out || !a->kv_lens) return cudaErrorInvalidValue;
  // (no pages, entries or positions: no memory of them either)
  if ((a->pages > 0 && (!a->k_cache || !a->v_cache)) || (a->table_width > 0 && !a->block_table) ||
      (a->rope_rows > 0 && (!a->cos_table || !a->sin_table)))
    return cudaErrorInvalidValue;
  if (!aligned16(a->qkv) || !aligned16(a->q_norm) || !aligned16(a->k_norm) || !aligned16(a->cos_table) ||
      !aligned16(a->sin_table) || !aligned16(a->q_out) || !aligned16(a->k_out) || !aligned16(a->k_cache) ||
      !aligned16(a->v_cache) || !strides_ok(a->qkv_stride, 2, a->source_dtype == MKB_FP32 ? 4 : 8) || !strides_ok(a->k_stride, 3) ||
      !strides_ok(a->v_stride, 3))
    return cudaErrorMisalignedAddress;
  for (const int64_t* s : {a->k_stride, a->v_stride})  // every row is written at a place of its own
    if (a->pages > 0 && ((a->pages > 1 && !s[0]) || (a->kv_heads > 1 && !s[1]) || !s[2])) return cudaErrorInvalidValue;
  return a->dtype == MKB_BF16 ? append_source<__nv_bfloat16>(*a, stream) : append_source<__half>(*a, stream);
}
