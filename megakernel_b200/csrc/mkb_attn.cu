// Attention of a packed batch: prompt_attention (keys packed like the queries) and
// paged_attention (keys in the paged cache).
//
//   out_i = sum_j p_ij v_j / sum_j p_ij,  p_ij = exp(scale q_i.k_j - max_j),  j <= pos(i)
//
// One warp per token and query head: a lane scores one key of 32 at a time, the
// running maximum and sum are kept in FP32, and the lanes then share the head's
// dimensions for the weighted sum of the 32 value rows.

#include <cmath>

#include "mkb_serving.cuh"

namespace mkb {
namespace sv {

template <typename T, int D, bool kPaged>
__global__ void __launch_bounds__(128) attn_rows_kernel(const mkb_attn_args a) {
  __shared__ float qs[4][D];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int64_t job = (int64_t)blockIdx.x * 4 + warp;
  const int t = static_cast<int>(job / a.heads), h = static_cast<int>(job % a.heads);
  if (t >= a.tokens) return;
  const int hk = h / (a.heads / a.kv_heads);
  const Request rq = request_at(a.cu_q, a.batch, a.q_len, a.tokens, t);
  const int b = rq.b, first = rq.first, at = t - first;
  const int len = kPaged ? a.kv_lens[b] : rq.n;
  const int keys = at >= 0 && at < rq.n ? len - rq.n + at + 1 : 0;  // the keys this token sees
  const T* q = static_cast<const T*>(a.q) + t * a.q_stride[0] + h * a.q_stride[1];
  for (int d = lane; d < D / 2; d += 32) {
    const float2 f = Pair<T>::get(reinterpret_cast<const uint32_t*>(q)[d]);
    qs[warp][2 * d] = f.x;
    qs[warp][2 * d + 1] = f.y;
  }
  __syncwarp();
  constexpr int kPer = D / 32;  // dimensions of a lane in the weighted sum
  float m = -INFINITY, l = 0.f, o[kPer] = {};
  uint32_t bad = 0;
  if (kPaged && (int64_t)len > (int64_t)a.table_width * a.page_size) bad = MKB_SERVE_BAD_LENGTH;
  for (int j0 = 0; j0 < keys && bad == 0; j0 += 32) {
    const int j = j0 + lane;
    int64_t ko = 0, vo = 0;
    bool sees = j < keys;
    if (sees) {
      if (kPaged) {
        const int64_t page = a.block_table[b * a.table_stride + j / a.page_size], slot = j % a.page_size;
        if (page < 0 || page >= a.pages) {
          bad = MKB_SERVE_BAD_PAGE;
          sees = false;
        } else {
          ko = page * a.k_stride[0] + hk * a.k_stride[1] + slot * a.k_stride[2];
          vo = page * a.v_stride[0] + hk * a.v_stride[1] + slot * a.v_stride[2];
        }
      } else {
        ko = (int64_t)(first + j) * a.k_stride[0] + hk * a.k_stride[1];
        vo = (int64_t)(first + j) * a.v_stride[0] + hk * a.v_stride[1];
      }
    }
    bad = __reduce_max_sync(0xffffffffu, bad);
    if (bad != 0) break;
    float s = -INFINITY;
    if (sees) {
      const T* k = static_cast<const T*>(a.k) + ko;
      s = 0.f;
#pragma unroll 4
      for (int d = 0; d < D; d += 8) {
        float kv[8];
        load8(k + d, kv);
#pragma unroll
        for (int i = 0; i < 8; ++i) s += qs[warp][d + i] * kv[i];
      }
      s *= a.scale;
    }
    float mx = s;
#pragma unroll
    for (int w = 16; w > 0; w >>= 1) {
      const float y = __shfl_xor_sync(0xffffffffu, mx, w);
      mx = (mx != mx || y != y) ? NAN : fmaxf(mx, y);
    }
    const float mn = mx != mx ? NAN : fmaxf(m, mx);
    const float sc = m == -INFINITY ? 0.f : expf(m - mn);  // nothing summed yet
    const float p = sees ? expf(s - mn) : 0.f;
    float ps = p;
#pragma unroll
    for (int w = 16; w > 0; w >>= 1) ps += __shfl_xor_sync(0xffffffffu, ps, w);
    l = l * sc + ps;
#pragma unroll
    for (int i = 0; i < kPer; ++i) o[i] *= sc;
    for (int jj = 0; jj < min(32, keys - j0); ++jj) {
      const float pj = __shfl_sync(0xffffffffu, p, jj);
      const T* v = static_cast<const T*>(a.v) + __shfl_sync(0xffffffffu, vo, jj);
#pragma unroll
      for (int i = 0; i < kPer / 2; ++i) {
        const float2 f = Pair<T>::get(reinterpret_cast<const uint32_t*>(v)[lane * (kPer / 2) + i]);
        o[2 * i] += pj * f.x;
        o[2 * i + 1] += pj * f.y;
      }
    }
    m = mn;
  }
  if (bad != 0 && lane == 0) report(a.status, bad);
  const float inv = bad != 0 ? NAN : keys > 0 ? 1.f / l : 0.f;
  T* out = static_cast<T*>(a.out) + t * a.out_stride[0] + h * a.out_stride[1];
#pragma unroll
  for (int i = 0; i < kPer / 2; ++i)
    reinterpret_cast<uint32_t*>(out)[lane * (kPer / 2) + i] = Pair<T>::put(o[2 * i] * inv, o[2 * i + 1] * inv);
}

template <typename T, int D, bool kPaged>
cudaError_t launch_rows(const mkb_attn_args& a, cudaStream_t stream) {
  const int64_t jobs = (int64_t)a.tokens * a.heads;
  attn_rows_kernel<T, D, kPaged><<<static_cast<unsigned>((jobs + 3) / 4), 128, 0, stream>>>(a);
  return cudaGetLastError();
}
template <typename T, bool kPaged>
cudaError_t launch_dim(const mkb_attn_args& a, cudaStream_t stream) {
  return a.head_dim == 128 ? launch_rows<T, 128, kPaged>(a, stream) : launch_rows<T, 64, kPaged>(a, stream);
}


cudaError_t attn_tc(const mkb_attn_args& a, bool paged, cudaStream_t stream);  // mkb_attn_tc.cu
size_t tc_workspace(const mkb_attn_args& a);

static bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15u) == 0; }
static bool strides_ok(const int64_t* s, int n) {
  for (int i = 0; i < n; ++i)
    if (s[i] < 0 || s[i] % 8) return false;
  return true;
}

// What both entry points refuse before a launch.
static cudaError_t check_attn(const mkb_attn_args* a, bool paged) {
  if (a == nullptr || a->tokens < 0 || a->batch < 0) return cudaErrorInvalidValue;
  if (a->tokens > 0 && a->batch == 0) return cudaErrorInvalidValue;
  if (a->dtype != MKB_BF16 && a->dtype != MKB_FP16) return cudaErrorInvalidValue;
  if (a->head_dim != 64 && a->head_dim != 128) return cudaErrorInvalidValue;
  if (a->kv_heads < 1 || a->heads < 1 || a->heads % a->kv_heads) return cudaErrorInvalidValue;
  if (!(a->scale > 0.f) || std::isinf(a->scale)) return cudaErrorInvalidValue;
  if (a->tokens == 0) return cudaSuccess;
  if (a->cu_q == nullptr && (a->q_len < 1 || (int64_t)a->q_len * a->batch != a->tokens)) return cudaErrorInvalidValue;
  if (!a->q || !a->out) return cudaErrorInvalidValue;
  // rows of a KV head, and their blocks over all of them, are counted in 32 bits
  if (a->heads / a->kv_heads > 128 || static_cast<int64_t>(a->tokens) + a->batch > (1ll << 30) / a->heads)
    return cudaErrorInvalidValue;
  if (paged) {
    if (!a->kv_lens || a->table_width < 0 || a->pages < 0) return cudaErrorInvalidValue;
    if (a->table_width > 0 && !a->block_table) return cudaErrorInvalidValue;
    if (a->pages > 0 && (!a->k || !a->v)) return cudaErrorInvalidValue;
    if (a->page_size < 16 || (a->page_size & (a->page_size - 1))) return cudaErrorInvalidValue;
  } else if (!a->k || !a->v) {
    return cudaErrorInvalidValue;
  }
  if (!aligned16(a->q) || !aligned16(a->k) || !aligned16(a->v) || !aligned16(a->out) || !aligned16(a->workspace) ||
      !strides_ok(a->q_stride, 2) || !strides_ok(a->out_stride, 2) || !strides_ok(a->k_stride, paged ? 3 : 2) ||
      !strides_ok(a->v_stride, paged ? 3 : 2))
    return cudaErrorMisalignedAddress;
  // rows lie at places of their own; KV heads may share one
  if ((a->tokens > 1 && (!a->q_stride[0] || !a->out_stride[0])) || (a->heads > 1 && (!a->q_stride[1] || !a->out_stride[1])))
    return cudaErrorInvalidValue;
  if (paged ? a->pages > 0 && ((a->pages > 1 && (!a->k_stride[0] || !a->v_stride[0])) || !a->k_stride[2] || !a->v_stride[2])
            : a->tokens > 1 && (!a->k_stride[0] || !a->v_stride[0]))
    return cudaErrorInvalidValue;
  return cudaSuccess;
}

}  // namespace sv
}  // namespace mkb

extern "C" {

size_t mkb_attn_workspace_bytes(const mkb_attn_args* a) {
  return mkb::sv::tc_workspace(*a);
}

cudaError_t mkb_attn_workspace_reset(void* workspace, size_t bytes, cudaStream_t stream) {
  return cudaMemsetAsync(workspace, 0, bytes, stream);
}

cudaError_t mkb_prompt_attention(const mkb_attn_args* a, cudaStream_t stream) {
  using namespace mkb::sv;
  const cudaError_t e = check_attn(a, false);
  if (e != cudaSuccess || a->tokens == 0) return e;
  return attn_tc(*a, false, stream);
}

cudaError_t mkb_paged_attention(const mkb_attn_args* a, cudaStream_t stream) {
  using namespace mkb::sv;
  const cudaError_t e = check_attn(a, true);
  if (e != cudaSuccess || a->tokens == 0) return e;
  if (a->cu_q != nullptr || a->q_len > 1) return attn_tc(*a, true, stream);
  return a->dtype == MKB_BF16 ? launch_dim<__nv_bfloat16, true>(*a, stream) : launch_dim<__half, true>(*a, stream);
}
}
