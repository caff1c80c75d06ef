// The attention entry points: what they refuse, and which kernel runs.

#include <atomic>
#include <cmath>

#include "mkb_serving.cuh"

namespace mkb {
namespace sv {

cudaError_t attn_tc(const mkb_attn_args& a, bool paged, cudaStream_t stream);  // mkb_attn_tc.cu
size_t tc_workspace(const mkb_attn_args& a);
cudaError_t attn_decode(const mkb_attn_args& a, cudaStream_t stream);  // mkb_attn_decode.cu
size_t decode_workspace(const mkb_attn_args& a);
bool decode_fits(const mkb_attn_args& a);
size_t counter_bytes();  // at the start of either's workspace

static std::atomic<Withheld> g_withheld{Withheld{-1, 0}};
Withheld withheld() { return g_withheld.load(std::memory_order_relaxed); }

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
  if (a == nullptr || (a->head_dim != 64 && a->head_dim != 128)) return 0;
  // (their counters share their place: both leave them zero)
  const size_t t = mkb::sv::tc_workspace(*a), d = mkb::sv::decode_workspace(*a);
  return t > d ? t : d;
}

cudaError_t mkb_attn_workspace_reset(void* workspace, size_t bytes, cudaStream_t stream) {
  // the counters: partial results are written before they are read
  const size_t counters = mkb::sv::counter_bytes();
  return cudaMemsetAsync(workspace, 0, bytes < counters ? bytes : counters, stream);
}

void mkb_attn_withhold(int cta, int from) { mkb::sv::g_withheld.store({cta, from}); }

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
  // Few rows known from the shapes alone: bytes bound the call, and the streaming kernel reads
  // them fastest (both sides measured: decode_fits). More rows, or chunks of lengths that only
  // the device knows: the tensor-core tiles.
  return decode_fits(*a) ? attn_decode(*a, stream) : attn_tc(*a, true, stream);
}
}
