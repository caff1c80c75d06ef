// Attention of few new tokens a request over the paged cache: the decode step.
//
//   out_i = sum_j p_ij v_j / sum_j p_ij,  p_ij = 2^(c q_i.k_j - m_i),  c = scale log2(e),  j <= pos(i)
//
// Every key and value is read once from memory and used for the handful of rows (new
// tokens x the query heads that share the KV head, 16 at most) that need it: bytes bound
// this kernel, at 4 D bytes a key and KV head. It reads them straight into shared memory
// (cp.async, 16 bytes a lane, chunks swizzled within a row so that the matrix loads below
// meet no bank twice), a ring of stages per warp, with no barrier between warps: a warp
// waits for its own copies only.
//
// The products run on mma.sync m16n8k16 with the keys as the 16 rows of S^T = K Q^T and
// the queries as its columns (8 or 16 of them), so that the tile is filled by keys however
// few the queries are: S^T's accumulators, transposed by movmatrix, are the B operand of
// O^T += V^T P^T, and V^T comes from V by ldmatrix.trans. P enters as a 16-bit high part
// and the remainder: memory leaves time for the second product, and P then costs no
// precision.
//
// Work: the requests' tiles of 16 keys, KV head by KV head, are laid end to end and cut
// into equal ranges, one a CTA; a CTA's warps take every eighth tile of each
// stretch that belongs to one request and KV head, and add up at its end. A stretch that
// is not the whole of its keys leaves O, maximum and sum in memory; the last one to be done
// adds them up in order.

#include <cmath>

#include "mkb_serving.cuh"

namespace mkb {
namespace sv {

constexpr int kDecWarps = 8;
constexpr int kTileKeys = 16;  // keys of a tile: the rows of one mma
constexpr int kDecTileMin = 16;  // tiles (of 16 keys) that are worth a CTA

struct DecArgs {
  mkb_attn_args a;
  float sl2;
  int group, rows;     // query heads of a KV head; rows (q_len * group)
  uint32_t* counters;  // [ctas], zero between calls
  float* part;         // [2 ctas][D][16] O^T, then its maxima and sums [2 ctas][2][16]
  float* stat;
};

template <int D>
struct DecShape {
  static constexpr int kStages = D == 128 ? 3 : 6;       // tiles of a warp in flight (one being worked on)
  static constexpr int kStageBytes = kTileKeys * D * 2 * 2;  // K and V
  static constexpr size_t kSmem = static_cast<size_t>(kDecWarps) * kStages * kStageBytes;
};

__device__ __forceinline__ void cp_async16(uint32_t dst, const void* src, bool there) {
  const int n = there ? 16 : 0;  // 0: zeros, nothing is read
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(n) : "memory");
}
__device__ __forceinline__ void cp_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void cp_wait() {
  asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}
__device__ __forceinline__ void ldsm4(uint32_t addr, uint32_t r[4]) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0, %1, %2, %3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr));
}
__device__ __forceinline__ void ldsm4_t(uint32_t addr, uint32_t r[4]) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0, %1, %2, %3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr));
}
__device__ __forceinline__ uint32_t transpose8x8(uint32_t v) {
  uint32_t r;
  asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(v));
  return r;
}
template <typename T>
__device__ __forceinline__ void mma16816(float c[4], const uint32_t a[4], uint32_t b0, uint32_t b1) {
  if constexpr (Pair<T>::kDtype == MKB_BF16)
    asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
  else
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

// Tiles of a request (one for a request without keys: its zeros have to be written).
__device__ __forceinline__ int dec_tiles(const DecArgs& g, int b, int* len_out, bool* bad_out) {
  const int len = max(__ldg(g.a.kv_lens + b), 0);
  const bool bad = static_cast<int64_t>(len) > static_cast<int64_t>(g.a.table_width) * g.a.page_size;
  *len_out = len;
  *bad_out = bad;
  return bad ? 1 : max((len + kTileKeys - 1) / kTileKeys, 1);
}

// kN: columns of 8 rows each (1 or 2)
template <typename T, int D, int kN>
__global__ void __launch_bounds__(32 * kDecWarps, 1) attn_decode_kernel(const __grid_constant__ DecArgs g) {
  using Shape = DecShape<D>;
  constexpr int kStages = Shape::kStages, kChunks = D / 8;  // 16-byte chunks of a row
  extern __shared__ __align__(128) uint8_t smem[];
  __shared__ float red_m[kDecWarps][16], red_l[kDecWarps][16];
  __shared__ int flag;
  __shared__ uint32_t odd_rows;  // rows whose O is not finite
  const mkb_attn_args& a = g.a;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  depend_launch();
  const uint32_t ring = smem_addr(smem) + warp * (kStages * Shape::kStageBytes);
  depend_wait();

  // ---- this CTA's range of tiles ---------------------------------------------------------
  // (every warp works it out for itself; a lane keeps the first 32 requests' tiles)
  int len0 = 0;
  bool bad0 = false;
  const int tiles0 = lane < a.batch ? dec_tiles(g, lane, &len0, &bad0) : 0;
  int64_t total = 0;
  for (int b0 = 0; b0 < a.batch; b0 += 32) {
    int n = tiles0, x;
    bool y;
    if (b0 > 0) n = b0 + lane < a.batch ? dec_tiles(g, b0 + lane, &x, &y) : 0;
    total += __reduce_add_sync(0xffffffffu, n);
  }
  total *= a.kv_heads;
  // a CTA for every kDecTileMin tiles, or for every request and KV head if those are more
  const int64_t heads = static_cast<int64_t>(a.batch) * a.kv_heads;
  const int ctas = static_cast<int>(min(static_cast<int64_t>(gridDim.x), max(total / kDecTileMin, heads)));
  const int cta = blockIdx.x;
  if (cta >= ctas) return;
  const double per = static_cast<double>(total) / ctas;
  auto cut = [&](int c) { return c >= ctas ? total : static_cast<int64_t>(per * c); };
  const int64_t from = cut(cta), to = cut(cta + 1);
  int b = a.batch, n = 0, len = 0, hk = 0;
  bool bad = false;
  int64_t pos = 0;  // tiles before the stretch's request and KV head
  for (int b0 = 0; b0 < a.batch; b0 += 32) {
    int t = tiles0, ln = len0;
    bool bd = bad0;
    if (b0 > 0) t = b0 + lane < a.batch ? dec_tiles(g, b0 + lane, &ln, &bd) : 0;
    int64_t inc = static_cast<int64_t>(t) * a.kv_heads;
    const int64_t own = inc;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int64_t y = __shfl_up_sync(0xffffffffu, inc, o);
      if (lane >= o) inc += y;
    }
    const uint32_t who = __ballot_sync(0xffffffffu, from - pos < inc);
    if (who != 0) {
      const int src = __ffs(who) - 1;
      b = b0 + src;
      n = __shfl_sync(0xffffffffu, t, src);
      len = __shfl_sync(0xffffffffu, ln, src);
      bad = __shfl_sync(0xffffffffu, static_cast<int>(bd), src) != 0;
      pos += __shfl_sync(0xffffffffu, inc - own, src);
      hk = static_cast<int>((from - pos) / n);
      pos += static_cast<int64_t>(n) * hk;
      break;
    }
    pos += __shfl_sync(0xffffffffu, inc, 31);
  }

  // ---- stretches ----------------------------------------------------------------------------
  while (pos < to && b < a.batch) {
    const int t0 = static_cast<int>(max(from - pos, static_cast<int64_t>(0)));
    const int t1 = static_cast<int>(min(to - pos, static_cast<int64_t>(n)));
    uint32_t page_bad = 0;
    const T* kbase = static_cast<const T*>(a.k) + hk * a.k_stride[1];
    const T* vbase = static_cast<const T*>(a.v) + hk * a.v_stride[1];
    const int first_pos = len - a.q_len;  // position of the request's first new token
    // a tile of the warp into a stage: 16 keys lie in one page
    const int mine = t1 > t0 + warp ? (t1 - t0 - warp + kDecWarps - 1) / kDecWarps : 0;
    auto page_of = [&](int i) {
      return i < mine && !bad && len > 0
                 ? __ldg(a.block_table + b * a.table_stride + (t0 + warp + i * kDecWarps) * kTileKeys / a.page_size)
                 : 0;
    };
    int ahead[kStages];  // the pages of the next tiles to load, read that much earlier
#pragma unroll
    for (int i = 0; i < kStages; ++i) ahead[i] = page_of(i);
    auto load = [&](int i) {
      if (i < mine && !bad && len > 0) {
        const int key = (t0 + warp + i * kDecWarps) * kTileKeys;
        const int page = ahead[0];
        const bool ok = page >= 0 && page < a.pages;
        if (!ok) page_bad = 1;
        const int64_t ko = ok ? page * a.k_stride[0] : 0, vo = ok ? page * a.v_stride[0] : 0;
        const int slot = key & (a.page_size - 1);
        const uint32_t dst = ring + (i % kStages) * Shape::kStageBytes;
#pragma unroll
        for (int c0 = 0; c0 < kTileKeys * kChunks; c0 += 32) {
          const int c = c0 + lane, r = c / kChunks, x = c % kChunks;
          const bool there = ok && key + r < len;  // (past the last key: zeros, whatever lies there)
          const uint32_t at = dst + r * (D * 2) + ((x ^ (r & 7)) << 4);
          cp_async16(at, there ? static_cast<const void*>(kbase + ko + (slot + r) * a.k_stride[2] + 8 * x) : a.k, there);
          cp_async16(at + Shape::kStageBytes / 2,
                     there ? static_cast<const void*>(vbase + vo + (slot + r) * a.v_stride[2] + 8 * x) : a.k, there);
        }
      }
      cp_commit();
#pragma unroll
      for (int s = 0; s + 1 < kStages; ++s) ahead[s] = ahead[s + 1];
      ahead[kStages - 1] = page_of(i + kStages);
    };
#pragma unroll
    for (int i = 0; i < kStages - 1; ++i) load(i);

    // Q^T as the B operand: columns are rows of Q (row = token * group + head)
    uint32_t qf[kN][D / 16][2];
#pragma unroll
    for (int nn = 0; nn < kN; ++nn) {
      const int r = 8 * nn + lane / 4;
      const bool live = r < g.rows;
      const int tok = live ? r / g.group : 0, h = hk * g.group + (live ? r - tok * g.group : 0);
      const uint32_t* q = reinterpret_cast<const uint32_t*>(static_cast<const T*>(a.q) +
                                                            (static_cast<int64_t>(b) * a.q_len + tok) * a.q_stride[0] +
                                                            h * a.q_stride[1]);
#pragma unroll
      for (int kk = 0; kk < D / 16; ++kk) {
        qf[nn][kk][0] = live ? __ldg(q + 8 * kk + lane % 4) : 0;
        qf[nn][kk][1] = live ? __ldg(q + 8 * kk + 4 + lane % 4) : 0;
      }
    }
    // this lane's columns of S^T: rows 8 nn + 2 (lane % 4) + {0, 1}
    int lim[kN][2];
    float m[kN][2], l[kN][2], o[D / 16][kN][4];
#pragma unroll
    for (int nn = 0; nn < kN; ++nn)
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const int r = 8 * nn + 2 * (lane % 4) + e;
        lim[nn][e] = r < g.rows ? first_pos + r / g.group : -1;
        m[nn][e] = -INFINITY;
        l[nn][e] = 0.f;
      }
#pragma unroll
    for (int d = 0; d < D / 16; ++d)
#pragma unroll
      for (int nn = 0; nn < kN; ++nn)
#pragma unroll
        for (int e = 0; e < 4; ++e) o[d][nn][e] = 0.f;

    for (int i = 0; i < mine; ++i) {
      load(i + kStages - 1);
      cp_wait<kStages - 1>();
      __syncwarp();
      const uint32_t kt = ring + (i % kStages) * Shape::kStageBytes, vt = kt + Shape::kStageBytes / 2;
      const int key = (t0 + warp + i * kDecWarps) * kTileKeys;
      float s[kN][4] = {};
#pragma unroll
      for (int kk = 0; kk < D / 16; ++kk) {  // A: keys by dims
        uint32_t ka[4];
        const int r = lane % 16, x = 2 * kk + lane / 16;
        ldsm4(kt + r * (D * 2) + ((x ^ (r & 7)) << 4), ka);
#pragma unroll
        for (int nn = 0; nn < kN; ++nn) mma16816<T>(s[nn], ka, qf[nn][kk][0], qf[nn][kk][1]);
      }
      // s[nn][e], s[nn][2 + e]: keys lane / 4 and lane / 4 + 8, row 8 nn + 2 (lane % 4) + e
      uint32_t ph[kN][2], pl[kN][2];
#pragma unroll
      for (int nn = 0; nn < kN; ++nn) {
        float p[4];
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          const int j = key + lane / 4;
          float x0 = j <= lim[nn][e] && j < len ? s[nn][e] * g.sl2 : -INFINITY;
          float x1 = j + 8 <= lim[nn][e] && j + 8 < len ? s[nn][2 + e] * g.sl2 : -INFINITY;
          float mx = fmaxf(x0, x1);
#pragma unroll
          for (int w = 4; w < 32; w <<= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, w));
          const float mn = fmaxf(m[nn][e], mx);
          const float ref = mn == -INFINITY ? 0.f : mn;  // nothing seen yet: weights of 0
          const float sc = ex2_approx(m[nn][e] - ref);
          m[nn][e] = mn;
          p[e] = ex2_approx(x0 - ref);
          p[2 + e] = ex2_approx(x1 - ref);
          l[nn][e] = l[nn][e] * sc + (p[e] + p[2 + e]);  // of this lane's keys: added up at the end
          if (__any_sync(0xffffffffu, sc != 1.f)) {
#pragma unroll
            for (int d = 0; d < D / 16; ++d) {
              o[d][nn][e] *= sc;
              o[d][nn][2 + e] *= sc;
            }
          }
        }
        // transposed into the B operand: keys down, rows across; high part and remainder
        const uint32_t h0 = Pair<T>::put(p[0], p[1]), h1 = Pair<T>::put(p[2], p[3]);
        const float2 f0 = Pair<T>::get(h0), f1 = Pair<T>::get(h1);
        ph[nn][0] = transpose8x8(h0);
        ph[nn][1] = transpose8x8(h1);
        pl[nn][0] = transpose8x8(Pair<T>::put(p[0] - f0.x, p[1] - f0.y));
        pl[nn][1] = transpose8x8(Pair<T>::put(p[2] - f1.x, p[3] - f1.y));
      }
#pragma unroll
      for (int d = 0; d < D / 16; ++d) {  // A: dims by keys, V transposed on the way
        uint32_t va[4];
        const int r = lane % 8 + 8 * (lane / 16), x = 2 * d + (lane / 8) % 2;
        ldsm4_t(vt + r * (D * 2) + ((x ^ (r & 7)) << 4), va);
#pragma unroll
        for (int nn = 0; nn < kN; ++nn) {
          mma16816<T>(o[d][nn], va, ph[nn][0], ph[nn][1]);
          mma16816<T>(o[d][nn], va, pl[nn][0], pl[nn][1]);
        }
      }
      __syncwarp();  // the stage may be filled again
    }
    cp_wait<0>();

    // ---- the warps' shares -------------------------------------------------------------------
#pragma unroll
    for (int nn = 0; nn < kN; ++nn)
#pragma unroll
      for (int e = 0; e < 2; ++e) {
#pragma unroll
        for (int w = 4; w < 32; w <<= 1) l[nn][e] += __shfl_xor_sync(0xffffffffu, l[nn][e], w);
        if (lane < 4) {
          red_m[warp][8 * nn + 2 * lane + e] = m[nn][e];
          red_l[warp][8 * nn + 2 * lane + e] = l[nn][e];
        }
      }
    if (threadIdx.x == 0) odd_rows = 0;
    const bool page_out = __syncthreads_or(page_bad != 0);
    float* buf = reinterpret_cast<float*>(smem);  // [warp][D][8 kN], over the ring
#pragma unroll
    for (int nn = 0; nn < kN; ++nn)
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const int r = 8 * nn + 2 * (lane % 4) + e;
        float mm = -INFINITY;
#pragma unroll
        for (int w = 0; w < kDecWarps; ++w) mm = fmaxf(mm, red_m[w][r]);
        const float f = ex2_approx(m[nn][e] - (mm == -INFINITY ? 0.f : mm));
#pragma unroll
        for (int d = 0; d < D / 16; ++d) {
          buf[(warp * D + 16 * d + lane / 4) * (8 * kN) + r] = o[d][nn][e] * f;
          buf[(warp * D + 16 * d + 8 + lane / 4) * (8 * kN) + r] = o[d][nn][2 + e] * f;
        }
      }
    __syncthreads();
    const bool whole = t0 == 0 && t1 == n;
    const bool wrong = bad || page_out;
    if (threadIdx.x == 0 && wrong) report(a.status, bad ? MKB_SERVE_BAD_LENGTH : MKB_SERVE_BAD_PAGE);
    // (first part: slot 2 cta + 1, others: slot 2 cta)
    const int slot = 2 * cta + (t0 == 0);
    for (int i = threadIdx.x; i < D * 8 * kN; i += 32 * kDecWarps) {
      const int r = i % (8 * kN);
      if (r >= g.rows) continue;
      float v = 0.f;
#pragma unroll
      for (int w = 0; w < kDecWarps; ++w) v += buf[w * D * 8 * kN + i];
      float mm = -INFINITY, ll = 0.f;
#pragma unroll
      for (int w = 0; w < kDecWarps; ++w) mm = fmaxf(mm, red_m[w][r]);
#pragma unroll
      for (int w = 0; w < kDecWarps; ++w) ll += red_l[w][r] * ex2_approx(red_m[w][r] - (mm == -INFINITY ? 0.f : mm));
      if (wrong) ll = NAN;
      if (a.q_len > 1 && v * 0.f != 0.f) atomicOr(&odd_rows, 1u << r);
      if (whole) {
        const int d = i / (8 * kN), tok = r / g.group, h = hk * g.group + r - tok * g.group;
        const bool zero = first_pos + tok < 0 && !wrong;
        T* out = static_cast<T*>(a.out) + (static_cast<int64_t>(b) * a.q_len + tok) * a.out_stride[0] + h * a.out_stride[1];
        const uint32_t w2 = Pair<T>::put(zero ? 0.f : v / ll, 0.f);
        reinterpret_cast<uint16_t*>(out)[d] = static_cast<uint16_t>(w2 & 0xffffu);
      } else {
        g.part[static_cast<size_t>(slot) * D * 16 + i] = v;
        if (i < 8 * kN) {
          g.stat[slot * 32 + r] = mm;
          g.stat[slot * 32 + 16 + r] = ll;
        }
      }
    }
    // Where rows see different keys, V that is not finite reaches those that do not see it:
    // such rows are computed again key by key.
    if (a.q_len > 1) {
      __syncthreads();
      for (int r = warp; r < g.rows && !wrong; r += kDecWarps) {
        if (!(odd_rows >> r & 1u)) continue;
        const int tok = r / g.group, h = hk * g.group + r - tok * g.group;
        constexpr int kPer = D / 32;
        float x[kPer], mm, ll;
        row_by_key<T, D, true>(a, g.sl2, b, 0, b * a.q_len + tok, h, hk, t0 * kTileKeys,
                               min(min(t1 * kTileKeys, len), first_pos + tok + 1), x, &mm, &ll);
#pragma unroll
        for (int i = 0; i < kPer; ++i) {
          const int d = lane * kPer + i;
          if (whole) {
            T* out = static_cast<T*>(a.out) + (static_cast<int64_t>(b) * a.q_len + tok) * a.out_stride[0] + h * a.out_stride[1];
            const uint32_t w2 = Pair<T>::put(first_pos + tok < 0 ? 0.f : x[i] / ll, 0.f);
            reinterpret_cast<uint16_t*>(out)[d] = static_cast<uint16_t>(w2 & 0xffffu);
          } else {
            g.part[static_cast<size_t>(slot) * D * 16 + d * 8 * kN + r] = x[i];
          }
        }
        if (!whole && lane == 0) {
          g.stat[slot * 32 + r] = mm;
          g.stat[slot * 32 + 16 + r] = ll;
        }
      }
    }
    if (!whole) {
      int c0 = cta, c1 = cta;  // the CTAs of the request's first and last stretch for this KV head
      while (cut(c0) > pos) --c0;
      while (cut(c1 + 1) < pos + n) ++c1;
      __threadfence();
      __syncthreads();
      if (threadIdx.x == 0) flag = atomicInc(g.counters + c0, c1 - c0) == static_cast<uint32_t>(c1 - c0);
      __syncthreads();
      if (flag) {
        __threadfence();
        for (int i = threadIdx.x; i < D * 8 * kN; i += 32 * kDecWarps) {
          const int r = i % (8 * kN);
          if (r >= g.rows) continue;
          float mm = -INFINITY, ll = 0.f, v = 0.f;
          for (int c = c0; c <= c1; ++c) mm = fmaxf(mm, __ldcg(g.stat + (2 * c + (c == c0)) * 32 + r));
          const float ref = mm == -INFINITY ? 0.f : mm;
          for (int c = c0; c <= c1; ++c) {
            const int s = 2 * c + (c == c0);
            const float f = ex2_approx(__ldcg(g.stat + s * 32 + r) - ref);
            ll += __ldcg(g.stat + s * 32 + 16 + r) * f;
            v += __ldcg(g.part + static_cast<size_t>(s) * D * 16 + i) * f;
          }
          const int d = i / (8 * kN), tok = r / g.group, h = hk * g.group + r - tok * g.group;
          T* out = static_cast<T*>(a.out) + (static_cast<int64_t>(b) * a.q_len + tok) * a.out_stride[0] + h * a.out_stride[1];
          const uint32_t w2 = Pair<T>::put(first_pos + tok < 0 ? 0.f : v / ll, 0.f);
          reinterpret_cast<uint16_t*>(out)[d] = static_cast<uint16_t>(w2 & 0xffffu);
        }
      }
    }
    __syncthreads();  // the ring and the reductions are free again
    // on to the next stretch
    pos += n;
    if (++hk == a.kv_heads) {
      hk = 0;
      if (++b < a.batch) n = dec_tiles(g, b, &len, &bad);
    }
  }
}

// ---- host side -----------------------------------------------------------------------

int sm_count();  // mkb_attn_tc.cu
size_t counter_bytes();

size_t decode_workspace(const mkb_attn_args& a) {
  return counter_bytes() + 2 * static_cast<size_t>(sm_count()) * (32 + static_cast<size_t>(a.head_dim) * 16) * 4;
}

template <typename T, int D, int kN>
static cudaError_t decode_launch(const mkb_attn_args& a, cudaStream_t stream) {
  DecArgs g;
  g.a = a;
  g.sl2 = a.scale * 1.4426950408889634f;
  g.group = a.heads / a.kv_heads;
  g.rows = a.q_len * g.group;
  uint8_t* ws = static_cast<uint8_t*>(a.workspace);
  if (ws == nullptr) return cudaErrorInvalidValue;
  g.counters = reinterpret_cast<uint32_t*>(ws);
  g.stat = reinterpret_cast<float*>(ws + counter_bytes());
  g.part = g.stat + 2 * static_cast<size_t>(sm_count()) * 32;
  constexpr size_t ring = DecShape<D>::kSmem, sums = static_cast<size_t>(kDecWarps) * D * 8 * kN * 4;
  constexpr size_t bytes = ring > sums ? ring : sums;
  static bool configured[64] = {false};
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e != cudaSuccess) return e;
  if (dev < 0 || dev >= 64) return cudaErrorInvalidDevice;
  if (!configured[dev]) {
    e = cudaFuncSetAttribute(attn_decode_kernel<T, D, kN>, cudaFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(bytes));
    if (e != cudaSuccess) return e;
    configured[dev] = true;
  }
  // a CTA for every SM that the tiles could keep busy
  const int64_t most = static_cast<int64_t>(a.batch) * a.kv_heads *
                       (static_cast<int64_t>(a.table_width) * a.page_size / (kTileKeys * kDecTileMin) + 1);
  const int grid = static_cast<int>(most < sm_count() ? most : sm_count());
  return launch_early(attn_decode_kernel<T, D, kN>, grid, 32 * kDecWarps, bytes, stream, g);
}

// Few enough rows a KV head for one tile of columns.
bool decode_fits(const mkb_attn_args& a) {
  return a.cu_q == nullptr && static_cast<int64_t>(a.q_len) * (a.heads / a.kv_heads) <= 16;
}

template <typename T>
static cudaError_t decode_type(const mkb_attn_args& a, cudaStream_t stream) {
  const bool one = a.q_len * (a.heads / a.kv_heads) <= 8;
  if (a.head_dim == 128) return one ? decode_launch<T, 128, 1>(a, stream) : decode_launch<T, 128, 2>(a, stream);
  return one ? decode_launch<T, 64, 1>(a, stream) : decode_launch<T, 64, 2>(a, stream);
}

cudaError_t attn_decode(const mkb_attn_args& a, cudaStream_t stream) {
  return a.dtype == MKB_BF16 ? decode_type<__nv_bfloat16>(a, stream) : decode_type<__half>(a, stream);
}

}  // namespace sv
}  // namespace mkb
