// Attention of few new tokens a request over the paged cache: the decode step.
//
//   out_i = sum_j p_ij v_j / sum_j p_ij,  p_ij = 2^(c q_i.k_j - m_i),  c = scale log2(e),  j <= pos(i)
//
// Every key and value is read once from memory and used for the handful of rows (new
// tokens x the query heads that share the KV head, 8 at most) that need it: bytes bound
// this kernel, at 4 D bytes a key and KV head. TMA brings them into shared memory (a box
// of 16 keys x 64 values, 128-byte swizzle, so that the matrix loads below meet no bank
// twice), a ring of tiles per warp, with no barrier between warps.
//
// The products run on mma.sync m16n8k16 with the keys as the 16 rows of S^T = K Q^T and
// the queries as its 8 columns, so that the tile is filled by keys however few the queries
// are: S^T's accumulators, transposed by movmatrix, are the B operand of
// O^T += V^T P^T, and V^T comes from V by ldmatrix.trans. P enters as a 16-bit high part
// and the remainder: memory leaves time for the second product, and P then costs no
// precision (in FP16, which ends at 2^-24, P is 2^15 times larger). The products take finite values of V only: a remainder of 0, or a row that
// does not see the key, would make NaN of an infinity. A tile is looked over for the others
// first (48 requests of 1-4,096 keys 57.9 us, 57.7 without; three of 9,001-60,000 78.7 and
// 78.1); they are added to the rows that see them, as they are, and cleared.
//
// Work: the tiles of 16 keys, request by request and KV head by KV head, are laid end to
// end and cut into equal ranges, one a CTA, and those into eight, one a warp. A warp runs
// through its range on its own, its copies a few tiles ahead and across the ends of
// requests; what lies in one warp's range as a whole it writes out itself. The others
// leave O, maximum and sum in shared memory, where the CTA adds them up at its end; those
// that go on in another CTA, in memory, where the last CTA to be done adds them up in
// order of their keys.
//
// 48 requests of 1-4,096 keys, 16 heads over 8 of 128: 58 us for 273 MB. While every SM streams
// it reads 6.2 TB/s of the 6.6 that a copy reaches, with 192 KB of copies in flight an SM (tiles
// of 16 keys keep a ring a warp in that): 44 us. 4 us pass before the first tile is there
// (launch, lengths, page table, one after another) and 2 after the last (sums over warps and
// CTAs); the other 8 are the slower SMs' last tiles, as the ranges are equal and the SMs are not
// (they are active for 78 % of the kernel's cycles on average).

#include <cmath>

#include "mkb_serving.cuh"
#include "mkb_tc.cuh"

namespace mkb {
namespace sv {

constexpr int kDecWarps = 8;
constexpr int kDecRows = 8;      // rows of a KV head: the columns of one mma
constexpr int kTileKeys = 16;    // keys of a tile: the rows of one mma
// A CTA for every request and KV head, unless those have more than kLongTiles tiles on
// average: then one for every kCtaTiles, as far as there are SMs. (8 requests of 700 keys: 12.4
// us, spread out further 17.6, the sums over CTAs cost more than the keys; one of 4,000: 18.7
// spread out, 40.7 not. With 64 tiles a CTA that one takes 23.7; with 4, 18.8, and one of 900
// keys 17.2 instead of 16.0.)
constexpr int kCtaTiles = 16;
constexpr int kLongTiles = 64;
// Below kWholeTiles a request's tiles of a KV head stay together: in one warp, or in one CTA
// where there are enough of those for each. (256 requests of 100 keys: 32.3 us, 41.1 when they
// are cut anywhere; 48 of 1-4,096 keys: 58.1, 58.8 cut anywhere, 59.8 with 32 tiles. One of 33
// keys: 7.4, 8.1 in one warp.)
constexpr int kWholeTiles = 8;
constexpr int kDecTryNs = 20000, kDecTries = 50000;  // bound of a wait: a second at most (0.2 s)

struct DecArgs {
  mkb_attn_args a;
  float sl2;
  int k_head, v_head;  // 0 where every KV head lies at the same place (stride 0), else 1
  int group, rows;     // query heads of a KV head; rows (q_len * group)
  int cols;            // rows up to a power of two: columns of a part
  uint32_t* counters;  // [ctas], zero between calls
  float* part;         // [2 ctas][D][cols] O^T, the maxima and sums in stat [2 ctas][2][kDecRows]
  float* stat;
  Withheld withheld;   // testing: a CTA that loads nothing
};

template <int D>
constexpr int kStageBytes = kTileKeys * D * 2 * 2;  // K and V of a tile
// Tiles of a warp's ring: 24 KB, which leaves room for a part beside each of the eight.
template <int D>
constexpr int kStages = 24 * 1024 / kStageBytes<D>;
// A warp's shared memory: the ring, then the part that it does not begin.
template <int D>
constexpr int kWarpBytes = kStages<D> * kStageBytes<D> + D * kDecRows * 4;

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
  const int len = max(g.a.kv_lens[b], 0);
  const bool bad = len > kMaxKeys || static_cast<int64_t>(len) > static_cast<int64_t>(g.a.table_width) * g.a.page_size;
  *len_out = len;
  *bad_out = bad;
  return bad ? 1 : max((len + kTileKeys - 1) / kTileKeys, 1);
}

// A place in the work: tile t of [.., t_end) of request b, KV head hk, whose tiles follow
// `pos` and one unit for its fixed cost.
struct Cursor {
  int b, hk, n, len, t, t_end;
  bool bad;
  int64_t pos;
};

template <typename T, int D>
__global__ void __launch_bounds__(32 * kDecWarps, 1)
    attn_decode_kernel(const __grid_constant__ CUtensorMap tk, const __grid_constant__ CUtensorMap tv,
                       const __grid_constant__ DecArgs g) {
  constexpr int kBytes = kStageBytes<D>, kHalf = kTileKeys * 128;  // (64 values of 16 keys)
  constexpr int kRing = kStages<D>;
  constexpr float kLift = Pair<T>::kDtype == MKB_FP16 ? 15.f : 0.f;  // P and its sum times 2^kLift
  extern __shared__ uint8_t smem_raw[];
  uint8_t* const smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  __shared__ uint64_t full[kDecWarps][kRing];
  __shared__ float part_m[kDecWarps][2][kDecRows], part_l[kDecWarps][2][kDecRows];
  __shared__ int64_t part_pos[kDecWarps][2];                   // the request's and KV head's place, -1: none
  __shared__ int part_at[kDecWarps][2][4];                     // b, hk, len, n
  __shared__ int flags[2][2], err;
  const mkb_attn_args& a = g.a;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  depend_launch();
  uint8_t* const mine = smem + warp * kWarpBytes<D>;
  const uint32_t ring = smem_addr(mine);
  // parts: 0 goes on from the warp before, 1 begins here (and lies over the ring, at the end)
  float* const part_o[2] = {reinterpret_cast<float*>(mine + kRing * kBytes), reinterpret_cast<float*>(mine)};
  if (lane < 2) part_pos[warp][lane] = -1;
  if (lane == 0) {
    tc::prefetch_tensormap(&tk);
    tc::prefetch_tensormap(&tv);
    for (int i = 0; i < kRing; ++i) mbar_init(&full[warp][i], 1);
    fence_mbar_init();
  }
  if (threadIdx.x == 0) err = 0;
  __syncthreads();
  depend_wait();

  // ---- the work, and this warp's range of it ----------------------------------------------
  int len0 = 0;
  bool bad0 = false;
  auto units = [&](int b, int* len, bool* bad) {
    return b < a.batch ? static_cast<int64_t>(dec_tiles(g, b, len, bad) + 1) * a.kv_heads : 0;
  };
  auto upto = [&](int64_t x) {  // sums over the lanes up to this one
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int64_t y = __shfl_up_sync(0xffffffffu, x, o);
      if (lane >= o) x += y;
    }
    return x;
  };
  const int64_t units0 = units(lane, &len0, &bad0), upto0 = upto(units0);  // (a lane keeps its first request's)
  int64_t total = __shfl_sync(0xffffffffu, upto0, 31);
  for (int b0 = 32; b0 < a.batch; b0 += 32) {
    int x;
    bool y;
    total += __shfl_sync(0xffffffffu, upto(units(b0 + lane, &x, &y)), 31);
  }
  const int64_t heads = static_cast<int64_t>(a.batch) * a.kv_heads;
  const int ctas = static_cast<int>(min(static_cast<int64_t>(gridDim.x),
                                        total > heads * kLongTiles ? max(total / kCtaTiles, heads) : heads));
  const int cta = blockIdx.x;
  if (cta >= ctas) return;
  const double per = static_cast<double>(total) / ctas;
  auto cut = [&](int c) { return c >= ctas ? total : static_cast<int64_t>(per * c); };
  const int64_t cta_from = cut(cta), cta_units = cut(cta + 1) - cta_from;
  const int64_t from = cta_from + cta_units * warp / kDecWarps, to = cta_from + cta_units * (warp + 1) / kDecWarps;
  Cursor ahead;  // of the next tile to load
  ahead.b = a.batch;
  ahead.pos = 0;
  for (int b0 = 0; b0 < a.batch && from < to; b0 += 32) {
    int64_t own = units0, inc = upto0;
    int ln = len0;
    bool bd = bad0;
    if (b0 > 0) {
      own = units(b0 + lane, &ln, &bd);
      inc = upto(own);
    }
    const uint32_t who = __ballot_sync(0xffffffffu, from - ahead.pos < inc);
    if (who != 0) {
      const int src = __ffs(who) - 1;
      ahead.b = b0 + src;
      ahead.n = static_cast<int>(__shfl_sync(0xffffffffu, own, src) / a.kv_heads) - 1;
      ahead.len = __shfl_sync(0xffffffffu, ln, src);
      ahead.bad = __shfl_sync(0xffffffffu, static_cast<int>(bd), src) != 0;
      ahead.pos += __shfl_sync(0xffffffffu, inc - own, src);
      ahead.hk = static_cast<int>((from - ahead.pos) / (ahead.n + 1));
      ahead.pos += static_cast<int64_t>(ahead.n + 1) * ahead.hk;
      break;
    }
    ahead.pos += __shfl_sync(0xffffffffu, inc, 31);
  }
  // a cut at x as a tile of the request and KV head that starts at pos; one between CTAs
  // (every cut, where there is more than one of those a CTA) leaves short ones whole
  auto tile_in = [&](int64_t x, int64_t pos, int n, bool whole) {
    const int64_t y = x - pos;
    if (y <= 0) return 0;
    if (y >= n + 1) return n;
    if (whole && n < kWholeTiles) return 2 * y >= n + 1 ? n : 0;
    return static_cast<int>(y) - 1;
  };
  auto tile_at = [&](int64_t x, int64_t pos, int n) { return tile_in(x, pos, n, true); };
  const bool many = heads > ctas;
  auto enter = [&](Cursor& c) {  // the part of c's tiles that is this warp's
    c.t = tile_at(from, c.pos, c.n);
    c.t_end = tile_at(to, c.pos, c.n);
    if (many || c.n >= kWholeTiles) return;
    const int lo = tile_at(cta_from, c.pos, c.n), hi = tile_at(cta_from + cta_units, c.pos, c.n);  // its CTA's part
    if (from != cta_from) c.t = min(max(tile_in(from, c.pos, c.n, false), lo), hi);
    if (to != cta_from + cta_units) c.t_end = min(max(tile_in(to, c.pos, c.n, false), lo), hi);
  };
  auto leave = [&](Cursor& c) {  // on to the next request and KV head
    c.pos += c.n + 1;
    if (++c.hk == a.kv_heads) {
      c.hk = 0;
      if (++c.b < a.batch) c.n = dec_tiles(g, c.b, &c.len, &c.bad);
    }
    enter(c);
  };
  auto open = [&](const Cursor& c) { return c.b < a.batch && c.pos < to; };
  enter(ahead);
  Cursor cur = ahead;

  bool dead = false;             // a wait has expired: nothing is waited for any more
  bool stop = g.withheld.here(); // ... nor loaded
  int fill = 0;                  // the ring's next stage to load
  int pages = 0, pages_at = -1;  // the lanes' pages of tiles pages_at .. + 31 of request pages_b
  int pages_b = -1;
  uint32_t bad_pages = 0;          // of the tiles in flight, a bit each, whether their page is outside the pool
  int load_bit = 0, bad_bit = 0;
  auto load = [&]() {
    while (open(ahead) && ahead.t >= ahead.t_end) leave(ahead);
    if (stop || !open(ahead)) return;
    bool oob = false;
    if (!ahead.bad && ahead.len > 0) {
      if (pages_b != ahead.b || ahead.t < pages_at || ahead.t >= pages_at + 32) {
        pages_b = ahead.b;
        pages_at = ahead.t;
        const int key = (ahead.t + lane) * kTileKeys;  // 16 keys lie in one page
        pages = key < ahead.len ? a.block_table[ahead.b * a.table_stride + key / a.page_size] : 0;
        if (pages < 0 || pages >= a.pages) {
          report(a.status, MKB_SERVE_BAD_PAGE);
          pages = -1;
        }
      }
      const int page = __shfl_sync(0xffffffffu, pages, ahead.t - pages_at);
      const int slot = ahead.t * kTileKeys & (a.page_size - 1);
      oob = page < 0;
      uint64_t* const bar = &full[warp][fill];
      const int at = oob ? max(a.pages, 1) : page;  // (outside the pool and its map: zeros)
      if (lane == 0) mbar_arrive_expect_tx(bar, kBytes);
      __syncwarp();
      if (lane < 2) {  // K and V
        tc::tma_load_5d(mine + fill * kBytes + lane * (kBytes / 2), lane ? &tv : &tk, 0, slot, 0, ahead.hk * (lane ? g.v_head : g.k_head), at, bar);
      }
    } else if (lane == 0) {
      mbar_arrive(&full[warp][fill]);  // nothing to bring
    }
    bad_pages = (bad_pages & ~(1u << load_bit)) | static_cast<uint32_t>(oob) << load_bit;
    load_bit = (load_bit + 1) & 31;
    if (++fill == kRing) fill = 0;
    ++ahead.t;
  };
#pragma unroll 1
  for (int i = 0; i < kRing - 1; ++i) load();

  uint32_t phase = 0;
  int stage = 0;
  for (; open(cur); leave(cur)) {
    if (cur.t >= cur.t_end) continue;
    const int t0 = cur.t, t1 = cur.t_end, b = cur.b, hk = cur.hk, len = cur.len;
    const int first_pos = len - a.q_len;  // position of the request's first new token
    // Q^T as the B operand: columns are rows of Q (row = token * group + head)
    uint32_t qf[D / 16][2];
    int lim[2];  // of this lane's columns of S^T, rows 2 (lane % 4) + {0, 1}
    float m[2], l[2], o[D / 16][4];
    const int r = lane / 4;
    const bool live = r < g.rows;
    const int tok = live ? r / g.group : 0, h = hk * g.group + (live ? r - tok * g.group : 0);
    const uint32_t* q = reinterpret_cast<const uint32_t*>(static_cast<const T*>(a.q) +
                                                          (static_cast<int64_t>(b) * a.q_len + tok) * a.q_stride[0] +
                                                          h * a.q_stride[1]);
#pragma unroll
    for (int kk = 0; kk < D / 16; ++kk) {
      qf[kk][0] = live ? q[8 * kk + lane % 4] : 0;
      qf[kk][1] = live ? q[8 * kk + 4 + lane % 4] : 0;
    }
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      const int re = 2 * (lane % 4) + e;
      lim[e] = re < g.rows ? min(first_pos + re / g.group, len - 1) : -1;
      m[e] = -INFINITY;
      l[e] = 0.f;
    }
#pragma unroll
    for (int d = 0; d < D / 16; ++d)
#pragma unroll
      for (int e = 0; e < 4; ++e) o[d][e] = 0.f;

    for (int t = t0; t < t1; ++t) {
      load();
      if (!dead)
        for (int i = 0; !__all_sync(0xffffffffu, mbar_wait(&full[warp][stage], phase, kDecTryNs)); ++i)
          if (i > kDecTries) {
            err = 1;
            dead = stop = true;
            break;
          }
      const uint32_t kt = ring + stage * kBytes, vt = kt + kBytes / 2;
      const int stage_v = stage * kBytes + kBytes / 2;
      const int key = t * kTileKeys;
      if (key + kTileKeys > len) {  // past the last key a page holds anything: P = 0 must give 0
        const int there = max(len - key, 0);
        for (int i = lane; i < (kTileKeys - there) * (D / 8); i += 32)
          *reinterpret_cast<uint4*>(mine + stage_v + (i / 8 % (D / 64)) * kHalf +
                                    (there + i / (D / 8)) * 128 + (i % 8) * 16) = make_uint4(0, 0, 0, 0);
        fence_proxy_async_shared();
        __syncwarp();
      }
      if (++stage == kRing) {
        stage = 0;
        phase ^= 1;
      }
      float s[4] = {}, s1[4] = {};  // (two sums: half the chain)
#pragma unroll
      for (int kk = 0; kk < D / 16; ++kk) {  // A: keys by dims
        uint32_t ka[4];
        const int r = lane % 16, x = 2 * (kk % 4) + lane / 16;
        ldsm4(kt + kk / 4 * kHalf + r * 128 + ((x ^ (r & 7)) << 4), ka);
        mma16816<T>(kk & 1 ? s1 : s, ka, qf[kk][0], qf[kk][1]);
      }
#pragma unroll
      for (int e = 0; e < 4; ++e) s[e] += s1[e];
      // s[e], s[2 + e]: keys lane / 4 and lane / 4 + 8, row 2 (lane % 4) + e
      if (bad_pages >> bad_bit & 1u) {  // a page outside the pool: its keys are NaN
#pragma unroll
        for (int e = 0; e < 4; ++e) s[e] = NAN;
      }
      bad_bit = (bad_bit + 1) & 31;
      float p[4];
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const int j = key + lane / 4;
        const float x0 = j <= lim[e] ? s[e] * g.sl2 : -INFINITY;
        const float x1 = j + 8 <= lim[e] ? s[2 + e] * g.sl2 : -INFINITY;
        float mx = fmaxf(x0, x1);
#pragma unroll
        for (int w = 4; w < 32; w <<= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, w));
        const float mn = fmaxf(m[e], mx);
        const float ref = mn == -INFINITY ? 0.f : mn;  // nothing seen yet: weights of 0
        const float sc = ex2_approx(m[e] - ref);
        m[e] = mn;
        p[e] = ex2_approx(x0 - (ref - kLift));
        p[2 + e] = ex2_approx(x1 - (ref - kLift));
        l[e] = l[e] * sc + (p[e] + p[2 + e]);  // of this lane's keys: added up at the end
        if (__any_sync(0xffffffffu, sc != 1.f)) {
#pragma unroll
          for (int d = 0; d < D / 16; ++d) {
            o[d][e] *= sc;
            o[d][2 + e] *= sc;
          }
        }
      }
      // V that is not finite: added as it is to the rows that see it, then cleared
      {
        uint8_t* const v = mine + stage_v;
        uint32_t n[2] = {};
#pragma unroll
        for (int i = 0; i < kTileKeys * D / 8 / 32; ++i)
          n[i & 1] = odd8<T>(*reinterpret_cast<const uint4*>(v + (32 * i + lane) * 16), n[i & 1]);
        if (__any_sync(0xffffffffu, (n[0] | n[1]) != 0)) {
#pragma unroll 1
          for (int j = 0; j < kTileKeys; ++j) {
            const bool sees[2] = {key + j <= lim[0], key + j <= lim[1]};
#pragma unroll
            for (int d = 0; d < D / 8; ++d) {  // value 8 d + lane / 4 of the key
              const uint16_t x = *reinterpret_cast<const uint16_t*>(v + d / 8 * kHalf + j * 128 + ((d % 8 ^ (j & 7)) << 4) +
                                                                    lane / 4 * 2);
              if (finite<T>(x)) continue;
              const float f = Pair<T>::get(x).x;
#pragma unroll
              for (int e = 0; e < 2; ++e)
                if (sees[e]) o[d / 2][2 * (d % 2) + e] += f;
            }
          }
          __syncwarp();
#pragma unroll 1
          for (int i = lane; i < kTileKeys * D; i += 32) {
            uint16_t* const x = reinterpret_cast<uint16_t*>(v) + i;
            if (!finite<T>(*x)) *x = 0;
          }
          fence_proxy_async_shared();
          __syncwarp();
        }
      }
      // transposed into the B operand: keys down, rows across; high part and remainder
      const uint32_t h0 = Pair<T>::put(p[0], p[1]), h1 = Pair<T>::put(p[2], p[3]);
      const float2 f0 = Pair<T>::get(h0), f1 = Pair<T>::get(h1);
      const uint32_t ph[2] = {transpose8x8(h0), transpose8x8(h1)};
      const uint32_t pl[2] = {transpose8x8(Pair<T>::put(p[0] - f0.x, p[1] - f0.y)),
                              transpose8x8(Pair<T>::put(p[2] - f1.x, p[3] - f1.y))};
#pragma unroll
      for (int d = 0; d < D / 16; ++d) {  // A: dims by keys, V transposed on the way
        uint32_t va[4];
        const int r = lane % 8 + 8 * (lane / 16), x = 2 * (d % 4) + (lane / 8) % 2;
        ldsm4_t(vt + d / 4 * kHalf + r * 128 + ((x ^ (r & 7)) << 4), va);
        mma16816<T>(o[d], va, ph[0], ph[1]);
        mma16816<T>(o[d], va, pl[0], pl[1]);
      }
      __syncwarp();  // the stage may be filled again
    }

    // ---- the end of a request's part ------------------------------------------------------
    const bool wrong = cur.bad || dead;
    if (cur.bad && lane == 0) report(a.status, MKB_SERVE_BAD_LENGTH);
    const bool whole = t0 == 0 && t1 == cur.n;
    const int which = t0 == 0;
#pragma unroll
    for (int e = 0; e < 2; ++e) {
#pragma unroll
      for (int w = 4; w < 32; w <<= 1) l[e] += __shfl_xor_sync(0xffffffffu, l[e], w);
      if (wrong) l[e] = NAN;
      const int r = 2 * (lane % 4) + e;
      if (whole) {
        if (r < g.rows) {
          const int tok = r / g.group, h = hk * g.group + r - tok * g.group;
          const bool zero = lim[e] < 0 && !wrong;  // a row that sees no key
          const float inv = 1.f / l[e];
          uint16_t* out = reinterpret_cast<uint16_t*>(static_cast<T*>(a.out) + (static_cast<int64_t>(b) * a.q_len + tok) * a.out_stride[0] +
                                                      h * a.out_stride[1]);
#pragma unroll
          for (int d = 0; d < D / 16; ++d) {
            const uint32_t w2 = Pair<T>::put(o[d][e] * inv, o[d][2 + e] * inv);
            out[16 * d + lane / 4] = zero ? 0 : static_cast<uint16_t>(w2);
            out[16 * d + 8 + lane / 4] = zero ? 0 : static_cast<uint16_t>(w2 >> 16);
          }
        }
      } else {
#pragma unroll
        for (int d = 0; d < D / 16; ++d) {
          if (r < g.cols) {
            part_o[which][(16 * d + lane / 4) * g.cols + r] = o[d][e];
            part_o[which][(16 * d + 8 + lane / 4) * g.cols + r] = o[d][2 + e];
          }
        }
        if (lane < 4) {
          part_m[warp][which][r] = m[e];
          part_l[warp][which][r] = l[e];
        }
      }
    }
    if (!whole && lane == 0) {
      part_pos[warp][which] = cur.pos;
      part_at[warp][which][0] = b;
      part_at[warp][which][1] = hk;
      part_at[warp][which][2] = len;
      part_at[warp][which][3] = cur.n;
    }
  }
  for (int i = 0; dead && i < 1000; ++i) __nanosleep(100000);  // (copies still in flight)
  __syncthreads();
  if (threadIdx.x == 0 && err) report(a.status, MKB_SERVE_TIMEOUT);

  // value i (a dim of a row) of a request: the sum v over the weights' sum
  auto write_out = [&](int b, int hk, int len, int i, float v, float ll) {
    const int r = i & (g.cols - 1), d = i / g.cols, tok = r / g.group, h = hk * g.group + r - tok * g.group;
    const float x = len - a.q_len + tok < 0 && ll == ll ? 0.f : v / ll;  // (a row that sees no key is zero)
    reinterpret_cast<uint16_t*>(static_cast<T*>(a.out) + (static_cast<int64_t>(b) * a.q_len + tok) * a.out_stride[0] +
                                h * a.out_stride[1])[d] = static_cast<uint16_t>(Pair<T>::put(x, 0.f));
  };

  // ---- requests that several warps have parts of --------------------------------------------
  // Part p = 2 warp + (0 or 1), in order of their keys; those of one request and KV head are
  // neighbours. First every part's weight beside the largest maximum of its row, a lane a part:
  constexpr int kParts = 2 * kDecWarps;
  // (these lie over the first warp's ring, behind its part)
  float(*const fac)[kDecRows] = reinterpret_cast<float(*)[kDecRows]>(smem + D * kDecRows * 4);
  float(*const sum_m)[kDecRows] = fac + kParts;
  float(*const sum_l)[kDecRows] = sum_m + kParts;
  static_assert((D + 3 * kParts) * kDecRows * 4 <= kRing * kBytes, "room of the first warp's ring");
  const int64_t my_pos = lane < kParts ? part_pos[lane / 2][lane % 2] : -1;
  // the parts that go with the lane's
  const uint32_t same = __match_any_sync(0xffffffffu, static_cast<unsigned long long>(my_pos)) & (my_pos >= 0 ? ~0u : 0u);
  const uint32_t firsts = __ballot_sync(0xffffffffu, my_pos >= 0 && (same & ((1u << lane) - 1)) == 0);
  if (firsts == 0) return;  // (the same for every warp)
  for (int r = warp; r < g.rows; r += kDecWarps) {
    const float m = my_pos >= 0 ? part_m[lane / 2][lane % 2][r] : -INFINITY;
    float mm = -INFINITY, ll = 0.f;
#pragma unroll
    for (int j = 0; j < kParts; ++j) {
      const float x = __shfl_sync(0xffffffffu, m, j);
      if (same >> j & 1u) mm = fmaxf(mm, x);
    }
    const float f = ex2_approx(m - (mm == -INFINITY ? 0.f : mm));
    const float l = my_pos >= 0 ? part_l[lane / 2][lane % 2][r] * f : 0.f;
#pragma unroll
    for (int j = 0; j < kParts; ++j) {
      const float x = __shfl_sync(0xffffffffu, l, j);
      if (same >> j & 1u) ll += x;
    }
    if (lane < kParts) {
      fac[lane][r] = f;
      sum_m[lane][r] = mm;
      sum_l[lane][r] = ll;
    }
  }
  __syncthreads();
  // then the sums: written out where the CTA has all of a request's keys, else left in memory
  // (that can be the CTA's first and its last: `cross`)
  int cross[2], crosses = 0;
  for (uint32_t todo = firsts; todo != 0; todo &= todo - 1) {
    const int p0 = __ffs(todo) - 1;
    const uint32_t parts = __shfl_sync(0xffffffffu, same, p0);
    const int64_t pos = part_pos[p0 / 2][p0 % 2];
    const int* at = part_at[p0 / 2][p0 % 2];
    const int b = at[0], hk = at[1], len = at[2], n = at[3];
    const bool begins = tile_at(cta_from, pos, n) == 0, here = begins && tile_at(cta_from + cta_units, pos, n) == n;
    const int slot = 2 * cta + begins;
    for (int i = threadIdx.x; i < D * g.cols; i += 32 * kDecWarps) {
      const int r = i & (g.cols - 1);
      if (r >= g.rows) continue;
      float v = 0.f;
      for (uint32_t u = parts; u != 0; u &= u - 1) {
        const int p = __ffs(u) - 1;
        const uint8_t* base = smem + (p / 2) * kWarpBytes<D> + (p % 2 == 0 ? kRing * kBytes : 0);
        v += reinterpret_cast<const float*>(base)[i] * fac[p][r];
      }
      if (here) write_out(b, hk, len, i, v, sum_l[p0][r]);
      else g.part[static_cast<size_t>(slot) * D * kDecRows + i] = v;
    }
    if (!here) {
      if (threadIdx.x < g.rows) {
        g.stat[slot * 2 * kDecRows + threadIdx.x] = sum_m[p0][threadIdx.x];
        g.stat[(slot * 2 + 1) * kDecRows + threadIdx.x] = sum_l[p0][threadIdx.x];
      }
      cross[crosses++ & 1] = p0;
    }
  }
  if (crosses == 0) return;
  __threadfence();
  __syncthreads();
  for (int x = 0; x < crosses; ++x) {
    const int p0 = cross[x], n = part_at[p0 / 2][p0 % 2][3];
    const int64_t pos = part_pos[p0 / 2][p0 % 2];
    if (threadIdx.x == 32 * x) {
      int c0 = cta, c1 = cta;  // the CTAs of its first and last part
      while (tile_at(cut(c0), pos, n) > 0) --c0;
      while (tile_at(cut(c1 + 1), pos, n) < n) ++c1;
      const bool last = atomicInc(g.counters + c0, c1 - c0) == static_cast<uint32_t>(c1 - c0);
      flags[x][0] = last ? c0 : -1;
      flags[x][1] = c1;
    }
  }
  __syncthreads();
  for (int x = 0; x < crosses; ++x) {
    const int c0 = flags[x][0], c1 = flags[x][1], p0 = cross[x];
    if (c0 < 0) continue;
    __threadfence();
    const int* at = part_at[p0 / 2][p0 % 2];
    const int b = at[0], hk = at[1], len = at[2];
    for (int r = warp; r < g.rows; r += kDecWarps) {  // a warp a row, a lane a CTA
      float mm = -INFINITY, ll = 0.f;
      for (int c = c0 + lane; c <= c1; c += 32) mm = fmaxf(mm, __ldcg(g.stat + (2 * c + (c == c0)) * 2 * kDecRows + r));
#pragma unroll
      for (int w = 16; w > 0; w >>= 1) mm = fmaxf(mm, __shfl_xor_sync(0xffffffffu, mm, w));
      const float ref = mm == -INFINITY ? 0.f : mm;
      for (int c = c0 + lane; c <= c1; c += 32) {
        const float* st = g.stat + (2 * c + (c == c0)) * 2 * kDecRows + r;
        ll += __ldcg(st + kDecRows) * ex2_approx(__ldcg(st) - ref);
      }
#pragma unroll
      for (int w = 16; w > 0; w >>= 1) ll += __shfl_xor_sync(0xffffffffu, ll, w);
      if (lane == 0) {
        sum_m[p0][r] = ref;
        sum_l[p0][r] = ll;
      }
    }
    __syncthreads();
    for (int i = threadIdx.x; i < D * g.cols; i += 32 * kDecWarps) {
      const int r = i & (g.cols - 1);
      if (r >= g.rows) continue;
      const float ref = sum_m[p0][r];
      float v = 0.f;
#pragma unroll 8
      for (int c = c0; c <= c1; ++c) {
        const int s = 2 * c + (c == c0);
        v += __ldcg(g.part + static_cast<size_t>(s) * D * kDecRows + i) * ex2_approx(__ldcg(g.stat + s * 2 * kDecRows + r) - ref);
      }
      write_out(b, hk, len, i, v, sum_l[p0][r]);
    }
    __syncthreads();
  }
}

// ---- host side -----------------------------------------------------------------------

int sm_count();  // these three: mkb_attn_tc.cu
cudaError_t map_rows(CUtensorMap* m, int dtype, const void* base, int D, int rank, const uint64_t* dims,
                     const int64_t* strides, const uint32_t* box);
size_t counter_bytes();

size_t decode_workspace(const mkb_attn_args& a) {
  return counter_bytes() + 2 * static_cast<size_t>(sm_count()) * (2 + static_cast<size_t>(a.head_dim)) * kDecRows * 4;
}

template <typename T, int D>
static cudaError_t decode_launch(const mkb_attn_args& a, cudaStream_t stream) {
  DecArgs g;
  g.a = a;
  g.sl2 = a.scale * 1.4426950408889634f;
  g.k_head = a.k_stride[1] != 0;
  g.v_head = a.v_stride[1] != 0;
  g.group = a.heads / a.kv_heads;
  g.rows = a.q_len * g.group;
  g.withheld = withheld();
  uint8_t* ws = static_cast<uint8_t*>(a.workspace);
  if (ws == nullptr) return cudaErrorInvalidValue;
  g.counters = reinterpret_cast<uint32_t*>(ws);
  g.stat = reinterpret_cast<float*>(ws + counter_bytes());
  g.part = g.stat + 2 * static_cast<size_t>(sm_count()) * 2 * kDecRows;
  for (g.cols = 2; g.cols < g.rows;) g.cols *= 2;
  constexpr int bytes = kDecWarps * kWarpBytes<D> + 1024;
  static_assert(kWarpBytes<D> % 1024 == 0, "swizzle atoms");
  static bool configured[64] = {false};
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e != cudaSuccess) return e;
  CUtensorMap mk, mv;
  const void* kb = a.pages > 0 ? a.k : a.q;  // an empty pool is never read: any address will do
  const void* vb = a.pages > 0 ? a.v : a.q;
  // (a row's blocks of 64 values are a dimension of their own: one copy brings them all, block
  // by block)
  const uint64_t dims[4] = {static_cast<uint64_t>(a.page_size), D / 64, static_cast<uint64_t>(a.kv_heads),
                            static_cast<uint64_t>(a.pages)};
  const int64_t ks[4] = {a.k_stride[2], 64, a.k_stride[1], a.k_stride[0]};
  const int64_t vs[4] = {a.v_stride[2], 64, a.v_stride[1], a.v_stride[0]};
  const uint32_t box[4] = {kTileKeys, D / 64, 1, 1};
  if ((e = map_rows(&mk, a.dtype, kb, 64, 4, dims, ks, box)) != cudaSuccess) return e;
  if ((e = map_rows(&mv, a.dtype, vb, 64, 4, dims, vs, box)) != cudaSuccess) return e;
  if (dev < 0 || dev >= 64) return cudaErrorInvalidDevice;
  if (!configured[dev]) {
    e = cudaFuncSetAttribute(attn_decode_kernel<T, D>, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes);
    if (e != cudaSuccess) return e;
    configured[dev] = true;
  }
  // a CTA for every SM that the tiles could keep busy
  const int64_t most = static_cast<int64_t>(a.batch) * a.kv_heads *
                       (static_cast<int64_t>(a.table_width) * a.page_size / (kTileKeys * kCtaTiles) + 1);
  const int grid = static_cast<int>(most < sm_count() ? most : sm_count());
  return launch_early(attn_decode_kernel<T, D>, grid, 32 * kDecWarps, bytes, stream, mk, mv, g);
}

// Rows (new tokens x query heads of a KV head) known from the shapes alone, and few: up to 4;
// up to 8 where there are few requests and KV heads, whose keys have to be shared out over the
// SMs, and the table has room for long ones (how long they are only the device knows). This
// kernel against the tensor-core tiles, heads 16 over 8 of 128 unless named, us:
//   2 rows: 48 requests of 1-4,096 keys 58 and 66, 9,001-60,000 keys 78 and 95, 33 keys 7.3 and 9.2
//   8 rows: 48 requests 71 and 66; three of 500-1,000 keys 26.9 and 17.6, of 4,000-8,000 37.7 and
//           36.0, of 16,000-32,000 69.7 and 72.6; one of 700 keys 15.0 and 15.2, of 8,000 34.4 and
//           33.8, of 16,000 40.8 and 44.3
//   8 rows, heads 16 over 2: four of 300-1,000 keys 23.5 and 16.9, 12 of 300-1,000 27.2 and 17.2, of
//           666-8,000 35.5 and 34.1, of 1,333-16,000 43.9 and 45.2, of 2,666-32,000 58.7 and 64.5
//   16 rows, by two columns of products: 48 requests 100 and 71
constexpr int kLongTable = 16384;
bool decode_fits(const mkb_attn_args& a) {
  if (a.cu_q != nullptr) return false;
  const int64_t rows = static_cast<int64_t>(a.q_len) * (a.heads / a.kv_heads);
  const bool few = static_cast<int64_t>(a.batch) * a.kv_heads * 6 <= sm_count();
  const bool longer = static_cast<int64_t>(a.table_width) * a.page_size >= kLongTable;
  return rows <= (few && longer ? kDecRows : kDecRows / 2);
}

template <typename T>
static cudaError_t decode_type(const mkb_attn_args& a, cudaStream_t stream) {
  return a.head_dim == 128 ? decode_launch<T, 128>(a, stream) : decode_launch<T, 64>(a, stream);
}

cudaError_t attn_decode(const mkb_attn_args& a, cudaStream_t stream) {
  return a.dtype == MKB_BF16 ? decode_type<__nv_bfloat16>(a, stream) : decode_type<__half>(a, stream);
}

}  // namespace sv
}  // namespace mkb
