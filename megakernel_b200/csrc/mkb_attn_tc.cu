// Attention of a packed batch on the tensor cores: prompts, and chunks of new tokens
// over the paged cache.
//
//   out_i = sum_j p_ij v_j / sum_j p_ij,  p_ij = 2^(c q_i.k_j - m_i),  c = scale log2(e),  j <= pos(i)
//
// A KV head's queries are rows: row r of a tile is token r / G, query head r % G of the
// G that share the KV head, so that one pass over the keys serves all of them; a tile
// holds the 128 / G tokens that fill (nearly) 128 rows. A CTA takes two tiles (A and B)
// of one request and KV head and walks its keys 128 at a time; where there are rows for
// one only, A takes them with the even and B with the odd tiles of keys, and A adds the
// two up in the end:
//
//   warp 11     which piece of work comes next
//   warp 9      its Q, K and V tiles by TMA (128-byte swizzle; K and V through a ring, pages
//               are boxes of page_size rows)
//   warps 8, 10 tcgen05.mma of tile A, B: S = Q K^T (Q and K in shared memory), O += P V with P from
//               tensor memory and V as it lies, keys by dims (an MN-major operand: no
//               transposed copy of V is made)
//   warps 0-3   softmax of tile A, a thread per row: S out of tensor memory, running
//   warps 4-7   maximum and sum in FP32 registers, P into tensor memory; tile B
//
// While one tile's softmax runs, the tensor core works on the other's products. Tensor core
// (8 D cycles for the two products of a 128 x 128 tile: 1,024 at D = 128) and exponentials
// (1,024: 16 a cycle and SM) bound a pair of tiles at 2,048 cycles each; the chain of one tile
// (load 215, maximum 450, weights 1,450, the rest of PV and the next S 1,100) makes it 3,250.
// That is for two tiles of rows; where there is one and the tiles take turns with the keys, the
// products have no order and a pair takes about 5,000 (four chunks of 512: 24 tiles of keys an
// SM, tensor core 31 % busy). 15,999 tokens, 16 heads over 8 of 128: 820-850 us, 1,280 TFLOP/s
// (of 1,640 that a library GEMM reaches), both units 63 % busy; 955 us once the power limit
// holds the clock (1,100 of 1,370 TFLOP/s).
// What did not shorten the chain: P in columns of its own, so that the next S need not wait
// for it (80 keys a tile at D = 128: 2,330 cycles a pair; both tiles' softmax then run at
// once); the next S in halves, the upper one while the weights are worked out (3-10 % slower:
// 64 columns cost the tensor core three quarters of 128); S read twice, 32 columns at a time
// (5-25 % slower); part of the exponentials as polynomials (no gain).
//
// The running maximum that P is relative to moves only when a row's grows by more than 8
// (a factor 256): O, in tensor memory, is then rescaled by the softmax warps; between
// moves P stays below 2^8, which FP32 sums and BF16 hold without loss. P is rounded to the
// operands' 16-bit type, as the output is: the same relative error. FP16 has no relative
// error below 2^-14, and nothing below 2^-25: there P is 2^7 times larger (2^15 at most), so
// that a weight is rounded by 2^-32 of the row's largest at most.
//
// Work: a piece is (request, KV head, one or two tiles of rows, a range of key tiles).
// Every CTA works the list out for itself from the lengths, the longest pieces first, and
// takes the next one when the loads of the last are nearly through (a counter in memory).
// Rows whose keys are more than a fair share are split over several pieces; each leaves its
// O, maximum and sum in memory, and the last one to be done adds them up in order of their
// keys, so results do not depend on timing. Nothing is asked of the host.
//
// Masked places: scores are replaced, not added to. V rows past the request's last key
// are cleared in shared memory. V that is not finite and stands where some row does not
// look would reach that row as 0 * inf = NaN. That can happen only in the key tiles that the
// piece's first row does not see in full (its last three at most): the warp that issues the
// product looks those over while it waits for P, and where it finds such a value clears it;
// the softmax warps then add it to the rows that see it, as it is. What every row of the
// piece sees goes through the product: a weight that rounds to 0 makes NaN of an infinity.
// (Looking over takes instructions from the softmax warps, which the comparisons below do not
// have in them yet: 12 prompts of 1-1,411 tokens 36.3 us, 34.7 without; 2,049, 1,000 and 4,097 tokens of 64-wide FP16 118.8, 117.1; two of 4,096 125.3,
// 123.0. 15,999 tokens 802 us; with NaN in all of the first key 834, all of V infinite 1,381.)

#include <cmath>
#include <cuda.h>

#include "mkb_serving.cuh"
#include "mkb_tc.cuh"

namespace mkb {
namespace sv {

constexpr int kTcThreads = 384;
// Registers of a thread: the launch's 168 are shared out again, to the softmax warps
// that hold 128 scores a thread (2 x 128 x 208 + 128 x 88 = 384 x 168).
constexpr int kSoftmaxRegs = 208, kOtherRegs = 88;
constexpr int kRows = 256, kKeys = 128;   // rows of a piece (two tiles), keys of a tile
constexpr int kFirstKeys = 96;            // of a tile's weights, what the second product starts on (2 x 4,096
                                          // tokens: 123 us; 126 with 64)
constexpr int kHalf = 128 * 128;          // 16 KB: 128 rows x 64 values, 128-byte swizzle
// Key tiles (turns, of one tile's rows) below which rows are not split: 1,200 tokens take 20.3
// us, with 3 35.8, with 12 24.8.
constexpr int kMinSplit = 6;
// Key tiles still to load when a CTA asks for its next piece: 12 prompts of 1-1,411 tokens take
// 35.4 us, with 8 37.3 (pieces are taken too long before their turn).
constexpr int kAskTiles = 3;
// Requests up to which pieces are taken longest first: 28 decoding and two chunks 62.3 us, as
// they come 68.2; 200 prompts of 30-930 tokens 516 us, as they come 463.
constexpr int kSortBatch = 128;
constexpr int kTryNs = 20000, kTries = 50000;  // bound of every wait: a second at most (tries end sooner: 0.2 s)

// A page or length is wrong; values of V that are not finite were cleared in the piece's tiles.
constexpr int kBad = 1, kOdd = 2;

struct Piece {
  int b;            // request, -1: no more work
  int hk;
  int first;        // the request's first packed token
  int tok0, toks;   // the piece's tokens
  int ctx, len;     // keys before the new tokens, all keys
  int k0, total;    // first key tile, how many
  int n[2];         // those of tiles A and B
  int halves;       // A and B have the same rows, and every other key tile
  int splits, split, slot;  // ranges of the rows' keys, which this is, where the first leaves its results
  int flags;        // of kBad, kOdd
};

template <int D>
struct TcShape {
  static constexpr int kSlots = D == 128 ? 4 : 8;       // K and V tiles in flight
  static constexpr int kTileBytes = kKeys * D * 2;
  // tensor memory columns: S of tile t at 128 t (P over its first half), O from kO on
  static constexpr uint32_t kO = 512 - 2 * D;
};

template <int D>
struct TcSmem {
  using Shape = TcShape<D>;
  uint8_t q[2][Shape::kTileBytes];
  uint8_t kv[Shape::kSlots][Shape::kTileBytes];
  uint8_t stage[8][32 * 128];                           // a warp's 32 rows x 64 values on their way out
  uint64_t kv_full[Shape::kSlots], kv_empty[Shape::kSlots];
  uint64_t q_full[2], q_empty[2], s_full[2], p_part[2], p_full[2], o_full[2];
  uint64_t info_full[2], info_empty[2], ask;
  uint64_t tile_bar[2];   // the four softmax warps of a tile
  uint64_t pair_full, pair_empty;
  float2 pair[128];       // maximum and sum of B's rows, where they are A's too
  Piece piece[2];
  Piece lost;             // taken off the list after a stop
  uint32_t tmem_base;
  int err;
  int handed, open, pending;  // pieces given out; after a stop: the list goes on, with this one if not -1
  int left[8];            // the first piece that a softmax warp has not finished
  int counted[2];         // pieces up to the last split one that a tile has counted
  int last[2];
  int turn;               // turns of A's products issued so far
};

struct TcArgs {
  mkb_attn_args a;
  float sl2;            // scale * log2(e)
  int group;            // query heads of a KV head
  int tile_tokens;      // tokens of a tile: 128 / group
  int group_mul;        // r / group = r * group_mul >> 16 for r < 128
  int warp_tokens;      // tokens of a warp's 32 rows, 0 where they are not whole
  int box;              // keys of a TMA box
  int folded;           // pages and KV heads are one dimension of the maps: see tc_launch
  int kx[3], vx[3];     // ... and lie there at page * [0] + head * [1], outside at [2]
  int k_head, v_head;   // 0 where every KV head lies at the same place (stride 0), else 1
  unsigned tile_mul;    // x / tile_tokens is x * tile_mul >> 32, or one less (0: tile_tokens is 1)
  uint32_t* work;       // the next piece, CTAs that have finished; both zero between calls
  uint32_t* counters;   // [slots][2], of the splits that are done, by tile; zero between calls
  float4* part;         // [slots][D / 4][256]
  float2* stat;         // [slots][256]: maximum, sum
  Withheld withheld;    // testing: a CTA that stops loading
};

// A warp's wait for a phase of a barrier. Bounded: each try suspends for 20 us at most.
// Once one has expired (here or in another warp) the warp is `dead`: it waits for nothing and
// issues nothing any more, makes the rows it is at NaN and leaves. What
// the CTA was given and has not finished, and the rest of the list, are then made NaN too and
// counted where others count on them (clean_up): every row of the call is right or NaN, and the
// counters are zero after it.
// (Short on purpose: the loops of the softmax warps fill the instruction caches, and what
// the other warps run between two MMAs is fetched anew every time.)
__device__ __forceinline__ void wait_for(uint64_t* bar, uint32_t ph, int* err, bool& dead) {
  if (__all_sync(0xffffffffu, mbar_test(bar, ph)) || dead) return;
#pragma unroll 1
  for (int i = 0; !__all_sync(0xffffffffu, mbar_wait(bar, ph, kTryNs)); ++i) {
    const bool other = *reinterpret_cast<volatile int*>(err) != 0;
    if (__any_sync(0xffffffffu, i > kTries || other)) {
      *reinterpret_cast<volatile int*>(err) = 1;
      dead = true;
      return;
    }
  }
}

__device__ __forceinline__ void tma_store_3d(const void* src, const CUtensorMap* map, int x, int y, int z) {
  asm volatile("cp.async.bulk.tensor.3d.global.shared::cta.tile.bulk_group [%0, {%2, %3, %4}], [%1];\n\t"
               "cp.async.bulk.commit_group;"
               ::"l"(reinterpret_cast<uint64_t>(map)), "r"(smem_addr(src)), "r"(x), "r"(y), "r"(z)
               : "memory");
}
// this thread's stores: their shared memory has been read / they are done
__device__ __forceinline__ void tma_store_read() { asm volatile("cp.async.bulk.wait_group.read 0;" ::: "memory"); }
__device__ __forceinline__ void tma_store_done() { asm volatile("cp.async.bulk.wait_group 0;" ::: "memory"); }

// Descriptor of an operand whose contiguous dimension is N, written by TMA with the
// 128-byte swizzle: 64 values of N a row, eight rows (of K) to an atom of 1024 bytes;
// `n_bytes` between 64-value blocks of N (leading offset), `k_bytes` between atoms of K
// (stride offset).
__device__ __forceinline__ uint64_t desc_mn_sw128(uint32_t addr, uint32_t n_bytes, uint32_t k_bytes) {
  uint64_t d = 0;
  d |= static_cast<uint64_t>((addr >> 4) & 0x3fffu);
  d |= static_cast<uint64_t>((n_bytes >> 4) & 0x3fffu) << 16;
  d |= static_cast<uint64_t>(k_bytes >> 4) << 32;
  d |= static_cast<uint64_t>(1u) << 46;
  d |= static_cast<uint64_t>(2u) << 61;
  return d;
}
// FP32 accumulator, A and B of type T (FP16 0, BF16 1), B N-major where `mn`
template <typename T>
__host__ __device__ constexpr uint32_t idesc16(int m, int n, bool mn) {
  constexpr uint32_t f = Pair<T>::kDtype == MKB_BF16 ? 1u : 0u;
  return (1u << 4) | (f << 7) | (f << 10) | (mn ? 1u << 16 : 0u) | (static_cast<uint32_t>(n >> 3) << 17) |
         (static_cast<uint32_t>(m >> 4) << 24);
}
// One lane of a converged warp.
__device__ __forceinline__ uint32_t elect_one() {
  uint32_t r;
  asm volatile(
      "{\n\t.reg .pred p;\n\t.reg .b32 t;\n\t"
      "elect.sync t|p, 0xffffffff;\n\t"
      "selp.u32 %0, 1, 0, p;\n\t}"
      : "=r"(r));
  return r;
}
// A value that every lane holds, in a uniform register.
__device__ __forceinline__ int uniform(int v) { return __reduce_max_sync(0xffffffffu, v); }
// The tensor-core instructions are issued by one lane (`leader`), but the whole warp runs
// through them, predicated: their operands then stay warp-uniform. Inside a branch of one
// lane every one of them costs a round of moves into uniform registers (80 cycles an
// MMA, measured, against 64 of tensor-core work for 128 x 128 x 16).
// D[tmem] (+)= A[smem desc] B[smem desc]
__device__ __forceinline__ void mma_ss(uint32_t leader, uint32_t d, uint64_t a, uint64_t b, uint32_t idesc,
                                       uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p, q;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "setp.ne.b32 q, %5, 0;\n\t"
      "@q tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}"
      ::"r"(d), "l"(a), "l"(b), "r"(idesc), "r"(accumulate), "r"(leader)
      : "memory");
}
// D[tmem] (+)= A[tmem] B[smem desc]
__device__ __forceinline__ void mma_ts(uint32_t leader, uint32_t d, uint32_t a, uint64_t b, uint32_t idesc,
                                       uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p, q;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "setp.ne.b32 q, %5, 0;\n\t"
      "@q tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}"
      ::"r"(d), "r"(a), "l"(b), "r"(idesc), "r"(accumulate), "r"(leader)
      : "memory");
}
// Arrive on `bar` once all that the leader issued before has completed.
__device__ __forceinline__ void commit(uint32_t leader, uint64_t* bar) {
  asm volatile(
      "{\n\t.reg .pred q;\n\t"
      "setp.ne.b32 q, %1, 0;\n\t"
      "@q tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];\n\t}"
      ::"r"(smem_addr(bar)), "r"(leader)
      : "memory");
}
__device__ __forceinline__ void tmem_st16(uint32_t taddr, const uint32_t v[16]) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, "
      "%15, %16};"
      ::"r"(taddr), "r"(v[0]), "r"(v[1]), "r"(v[2]), "r"(v[3]), "r"(v[4]), "r"(v[5]), "r"(v[6]), "r"(v[7]), "r"(v[8]),
        "r"(v[9]), "r"(v[10]), "r"(v[11]), "r"(v[12]), "r"(v[13]), "r"(v[14]), "r"(v[15])
      : "memory");
}
// 16 columns of this thread's lane; valid after tmem_wait_ld, which takes the first of
// several such loads (the others go through pin16, so that no use moves before it)
__device__ __forceinline__ void tmem_ld16(uint32_t taddr, uint32_t* r) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15}, "
      "[%16];"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]),
        "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
      : "r"(taddr));
}
#define MKB_PIN16(text)                                                                                              \
  asm volatile(text                                                                                                  \
               : "+r"(r[0]), "+r"(r[1]), "+r"(r[2]), "+r"(r[3]), "+r"(r[4]), "+r"(r[5]), "+r"(r[6]), "+r"(r[7]),     \
                 "+r"(r[8]), "+r"(r[9]), "+r"(r[10]), "+r"(r[11]), "+r"(r[12]), "+r"(r[13]), "+r"(r[14]), "+r"(r[15]) \
               :: "memory")
__device__ __forceinline__ void tmem_wait_ld(uint32_t* r) { MKB_PIN16("tcgen05.wait::ld.sync.aligned;"); }
__device__ __forceinline__ void pin16(uint32_t* r) { MKB_PIN16(""); }
#undef MKB_PIN16
__device__ __forceinline__ void tmem_wait_st() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }

// two FP32 operations in one instruction
__device__ __forceinline__ uint64_t pack2(float a, float b) {
  uint64_t r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(a), "f"(b));
  return r;
}
__device__ __forceinline__ float2 unpack2(uint64_t v) {
  float2 f;
  asm("mov.b64 {%0, %1}, %2;" : "=f"(f.x), "=f"(f.y) : "l"(v));
  return f;
}
__device__ __forceinline__ uint64_t fma2(uint64_t a, uint64_t b, uint64_t c) {
  uint64_t r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
  return r;
}
__device__ __forceinline__ uint64_t add2(uint64_t a, uint64_t b) {
  uint64_t r;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}

// the largest of three; NaN where one is
__device__ __forceinline__ float max3(float a, float b, float c) {
  float r;
  asm("max.NaN.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
  return r;
}
// ---- the list of pieces, worked out by one warp -------------------------------------

// One request as the list sees it.
struct Load {
  int first, q, len, ctx, tiles, bad;
  int blocks, turns, splits;  // its blocks of rows, the turns of the last of them, the ranges of each one's keys
};
template <bool kPaged>
__device__ __forceinline__ Load load_of(const TcArgs& g, int b) {
  const Request rq = request_rows(g.a.cu_q, b, g.a.q_len, g.a.tokens);
  Load l;
  l.first = rq.first;
  l.q = rq.n;
  l.len = kPaged ? max(g.a.kv_lens[b], 0) : rq.n;
  l.bad = kPaged && (l.len > kMaxKeys || static_cast<int64_t>(l.len) > static_cast<int64_t>(g.a.table_width) * g.a.page_size);
  l.ctx = l.len - l.q;
  l.tiles = l.bad || l.q == 0 ? 0 : static_cast<int>((static_cast<unsigned>(l.len) + kKeys - 1) / kKeys);
  return l;
}
// key tiles that the first `toks` tokens of the request see
__device__ __forceinline__ int tiles_of(const Load& l, int toks) {
  const int keys = l.ctx + min(toks, l.q);
  return l.bad || keys <= 0 ? 0 : static_cast<int>((static_cast<unsigned>(keys) + kKeys - 1) / kKeys);
}
// Blocks of `span` tokens, `tiles` tiles of rows each (1 or 2).
struct Blocks {
  int tiles, span;
  unsigned tile_mul;
  __device__ __forceinline__ int over(unsigned x) const {  // x / span
    const unsigned y = tiles == 2 ? x >> 1 : x;  // (span = tiles * tile_tokens)
    if (tile_mul == 0) return y;
    int i = __umulhi(y, tile_mul);
    return i * (span >> (tiles - 1)) > y ? i - 1 : i;
  }
  __device__ __forceinline__ int of(const Load& l) const { return l.q > 0 ? over(l.q - 1) + 1 : 0; }
  // rows for one tile take two key tiles at a time
  __device__ __forceinline__ bool halves(const Load& l) const { return tiles == 1 || 2 * l.q <= span; }
  // turns that a block with n key tiles takes
  __device__ __forceinline__ int turns(const Load& l, int n) const { return halves(l) ? (n + 1) / 2 : n; }
  // how many of the request's blocks take more than x turns (they come last)
  __device__ __forceinline__ int above(const Load& l, int x) const {
    if (x < 0) return l.blocks;
    if (l.turns <= x) return 0;
    const int n = halves(l) ? 2 * x : x;  // more than n key tiles
    const int y = n * kKeys - l.ctx;      // the first token that sees more (n < tiles: no overflow)
    return y <= 0 ? l.blocks : l.blocks - over(y);
  }
};

// The rows of a piece that is not to be worked out any more: NaN. Where they are one of several
// ranges of keys, this one is NaN for whoever adds them up, and counted: `count` has a bit for
// each tile that has not been. Warp-wide.
template <typename T, int D>
__device__ __noinline__ void void_piece(const TcArgs& g, const Piece& p, int count) {
  const mkb_attn_args& a = g.a;
  const int lane = threadIdx.x & 31;
  constexpr int kLanes = D / 8;  // of a row
  for (int i = lane / kLanes; i < p.toks * g.group; i += 32 / kLanes) {
    const int tok = i / g.group;
    T* const out = static_cast<T*>(a.out) + (p.first + p.tok0 + tok) * a.out_stride[0] +
                   (p.hk * g.group + i - tok * g.group) * a.out_stride[1];
    reinterpret_cast<uint4*>(out)[lane % kLanes] = make_uint4(0x7fff7fffu, 0x7fff7fffu, 0x7fff7fffu, 0x7fff7fffu);
  }
  if (p.splits == 1) return;
  for (int t = 0; t < (p.halves ? 1 : 2); ++t) {
    if (!(count >> t & 1)) continue;
    float2* const stat = g.stat + static_cast<size_t>(p.slot + p.split) * kRows + 128 * t;
    for (int i = lane; i < 128; i += 32) stat[i] = make_float2(0.f, NAN);
    __threadfence();
    __syncwarp();
    if (lane == 0) atomicInc(g.counters + 2 * p.slot + t, p.splits - 1);
  }
}

// Which piece comes next, worked out by one warp: handed to the CTA's other warps or, after a
// stop (kDrain), taken off the list and made NaN. `mine` is the lane's first request.
template <typename T, int D, bool kPaged, bool kDrain>
__device__ __forceinline__ void hand_out(const TcArgs& g, TcSmem<D>& sm, Load mine, bool& dead) {
  // (a warp of its own: the place in the list takes 5,000 cycles to work out, and the loads
  // of the next piece came that much late: 12 prompts of 1-1,411 tokens 37.7 us, now 35.3)
  const mkb_attn_args& a = g.a;
  const int lane = threadIdx.x & 31, kv_heads = a.kv_heads, grid = gridDim.x;
  // One pass over the requests: their blocks as pairs of tiles and as single ones, what
  // those come to in turns (linear in the block), and the longest.
  const Blocks pairs = {2, 2 * g.tile_tokens, g.tile_mul}, singles = {1, g.tile_tokens, g.tile_mul};
  int n2 = 0, n1 = 0, longest = 0, top = 0;
  float total2 = 0.f, total1 = 0.f;
  for (int b = lane; b < a.batch; b += 32) {
    const Load l = b < 32 ? mine : load_of<kPaged>(g, b);
    const int b2 = pairs.of(l), b1 = singles.of(l), t2 = pairs.turns(l, l.tiles), t1 = singles.turns(l, l.tiles);
    n2 += b2;
    n1 += b1;
    longest = max(longest, l.tiles);
    top = max(top, t2);
    total2 += 0.5f * (pairs.turns(l, tiles_of(l, pairs.span)) + t2) * b2;
    total1 += 0.5f * (singles.turns(l, tiles_of(l, singles.span)) + t1) * b1;
  }
  n2 = __reduce_add_sync(0xffffffffu, n2) * kv_heads;
  n1 = __reduce_add_sync(0xffffffffu, n1) * kv_heads;
  longest = __reduce_max_sync(0xffffffffu, longest);
  // pairs of tiles; single ones where the pairs are fewer than the CTAs, unless the keys are
  // few and not all of those would have a CTA either (1,200 tokens 20.3 us, in pairs 29.5)
  const bool single = n2 <= grid && (longest >= kMinSplit || n1 <= grid);
  const Blocks blocks = single ? singles : pairs;
  float total = single ? total1 : total2;
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) total += __shfl_xor_sync(0xffffffffu, total, o);
  top = single ? (longest + 1) / 2 : __reduce_max_sync(0xffffffffu, top);
  int count = single ? n1 : n2;  // of pieces
  // a fair share of the turns and a quarter; rows with more are split (but for those that stand
  // before position 0). 12 prompts of 1-1,411 tokens: 35.7 us, at the bare share 52.5.
  const int cap = max(kMinSplit, static_cast<int>(fminf(total * kv_heads * 1.25f / grid, 1e9f)) + 1);
  auto share = [&](Load& l) {
    l.blocks = blocks.of(l);
    l.turns = blocks.turns(l, l.tiles);
    l.splits = l.turns > cap && l.ctx >= 0 ? static_cast<int>((static_cast<unsigned>(l.turns) + cap - 1) / cap) : 1;
  };
  share(mine);
  auto request = [&](int b) {  // of lane b % 32
    if (b < 32) return mine;
    Load l = load_of<kPaged>(g, b);
    share(l);
    return l;
  };
  const bool any_split = top > cap;
  if (any_split) {
    top = count = 0;
    for (int b = lane; b < a.batch; b += 32) {
      const Load l = request(b);
      count += l.blocks * l.splits;
      top = max(top, (l.turns + l.splits - 1) / l.splits);
    }
    top = __reduce_max_sync(0xffffffffu, top);
    count = __reduce_add_sync(0xffffffffu, count) * kv_heads;
  }
  // pieces of more than x turns each, all requests
  auto pieces_above = [&](int x) {
    int n = 0;
#pragma unroll 1
    for (int b = lane; b < a.batch; b += 32) {
      const Load l = request(b);
      n += blocks.above(l, x * l.splits) * l.splits;
    }
    return __reduce_add_sync(0xffffffffu, n) * kv_heads;
  };
  // longest first, unless every piece has a CTA of its own (or the list is long: even anyway)
  const bool sorted = a.batch <= kSortBatch && count > grid;
  int k = 0, pending = kDrain ? sm.pending : blockIdx.x;  // (-1: none)
  for (;; ++k) {
    const int st = k & 1;
    int want = pending;
    if (kDrain ? k > 0 || want < 0 : k > 0) {
      pending = -1;
      if (!kDrain) wait_for(&sm.ask, (k - 1) & 1, &sm.err, dead);
      if (!kDrain && dead) break;
      if (lane == 0) want = grid + static_cast<int>(atomicAdd(g.work, 1u));
      want = __shfl_sync(0xffffffffu, want, 0);
    }
    // the level (turns of a piece) that `want` falls into, and its place there; the next
    // one wanted is never on a higher level
    int lo = 0, r = want;
    bool found = want < count;
    if (sorted && found) {
      int hi = top, at_hi = 0, n = 0;
      while (lo < hi) {
        const int mid = (lo + hi) / 2;
        if ((n = pieces_above(mid)) <= want) {
          hi = mid;
          at_hi = n;
        } else {
          lo = mid + 1;
        }
      }
      top = lo;
      r = want - (at_hi > 0 ? at_hi : pieces_above(lo));
    }
    if (!kDrain && k >= 2) {
      wait_for(&sm.info_empty[st], ((k >> 1) - 1) & 1, &sm.err, dead);
      if (dead) {
        pending = want;
        break;
      }
    }
    Piece& p = kDrain ? sm.lost : sm.piece[st];
    int slot_base = 0;
    for (int b0 = 0; b0 < a.batch && found; b0 += 32) {
      const int b = b0 + lane;
      Load l = {};
      int above = 0, here = 0, slots = 0, sp = 1;
      if (b < a.batch) {
        l = request(b);
        sp = l.splits;
        if (sorted) above = blocks.above(l, lo * sp);
        here = (sorted ? blocks.above(l, (lo - 1) * sp) - above : l.blocks) * sp * kv_heads;
        slots = sp > 1 ? l.blocks * sp * kv_heads : 0;
      }
      int inc = here, sinc = slots;  // inclusive prefix sums
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const int x = __shfl_up_sync(0xffffffffu, inc, o);
        if (lane >= o) inc += x;
      }
      if (any_split) {
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
          const int y = __shfl_up_sync(0xffffffffu, sinc, o);
          if (lane >= o) sinc += y;
        }
      }
      const bool is_it = r >= inc - here && r < inc;
      if (is_it) {
        unsigned at = static_cast<unsigned>(r) - (inc - here), split = 0;
        if (sp > 1) {
          split = at % static_cast<unsigned>(sp);
          at /= static_cast<unsigned>(sp);
        }
        const unsigned i0 = at / static_cast<unsigned>(kv_heads);
        const int hk = at - i0 * kv_heads, i = l.blocks - 1 - above - static_cast<int>(i0);  // longest first
        const int tok0 = i * blocks.span, toks = min(l.q - tok0, blocks.span);
        const int n = tiles_of(l, tok0 + toks);
        const int per = sp > 1 ? static_cast<int>((static_cast<unsigned>(n) + sp - 1) / sp) : n;
        const int k0 = min(static_cast<int>(split) * per, n), k1 = min(k0 + per, n), total = k1 - k0;
        const bool halves = toks <= g.tile_tokens;
        p.b = b;
        p.hk = hk;
        p.first = l.first;
        p.tok0 = tok0;
        p.toks = toks;
        p.ctx = l.ctx;
        p.len = l.len;
        p.k0 = k0;
        p.total = total;
        p.n[0] = halves ? (total + 1) / 2 : max(min(tiles_of(l, tok0 + g.tile_tokens), k1) - k0, 0);
        p.n[1] = halves ? total / 2 : total;
        p.halves = halves;
        p.splits = sp;
        p.split = split;
        p.slot = slot_base + sinc - slots + (i * kv_heads + hk) * sp;
        p.flags = l.bad ? kBad : 0;
        if (l.bad) report(a.status, MKB_SERVE_BAD_LENGTH);
      }
      if (__any_sync(0xffffffffu, is_it)) break;
      r -= __shfl_sync(0xffffffffu, inc, 31);
      slot_base += __shfl_sync(0xffffffffu, sinc, 31);
      found = b0 + 32 < a.batch;
    }
    if (!kDrain) {
      if (!found && lane == 0) p.b = -1;
      __syncwarp();
      if (lane == 0) mbar_arrive(&sm.info_full[st]);
    }
    if (!found) break;
    if (kDrain) {
      __syncwarp();
      void_piece<T, D>(g, p, 3);
      __syncwarp();
    }
  }
  if (!kDrain && lane == 0) {
    sm.handed = k;
    sm.open = dead;
    sm.pending = pending;
  }
  if (!kDrain && dead) return;  // (the rest of the list after the CTA's other warps)
  // the last CTA to have asked for its last piece puts the list back to its start
  if (lane == 0 && atomicInc(g.work + 1, grid - 1) == static_cast<uint32_t>(grid - 1)) atomicExch(g.work, 0u);
}
// What a CTA leaves that has stopped: the last two pieces that it was given, as far as they
// are not finished, and the rest of the list. Warp-wide.
template <typename T, int D, bool kPaged>
__device__ __noinline__ void clean_up(const TcArgs& g, TcSmem<D>& sm) {
  const int lane = threadIdx.x & 31;
  for (int k = max(sm.handed - 2, 0); k < sm.handed; ++k) {
    if (__any_sync(0xffffffffu, lane < 8 && sm.left[lane & 7] <= k))
      void_piece<T, D>(g, sm.piece[k & 1], (sm.counted[0] <= k) | (sm.counted[1] <= k) << 1);
    __syncwarp();
  }
  if (!sm.open) return;
  Load mine = {};
  if (lane < g.a.batch) mine = load_of<kPaged>(g, lane);
  bool dead = true;
  hand_out<T, D, kPaged, true>(g, sm, mine, dead);
}

template <typename T, int D, bool kPaged>
__global__ void __launch_bounds__(kTcThreads, 1)
    attn_tc_kernel(const __grid_constant__ CUtensorMap tk, const __grid_constant__ CUtensorMap tv,
                   const __grid_constant__ CUtensorMap tq, const __grid_constant__ CUtensorMap to,
                   const __grid_constant__ TcArgs g) {
  using Smem = TcSmem<D>;
  using Shape = TcShape<D>;
  constexpr int kSlots = Shape::kSlots, kTileBytes = Shape::kTileBytes;
  extern __shared__ uint8_t smem_raw[];
  Smem& sm = *reinterpret_cast<Smem*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  const mkb_attn_args& a = g.a;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  depend_launch();
  if (threadIdx.x == 0) {
    for (int s = 0; s < kSlots; ++s) {
      mbar_init(&sm.kv_full[s], 1);
      mbar_init(&sm.kv_empty[s], 2);  // both tiles' products
    }
    for (int t = 0; t < 2; ++t) {
      mbar_init(&sm.q_full[t], 1);
      mbar_init(&sm.q_empty[t], 1);
      mbar_init(&sm.s_full[t], 1);
      mbar_init(&sm.p_part[t], 4);
      mbar_init(&sm.p_full[t], 4);
      mbar_init(&sm.o_full[t], 1);
      mbar_init(&sm.info_full[t], 1);
      mbar_init(&sm.tile_bar[t], 4);
      mbar_init(&sm.info_empty[t], 11);  // eight softmax warps, two MMA warps, the loading warp
    }
    mbar_init(&sm.ask, 1);
    mbar_init(&sm.pair_full, 4);
    mbar_init(&sm.pair_empty, 4);
    for (int w = 0; w < 8; ++w) sm.left[w] = 0x7fffffff;
    sm.counted[0] = sm.counted[1] = 0;
    sm.err = sm.turn = 0;
    fence_mbar_init();
  }
  if (warp == 8) {
    tc::tmem_alloc(&sm.tmem_base, 512);
    tc::tmem_relinquish();
  }
  depend_wait();  // what came before in the stream is done: its results may be read
  Load mine = {};  // (a lane keeps its first request; the others are read again in every pass)
  if (warp == 11 && lane < a.batch) mine = load_of<kPaged>(g, lane);
  tc::fence_before_sync();
  __syncthreads();
  tc::fence_after_sync();
  // all 512 columns: the base is 0 then, which as a constant keeps the addresses out of registers
  constexpr uint32_t tbase = 0;
  bool dead = false;
  if (sm.tmem_base != 0) sm.err = 1;

  if (warp >= 8) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kOtherRegs));
  if (warp == 11) {
    hand_out<T, D, kPaged, false>(g, sm, mine, dead);
  } else if (warp == 9) {
    // ---- the loads of a piece -----------------------------------------------------------------
    if (lane == 0) {
      tc::prefetch_tensormap(&tk);
      tc::prefetch_tensormap(&tv);
      tc::prefetch_tensormap(&tq);
    }
    int slot = 0, q_uses[2] = {0, 0};  // the ring's next slot, and how often it has gone round
    uint32_t round = 0;
    for (int k = 0; !dead; ++k) {
      const int st = k & 1;
      wait_for(&sm.info_full[st], (k >> 1) & 1, &sm.err, dead);
      const Piece p = sm.piece[st];
      if (p.b < 0 || dead) break;
      if (g.withheld.here() && k >= g.withheld.from) break;
      // K(0), then K(j + 1) and V(j): the order in which the products take them
      const int n = p.total;
      int pages = 0, pages_at = 0, pages_end = 0;  // the lanes' pages: boxes of keys up to pages_end
      auto load = [&](const CUtensorMap* map, int head, int j) {
        const int s = slot;
        if (round > 0) wait_for(&sm.kv_empty[s], (round - 1) & 1, &sm.err, dead);
        if (dead) return;
        if (++slot == kSlots) {
          slot = 0;
          ++round;
        }
        const int key = (p.k0 + j) * kKeys;
        if (lane == 0) mbar_arrive_expect_tx(&sm.kv_full[s], kTileBytes);
        __syncwarp();
        if (kPaged) {
          // (a lane reads one entry of the table for several tiles to come: a lookup before every
          // copy, of K and of V, is what such loads took longest over)
          const int box = g.box;
          const int box_log = 31 - __clz(box);
          if (key + kKeys > pages_end) {
            pages_at = max(key - kKeys, 0);  // (V follows a tile behind K)
            pages_end = pages_at + 32 * box;
            const int at = pages_at + lane * box;
            pages = -2;  // past the last key: outside the pool, which reads as zeros
            if (at < p.len) {
              pages = a.block_table[p.b * a.table_stride + (at >> 31 - __clz(a.page_size))];
              if (pages < 0 || pages >= a.pages) pages = -1;
            }
          }
          const int page = __shfl_sync(0xffffffffu, pages, ((key - pages_at >> box_log) + lane) & 31);
          if (lane * box < kKeys) {
            if (page == -1) {
              atomicOr(&sm.piece[st].flags, kBad);
              report(a.status, MKB_SERVE_BAD_PAGE);
            }
            const int at = (key + lane * box) & (a.page_size - 1);
            if (g.folded) {
              const int* x = map == &tk ? g.kx : g.vx;
              tc::tma_load_5d(sm.kv[s] + lane * box * D * 2, map, 0, 0, 0, at >> 3, page < 0 ? x[2] : page * x[0] + p.hk * x[1],
                              &sm.kv_full[s]);
            } else {
#pragma unroll
              for (int d = 0; d < D / 64; ++d)
                tc::tma_load_4d(sm.kv[s] + d * kHalf + lane * box * 128, map, 64 * d, at, head,
                                page < 0 ? max(a.pages, 1) : page, &sm.kv_full[s]);
            }
          }
        } else if (lane == 0) {
#pragma unroll
          for (int d = 0; d < D / 64; ++d)
            tc::tma_load_3d(sm.kv[s] + d * kHalf, map, 64 * d, p.first + key, head, &sm.kv_full[s]);
        }
      };
      const int kh = p.hk * g.k_head, vh = p.hk * g.v_head;
      if (n > 0) load(&tk, kh, 0);
      for (int t = 0; t < 2; ++t) {  // Q once the last product of the tile's previous one has read it
        if (p.n[t] == 0) continue;
        if (q_uses[t] > 0) wait_for(&sm.q_empty[t], (q_uses[t] - 1) & 1, &sm.err, dead);
        if (dead) break;
        ++q_uses[t];
        if (lane == 0) {
          mbar_arrive_expect_tx(&sm.q_full[t], g.tile_tokens * g.group * D * 2);
#pragma unroll
          for (int d = 0; d < D / 64; ++d)
            tc::tma_load_3d(sm.q[t] + d * kHalf, &tq, 64 * d, p.hk * g.group, p.first + p.tok0 + (p.halves ? 0 : t * g.tile_tokens),
                   &sm.q_full[t]);
        }
        __syncwarp();
      }
      for (int j = 0; j < n && !dead; ++j) {
        if (lane == 0 && j == max(n - kAskTiles, 0)) mbar_arrive(&sm.ask);
        if (j + 1 < n) load(&tk, kh, j + 1);
        load(&tv, vh, j);
      }
      __syncwarp();
      if (lane == 0) {
        if (n == 0) mbar_arrive(&sm.ask);
        mbar_arrive(&sm.info_empty[st]);
      }
    }
    // after a stop, wait (bounded) for the copies still in flight before leaving
    if (sm.err) {
      int tries = 0;
      for (int s = 0; s < kSlots; ++s) {  // its last use: in this lap, or in the one before
        const uint32_t r = s < slot ? round : round - 1;
        while ((s < slot || round > 0) && !mbar_wait(&sm.kv_full[s], r & 1, kTryNs) && ++tries < kTries) {
        }
      }
      for (int t = 0; t < 2; ++t)
        while (q_uses[t] > 0 && !mbar_wait(&sm.q_full[t], (q_uses[t] - 1) & 1, kTryNs) && ++tries < kTries) {
        }
    }
  } else if (warp == 8 || warp == 10) {
    // ---- the products of a tile -------------------------------------------------------------------
    constexpr uint32_t id_s = idesc16<T>(128, kKeys, false), id_o = idesc16<T>(128, D, true);
    // K and V lie block of 64 values by block, all keys of a block one after another; where
    // they are folded, eight keys by eight, and in each the blocks
    const bool folded = kPaged && uniform(g.folded) != 0;
    const int block = folded ? 1024 : kHalf, row = folded ? D * 2 : 128;  // bytes between blocks; of a key
    const uint64_t dq0 = tc::desc_sw128(smem_addr(sm.q[0]));
    const uint64_t dk0 = tc::desc_sw128(smem_addr(sm.kv[0])) + (static_cast<uint64_t>(8 * row - 1024 >> 4) << 32);
    const uint64_t dv0 = desc_mn_sw128(smem_addr(sm.kv[0]), block, 8 * row);
    const uint32_t leader = elect_one();
    const int t = uniform((warp - 8) >> 1);
    const uint32_t ts = tbase + 128 * t, to_ = tbase + Shape::kO + D * t;
    const uint64_t dq = tc::desc_advance(dq0, t * kTileBytes);
    // the ring's next slot and the parity of its phase; K(j + 1) and V(j) of a turn are
    // neighbours in it, in that order
    int slot = 0, turn = 0;
    uint32_t ring = 0, p_ph = 0, q_ph = 0;
    auto next = [&]() {
      if (++slot == kSlots) {
        slot = 0;
        ring ^= 1;
      }
    };
    auto scores = [&](int s) {  // S = Q K^T (over the P that the last product has read: MMAs run in order)
      const uint64_t dk = tc::desc_advance(dk0, s * kTileBytes);
#pragma unroll
      for (int kk = 0; kk < D / 16; ++kk) {
        mma_ss(leader, ts, tc::desc_advance(dq, (kk >> 2) * kHalf + (kk & 3) * 32),
               tc::desc_advance(dk, (kk >> 2) * block + (kk & 3) * 32), id_s, kk != 0);
      }
      commit(leader, &sm.s_full[t]);  // covers O as well: S(j + 1) seen means PV(j) done
    };
#pragma unroll 1
    for (int k = 0; !dead; ++k) {
      const int st = k & 1;
      wait_for(&sm.info_full[st], (k >> 1) & 1, &sm.err, dead);
      // (uniform by construction: loop counts and ring slots feed the MMAs' descriptors)
      const int n = uniform(sm.piece[st].total), mine_n = uniform(sm.piece[st].n[t]);
      const int step = uniform(sm.piece[st].halves) ? 2 : 1, from = step == 2 ? t : 0;  // its key tiles
      const int last = from + step * (mine_n - 1);                                     // (below `from`: none)
      const int left = uniform(sm.piece[st].len) - uniform(sm.piece[st].k0) * kKeys;  // keys from the first tile on
      // the first tile of keys that the piece's first row does not see in full
      const int sees = uniform(sm.piece[st].ctx) + uniform(sm.piece[st].tok0) + 1;
      const int look = sees < uniform(sm.piece[st].len) ? max(sees / kKeys, 0) - uniform(sm.piece[st].k0) : 0x7fffffff;
      const bool end = uniform(sm.piece[st].b) < 0;
      if (dead) break;
      __syncwarp();
      if (lane == 0) mbar_arrive(&sm.info_empty[st]);
      if (end) break;
      if (n == 0) continue;
      if (mine_n > 0) {
        wait_for(&sm.q_full[t], q_ph, &sm.err, dead);
        q_ph ^= 1;
      }
      wait_for(&sm.kv_full[slot], ring, &sm.err, dead);
      if (dead) break;
      int todo = from, done = from;  // the next tile of scores, of outputs
      auto maybe_scores = [&](int j, int s) {
        if (j != todo || j > last) return;
        scores(s);
        if (j == last) commit(leader, &sm.q_empty[t]);
        todo += step;
      };
      maybe_scores(0, slot);
      commit(leader, &sm.kv_empty[slot]);
      next();
      // every K and V tile is released by both tiles' warps, by those too that have no use for it
#pragma unroll 1
      for (int j = 0; j < n; ++j) {
        const int sk = slot;
        if (j + 1 < n) {
          wait_for(&sm.kv_full[sk], ring, &sm.err, dead);  // K(j + 1)
          next();
        }
        // (in the other tile's turn the next scores need not wait for its V, which comes late over
        // pages: 28 requests decoding and two chunks 62.5 us, 64.4 in order; prompts lose 1 %)
        const bool mine = j == done && j <= last, early = kPaged && !mine && j + 1 < n;
        if (early) {
          if (dead) break;
          maybe_scores(j + 1, sk);
          commit(leader, &sm.kv_empty[sk]);
        }
        wait_for(&sm.kv_full[slot], ring, &sm.err, dead);  // V(j)
        if (dead) break;
        if (mine) {
          const int valid = left - j * kKeys;
          if (valid < kKeys) {  // rows past the last key: whatever lies there, P = 0 must give 0 (both warps clear them)
            const int chunks = (kKeys - valid) * 8;
#pragma unroll
            for (int d = 0; d < D / 64; ++d)
              for (int c = lane; c < chunks; c += 32)
                reinterpret_cast<uint4*>(sm.kv[slot] + (valid + c / 8 >> 3) * 8 * row + d * block + (valid + c / 8 & 7) * 128)[c % 8] =
                    make_uint4(0, 0, 0, 0);
            fence_proxy_async_shared();
            __syncwarp();
          }
          if (__builtin_expect(j >= look, 0)) {  // V that is not finite (both warps, side by side, to the same end)
            uint8_t* const v = sm.kv[slot];
            const int groups = (min(valid, kKeys) + 7) / 8;  // of eight keys
            uint32_t x[D / 32] = {}, any = 0;
#pragma unroll 2
            for (int i = 0; i < groups; ++i) {
#pragma unroll
              for (int d = 0; d < D / 32; ++d)
                x[d] = odd8<T>(reinterpret_cast<const uint4*>(v + 8 * row * i + block * (d / 2))[32 * (d % 2) + lane], x[d]);
            }
#pragma unroll
            for (int d = 0; d < D / 32; ++d) any |= x[d];
            if (__builtin_expect(__any_sync(0xffffffffu, any != 0), 0)) {
              if (lane == 0) atomicOr(&sm.piece[st].flags, kOdd);
              __threadfence_block();
              __syncwarp();
#pragma unroll 1
              for (int i = lane; i < kTileBytes / 2; i += 32) {
                uint16_t* const y = reinterpret_cast<uint16_t*>(v) + i;
                if (!finite<T>(*y)) *y = 0;
              }
            }
            fence_proxy_async_shared();
            __syncwarp();
          }
          const uint64_t dv = tc::desc_advance(dv0, slot * kTileBytes);
          // B's products queue behind A's of the same turn: side by side they would end
          // together, and both tiles' softmax run at once, on the same units (4,900 cycles
          // a turn instead of 3,250)
          if (t == 1 && step == 1) {
            for (int i = 0; *reinterpret_cast<volatile int*>(&sm.turn) - turn <= 0 && !dead; ++i) {
              __nanosleep(20);
              if (i > kTries * (kTryNs / 20) || *reinterpret_cast<volatile int*>(&sm.err) != 0)
                dead = *reinterpret_cast<volatile int*>(&sm.err) = 1;
            }
            dead = __any_sync(0xffffffffu, dead);
          }
          wait_for(&sm.p_part[t], p_ph, &sm.err, dead);
          if (dead) break;
          tc::fence_after_sync();
#pragma unroll
          for (int kk = 0; kk < kFirstKeys / 16; ++kk)  // O (+)= P V
            mma_ts(leader, to_, ts + 8 * kk, tc::desc_advance(dv, 16 * kk * row), id_o, (j - from | kk) != 0);
          wait_for(&sm.p_full[t], p_ph, &sm.err, dead);
          if (dead) break;
          p_ph ^= 1;
          tc::fence_after_sync();
#pragma unroll
          for (int kk = kFirstKeys / 16; kk < kKeys / 16; ++kk)
            mma_ts(leader, to_, ts + 8 * kk, tc::desc_advance(dv, 16 * kk * row), id_o, 1u);
          if (j == last) commit(leader, &sm.o_full[t]);
          done += step;
        }
        commit(leader, &sm.kv_empty[slot]);
        if (!early && j + 1 < n) {
          maybe_scores(j + 1, sk);
          commit(leader, &sm.kv_empty[sk]);
        }
        ++turn;
        if (t == 0 && lane == 0) *reinterpret_cast<volatile int*>(&sm.turn) = turn;
        next();
      }
    }
  }
  } else {
    asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(kSoftmaxRegs));
    // ---- softmax of a tile, a thread per row ----------------------------------------------
    const int t = warp >> 2;                 // tile
    const int row_in = threadIdx.x & 127;    // row of the tile = TMEM lane
    const uint32_t lanes = static_cast<uint32_t>(32 * (warp & 3)) << 16;
    const uint32_t t_s = tbase + lanes + 128 * t, t_o = tbase + lanes + Shape::kO + D * t;
    const float sl2 = g.sl2;
    constexpr float kLift = Pair<T>::kDtype == MKB_FP16 ? 7.f : 0.f;  // P and its sum times 2^kLift
    uint32_t s_ph = 0, o_ph = 0;
    const int tok_in = row_in * g.group_mul >> 16;
    uint32_t t_ph = 0, pair_ph = 0;
    auto tile_sync = [&]() {                 // a barrier of the tile's warps
      __syncwarp();
      if (lane == 0) mbar_arrive(&sm.tile_bar[t]);
      wait_for(&sm.tile_bar[t], t_ph, &sm.err, dead);
      t_ph ^= 1;
    };
    int k = 0;
#pragma unroll 1
    for (; !dead; ++k) {
      const int st = k & 1;
      wait_for(&sm.info_full[st], (k >> 1) & 1, &sm.err, dead);
      if (dead) break;
      const Piece p = sm.piece[st];
      auto release = [&]() {
        __syncwarp();
        if (lane == 0) mbar_arrive(&sm.info_empty[st]);
      };
      if (p.b < 0) {
        release();
        break;
      }
      const int n = p.n[t];
      const int tok_t = p.tok0 + (p.halves ? 0 : g.tile_tokens * t); // the tile's first token
      const bool live = row_in < g.tile_tokens * g.group && tok_t + tok_in < p.tok0 + p.toks;
      const int lim0 = p.ctx + tok_t;                                // the last key its first row sees
      const int lim = lim0 + tok_in;                                 // ... and this row
      float m = -INFINITY;                                           // in units of log2
      uint64_t l2 = 0;                                               // two partial sums
#pragma unroll 1
      for (int j = 0; j < n; ++j) {
        wait_for(&sm.s_full[t], s_ph, &sm.err, dead);
        if (dead) break;
        s_ph ^= 1;
        tc::fence_after_sync();
        uint32_t sr[kKeys];
#pragma unroll
        for (int c = 0; c < kKeys / 16; ++c) tmem_ld16(t_s + 16 * c, sr + 16 * c);
        tmem_wait_ld(sr);
#pragma unroll
        for (int c = 1; c < kKeys / 16; ++c) pin16(sr + 16 * c);
        const int key0 = (p.k0 + (p.halves ? 2 * j + t : j)) * kKeys;
        if (key0 + kKeys - 1 > lim0) {  // some row of the tile does not see all of these keys
#pragma unroll
          for (int i = 0; i < kKeys; ++i)
            if (key0 + i > lim) sr[i] = 0xff800000u;
        }
        float mx;
        {
          float x4[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
          for (int i = 0; i < kKeys; i += 2)
            x4[(i >> 1) & 3] = max3(x4[(i >> 1) & 3], __uint_as_float(sr[i]), __uint_as_float(sr[i + 1]));
          mx = live ? fmaxf(fmaxf(x4[0], x4[1]), fmaxf(x4[2], x4[3])) * sl2 : -INFINITY;
        }
        if (__any_sync(0xffffffffu, mx > m + 8.f)) {  // (also the first tile: m = -inf)
          const float mn = fmaxf(m, mx);
          const float sc = mn == -INFINITY ? 0.f : ex2_approx(m - mn);
          if (j > 0) {  // S(j) is there, so PV(j - 1) is done and O can be rescaled
#pragma unroll 1
            for (int c = 0; c < D / 32; ++c) {
              float o[32];
              tc::tmem_ld32(t_o + 32 * c, o);
#pragma unroll
              for (int i = 0; i < 32; ++i) o[i] *= sc;
              tc::tmem_st32(t_o + 32 * c, o);
            }
          }
          l2 = fma2(l2, pack2(sc, sc), 0);
          m = mn;
        }
        // an infinite maximum leaves no weights (inf - inf); none at all, weights of 0
        const float ref = m == -INFINITY ? 0.f : kLift - m;
        const uint64_t ref2 = pack2(ref, ref), sl22 = pack2(sl2, sl2);
        uint64_t la = 0, lb = 0;
        auto arrive = [&](uint64_t* bar) {
          tmem_wait_st();
          tc::fence_before_sync();
          __syncwarp();
          if (lane == 0) mbar_arrive(bar);
        };
#pragma unroll
        for (int c = 0; c < kKeys / 32; ++c) {
          uint32_t pw[16];
#pragma unroll
          for (int i = 0; i < 16; ++i) {
            const uint32_t* x2 = sr + 32 * c + 2 * i;
            const float2 x = unpack2(fma2(pack2(__uint_as_float(x2[0]), __uint_as_float(x2[1])), sl22, ref2));
            const float e0 = ex2_approx(x.x), e1 = ex2_approx(x.y);
            if (i & 1) lb = add2(lb, pack2(e0, e1));
            else la = add2(la, pack2(e0, e1));
            pw[i] = Pair<T>::put(e0, e1);
            if (32 * c == kFirstKeys && i == 7) arrive(&sm.p_part[t]);  // its stores have had time to land
          }
          tmem_st16(t_s + 16 * c, pw);
        }
        arrive(&sm.p_full[t]);
        l2 = add2(l2, add2(la, lb));
      }
      const float2 lf = unpack2(l2);
      float l = lf.x + lf.y;
      if (n > 0) {
        wait_for(&sm.o_full[t], o_ph, &sm.err, dead);
        o_ph ^= 1;
        tc::fence_after_sync();
      }
      // B's rows are A's: A adds the two up, each relative to its own maximum
      const bool pair = p.halves && p.n[1] > 0;
      float own = 1.f, other = 0.f;  // the weights of the two
      if (p.halves && t == 1) {
        release();
        if (pair) {
          sm.pair[row_in] = make_float2(m, l);
          tc::fence_before_sync();
          __syncwarp();
          if (lane == 0) mbar_arrive(&sm.pair_full);
          wait_for(&sm.pair_empty, pair_ph, &sm.err, dead);  // until A has read O
          pair_ph ^= 1;
        }
        continue;
      }
      if (pair) {
        wait_for(&sm.pair_full, pair_ph, &sm.err, dead);
        pair_ph ^= 1;
        tc::fence_after_sync();
        const float2 x = sm.pair[row_in];
        const float mm = fmaxf(m, x.x), ref = mm == -INFINITY ? 0.f : mm;
        own = ex2_approx(m - ref);
        other = ex2_approx(x.x - ref);
        l = l * own + x.y * other;
        m = mm;
      }
      const int flags = *reinterpret_cast<volatile int*>(&sm.piece[st].flags);
      const bool bad = (flags & kBad) != 0 || dead, odd = (flags & kOdd) != 0;
      release();
      const int k_end = min(p.len, (p.k0 + p.total) * kKeys);
      constexpr int kPer = D / 32;
      uint8_t* stage = sm.stage[warp];
      // Rows on their way out, 32 values at a time (a small loop: this code is not in the
      // instruction cache when a piece ends): 64 values of all 32 rows of the warp by a TMA
      // store where they are whole tokens of the request (and final), else a thread its own row
      const int tok_w = tok_t + g.warp_tokens * (warp & 3);
      const bool whole = g.warp_tokens > 0 && tok_w + g.warp_tokens <= p.tok0 + p.toks && !odd;
      auto emit = [&](int c, const uint32_t* w) {  // values 32 c .. + 31 of every row, packed
        if (!whole) {
          if (live) {
            T* out = static_cast<T*>(a.out) + (p.first + tok_t + tok_in) * a.out_stride[0] +
                     (p.hk * g.group + row_in - tok_in * g.group) * a.out_stride[1] + 32 * c;
#pragma unroll
            for (int i = 0; i < 4; ++i)
              reinterpret_cast<uint4*>(out)[i] = make_uint4(w[4 * i], w[4 * i + 1], w[4 * i + 2], w[4 * i + 3]);
          }
          return;
        }
        if ((c & 1) == 0) {
          if (lane == 0) tma_store_read();
          __syncwarp();
        }
#pragma unroll
        for (int i = 0; i < 4; ++i)
          *reinterpret_cast<uint4*>(stage + lane * 128 + (((4 * (c & 1) + i) ^ (lane & 7)) << 4)) =
              make_uint4(w[4 * i], w[4 * i + 1], w[4 * i + 2], w[4 * i + 3]);
        if ((c & 1) == 0) return;
        fence_proxy_async_shared();
        __syncwarp();
        if (lane == 0) tma_store_3d(stage, &to, 32 * (c - 1), p.hk * g.group, p.first + tok_w);
      };
      const bool split = p.splits > 1;
      const int at = 128 * t + row_in;
      auto slot_of = [&](int s) { return static_cast<size_t>(p.slot + s); };
      const size_t slot = slot_of(p.split);
      float4* part = g.part + slot * (D / 4) * kRows;
      // no weights at all (every score -inf) are no mean; a row that sees no key is zero
      const bool zero = lim < 0 && !bad, zeros = __any_sync(0xffffffffu, zero);
      const float inv = bad || m == -INFINITY ? NAN : 1.f / l;
      const uint64_t inv2 = pack2(inv, inv), own2 = pack2(own, own), other2 = pack2(other, other);
#pragma unroll 1
      for (int c = 0; c < D / 32; ++c) {
        uint32_t x[32];
        uint64_t o2[16];
        if (n > 0) {
          tmem_ld16(t_o + 32 * c, x);
          tmem_ld16(t_o + 32 * c + 16, x + 16);
          tmem_wait_ld(x);
          pin16(x + 16);
        } else {
#pragma unroll
          for (int i = 0; i < 32; ++i) x[i] = 0;
        }
#pragma unroll
        for (int i = 0; i < 16; ++i) o2[i] = pack2(__uint_as_float(x[2 * i]), __uint_as_float(x[2 * i + 1]));
        if (pair) {
          tmem_ld16(t_o + D + 32 * c, x);
          tmem_ld16(t_o + D + 32 * c + 16, x + 16);
          tmem_wait_ld(x);
          pin16(x + 16);
#pragma unroll
          for (int i = 0; i < 16; ++i)
            o2[i] = fma2(pack2(__uint_as_float(x[2 * i]), __uint_as_float(x[2 * i + 1])), other2, fma2(o2[i], own2, 0));
        }
        if (split) {  // one of several ranges of keys: left for whoever comes last
          if (live) {
#pragma unroll
            for (int i = 0; i < 8; ++i) {
              const float2 u = unpack2(o2[2 * i]), v = unpack2(o2[2 * i + 1]);
              part[(8 * c + i) * kRows + at] = make_float4(u.x, u.y, v.x, v.y);
            }
          }
        } else {
#pragma unroll
          for (int i = 0; i < 16; ++i) {
            const float2 u = unpack2(fma2(o2[i], inv2, 0));
            x[i] = Pair<T>::put(u.x, u.y);
          }
          if (zeros) {
#pragma unroll
            for (int i = 0; i < 16; ++i) x[i] = zero ? 0 : x[i];
          }
          emit(c, x);
        }
      }
      if (pair) {
        tc::fence_before_sync();
        __syncwarp();
        if (lane == 0) mbar_arrive(&sm.pair_empty);
      }
      if (split && live) g.stat[slot * kRows + at] = make_float2(m, bad ? NAN : l);
      // the values of V that were cleared, to the warp's rows that see them
      __syncwarp();
      if (odd && !bad) {
        int key = max(p.k0 * kKeys, max(p.ctx + p.tok0 + 1, 0) / kKeys * kKeys);
        float z[kPer] = {};  // (rows come in the order of their tokens: each sees what the one before saw)
#pragma unroll 1
        for (int r = 0; r < 32; ++r) {
          const int rt = 32 * (warp & 3) + r, tok = rt * g.group_mul >> 16;
          if (rt >= g.tile_tokens * g.group || tok_t + tok >= p.tok0 + p.toks) break;
          const int end = min(k_end, p.ctx + tok_t + tok + 1);
          if (key < end) {
            sum_odd<T, D, kPaged>(a, p.b, p.first, p.hk, key, end, z);
            key = end;
          }
#pragma unroll
          for (int i = 0; i < kPer; ++i) {
            const int d = lane * kPer + i;
            if (z[i] == 0.f) continue;
            if (split) {
              reinterpret_cast<float*>(part + (d / 4) * kRows + 128 * t + rt)[d % 4] += z[i];
            } else {
              T* const o = static_cast<T*>(a.out) + (p.first + tok_t + tok) * a.out_stride[0] +
                           (p.hk * g.group + rt - tok * g.group) * a.out_stride[1] + d;
              *o = static_cast<T>(static_cast<float>(*o) + z[i]);
            }
          }
        }
      }
      __syncwarp();
      if (split) {
        __threadfence();
        tile_sync();
        if (threadIdx.x % 128 == 0 && !dead) {
          *reinterpret_cast<volatile int*>(&sm.last[t]) =
              atomicInc(g.counters + 2 * p.slot + t, p.splits - 1) ==
              static_cast<uint32_t>(p.splits - 1);
          sm.counted[t] = k + 1;
        }
        tile_sync();
        if (!dead && *reinterpret_cast<volatile int*>(&sm.last[t]) != 0) {
          __threadfence();
          float mm = -INFINITY, ll = 0.f;
          for (int s = 0; s < p.splits && live; ++s) mm = fmaxf(mm, __ldcg(g.stat + slot_of(s) * kRows + at).x);
          const float ref = mm == -INFINITY ? 0.f : mm;
          for (int s = 0; s < p.splits && live; ++s) {
            const float2 x = __ldcg(g.stat + slot_of(s) * kRows + at);
            ll += x.y * ex2_approx(x.x - ref);
          }
          const float f0 = 1.f / ll;
          // a row's whole D at once: the loads of a range are all in flight together
          float o[D];
#pragma unroll
          for (int i = 0; i < D; ++i) o[i] = 0.f;
#pragma unroll 1
          for (int s = 0; s < p.splits && live; ++s) {
            const float w = __ldcg(g.stat + slot_of(s) * kRows + at).x;
            const float4* x4 = g.part + slot_of(s) * (D / 4) * kRows + at;
#pragma unroll
            for (int h = 0; h < D / 64; ++h) {
              float4 x[16];
#pragma unroll
              for (int i = 0; i < 16; ++i) x[i] = __ldcg(x4 + (16 * h + i) * kRows);
              if (w == -INFINITY) continue;  // that range holds no key this row sees
              const float f = ex2_approx(w - ref);
#pragma unroll
              for (int i = 0; i < 16; ++i) {
                o[64 * h + 4 * i] += f * x[i].x;
                o[64 * h + 4 * i + 1] += f * x[i].y;
                o[64 * h + 4 * i + 2] += f * x[i].z;
                o[64 * h + 4 * i + 3] += f * x[i].w;
              }
            }
          }
#pragma unroll
          for (int c = 0; c < D / 32; ++c) {
            uint32_t w[16];
#pragma unroll
            for (int i = 0; i < 16; ++i) w[i] = lim < 0 ? 0 : Pair<T>::put(o[32 * c + 2 * i] * f0, o[32 * c + 2 * i + 1] * f0);
            emit(c, w);
          }
        }
      }
      tc::fence_before_sync();  // O has been read: the next piece's first PV may overwrite it
    }
    if (lane == 0) {
      tma_store_done();
      if (dead) sm.left[warp] = k - 1;  // (the one it was at when it stopped, or the last before)
    }
  }
  tc::fence_before_sync();
  __syncthreads();
  if (sm.err) {
    if (threadIdx.x == 0) report(a.status, MKB_SERVE_TIMEOUT);
    for (int i = 0; i < 100; ++i) __nanosleep(100000);  // (products still in flight)
    if (warp == 11) clean_up<T, D, kPaged>(g, sm);
    __syncthreads();
  }
  if (warp == 8) {
    tc::fence_after_sync();
    tc::tmem_dealloc(tbase, 512);
  }
}

// ---- host side -----------------------------------------------------------------------

using EncodeTiled = CUresult (*)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*,
                                 const cuuint64_t*, const cuuint32_t*, const cuuint32_t*, CUtensorMapInterleave,
                                 CUtensorMapSwizzle, CUtensorMapL2promotion, CUtensorMapFloatOOBfill);
static EncodeTiled encoder() {
  static EncodeTiled fn = [] {
    void* p = nullptr;
    cudaDriverEntryPointQueryResult q;
    if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &p, cudaEnableDefault, &q) != cudaSuccess ||
        q != cudaDriverEntryPointSuccess)
      p = nullptr;
    return reinterpret_cast<EncodeTiled>(p);
  }();
  return fn;
}

// Rows of 64 values (of D); the dimensions after the row's are `dims` with strides of
// `strides` elements, a copy takes `box` of each. What lies outside reads as zeros.
cudaError_t map_rows(CUtensorMap* m, int dtype, const void* base, int D, int rank, const uint64_t* dims,
                            const int64_t* strides, const uint32_t* box) {
  const EncodeTiled enc = encoder();
  if (!enc) return cudaErrorNotSupported;
  cuuint64_t gd[5] = {static_cast<cuuint64_t>(D)}, gs[4];
  cuuint32_t bx[5] = {64, 1, 1, 1, 1}, es[5] = {1, 1, 1, 1, 1};
  for (int i = 0; i < rank; ++i) {
    gd[i + 1] = dims[i] > 0 ? dims[i] : 1;
    // a stride of 0 (one element, or the same place for all) is never stepped along
    gs[i] = static_cast<cuuint64_t>(strides[i] > 0 ? strides[i] : D) * 2;
    if (strides[i] == 0) gd[i + 1] = 1;
    bx[i + 1] = box[i];
  }
  const CUresult r = enc(m, dtype == MKB_BF16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16,
                         rank + 1, const_cast<void*>(base), gd, gs, bx, es, CU_TENSOR_MAP_INTERLEAVE_NONE,
                         CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                         CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  return r == CUDA_SUCCESS ? cudaSuccess : cudaErrorInvalidValue;
}

int sm_count() {
  static int n[64] = {0};
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 64) return 148;
  if (n[dev] == 0 && cudaDeviceGetAttribute(&n[dev], cudaDevAttrMultiProcessorCount, dev) != cudaSuccess) n[dev] = 0;
  return n[dev] > 0 ? n[dev] : 148;
}

// Upper bound of the pieces of a call before any split, all KV heads.
static int64_t tc_blocks(const mkb_attn_args& a) {
  return (a.tokens / (128 / (a.heads / a.kv_heads)) + a.batch) * static_cast<int64_t>(a.kv_heads);
}
// Partial results a call can leave. Rows are split only where their n turns are more than a
// cap C >= 5/4 U / grid of all U turns, into at most 2 n / C ranges; a request's blocks grow
// linearly, so that U counts at least half of n for each: at most 4 U / C < 4 grid.
static size_t tc_slots() { return 4 * static_cast<size_t>(sm_count()); }
// Counters (the place of both attention kernels', zero between calls), then partial results.
size_t counter_bytes() { return (16 + tc_slots() * 8 + 255) / 256 * 256; }
size_t tc_workspace(const mkb_attn_args& a) {
  return counter_bytes() + tc_slots() * kRows * (static_cast<size_t>(a.head_dim) * 4 + 8);
}

template <typename T, int D, bool kPaged>
static cudaError_t tc_launch(const mkb_attn_args& a, cudaStream_t stream) {
  TcArgs g;
  g.a = a;
  g.sl2 = a.scale * 1.4426950408889634f;
  g.group = a.heads / a.kv_heads;
  g.tile_tokens = 128 / g.group;
  g.warp_tokens = 32 % g.group == 0 ? 32 / g.group : 0;
  g.group_mul = 65536 / g.group + 1;
  g.k_head = a.k_stride[1] != 0;
  g.v_head = a.v_stride[1] != 0;
  g.withheld = withheld();
  uint8_t* ws = static_cast<uint8_t*>(a.workspace);
  if (ws == nullptr) return cudaErrorInvalidValue;
  g.tile_mul = g.tile_tokens > 1 ? static_cast<unsigned>((1ull << 32) / g.tile_tokens + 1) : 0;
  g.work = reinterpret_cast<uint32_t*>(ws);
  g.counters = g.work + 4;
  g.stat = reinterpret_cast<float2*>(ws + counter_bytes());
  g.part = reinterpret_cast<float4*>(g.stat + tc_slots() * kRows);
  CUtensorMap mk, mv, mq, mo;
  cudaError_t e;
  {
    const uint64_t dims[2] = {static_cast<uint64_t>(a.heads), static_cast<uint64_t>(a.tokens)};
    const int64_t qs[2] = {a.q_stride[1], a.q_stride[0]};
    const uint32_t box[2] = {static_cast<uint32_t>(g.group), static_cast<uint32_t>(g.tile_tokens)};
    if ((e = map_rows(&mq, a.dtype, a.q, D, 2, dims, qs, box)) != cudaSuccess) return e;
    mo = mq;
    if (g.warp_tokens > 0) {
      const int64_t os[2] = {a.out_stride[1], a.out_stride[0]};
      const uint32_t obox[2] = {box[0], static_cast<uint32_t>(g.warp_tokens)};
      if ((e = map_rows(&mo, a.dtype, a.out, D, 2, dims, os, obox)) != cudaSuccess) return e;
    }
  }
  g.box = kPaged && a.page_size < kKeys ? a.page_size : kKeys;
  const uint32_t kbox[3] = {static_cast<uint32_t>(g.box), 1, 1};
  const void *kb = a.k, *vb = a.v;
  if (kPaged && a.pages == 0) kb = vb = a.q;  // an empty pool is never read: any address will do
  // What a copy of a page's keys costs is the copy (80 cycles of the loading warp, and a tile has
  // 128 / page_size of them), so one brings all blocks of 64 values: keys are groups of eight, a
  // key of a group, blocks and groups three dimensions, laid down as the products' operands want
  // them. That leaves one of a map's five for page and KV head, which are folded: where one of
  // their strides is a multiple of the other. (28 requests decoding and two chunks, pages of 16:
  // 62.3 us, 73.5 by a copy a block; four chunks of 512, pages of 32: 44.5, 47.8.)
  g.folded = kPaged;
  uint64_t fold_dim[2];
  int64_t fold_stride[2];
  for (int i = 0; i < 2 && kPaged; ++i) {
    const int64_t *st = i ? a.v_stride : a.k_stride, ps = st[0], hs = a.kv_heads > 1 ? st[1] : 0;
    int64_t page_x = 1, head_x = 0, unit = ps;
    if (hs > 0 && a.pages <= 1) {
      page_x = 0, head_x = 1, unit = hs;
    } else if (hs > 0 && ps % hs == 0) {
      page_x = ps / hs, head_x = 1, unit = hs;
    } else if (hs > 0 && hs % ps == 0) {
      head_x = hs / ps;
    } else if (hs > 0) {
      g.folded = 0;
    }
    const int64_t pages = a.pages > 0 ? a.pages : 1;
    if (page_x > INT32_MAX / pages || head_x > INT32_MAX / a.kv_heads) {
      g.folded = 0;
      continue;
    }
    const int64_t end = (pages - 1) * page_x + (a.kv_heads - 1) * head_x + 1;
    if (end > INT32_MAX) g.folded = 0;
    int* const x = i ? g.vx : g.kx;
    x[0] = static_cast<int>(page_x);
    x[1] = static_cast<int>(head_x);
    x[2] = static_cast<int>(end);
    fold_dim[i] = static_cast<uint64_t>(end);
    fold_stride[i] = unit;
  }
  if (kPaged && g.folded) {
    const uint32_t box[4] = {8, D / 64, static_cast<uint32_t>(g.box / 8), 1};
    for (int i = 0; i < 2; ++i) {
      const int64_t slot = i ? a.v_stride[2] : a.k_stride[2];
      const uint64_t dims[4] = {8, D / 64, static_cast<uint64_t>(a.page_size / 8), fold_dim[i]};
      const int64_t strides[4] = {slot, 64, 8 * slot, fold_stride[i]};
      if ((e = map_rows(i ? &mv : &mk, a.dtype, i ? vb : kb, 64, 4, dims, strides, box)) != cudaSuccess) return e;
    }
  } else if (kPaged) {
    const uint64_t dims[3] = {static_cast<uint64_t>(a.page_size), static_cast<uint64_t>(a.kv_heads),
                              static_cast<uint64_t>(a.pages)};
    const int64_t ks[3] = {a.k_stride[2], a.k_stride[1], a.k_stride[0]};
    const int64_t vs[3] = {a.v_stride[2], a.v_stride[1], a.v_stride[0]};
    if ((e = map_rows(&mk, a.dtype, kb, D, 3, dims, ks, kbox)) != cudaSuccess) return e;
    if ((e = map_rows(&mv, a.dtype, vb, D, 3, dims, vs, kbox)) != cudaSuccess) return e;
  } else {
    const uint64_t dims[2] = {static_cast<uint64_t>(a.tokens), static_cast<uint64_t>(a.kv_heads)};
    if ((e = map_rows(&mk, a.dtype, kb, D, 2, dims, a.k_stride, kbox)) != cudaSuccess) return e;
    if ((e = map_rows(&mv, a.dtype, vb, D, 2, dims, a.v_stride, kbox)) != cudaSuccess) return e;
  }
  constexpr int bytes = sizeof(TcSmem<D>) + 1024;
  static_assert(bytes <= 232448, "shared memory of the attention kernel");
  static bool configured[64] = {false};
  int dev = 0;
  if ((e = cudaGetDevice(&dev)) != cudaSuccess) return e;
  if (dev < 0 || dev >= 64) return cudaErrorInvalidDevice;
  if (!configured[dev]) {
    e = cudaFuncSetAttribute(attn_tc_kernel<T, D, kPaged>, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes);
    if (e != cudaSuccess) return e;
    configured[dev] = true;
  }
  // at least one row block a CTA, unless keys are split: then every SM may have a part
  const int64_t blocks = tc_blocks(a) * (kPaged ? (static_cast<int64_t>(a.table_width) * a.page_size / kKeys) / kMinSplit + 1
                                                : a.tokens / (kKeys * kMinSplit) + 1);
  const int grid = static_cast<int>(blocks < sm_count() ? blocks : sm_count());
  return launch_early(attn_tc_kernel<T, D, kPaged>, grid, kTcThreads, bytes, stream, mk, mv, mq, mo, g);
}

template <typename T>
static cudaError_t tc_type(const mkb_attn_args& a, bool paged, cudaStream_t stream) {
  if (a.head_dim == 128) return paged ? tc_launch<T, 128, true>(a, stream) : tc_launch<T, 128, false>(a, stream);
  return paged ? tc_launch<T, 64, true>(a, stream) : tc_launch<T, 64, false>(a, stream);
}

cudaError_t attn_tc(const mkb_attn_args& a, bool paged, cudaStream_t stream) {
  return a.dtype == MKB_BF16 ? tc_type<__nv_bfloat16>(a, paged, stream) : tc_type<__half>(a, paged, stream);
}

}  // namespace sv
}  // namespace mkb
