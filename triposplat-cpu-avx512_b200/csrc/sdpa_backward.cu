// Exact attention for training, head_dim 64, scale 1/8, fp32 in and out: the forward pass on the
// attention kernel of sdpa.cu with each row's softmax statistics kept, and the backward pass,
// which recomputes the probabilities.  No Lq x Lk matrix is ever stored.
//
// Mathematics.  With x_ij = (q_i . k_j / 8 + b_j) log2 e, the forward pass keeps per row an integer
// reference m_i (at most 8 below the row's maximum) and l_i = sum_j e_ij, e_ij = 2^(x_ij - m_i).
// The backward pass folds 1 / l_i into the incoming gradient once per row,
//   g_i = dO_i / l_i,   delta_i = g_i . O_i,
// and then needs no other row factor:
//   dV_j = sum_i e_ij g_i ;  dS_ij = e_ij (g_i . v_j - delta_i) ;
//   dQ_i = sum_j dS_ij k_j / 8 ;  dK_j = sum_i dS_ij q_i / 8 ;  db_j = sum_i dS_ij.
//
// Key bias.  -inf means that the key does not exist: its K and V rows are read as zeros (they may
// hold anything) and its gradients are zero; a row without a key is zeros, forward and backward.
// Finite values are taken relative to their largest, which a softmax does not see, so that
// none overflows; where the largest is beyond 2^60 in magnitude (a mask of the type's lowest
// value on every key) the scores vanish next to it in any arithmetic, and the softmax is that of
// the bias alone.
//
// Two passes, each the owner of its outputs, instead of one with atomics on dQ: the results are
// the same bits on every run.  The keys' pass holds 128 keys and walks the queries
// (S^T, dP^T, dV, dK: four products), the queries' pass holds 128 queries and walks the keys (S, dP,
// dQ: three).  Both are one kernel and one launch: F1, F2 are the held operands (K, V or Q, g), G1, G2
// the walked ones (Q, g or K, V):
//   X = F1 G1^T ;  Y = F2 G2^T ;  e = 2^(c X + column + row) ;  ds = e (a Y - delta) ;
//   acc1 += ds G1   (dK or dQ) ;  acc2 += e G2   (dV, keys' pass only).
//
// Split precision as in sdpa.cu: every operand is an fp16 pair hi + lo after an exact power-of-two
// scale (one per 128-row tile; 2^7 for e <= 2^8, and for ds a power of two from the tiles' largest
// norms, |g . v - delta| <= |g| |v| + |delta|), each product is three tensor-core passes (hi.lo, lo.hi,
// hi.hi), and the products of two walked tiles go into a fresh accumulator in tensor memory that is
// added to fp32 registers: the tensor core's own fp32 accumulation truncates, and one accumulator over
// thousands of rows would drift.  Measured at 8193 x 8193: errors of 5e-7 (dq, dk, dv; 2-norm), 1.2e-6
// with hi.hi first; a tile per accumulator gives 4e-7 and takes 3% longer.
//
// CTA: 384 threads, one per SM, persistent over work items (pass, head, held tile, share of the walk).
// Warp 0 loads walked tiles (64 rows: 32 KB of planes and the tile's vectors, kStages deep), warp 1
// issues all MMAs, two warpgroups compute: thread = held row = tensor-memory lane, warpgroup = 32
// walked rows.  The held operands live in tensor memory as the A side of X and Y (128 columns), so
// that shared memory feeds the tensor core only the walked side: measured, an MMA of 128 x 64 x 16
// takes its 32 cycles with A in tensor memory and 48 with both operands in shared memory.  X and Y
// have two buffers of 64 columns each: the tensor core forms X, Y of the next tile while the
// warpgroups turn the current ones, in place, into the fp16 pairs of e and ds, the A side of the
// accumulating products.  G1, G2 are read from the same shared tile both ways: K-major for X
// and Y (the 64 head dimensions contracted), MN-major for the accumulators (rows contracted).
//
// Few held tiles (a handful of queries or keys): walks are cut into shares where that ends sooner
// (cut_walks), each share writes partial sums, and a last kernel adds them in their order.  Tiles of 128 keys
// without a key at either end of a row (padding) are left out.
//
// Bound.  8193 x 8193, 32 heads: forward 1.30 to 1.37 ms, backward 4.37 ms, preparation of the planes 64 and 102 us.
// Nine products (two forward, seven backward) in three passes each are 7.4 TFLOP: 1.3 PFLOP/s, 0.93 of what
// a library bf16 product sustains under the power cap (1.41, at the 1.35 to 1.65 GHz that it leaves); the clock, not
// the issue of MMAs, is what is left.  2049 x 1374 of two requests, one without keys: 62 and 120 us.
#include <stdint.h>

#include <atomic>
#include <initializer_list>

#include "common.cuh"
#include "runtime.h"
#include "sdpa_planes.h"

namespace tsb {
namespace sdpab {

constexpr int D = 64;
constexpr int HELD = 128;               // rows of a held tile
constexpr int WALK = 64;                // rows of a walked tile (two share their scales and accumulators)
constexpr int kThreads = 384;
constexpr int kStages = 4;
constexpr int PLANE = WALK * D * 2;     // 8 KB: one 64 x 64 fp16 tile
constexpr int STAGE = 4 * PLANE;                      // G1 hi, lo, G2 hi, lo
constexpr int VEC_STAGE = 2 * WALK * 4 + 16;          // column vector, deltas, the tile's scales
constexpr int SMEM_BYTES = 1024 + kStages * (STAGE + VEC_STAGE) + 32 * 8 + 16;
constexpr int TMEM_COLS = 512;
constexpr int F_COL = 0;                // F1 hi, F1 lo, F2 hi, F2 lo: 32 columns each
constexpr int XY_COL = 128;             // two buffers of X (64) and Y (64)
constexpr int ACC_COL = 384;            // acc1 (64), acc2 (64); queries' pass: two buffers of acc1
constexpr float LOG2E = 1.4426950408889634f;
constexpr float E_LIFT = 7.0f;          // e is formed as e * 2^7 <= 2^15, inside fp16's range
// Register split as in sdpa.cu: 168 a thread at launch, 56 for the control warps, 224 for the rest.
constexpr uint32_t REGS_LAUNCH = 168, REGS_CONTROL = 56, REGS_COMPUTE = 224;
static_assert((REGS_CONTROL + 2 * REGS_COMPUTE) * 128 <= REGS_LAUNCH * kThreads, "register split");

__device__ __forceinline__ float pow2i(int s) { return __int_as_float((127 + s) << 23); }

// s with mx * 2^s in [2^14, 2^15), within [-100, 100]; 0 for 0 and what is not finite
__device__ __forceinline__ int scale_shift(float mx) {
  if (!(mx > 0.0f) || !(mx <= 3.402823466e38f)) return 0;
  const int s = 14 - ilogbf(mx);
  return s < -100 ? -100 : (s > 100 ? 100 : s);
}

__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ uint64_t f2pack(float a, float b) {
  uint64_t r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(a), "f"(b));
  return r;
}
__device__ __forceinline__ void f2unpack(uint64_t v, float& a, float& b) {
  asm("mov.b64 {%0, %1}, %2;" : "=f"(a), "=f"(b) : "l"(v));
}
__device__ __forceinline__ uint64_t f2fma(uint64_t a, uint64_t b, uint64_t c) {
  uint64_t r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
  return r;
}
__device__ __forceinline__ uint64_t f2mul(uint64_t a, uint64_t b) {
  uint64_t r;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
__device__ __forceinline__ uint64_t f2add(uint64_t a, uint64_t b) {
  uint64_t r;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
__device__ __forceinline__ uint64_t f2sub(uint64_t a, uint64_t b) {
  uint64_t r;
  asm("sub.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}

// hi / lo fp16 pairs of two values: hi is the value with the 13 low mantissa bits cleared, lo the
// exact remainder
__device__ __forceinline__ void split2(uint64_t v, uint32_t& hi, uint32_t& lo) {
  float a, b;
  f2unpack(v, a, b);
  const float ha = __uint_as_float(__float_as_uint(a) & 0xFFFFE000u);
  const float hb = __uint_as_float(__float_as_uint(b) & 0xFFFFE000u);
  float la, lb;
  f2unpack(f2sub(v, f2pack(ha, hb)), la, lb);
  const __half2 h = __floats2half2_rn(ha, hb), l = __floats2half2_rn(la, lb);
  hi = *reinterpret_cast<const uint32_t*>(&h);
  lo = *reinterpret_cast<const uint32_t*>(&l);
}

// untiled bulk copy, global -> shared (16-byte aligned, a multiple of 16 bytes)
__device__ __forceinline__ void bulk_load(void* dst, const void* src, uint32_t bytes, uint64_t* bar) {
  asm volatile(
      "cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(
          smem_u32(dst)),
      "l"(src), "r"(bytes), "r"(smem_u32(bar))
      : "memory");
}

// D = A B (FRESH) or D += A B over 64 contracted elements in three passes.  A: hi and lo pairs A_STEP columns per
// 16 elements apart, lo A_LO columns behind hi; B: tiles hi and lo (PLANE apart), B_STEP 16-byte units
// per 16 elements.  The two small passes come first: every step truncates the sum so far, and this
// way it is small (2^-11 of the result) for all steps of a fresh product but the last four.
template <int A_STEP, int A_LO, int B_STEP, bool FRESH>
__device__ __forceinline__ void product(uint32_t d, uint32_t a, uint32_t b_lo, uint32_t idesc) {
#pragma unroll
  for (int kk = 0; kk < 4; ++kk) {
    const uint32_t ah = a + kk * A_STEP, bh = b_lo + kk * B_STEP;
    if (FRESH && kk == 0) mma_step_ts<false>(d, ah, bh + (PLANE >> 4), idesc);
    else mma_step_ts<true>(d, ah, bh + (PLANE >> 4), idesc);
    mma_step_ts<true>(d, ah + A_LO, bh, idesc);
  }
#pragma unroll
  for (int kk = 0; kk < 4; ++kk) mma_step_ts<true>(d, a + kk * A_STEP, b_lo + kk * B_STEP, idesc);
}

// One scale tile (128 rows) of the two tensors of a side.
struct TileScale {
  float inv1, inv2;   // inverse pre-scales of (Q, g) or (K, V)
  float norm, delta;  // queries: largest |g_i|, |delta_i|; keys: largest |v_j|, 0
};

// The two sides' planes, all [BH, rows padded to 128, 64] fp16, rows past the end zero.
struct Side {
  __half *hi1, *lo1, *hi2, *lo2;
  float *col;         // queries: 7 - m_i (-inf past the end and for rows without a key); keys: bias in log2 units
  float *delta;       // queries: -delta_i; keys: unused
  TileScale* scale;   // [BH, padded / 128]
  int L, Lt;          // rows, padded rows
};

// One pass: what it holds and walks, how its walk is cut, where its gradients go.
struct Pass {
  Side held, walk;
  float *out1, *out2;  // dK (or dQ), dV; with cuts, partial sums [cuts, BH, held.Lt, 64] instead
  int64_t s1b, s1h, s1l, s2b, s2h, s2l;  // element strides of out1, out2
  int T, Ft;           // walked tiles, held tiles per head
  int cuts, span;      // shares of the walk, walked tiles per share (even unless there is one share)
  int ragged;          // the last walked tile ends before its 64 rows
  int vec_out;         // 16-byte stores
};

struct Params {
  Pass keys, queries;
  const float2* head;  // [BH] head_stride apart: .y = 0 where the bias leaves the scores no weight, 1 otherwise
  int64_t head_stride;
  const int2* tiles;   // with a bias, [BH]: first 128-key tile with a key and the one past the last
  float* db;           // nullable: [cuts, 2, BH, Lt of the keys] sums of ds over each warpgroup's queries
  int H, BH;
  int key_items, items;
  int keys_last;       // the queries' items come first (the longer ones do)
  int* next;           // items handed out beyond the first of each CTA
  int* status;
};

struct Maps {
  CUtensorMap q1h, q1l, q2h, q2l, k1h, k1l, k2h, k2l;
};

// Work item j: the pass with the longer items first; shares of a walk next to each other, then held tiles,
// then heads.  A CTA starts with item blockIdx.x and then takes the next one that is left, so that
// items of different lengths fill the SMs evenly; which CTA works on an item changes no result.
// Tiles without a key at either end (padding) are left out: held ones have nothing to walk.
struct Item {
  bool keys;
  int bh, f0, t0, n, cut;  // head, first held row, walked tiles [t0, t0 + n)
};
template <bool BIAS>
__device__ __forceinline__ Item item_of(const Params& p, int j) {
  Item it;
  const int first = p.keys_last ? p.items - p.key_items : p.key_items;
  it.keys = (j < first) != (bool)p.keys_last;
  const Pass& s = it.keys ? p.keys : p.queries;
  if (j >= first) j -= first;
  it.cut = j % s.cuts;
  j /= s.cuts;
  it.bh = j / s.Ft;
  it.f0 = (j - it.bh * s.Ft) * HELD;
  it.t0 = it.cut * s.span;
  it.n = min(s.span, s.T - it.t0);
  if (BIAS) {
    const int2 r = __ldg(p.tiles + it.bh);
    if (it.keys) {
      if (it.f0 < r.x * HELD || it.f0 >= r.y * HELD) it.n = 0;
    } else {
      const int end = min(it.t0 + it.n, r.y * (HELD / WALK));
      it.t0 = max(it.t0, r.x * (HELD / WALK));
      it.n = max(end - it.t0, 0);
    }
  }
  return it;
}

// A wait of a whole warp: one lane polls.
__device__ __forceinline__ bool warp_wait(uint64_t* bar, uint32_t parity, int* status, int code, volatile int* abort_flag) {
  int ok = 1;
  if (lane_id() == 0) ok = mbar_wait(bar, parity, status, code, abort_flag);
  return __shfl_sync(0xffffffffu, ok, 0) != 0;
}

// Of one walked tile, the 32 columns of this thread's row that its warpgroup has: X and Y in, e
// (KEYS) and ds out as fp16 pairs over them.  The exponent's offset is a column's (COL) or the row's
// (ROW) or both; the column's and the row's delta come in the units of a * Y.
template <bool KEYS, bool COL, bool ROW>
__device__ __forceinline__ void tile_math(uint32_t x0, const uint32_t (&xv)[32], const uint32_t (&yv)[32],
                                          const float4* col, const float4* del, float c, float a, float up, float row,
                                          float row_delta, uint64_t& dsum) {
  // up: ds is formed times 2^kk, e is lifted by 2^7; the queries' pass has both in a and row_delta
  const uint64_t c2 = f2pack(c, c), a2 = f2pack(a, a), up2 = f2pack(up, up);
  const uint64_t row2 = f2pack(row, row), rd2 = f2pack(row_delta, row_delta);
#pragma unroll
  for (int ch = 0; ch < 2; ++ch) {  // 16 walked rows: 8 columns of hi pairs, 8 of lo pairs
    uint32_t pe[16], pd[16];
#pragma unroll
    for (int j = 0; j < 16; j += 4) {
      const int q = ch * 16 + j;
      const float4 cv = COL ? col[q / 4] : make_float4(0.f, 0.f, 0.f, 0.f);
      const float4 dv = KEYS ? del[q / 4] : make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const int k = q + 2 * h;
        uint64_t off = row2;
        if (COL) {
          off = h == 0 ? f2pack(cv.x, cv.y) : f2pack(cv.z, cv.w);
          if (ROW) off = f2add(off, row2);
        }
        float e0, e1;
        f2unpack(f2fma(f2pack(__uint_as_float(xv[k]), __uint_as_float(xv[k + 1])), c2, off), e0, e1);
        const uint64_t e = f2pack(ex2(e0), ex2(e1));
        const uint64_t nd = KEYS ? (h == 0 ? f2pack(dv.x, dv.y) : f2pack(dv.z, dv.w)) : rd2;
        const uint64_t y = f2fma(f2pack(__uint_as_float(yv[k]), __uint_as_float(yv[k + 1])), a2, nd);
        const uint64_t ds = f2mul(KEYS ? f2mul(e, up2) : e, y);
        if (KEYS) split2(e, pe[j / 2 + h], pe[8 + j / 2 + h]);
        if (KEYS && ROW) dsum = f2add(dsum, ds);
        split2(ds, pd[j / 2 + h], pd[8 + j / 2 + h]);
      }
    }
    if (KEYS) tmem_st16(x0 + ch * 16, pe);
    tmem_st16(x0 + 64 + ch * 16, pd);
  }
}

// Barriers and shared memory of a CTA, and the counts that its roles keep in step: walked tiles (G)
// and pairs of them (P) so far, over all items.
struct Shared {
  uint8_t *tiles, *vecs;  // [kStages] G1 hi, lo, G2 hi, lo; [kStages] columns, deltas, scales
  uint64_t* full;         // [kStages] walked tile loaded
  uint64_t* empty;        // [kStages] both products of the tile retired
  uint64_t* xy_full;      // [2] X, Y formed
  uint64_t* ed_full;      // [2] e, ds written over them (8 warps)
  uint64_t* acc_full;     // [2] accumulators of a pair formed
  uint64_t* acc_free;     // [2] ... and folded into registers (8 warps)
  uint64_t* held_full;    // the item's held operands are in tensor memory (8 warps)
  uint64_t* all_done;
  uint64_t* item_full;    // [2] the next item's number is in items[]
  uint64_t* item_empty;   // [2] ... and read (MMA thread, 8 warps)
  volatile int* items;    // [2]
  uint32_t* tmem_slot;
  volatile int* abort_flag;
};

__device__ __forceinline__ Shared carve(uint8_t* raw) {
  Shared s;
  s.tiles = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(raw) + 1023) & ~static_cast<uintptr_t>(1023));
  s.vecs = s.tiles + kStages * STAGE;
  s.full = reinterpret_cast<uint64_t*>(s.vecs + kStages * VEC_STAGE);
  s.empty = s.full + kStages;
  s.xy_full = s.empty + kStages;
  s.ed_full = s.xy_full + 2;
  s.acc_full = s.ed_full + 2;
  s.acc_free = s.acc_full + 2;
  s.held_full = s.acc_free + 2;
  s.all_done = s.held_full + 1;
  s.item_full = s.all_done + 1;
  s.item_empty = s.item_full + 2;
  s.items = reinterpret_cast<volatile int*>(s.item_empty + 2);
  s.tmem_slot = reinterpret_cast<uint32_t*>(const_cast<int*>(s.items) + 2);
  s.abort_flag = reinterpret_cast<volatile int*>(s.tmem_slot + 1);
  return s;
}

// Warp 0, one thread: an item's walked tiles.
template <bool KEYS>
__device__ __forceinline__ bool load_item(const Params& p, const Pass& ps, const Item& it, const CUtensorMap* m1h,
                                          const CUtensorMap* m1l, const CUtensorMap* m2h, const CUtensorMap* m2l,
                                          const Shared& sh, int& G) {
  for (int t = it.t0; t < it.t0 + it.n; ++t, ++G) {
    const int st = G % kStages;
    if (G >= kStages &&
        !mbar_wait(&sh.empty[st], ((G / kStages) & 1) ^ 1, p.status, kDevTimeoutProducer, sh.abort_flag))
      return false;
    uint8_t* d = sh.tiles + st * STAGE;
    uint8_t* v = sh.vecs + st * VEC_STAGE;
    const int64_t row = (int64_t)it.bh * ps.walk.Lt + t * WALK;
    mbar_arrive_expect_tx(&sh.full[st], STAGE + WALK * 4 * (KEYS ? 2 : 1) + 16);
    tma_load_3d(d, m1h, &sh.full[st], 0, t * WALK, it.bh);
    tma_load_3d(d + PLANE, m1l, &sh.full[st], 0, t * WALK, it.bh);
    tma_load_3d(d + 2 * PLANE, m2h, &sh.full[st], 0, t * WALK, it.bh);
    tma_load_3d(d + 3 * PLANE, m2l, &sh.full[st], 0, t * WALK, it.bh);
    bulk_load(v, ps.walk.col + row, WALK * 4, &sh.full[st]);
    if (KEYS) bulk_load(v + WALK * 4, ps.walk.delta + row, WALK * 4, &sh.full[st]);
    bulk_load(v + 2 * WALK * 4, ps.walk.scale + row / HELD, 16, &sh.full[st]);
  }
  return true;
}

// Warp 1, one thread: an item's MMAs.  X, Y of tile t + 1 are issued ahead of tile t's accumulating
// products, so the tensor core has them to do while e, ds of tile t are formed.  Their buffer's last
// readers, the products of tile t - 1, come before them in the same order.
template <bool KEYS>
__device__ __forceinline__ bool mma_item(const Params& p, int n, const Shared& sh, uint32_t tmem, int& G, int& P) {
  constexpr uint32_t idesc_xy = idesc_f16_f32(HELD, WALK);
  constexpr uint32_t idesc_acc = idesc_f16_f32(HELD, D) | (1u << 16);  // B MN-major
  auto form_xy = [&](int g_) -> bool {
    const int st = g_ % kStages;
    if (!mbar_wait(&sh.full[st], (g_ / kStages) & 1, p.status, kDevTimeoutMma, sh.abort_flag)) return false;
    tc_fence_after();
    const uint32_t g = sw128_desc_lo(smem_u32(sh.tiles + st * STAGE));
    const uint32_t x = tmem + XY_COL + (g_ & 1) * 128;
    product<8, 32, 32 / 16, true>(x, tmem + F_COL, g, idesc_xy);                                // F1 G1^T
    product<8, 32, 32 / 16, true>(x + 64, tmem + F_COL + 64, g + (2 * PLANE >> 4), idesc_xy);  // F2 G2^T
    mma_commit(&sh.xy_full[g_ & 1]);
    return true;
  };
  if (n > 0 && !form_xy(G)) return false;
  for (int t = 0; t < n; ++t, ++G) {
    const int st = G % kStages;
    if (t + 1 < n && !form_xy(G + 1)) return false;
    // accumulators of pair P: the keys' pass has one buffer, the queries' two
    const int prev = KEYS ? P - 1 : P - 2;
    if (!mbar_wait(&sh.ed_full[G & 1], (G >> 1) & 1, p.status, kDevTimeoutMma, sh.abort_flag)) return false;
    if (!(t & 1) && prev >= 0 &&
        !mbar_wait(&sh.acc_free[prev & 1], (prev >> 1) & 1, p.status, kDevTimeoutMma, sh.abort_flag))
      return false;
    tc_fence_after();
    const uint32_t g = sw128_desc_lo(smem_u32(sh.tiles + st * STAGE));
    const uint32_t x = tmem + XY_COL + (G & 1) * 128;
    const uint32_t acc1 = tmem + ACC_COL + (KEYS ? 0 : (P & 1) * 64);
    if (t & 1) {
      if (KEYS) product<16, 8, 2048 / 16, false>(acc1 + 64, x, g + (2 * PLANE >> 4), idesc_acc);  // e G2
      product<16, 8, 2048 / 16, false>(acc1, x + 64, g, idesc_acc);                              // ds G1
    } else {
      if (KEYS) product<16, 8, 2048 / 16, true>(acc1 + 64, x, g + (2 * PLANE >> 4), idesc_acc);
      product<16, 8, 2048 / 16, true>(acc1, x + 64, g, idesc_acc);
    }
    mma_commit(&sh.empty[st]);
    if ((t & 1) || t + 1 == n) {
      mma_commit(&sh.acc_full[P & 1]);
      ++P;
    }
  }
  return true;
}

// The two compute warpgroups: an item's e, ds, folds and gradients.
template <bool KEYS, bool BIAS>
__device__ __forceinline__ bool compute_item(const Params& p, const Pass& ps, const Item& it, const Shared& sh,
                                             uint32_t tmem, int& G, int& P) {
  const uint32_t warp = warp_id(), lane = lane_id(), sub = warp & 3;
  const int w = (warp - 4) >> 2;  // warpgroup w has walked rows 32w..32w+31
  const int r = sub * 32 + lane;  // held row == tensor-memory lane
  const uint32_t trow = tmem + ((sub * 32) << 16);
  constexpr int NACC = KEYS ? 64 : 32;  // keys: w = 0 keeps dV, w = 1 dK; queries: half of dQ each
  const int64_t frow = (int64_t)it.bh * ps.held.Lt + it.f0 + r;
  {
    // held operands into tensor memory: this warpgroup's pair of planes
    const __half* hi = w == 0 ? ps.held.hi1 : ps.held.hi2;
    const __half* lo = w == 0 ? ps.held.lo1 : ps.held.lo2;
#pragma unroll
    for (int pl = 0; pl < 2; ++pl) {
      const uint4* src = reinterpret_cast<const uint4*>((pl == 0 ? hi : lo) + frow * D);
      uint32_t v[32];
#pragma unroll
      for (int k = 0; k < 8; ++k) {
        const uint4 u = __ldg(src + k);
        v[4 * k] = u.x; v[4 * k + 1] = u.y; v[4 * k + 2] = u.z; v[4 * k + 3] = u.w;
      }
      tmem_st32(trow + F_COL + w * 64 + pl * 32, v);
    }
    tmem_wait_st();
    tc_fence_before();
    __syncwarp();
    if (lane == 0) mbar_arrive(sh.held_full);
  }
  const TileScale fs = ps.held.scale[frow / HELD];
  const float c0 = 0.125f * LOG2E * p.head[it.bh * p.head_stride].y * fs.inv1;
  // row constants: queries' pass 7 - m_i and -delta_i, keys' pass b_j
  const float row = ps.held.col[frow], row_delta = KEYS ? 0.0f : ps.held.delta[frow];
  uint64_t acc[NACC / 2];
#pragma unroll
  for (int k = 0; k < NACC / 2; ++k) acc[k] = 0ull;
  float db = 0.0f, fold_scale = 0.0f;
  // adds the accumulators of the next pair to the registers
  auto fold = [&]() -> bool {
    if (!warp_wait(&sh.acc_full[P & 1], (P >> 1) & 1, p.status, kDevTimeoutConsumer, sh.abort_flag)) return false;
    tc_fence_after();
    const uint32_t src = trow + ACC_COL + (KEYS ? (w == 0 ? 64 : 0) : (P & 1) * 64 + w * 32);
    const uint64_t s2 = f2pack(fold_scale, fold_scale);
    uint32_t v[NACC / 32][32];
#pragma unroll
    for (int c = 0; c < NACC / 32; ++c) tmem_ld32(src + c * 32, v[c]);
    tmem_wait_ld();
#pragma unroll
    for (int c = 0; c < NACC / 32; ++c) reg_fence(v[c]);
    tc_fence_before();
    __syncwarp();
    if (lane == 0) mbar_arrive(&sh.acc_free[P & 1]);
    ++P;
#pragma unroll
    for (int c = 0; c < NACC / 32; ++c)
#pragma unroll
      for (int k = 0; k < 32; k += 2)
        acc[c * 16 + k / 2] = f2fma(f2pack(__uint_as_float(v[c][k]), __uint_as_float(v[c][k + 1])), s2, acc[c * 16 + k / 2]);
    return true;
  };
  for (int t = 0; t < it.n; ++t, ++G) {
    const int st = G % kStages;
    // the tile's vectors (their copy's completion seen by this warp) and its X, Y
    if (!warp_wait(&sh.full[st], (G / kStages) & 1, p.status, kDevTimeoutConsumer, sh.abort_flag) ||
        !warp_wait(&sh.xy_full[G & 1], (G >> 1) & 1, p.status, kDevTimeoutConsumer, sh.abort_flag))
      return false;
    tc_fence_after();
    const uint32_t x0 = trow + XY_COL + (G & 1) * 128 + w * 32;
    uint32_t xv[32], yv[32];
    tmem_ld32(x0, xv);
    tmem_ld32(x0 + 64, yv);
    const uint8_t* v = sh.vecs + st * VEC_STAGE;
    const float4* col = reinterpret_cast<const float4*>(v) + w * 8;
    const float4* del = reinterpret_cast<const float4*>(v + WALK * 4) + w * 8;
    const TileScale ws = *reinterpret_cast<const TileScale*>(v + 2 * WALK * 4);
    const float c = c0 * ws.inv1, a = fs.inv2 * ws.inv2;
    // ds is formed as ds * 2^kk with |ds| 2^kk <= 2^15: e <= 2^8, |Y - delta| <= bound < 2^(ilogb + 1)
    const float bound = fs.norm * ws.norm + (KEYS ? ws.delta : fs.delta);
    int kk = 6 - ((__float_as_int(bound) >> 23) - 127);
    kk = kk > 100 ? 100 : (kk < -100 ? -100 : kk);
    const float up = pow2i(kk) * 0x1p-7f, down = pow2i(-kk);
    uint64_t dsum = 0ull;
    tmem_wait_ld();
    reg_fence(xv);
    reg_fence(yv);
    if (KEYS)
      tile_math<true, true, BIAS>(x0, xv, yv, col, del, c, a, up, row, 0.0f, dsum);
    else if (BIAS || (ps.ragged && it.t0 + t + 1 == ps.T))
      tile_math<false, true, true>(x0, xv, yv, col, del, c, a * up, 1.0f, row, row_delta * up, dsum);
    else
      tile_math<false, false, true>(x0, xv, yv, col, del, c, a * up, 1.0f, row, row_delta * up, dsum);
    tmem_wait_st();
    tc_fence_before();
    __syncwarp();
    if (lane == 0) mbar_arrive(&sh.ed_full[G & 1]);
    if (t >= 2 && !(t & 1) && !fold()) return false;
    // scales of the pair that this tile is in (both of its tiles have the same)
    fold_scale = KEYS && w == 0 ? ws.inv2 * 0x1p-7f : ws.inv1 * down;
    if (KEYS && BIAS) {
      float d0, d1;
      f2unpack(dsum, d0, d1);
      db = fmaf(d0 + d1, down, db);
    }
  }
  if (it.n > 0 && !fold()) return false;
  // ---- the held rows' gradients ----
  const bool first = !KEYS || w == 1;  // out1 (dK, dQ) or out2 (dV)
  float* dst = first ? ps.out1 : ps.out2;
  bool vec = true;
  if (ps.cuts > 1) {
    dst += (((int64_t)it.cut * p.BH + it.bh) * ps.held.Lt + it.f0 + r) * D;
  } else {
    const int b = it.bh / p.H, h = it.bh - b * p.H;
    dst += first ? b * ps.s1b + h * ps.s1h + (it.f0 + r) * ps.s1l : b * ps.s2b + h * ps.s2h + (it.f0 + r) * ps.s2l;
    vec = ps.vec_out;
  }
  if (!KEYS) dst += w * 32;
  if (it.f0 + r < ps.held.L) {
    const float s = first ? 0.125f : 1.0f;
    if (vec) {
#pragma unroll
      for (int k = 0; k < NACC; k += 4) {
        float4 o;
        f2unpack(acc[k / 2], o.x, o.y);
        f2unpack(acc[k / 2 + 1], o.z, o.w);
        *reinterpret_cast<float4*>(dst + k) = make_float4(o.x * s, o.y * s, o.z * s, o.w * s);
      }
    } else {
#pragma unroll
      for (int k = 0; k < NACC; k += 2) {
        float o0, o1;
        f2unpack(acc[k / 2], o0, o1);
        dst[k] = o0 * s;
        dst[k + 1] = o1 * s;
      }
    }
  }
  if (KEYS && BIAS && p.db) p.db[(int64_t)(it.cut * 2 + w) * p.BH * ps.held.Lt + frow] = db;
  return true;
}

// BIAS: the call has a key bias (without one, the keys' pass has no row offset and the queries' pass
// needs column offsets only for the tile past the last key).
template <bool BIAS>
__global__ void __launch_bounds__(kThreads, 1) sdpa_bwd_tc(const __grid_constant__ Maps m, const __grid_constant__ Params p) {
  extern __shared__ uint8_t smem_raw[];
  const Shared sh = carve(smem_raw);
  const uint32_t warp = warp_id();
  if (threadIdx.x == 0) {
    for (int i = 0; i < kStages; ++i) { mbar_init(&sh.full[i], 1); mbar_init(&sh.empty[i], 1); }
    for (int i = 0; i < 2; ++i) {
      mbar_init(&sh.xy_full[i], 1);
      mbar_init(&sh.ed_full[i], 8);
      mbar_init(&sh.acc_full[i], 1);
      mbar_init(&sh.acc_free[i], 8);
      mbar_init(&sh.item_full[i], 1);
      mbar_init(&sh.item_empty[i], 9);
    }
    mbar_init(sh.held_full, 8);
    mbar_init(sh.all_done, 1);
    *sh.abort_flag = 0;
    fence_barrier_init();
  }
  if (warp == 1) {
    tmem_alloc(sh.tmem_slot, TMEM_COLS);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *sh.tmem_slot;
  grid_release();
  grid_wait();
  int G = 0, P = 0;
  bool ok = true;
  if (warp < 4) {
    setmaxnreg_dec<REGS_CONTROL>();
    if (warp == 0) {
      if (elect_one()) {
        for (int i = 0; ok; ++i) {
          const int j = i == 0 ? (int)blockIdx.x : (int)gridDim.x + atomicAdd(p.next, 1);
          if (i >= 2 && !mbar_wait(&sh.item_empty[i & 1], ((i >> 1) & 1) ^ 1, p.status, kDevTimeoutProducer, sh.abort_flag)) break;
          sh.items[i & 1] = j;
          mbar_arrive(&sh.item_full[i & 1]);
          if (j >= p.items) break;
          const Item it = item_of<BIAS>(p, j);
          ok = it.keys ? load_item<true>(p, p.keys, it, &m.q1h, &m.q1l, &m.q2h, &m.q2l, sh, G)
                       : load_item<false>(p, p.queries, it, &m.k1h, &m.k1l, &m.k2h, &m.k2l, sh, G);
        }
        if (*sh.abort_flag)  // never leave the CTA while a bulk copy may still write its shared memory
          for (int g = G < kStages ? 0 : G - kStages; g < G; ++g)
            mbar_wait(&sh.full[g % kStages], (g / kStages) & 1, p.status, kDevTimeoutProducer, nullptr);
      }
    } else if (warp == 1) {
      if (elect_one()) {
        for (int i = 0; ok; ++i) {
          ok = mbar_wait(&sh.item_full[i & 1], (i >> 1) & 1, p.status, kDevTimeoutMma, sh.abort_flag);
          if (!ok) break;
          const int j = sh.items[i & 1];
          mbar_arrive(&sh.item_empty[i & 1]);
          if (j >= p.items) break;
          const Item it = item_of<BIAS>(p, j);
          ok = mbar_wait(sh.held_full, i & 1, p.status, kDevTimeoutMma, sh.abort_flag);
          if (!ok) break;
          tc_fence_after();
          ok = it.keys ? mma_item<true>(p, it.n, sh, tmem, G, P) : mma_item<false>(p, it.n, sh, tmem, G, P);
        }
        mma_commit(sh.all_done);
        mbar_wait(sh.all_done, 0, p.status, kDevTimeoutMma, nullptr);
      }
    }
  } else {
    setmaxnreg_inc<REGS_COMPUTE>();
    for (int i = 0; ok; ++i) {
      ok = warp_wait(&sh.item_full[i & 1], (i >> 1) & 1, p.status, kDevTimeoutConsumer, sh.abort_flag);
      if (!ok) break;
      const int j = sh.items[i & 1];
      __syncwarp();
      if (lane_id() == 0) mbar_arrive(&sh.item_empty[i & 1]);
      if (j >= p.items) break;
      const Item it = item_of<BIAS>(p, j);
      ok = it.keys ? compute_item<true, BIAS>(p, p.keys, it, sh, tmem, G, P)
                   : compute_item<false, BIAS>(p, p.queries, it, sh, tmem, G, P);
    }
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  if (warp == 1) {
    __syncwarp();
    tmem_dealloc(tmem, TMEM_COLS);
  }
}

// ---------------------------------------------------------------------------
// Preparation
// ---------------------------------------------------------------------------

// The key bias of the softmax: relative to the row's largest, clamped to -1e6 (2^-1e6 is zero next to
// the largest), -inf kept.
__device__ __forceinline__ float relative_bias(float v, float mx) {
  const float d = v - mx;  // NaN for NaN and for +inf
  return v == -INFINITY ? v : (d < -1.0e6f ? -1.0e6f : d);
}

// A row's largest bias and whether the scores count beside it (0 beyond 2^60 in magnitude).
__device__ __forceinline__ float2 bias_head(float mx) {
  return make_float2(mx, mx > -INFINITY && fabsf(mx) > 0x1p60f ? 0.0f : 1.0f);
}

// Which bias row (b, h) reads: [bias_b, bias_h, Lk] with 1 for a shared dimension.
struct Bias {
  const float* p;
  int b, h, L;
  __device__ __forceinline__ const float* row(int ib, int ih) const {
    return p + ((int64_t)(b == 1 ? 0 : ib) * h + (h == 1 ? 0 : ih)) * L;
  }
};

// The first 128-key tile of a bias row with a key and the one past the last; (0, 0) without any.  A block
// of 256 threads; lo, hi: of the keys that the thread has seen.
__device__ __forceinline__ int2 tile_range(int lo, int hi, int2* sm) {
  lo = __reduce_min_sync(0xffffffffu, lo);
  hi = __reduce_max_sync(0xffffffffu, hi);
  if ((threadIdx.x & 31) == 0) sm[threadIdx.x >> 5] = make_int2(lo, hi);
  __syncthreads();
#pragma unroll
  for (int k = 0; k < 8; ++k) {
    lo = min(lo, sm[k].x);
    hi = max(hi, sm[k].y);
  }
  return hi < 0 ? make_int2(0, 0) : make_int2(lo / HELD, hi / HELD + 1);
}

// One block per (b, h): the row's head, behind the statistics for the backward pass, and (out not null) the
// relative bias and the range of tiles with a key.
__global__ void __launch_bounds__(256) bias_rows_k(Bias bias, int H, float* __restrict__ out, int2* __restrict__ tiles,
                                                   float2* head, int64_t head_stride) {
  __shared__ float sm[8];
  __shared__ int2 sm_range[8];
  grid_release();
  const int bh = blockIdx.x, b = bh / H, h = bh - b * H;
  const float* src = bias.row(b, h);
  float mx = -INFINITY;
  int lo = 0x7fffffff, hi = -1;
#pragma unroll 8
  for (int j = threadIdx.x; j < bias.L; j += 256) {
    const float v = src[j];
    mx = fmaxf(mx, v);
    if (v != -INFINITY) {
      lo = min(lo, j);
      hi = j;
    }
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, o));
  if ((threadIdx.x & 31) == 0) sm[threadIdx.x >> 5] = mx;
  const int2 range = tile_range(lo, hi, sm_range);  // also orders sm
#pragma unroll
  for (int k = 0; k < 8; ++k) mx = fmaxf(mx, sm[k]);
  if (threadIdx.x == 0) head[bh * head_stride] = bias_head(mx);
  if (!out) return;
  if (threadIdx.x == 0) tiles[bh] = range;
  for (int j = threadIdx.x; j < bias.L; j += 256) out[(int64_t)bh * bias.L + j] = relative_bias(src[j], mx);
}

struct Rows {
  const float* p;
  int64_t b, h, l;
  __device__ __forceinline__ const float* at(int ib, int ih, int64_t il) const { return p + ib * b + ih * h + il * l; }
};

// Four lanes share a 64-dimensional row: lane q has columns col16(q, 0..15), four runs of four, 16
// columns apart, so that one access of the four lanes covers 64 bytes side by side.
__device__ __forceinline__ int col16(int q, int e) { return (e >> 2) * 16 + q * 4 + (e & 3); }

__device__ __forceinline__ void load16(const float* row, int q, bool vec, float (&v)[16]) {
  if (vec) {
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      const float4 f = *reinterpret_cast<const float4*>(row + col16(q, 4 * k));
      v[4 * k] = f.x; v[4 * k + 1] = f.y; v[4 * k + 2] = f.z; v[4 * k + 3] = f.w;
    }
  } else {
#pragma unroll
    for (int k = 0; k < 16; ++k) v[k] = row[col16(q, k)];
  }
}

// largest finite magnitude: a scale is shared by the rows of a tile, and one that is not finite is
// none of the others' business
__device__ __forceinline__ float absmax16(const float (&v)[16]) {
  float m = 0.0f;
#pragma unroll
  for (int k = 0; k < 16; ++k) {
    const float a = fabsf(v[k]);
    m = a <= 3.402823466e38f ? fmaxf(m, a) : m;
  }
  return m;
}

// hi / lo planes of four consecutive values times a power of two
__device__ __forceinline__ void store_split4(const float* v, float up, __half* hi, __half* lo) {
  __align__(8) __half2 h[2], l[2];
#pragma unroll
  for (int k = 0; k < 2; ++k) {
    const float a = v[2 * k] * up, b = v[2 * k + 1] * up;
    h[k] = __floats2half2_rn(a, b);
    const float2 f = __half22float2(h[k]);
    l[k] = __floats2half2_rn(a - f.x, b - f.y);
  }
  *reinterpret_cast<uint2*>(hi) = *reinterpret_cast<const uint2*>(h);
  *reinterpret_cast<uint2*>(lo) = *reinterpret_cast<const uint2*>(l);
}

// ... of a lane's 16 columns of a row
__device__ __forceinline__ void store_split16(const float (&v)[16], int q, float up, __half* hi, __half* lo) {
#pragma unroll
  for (int k = 0; k < 4; ++k) store_split4(v + 4 * k, up, hi + col16(q, 4 * k), lo + col16(q, 4 * k));
}

// largest of four values over a block of 256 threads
__device__ __forceinline__ float4 block_max4(float4 v, float4* sm) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    v.x = fmaxf(v.x, __shfl_xor_sync(0xffffffffu, v.x, o));
    v.y = fmaxf(v.y, __shfl_xor_sync(0xffffffffu, v.y, o));
    v.z = fmaxf(v.z, __shfl_xor_sync(0xffffffffu, v.z, o));
    v.w = fmaxf(v.w, __shfl_xor_sync(0xffffffffu, v.w, o));
  }
  if ((threadIdx.x & 31) == 0) sm[threadIdx.x >> 5] = v;
  __syncthreads();
  v = sm[0];
#pragma unroll
  for (int k = 1; k < 8; ++k) {
    const float4 u = sm[k];
    v = make_float4(fmaxf(v.x, u.x), fmaxf(v.y, u.y), fmaxf(v.z, u.z), fmaxf(v.w, u.w));
  }
  return v;
}

// The planes, vectors and scales of both sides of the backward pass.  One block per (b h, 128-row
// tile), the keys' tiles first; a thread has a quarter of rows j and j + 64.  Keys: K and V, rows with
// a bias of -inf as zeros, the relative bias in log2 units (-inf past the end).  Queries: Q and
// g = dO / l, 7 - m, -delta; the first of them also finds the head's range of tiles with a key.
__global__ void __launch_bounds__(256) bwd_split_k(Rows q, Rows dout, Rows out, Rows k, Rows v, Bias bias,
                                                   const float2* __restrict__ stats, int64_t stats_ld, int H, int vec,
                                                   Side qs, Side ks, int* next, int2* __restrict__ tiles) {
  __shared__ float4 sm[8];
  __shared__ int2 sm_range[8];
  grid_release();
  const int bh = blockIdx.x, b = bh / H, h = bh - b * H, lq = threadIdx.x & 3;
  const int key_tiles = ks.Lt / HELD;
  if (bh == 0 && blockIdx.y == 0 && threadIdx.x == 0) *next = 0;  // the main kernel's item counter
  const bool keys = (int)blockIdx.y < key_tiles;
  if (bias.p && (int)blockIdx.y == key_tiles) {
    const float* src = bias.row(b, h);
    int lo = 0x7fffffff, hi = -1;
#pragma unroll 8
    for (int j = threadIdx.x; j < ks.L; j += 256) {
      if (src[j] != -INFINITY) {
        lo = min(lo, j);
        hi = j;
      }
    }
    const int2 range = tile_range(lo, hi, sm_range);
    if (threadIdx.x == 0) tiles[bh] = range;
  }
  const Side& s = keys ? ks : qs;
  const int row0 = (keys ? blockIdx.y : blockIdx.y - key_tiles) * HELD + (threadIdx.x >> 2);
  float x[2][16], y[2][16], sq[2] = {0.0f, 0.0f}, delta[2] = {0.0f, 0.0f}, col[2] = {-INFINITY, -INFINITY};
  if (keys) {
    const float mx = bias.p ? stats[bh * stats_ld + stats_ld - 1].x : 0.0f;
#pragma unroll
    for (int u = 0; u < 2; ++u) {
      const int row = row0 + 64 * u;
#pragma unroll
      for (int e = 0; e < 16; ++e) x[u][e] = y[u][e] = 0.0f;
      if (row < s.L) col[u] = bias.p ? relative_bias(bias.row(b, h)[row], mx) * LOG2E : 0.0f;
      if (col[u] != -INFINITY) {
        load16(k.at(b, h, row), lq, vec, x[u]);
        load16(v.at(b, h, row), lq, vec, y[u]);
      }
    }
  } else {
#pragma unroll
    for (int u = 0; u < 2; ++u) {
      const int row = row0 + 64 * u;
      float ov[16];
      float2 ml = make_float2(0.0f, 0.0f);
#pragma unroll
      for (int e = 0; e < 16; ++e) x[u][e] = y[u][e] = ov[e] = 0.0f;
      if (row < s.L) {
        load16(q.at(b, h, row), lq, vec, x[u]);
        load16(dout.at(b, h, row), lq, vec, y[u]);
        load16(out.at(b, h, row), lq, vec, ov);
        ml = stats[bh * stats_ld + row];
      }
      const bool any = ml.y != 0.0f;  // a row without a key gives nothing, whatever dO holds
      const float inv = any ? 1.0f / ml.y : 0.0f;
      if (any) col[u] = E_LIFT - ml.x;
#pragma unroll
      for (int e = 0; e < 16; ++e) {
        y[u][e] = any ? y[u][e] * inv : 0.0f;
        delta[u] = fmaf(y[u][e], ov[e], delta[u]);
      }
    }
  }
  const float top[2] = {absmax16(y[0]), absmax16(y[1])};
  float4 mx = make_float4(fmaxf(absmax16(x[0]), absmax16(x[1])), fmaxf(top[0], top[1]), 0.0f, 0.0f);
#pragma unroll
  for (int u = 0; u < 2; ++u) {
    float all = top[u];
#pragma unroll
    for (int e = 0; e < 16; ++e) sq[u] = fmaf(y[u][e], y[u][e], sq[u]);
#pragma unroll
    for (int i = 1; i < 4; i <<= 1) {
      sq[u] += __shfl_xor_sync(0xffffffffu, sq[u], i);
      delta[u] += __shfl_xor_sync(0xffffffffu, delta[u], i);
      all = fmaxf(all, __shfl_xor_sync(0xffffffffu, all, i));
    }
    // the row's norm, or sqrt(64) times its largest element where the squares leave the type's range
    mx.z = fmaxf(mx.z, sq[u] >= 0x1p-100f && sq[u] <= 0x1p120f ? sqrtf(sq[u]) : 8.0f * all);
    if (fabsf(delta[u]) <= 3.402823466e38f) mx.w = fmaxf(mx.w, fabsf(delta[u]));
  }
  mx = block_max4(mx, sm);
  const int s1 = scale_shift(mx.x), s2 = scale_shift(mx.y);
  const int64_t prow0 = (int64_t)bh * s.Lt + row0;
  if (threadIdx.x == 0)  // the norms a little up: they bound what is formed from rounded values
    s.scale[prow0 / HELD] = {pow2i(-s1), pow2i(-s2), mx.z * 1.0001f, mx.w * 1.0001f};
#pragma unroll
  for (int u = 0; u < 2; ++u) {
    const int64_t prow = prow0 + 64 * u;
    if ((threadIdx.x & 3) == 0) {
      s.col[prow] = col[u];
      if (!keys) s.delta[prow] = -delta[u];
    }
    store_split16(x[u], lq, pow2i(s1), s.hi1 + prow * D, s.lo1 + prow * D);
    store_split16(y[u], lq, pow2i(s2), s.hi2 + prow * D, s.lo2 + prow * D);
  }
}

// The forward kernel's planes (sdpa_planes.h) from strided tensors.  One block per (b h, 128-row tile),
// the keys' tiles first, threads as above.  Keys: one scale each for K and V of a tile, V through
// shared memory to its transposed planes.  Queries: one scale per row.
constexpr int KT = 128;
__global__ void __launch_bounds__(256) fwd_split_k(Rows q, Rows k, Rows v, Bias bias, float2* head, int64_t head_stride,
                                                   int H, int Lq, int Lk, int vec, SplitPlanesSdpa sp) {
  __shared__ float vt[KT][D + 1];
  __shared__ float4 sm[8];
  grid_release();
  grid_wait();
  const int bh = blockIdx.x, b = bh / H, h = bh - b * H, lq = threadIdx.x & 3;
  float x[2][16];
  if ((int)blockIdx.y >= sp.T) {
    const int row0 = (blockIdx.y - sp.T) * KT + (threadIdx.x >> 2);
    float weight = 1.0f;
    if (bias.p) weight = head[bh * head_stride].y;
    else if (row0 == 0 && threadIdx.x == 0) head[bh * head_stride] = make_float2(0.0f, 1.0f);
#pragma unroll
    for (int u = 0; u < 2; ++u) {
#pragma unroll
      for (int e = 0; e < 16; ++e) x[u][e] = 0.0f;
      if (row0 + 64 * u < Lq) load16(q.at(b, h, row0 + 64 * u), lq, vec, x[u]);
    }
#pragma unroll
    for (int u = 0; u < 2; ++u) {
      float mx = absmax16(x[u]);
#pragma unroll
      for (int i = 1; i < 4; i <<= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, i));
      if (row0 + 64 * u >= Lq) continue;
      const int s = scale_shift(mx);
      const int64_t prow = (int64_t)bh * Lq + row0 + 64 * u;
      store_split16(x[u], lq, pow2i(s), sp.qhi + prow * D, sp.qlo + prow * D);
      if ((threadIdx.x & 3) == 0) sp.qinv[prow] = pow2i(-s) * weight;
    }
    return;
  }
  const int tile = blockIdx.y, row0 = tile * KT + (threadIdx.x >> 2);
  float kmx = 0.0f, vmx = 0.0f;
#pragma unroll
  for (int u = 0; u < 2; ++u) {
    const int j = u * 64 + (threadIdx.x >> 2), row = row0 + u * 64;
    float y[16];
#pragma unroll
    for (int e = 0; e < 16; ++e) x[u][e] = y[e] = 0.0f;
    if (row < Lk && !(bias.p && bias.row(b, h)[row] == -INFINITY)) {
      load16(k.at(b, h, row), lq, vec, x[u]);
      load16(v.at(b, h, row), lq, vec, y);
    }
#pragma unroll
    for (int e = 0; e < 16; ++e) vt[j][col16(lq, e)] = y[e];
    kmx = fmaxf(kmx, absmax16(x[u]));
    vmx = fmaxf(vmx, absmax16(y));
  }
  const float4 mx = block_max4(make_float4(kmx, vmx, 0.0f, 0.0f), sm);  // also orders vt
  // within the +-60 that the forward kernel's exponent arithmetic on V's scales expects
  const int sk = max(-60, min(60, scale_shift(mx.x)));
  // the forward kernel lifts probabilities by a tile's V scale relative to the head's largest: a tile
  // of zeros (keys that do not exist) takes the smallest, so that it leaves the others' lift alone
  const int sv = mx.y == 0.0f ? 60 : max(-60, min(60, scale_shift(mx.y)));
#pragma unroll
  for (int u = 0; u < 2; ++u) {
    const int64_t prow = (int64_t)bh * sp.Lkt + row0 + u * 64;
    store_split16(x[u], lq, pow2i(sk), sp.khi + prow * D, sp.klo + prow * D);
  }
  // a warp per row of V^T: two keys per lane, 128 bytes side by side
  for (int d = threadIdx.x >> 5; d < D; d += 8) {
#pragma unroll
    for (int u = 0; u < 2; ++u) {
      const int j = 64 * u + 2 * (threadIdx.x & 31);
      const float a0 = vt[j][d] * pow2i(sv), a1 = vt[j + 1][d] * pow2i(sv);
      const __half2 h = __floats2half2_rn(a0, a1);
      const float2 f = __half22float2(h);
      const int64_t off = ((int64_t)bh * D + d) * sp.Lkt + tile * KT + j;
      *reinterpret_cast<__half2*>(sp.vhi + off) = h;
      *reinterpret_cast<__half2*>(sp.vlo + off) = __floats2half2_rn(a0 - f.x, a1 - f.y);
    }
  }
  if (threadIdx.x == 0) {
    sp.kinv[(int64_t)bh * sp.T + tile] = pow2i(-sk);
    sp.vinv[(int64_t)bh * sp.T + tile] = pow2i(-sv);
  }
}

// Gradients of passes whose walks were cut: a tensor's partial sums [cuts, BH, Lt, 64] added over the shares.
// blockIdx.y is the tensor; a thread has 4 of a row's 64 elements and every W-th share (W = 8 where there
// are more than that: few rows, else 1), whose sums are then added in order.
struct Join {
  const float* part;
  float* out;
  int64_t sb, sh, sl;  // element strides of out
  int cuts, L, Lt;
  __host__ __device__ int threads() const { return cuts > 8 ? 8 : 1; }  // per 4 elements
};
struct Joins {
  Join t[3];
  int H, BH, vec_out;
};
__global__ void __launch_bounds__(256) join_k(const Joins a) {
  __shared__ float4 sm[256];
  grid_release();
  grid_wait();
  const Join& t = a.t[blockIdx.y];
  const int W = t.threads();
  const int lane = threadIdx.x % 16, y = threadIdx.x / 16 % W;
  const int64_t i = (int64_t)blockIdx.x * (16 / W) + threadIdx.x / (16 * W);
  const bool here = i < (int64_t)a.BH * t.L;
  const int64_t row = i % t.L;
  const int bh = (int)(i / t.L), b = bh / a.H, h = bh - b * a.H;
  const int64_t step = (int64_t)a.BH * t.Lt * (D / 4);
  float4 s = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
  if (here) {
    const float4* src = reinterpret_cast<const float4*>(t.part) + ((int64_t)bh * t.Lt + row) * (D / 4) + lane;
#pragma unroll 4
    for (int c = y; c < t.cuts; c += W) {
      const float4 v = src[c * step];
      s.x += v.x; s.y += v.y; s.z += v.z; s.w += v.w;
    }
  }
  if (W > 1) {
    sm[threadIdx.x] = s;
    __syncthreads();
    if (y != 0) return;
#pragma unroll
    for (int k = 1; k < 8; ++k) {
      const float4 v = sm[threadIdx.x + 16 * k];
      s.x += v.x; s.y += v.y; s.z += v.z; s.w += v.w;
    }
  }
  if (!here) return;
  float* dst = t.out + b * t.sb + h * t.sh + row * t.sl + lane * 4;
  if (a.vec_out) {
    *reinterpret_cast<float4*>(dst) = s;
  } else {
    dst[0] = s.x; dst[1] = s.y; dst[2] = s.z; dst[3] = s.w;
  }
}

// Shares of the keys joined: partial outputs [cuts, BH or B, Lq, ...] as normalised by their own sums,
// with their statistics.  W warps per row (8 where there are more shares than that, else 1): warp w adds
// shares w, w + W, ..., then the warps' sums are added in order.  last: the statistics' last row has
// no bias kernel to set it.
template <int W>
__global__ void __launch_bounds__(256) attn_join_k(const float* __restrict__ o, const float2* __restrict__ st, int cuts,
                                                   int64_t cut_o, int64_t cut_st, int64_t st_ld, int by_head, int64_t n,
                                                   int H, int Lq, int last, float* __restrict__ out,
                                                   float2* __restrict__ stats) {
  __shared__ float sm_l[8];
  __shared__ float2 sm_v[8][32];
  grid_release();
  grid_wait();
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int64_t i = W == 1 ? (int64_t)blockIdx.x * 8 + warp : blockIdx.x;
  if (i >= n) return;
  const int bh = (int)(i / Lq), row = (int)(i - (int64_t)bh * Lq), b = bh / H, h = bh - b * H;
  const int64_t dst = (((int64_t)b * Lq + row) * H + h) * D + lane * 2;
  const float* src = o + (by_head ? i * D + lane * 2 : dst);
  const float2* s = st + bh * st_ld + row;
  float m = -INFINITY;
  for (int c = lane; c < cuts; c += 32) m = fmaxf(m, s[c * cut_st].x);
#pragma unroll
  for (int k = 16; k > 0; k >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, k));
  float l = 0.0f;
  float2 v = make_float2(0.0f, 0.0f);
#pragma unroll 8
  for (int c = W == 1 ? 0 : warp; c < cuts; c += W) {
    const float2 ml = s[c * cut_st];
    const float w = ml.y * (ml.x == m ? 1.0f : ex2(ml.x - m));
    const float2 x = *reinterpret_cast<const float2*>(src + c * cut_o);
    l += w;
    v.x = fmaf(w, x.x, v.x);
    v.y = fmaf(w, x.y, v.y);
  }
  if (W > 1) {
    sm_v[warp][lane] = v;
    if (lane == 0) sm_l[warp] = l;
    __syncthreads();
    if (warp != 0) return;
#pragma unroll
    for (int w = 1; w < 8; ++w) {
      l += sm_l[w];
      v.x += sm_v[w][lane].x;
      v.y += sm_v[w][lane].y;
    }
  }
  const float inv = l == 0.0f ? 0.0f : 1.0f / l;
  *reinterpret_cast<float2*>(out + dst) = make_float2(v.x * inv, v.y * inv);
  if (lane == 0) stats[(int64_t)bh * (Lq + 1) + row] = make_float2(m, l);
  if (last && row == 0 && lane == 1) stats[(int64_t)bh * (Lq + 1) + Lq] = make_float2(0.0f, 1.0f);
}

// db [bias_b, bias_h, Lk]: part [parts, B, H, Lt] added over the parts and the batch entries and heads
// that share a row.  32 columns per block, eight threads each: thread y adds terms y, y + 8, ..., then the
// eight sums are added in order.
__global__ void __launch_bounds__(256) bias_grad_k(const float* __restrict__ part, int parts, int B, int H, int bias_b,
                                                   int bias_h, int Lk, int Lt, float* __restrict__ db) {
  __shared__ float sm[8][32];
  grid_release();
  grid_wait();
  const int j = blockIdx.x * 32 + threadIdx.x, y = threadIdx.y, row = blockIdx.y;
  const int rb = row / bias_h, rh = row - rb * bias_h;
  const int b0 = bias_b == 1 ? 0 : rb, nb = bias_b == 1 ? B : 1;
  const int h0 = bias_h == 1 ? 0 : rh, nh = bias_h == 1 ? H : 1;
  float s = 0.0f;
  if (j < Lk) {
    const float* p = part + ((int64_t)b0 * H + h0) * Lt + j;
    const int n = parts * nb * nh;
#pragma unroll 4
    for (int i = y; i < n; i += 8) {
      const int h = i % nh, gb = i / nh, b = gb % nb, g = gb / nb;
      s += p[(((int64_t)g * B + b) * H + h) * Lt];
    }
  }
  sm[y][threadIdx.x] = s;
  __syncthreads();
  if (y != 0 || j >= Lk) return;
#pragma unroll
  for (int k = 1; k < 8; ++k) s += sm[k][threadIdx.x];
  db[(int64_t)row * Lk + j] = s;
}

// ---------------------------------------------------------------------------
// Host
// ---------------------------------------------------------------------------
static size_t al256(size_t x) { return (x + 255) & ~static_cast<size_t>(255); }

// Carves one side out of the workspace (base null: only counts) and returns its bytes.
static size_t side_layout(uint8_t* base, int64_t BH, int L, bool delta, Side& s) {
  s.L = L;
  s.Lt = (L + HELD - 1) / HELD * HELD;
  const size_t rows = (size_t)BH * s.Lt;
  size_t at = 0;
  auto take = [&](size_t bytes) {
    uint8_t* p = base ? base + at : nullptr;
    at += al256(bytes);
    return p;
  };
  s.hi1 = reinterpret_cast<__half*>(take(rows * D * 2));
  s.lo1 = reinterpret_cast<__half*>(take(rows * D * 2));
  s.hi2 = reinterpret_cast<__half*>(take(rows * D * 2));
  s.lo2 = reinterpret_cast<__half*>(take(rows * D * 2));
  s.col = reinterpret_cast<float*>(take(rows * 4));
  s.delta = reinterpret_cast<float*>(take(delta ? rows * 4 : 0));
  s.scale = reinterpret_cast<TileScale*>(take(rows / HELD * sizeof(TileScale)));
  return at;
}

static bool plane_map(CUtensorMap* m, const __half* base, int64_t BH, int Lt) {
  const uint64_t dims[3] = {D, (uint64_t)Lt, (uint64_t)BH};
  const uint64_t strides[2] = {D * 2, (uint64_t)Lt * D * 2};
  const uint32_t box[3] = {D, WALK, 1};
  return encode_tmap(m, CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 3, const_cast<__half*>(base), dims, strides, box,
                     CU_TENSOR_MAP_SWIZZLE_128B);
}

// Shared-memory opt-in and the register check of the split budgets, once per device: with fewer
// registers compiled in, setmaxnreg.inc would wait for ever.
template <bool BIAS>
static int ensure_kernel() {
  static std::atomic<uint64_t> done{0};
  int dev = 0;
  cudaGetDevice(&dev);
  if (done.load(std::memory_order_acquire) >> (dev & 63) & 1) return kOk;
  cudaFuncAttributes fa{};
  if (cudaFuncGetAttributes(&fa, sdpa_bwd_tc<BIAS>) != cudaSuccess || fa.numRegs < (int)REGS_LAUNCH) {
    set_last_error("sdpa_bwd_tc was compiled with fewer registers than its warpgroup budget needs");
    return kLaunchFailed;
  }
  if (cudaFuncSetAttribute(sdpa_bwd_tc<BIAS>, cudaFuncAttributeMaxDynamicSharedMemorySize, SMEM_BYTES) != cudaSuccess)
    return launch_status();
  done.fetch_or(1ull << (dev & 63), std::memory_order_acq_rel);
  return kOk;
}

// When the last of the SMs is done that take n1 items of c1 and then n2 items of c2 <= c1 one by one.
static int64_t makespan(int64_t n1, int64_t c1, int64_t n2, int64_t c2, int64_t sms) {
  // two groups of SMs, those with one item of the first kind more than the others
  int64_t more = n1 % sms, less = sms - more, low = n1 / sms * c1, high = low + c1, end = more ? high : low;
  while (n2 > 0) {
    const bool to_low = !more || low <= high;
    int64_t &load = to_low ? low : high, size = to_low ? less : more;
    load += c2;
    n2 -= size;
    if (load > end) end = load;
  }
  return end;
}

// Into how many shares the two passes' walks are cut (few held tiles: their items would leave SMs idle or
// end at very different times), by the time until the last SM is done.  Costs in products of a 64-row tile,
// some 0.38 us (keys' pass 4 per tile, queries' pass 3), an item's start as much as 4 tiles; a cut costs the
// join of its partial sums: 8, and 1 per MB of them.  (2000 x 2000, 4 heads, uncut by this rule: 57 us; its
// 128 + 64 items of a rule that cuts down to an SM's fair share 61 and 18 for the joins.)
static void cut_walks(Pass& keys, Pass& queries, int64_t BH) {
  static const int kCuts[] = {1, 2, 3, 4, 6, 8, 12, 16, 24, 32, 48, 64};
  const int64_t sms = sm_count();
  Pass* s[2] = {&keys, &queries};
  for (Pass* q : s) {
    q->cuts = 1;
    q->span = q->T;
  }
  if (BH * (keys.Ft + queries.Ft) > 8 * sms) return;
  int64_t best = -1;
  int span[2] = {keys.T, queries.T};
  for (int a : kCuts) {
    const int sk = ((keys.T + a - 1) / a + 1) / 2 * 2;
    if (a > 1 && sk < 4) break;
    const int64_t nk = BH * keys.Ft * (a == 1 ? 1 : (keys.T + sk - 1) / sk), ck = ((a == 1 ? keys.T : sk) + 4) * 4;
    for (int b : kCuts) {
      const int sq = ((queries.T + b - 1) / b + 1) / 2 * 2;
      if (b > 1 && sq < 4) break;
      const int64_t nq = BH * queries.Ft * (b == 1 ? 1 : (queries.T + sq - 1) / sq), cq = ((b == 1 ? queries.T : sq) + 4) * 3;
      int64_t t = ck >= cq ? makespan(nk, ck, nq, cq, sms) : makespan(nq, cq, nk, ck, sms);
      if (a > 1 || b > 1) t += 8 + ((a > 1 ? 2 * nk : 0) + (b > 1 ? nq : 0)) * HELD * D * 4 / (1 << 20);
      if (best < 0 || t < best) {
        best = t;
        span[0] = a == 1 ? keys.T : sk;
        span[1] = b == 1 ? queries.T : sq;
      }
    }
  }
  for (int i = 0; i < 2; ++i) {
    s[i]->span = span[i];
    s[i]->cuts = (s[i]->T + span[i] - 1) / span[i];
  }
}

// sizes a launch can hold: items * tiles counted in ints, grid rows in 16 bits
static int check_sizes(int B, int H, int Lq, int Lk, const void* bias, int bias_b, int bias_h) {
  if (B <= 0 || H <= 0 || Lq <= 0 || Lk <= 0) return kBadDims;
  const int64_t BH = (int64_t)B * H;
  if (BH > 65535 || Lq > 64 * 65535 || Lk > 64 * 65535) return kBadDims;
  const int64_t tiles = (int64_t)((Lq + 127) / 128) * ((Lk + 127) / 128) * 2;
  if (BH * tiles > 2147483647) return kBadDims;
  if (bias && ((bias_b != 1 && bias_b != B) || (bias_h != 1 && bias_h != H))) return kBadRange;
  return kOk;
}

static bool misaligned(std::initializer_list<const void*> ps, uintptr_t low) {
  for (const void* p : ps)
    if (reinterpret_cast<uintptr_t>(p) & low) return true;
  return false;
}

// whether every row of the tensors starts on a 16-byte boundary
static bool rows16(std::initializer_list<const void*> ps, const int64_t* strides, int n) {
  if (misaligned(ps, 15)) return false;
  for (int i = 0; i < 3 * n; ++i)
    if (strides[i] % 4) return false;
  return true;
}

#include "sdpa_few.cuh"

static Rows rows_of(const void* p, const int64_t* s) { return {static_cast<const float*>(p), s[0], s[1], s[2]}; }

}  // namespace sdpab
}  // namespace tsb

extern "C" {

int triposplat_b200_attention_forward(const float* q, const float* k, const float* v, const int64_t* strides,
                                      const float* key_bias, int bias_batches, int bias_heads, float* out_blhd,
                                      float* stats, int B, int H, int Lq, int Lk) {
  using namespace tsb;
  using namespace tsb::sdpab;
  if (!q || !k || !v || !strides || !out_blhd || !stats) return kNullPointer;
  int st = check_sizes(B, H, Lq, Lk, key_bias, bias_batches, bias_heads);
  if (st != kOk) return st;
  if (misaligned({q, k, v, key_bias}, 3) || misaligned({out_blhd}, 15) || misaligned({stats}, 7)) return kBadAlignment;
  st = entry_check();
  if (st != kOk) return st;
  for (const void* p : {q, k, v, key_bias, static_cast<const float*>(out_blhd), static_cast<const float*>(stats)})
    if (p && !is_device_pointer(p)) return kNotDevicePointer;
  cudaStream_t stream = current_stream();
  const int64_t BH = (int64_t)B * H;
  float2* rows = reinterpret_cast<float2*>(stats);
  const Bias bias{key_bias, bias_batches, bias_heads, Lk};
  const int vec = rows16({q, k, v}, strides, 3);
  auto bias_rows = [&](float* relative, int2* tiles) {
    LaunchScope scope(kKSdpaSplit, stream);
    bias_rows_k<<<(unsigned)BH, 256, 0, stream>>>(bias, H, relative, tiles, rows + Lq, Lq + 1);
  };
  auto join = [&](const float* o, const float2* part, int cuts, int64_t cut_o, int64_t cut_st, int64_t st_ld, int by_head,
                  int last) {
    LaunchScope scope(kKSdpaSplit, stream);
    if (cuts > 8)
      launch_chained(attn_join_k<8>, dim3((unsigned)(BH * Lq)), dim3(256), 0, stream, o, part, cuts, cut_o, cut_st, st_ld, by_head,
                     BH * Lq, H, Lq, last, out_blhd, rows);
    else
      launch_chained(attn_join_k<1>, dim3((unsigned)((BH * Lq + 7) / 8)), dim3(256), 0, stream, o, part, cuts, cut_o, cut_st, st_ld,
                     by_head, BH * Lq, H, Lq, last, out_blhd, rows);
  };
  FewArgs a{};
  a.H = H; a.BH = (int)BH; a.Lq = Lq; a.Lk = Lk;
  if (few(a)) {
    a.q = rows_of(q, strides); a.k = rows_of(k, strides + 3); a.v = rows_of(v, strides + 6);
    a.bias = bias;
    a.head = rows + Lq; a.head_stride = Lq + 1;
    a.o = out_blhd; a.stats_out = rows;
    a.vec = vec;
    if (a.shares > 1) {
      const size_t obytes = al256((size_t)a.shares * BH * Lq * D * 4);
      uint8_t* ws = static_cast<uint8_t*>(workspace(obytes + (size_t)a.shares * BH * Lq * 8, stream));
      if (!ws) return kWorkspace;
      a.o = reinterpret_cast<float*>(ws);
      a.stats_out = reinterpret_cast<float2*>(ws + obytes);
    }
    const bool apart = key_bias && Lk > kFewBias;
    if (apart) bias_rows(nullptr, nullptr);
    else if (key_bias) a.head_out = rows + Lq;
    few_fwd(a, apart, stream);
    if (a.shares > 1) join(a.o, a.stats_out, a.shares, BH * Lq * D, BH * Lq, Lq, 1, key_bias == nullptr);
    return launch_status();
  }
  // few work items: the keys in shares of two tiles or more, so that most SMs have one
  const int Qt = (Lq + KT - 1) / KT, T = (Lk + KT - 1) / KT;
  const int64_t fit = sm_count() / (Qt * BH);
  const int cuts = fit < 2 || T < 4 ? 1 : (int)(fit < T / 2 ? fit : T / 2);
  const size_t row_bytes = key_bias ? al256((size_t)BH * Lk * 4) : 0;
  const size_t bias_bytes = key_bias ? row_bytes + al256((size_t)BH * sizeof(int2)) : 0;
  const size_t part_bytes = cuts > 1 ? al256((size_t)cuts * BH * Lq * D * 4) : 0;
  SplitPlanesSdpa sp;
  void* behind = nullptr;
  st = sdpa_planes_extra(BH, Lq, Lk, bias_bytes + part_bytes + (cuts > 1 ? (size_t)cuts * BH * Lq * 8 : 0), stream, sp,
                         &behind);
  if (st != kOk) return st;
  float* relative = key_bias ? static_cast<float*>(behind) : nullptr;
  int2* tiles = key_bias ? reinterpret_cast<int2*>(static_cast<uint8_t*>(behind) + row_bytes) : nullptr;
  float* part = reinterpret_cast<float*>(static_cast<uint8_t*>(behind) + bias_bytes);
  float2* part_st = reinterpret_cast<float2*>(static_cast<uint8_t*>(behind) + bias_bytes + part_bytes);
  if (key_bias) bias_rows(relative, tiles);
  {
    LaunchScope scope(kKSdpaSplit, stream);
    const dim3 grid((unsigned)BH, sp.T + Qt);
    const Rows rq = rows_of(q, strides), rk = rows_of(k, strides + 3), rv = rows_of(v, strides + 6);
    if (key_bias) launch_chained(fwd_split_k, grid, dim3(256), 0, stream, rq, rk, rv, bias, rows + Lq, Lq + 1, H, Lq, Lk, vec, sp);
    else fwd_split_k<<<grid, 256, 0, stream>>>(rq, rk, rv, bias, rows + Lq, Lq + 1, H, Lq, Lk, vec, sp);
  }
  if ((st = launch_status()) != kOk) return st;
  if (cuts == 1)
    return sdpa_attend_stats(sp, relative, Lk, tiles, out_blhd, rows, Lq + 1, BH, H, Lq, Lk, 1, 0, 0, stream);
  st = sdpa_attend_stats(sp, relative, Lk, tiles, part, part_st, Lq, BH, H, Lq, Lk, cuts, BH * Lq * D, BH * Lq, stream);
  if (st != kOk) return st;
  join(part, part_st, cuts, BH * Lq * D, BH * Lq, Lq, 0, 0);
  return launch_status();
}

int triposplat_b200_attention_backward(const float* dout, const float* q, const float* k, const float* v,
                                       const float* out, const float* stats, const int64_t* strides,
                                       const float* key_bias, int bias_batches, int bias_heads, float* dq, float* dk,
                                       float* dv, float* dbias, int B, int H, int Lq, int Lk) {
  using namespace tsb;
  using namespace tsb::sdpab;
  if (!dout || !q || !k || !v || !out || !stats || !strides || !dq || !dk || !dv || (dbias && !key_bias))
    return kNullPointer;
  int st = check_sizes(B, H, Lq, Lk, key_bias, bias_batches, bias_heads);
  if (st != kOk) return st;
  if (misaligned({dout, q, k, v, out, key_bias, dq, dk, dv, dbias}, 3) || misaligned({stats}, 7)) return kBadAlignment;
  st = entry_check();
  if (st != kOk) return st;
  for (const float* p : {dout, q, k, v, out, stats, key_bias, static_cast<const float*>(dq), static_cast<const float*>(dk),
                         static_cast<const float*>(dv), static_cast<const float*>(dbias)})
    if (p && !is_device_pointer(p)) return kNotDevicePointer;
  cudaStream_t stream = current_stream();
  const int64_t BH = (int64_t)B * H;
  const int64_t* go = strides + 15;  // dq, dk, dv
  const int vec = rows16({dout, q, k, v, out}, strides, 5), vec_out = rows16({dq, dk, dv}, go, 3);
  const float2* rows = reinterpret_cast<const float2*>(stats);
  const Bias bias{key_bias, bias_batches, bias_heads, Lk};
  Joins joins{{}, H, (int)BH, vec_out};
  int parts = 0;
  auto add_join = [&](const float* part, int cuts, int L, int Lt, float* dst, const int64_t* g) {
    joins.t[parts++] = {part, dst, g[0], g[1], g[2], cuts, L, Lt};
  };
  auto join = [&]() {
    if (parts == 0) return;
    int64_t blocks = 0;
    for (int i = 0; i < parts; ++i) {
      const int rows = 16 / joins.t[i].threads();
      const int64_t n = (BH * joins.t[i].L + rows - 1) / rows;
      blocks = n > blocks ? n : blocks;
    }
    LaunchScope scope(kKSdpaSplit, stream);
    launch_chained(join_k, dim3((unsigned)blocks, parts), dim3(256), 0, stream, joins);
  };
  auto bias_grad = [&](const float* part, int terms, int Lt) {
    LaunchScope scope(kKSdpaSplit, stream);
    launch_chained(bias_grad_k, dim3((Lk + 31) / 32, bias_batches * bias_heads), dim3(32, 8), 0, stream, part, terms, B, H,
                   bias_batches, bias_heads, Lk, Lt, dbias);
  };
  FewArgs a{};
  a.H = H; a.BH = (int)BH; a.Lq = Lq; a.Lk = Lk;
  if (few(a)) {
    a.dout = rows_of(dout, strides); a.q = rows_of(q, strides + 3); a.k = rows_of(k, strides + 6);
    a.v = rows_of(v, strides + 9); a.out = rows_of(out, strides + 12);
    a.bias = bias;
    a.head = rows + Lq; a.head_stride = Lq + 1;
    a.stats = rows;
    a.dk = dk; a.kb = go[3]; a.kh = go[4]; a.kl = go[5];
    a.dv = dv; a.vb = go[6]; a.vh = go[7]; a.vl = go[8];
    a.vec = vec; a.vec_out = vec_out;
    const size_t qbytes = al256((size_t)a.shares * BH * Lq * D * 4);
    const size_t kbytes = a.groups > 1 ? al256((size_t)a.groups * BH * Lk * D * 4) : 0;
    uint8_t* ws = static_cast<uint8_t*>(workspace(qbytes + 2 * kbytes + (dbias ? (size_t)a.groups * BH * Lk * 4 : 0), stream));
    if (!ws) return kWorkspace;
    a.dq = reinterpret_cast<float*>(ws);
    a.dk_part = reinterpret_cast<float*>(ws + qbytes);
    a.dv_part = reinterpret_cast<float*>(ws + qbytes + kbytes);
    a.db = dbias ? reinterpret_cast<float*>(ws + qbytes + 2 * kbytes) : nullptr;
    if (a.groups > 1) a.vec_out = 1;  // into the partial sums, joined by a last kernel as dq's are
    few_bwd(a, stream);
    add_join(a.dq, a.shares, Lq, Lq, dq, go);
    if (a.groups > 1) {
      add_join(a.dk_part, a.groups, Lk, Lk, dk, go + 3);
      add_join(a.dv_part, a.groups, Lk, Lk, dv, go + 6);
    }
    join();
    if (dbias) bias_grad(a.db, a.groups, Lk);
    return launch_status();
  }
  st = key_bias ? ensure_kernel<true>() : ensure_kernel<false>();
  if (st != kOk) return st;
  Params p{};
  Side qs{}, ks{};
  const size_t qbytes = side_layout(nullptr, BH, Lq, true, qs), kbytes = side_layout(nullptr, BH, Lk, false, ks);
  p.keys.T = (Lq + WALK - 1) / WALK;
  p.keys.Ft = (Lk + HELD - 1) / HELD;
  p.keys.ragged = Lq % WALK != 0;
  p.queries.T = (Lk + WALK - 1) / WALK;
  p.queries.Ft = (Lq + HELD - 1) / HELD;
  p.queries.ragged = Lk % WALK != 0;
  cut_walks(p.keys, p.queries, BH);
  const size_t kpart = p.keys.cuts > 1 ? al256((size_t)p.keys.cuts * BH * ks.Lt * D * 4) : 0;
  const size_t qpart = p.queries.cuts > 1 ? al256((size_t)p.queries.cuts * BH * qs.Lt * D * 4) : 0;
  const size_t db_bytes = dbias ? al256((size_t)2 * p.keys.cuts * BH * ks.Lt * 4) : 0;
  const size_t tile_bytes = key_bias ? al256((size_t)BH * sizeof(int2)) : 0;
  uint8_t* ws = static_cast<uint8_t*>(workspace(qbytes + kbytes + 2 * kpart + qpart + db_bytes + tile_bytes + 256, stream));
  if (!ws) return kWorkspace;
  side_layout(ws, BH, Lq, true, qs);
  side_layout(ws + qbytes, BH, Lk, false, ks);
  uint8_t* at = ws + qbytes + kbytes;
  p.keys.held = ks;
  p.keys.walk = qs;
  p.keys.out1 = kpart ? reinterpret_cast<float*>(at) : dk;
  p.keys.out2 = kpart ? reinterpret_cast<float*>(at + kpart) : dv;
  p.keys.s1b = go[3]; p.keys.s1h = go[4]; p.keys.s1l = go[5];
  p.keys.s2b = go[6]; p.keys.s2h = go[7]; p.keys.s2l = go[8];
  p.keys.vec_out = vec_out;
  p.queries.held = qs;
  p.queries.walk = ks;
  p.queries.out1 = qpart ? reinterpret_cast<float*>(at + 2 * kpart) : dq;
  p.queries.s1b = go[0]; p.queries.s1h = go[1]; p.queries.s1l = go[2];
  p.queries.vec_out = vec_out;
  p.db = dbias ? reinterpret_cast<float*>(at + 2 * kpart + qpart) : nullptr;
  int2* tiles = key_bias ? reinterpret_cast<int2*>(at + 2 * kpart + qpart + db_bytes) : nullptr;
  p.tiles = tiles;
  p.next = reinterpret_cast<int*>(at + 2 * kpart + qpart + db_bytes + tile_bytes);
  p.keys_last = 4 * (p.keys.span + 4) < 3 * (p.queries.span + 4);
  p.head = rows + Lq;
  p.head_stride = Lq + 1;
  p.H = H;
  p.BH = (int)BH;
  p.key_items = (int)(BH * p.keys.Ft * p.keys.cuts);
  p.items = p.key_items + (int)(BH * p.queries.Ft * p.queries.cuts);
  p.status = device_status();
  Maps m;
  if (!plane_map(&m.q1h, qs.hi1, BH, qs.Lt) || !plane_map(&m.q1l, qs.lo1, BH, qs.Lt) ||
      !plane_map(&m.q2h, qs.hi2, BH, qs.Lt) || !plane_map(&m.q2l, qs.lo2, BH, qs.Lt) ||
      !plane_map(&m.k1h, ks.hi1, BH, ks.Lt) || !plane_map(&m.k1l, ks.lo1, BH, ks.Lt) ||
      !plane_map(&m.k2h, ks.hi2, BH, ks.Lt) || !plane_map(&m.k2l, ks.lo2, BH, ks.Lt))
    return kLaunchFailed;
  {
    LaunchScope scope(kKSdpaSplit, stream);
    bwd_split_k<<<dim3((unsigned)BH, (ks.Lt + qs.Lt) / HELD), 256, 0, stream>>>(
        rows_of(q, strides + 3), rows_of(dout, strides), rows_of(out, strides + 12), rows_of(k, strides + 6),
        rows_of(v, strides + 9), bias, rows, Lq + 1, H, vec, qs, ks, p.next, tiles);
  }
  {
    LaunchScope scope(kKSdpaAttn, stream);
    const unsigned grid = (unsigned)(p.items < sm_count() ? p.items : sm_count());
    launch_chained(key_bias ? sdpa_bwd_tc<true> : sdpa_bwd_tc<false>, dim3(grid), dim3(kThreads), SMEM_BYTES, stream, m, p);
  }
  if (qpart) add_join(p.queries.out1, p.queries.cuts, Lq, qs.Lt, dq, go);
  if (kpart) {
    add_join(p.keys.out1, p.keys.cuts, Lk, ks.Lt, dk, go + 3);
    add_join(p.keys.out2, p.keys.cuts, Lk, ks.Lt, dv, go + 6);
  }
  join();
  if (dbias) bias_grad(p.db, 2 * p.keys.cuts, ks.Lt);
  return launch_status();
}

}  // extern "C"
