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
// dQ: three).  Both are one kernel: F1, F2 are the held operands (K, V or Q, g), G1, G2 the walked
// ones (Q, g or K, V):
//   X = F1 G1^T ;  Y = F2 G2^T ;  e = 2^(c X + column + row) ;  ds = e (a Y - delta) ;
//   acc1 += ds G1   (dK or dQ) ;  acc2 += e G2   (dV, keys' pass only).
//
// Split precision as in sdpa.cu: every operand is an fp16 pair hi + lo after an exact power-of-two
// scale (one per 64-row tile; for e and ds a power of two from the bound 2^8 on e, and for ds from
// the tiles' largest row norms, |g . v - delta| <= |g| |v| + |delta|), each product is three
// tensor-core passes (hi.hi, hi.lo, lo.hi), and a walked tile's products go into a fresh
// accumulator in tensor memory that is added to fp32 registers: the tensor core's own fp32
// accumulation truncates, and one accumulator over thousands of rows would drift.
//
// CTA: 384 threads, one per SM, persistent over (head, held tile).  Warp 0 loads walked tiles
// (64 rows: 32 KB of planes and the tile's vectors, kStages deep), warp 1 issues all MMAs, two
// warpgroups compute.  The held operands live in tensor memory as the A side of X and Y (128
// columns), so that shared memory feeds the tensor core only the walked side.  X and Y have
// two buffers of 64 columns each: the tensor core forms X, Y of the next tile while the
// warpgroups turn the current ones, in place, into the fp16 pairs of e and ds, the A side of the
// accumulating products.  G1, G2 are read from the same shared tile both ways: K-major for X
// and Y (the 64 head dimensions contracted), MN-major for the accumulators (rows contracted).
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
constexpr int WALK = 64;                // rows of a walked tile, and of a scale tile
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

// Shared-memory descriptor of a 64-column fp16 tile (128-byte rows, 128-byte swizzle) read
// MN-major: the 64 columns are the operand's N, rows its K; groups of 8 rows are 1024 bytes apart.
__device__ __forceinline__ uint64_t sw128_mnmajor_desc(uint32_t smem_addr) {
  uint64_t d = 0;
  d |= (uint64_t)((smem_addr >> 4) & 0x3FFFu);
  d |= (uint64_t)(1024u >> 4) << 16;  // next 64 columns (N = 64: not used)
  d |= (uint64_t)(1024u >> 4) << 32;  // next 8 rows
  d |= (uint64_t)1u << 46;
  d |= (uint64_t)2u << 61;
  return d;
}

// One scale tile (64 rows) of the two tensors of a side.
struct TileScale {
  float inv1, inv2;   // inverse pre-scales of (Q, g) or (K, V)
  float norm, delta;  // queries: largest |g_i|, |delta_i|; keys: largest |v_j|, 0
};

// The two sides' planes, all [BH, rows padded to 128, 64] fp16, rows past the end zero.
struct Side {
  __half *hi1, *lo1, *hi2, *lo2;
  float *col;         // queries: -m_i (-inf past the end and for rows without a key); keys: bias in log2 units
  float *delta;       // queries: -delta_i; keys: unused
  TileScale* scale;   // [BH, padded / 64]
  int L, Lt;          // rows, padded rows
};

struct Params {
  Side held, walk;
  const float* head;  // [BH]: 0 where the bias leaves the scores no weight, 1 otherwise
  float *out1, *out2; // dK (or dQ), dV
  float* db;          // nullable: [2, BH, Lt of the keys] sums of ds over each warpgroup's queries
  int64_t s1b, s1h, s1l, s2b, s2h, s2l;  // element strides of out1, out2
  int H, BH, T, Ft, vec_out;  // T walked tiles, Ft held tiles per head
  int* status;
};

template <bool KEYS>
__global__ void __launch_bounds__(kThreads, 1)
    sdpa_bwd_tc(const __grid_constant__ CUtensorMap tm1h, const __grid_constant__ CUtensorMap tm1l,
                const __grid_constant__ CUtensorMap tm2h, const __grid_constant__ CUtensorMap tm2l,
                const Params p) {
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>(
      (reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~static_cast<uintptr_t>(1023));
  uint8_t* tiles = smem;                                     // [kStages] G1 hi, lo, G2 hi, lo
  uint8_t* vecs = tiles + kStages * STAGE;                   // [kStages] columns, deltas, scales
  uint64_t* bars = reinterpret_cast<uint64_t*>(vecs + kStages * VEC_STAGE);
  uint64_t* full = bars;               // [kStages] walked tile loaded
  uint64_t* empty = full + kStages;    // [kStages] both products of the tile retired
  uint64_t* xy_full = empty + kStages; // [2] X, Y formed
  uint64_t* ed_full = xy_full + 2;     // [2] e, ds written over them (8 warps)
  uint64_t* acc_full = ed_full + 2;    // [2] accumulators of a tile formed
  uint64_t* acc_free = acc_full + 2;   // [2] ... and folded into registers (8 warps)
  uint64_t* held_full = acc_free + 2;  // the item's held operands are in tensor memory (8 warps)
  uint64_t* all_done = held_full + 1;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(all_done + 1);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);

  const uint32_t warp = warp_id(), lane = lane_id();
  const int T = p.T;
  const int items = p.Ft * p.BH;
  const int my_items = (int)blockIdx.x < items ? (items - 1 - (int)blockIdx.x) / (int)gridDim.x + 1 : 0;
  auto item_of = [&](int i, int& bh, int& f0) {
    const int j = blockIdx.x + i * gridDim.x;
    bh = j / p.Ft;
    f0 = (j - bh * p.Ft) * HELD;
  };

  if (threadIdx.x == 0) {
    for (int i = 0; i < kStages; ++i) { mbar_init(&full[i], 1); mbar_init(&empty[i], 1); }
    for (int i = 0; i < 2; ++i) {
      mbar_init(&xy_full[i], 1);
      mbar_init(&ed_full[i], 8);
      mbar_init(&acc_full[i], 1);
      mbar_init(&acc_free[i], 8);
    }
    mbar_init(held_full, 8);
    mbar_init(all_done, 1);
    *abort_flag = 0;
    fence_barrier_init();
  }
  if (warp == 0 && lane == 0) {
    tma_prefetch_desc(&tm1h); tma_prefetch_desc(&tm1l);
    tma_prefetch_desc(&tm2h); tma_prefetch_desc(&tm2l);
  }
  if (warp == 1) {
    tmem_alloc(tmem_slot, TMEM_COLS);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;

  if (warp < 4) {
    setmaxnreg_dec<REGS_CONTROL>();
    if (warp == 0) {
      // ---------------- walked tiles ----------------
      if (elect_one()) {
        int issued[kStages];
        for (int s = 0; s < kStages; ++s) issued[s] = -1;
        bool ok = true;
        for (int i = 0; i < my_items && ok; ++i) {
          int bh, f0;
          item_of(i, bh, f0);
          for (int t = 0; t < T; ++t) {
            const int G = i * T + t, st = G % kStages;
            if (G >= kStages &&
                !mbar_wait(&empty[st], ((G / kStages) & 1) ^ 1, p.status, kDevTimeoutProducer, abort_flag)) {
              ok = false;
              break;
            }
            uint8_t* d = tiles + st * STAGE;
            uint8_t* v = vecs + st * VEC_STAGE;
            const int64_t row = (int64_t)bh * p.walk.Lt + t * WALK;
            mbar_arrive_expect_tx(&full[st], STAGE + WALK * 4 * (KEYS ? 2 : 1) + 16);
            tma_load_3d(d, &tm1h, &full[st], 0, t * WALK, bh);
            tma_load_3d(d + PLANE, &tm1l, &full[st], 0, t * WALK, bh);
            tma_load_3d(d + 2 * PLANE, &tm2h, &full[st], 0, t * WALK, bh);
            tma_load_3d(d + 3 * PLANE, &tm2l, &full[st], 0, t * WALK, bh);
            bulk_load(v, p.walk.col + row, WALK * 4, &full[st]);
            if (KEYS) bulk_load(v + WALK * 4, p.walk.delta + row, WALK * 4, &full[st]);
            bulk_load(v + 2 * WALK * 4, p.walk.scale + row / WALK, 16, &full[st]);
            issued[st] = G;
          }
        }
        if (*abort_flag)  // never leave the CTA while a bulk copy may still write its shared memory
          for (int s = 0; s < kStages; ++s)
            if (issued[s] >= 0) mbar_wait(&full[s], (issued[s] / kStages) & 1, p.status, kDevTimeoutProducer, nullptr);
      }
    } else if (warp == 1) {
      // ---------------- all MMAs, in one thread's order ----------------
      // X, Y of tile t + 1 are issued ahead of tile t's accumulating products, so the tensor core
      // has them to do while e, ds of tile t are formed.  Their buffer's last readers, the
      // products of tile t - 1, come before them in the same order.
      if (elect_one()) {
        constexpr uint32_t idesc_xy = idesc_f16_f32(HELD, WALK);
        constexpr uint32_t idesc_acc = idesc_f16_f32(HELD, D) | (1u << 16);  // B MN-major
        bool ok = true;
        auto form_xy = [&](int G) -> bool {
          const int st = G % kStages;
          if (!mbar_wait(&full[st], (G / kStages) & 1, p.status, kDevTimeoutMma, abort_flag)) return false;
          tc_fence_after();
          const uint32_t g = smem_u32(tiles + st * STAGE);
          const uint32_t x = tmem + XY_COL + (G & 1) * 128;
#pragma unroll 1
          for (int o = 0; o < 2; ++o) {  // X from F1, G1, then Y from F2, G2
            const uint32_t f = tmem + F_COL + o * 64, gh = g + o * 2 * PLANE, d = x + o * 64;
#pragma unroll 1
            for (int kk = 0; kk < D / 16; ++kk) {
              const uint64_t b_h = sw128_kmajor_desc(gh + kk * 32), b_l = sw128_kmajor_desc(gh + PLANE + kk * 32);
              mma_f16_ts(d, f + kk * 8, b_h, idesc_xy, kk != 0);
              mma_f16_ts(d, f + kk * 8, b_l, idesc_xy, 1);
              mma_f16_ts(d, f + 32 + kk * 8, b_h, idesc_xy, 1);
            }
          }
          mma_commit(&xy_full[G & 1]);
          return true;
        };
        for (int i = 0; i < my_items && ok; ++i) {
          ok = mbar_wait(held_full, i & 1, p.status, kDevTimeoutMma, abort_flag);
          if (ok) {
            tc_fence_after();
            ok = form_xy(i * T);
          }
          for (int t = 0; t < T && ok; ++t) {
            const int G = i * T + t, st = G % kStages;
            if (t + 1 < T) ok = form_xy(G + 1);
            // the keys' pass has one buffer of accumulators, the queries' pass two
            const int prev = KEYS ? G - 1 : G - 2;
            ok = ok && mbar_wait(&ed_full[G & 1], (G >> 1) & 1, p.status, kDevTimeoutMma, abort_flag) &&
                 (prev < 0 || mbar_wait(&acc_free[prev & 1], (prev >> 1) & 1, p.status, kDevTimeoutMma, abort_flag));
            if (!ok) break;
            tc_fence_after();
            const uint32_t g = smem_u32(tiles + st * STAGE);
            const uint32_t x = tmem + XY_COL + (G & 1) * 128;
#pragma unroll 1
            for (int o = KEYS ? 0 : 1; o < 2; ++o) {  // acc2 from e and G2, then acc1 from ds and G1
              const uint32_t a = x + o * 64, gh = g + (1 - o) * 2 * PLANE;
              const uint32_t d = tmem + ACC_COL + (KEYS ? (1 - o) * 64 : (G & 1) * 64);
#pragma unroll 1
              for (int kk = 0; kk < WALK / 16; ++kk) {
                const uint64_t b_h = sw128_mnmajor_desc(gh + kk * 2048), b_l = sw128_mnmajor_desc(gh + PLANE + kk * 2048);
                mma_f16_ts(d, a + kk * 16, b_h, idesc_acc, kk != 0);
                mma_f16_ts(d, a + kk * 16, b_l, idesc_acc, 1);
                mma_f16_ts(d, a + kk * 16 + 8, b_h, idesc_acc, 1);
              }
            }
            mma_commit(&empty[st]);
            mma_commit(&acc_full[G & 1]);
          }
        }
        mma_commit(all_done);
        mbar_wait(all_done, 0, p.status, kDevTimeoutMma, nullptr);
      }
    }
  } else {
    setmaxnreg_inc<REGS_COMPUTE>();
    // ---------------- e, ds and the folds: warpgroup w has walked rows 32w..32w+31 ----------------
    const int w = (warp - 4) >> 2;
    const uint32_t sub = warp & 3;
    const int r = sub * 32 + lane;  // held row == tensor-memory lane
    const uint32_t trow = tmem + ((sub * 32) << 16);
    constexpr int NACC = KEYS ? 64 : 32;  // keys: w = 0 keeps dV, w = 1 dK; queries: half of dQ each
    bool ok = true;
    for (int i = 0; i < my_items && ok; ++i) {
      int bh, f0;
      item_of(i, bh, f0);
      const int64_t frow = (int64_t)bh * p.held.Lt + f0 + r;
      {
        // held operands into tensor memory: this warpgroup's pair of planes
        const __half* hi = w == 0 ? p.held.hi1 : p.held.hi2;
        const __half* lo = w == 0 ? p.held.lo1 : p.held.lo2;
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
        if (lane == 0) mbar_arrive(held_full);
      }
      const TileScale fs = p.held.scale[frow / WALK];
      const float head = p.head[bh];
      // row constants: queries' pass -m_i and -delta_i, keys' pass b_j
      const float row = p.held.col[frow] + E_LIFT;
      const float row_delta = KEYS ? 0.0f : p.held.delta[frow];
      const uint64_t row2 = f2pack(row, row);
      float acc[NACC];
#pragma unroll
      for (int k = 0; k < NACC; ++k) acc[k] = 0.0f;
      float db = 0.0f, fold_scale = 0.0f;
      // adds the accumulators of tile G to the registers
      auto fold = [&](int G) -> bool {
        if (!__all_sync(0xffffffffu, mbar_wait(&acc_full[G & 1], (G >> 1) & 1, p.status, kDevTimeoutConsumer, abort_flag)))
          return false;
        tc_fence_after();
        const uint32_t src = trow + ACC_COL + (KEYS ? (w == 0 ? 64 : 0) : (G & 1) * 64 + w * 32);
        const uint64_t s2 = f2pack(fold_scale, fold_scale);
#pragma unroll
        for (int c = 0; c < NACC / 32; ++c) {
          uint32_t v[32];
          tmem_ld32(src + c * 32, v);
          tmem_wait_ld();
          reg_fence(v);
#pragma unroll
          for (int k = 0; k < 32; k += 2)
            f2unpack(f2fma(f2pack(__uint_as_float(v[k]), __uint_as_float(v[k + 1])), s2,
                           f2pack(acc[c * 32 + k], acc[c * 32 + k + 1])),
                     acc[c * 32 + k], acc[c * 32 + k + 1]);
        }
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(&acc_free[G & 1]);
        return true;
      };
      for (int t = 0; t < T; ++t) {
        const int G = i * T + t, st = G % kStages;
        // the tile's vectors (their copy's completion seen by this thread) and its X, Y
        ok = mbar_wait(&full[st], (G / kStages) & 1, p.status, kDevTimeoutConsumer, abort_flag) &&
             mbar_wait(&xy_full[G & 1], (G >> 1) & 1, p.status, kDevTimeoutConsumer, abort_flag);
        if (!__all_sync(0xffffffffu, ok)) { ok = false; break; }
        tc_fence_after();
        const uint8_t* v = vecs + st * VEC_STAGE;
        const float4* col = reinterpret_cast<const float4*>(v) + w * 8;
        const float4* del = reinterpret_cast<const float4*>(v + WALK * 4) + w * 8;
        const TileScale ws = *reinterpret_cast<const TileScale*>(v + 2 * WALK * 4);
        const float c = 0.125f * LOG2E * head * fs.inv1 * ws.inv1;
        // ds is formed as ds * 2^kk with |ds| 2^kk <= 2^15: e <= 2^8, |Y - delta| <= bound < 2^(ilogb + 1)
        const float bound = fs.norm * ws.norm + (KEYS ? ws.delta : fs.delta);
        int kk = 6 - ((__float_as_int(bound) >> 23) - 127);
        kk = kk > 100 ? 100 : (kk < -100 ? -100 : kk);
        const float up = pow2i(kk);
        const float a = fs.inv2 * ws.inv2;
        const uint64_t c2 = f2pack(c, c), a2 = f2pack(a, a);
        const uint64_t b2 = f2pack(up * 0x1p-7f, up * 0x1p-7f);  // takes the lift of e back
        const uint64_t rd2 = f2pack(row_delta, row_delta);
        const uint32_t x0 = trow + XY_COL + (G & 1) * 128 + w * 32;
        uint32_t xv[32], yv[32];
        tmem_ld32(x0, xv);
        tmem_ld32(x0 + 64, yv);
        tmem_wait_ld();
        reg_fence(xv);
        reg_fence(yv);
        uint64_t dsum = 0ull;
#pragma unroll
        for (int ch = 0; ch < 2; ++ch) {  // 16 walked rows: 8 columns of hi pairs, 8 of lo pairs
          uint32_t pe[16], pd[16];
#pragma unroll
          for (int j = 0; j < 16; j += 4) {
            const int q = ch * 16 + j;
            const float4 cv = col[q / 4];
            const float4 dv = KEYS ? del[q / 4] : make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
            for (int h = 0; h < 2; ++h) {
              const int k = q + 2 * h;
              const uint64_t off = f2add(h == 0 ? f2pack(cv.x, cv.y) : f2pack(cv.z, cv.w), row2);
              float e0, e1;
              f2unpack(f2fma(f2pack(__uint_as_float(xv[k]), __uint_as_float(xv[k + 1])), c2, off), e0, e1);
              e0 = ex2(e0);
              e1 = ex2(e1);
              const uint64_t e = f2pack(e0, e1);
              const uint64_t nd = KEYS ? (h == 0 ? f2pack(dv.x, dv.y) : f2pack(dv.z, dv.w)) : rd2;
              const uint64_t y = f2fma(f2pack(__uint_as_float(yv[k]), __uint_as_float(yv[k + 1])), a2, nd);
              const uint64_t ds = f2mul(f2mul(e, b2), y);
              if (KEYS) {
                split2(e, pe[j / 2 + h], pe[8 + j / 2 + h]);
                dsum = f2add(dsum, ds);
              }
              split2(ds, pd[j / 2 + h], pd[8 + j / 2 + h]);
            }
          }
          if (KEYS) tmem_st16(x0 + ch * 16, pe);
          tmem_st16(x0 + 64 + ch * 16, pd);
        }
        tmem_wait_st();
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(&ed_full[G & 1]);
        if (t > 0 && !fold(G - 1)) { ok = false; break; }
        const float down = pow2i(-kk);
        if (KEYS) {
          fold_scale = w == 0 ? ws.inv2 * 0x1p-7f : ws.inv1 * down;
          float d0, d1;
          f2unpack(dsum, d0, d1);
          db = fmaf(d0 + d1, down, db);
        } else {
          fold_scale = ws.inv1 * down;
        }
      }
      if (ok && T > 0) ok = fold(i * T + T - 1);
      if (!ok) break;
      // ---- the held rows' gradients ----
      const int b = bh / p.H, h = bh - b * p.H;
      if (f0 + r < p.held.L) {
        const bool first = !KEYS || w == 1;  // out1 (dK, dQ) or out2 (dV)
        float* dst = first ? p.out1 + b * p.s1b + h * p.s1h + (int64_t)(f0 + r) * p.s1l + (KEYS ? 0 : w * 32)
                           : p.out2 + b * p.s2b + h * p.s2h + (int64_t)(f0 + r) * p.s2l;
        const float s = first ? 0.125f : 1.0f;
        if (p.vec_out) {
#pragma unroll
          for (int k = 0; k < NACC; k += 4)
            *reinterpret_cast<float4*>(dst + k) =
                make_float4(acc[k] * s, acc[k + 1] * s, acc[k + 2] * s, acc[k + 3] * s);
        } else {
#pragma unroll
          for (int k = 0; k < NACC; ++k) dst[k] = acc[k] * s;
        }
      }
      if (KEYS && p.db) p.db[(int64_t)w * p.BH * p.held.Lt + frow] = db;
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

// One block per (b, h): the key bias relative to its largest finite value, times `unit`, clamped to
// -1e6 (2^-1e6 is zero next to the largest), -inf kept; zeros without a bias; -inf past Lk.  head[bh]
// = 0 where the largest is beyond 2^60 in magnitude.
__global__ void __launch_bounds__(256) bias_rows_k(const float* __restrict__ bias, int bias_b, int bias_h, int H,
                                                   int Lk, int Lt, float unit, float* __restrict__ out,
                                                   float* __restrict__ head) {
  __shared__ float sm[8];
  const int bh = blockIdx.x, b = bh / H, h = bh - b * H;
  const float* src = bias ? bias + ((int64_t)(bias_b == 1 ? 0 : b) * bias_h + (bias_h == 1 ? 0 : h)) * Lk : nullptr;
  float mx = -INFINITY;
  if (src)
    for (int j = threadIdx.x; j < Lk; j += 256) mx = fmaxf(mx, src[j]);
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, o));
  if ((threadIdx.x & 31) == 0) sm[threadIdx.x >> 5] = mx;
  __syncthreads();
#pragma unroll
  for (int k = 0; k < 8; ++k) mx = fmaxf(mx, sm[k]);
  if (threadIdx.x == 0) head[bh] = mx > -INFINITY && fabsf(mx) > 0x1p60f ? 0.0f : 1.0f;
  for (int j = threadIdx.x; j < Lt; j += 256) {
    float v = j < Lk ? 0.0f : -INFINITY;
    if (src && j < Lk) {
      v = src[j];
      if (v != -INFINITY) {
        v -= mx;
        if (v < -1.0e6f) v = -1.0e6f;
        v *= unit;
      }
    }
    out[(int64_t)bh * Lt + j] = v;
  }
}

struct Rows {
  const float* p;
  int64_t b, h, l;
  __device__ __forceinline__ const float* at(int ib, int ih, int64_t il) const { return p + ib * b + ih * h + il * l; }
};

// 16 consecutive values
__device__ __forceinline__ void load16(const float* p, bool vec, float (&v)[16]) {
  if (vec) {
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      const float4 f = *reinterpret_cast<const float4*>(p + 4 * k);
      v[4 * k] = f.x; v[4 * k + 1] = f.y; v[4 * k + 2] = f.z; v[4 * k + 3] = f.w;
    }
  } else {
#pragma unroll
    for (int k = 0; k < 16; ++k) v[k] = p[k];
  }
}

__device__ __forceinline__ float absmax16(const float (&v)[16]) {
  float m = 0.0f;
#pragma unroll
  for (int k = 0; k < 16; ++k) m = fmaxf(m, fabsf(v[k]));
  return m;
}

__device__ __forceinline__ void store_split16(const float (&v)[16], float up, __half* hi, __half* lo) {
  __align__(16) __half2 h[8], l[8];
#pragma unroll
  for (int k = 0; k < 8; ++k) {
    const float a = v[2 * k] * up, b = v[2 * k + 1] * up;
    h[k] = __floats2half2_rn(a, b);
    const float2 f = __half22float2(h[k]);
    l[k] = __floats2half2_rn(a - f.x, b - f.y);
  }
#pragma unroll
  for (int k = 0; k < 2; ++k) {
    reinterpret_cast<uint4*>(hi)[k] = reinterpret_cast<const uint4*>(h)[k];
    reinterpret_cast<uint4*>(lo)[k] = reinterpret_cast<const uint4*>(l)[k];
  }
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

// One block per (b h, 64-row tile), four threads per row: the planes, vectors and scales of one side.
// Queries (KEYS = false): Q and g = dO / l, -m, -delta.  Keys: K and V, rows with a bias of -inf as zeros.
template <bool KEYS>
__global__ void __launch_bounds__(256) bwd_split_k(Rows t1, Rows t2, Rows o, const float2* __restrict__ stats,
                                                   int H, int vec, Side s) {
  __shared__ float4 sm[8];
  const int bh = blockIdx.x, b = bh / H, h = bh - b * H;
  const int row = blockIdx.y * WALK + (threadIdx.x >> 2), c0 = (threadIdx.x & 3) * 16;
  const int64_t prow = (int64_t)bh * s.Lt + row;
  float x[16], y[16];
#pragma unroll
  for (int k = 0; k < 16; ++k) x[k] = y[k] = 0.0f;
  float delta = 0.0f;
  if (row < s.L) {
    if (KEYS) {
      if (s.col[prow] != -INFINITY) {
        load16(t1.at(b, h, row) + c0, vec, x);
        load16(t2.at(b, h, row) + c0, vec, y);
      }
    } else {
      const float2 ml = stats[(int64_t)bh * s.L + row];
      load16(t1.at(b, h, row) + c0, vec, x);
      if (ml.y != 0.0f) {
        float ov[16];
        load16(t2.at(b, h, row) + c0, vec, y);
        load16(o.at(b, h, row) + c0, vec, ov);
        const float inv = 1.0f / ml.y;
#pragma unroll
        for (int k = 0; k < 16; ++k) {
          y[k] *= inv;
          delta = fmaf(y[k], ov[k], delta);
        }
      }
    }
  }
  float sq = 0.0f;
#pragma unroll
  for (int k = 0; k < 16; ++k) sq = fmaf(y[k], y[k], sq);
#pragma unroll
  for (int i = 1; i < 4; i <<= 1) {
    sq += __shfl_xor_sync(0xffffffffu, sq, i);
    delta += __shfl_xor_sync(0xffffffffu, delta, i);
  }
  if (!KEYS && (threadIdx.x & 3) == 0) {
    const float2 ml = row < s.L ? stats[(int64_t)bh * s.L + row] : make_float2(0.0f, 0.0f);
    s.col[prow] = ml.y != 0.0f ? -ml.x : -INFINITY;
    s.delta[prow] = -delta;
  }
  const float4 mx = block_max4(make_float4(absmax16(x), absmax16(y), sqrtf(sq), fabsf(delta)), sm);
  const int s1 = scale_shift(mx.x), s2 = scale_shift(mx.y);
  if (threadIdx.x == 0)
    s.scale[prow / WALK] = {pow2i(-s1), pow2i(-s2), mx.z * 1.0001f, KEYS ? 0.0f : mx.w * 1.0001f};
  store_split16(x, pow2i(s1), s.hi1 + prow * D + c0, s.lo1 + prow * D + c0);
  store_split16(y, pow2i(s2), s.hi2 + prow * D + c0, s.lo2 + prow * D + c0);
}

// The forward kernel's planes (sdpa_planes.h) from strided tensors.  Queries: one scale per row,
// four threads per row, 64 rows per block.
__global__ void __launch_bounds__(256) fwd_split_q_k(Rows q, const float* __restrict__ head, int H, int Lq, int vec,
                                                     __half* __restrict__ hi, __half* __restrict__ lo,
                                                     float* __restrict__ qinv) {
  const int bh = blockIdx.x, b = bh / H, h = bh - b * H;
  const int row = blockIdx.y * WALK + (threadIdx.x >> 2), c0 = (threadIdx.x & 3) * 16;
  float x[16];
#pragma unroll
  for (int k = 0; k < 16; ++k) x[k] = 0.0f;
  if (row < Lq) load16(q.at(b, h, row) + c0, vec, x);
  float mx = absmax16(x);
#pragma unroll
  for (int i = 1; i < 4; i <<= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, i));
  if (row >= Lq) return;
  const int s = scale_shift(mx);
  const int64_t prow = (int64_t)bh * Lq + row;
  store_split16(x, pow2i(s), hi + prow * D + c0, lo + prow * D + c0);
  if ((threadIdx.x & 3) == 0) qinv[prow] = pow2i(-s) * head[bh];
}

// Keys: one block per 128-key tile (one scale each for K and V), eight warps of 16 keys; V goes
// through shared memory to its transposed planes.
constexpr int KT = 128;
__global__ void __launch_bounds__(256) fwd_split_kv_k(Rows kr, Rows vr, const float* __restrict__ bias, int H, int Lk,
                                                      int Lkt, int vec, __half* __restrict__ khi,
                                                      __half* __restrict__ klo, __half* __restrict__ vhi,
                                                      __half* __restrict__ vlo, float* __restrict__ kinv,
                                                      float* __restrict__ vinv) {
  __shared__ float vt[KT][D + 1];
  __shared__ float4 sm[8];
  const int bh = blockIdx.x, b = bh / H, h = bh - b * H, tile = blockIdx.y;
  float x[2][16];
  float kmx = 0.0f, vmx = 0.0f;
#pragma unroll
  for (int u = 0; u < 2; ++u) {
    const int j = u * 64 + (threadIdx.x >> 2), row = tile * KT + j, c0 = (threadIdx.x & 3) * 16;
    float y[16];
#pragma unroll
    for (int k = 0; k < 16; ++k) x[u][k] = y[k] = 0.0f;
    if (row < Lk && !(bias && bias[(int64_t)bh * Lk + row] == -INFINITY)) {
      load16(kr.at(b, h, row) + c0, vec, x[u]);
      load16(vr.at(b, h, row) + c0, vec, y);
    }
#pragma unroll
    for (int k = 0; k < 16; ++k) vt[j][c0 + k] = y[k];
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
    const int64_t prow = (int64_t)bh * Lkt + tile * KT + u * 64 + (threadIdx.x >> 2);
    const int c0 = (threadIdx.x & 3) * 16;
    store_split16(x[u], pow2i(sk), khi + prow * D + c0, klo + prow * D + c0);
  }
  for (int e = threadIdx.x; e < D * (KT / 16); e += 256) {
    const int d = e % D, jb = e / D * 16;
    float v[16];
#pragma unroll
    for (int k = 0; k < 16; ++k) v[k] = vt[jb + k][d];
    const int64_t off = ((int64_t)bh * D + d) * Lkt + tile * KT + jb;
    store_split16(v, pow2i(sv), vhi + off, vlo + off);
  }
  if (threadIdx.x == 0) {
    kinv[(int64_t)bh * (Lkt / KT) + tile] = pow2i(-sk);
    vinv[(int64_t)bh * (Lkt / KT) + tile] = pow2i(-sv);
  }
}

// db [bias_b, bias_h, Lk]: part [2, B, H, Lt] added over the halves and the batch entries and heads
// that share a row, in their order.
__global__ void __launch_bounds__(256) bias_grad_k(const float* __restrict__ part, int B, int H, int bias_b,
                                                   int bias_h, int Lk, int Lt, float* __restrict__ db) {
  const int j = blockIdx.x * 256 + threadIdx.x, row = blockIdx.y;
  if (j >= Lk) return;
  const int rb = row / bias_h, rh = row - rb * bias_h;
  const int b0 = bias_b == 1 ? 0 : rb, b1 = bias_b == 1 ? B : rb + 1;
  const int h0 = bias_h == 1 ? 0 : rh, h1 = bias_h == 1 ? H : rh + 1;
  float s = 0.0f;
  for (int b = b0; b < b1; ++b)
    for (int h = h0; h < h1; ++h) {
      const int64_t i = ((int64_t)b * H + h) * Lt + j;
      s += part[i] + part[i + (int64_t)B * H * Lt];
    }
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
  s.scale = reinterpret_cast<TileScale*>(take(rows / WALK * sizeof(TileScale)));
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
template <bool KEYS>
static int ensure_kernel() {
  static std::atomic<uint64_t> done{0};
  int dev = 0;
  cudaGetDevice(&dev);
  if (done.load(std::memory_order_acquire) >> (dev & 63) & 1) return kOk;
  cudaFuncAttributes fa{};
  if (cudaFuncGetAttributes(&fa, sdpa_bwd_tc<KEYS>) != cudaSuccess || fa.numRegs < (int)REGS_LAUNCH) {
    set_last_error("sdpa_bwd_tc was compiled with fewer registers than its warpgroup budget needs");
    return kLaunchFailed;
  }
  if (cudaFuncSetAttribute(sdpa_bwd_tc<KEYS>, cudaFuncAttributeMaxDynamicSharedMemorySize, SMEM_BYTES) != cudaSuccess)
    return launch_status();
  done.fetch_or(1ull << (dev & 63), std::memory_order_acq_rel);
  return kOk;
}

template <bool KEYS>
static int launch_bwd(const Params& p, int64_t BH, cudaStream_t stream) {
  int st = ensure_kernel<KEYS>();
  if (st != kOk) return st;
  CUtensorMap m1h, m1l, m2h, m2l;
  if (!plane_map(&m1h, p.walk.hi1, BH, p.walk.Lt) || !plane_map(&m1l, p.walk.lo1, BH, p.walk.Lt) ||
      !plane_map(&m2h, p.walk.hi2, BH, p.walk.Lt) || !plane_map(&m2l, p.walk.lo2, BH, p.walk.Lt))
    return kLaunchFailed;
  const int64_t items = (int64_t)p.Ft * BH;
  const int sms = sm_count();
  LaunchScope scope(kKSdpaAttn, stream);
  sdpa_bwd_tc<KEYS><<<(unsigned)(items < sms ? items : sms), kThreads, SMEM_BYTES, stream>>>(m1h, m1l, m2h, m2l, p);
  return launch_status();
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
  SplitPlanesSdpa sp;
  void* behind = nullptr;
  const size_t bias_bytes = al256((size_t)BH * Lk * 4);
  st = sdpa_planes_extra(BH, Lq, Lk, bias_bytes + al256((size_t)BH * 4), stream, sp, &behind);
  if (st != kOk) return st;
  float* bias = static_cast<float*>(behind);
  float* head = reinterpret_cast<float*>(static_cast<uint8_t*>(behind) + bias_bytes);
  const int vec = rows16({q, k, v}, strides, 3);
  {
    LaunchScope scope(kKSdpaSplit, stream);
    bias_rows_k<<<(unsigned)BH, 256, 0, stream>>>(key_bias, bias_batches, bias_heads, H, Lk, Lk, 1.0f, bias, head);
  }
  {
    LaunchScope scope(kKSdpaSplit, stream);
    fwd_split_q_k<<<dim3((unsigned)BH, (Lq + WALK - 1) / WALK), 256, 0, stream>>>(rows_of(q, strides), head, H, Lq, vec,
                                                                             sp.qhi, sp.qlo, sp.qinv);
  }
  {
    LaunchScope scope(kKSdpaSplit, stream);
    fwd_split_kv_k<<<dim3((unsigned)BH, sp.T), 256, 0, stream>>>(rows_of(k, strides + 3), rows_of(v, strides + 6),
                                                                 key_bias ? bias : nullptr, H, Lk, sp.Lkt, vec, sp.khi,
                                                                 sp.klo, sp.vhi, sp.vlo, sp.kinv, sp.vinv);
  }
  if ((st = launch_status()) != kOk) return st;
  return sdpa_attend_stats(sp, key_bias ? bias : nullptr, Lk, out_blhd, reinterpret_cast<float2*>(stats), BH, H, Lq, Lk,
                           stream);
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
  Side qs{}, ks{};
  const size_t qbytes = side_layout(nullptr, BH, Lq, true, qs), kbytes = side_layout(nullptr, BH, Lk, false, ks);
  const size_t head_bytes = al256((size_t)BH * 4), db_bytes = dbias ? al256((size_t)2 * BH * ks.Lt * 4) : 0;
  uint8_t* ws = static_cast<uint8_t*>(workspace(qbytes + kbytes + head_bytes + db_bytes, stream));
  if (!ws) return kWorkspace;
  side_layout(ws, BH, Lq, true, qs);
  side_layout(ws + qbytes, BH, Lk, false, ks);
  float* head = reinterpret_cast<float*>(ws + qbytes + kbytes);
  float* part = dbias ? reinterpret_cast<float*>(ws + qbytes + kbytes + head_bytes) : nullptr;
  const int vec = rows16({dout, q, k, v, out}, strides, 5);
  {
    LaunchScope scope(kKSdpaSplit, stream);
    bias_rows_k<<<(unsigned)BH, 256, 0, stream>>>(key_bias, bias_batches, bias_heads, H, Lk, ks.Lt, LOG2E, ks.col, head);
  }
  {
    LaunchScope scope(kKSdpaSplit, stream);
    bwd_split_k<true><<<dim3((unsigned)BH, ks.Lt / WALK), 256, 0, stream>>>(
        rows_of(k, strides + 6), rows_of(v, strides + 9), Rows{}, nullptr, H, vec, ks);
  }
  {
    LaunchScope scope(kKSdpaSplit, stream);
    bwd_split_k<false><<<dim3((unsigned)BH, qs.Lt / WALK), 256, 0, stream>>>(
        rows_of(q, strides + 3), rows_of(dout, strides), rows_of(out, strides + 12),
        reinterpret_cast<const float2*>(stats), H, vec, qs);
  }
  if ((st = launch_status()) != kOk) return st;
  const int64_t* go = strides + 15;  // dq, dk, dv
  Params p{};
  p.head = head;
  p.H = H;
  p.BH = (int)BH;
  p.vec_out = rows16({dq, dk, dv}, go, 3);
  p.status = device_status();
  p.held = ks;
  p.walk = qs;
  p.T = (Lq + WALK - 1) / WALK;
  p.Ft = (Lk + HELD - 1) / HELD;
  p.out1 = dk; p.s1b = go[3]; p.s1h = go[4]; p.s1l = go[5];
  p.out2 = dv; p.s2b = go[6]; p.s2h = go[7]; p.s2l = go[8];
  p.db = part;
  if ((st = launch_bwd<true>(p, BH, stream)) != kOk) return st;
  p.held = qs;
  p.walk = ks;
  p.T = (Lk + WALK - 1) / WALK;
  p.Ft = (Lq + HELD - 1) / HELD;
  p.out1 = dq; p.s1b = go[0]; p.s1h = go[1]; p.s1l = go[2];
  p.out2 = nullptr;
  p.db = nullptr;
  if ((st = launch_bwd<false>(p, BH, stream)) != kOk) return st;
  if (dbias) {
    LaunchScope scope(kKSdpaSplit, stream);
    bias_grad_k<<<dim3((Lk + 255) / 256, bias_batches * bias_heads), 256, 0, stream>>>(part, B, H, bias_batches,
                                                                                     bias_heads, Lk, ks.Lt, dbias);
  }
  return launch_status();
}

}  // extern "C"
