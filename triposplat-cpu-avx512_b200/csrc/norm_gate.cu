// Norms before and after a block, fused with the block's gate, residual scale and modulation:
//   z = x + rho * gate[b] * w_post * post(y)
//   h = w_pre * pre(z) * (1 + scale[b]) + shift[b]
// post in {none, layer, rms}, pre in {none, layer, rms}; layer(v) = (v - mean) * r with
// r = 1 / sqrt(mean((v - mean)^2) + eps), rms(v) = v / sqrt(mean(v^2) + eps).
//
// Backward, with m = post(y), n = pre(z) (rebuilt from x, y and four saved numbers per row, so
// that 16-bit tensors add no rounding between the two directions):
//   dn = dh (1 + scale) w_pre ;  dz' = dz + r_n (dn - [layer] mean(dn) - n mean(dn n)) = dx
//   dm = dz' rho gate w_post  ;  dy = r_m (dm - [layer] mean(dm) - m mean(dm m))   (none: dm)
//   S0 = sum dh, S1 = sum dh n, S2 = sum dz' m over a batch entry's rows, per column:
//   dshift = S0, dscale = w_pre S1, dgate = rho w_post S2,
//   dw_pre = sum_b (1 + scale) S1, dw_post = sum_b rho gate S2
// so three column sums carry all five parameter gradients.  Each row group adds its rows in
// order in registers and writes one partial row; a second kernel adds the partial rows in a
// fixed order: no atomics, the same bits on every run.
//
// Bound by HBM: every tensor is read or written once.  A row is held in registers (4, 8 or 16
// elements per thread) by one warp (up to 128 columns) or one block, statistics are taken
// in two passes over the registers (mean, then centred squares) in fp32.  A row group keeps its
// columns' coefficients (rho gate w_post, (1 + scale) w_pre, shift) in registers over all its rows,
// and (up to 4096 columns; beyond, registers are short) the next row's loads are in flight while a
// row is worked on.  Measured, 8193 x 1024 x 2 in fp32: forward 46 us (5.8 TB/s), backward 70 us (5.75)
// and 7 for the column sums; with 4 elements per thread, twice the warps per barrier, 55 and 94 us,
// with a warp per row and coefficients in shared memory (no barriers, 200 registers) 96 and 134.
// Odd widths, 2051 x 1111 x 3 in bf16: forward 24 us, backward 37; element by element, without the shift
// (Columns), 34 and 62.  16-bit rows are short: the two sums per row and direction, each a barrier, and 8 to 12 warps
// per SM bound them (3000 x 1024 x 2: 15 and 21 us in bf16, 19 and 31 in fp32).
#include <stdint.h>

#include <atomic>
#include <initializer_list>

#include "common.cuh"
#include "runtime.h"
#include "vecio.cuh"

namespace tsb {
namespace ng {

enum Kind : int { kNone = 0, kLayer = 1, kRms = 2 };
constexpr int kMaxThreads = 512;   // per row: 4 columns each up to 512, 8 up to 4096, 16 beyond
// blocks of up to this many threads: up to 168 registers, three warps in each quarter of an SM (free to take
// more, the backward kernel takes 176 to 192, and only two fit: 8193 x 1024 x 2 80 us)
constexpr int kFewThreads = 384;
constexpr int kMaxColumns = 8192;

struct Args {
  const void *x, *y, *dz, *dh;             // T; dz and dh only in the backward pass
  int64_t xb, xl, yb, yl, zb, zl, hb, hl;  // element strides (batch, row) of x, y, dz, dh
  const float *gate, *scale, *shift, *wpre, *wpost;  // [B, C], [B, C], [B, C], [C], [C] or null
  void *out0, *out1;                       // z, h or dx, dy: [B, L, C] contiguous
  float* stats;                            // [B * L, 4]: mean, r of post; mean, r of pre
  float* part;                             // [B, groups, 3, C] partial column sums
  int64_t L;
  int B, C, pre, post, groups;
  float rho, eps;
};

// Sums over a row's threads: one warp, or the whole block (`sm` [2][16] per summed value, alternated
// by `turn`, so one barrier per sum is enough; slots of warps that a block lacks are zero).
struct RowSum {
  float2 (*sm)[16];
  int turn;
  __device__ __forceinline__ RowSum(float2 (*s)[16]) : sm(s), turn(0) {
    const int t = threadIdx.y * blockDim.x + threadIdx.x;
    if (t < 32) sm[t / 16][t % 16] = make_float2(0.0f, 0.0f);
    if (blockDim.x > 32) __syncthreads();
  }
  __device__ __forceinline__ float2 operator()(float2 v) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
      v.x += __shfl_xor_sync(0xffffffffu, v.x, o);
      v.y += __shfl_xor_sync(0xffffffffu, v.y, o);
    }
    if (blockDim.x == 32) return v;
    const float4* s = share(v);
    float4 r = s[0];
#pragma unroll
    for (int w = 1; w < 8; ++w) {
      if (w * 64 >= blockDim.x) break;
      const float4 u = s[w];
      r.x += u.x; r.y += u.y; r.z += u.z; r.w += u.w;
    }
    return make_float2(r.x + r.z, r.y + r.w);
  }
  __device__ __forceinline__ float operator()(float v) {
    v = warp_sum(v);
    if (blockDim.x == 32) return v;
    const float4* s = share(make_float2(v, 0.0f));
    float r = s[0].x + s[0].z;
#pragma unroll
    for (int w = 1; w < 8; ++w) {
      if (w * 64 >= blockDim.x) break;
      r += s[w].x + s[w].z;
    }
    return r;
  }

 private:
  __device__ __forceinline__ const float4* share(float2 v) {
    float2* s = sm[turn];
    turn ^= 1;
    if ((threadIdx.x & 31) == 0) s[threadIdx.x >> 5] = v;
    __syncthreads();
    return reinterpret_cast<const float4*>(s);
  }
};

// Which columns a thread has: runs of VEC, one every blockDim.x * VEC.  Rows of an odd width start between
// two access boundaries; there (SHIFT) a thread's runs lie on the boundaries, `shift` elements before
// the row's own multiples, and the first and the last run of a row may be partly outside it: their bits there
// are cleared after the load (keep), whatever the neighbouring rows hold.  Nothing of this branches but the
// stores: a branch around what is fetched ahead, or around its use, took what the wide accesses gain.
template <class T, int VEC, int NI, bool SHIFT>
struct Columns {
  int C, shift;
  Raw<T, VEC> keep[SHIFT ? NI : 1];
  __device__ __forceinline__ Columns(int c, int s) : C(c), shift(s) {
    if constexpr (SHIFT) {
#pragma unroll
      for (int i = 0; i < NI; ++i) keep[i].mask(-at(i), C - at(i));
    }
  }
  __device__ __forceinline__ int at(int i) const {
    return (i * (int)blockDim.x + (int)threadIdx.x) * VEC - (SHIFT ? shift : 0);
  }
  __device__ __forceinline__ bool whole(int i) const { return (!SHIFT || at(i) >= 0) && at(i) + (SHIFT ? VEC : 1) <= C; }
  __device__ __forceinline__ bool has(int i, int e) const {
    return SHIFT ? (unsigned)(at(i) + e) < (unsigned)C : at(i) < C;
  }
};

// mean (0 for rms) and r of a row held in registers; elements past C are zero and stay out of
// the centred sum
template <class T, int VEC, int NI, bool SHIFT>
__device__ __forceinline__ float2 row_stats(const float (&v)[NI][VEC], int kind, const Columns<T, VEC, NI, SHIFT>& cols,
                                            float inv_c, float eps, RowSum& sum) {
  float mean = 0.0f, q = 0.0f;
  if (kind == kLayer) {
    float s = 0.0f;
#pragma unroll
    for (int i = 0; i < NI; ++i)
#pragma unroll
      for (int e = 0; e < VEC; ++e) s += v[i][e];
    mean = sum(s) * inv_c;
#pragma unroll
    for (int i = 0; i < NI; ++i)
#pragma unroll
      for (int e = 0; e < VEC; ++e) {
        const float d = cols.has(i, e) ? v[i][e] - mean : 0.0f;
        q = fmaf(d, d, q);
      }
  } else {  // elements outside are zeros
#pragma unroll
    for (int i = 0; i < NI; ++i)
#pragma unroll
      for (int e = 0; e < VEC; ++e) q = fmaf(v[i][e], v[i][e], q);
  }
  return make_float2(mean, rsqrtf(fmaf(sum(q), inv_c, eps)));
}

// A row's elements of one tensor as they lie in memory, and as numbers (zeros outside the row).  With a shift, runs
// at a row's ends read on into its neighbours; only where that would pass the end of the tensor (`room`
// elements behind the row's start: the last row) are they read word by word.
template <class T, int VEC, int NI, bool SHIFT>
struct RawRow {
  Raw<T, VEC> v[NI];
  __device__ __forceinline__ void clear() {  // all types' zero is zero bits
#pragma unroll
    for (int i = 0; i < NI; ++i) v[i].b = {};
  }
  __device__ __forceinline__ void load(const T* p, const Columns<T, VEC, NI, SHIFT>& cols, int64_t room) {
    if constexpr (SHIFT) {
      if (room < cols.C + VEC - 1) {  // the same in all threads of the row
#pragma unroll
        for (int i = 0; i < NI; ++i)
          if (cols.at(i) < cols.C) v[i].load_first(p + cols.at(i), cols.C - cols.at(i));
        return;
      }
    }
#pragma unroll
    for (int i = 0; i < NI; ++i) {
      const int c = cols.at(i);  // where it is negative: the boundary before the row, inside the tensor
      if (c < cols.C) v[i].load(p + c);
    }
  }
  __device__ __forceinline__ void get(float (&f)[NI][VEC], const Columns<T, VEC, NI, SHIFT>& cols) const {
#pragma unroll
    for (int i = 0; i < NI; ++i) {
      Raw<T, VEC> r = v[i];
      if constexpr (SHIFT) r = r & cols.keep[i];
#pragma unroll
      for (int e = 0; e < VEC; ++e) f[i][e] = r[e];
    }
  }
};

template <class T, int VEC, int NI, bool SHIFT>
__device__ __forceinline__ void store_row(T* p, const Columns<T, VEC, NI, SHIFT>& cols, const float (&v)[NI][VEC]) {
#pragma unroll
  for (int i = 0; i < NI; ++i) {
    const int c = cols.at(i);
    if (cols.whole(i)) store_vec<T, VEC>(p + c, v[i]);
    else if (SHIFT && c < cols.C) {
#pragma unroll
      for (int e = 0; e < VEC; ++e)
        if (cols.has(i, e)) p[c + e] = from_f32<T>(v[i][e]);
    }
  }
}

// a[c] * (b[c] + add) (null: a = 1, b = 0), zeros outside the row
template <class T, int VEC, int NI, bool SHIFT>
__device__ __forceinline__ void load_coef(const float* a, const float* b, float add, const Columns<T, VEC, NI, SHIFT>& cols,
                                          float (&v)[NI][VEC]) {
#pragma unroll
  for (int i = 0; i < NI; ++i) {
    const int c = cols.at(i);
#pragma unroll
    for (int e = 0; e < VEC; ++e)
      v[i][e] = cols.has(i, e) ? (a ? __ldg(a + c + e) : 1.0f) * ((b ? __ldg(b + c + e) : 0.0f) + add) : 0.0f;
  }
}

// Row group g of batch entry blockIdx.y takes the entry's rows g, g + groups, g + 2 groups, ...
template <class T, int VEC, int NI, int MAXT, bool SHIFT>
__global__ void __launch_bounds__(MAXT, 1) norm_gate_k(const Args a) {
  __shared__ __align__(16) float2 sm[2][16];
  RowSum sum(sm);
  const float inv_c = 1.0f / (float)a.C;
  const int64_t b = blockIdx.y, g = (int64_t)blockIdx.x * blockDim.y + threadIdx.y;
  const T* x = static_cast<const T*>(a.x) + b * a.xb + g * a.xl;
  const T* y = static_cast<const T*>(a.y) + b * a.yb + g * a.yl;
  const int64_t dx = a.groups * a.xl, dy = a.groups * a.yl;
  // the same shift in all tensors and all rows of the group (see launch)
  const Columns<T, VEC, NI, SHIFT> cols(a.C, SHIFT ? (int)((b * a.xb + g * a.xl) % VEC) : 0);
  int64_t roomx = (a.B - 1 - b) * a.xb + (a.L - 1 - g) * a.xl + a.C;
  int64_t roomy = (a.B - 1 - b) * a.yb + (a.L - 1 - g) * a.yl + a.C;
  RawRow<T, VEC, NI, SHIFT> ry, rx;
  ry.clear();
  rx.clear();
  auto fetch = [&]() {  // the next row of the group
    ry.load(y, cols, roomy);
    rx.load(x, cols, roomx);
    y += dy;
    x += dx;
    roomy -= dy;
    roomx -= dx;
  };
  constexpr bool kAhead = NI * VEC <= 8;
  const int64_t first = g < a.groups ? g : a.L;  // a block of several groups may hold more than there are
  if (kAhead && first < a.L) fetch();
  float gw[NI][VEC], sw[NI][VEC], sh[NI][VEC];
  load_coef<T, VEC, NI, SHIFT>(a.wpost, a.gate ? a.gate + b * a.C : nullptr, a.gate ? 0.0f : 1.0f, cols, gw);
  load_coef<T, VEC, NI, SHIFT>(a.wpre, a.scale ? a.scale + b * a.C : nullptr, 1.0f, cols, sw);
  load_coef<T, VEC, NI, SHIFT>(nullptr, a.shift ? a.shift + b * a.C : nullptr, 0.0f, cols, sh);
#pragma unroll 1
  for (int64_t l = first; l < a.L; l += a.groups) {
    const int64_t r = b * a.L + l;
    float z[NI][VEC], m[NI][VEC];
    if (!kAhead) fetch();
    ry.get(m, cols);
    rx.get(z, cols);
    if (kAhead && l + a.groups < a.L) fetch();
    float2 sp = make_float2(0.0f, 1.0f), sn = make_float2(0.0f, 1.0f);
    if (a.post != kNone) sp = row_stats<T, VEC, NI, SHIFT>(m, a.post, cols, inv_c, a.eps, sum);
    const float rs = sp.y * a.rho;
#pragma unroll
    for (int i = 0; i < NI; ++i)
#pragma unroll
      for (int e = 0; e < VEC; ++e) z[i][e] = fmaf((m[i][e] - sp.x) * rs, gw[i][e], z[i][e]);
    store_row<T, VEC, NI, SHIFT>(static_cast<T*>(a.out0) + r * a.C, cols, z);
    if (a.pre != kNone) {
      sn = row_stats<T, VEC, NI, SHIFT>(z, a.pre, cols, inv_c, a.eps, sum);
#pragma unroll
      for (int i = 0; i < NI; ++i)
#pragma unroll
        for (int e = 0; e < VEC; ++e) z[i][e] = fmaf((z[i][e] - sn.x) * sn.y, sw[i][e], sh[i][e]);
      store_row<T, VEC, NI, SHIFT>(static_cast<T*>(a.out1) + r * a.C, cols, z);
    }
    if (threadIdx.x == 0)
      *reinterpret_cast<float4*>(a.stats + 4 * r) = make_float4(sp.x, sp.y, sn.x, sn.y);
  }
}

template <class T, int VEC, int NI, int MAXT, bool SHIFT>
__global__ void __launch_bounds__(MAXT, 1) norm_gate_bwd_k(const Args a) {
  __shared__ __align__(16) float2 sm[2][16];
  grid_release();
  RowSum sum(sm);
  const int64_t b = blockIdx.y, g = (int64_t)blockIdx.x * blockDim.y + threadIdx.y;
  const float inv_c = 1.0f / (float)a.C;
  const bool has_h = a.dh != nullptr, has_z = a.dz != nullptr;
  const T* x = static_cast<const T*>(a.x) + b * a.xb + g * a.xl;
  const T* y = static_cast<const T*>(a.y) + b * a.yb + g * a.yl;
  const T* dh = has_h ? static_cast<const T*>(a.dh) + b * a.hb + g * a.hl : nullptr;
  const T* dz = has_z ? static_cast<const T*>(a.dz) + b * a.zb + g * a.zl : nullptr;
  const float4* stats = reinterpret_cast<const float4*>(a.stats) + b * a.L + g;
  const int64_t ix = a.groups * a.xl, iy = a.groups * a.yl, ih = a.groups * a.hl, iz = a.groups * a.zl;
  const Columns<T, VEC, NI, SHIFT> cols(a.C, SHIFT ? (int)((b * a.xb + g * a.xl) % VEC) : 0);
  // elements from this row's start to the tensors' ends: the least of the four
  auto room_of = [&](int64_t sb, int64_t sl) { return (a.B - 1 - b) * sb + (a.L - 1 - g) * sl + a.C; };
  int64_t room = SHIFT ? min(room_of(a.xb, a.xl), room_of(a.yb, a.yl)) : 0, step = SHIFT ? max(ix, iy) : 0;
  if (SHIFT && has_h) { room = min(room, room_of(a.hb, a.hl)); step = max(step, ih); }
  if (SHIFT && has_z) { room = min(room, room_of(a.zb, a.zl)); step = max(step, iz); }
  RawRow<T, VEC, NI, SHIFT> ry, rx, rh, rz;
  ry.clear();
  rx.clear();
  rh.clear();
  rz.clear();
  float4 st = make_float4(0.0f, 1.0f, 0.0f, 1.0f);
  auto fetch = [&]() {  // the next row of the group
    ry.load(y, cols, room);
    rx.load(x, cols, room);
    if (has_h) rh.load(dh, cols, room);
    if (has_z) rz.load(dz, cols, room);
    room -= step;
    st = __ldg(stats);
    y += iy;
    x += ix;
    dh += ih;
    dz += iz;
    stats += a.groups;
  };
  constexpr bool kAhead = NI * VEC <= 8;
  const int64_t first = g < a.groups ? g : a.L;  // a block of several groups may hold more than there are
  if (kAhead && first < a.L) fetch();
  float gw[NI][VEC], sw[NI][VEC];
  load_coef<T, VEC, NI, SHIFT>(a.wpost, a.gate ? a.gate + b * a.C : nullptr, a.gate ? 0.0f : 1.0f, cols, gw);
  load_coef<T, VEC, NI, SHIFT>(a.wpre, a.scale ? a.scale + b * a.C : nullptr, 1.0f, cols, sw);
  float a0[NI][VEC], a1[NI][VEC], a2[NI][VEC];
#pragma unroll
  for (int i = 0; i < NI; ++i)
#pragma unroll
    for (int e = 0; e < VEC; ++e) {
      a0[i][e] = a1[i][e] = a2[i][e] = 0.0f;
      gw[i][e] *= a.rho;
    }
#pragma unroll 1
  for (int64_t l = first; l < a.L; l += a.groups) {
    const int64_t r = b * a.L + l;
    float n[NI][VEC], m[NI][VEC], d[NI][VEC], dzv[NI][VEC];
    if (!kAhead) fetch();
    ry.get(m, cols);
    rx.get(n, cols);
    const float4 s4 = st;
    if (has_h) rh.get(d, cols);
    if (has_z) rz.get(dzv, cols);
    if (kAhead && l + a.groups < a.L) fetch();
#pragma unroll
    for (int i = 0; i < NI; ++i)
#pragma unroll
      for (int e = 0; e < VEC; ++e) {
        m[i][e] = (m[i][e] - s4.x) * s4.y;
        n[i][e] = (fmaf(m[i][e], gw[i][e], n[i][e]) - s4.z) * s4.w;
      }
    if (has_h) {
      // columns past C hold d = 0 (and a coefficient of 0), whatever n is there
      float2 s = make_float2(0.0f, 0.0f);
#pragma unroll
      for (int i = 0; i < NI; ++i)
#pragma unroll
        for (int e = 0; e < VEC; ++e) {
          a0[i][e] += d[i][e];
          a1[i][e] = fmaf(d[i][e], n[i][e], a1[i][e]);
          d[i][e] *= sw[i][e];
          s.x += d[i][e];
          s.y = fmaf(d[i][e], n[i][e], s.y);
        }
      s = sum(s);
      const float mean = a.pre == kLayer ? s.x * inv_c : 0.0f, dot = s.y * inv_c;
#pragma unroll
      for (int i = 0; i < NI; ++i)
#pragma unroll
        for (int e = 0; e < VEC; ++e) d[i][e] = s4.w * (d[i][e] - mean - n[i][e] * dot);
    } else {
#pragma unroll
      for (int i = 0; i < NI; ++i)
#pragma unroll
        for (int e = 0; e < VEC; ++e) d[i][e] = 0.0f;
    }
    if (has_z) {
#pragma unroll
      for (int i = 0; i < NI; ++i)
#pragma unroll
        for (int e = 0; e < VEC; ++e) d[i][e] += dzv[i][e];
    }
    store_row<T, VEC, NI, SHIFT>(static_cast<T*>(a.out0) + r * a.C, cols, d);
    // gw is 0 past C: those columns stay out of the sums, and a2 there is never stored
    float2 s = make_float2(0.0f, 0.0f);
#pragma unroll
    for (int i = 0; i < NI; ++i)
#pragma unroll
      for (int e = 0; e < VEC; ++e) {
        a2[i][e] = fmaf(d[i][e], m[i][e], a2[i][e]);
        d[i][e] *= gw[i][e];
        s.x += d[i][e];
        s.y = fmaf(d[i][e], m[i][e], s.y);
      }
    if (a.post != kNone) {
      s = sum(s);
      const float mean = a.post == kLayer ? s.x * inv_c : 0.0f, dot = s.y * inv_c;
#pragma unroll
      for (int i = 0; i < NI; ++i)
#pragma unroll
        for (int e = 0; e < VEC; ++e) d[i][e] = s4.y * (d[i][e] - mean - m[i][e] * dot);
    }
    store_row<T, VEC, NI, SHIFT>(static_cast<T*>(a.out1) + r * a.C, cols, d);
  }
  if (a.part == nullptr || g >= a.groups) return;
  float* p = a.part + (b * a.groups + g) * 3 * a.C;
#pragma unroll
  for (int i = 0; i < NI; ++i) {
    const int c = cols.at(i);
#pragma unroll
    for (int e = 0; e < VEC; ++e)
      if (cols.has(i, e)) {
        p[c + e] = a0[i][e];
        p[a.C + c + e] = a1[i][e];
        p[2 * a.C + c + e] = a2[i][e];
      }
  }
}

struct ReduceArgs {
  const float *part, *gate, *scale, *wpre, *wpost;
  float *dgate, *dscale, *dshift, *dwpre, *dwpost;  // nullable
  int B, C, groups;
  float rho;
};

// 32 columns of one of the three sums (blockIdx.y) per block, 32 threads per column; partial rows
// added in a fixed order, four batch entries at a time so that their loads overlap.
__global__ void __launch_bounds__(1024) norm_gate_reduce_k(const ReduceArgs a) {
  constexpr int NB = 4;
  __shared__ float sm[NB][32][33];
  grid_release();
  grid_wait();
  const int c = blockIdx.x * 32 + threadIdx.x, y = threadIdx.y, q = blockIdx.y;
  float dw = 0.0f;
  for (int b0 = 0; b0 < a.B; b0 += NB) {
    float s[NB];
#pragma unroll
    for (int u = 0; u < NB; ++u) {
      s[u] = 0.0f;
      if (c < a.C && b0 + u < a.B) {
        const float* p = a.part + ((int64_t)(b0 + u) * a.groups * 3 + q) * a.C + c;
#pragma unroll 8
        for (int g = y; g < a.groups; g += 32) s[u] += p[(int64_t)g * 3 * a.C];
      }
    }
#pragma unroll
    for (int u = 0; u < NB; ++u) sm[u][threadIdx.x][y] = s[u];
    __syncthreads();
    // warp u adds entry u's column sums
    float t = 0.0f;
    if (y < NB) {
#pragma unroll
      for (int j = 0; j < 32; ++j) t += sm[y][threadIdx.x][j];
      sm[y][threadIdx.x][32] = t;
    }
    __syncthreads();
    if (y == 0 && c < a.C) {
      for (int u = 0; u < NB && b0 + u < a.B; ++u) {
        const float v = sm[u][threadIdx.x][32];
        const int64_t bc = (int64_t)(b0 + u) * a.C + c;
        if (q == 0) {
          if (a.dshift) a.dshift[bc] = v;
        } else if (q == 1) {
          if (a.dscale) a.dscale[bc] = v * (a.wpre ? a.wpre[c] : 1.0f);
          dw = fmaf(1.0f + (a.scale ? a.scale[bc] : 0.0f), v, dw);
        } else {
          if (a.dgate) a.dgate[bc] = v * a.rho * (a.wpost ? a.wpost[c] : 1.0f);
          dw = fmaf(a.rho * (a.gate ? a.gate[bc] : 1.0f), v, dw);
        }
      }
    }
    __syncthreads();
  }
  if (y == 0 && c < a.C) {
    if (q == 1 && a.dwpre) a.dwpre[c] = dw;
    if (q == 2 && a.dwpost) a.dwpost[c] = dw;
  }
}

// How rows are accessed: by runs of four elements where every row of every tensor starts on a boundary of
// four (kWide); where the tensors start on one and their strides leave the same remainder, as contiguous
// ones of odd width do, by runs of four with a shift (kShifted); element by element otherwise (some sliced
// views).  6000 x 1999 in bf16, shifted and by elements: see above.
enum Access : int { kWide = 0, kShifted = 1, kSingle = 2 };

static Access access_of(const Args& a, int size) {
  bool wide = a.C % 4 == 0, shifted = a.C <= kMaxColumns - 3;
  auto look = [&](const void* p, int64_t sb, int64_t sl) {
    if (!p) return;
    if (reinterpret_cast<uintptr_t>(p) & (4 * size - 1)) wide = shifted = false;
    if (sb % 4 || sl % 4) wide = false;
    if ((sb - a.L * a.C) % 4 || (sl - a.C) % 4 || sb < 0 || sl < 0) shifted = false;
  };
  look(a.x, a.xb, a.xl);
  look(a.y, a.yb, a.yl);
  look(a.dz, a.zb, a.zl);
  look(a.dh, a.hb, a.hl);
  look(a.out0, a.L * a.C, a.C);
  look(a.out1, a.L * a.C, a.C);
  return wide ? kWide : (shifted ? kShifted : kSingle);
}

struct Shape {
  Access access;
  dim3 block;
  int per;  // elements per thread
};

static Shape shape_of(const Args& a, int size) {
  Shape s;
  s.access = access_of(a, size);
  const int C = a.C + (s.access == kShifted ? 3 : 0);
  s.per = C <= 512 ? 4 : (C <= 8 * kMaxThreads ? 8 : 16);
  const int t = ((C + s.per - 1) / s.per + 31) / 32 * 32;
  s.block = t == 32 ? dim3(32, 4) : dim3(t, 1);
  return s;
}

using Kernel = void (*)(Args);

template <class T, int VEC, int PER, bool BWD, bool SHIFT>
static Kernel kernel_for(const Shape& s) {
  constexpr int NI = PER / VEC;
  if (s.block.x * s.block.y > kFewThreads)
    return BWD ? norm_gate_bwd_k<T, VEC, NI, kMaxThreads, SHIFT> : norm_gate_k<T, VEC, NI, kMaxThreads, SHIFT>;
  return BWD ? norm_gate_bwd_k<T, VEC, NI, kFewThreads, SHIFT> : norm_gate_k<T, VEC, NI, kFewThreads, SHIFT>;
}

template <class T, int PER, bool BWD>
static Kernel kernel_for_access(const Shape& s) {
  if (s.access == kWide) return kernel_for<T, 4, PER, BWD, false>(s);
  if (s.access == kShifted) return kernel_for<T, 4, PER, BWD, true>(s);
  return kernel_for<T, 1, PER, BWD, false>(s);
}

template <class T, bool BWD>
static Kernel kernel_for_type(const Shape& s) {
  if (s.per == 4) return kernel_for_access<T, 4, BWD>(s);
  if (s.per == 8) return kernel_for_access<T, 8, BWD>(s);
  return kernel_for_access<T, 16, BWD>(s);
}

struct Plan {
  Kernel kernel;
  dim3 grid, block;
};

// The kernel of a call, and as many row groups per batch entry as fill the GPU once, one row per group at least
// (8193 x 1024 x 2: with twice as many, whose second half waits for the first, 46 us forward and 82 backward, with 1.5
// times as many 53 and more).  With a shift, a multiple of four, so that all rows of a group have the same one.
template <bool BWD>
static Plan plan_of(Args& a, int dtype) {
  const Shape s = shape_of(a, dtype_size(dtype));
  Plan p;
  p.kernel = dtype == kF32 ? kernel_for_type<float, BWD>(s)
                           : (dtype == kBF16 ? kernel_for_type<__nv_bfloat16, BWD>(s) : kernel_for_type<__half, BWD>(s));
  p.block = s.block;
  const int threads = (int)(s.block.x * s.block.y);
  // resident blocks per SM, asked for once per kernel and block size
  static std::atomic<int> known[3][3][3][kMaxThreads / 32 + 1];
  std::atomic<int>& blocks = known[dtype][s.access][s.per / 8][threads / 32];
  int n = blocks.load(std::memory_order_relaxed);
  if (n == 0) {
    if (cudaOccupancyMaxActiveBlocksPerMultiprocessor(&n, p.kernel, threads, 0) != cudaSuccess || n < 1) n = 1;
    blocks.store(n, std::memory_order_relaxed);
  }
  const int64_t want = ((int64_t)sm_count() * n * s.block.y + a.B - 1) / a.B;
  a.groups = (int)(want < a.L ? want : a.L);
  if (s.access == kShifted && a.groups < a.L) a.groups = a.groups < 4 ? 4 : a.groups / 4 * 4;
  p.grid = dim3((a.groups + s.block.y - 1) / s.block.y, a.B);
  return p;
}

static void launch(const Args& a, const Plan& p, cudaStream_t stream) {
  LaunchScope scope(kKElementwise, stream);
  p.kernel<<<p.grid, p.block, 0, stream>>>(a);
}

// whether a tensor's pointer is not a multiple of its element's size
static bool misaligned(const void* p, int size) { return reinterpret_cast<uintptr_t>(p) & (size - 1); }

static int check(const Args& a, int dtype) {
  if (a.B <= 0 || a.B > 65535 || a.L <= 0 || a.C <= 0 || a.C > kMaxColumns) return kBadDims;
  if (dtype < kF32 || dtype > kF16 || a.pre < kNone || a.pre > kRms || a.post < kNone || a.post > kRms)
    return kBadRange;
  if ((a.scale == nullptr) != (a.shift == nullptr)) return kNullPointer;
  if (a.pre == kNone && (a.scale || a.wpre)) return kBadRange;
  for (const void* p : {a.x, a.y, a.dz, a.dh, static_cast<const void*>(a.out0), static_cast<const void*>(a.out1)})
    if (misaligned(p, dtype_size(dtype))) return kBadAlignment;
  for (const float* p : {a.gate, a.scale, a.shift, a.wpre, a.wpost})
    if (misaligned(p, 4)) return kBadAlignment;
  if (misaligned(a.stats, 16)) return kBadAlignment;
  return kOk;
}

}  // namespace ng
}  // namespace tsb

extern "C" {

int triposplat_b200_norm_gate(const void* x, const void* y, const int64_t* strides, const float* gate,
                              const float* scale, const float* shift, const float* pre_weight,
                              const float* post_weight, void* z, void* h, float* stats, int dtype,
                              int B, int64_t L, int C, int pre, int post, float residual_scale,
                              float eps) {
  using namespace tsb;
  if (!x || !y || !strides || !z || !stats || (pre != ng::kNone && !h)) return kNullPointer;
  ng::Args a{};
  a.x = x; a.y = y;
  a.xb = strides[0]; a.xl = strides[1]; a.yb = strides[2]; a.yl = strides[3];
  a.gate = gate; a.scale = scale; a.shift = shift; a.wpre = pre_weight; a.wpost = post_weight;
  a.out0 = z; a.out1 = pre == ng::kNone ? nullptr : h; a.stats = stats;
  a.L = L; a.B = B; a.C = C; a.pre = pre; a.post = post; a.rho = residual_scale; a.eps = eps;
  int st = ng::check(a, dtype);
  if (st != kOk) return st;
  st = entry_check();
  if (st != kOk) return st;
  for (const void* p : {x, y, static_cast<const void*>(z), static_cast<const void*>(a.out1),
                        static_cast<const void*>(stats), static_cast<const void*>(gate),
                        static_cast<const void*>(scale), static_cast<const void*>(shift),
                        static_cast<const void*>(pre_weight), static_cast<const void*>(post_weight)})
    if (p && !is_device_pointer(p)) return kNotDevicePointer;
  const ng::Plan plan = ng::plan_of<false>(a, dtype);
  ng::launch(a, plan, current_stream());
  return launch_status();
}

int triposplat_b200_norm_gate_backward(const void* dz, const void* dh, const void* x, const void* y,
                                       const int64_t* strides, const float* stats, const float* gate,
                                       const float* scale, const float* pre_weight,
                                       const float* post_weight, void* dx, void* dy, float* dgate,
                                       float* dscale, float* dshift, float* dpre_weight,
                                       float* dpost_weight, int dtype, int B, int64_t L, int C, int pre,
                                       int post, float residual_scale) {
  using namespace tsb;
  if (!x || !y || !strides || !stats || !dx || !dy || (!dz && !dh)) return kNullPointer;
  ng::Args a{};
  a.x = x; a.y = y; a.dz = dz; a.dh = dh;
  a.xb = strides[0]; a.xl = strides[1]; a.yb = strides[2]; a.yl = strides[3];
  a.zb = strides[4]; a.zl = strides[5]; a.hb = strides[6]; a.hl = strides[7];
  a.gate = gate; a.scale = scale; a.shift = scale; a.wpre = pre_weight; a.wpost = post_weight;
  a.out0 = dx; a.out1 = dy; a.stats = const_cast<float*>(stats);
  a.L = L; a.B = B; a.C = C; a.pre = pre; a.post = post; a.rho = residual_scale;
  int st = ng::check(a, dtype);
  if (st != kOk) return st;
  if (pre == ng::kNone && dh) return kBadRange;
  st = entry_check();
  if (st != kOk) return st;
  for (const void* p : {dz, dh, x, y, static_cast<const void*>(stats), static_cast<const void*>(gate),
                        static_cast<const void*>(scale), static_cast<const void*>(pre_weight),
                        static_cast<const void*>(post_weight), static_cast<const void*>(dx),
                        static_cast<const void*>(dy), static_cast<const void*>(dgate),
                        static_cast<const void*>(dscale), static_cast<const void*>(dshift),
                        static_cast<const void*>(dpre_weight), static_cast<const void*>(dpost_weight)})
    if (p && !is_device_pointer(p)) return kNotDevicePointer;
  cudaStream_t stream = current_stream();
  const ng::Plan plan = ng::plan_of<true>(a, dtype);
  const bool sums = dgate || dscale || dshift || dpre_weight || dpost_weight;
  if (sums) {
    a.part = static_cast<float*>(workspace((size_t)B * a.groups * 3 * C * sizeof(float), stream));
    if (!a.part) return kWorkspace;
  }
  ng::launch(a, plan, stream);
  if (sums) {
    const ng::ReduceArgs ra{a.part, gate, scale, pre_weight, post_weight, dgate, dscale, dshift, dpre_weight,
                            dpost_weight, B, C, a.groups, residual_scale};
    LaunchScope scope(kKElementwise, stream);
    launch_chained(ng::norm_gate_reduce_k, dim3((C + 31) / 32, 3), dim3(32, 32), 0, stream, ra);
  }
  return launch_status();
}

}  // extern "C"
