// Rotary positions with several axes (a grid's or a video's), from position numbers, with the
// per-head norm the flow model puts after the rotation:
//   r = R(pos) x ;  y = r  or  y = r * sqrt(D) / max(|r|, 1e-12) * gamma[h]
// Pair p of axis a turns by pos[a] * inv_freq[p].  A pair is (2p, 2p + 1) ("interleaved") or
// (p, P + p) ("halves", P pairs in all); elements past 2P pass unrotated.
// Backward, with s = sqrt(D), n = |r|, g = dy * gamma:
//   dr = s/n (g - r (r . g) / n^2)  where n > 1e-12, s/1e-12 g otherwise (no norm: dr = dy)
//   dx = R(-pos) dr ;  dgamma[h] = sum over tokens of dy * r * s / max(n, 1e-12)
//
// Angles are formed and reduced to [-pi, pi] in fp64 (position numbers of any size keep
// their accuracy; a pair and token costs one, all heads share it), sine and cosine in fp32.
//
// Bound by HBM: x is read and y written once.  A head's vector belongs to a group of 1 to 32
// lanes, VEC pairs (two 16-byte accesses) each; the groups of a block take different heads of
// one token (adjacent in memory) and, with few heads, several tokens.  A block walks tiles of a few
// tokens: it issues the tile's loads, then its threads put the tokens' cosines and sines into
// shared memory (two buffers, one barrier per tile), then each group turns its vectors.  A group
// keeps its head: gamma stays in registers, and so does its part of dgamma, over all tiles of
// the block; a second kernel adds the blocks' partial rows in a fixed order (no atomics).
#include <stdint.h>

#include <initializer_list>

#include "common.cuh"
#include "runtime.h"
#include "vecio.cuh"

namespace tsb {
namespace rope {

constexpr int kMaxAxes = 4;
constexpr int kMaxDim = 256;
constexpr int kThreads = 256;

enum PosType : int { kInt32 = 0, kInt64 = 1, kFloat = 2 };

struct Args {
  const void *x, *dy;
  void* y;                       // y, or dx
  const void* pos;
  const float *inv_freq, *gamma;
  float* part;                   // [gridDim.x * token_groups, H, D] partial dgamma
  int64_t xb, xl, xh, db, dl, dh, yb, yl, yh;  // element strides (batch, token, head)
  int64_t pos_batch;             // elements between batch entries' positions (0: shared)
  int64_t L;
  int H, D, P, axes, pos_type, halves;
  int ends[kMaxAxes];            // first pair past each axis
  float sq;                      // sqrt(D)
  int B, lanes;                  // lanes per vector (a power of two)
  int heads, token_groups;       // heads and token groups of a block
  int64_t tiles;                 // tiles per batch entry
};

__device__ __forceinline__ double position(const Args& a, int64_t i) {
  if (a.pos_type == kInt32) return (double)static_cast<const int*>(a.pos)[i];
  if (a.pos_type == kInt64) return (double)static_cast<const int64_t*>(a.pos)[i];
  return (double)static_cast<const float*>(a.pos)[i];
}

// cosine and sine of pos * f: the product and its reduction by 2 pi in fp64, the reduced
// angle's low part put back to first order
__device__ __forceinline__ float2 turn_of(double pos, float f) {
  const double t = pos * (double)f;
  const double k = rint(t * 0.15915494309189533577);  // 1 / (2 pi)
  const double red = fma(-k, 2.4492935982947064e-16, fma(-k, 6.283185307179586, t));
  const float hi = (float)red, lo = (float)(red - (double)hi);
  float s, c;
  sincosf(hi, &s, &c);
  return make_float2(fmaf(-s, lo, c), fmaf(c, lo, s));
}

// VEC pairs of a head, as two runs of VEC elements.  Interleaved, the runs follow each other and
// pair i is (2i, 2i + 1) of both together; in halves, pair i is element i of each run.
template <class T, int VEC>
struct Slot {
  Pack<T, VEC> a, b;
  __device__ __forceinline__ void load(const T* p, int e0, int e1) {
    a = *reinterpret_cast<const Pack<T, VEC>*>(p + e0);
    b = *reinterpret_cast<const Pack<T, VEC>*>(p + e1);
  }
  __device__ __forceinline__ void store(T* p, int e0, int e1) const {
    *reinterpret_cast<Pack<T, VEC>*>(p + e0) = a;
    *reinterpret_cast<Pack<T, VEC>*>(p + e1) = b;
  }
  template <bool HALVES>
  __device__ __forceinline__ float2 pair(int i) const {
    if (HALVES) return make_float2(to_f32(a.v[i]), to_f32(b.v[i]));
    const int e = 2 * i;
    return e < VEC ? make_float2(to_f32(a.v[e]), to_f32(e + 1 < VEC ? a.v[(e + 1) % VEC] : b.v[0]))
                   : make_float2(to_f32(b.v[e - VEC]), to_f32(b.v[(e + 1 - VEC) % VEC]));
  }
  template <bool HALVES>
  __device__ __forceinline__ void put(int i, float2 v) {
    if (HALVES) {
      a.v[i] = from_f32<T>(v.x);
      b.v[i] = from_f32<T>(v.y);
      return;
    }
    const int e = 2 * i;
    if (e < VEC) {
      a.v[e] = from_f32<T>(v.x);
      if (e + 1 < VEC) a.v[(e + 1) % VEC] = from_f32<T>(v.y);
      else b.v[0] = from_f32<T>(v.y);
    } else {
      b.v[e - VEC] = from_f32<T>(v.x);
      b.v[(e + 1 - VEC) % VEC] = from_f32<T>(v.y);
    }
  }
};

// tokens that a group has in flight at once
template <bool BWD, int K>
__host__ __device__ constexpr int tokens_at_once() { return K > 1 ? 1 : (BWD ? 2 : 4); }

// K slots per lane, `lanes` apart.
template <class T, int VEC, int K, bool HALVES, bool BWD>
__global__ void __launch_bounds__(kThreads) axis_rope_k(const Args a) {
  constexpr int U = tokens_at_once<BWD, K>();
  extern __shared__ float2 table[];  // [2][tile tokens][D / 2]
  const int half = a.D / 2, tile_tokens = a.token_groups * U;
  const int lane = threadIdx.x & (a.lanes - 1), group = threadIdx.x / a.lanes;
  const int tg = group / a.heads, h = blockIdx.y * a.heads + group - tg * a.heads;
  const bool active = tg < a.token_groups && h < a.H;
  int e0[K], e1[K], p0[K];
  bool live[K];
  float2 g[K][VEC], acc[K][VEC];
#pragma unroll
  for (int k = 0; k < K; ++k) {
    p0[k] = (lane + k * a.lanes) * VEC;
    live[k] = active && p0[k] < half;
    const bool apart = HALVES && p0[k] < a.P;
    e0[k] = apart ? p0[k] : 2 * p0[k];
    e1[k] = apart ? a.P + p0[k] : e0[k] + VEC;
    Slot<float, VEC> gs;
#pragma unroll
    for (int i = 0; i < VEC; ++i) gs.a.v[i] = gs.b.v[i] = 1.0f;
    if (a.gamma && live[k]) {
      const float* gp = a.gamma + (int64_t)h * a.D;
#pragma unroll
      for (int i = 0; i < VEC; ++i) {
        gs.a.v[i] = __ldg(gp + e0[k] + i);
        gs.b.v[i] = __ldg(gp + e1[k] + i);
      }
    }
#pragma unroll
    for (int i = 0; i < VEC; ++i) {
      g[k][i] = gs.template pair<HALVES>(i);
      acc[k][i] = make_float2(0.0f, 0.0f);
    }
  }
  int turn = 0;
  const int64_t all = a.tiles * a.B;
#pragma unroll 1
  for (int64_t tile = blockIdx.x; tile < all; tile += gridDim.x) {
    const int64_t b = tile / a.tiles, l0 = (tile - b * a.tiles) * tile_tokens;
    Slot<T, VEC> xs[U][K], ds[U][K];
    // the tile's loads first: they fly while the table is made
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int64_t l = l0 + u * a.token_groups + tg;
#pragma unroll
      for (int k = 0; k < K; ++k)
        if (live[k] && l < a.L) {
          if (!BWD || a.gamma) xs[u][k].load(static_cast<const T*>(a.x) + b * a.xb + l * a.xl + h * a.xh, e0[k], e1[k]);
          if (BWD) ds[u][k].load(static_cast<const T*>(a.dy) + b * a.db + l * a.dl + h * a.dh, e0[k], e1[k]);
        }
    }
    float2* cs = table + turn * tile_tokens * half;
    turn ^= 1;
    for (int i = threadIdx.x; i < tile_tokens * half; i += kThreads) {
      const int t = i / half, p = i - t * half;
      float2 w = make_float2(1.0f, 0.0f);
      if (p < a.P && l0 + t < a.L) {
        int axis = 0;
        while (p >= a.ends[axis]) ++axis;
        w = turn_of(position(a, b * a.pos_batch + (l0 + t) * a.axes + axis), a.inv_freq[p]);
      }
      cs[i] = w;
    }
    __syncthreads();
    float2 r[U][K][VEC];
    float ss[U], dot[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      ss[u] = dot[u] = 0.0f;
#pragma unroll
      for (int k = 0; k < K; ++k)
#pragma unroll
        for (int i = 0; i < VEC; ++i) {
          r[u][k][i] = make_float2(0.0f, 0.0f);
          if (!live[k]) continue;
          if (!BWD || a.gamma) {
            const float2 w = cs[(u * a.token_groups + tg) * half + p0[k] + i];
            const float2 v = xs[u][k].template pair<HALVES>(i);
            r[u][k][i] = make_float2(v.x * w.x - v.y * w.y, v.x * w.y + v.y * w.x);
            ss[u] = fmaf(r[u][k][i].x, r[u][k][i].x, fmaf(r[u][k][i].y, r[u][k][i].y, ss[u]));
            if (BWD) {
              const float2 d = ds[u][k].template pair<HALVES>(i);
              dot[u] = fmaf(d.x * g[k][i].x, r[u][k][i].x, fmaf(d.y * g[k][i].y, r[u][k][i].y, dot[u]));
            }
          }
        }
    }
    float f[U], back[U];
#pragma unroll
    for (int u = 0; u < U; ++u) f[u] = 1.0f, back[u] = 0.0f;
    if (a.gamma) {
#pragma unroll 1
      for (int o = a.lanes / 2; o > 0; o >>= 1)
#pragma unroll
        for (int u = 0; u < U; ++u) {
          ss[u] += __shfl_xor_sync(0xffffffffu, ss[u], o);
          if (BWD) dot[u] += __shfl_xor_sync(0xffffffffu, dot[u], o);
        }
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const float n = sqrtf(ss[u]);
        f[u] = a.sq / fmaxf(n, 1.0e-12f);
        if (BWD) back[u] = n > 1.0e-12f ? dot[u] / (n * n) : 0.0f;
      }
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int64_t l = l0 + u * a.token_groups + tg;
#pragma unroll
      for (int k = 0; k < K; ++k) {
        if (!live[k] || l >= a.L) continue;
        Slot<T, VEC> o;
#pragma unroll
        for (int i = 0; i < VEC; ++i) {
          float2 v = r[u][k][i];
          if (BWD) {
            const float2 w = cs[(u * a.token_groups + tg) * half + p0[k] + i];
            const float2 d = ds[u][k].template pair<HALVES>(i);
            float2 e = d;
            if (a.gamma) {
              acc[k][i].x = fmaf(d.x, v.x * f[u], acc[k][i].x);
              acc[k][i].y = fmaf(d.y, v.y * f[u], acc[k][i].y);
              e.x = f[u] * fmaf(-v.x, back[u], d.x * g[k][i].x);
              e.y = f[u] * fmaf(-v.y, back[u], d.y * g[k][i].y);
            }
            v = make_float2(e.x * w.x + e.y * w.y, e.y * w.x - e.x * w.y);
          } else {
            v = make_float2(v.x * f[u] * g[k][i].x, v.y * f[u] * g[k][i].y);
          }
          o.template put<HALVES>(i, v);
        }
        o.store(static_cast<T*>(a.y) + b * a.yb + l * a.yl + h * a.yh, e0[k], e1[k]);
      }
    }
  }
  if (BWD && a.part) {
    float* q = a.part + (((int64_t)blockIdx.x * a.token_groups + tg) * a.H + h) * a.D;
#pragma unroll
    for (int k = 0; k < K; ++k) {
      if (!live[k]) continue;
      Slot<float, VEC> o;
#pragma unroll
      for (int i = 0; i < VEC; ++i) o.template put<HALVES>(i, acc[k][i]);
#pragma unroll
      for (int i = 0; i < VEC; ++i) {
        q[e0[k] + i] = o.a.v[i];
        q[e1[k] + i] = o.b.v[i];
      }
    }
  }
}

// dgamma[i] = sum of part[., i] over the partial rows, in a fixed order: 32 columns per block,
// 32 threads per column.
__global__ void __launch_bounds__(1024) column_sum_k(const float* __restrict__ part, int64_t rows, int cols,
                                                     float* __restrict__ out) {
  __shared__ float sm[32][33];
  const int c = blockIdx.x * 32 + threadIdx.x, y = threadIdx.y;
  float s = 0.0f;
  if (c < cols) {
#pragma unroll 8
    for (int64_t r = y; r < rows; r += 32) s += part[r * cols + c];
  }
  sm[threadIdx.x][y] = s;
  __syncthreads();
  if (y == 0 && c < cols) {
    float t = 0.0f;
#pragma unroll
    for (int j = 0; j < 32; ++j) t += sm[threadIdx.x][j];
    out[c] = t;
  }
}

static int fill(Args& a, int dtype, int pos_type, int B, int64_t L, int H, int D, const int* axis_pairs,
                int axes, int layout) {
  if (B <= 0 || B > 65535 || L <= 0 || H <= 0 || D <= 0 || D % 2 || D > kMaxDim || axes <= 0 || axes > kMaxAxes)
    return kBadDims;
  if (dtype < kF32 || dtype > kF16 || pos_type < kInt32 || pos_type > kFloat || layout < 0 || layout > 1)
    return kBadRange;
  int p = 0;
  for (int i = 0; i < axes; ++i) {
    if (axis_pairs[i] < 0 || axis_pairs[i] > D / 2) return kBadRange;
    p += axis_pairs[i];
    a.ends[i] = p;
  }
  if (p > D / 2) return kBadRange;
  if (pos_type == kInt64 && (reinterpret_cast<uintptr_t>(a.pos) & 7)) return kBadAlignment;
  a.L = L; a.H = H; a.D = D; a.P = p; a.axes = axes; a.pos_type = pos_type; a.halves = layout;
  a.sq = sqrtf((float)D);
  a.B = B;
  return kOk;
}

// whether a pointer is not a multiple of its element's size
static bool misaligned(int dtype, std::initializer_list<const void*> ps) {
  for (const void* p : ps)
    if (reinterpret_cast<uintptr_t>(p) & (dtype_size(dtype) - 1)) return true;
  return false;
}

// How a call's vectors are cut: VEC pairs per lane where every run of VEC elements lies on its own
// boundary (16 bytes for 4 of fp32 or 8 of a 16-bit type, 8 bytes for 4 of a 16-bit type), single pairs
// otherwise (odd widths, sliced views).
struct Plan {
  int vec, k, u;
  unsigned grid_x, grid_y;
};

static Plan plan_of(Args& a, int dtype, bool bwd) {
  const int half = a.D / 2;
  auto fits = [&](int vec) {
    const uintptr_t bytes = (uintptr_t)vec * dtype_size(dtype) - 1;
    if (half % vec || (a.halves && a.P % vec)) return false;
    if ((reinterpret_cast<uintptr_t>(a.x) | reinterpret_cast<uintptr_t>(a.dy) | reinterpret_cast<uintptr_t>(a.y)) & bytes)
      return false;
    for (int64_t s : {a.xb, a.xl, a.xh, a.db, a.dl, a.dh, a.yb, a.yl, a.yh})
      if (s % vec) return false;
    return true;
  };
  Plan p;
  p.vec = dtype != kF32 && fits(8) ? 8 : (fits(4) ? 4 : 1);
  const int slots = half / p.vec;
  a.lanes = 1;
  while (a.lanes < slots && a.lanes < 32) a.lanes *= 2;
  p.k = slots > a.lanes ? 4 : 1;
  p.u = p.k > 1 ? tokens_at_once<false, 4>() : (bwd ? tokens_at_once<true, 1>() : tokens_at_once<false, 1>());
  const int groups = kThreads / a.lanes;
  a.heads = a.H < groups ? a.H : groups;
  p.grid_y = (unsigned)((a.H + a.heads - 1) / a.heads);
  a.heads = (int)((a.H + p.grid_y - 1) / p.grid_y);  // even shares
  a.token_groups = groups / a.heads;
  // no more tokens at a time than there are, and a table of at most 32 KB
  const int64_t need = (a.L + p.u - 1) / p.u;
  const int room = 32768 / (int)(2 * p.u * half * sizeof(float2));
  if (a.token_groups > need) a.token_groups = (int)need;
  if (a.token_groups > room) a.token_groups = room > 0 ? room : 1;
  const int64_t tokens = (int64_t)a.token_groups * p.u;
  a.tiles = (a.L + tokens - 1) / tokens;
  const int64_t all = a.tiles * a.B;
  const int64_t cap = ((int64_t)sm_count() * (bwd ? 2 : 4) + p.grid_y - 1) / p.grid_y;
  p.grid_x = (unsigned)(all < cap ? all : cap);
  return p;
}

template <class T, int VEC, int K, bool BWD>
static void start(const Args& a, const Plan& p, cudaStream_t stream) {
  const size_t smem = (size_t)2 * a.token_groups * p.u * (a.D / 2) * sizeof(float2);
  const dim3 grid(p.grid_x, p.grid_y);
  if (a.halves) axis_rope_k<T, VEC, K, true, BWD><<<grid, kThreads, smem, stream>>>(a);
  else axis_rope_k<T, VEC, K, false, BWD><<<grid, kThreads, smem, stream>>>(a);
}

template <bool BWD>
static void launch(const Args& a, const Plan& p, int dtype, cudaStream_t stream) {
  LaunchScope scope(kKElementwise, stream);
  if (dtype == kF32) {
    if (p.vec == 4) start<float, 4, 1, BWD>(a, p, stream);
    else if (p.k == 1) start<float, 1, 1, BWD>(a, p, stream);
    else start<float, 1, 4, BWD>(a, p, stream);
  } else if (dtype == kBF16) {
    if (p.vec == 8) start<__nv_bfloat16, 8, 1, BWD>(a, p, stream);
    else if (p.vec == 4) start<__nv_bfloat16, 4, 1, BWD>(a, p, stream);
    else if (p.k == 1) start<__nv_bfloat16, 1, 1, BWD>(a, p, stream);
    else start<__nv_bfloat16, 1, 4, BWD>(a, p, stream);
  } else {
    if (p.vec == 8) start<__half, 8, 1, BWD>(a, p, stream);
    else if (p.vec == 4) start<__half, 4, 1, BWD>(a, p, stream);
    else if (p.k == 1) start<__half, 1, 1, BWD>(a, p, stream);
    else start<__half, 1, 4, BWD>(a, p, stream);
  }
}

}  // namespace rope
}  // namespace tsb

extern "C" {

int triposplat_b200_axis_rope(const void* x, const void* positions, const float* inv_freq,
                              const float* gamma, void* y, const int64_t* strides, int dtype,
                              int position_type, int64_t position_batch_stride, int B, int64_t L, int H,
                              int D, const int* axis_pairs, int axes, int layout) {
  using namespace tsb;
  if (!x || !positions || !inv_freq || !y || !strides || !axis_pairs) return kNullPointer;
  rope::Args a{};
  a.pos = positions;
  int st = rope::fill(a, dtype, position_type, B, L, H, D, axis_pairs, axes, layout);
  if (st != kOk) return st;
  if (rope::misaligned(dtype, {x, y}) || rope::misaligned(kF32, {inv_freq, gamma, positions})) return kBadAlignment;
  st = entry_check();
  if (st != kOk) return st;
  for (const void* p : {x, positions, static_cast<const void*>(inv_freq), static_cast<const void*>(gamma),
                        static_cast<const void*>(y)})
    if (p && !is_device_pointer(p)) return kNotDevicePointer;
  a.x = x; a.y = y; a.pos = positions; a.inv_freq = inv_freq; a.gamma = gamma;
  a.xb = strides[0]; a.xl = strides[1]; a.xh = strides[2];
  a.yb = strides[3]; a.yl = strides[4]; a.yh = strides[5];
  a.pos_batch = position_batch_stride;
  const rope::Plan plan = rope::plan_of(a, dtype, false);
  rope::launch<false>(a, plan, dtype, current_stream());
  return launch_status();
}

int triposplat_b200_axis_rope_backward(const void* dy, const void* x, const void* positions,
                                       const float* inv_freq, const float* gamma, void* dx, float* dgamma,
                                       const int64_t* strides, int dtype, int position_type,
                                       int64_t position_batch_stride, int B, int64_t L, int H, int D,
                                       const int* axis_pairs, int axes, int layout) {
  using namespace tsb;
  if (!dy || !positions || !inv_freq || !dx || !strides || !axis_pairs || (gamma && !x) || (dgamma && !gamma))
    return kNullPointer;
  rope::Args a{};
  a.pos = positions;
  int st = rope::fill(a, dtype, position_type, B, L, H, D, axis_pairs, axes, layout);
  if (st != kOk) return st;
  if ((int64_t)H * D > 2147483647) return kBadDims;
  if (rope::misaligned(dtype, {dy, x, dx}) || rope::misaligned(kF32, {inv_freq, gamma, positions, dgamma}))
    return kBadAlignment;
  st = entry_check();
  if (st != kOk) return st;
  for (const void* p : {dy, x, positions, static_cast<const void*>(inv_freq), static_cast<const void*>(gamma),
                        static_cast<const void*>(dx), static_cast<const void*>(dgamma)})
    if (p && !is_device_pointer(p)) return kNotDevicePointer;
  a.x = x; a.dy = dy; a.y = dx; a.pos = positions; a.inv_freq = inv_freq; a.gamma = gamma;
  a.db = strides[0]; a.dl = strides[1]; a.dh = strides[2];
  a.xb = strides[3]; a.xl = strides[4]; a.xh = strides[5];
  a.yb = strides[6]; a.yl = strides[7]; a.yh = strides[8];
  a.pos_batch = position_batch_stride;
  cudaStream_t stream = current_stream();
  const rope::Plan plan = rope::plan_of(a, dtype, true);
  const int64_t rows = (int64_t)plan.grid_x * a.token_groups;
  if (dgamma) {
    a.part = static_cast<float*>(workspace((size_t)rows * H * D * sizeof(float), stream));
    if (!a.part) return kWorkspace;
  }
  rope::launch<true>(a, plan, dtype, stream);
  if (dgamma) {
    LaunchScope scope(kKElementwise, stream);
    rope::column_sum_k<<<(H * D + 31) / 32, dim3(32, 32), 0, stream>>>(a.part, rows, H * D, dgamma);
  }
  return launch_status();
}

}  // extern "C"
