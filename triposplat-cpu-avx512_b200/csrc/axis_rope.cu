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
// lanes, four pairs (two accesses of 16 bytes, or 8 of a 16-bit type; eight pairs of one from 96
// dimensions on) each; the groups of a block
// take different heads of one token (adjacent in memory) and, with few heads, several tokens.  A block
// walks chunks of tokens: its threads put the chunk's cosines and sines into shared memory once,
// then each group walks its head's vectors with the next step's loads in flight.  gamma stays in
// registers, and so does a group's part of dgamma, over all chunks of the block; a second kernel
// adds the blocks' partial rows in a fixed order (no atomics).
//
// Measured, 8193 x 2 x 32 x 64 in fp32 with the norm: forward 49 us (5.5 TB/s), backward 71 us (5.7) and 4 for
// dgamma.  5985 x 24 x 128 in bf16 without it: 17.6 us each way (4.2 TB/s), half the bytes for the same
// instructions.
#include <stdint.h>

#include <initializer_list>

#include "common.cuh"
#include "runtime.h"
#include "vecio.cuh"

namespace tsb {
namespace rope {

constexpr int kMaxAxes = 4;
constexpr int kMaxDim = 256;
constexpr int kThreads = 384;  // most per block

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
  int steps;                     // steps of U * token_groups tokens in a chunk
  int64_t chunks;                // chunks per batch entry
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
// pair i is (2i, 2i + 1) of both together; in halves, pair i is element i of each run.  A single
// pair is the same either way and uses the second form.
template <int VEC>
struct Runs {
  float v[2][VEC];
  template <bool HALVES>
  __device__ __forceinline__ float2 pair(int i) const {
    if (HALVES) return make_float2(v[0][i], v[1][i]);
    return make_float2(v[2 * i / VEC][2 * i % VEC], v[(2 * i + 1) / VEC][(2 * i + 1) % VEC]);
  }
  template <bool HALVES>
  __device__ __forceinline__ void put(int i, float2 p) {
    if (HALVES) {
      v[0][i] = p.x;
      v[1][i] = p.y;
    } else {
      v[2 * i / VEC][2 * i % VEC] = p.x;
      v[(2 * i + 1) / VEC][(2 * i + 1) % VEC] = p.y;
    }
  }
  template <class T>
  __device__ __forceinline__ void store(T* p, int e0, int e1) const {
    store_vec<T, VEC>(p + e0, v[0]);
    store_vec<T, VEC>(p + e1, v[1]);
  }
};

// ... as they lie in memory
template <class T, int VEC>
struct Slot {
  Raw<T, VEC> a, b;
  __device__ __forceinline__ void load(const T* p, int e0, int e1) {
    a.load(p + e0);
    b.load(p + e1);
  }
  __device__ __forceinline__ Runs<VEC> get() const {
    Runs<VEC> r;
#pragma unroll
    for (int i = 0; i < VEC; ++i) {
      r.v[0][i] = a[i];
      r.v[1][i] = b[i];
    }
    return r;
  }
};

// tokens of one step of a group
template <bool BWD, int K>
__host__ __device__ constexpr int tokens_at_once() { return K > 1 || BWD ? 1 : 2; }

// K slots per lane, `lanes` apart.
template <class T, int VEC, int K, bool HALVES, bool BWD, bool NORM>
__global__ void __launch_bounds__(kThreads, K > 1 ? 1 : 2) axis_rope_k(const Args a) {
  constexpr int U = tokens_at_once<BWD, K>();
  // [chunk tokens][VEC][D / 2 / VEC]: the lanes of a vector read neighbouring entries
  extern __shared__ float2 cs[];
  if (BWD) grid_release();
  const int half = a.D / 2, step_tokens = a.token_groups * U, chunk_tokens = step_tokens * a.steps;
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
    const bool apart = a.halves && p0[k] < a.P;
    e0[k] = apart ? p0[k] : 2 * p0[k];
    e1[k] = apart ? a.P + p0[k] : e0[k] + VEC;
    if (NORM) {
      Runs<VEC> gs;
#pragma unroll
      for (int i = 0; i < VEC; ++i) {
        gs.v[0][i] = live[k] ? __ldg(a.gamma + (int64_t)h * a.D + e0[k] + i) : 0.0f;
        gs.v[1][i] = live[k] ? __ldg(a.gamma + (int64_t)h * a.D + e1[k] + i) : 0.0f;
      }
#pragma unroll
      for (int i = 0; i < VEC; ++i) {
        g[k][i] = gs.template pair<HALVES>(i);
        acc[k][i] = make_float2(0.0f, 0.0f);
      }
    }
  }
  const int slots = half / VEC;
  const int64_t all = a.chunks * a.B;
#pragma unroll 1
  for (int64_t chunk = blockIdx.x; chunk < all; chunk += gridDim.x) {
    const int64_t b = chunk / a.chunks, l0 = (chunk - b * a.chunks) * chunk_tokens;
    const int tokens = (int)min((int64_t)chunk_tokens, a.L - l0);
    const T* x = static_cast<const T*>(a.x) + h * a.xh + b * a.xb + (l0 + tg) * a.xl;
    const T* dy = static_cast<const T*>(a.dy) + h * a.dh + b * a.db + (l0 + tg) * a.dl;
    T* y = static_cast<T*>(a.y) + h * a.yh + b * a.yb + (l0 + tg) * a.yl;
    const int64_t dxl = a.token_groups * a.xl, ddl = a.token_groups * a.dl, dyl = a.token_groups * a.yl;
    Slot<T, VEC> xs[U][K], ds[U][K];
    // the next step's loads (nothing past the chunk's end)
    auto fetch = [&](int t) {
#pragma unroll
      for (int u = 0; u < U; ++u, t += a.token_groups, x += dxl, dy += ddl) {
#pragma unroll
        for (int k = 0; k < K; ++k)
          if (live[k] && t < tokens) {
            if (!BWD || NORM) xs[u][k].load(x, e0[k], e1[k]);
            if (BWD) ds[u][k].load(dy, e0[k], e1[k]);
          }
      }
    };
    fetch(tg);  // in flight while the table is made
    for (int i = threadIdx.x; i < tokens * half; i += blockDim.x) {
      const int t = i / half, q = i - t * half, p = q % slots * VEC + q / slots;
      float2 w = make_float2(1.0f, 0.0f);
      if (p < a.P) {
        int axis = 0;
        while (p >= a.ends[axis]) ++axis;
        w = turn_of(position(a, b * a.pos_batch + (l0 + t) * a.axes + axis), a.inv_freq[p]);
      }
      cs[i] = w;
    }
    __syncthreads();
#pragma unroll 1
    for (int t0 = 0; t0 < tokens; t0 += step_tokens) {
      Slot<T, VEC> xc[U][K], dc[U][K];
#pragma unroll
      for (int u = 0; u < U; ++u)
#pragma unroll
        for (int k = 0; k < K; ++k) {
          if (!BWD || NORM) xc[u][k] = xs[u][k];
          if (BWD) dc[u][k] = ds[u][k];
        }
      fetch(t0 + step_tokens + tg);
#pragma unroll
      for (int u = 0; u < U; ++u, y += dyl) {
        const int t = t0 + u * a.token_groups + tg;
        const bool here = t < tokens;
        const float2* w = cs + (here ? t : 0) * half + lane;
        Runs<VEC> xr[K], dr[K];
#pragma unroll
        for (int k = 0; k < K; ++k) {
          if (!BWD || NORM) xr[k] = xc[u][k].get();
          if (BWD) dr[k] = dc[u][k].get();
        }
        float2 r[K][VEC];
        float ss = 0.0f, dot = 0.0f;
        if (!BWD || NORM) {
#pragma unroll
          for (int k = 0; k < K; ++k)
#pragma unroll
            for (int i = 0; i < VEC; ++i) {
              r[k][i] = make_float2(0.0f, 0.0f);
              if (!live[k] || !here) continue;
              const float2 c = w[i * slots + k * a.lanes], v = xr[k].template pair<HALVES>(i);
              r[k][i] = make_float2(v.x * c.x - v.y * c.y, v.x * c.y + v.y * c.x);
              if (NORM) {
                ss = fmaf(r[k][i].x, r[k][i].x, fmaf(r[k][i].y, r[k][i].y, ss));
                if (BWD) {
                  const float2 d = dr[k].template pair<HALVES>(i);
                  dot = fmaf(d.x * g[k][i].x, r[k][i].x, fmaf(d.y * g[k][i].y, r[k][i].y, dot));
                }
              }
            }
        }
        float f = 1.0f, back = 0.0f;
        if (NORM) {
          for (int o = a.lanes / 2; o > 0; o >>= 1) {
            ss += __shfl_xor_sync(0xffffffffu, ss, o);
            if (BWD) dot += __shfl_xor_sync(0xffffffffu, dot, o);
          }
          const float n = sqrtf(ss);
          f = a.sq / fmaxf(n, 1.0e-12f);
          if (BWD) back = n > 1.0e-12f ? dot / (n * n) : 0.0f;
        }
#pragma unroll
        for (int k = 0; k < K; ++k) {
          if (!live[k] || !here) continue;
          Runs<VEC> o;
#pragma unroll
          for (int i = 0; i < VEC; ++i) {
            float2 v;
            if (BWD) {
              const float2 d = dr[k].template pair<HALVES>(i), c = w[i * slots + k * a.lanes];
              float2 e = d;
              if (NORM) {
                const float2 q = r[k][i];
                acc[k][i].x = fmaf(d.x, q.x * f, acc[k][i].x);
                acc[k][i].y = fmaf(d.y, q.y * f, acc[k][i].y);
                e.x = f * fmaf(-q.x, back, d.x * g[k][i].x);
                e.y = f * fmaf(-q.y, back, d.y * g[k][i].y);
              }
              v = make_float2(e.x * c.x + e.y * c.y, e.y * c.x - e.x * c.y);
            } else {
              v = r[k][i];
              if (NORM) v = make_float2(v.x * f * g[k][i].x, v.y * f * g[k][i].y);
            }
            o.template put<HALVES>(i, v);
          }
          o.store(y, e0[k], e1[k]);
        }
      }
    }
    __syncthreads();  // the table is free for the next chunk
  }
  if (BWD && NORM && a.part) {
    float* q = a.part + (((int64_t)blockIdx.x * a.token_groups + tg) * a.H + h) * a.D;
#pragma unroll
    for (int k = 0; k < K; ++k) {
      if (!live[k]) continue;
      Runs<VEC> o;
#pragma unroll
      for (int i = 0; i < VEC; ++i) o.template put<HALVES>(i, acc[k][i]);
#pragma unroll
      for (int i = 0; i < VEC; ++i) {
        q[e0[k] + i] = o.v[0][i];
        q[e1[k] + i] = o.v[1][i];
      }
    }
  }
}

// dgamma[i] = sum of part[., i] over the partial rows, in a fixed order: 32 columns per block,
// 32 threads per column.
__global__ void __launch_bounds__(1024) column_sum_k(const float* __restrict__ part, int64_t rows, int cols,
                                                     float* __restrict__ out) {
  __shared__ float sm[32][33];
  grid_release();
  grid_wait();
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

// How a call's vectors are cut: four pairs per lane where every run of as many elements lies on its own boundary,
// single pairs otherwise (odd widths, sliced views).  Eight pairs of a 16-bit type (16-byte accesses) from 96 dimensions
// on, but not for the backward pass of the norm, whose registers they do not leave enough of: 4000 x 2 x 16 x 96 in bf16,
// eight and four: 13.4 and 16.0 us forward, 15.1 and 17.6 backward, with the norm 20.7 and 23.5 forward but 47 and
// 31 backward; 4000 x 2 x 16 x 64: 8.5 and 8.6, 10.5 and 9.7, 14.3 and 13.0, 29 and 19.
struct Plan {
  int vec, k, u;
  unsigned grid_x, grid_y, threads;
  size_t smem;
};

static Plan plan_of(Args& a, int dtype, bool bwd) {
  const int half = a.D / 2, size = dtype_size(dtype);
  const uintptr_t starts =
      reinterpret_cast<uintptr_t>(a.x) | reinterpret_cast<uintptr_t>(a.dy) | reinterpret_cast<uintptr_t>(a.y);
  Plan p;
  for (p.vec = size == 2 && half >= 48 && !(bwd && a.gamma) ? 8 : 4; p.vec > 1; p.vec = p.vec > 4 ? 4 : 1) {
    bool fits = half % p.vec == 0 && !(a.halves && a.P % p.vec) && !(starts & (p.vec * size - 1));
    for (int64_t s : {a.xb, a.xl, a.xh, a.db, a.dl, a.dh, a.yb, a.yl, a.yh})
      if (s % p.vec) fits = false;
    if (fits) break;
  }
  const int slots = half / p.vec;
  a.lanes = 1;
  while (a.lanes < slots && a.lanes < 32) a.lanes *= 2;
  p.k = slots > a.lanes ? 4 : 1;
  p.u = p.k > 1 || bwd ? tokens_at_once<true, 4>() : tokens_at_once<false, 1>();
  const int groups = kThreads / a.lanes;
  a.heads = a.H < groups ? a.H : groups;
  p.grid_y = (unsigned)((a.H + a.heads - 1) / a.heads);
  a.heads = (int)((a.H + p.grid_y - 1) / p.grid_y);  // even shares
  // no more tokens at a time than there are, and a table of at most 32 KB
  const int room = 32768 / (int)(half * sizeof(float2));
  a.token_groups = groups / a.heads;
  if (a.token_groups > (a.L + p.u - 1) / p.u) a.token_groups = (int)((a.L + p.u - 1) / p.u);
  if (a.token_groups > room / p.u) a.token_groups = room / p.u;
  const int step = a.token_groups * p.u;
  p.threads = (a.heads * a.token_groups * a.lanes + 31) / 32 * 32;
  // one chunk per block of a full GPU (some 768 threads per SM), within the table's room
  const int per_sm = 768 / (int)p.threads > 16 ? 16 : 768 / (int)p.threads;
  const int64_t blocks = ((int64_t)sm_count() * per_sm + p.grid_y - 1) / p.grid_y;
  const int64_t share = (a.L * a.B + blocks - 1) / blocks;
  int64_t steps = (share + step - 1) / step;
  if (steps > room / step) steps = room / step;
  a.steps = (int)steps;
  a.chunks = (a.L + steps * step - 1) / (steps * step);
  const int64_t all = a.chunks * a.B;
  p.grid_x = (unsigned)(all < blocks ? all : blocks);
  p.smem = (size_t)a.steps * step * half * sizeof(float2);
  return p;
}

template <class T, bool BWD, bool NORM>
static void start(const Args& a, const Plan& p, cudaStream_t st) {
  const dim3 grid(p.grid_x, p.grid_y);
  if constexpr (sizeof(T) == 2 && !(BWD && NORM)) {
    if (p.vec == 8) {
      if (a.halves) axis_rope_k<T, 8, 1, true, BWD, NORM><<<grid, p.threads, p.smem, st>>>(a);
      else axis_rope_k<T, 8, 1, false, BWD, NORM><<<grid, p.threads, p.smem, st>>>(a);
      return;
    }
  }
  if (p.vec == 4 && a.halves) axis_rope_k<T, 4, 1, true, BWD, NORM><<<grid, p.threads, p.smem, st>>>(a);
  else if (p.vec == 4) axis_rope_k<T, 4, 1, false, BWD, NORM><<<grid, p.threads, p.smem, st>>>(a);
  else if (p.k == 1) axis_rope_k<T, 1, 1, true, BWD, NORM><<<grid, p.threads, p.smem, st>>>(a);
  else axis_rope_k<T, 1, 4, true, BWD, NORM><<<grid, p.threads, p.smem, st>>>(a);
}

template <bool BWD>
static void launch(const Args& a, const Plan& p, int dtype, cudaStream_t st) {
  LaunchScope scope(kKElementwise, st);
  if (dtype == kF32) a.gamma ? start<float, BWD, true>(a, p, st) : start<float, BWD, false>(a, p, st);
  else if (dtype == kBF16)
    a.gamma ? start<__nv_bfloat16, BWD, true>(a, p, st) : start<__nv_bfloat16, BWD, false>(a, p, st);
  else a.gamma ? start<__half, BWD, true>(a, p, st) : start<__half, BWD, false>(a, p, st);
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
    launch_chained(rope::column_sum_k, dim3((H * D + 31) / 32), dim3(32, 32), 0, stream, a.part, rows, H * D, dgamma);
  }
  return launch_status();
}

}  // extern "C"
