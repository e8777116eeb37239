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
// Bound by HBM: x is read and y written once.  A block takes 32 tokens of one batch entry:
// its threads first put the tokens' cosines and sines into shared memory, then each warp
// walks the heads, one head's vector per warp at a time.  dgamma: a warp keeps its head's
// sums in registers over the block's tokens and writes one partial row, a second kernel adds
// the partial rows in a fixed order (no atomics).
#include <stdint.h>

#include <initializer_list>

#include "common.cuh"
#include "runtime.h"
#include "vecio.cuh"

namespace tsb {
namespace rope {

constexpr int kMaxAxes = 4;
constexpr int kMaxDim = 256;
constexpr int kTokens = 32;   // tokens per block
constexpr int kThreads = 256;
constexpr int kPairsPerLane = kMaxDim / 2 / 32;

enum PosType : int { kInt32 = 0, kInt64 = 1, kFloat = 2 };

struct Args {
  const void *x, *dy;
  void* y;                       // y, or dx
  const void* pos;
  const float *inv_freq, *gamma;
  float* part;                   // [blocks, H, D] partial dgamma
  int64_t xb, xl, xh, db, dl, dh, yb, yl, yh;  // element strides (batch, token, head)
  int64_t pos_batch;             // elements between batch entries' positions (0: shared)
  int64_t L;
  int H, D, P, axes, pos_type, halves;
  int ends[kMaxAxes];            // first pair past each axis
  float sq;                      // sqrt(D)
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

__device__ __forceinline__ void pair_index(const Args& a, int p, int& i0, int& i1) {
  if (a.halves && p < a.P) {
    i0 = p;
    i1 = a.P + p;
  } else {
    i0 = 2 * p;
    i1 = 2 * p + 1;
  }
}

template <class T, bool BWD>
__global__ void __launch_bounds__(kThreads) axis_rope_k(const Args a) {
  extern __shared__ float2 cs[];  // [kTokens][P]
  const int64_t l0 = (int64_t)blockIdx.x * kTokens;
  const int b = blockIdx.y;
  const int tokens = (int)min((int64_t)kTokens, a.L - l0);
  for (int i = threadIdx.x; i < tokens * a.P; i += kThreads) {
    const int t = i / a.P, p = i - t * a.P;
    int axis = 0;
    while (p >= a.ends[axis]) ++axis;
    cs[i] = turn_of(position(a, b * a.pos_batch + (l0 + t) * a.axes + axis), a.inv_freq[p]);
  }
  __syncthreads();
  const int lane = threadIdx.x & 31, half = a.D / 2;
  for (int h = threadIdx.x >> 5; h < a.H; h += kThreads / 32) {
    float2 g[kPairsPerLane], acc[kPairsPerLane];
#pragma unroll
    for (int k = 0; k < kPairsPerLane; ++k) {
      g[k] = make_float2(1.0f, 1.0f);
      acc[k] = make_float2(0.0f, 0.0f);
      const int p = lane + 32 * k;
      if (a.gamma && p < half) {
        int i0, i1;
        pair_index(a, p, i0, i1);
        g[k] = make_float2(a.gamma[(int64_t)h * a.D + i0], a.gamma[(int64_t)h * a.D + i1]);
      }
    }
#pragma unroll 1
    for (int t = 0; t < tokens; ++t) {
      const T* x = static_cast<const T*>(a.x) + b * a.xb + (l0 + t) * a.xl + h * a.xh;
      T* y = static_cast<T*>(a.y) + b * a.yb + (l0 + t) * a.yl + h * a.yh;
      const T* d = BWD ? static_cast<const T*>(a.dy) + b * a.db + (l0 + t) * a.dl + h * a.dh : nullptr;
      float2 r[kPairsPerLane], w[kPairsPerLane], dv[kPairsPerLane];
      float ss = 0.0f, dot = 0.0f;
#pragma unroll
      for (int k = 0; k < kPairsPerLane; ++k) {
        r[k] = dv[k] = make_float2(0.0f, 0.0f);
        w[k] = make_float2(1.0f, 0.0f);
        const int p = lane + 32 * k;
        if (p >= half) continue;
        int i0, i1;
        pair_index(a, p, i0, i1);
        if (p < a.P) w[k] = cs[t * a.P + p];
        if (BWD) dv[k] = make_float2(to_f32(d[i0]), to_f32(d[i1]));
        if (!BWD || a.gamma) {
          const float2 v = make_float2(to_f32(x[i0]), to_f32(x[i1]));
          r[k] = make_float2(v.x * w[k].x - v.y * w[k].y, v.x * w[k].y + v.y * w[k].x);
          ss = fmaf(r[k].x, r[k].x, fmaf(r[k].y, r[k].y, ss));
        }
        if (BWD && a.gamma)
          dot = fmaf(dv[k].x * g[k].x, r[k].x, fmaf(dv[k].y * g[k].y, r[k].y, dot));
      }
      float f = 1.0f, back = 0.0f;
      if (a.gamma) {
        const float n = sqrtf(warp_sum(ss));
        f = a.sq / fmaxf(n, 1.0e-12f);
        if (BWD) {
          dot = warp_sum(dot);
          back = n > 1.0e-12f ? dot / (n * n) : 0.0f;
        }
      }
#pragma unroll
      for (int k = 0; k < kPairsPerLane; ++k) {
        const int p = lane + 32 * k;
        if (p >= half) continue;
        int i0, i1;
        pair_index(a, p, i0, i1);
        float2 o;
        if (BWD) {
          float2 e = dv[k];
          if (a.gamma) {
            acc[k].x = fmaf(dv[k].x, r[k].x * f, acc[k].x);
            acc[k].y = fmaf(dv[k].y, r[k].y * f, acc[k].y);
            e.x = f * fmaf(-r[k].x, back, dv[k].x * g[k].x);
            e.y = f * fmaf(-r[k].y, back, dv[k].y * g[k].y);
          }
          o = make_float2(e.x * w[k].x + e.y * w[k].y, e.y * w[k].x - e.x * w[k].y);
        } else {
          o = make_float2(r[k].x * f * g[k].x, r[k].y * f * g[k].y);
        }
        y[i0] = from_f32<T>(o.x);
        y[i1] = from_f32<T>(o.y);
      }
    }
    if (BWD && a.part) {
      float* q = a.part + (((int64_t)b * gridDim.x + blockIdx.x) * a.H + h) * a.D;
#pragma unroll
      for (int k = 0; k < kPairsPerLane; ++k) {
        const int p = lane + 32 * k;
        if (p >= half) continue;
        int i0, i1;
        pair_index(a, p, i0, i1);
        q[i0] = acc[k].x;
        q[i1] = acc[k].y;
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
  if ((L + kTokens - 1) / kTokens > 2147483647) return kBadDims;
  if (pos_type == kInt64 && (reinterpret_cast<uintptr_t>(a.pos) & 7)) return kBadAlignment;
  a.L = L; a.H = H; a.D = D; a.P = p; a.axes = axes; a.pos_type = pos_type; a.halves = layout;
  a.sq = sqrtf((float)D);
  return kOk;
}

// whether a pointer is not a multiple of its element's size
static bool misaligned(int dtype, std::initializer_list<const void*> ps) {
  for (const void* p : ps)
    if (reinterpret_cast<uintptr_t>(p) & (dtype_size(dtype) - 1)) return true;
  return false;
}

template <bool BWD>
static void launch(const Args& a, int dtype, int B, cudaStream_t stream) {
  const dim3 grid((unsigned)((a.L + kTokens - 1) / kTokens), B);
  const size_t smem = (size_t)kTokens * a.P * sizeof(float2);
  LaunchScope scope(kKElementwise, stream);
  if (dtype == kF32) axis_rope_k<float, BWD><<<grid, kThreads, smem, stream>>>(a);
  else if (dtype == kBF16) axis_rope_k<__nv_bfloat16, BWD><<<grid, kThreads, smem, stream>>>(a);
  else axis_rope_k<__half, BWD><<<grid, kThreads, smem, stream>>>(a);
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
  rope::launch<false>(a, dtype, B, current_stream());
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
  const int64_t rows = (L + rope::kTokens - 1) / rope::kTokens * B;
  if (dgamma) {
    a.part = static_cast<float*>(workspace((size_t)rows * H * D * sizeof(float), stream));
    if (!a.part) return kWorkspace;
  }
  rope::launch<true>(a, dtype, B, stream);
  if (dgamma) {
    LaunchScope scope(kKElementwise, stream);
    rope::column_sum_k<<<(H * D + 31) / 32, dim3(32, 32), 0, stream>>>(a.part, rows, H * D, dgamma);
  }
  return launch_status();
}

}  // extern "C"
