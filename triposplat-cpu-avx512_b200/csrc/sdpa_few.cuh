// Attention of up to eight query rows per head (a pooled token, a decoded one), and of any small number of
// queries and keys in groups of four rows, forward and backward, in fp32 on the CUDA cores.  With so
// few rows the work is reading K and V once (and, backward, writing their gradients): the tensor-core
// path would first write both as fp16 pairs and read those back, and walk them with one held tile
// per head.  With several groups, each writes its part of dK and dV, joined like the shares of dQ.
//
// Four lanes per key, 16 of its 64 dimensions each; a score is 16 products per lane and two shuffles.
// A block takes a share of a head's keys, four warps of eight keys at a time.  Forward: each group
// of four lanes keeps a softmax of its own (integer reference m in log2 units, raised when a score
// passes it by more than 8, so that its factor is a power of two; l; 16 output values per row),
// joined over the warp by shuffles, over the block in shared memory, and over the shares of the keys by
// a last kernel in their order.  Backward: per key e and ds of every row give its dK, dV at once, dQ is
// kept in registers and joined the same way.
//
// Bound by HBM: 32 heads of 8193 keys are 134 MB of K and V, 28 us forward for one query (4.8 TB/s), and 268 MB with
// their gradients, 45 us backward (6.0); four queries take 50 and 72 us, bound by instructions (80 FMAs per
// key, lane and query backward).
//
// Included by sdpa_backward.cu, whose Rows, Bias and helpers it uses.

constexpr int kFewRows = 8;
constexpr int kFewThreads = 128;
// Keys up to which the forward blocks look for a bias row's largest value themselves, instead of a launch of its own:
// 2 us less of 20 to 30 (32 heads 1 x 2000 31 and 33); every block reads the row, so long rows keep the launch.
constexpr int kFewBias = 2048;

struct FewArgs {
  Rows q, k, v, out, dout;
  Bias bias;               // .p null: none
  const float2* head;      // [BH] head_stride apart: (largest bias, weight of the scores); only with a bias
  float2* head_out;        // forward: where not null, each block finds its row's head, and writes it here
  int64_t head_stride;
  const float2* stats;     // backward: [BH, Lq + 1]
  float *o, *dk, *dv;      // forward: [B, Lq, H, 64] or partial [shares, BH, Lq, 64]; backward: with strides
  float2* stats_out;       // forward: [BH, Lq + 1] or partial [shares, BH, Lq]
  float* dq;               // partial [shares, BH, Lq, 64]
  float* db;               // nullable: [BH, Lk]
  int64_t kb, kh, kl, vb, vh, vl;  // strides of dk, dv
  float *dk_part, *dv_part;  // several groups: [groups, BH, Lk, 64] in place of dk, dv; db then [groups, BH, Lk]
  int H, BH, Lq, Lk, vec, vec_out, shares, span;
  int rows, groups;        // groups of NQ = rows query rows, a block each (blockIdx.z)
};

// sum over the lanes of a warp that hold the same dimensions (lane mod 4)
__device__ __forceinline__ float sum_groups(float v) {
#pragma unroll
  for (int o = 4; o < 32; o <<= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}
// sum over the four lanes of a key
__device__ __forceinline__ float sum_key(float v) {
  v += __shfl_xor_sync(0xffffffffu, v, 1);
  return v + __shfl_xor_sync(0xffffffffu, v, 2);
}

template <int NQ>
__global__ void __launch_bounds__(kFewThreads) few_fwd_k(const FewArgs a) {
  __shared__ float qs[NQ][D];
  __shared__ float sm_m[kFewThreads / 32][NQ], sm_l[kFewThreads / 32][NQ], sm_o[kFewThreads / 32][NQ][D];
  grid_release();
  grid_wait();
  const int bh = blockIdx.y, b = bh / a.H, h = bh - b * a.H;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, lq = lane & 3;
  const int r0 = blockIdx.z * NQ, rows = min(NQ, a.Lq - r0);
  float2 head = make_float2(0.0f, 1.0f);
  if (a.bias.p && a.head_out) {
    __shared__ float sm_b[kFewThreads / 32];
    const float* row = a.bias.row(b, h);
    float mx = -INFINITY;
#pragma unroll 8
    for (int j = threadIdx.x; j < a.Lk; j += kFewThreads) mx = fmaxf(mx, row[j]);
#pragma unroll
    for (int i = 16; i > 0; i >>= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, i));
    if (lane == 0) sm_b[warp] = mx;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < kFewThreads / 32; ++w) mx = fmaxf(mx, sm_b[w]);
    head = bias_head(mx);
    if (blockIdx.x == 0 && blockIdx.z == 0 && threadIdx.x == 0) a.head_out[bh * a.head_stride] = head;
  } else if (a.bias.p) {
    head = a.head[bh * a.head_stride];
  }
  for (int i = threadIdx.x; i < NQ * D; i += kFewThreads) {
    const int r = i / D, d = i - r * D;
    qs[r][d] = r < rows && head.y != 0.0f ? a.q.at(b, h, r0 + r)[d] * (0.125f * LOG2E) : 0.0f;
  }
  __syncthreads();
  float m[NQ], l[NQ], o[NQ][16];
#pragma unroll
  for (int r = 0; r < NQ; ++r) {
    m[r] = -INFINITY;
    l[r] = 0.0f;
#pragma unroll
    for (int e = 0; e < 16; ++e) o[r][e] = 0.0f;
  }
  const int j1 = min(a.Lk, (int)(blockIdx.x + 1) * a.span);
#pragma unroll 1
  for (int jb = blockIdx.x * a.span + warp * 8; jb < j1; jb += kFewThreads / 4) {  // uniform over the warp
    const int j = jb + (lane >> 2);
    asm volatile("" ::: "memory");  // the rows stay in shared memory: registers are short
    float off = -INFINITY, kv[16], vv[16];
#pragma unroll
    for (int e = 0; e < 16; ++e) kv[e] = vv[e] = 0.0f;
    if (j < j1) off = a.bias.p ? relative_bias(a.bias.row(b, h)[j], head.x) * LOG2E : 0.0f;
    if (off != -INFINITY) {
      load16(a.k.at(b, h, j), lq, a.vec, kv);
      load16(a.v.at(b, h, j), lq, a.vec, vv);
    }
#pragma unroll
    for (int r = 0; r < NQ; ++r) {
      float s = 0.0f;
#pragma unroll
      for (int e = 0; e < 16; ++e) s = fmaf(qs[r][col16(lq, e)], kv[e], s);
      s = sum_key(s) + off;
      if (s > m[r] + 8.0f) {  // the same in the key's four lanes
        const float up = ceilf(s), f = ex2(m[r] - up);  // 0 from -inf
        m[r] = up;
        l[r] *= f;
#pragma unroll
        for (int e = 0; e < 16; ++e) o[r][e] *= f;
      }
      // a missing key gives 0, also while m is -inf; NaN stays
      const float w = s == -INFINITY ? 0.0f : ex2(s - m[r]);
      l[r] += w;
#pragma unroll
      for (int e = 0; e < 16; ++e) o[r][e] = fmaf(w, vv[e], o[r][e]);
    }
  }
#pragma unroll
  for (int r = 0; r < NQ; ++r) {
    float top = m[r];
#pragma unroll
    for (int i = 4; i < 32; i <<= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, i));
    const float f = m[r] == top ? 1.0f : ex2(m[r] - top);
    const float ls = sum_groups(l[r] * f);
#pragma unroll
    for (int e = 0; e < 16; ++e) {
      const float v = sum_groups(o[r][e] * f);
      if (lane < 4) sm_o[warp][r][col16(lq, e)] = v;
    }
    if (lane == 0) {
      sm_m[warp][r] = top;
      sm_l[warp][r] = ls;
    }
  }
  __syncthreads();
  for (int i = threadIdx.x; i < NQ * D; i += kFewThreads) {
    const int r = i / D, d = i - r * D;
    if (r >= rows) continue;
    float top = -INFINITY, ls = 0.0f, os = 0.0f;
#pragma unroll
    for (int w = 0; w < kFewThreads / 32; ++w) top = fmaxf(top, sm_m[w][r]);
#pragma unroll
    for (int w = 0; w < kFewThreads / 32; ++w) {
      const float f = sm_m[w][r] == top ? 1.0f : ex2(sm_m[w][r] - top);
      ls = fmaf(sm_l[w][r], f, ls);
      os = fmaf(sm_o[w][r][d], f, os);
    }
    os = ls == 0.0f ? 0.0f : os / ls;
    if (a.shares > 1) {
      const int64_t row = ((int64_t)blockIdx.x * a.BH + bh) * a.Lq + r0 + r;
      a.o[row * D + d] = os;
      if (d == 0) a.stats_out[row] = make_float2(top, ls);
    } else {
      a.o[(((int64_t)b * a.Lq + r0 + r) * a.H + h) * D + d] = os;
      if (d == 0) a.stats_out[(int64_t)bh * (a.Lq + 1) + r0 + r] = make_float2(top, ls);
    }
  }
  if (!a.bias.p && blockIdx.x == 0 && blockIdx.z == 0 && threadIdx.x == 0 && a.shares == 1)
    a.stats_out[(int64_t)bh * (a.Lq + 1) + a.Lq] = make_float2(0.0f, 1.0f);
}

template <int NQ>
__global__ void __launch_bounds__(kFewThreads) few_bwd_k(const FewArgs a) {
  __shared__ float qs[NQ][D], gs[NQ][D], sm_m[NQ], sm_d[NQ];
  __shared__ float sm_q[kFewThreads / 32][NQ][D];
  grid_release();
  const int bh = blockIdx.y, b = bh / a.H, h = bh - b * a.H;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, lq = lane & 3;
  const float2 head = a.bias.p ? a.head[bh * a.head_stride] : make_float2(0.0f, 1.0f);
  const float c = 0.125f * LOG2E * head.y;
  const int r0 = blockIdx.z * NQ, rows = min(NQ, a.Lq - r0);
  for (int r = warp; r < NQ; r += kFewThreads / 32) {  // a warp per row: q, g = dO / l, delta = g . O, m
    float delta = 0.0f, m = INFINITY;
    float q[2] = {0.0f, 0.0f}, g[2] = {0.0f, 0.0f};
    if (r < rows) {
      const float2 ml = a.stats[(int64_t)bh * (a.Lq + 1) + r0 + r];
#pragma unroll
      for (int u = 0; u < 2; ++u) {
        q[u] = a.q.at(b, h, r0 + r)[lane + 32 * u];
        if (ml.y != 0.0f) {
          g[u] = a.dout.at(b, h, r0 + r)[lane + 32 * u] / ml.y;
          delta = fmaf(g[u], a.out.at(b, h, r0 + r)[lane + 32 * u], delta);
        }
      }
      if (ml.y != 0.0f) m = ml.x;  // else +inf: e = 0 throughout
    }
    delta = warp_sum(delta);
    qs[r][lane] = q[0]; qs[r][lane + 32] = q[1];
    gs[r][lane] = g[0]; gs[r][lane + 32] = g[1];
    if (lane == 0) {
      sm_m[r] = m;
      sm_d[r] = delta;
    }
  }
  __syncthreads();
  float dq[NQ][16];
#pragma unroll
  for (int r = 0; r < NQ; ++r)
#pragma unroll
    for (int e = 0; e < 16; ++e) dq[r][e] = 0.0f;
  const int j1 = min(a.Lk, (int)(blockIdx.x + 1) * a.span);
#pragma unroll 1
  for (int jb = blockIdx.x * a.span + warp * 8; jb < j1; jb += kFewThreads / 4) {
    const int j = jb + (lane >> 2);
    asm volatile("" ::: "memory");  // the rows stay in shared memory: registers are short
    float off = -INFINITY, kv[16], vv[16], dk[16], dv[16], db = 0.0f;
#pragma unroll
    for (int e = 0; e < 16; ++e) kv[e] = vv[e] = dk[e] = dv[e] = 0.0f;
    if (j < j1) off = a.bias.p ? relative_bias(a.bias.row(b, h)[j], head.x) * LOG2E : 0.0f;
    if (off != -INFINITY) {
      load16(a.k.at(b, h, j), lq, a.vec, kv);
      load16(a.v.at(b, h, j), lq, a.vec, vv);
    }
#pragma unroll
    for (int r = 0; r < NQ; ++r) {
      float s = 0.0f, dp = 0.0f;
#pragma unroll
      for (int e = 0; e < 16; ++e) {
        s = fmaf(qs[r][col16(lq, e)], kv[e], s);
        dp = fmaf(gs[r][col16(lq, e)], vv[e], dp);
      }
      s = sum_key(s);
      dp = sum_key(dp);
      const float w = ex2(fmaf(s, c, off - sm_m[r])), ds = w * (dp - sm_d[r]);
      db += ds;
#pragma unroll
      for (int e = 0; e < 16; ++e) {
        dk[e] = fmaf(ds, qs[r][col16(lq, e)], dk[e]);
        dv[e] = fmaf(w, gs[r][col16(lq, e)], dv[e]);
        dq[r][e] = fmaf(ds, kv[e], dq[r][e]);
      }
    }
    if (j < j1) {
      float* pk = a.dk + b * a.kb + h * a.kh + j * a.kl;
      float* pv = a.dv + b * a.vb + h * a.vh + j * a.vl;
      const int64_t part = ((int64_t)blockIdx.z * a.BH + bh) * a.Lk + j;
      if (a.groups > 1) {
        pk = a.dk_part + part * D;
        pv = a.dv_part + part * D;
      }
#pragma unroll
      for (int e = 0; e < 16; ++e) dk[e] *= 0.125f;
      if (a.vec_out) {
#pragma unroll
        for (int e = 0; e < 16; e += 4) {
          *reinterpret_cast<float4*>(pk + col16(lq, e)) = make_float4(dk[e], dk[e + 1], dk[e + 2], dk[e + 3]);
          *reinterpret_cast<float4*>(pv + col16(lq, e)) = make_float4(dv[e], dv[e + 1], dv[e + 2], dv[e + 3]);
        }
      } else {
#pragma unroll
        for (int e = 0; e < 16; ++e) {
          pk[col16(lq, e)] = dk[e];
          pv[col16(lq, e)] = dv[e];
        }
      }
      if (a.db && (lane & 3) == 0) a.db[part] = db;
    }
  }
#pragma unroll
  for (int r = 0; r < NQ; ++r)
#pragma unroll
    for (int e = 0; e < 16; ++e) {
      const float v = sum_groups(dq[r][e]);
      if (lane < 4) sm_q[warp][r][col16(lq, e)] = v;
    }
  __syncthreads();
  for (int i = threadIdx.x; i < NQ * D; i += kFewThreads) {
    const int r = i / D, d = i - r * D;
    if (r >= rows) continue;
    float s = 0.0f;
#pragma unroll
    for (int w = 0; w < kFewThreads / 32; ++w) s += sm_q[w][r][d];
    a.dq[(((int64_t)blockIdx.x * a.BH + bh) * a.Lq + r0 + r) * D + d] = s * 0.125f;
  }
}

// Groups of query rows, and keys per block so that the GPU has some eight blocks per SM, a multiple of the 32 that a
// block takes at a time and no less than four times that.
static void few_shares(FewArgs& a, int rows) {
  a.rows = rows;
  a.groups = (a.Lq + rows - 1) / rows;
  const int64_t blocks = (int64_t)a.BH * a.groups, want = ((int64_t)sm_count() * 8 + blocks - 1) / blocks;
  const int64_t span = (a.Lk + want - 1) / want;
  a.span = (int)((span < 128 ? 128 : span + 31) / 32 * 32);
  a.shares = (a.Lk + a.span - 1) / a.span;
}

// Whether a call takes this path: up to eight query rows, or so little work that the tensor-core path (29 to 36 us for
// forward and backward of anything small) is all starts and ends.  This one takes some 17 us, 1.6 for every 100
// blocks and 1 for every 10,000 pairs of a query and a key; measured, here and there: 4 heads 65 x 17 17.5 and 32, 4 heads
// 200 x 20 17 and 35, 8 heads 16 x 1000 29 and 37, 32 heads 65 x 17 27 and 33, 32 heads 20 x 200 37 and 33, 4 heads
// 1000 x 16 43 and 37, 32 heads 90 x 90 50 and 34.  Five to eight rows of more than that are one group of eight (few
// registers left for loads in flight, but K and V are read once): 32 heads 8 x 8193 225 us, there 290, 8 heads 8 x 3000 40
// and 55, 32 heads 8 x 1000 39 and 62; of less, 8 heads 8 x 300, 33 us, as two groups of four 23.
static bool few(FewArgs& a) {
  if (a.Lq <= 4) {
    few_shares(a, a.Lq == 3 ? 4 : a.Lq);
    return true;
  }
  if ((int64_t)a.BH * a.Lq <= 140000) {
    few_shares(a, 4);
    if ((int64_t)a.BH * a.Lq * a.Lk + 160ll * a.BH * a.groups * a.shares <= 140000) return true;
  }
  if (a.Lq > kFewRows) return false;
  few_shares(a, 8);
  return true;
}

// chained: behind the bias's rows
static void few_fwd(const FewArgs& a, bool chained, cudaStream_t stream) {
  LaunchScope scope(kKSdpaAttn, stream);
  const dim3 grid(a.shares, a.BH, a.groups);
  auto kernel = a.rows == 1 ? few_fwd_k<1> : (a.rows == 2 ? few_fwd_k<2> : (a.rows == 4 ? few_fwd_k<4> : few_fwd_k<8>));
  if (chained) launch_chained(kernel, grid, dim3(kFewThreads), 0, stream, a);
  else kernel<<<grid, kFewThreads, 0, stream>>>(a);
}

static void few_bwd(const FewArgs& a, cudaStream_t stream) {
  LaunchScope scope(kKSdpaAttn, stream);
  auto kernel = a.rows == 1 ? few_bwd_k<1> : (a.rows == 2 ? few_bwd_k<2> : (a.rows == 4 ? few_bwd_k<4> : few_bwd_k<8>));
  kernel<<<dim3(a.shares, a.BH, a.groups), kFewThreads, 0, stream>>>(a);
}
