// What the attention's training entries (sdpa_backward.cu) share with the attention itself: the
// split-format inputs of the forward kernel and its launch with the row statistics kept.
#pragma once

#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <stdint.h>

namespace tsb {

// Attention inputs in the split format, in the library workspace of the current stream.
struct SplitPlanesSdpa {
  __half *qhi, *qlo, *khi, *klo, *vhi, *vlo;
  float *qinv, *kinv, *vinv;
  int T, Lkt;
};

// Planes for BH heads in the workspace, and `extra` bytes behind them (256-byte aligned).
int sdpa_planes_extra(int64_t BH, int Lq, int Lk, size_t extra, cudaStream_t stream, SplitPlanesSdpa& sp,
                      void** behind);

// The attention kernel on split planes, BLHD output, with each row's (reference maximum in log2
// units, sum of 2^(score - maximum)) written to stats [BH, stats_ld] (row r of head bh at
// bh * stats_ld + r).  cuts > 1: the keys' tiles in that many shares, each with its own output and
// statistics, cut_out floats and cut_stats rows apart (few rows: more work items).  tiles (nullable, [BH]):
// the first 128-key tile with a key and the one past the last, where the bias is -inf outside.  A row without a key (every bias
// -inf) gives zeros and (-inf, 0).
int sdpa_attend_stats(const SplitPlanesSdpa& sp, const float* bias, int64_t bias_bh_stride, const int2* tiles,
                      float* out_blhd, float2* stats, int64_t stats_ld, int64_t BH, int H, int Lq, int Lk, int cuts, int64_t cut_out,
                      int64_t cut_stats, cudaStream_t stream);

}  // namespace tsb
