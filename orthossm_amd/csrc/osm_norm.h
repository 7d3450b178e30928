// Parameters of the layer norm's and the gradient clipping's kernels
// (osm_norm.hip, osm_clip.hip).
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

namespace osm {

struct NormParams {
  const void* x;                 // rows x_stride elements apart
  const float* weight;           // [D], or NULL: ones
  const float* bias;             // [D], or NULL: zeros
  void* y;
  float* mean;                   // [rows]: written by the forward (or NULL), read by the backward
  float* rstd;
  const void* gy;                // the backward's
  void* gx;                      // or NULL
  float* part;                   // [norm_lines][2][D]
  int64_t x_stride, y_stride, gy_stride, gx_stride, rows, D;
  float eps;
  int vec;                       // rows start at multiples of 16 bytes, D is whole 16-byte units
};

int norm_lines(int64_t rows, int64_t D);
hipError_t launch_layer_norm_fwd(const NormParams& p, int dtype, hipStream_t stream);
hipError_t launch_layer_norm_bwd(const NormParams& p, float* dw, float* db, int dtype, hipStream_t stream);

// A launch's tensors, passed by value: kernel arguments hold 4 KB.
constexpr int kClipTensors = 150;
struct ClipTable {
  void* p[kClipTensors];
  int64_t n[kClipTensors];       // elements
  int first[kClipTensors + 1];   // first chunk of each tensor; [count]: all chunks
  unsigned char bf16[kClipTensors];
  unsigned char vec[kClipTensors];   // 16-byte aligned
  int count;
  int part0, parts;              // this launch's first partial sum and number of them
};

constexpr int kClipChunk = 8192;     // elements
constexpr int kClipMaxGroups = 1024; // workgroups, and partial sums, of a launch

hipError_t launch_clip_sums(const ClipTable& t, double* part, hipStream_t stream);
// norm = sqrt(the sum of all `parts` partial sums); with scale, every element
// times min(1, max_norm / (norm + eps)).
hipError_t launch_clip_scale(const ClipTable& t, const double* part, int parts, double max_norm, double eps, float* norm,
                             bool scale, hipStream_t stream);

}  // namespace osm
