// Parameters of the residual norm's kernels (osm_resnorm.hip).
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

namespace osm {

struct ResnormParams {
  const void *x, *y, *gate;      // rows a stride apart; gate may be NULL
  const float *scale, *weight, *bias;   // [D], or NULL
  void *r, *n;
  float* stats;                  // [rows][4], or NULL: mean and 1 / spread of y, of r
  const void *gr, *gn;           // the backward's; each may be NULL
  void *gx, *gy, *gg;
  float* part;                   // [lines][3][D]: weight, bias, scale
  float* sums;                   // [rows][2], of long rows
  int64_t x_s, y_s, gate_s, r_s, n_s, gr_s, gn_s, gx_s, gy_s, gg_s, rows, D;
  float eps;
  int norm_y, rms;
  int vec;                       // rows start at multiples of 16 bytes, D is whole units
};

// Whether rows of D are too long for registers (then the backward needs `sums`).
bool resnorm_long(int64_t D);
hipError_t launch_resnorm_fwd(const ResnormParams& p, int stream_dtype, int block_dtype, hipStream_t stream);
hipError_t launch_resnorm_bwd(const ResnormParams& p, float* dw, float* db, float* ds, int stream_dtype, int block_dtype,
                              hipStream_t stream);

}  // namespace osm
