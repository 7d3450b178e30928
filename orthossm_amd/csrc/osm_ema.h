// Parameters of the gated EMA's kernels (osm_ema.hip).
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

namespace osm {

constexpr int kEmaLanes = 128;     // channels of a lane-block
constexpr int kEmaWaves = 8;       // token groups of a tile, one a wave
constexpr int kEmaRun = 16;        // tokens of a group, forward
constexpr int kEmaBwdRun = 8;      // backward, which holds twice as much of a token
constexpr int kEmaTile = kEmaWaves * kEmaRun, kEmaBwdTile = kEmaWaves * kEmaBwdRun;
constexpr int kEmaGroup = 8;       // tiles from checkpoint to checkpoint
// A lane-block's line of the workspace: its counter at this word.  The first's holds the launch's
// fault word too, where the headers of the other look-backs' workspaces do.
constexpr int kEmaLine = 32, kEmaTicket = 1;

struct EmaSeq {
  void* p;
  int64_t sb, ss;
};

struct EmaParams {
  EmaSeq x, gate, out;
  const int* lengths;            // [B], or NULL
  const float* init;             // [B,D], or NULL
  float* fin;                    // [B,D], or NULL
  float* saved;                  // [B][n_saved][D]: the state ahead of each of the backward's tiles, or NULL
  EmaSeq go, gx, gg;             // the backward's
  const float* gstate;           // [B,D], or NULL
  float* ginit;                  // [B,D], or NULL
  unsigned long long* words;     // zeroed: [lane-blocks][tiles][kEmaLanes] tile maps
  unsigned long long* marks;     // zeroed: [lane-blocks][groups][kEmaLanes] states after whole groups
  unsigned* lines;               // zeroed: [lane-blocks][kEmaLine]
  int B, S, D, n_lbd, n_lb, n_tiles, n_groups, n_saved;
  int vec;                       // rows and D in pairs of channels, aligned
  unsigned poll_limit;           // of a wait: kSpinLimit, or 0 under OSM_FLAG_POLL_LIMIT_ZERO
};

struct EmaStepParams {
  EmaSeq x, gate, out;
  float* state;
  int64_t state_s, n_slots;
  const int64_t* slots;
  int B, D;
  int vec;                       // groups of 4 channels, aligned
};

hipError_t launch_ema_fwd(const EmaParams& p, int dtype, hipStream_t stream);
hipError_t launch_ema_bwd(const EmaParams& p, int dtype, hipStream_t stream);
hipError_t launch_ema_step(const EmaStepParams& p, int dtype, hipStream_t stream);

}  // namespace osm
