// Parameters of the vocabulary's cross entropy (osm_loss.hip).
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

namespace osm {

constexpr int kLossPad = 256;      // rows of compacted tokens, columns of a piece: multiples of this

// The tokens that count, one after the other.  All NULL in a short forward, whose tokens
// are all in their own places, those that do not count too.
struct LossTokens {
  int* targets;                    // [N]: by place, -1: outside the vocabulary
  float2* factors;                 // [N]: by place, log2(e) lse and grad_losses (1 without); the backward's
  int* places;                     // [N]: the place of each token, -1: does not count
  int* count;                      // device scalar: how many
};

struct LossParams {
  int64_t N, D, V;
  int Npad, Dpad, parts, p_parts;  // parts of hidden and weight: 1 (bf16), 3 (fp32); of p: 2 of few bf16 tokens
  const void* hidden;
  int64_t hidden_s;
  const void* weight;
  int64_t weight_s;
  const int64_t* targets;
  int64_t ignore;
  LossTokens tok;
  const __bf16* h;                 // [parts][h_rows][h_ld], h_part apart: the hidden rows that count, zeros after them up to a whole step
  int64_t h_ld, h_part;
  int h_rows;
  // a piece of the vocabulary
  int64_t v0;
  int vn, vpad;                    // its classes; columns of p
  const __bf16* w;                 // [parts][vn][w_ld], w_part apart
  int64_t w_ld, w_part;
  __bf16* p;                       // [p_parts][Npad][vpad]: probabilities less the targets'
  float* dh;                       // [splits][Npad][Dpad]
  int splits, first;               // first: dh is written, not added to
  // statistics
  float2* stat;                    // [tiles of the vocabulary][Npad]: largest logit, sum of exp of what is below it
  int tile0;                       // the piece's first tile
  float* own;                      // [Npad]: the target's logit
  float *losses, *lse, *loss, *count;
  int mean;
  const float *grad, *grad_losses, *count_in;
  void *grad_h, *grad_w;
};

hipError_t launch_loss_rows(const LossParams& p, __bf16* h, __bf16* w, int dtype, bool bwd, hipStream_t stream);   // tok, h; w: or NULL
hipError_t launch_loss_weight(const LossParams& p, __bf16* w, int dtype, hipStream_t stream);   // parts of the piece's rows
int loss_tile_rows(const LossParams& p);                                                    // classes of a forward's tile of logits, by N, V and parts
hipError_t launch_loss_logits(const LossParams& p, hipStream_t stream);                     // stat, own
hipError_t launch_loss_join(const LossParams& p, int tiles, hipStream_t stream);            // losses, lse, loss, count
hipError_t launch_loss_none(float* loss, float* count, hipStream_t stream);
hipError_t launch_loss_probs(const LossParams& p, hipStream_t stream);                      // p
hipError_t launch_loss_dh(const LossParams& p, hipStream_t stream);
hipError_t launch_loss_dw(LossParams p, int from, int n, hipStream_t stream);                // of n of the piece's classes
hipError_t launch_loss_zero(void* to, int64_t n, int dtype, hipStream_t stream);
hipError_t launch_loss_finish(const LossParams& p, int dtype, hipStream_t stream);          // grad_h

}  // namespace osm
