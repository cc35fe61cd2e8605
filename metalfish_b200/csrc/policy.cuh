// policy.cuh -- operators on policy logits and legal-move lists (policy.cu).
#pragma once
#include <cuda_runtime.h>

#include <cstdint>

namespace mfb200 {

// A batch of policy rows with their legal moves, on the device (the fields of
// mfb200_policy_rows; off[0] is the position of index[0]).
struct PolicyRows {
  const void *logits;
  long long stride;  // elements between rows
  int type;          // MFB200_TYPE_*
  int batch, classes;
  const int32_t *off;     // [batch + 1]
  const int16_t *index;   // [num_moves]
  long long num_moves;
  const int32_t *played;  // [batch] edge numbers, or null
  double temp, inv_temp64;  // 1 / temp
  float inv_temp;
};

// Log-probabilities of the legal moves, of the played move and the entropy;
// each output may be null.
cudaError_t launch_move_logprobs(const PolicyRows &r, float *move_logp, float *played_logp,
                                 float *entropy, cudaStream_t s);

}  // namespace mfb200
