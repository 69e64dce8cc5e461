// beam.h -- beam search's selection (k_beam.hip).
#pragma once

#include "kernels.h"

namespace g4 {

constexpr int BEAM_MOST = 64;                    // beams of a group, outputs of a group
constexpr int BEAM_VOCAB = 1 << 24;

struct BeamSelect {
    const float *x;                              // logits, rows `stride` floats apart
    size_t stride;
    int n_group, n_beam, n_vocab, n_out;
    const float *score;
    const int *ended;                            // or null
    float *score_out;
    int *row_out, *token_out;
    int lists, span;                             // workgroups a row, and the tokens of each
    float2 *ms;                                  // [row][list] maximum, sum of exp(x - maximum)
    uint64_t *top;                               // [row][list][n_out] candidates, descending; 0: none
};
// workspace of a call; and enough for it and all calls of fewer groups
size_t beam_workspace(int n_group, int n_beam, int n_vocab, int n_out);
size_t beam_workspace_most(int n_group, int n_beam, int n_vocab, int n_out);
hipError_t launch_beam_select(BeamSelect a, uint8_t *ws, hipStream_t s);

}  // namespace g4
