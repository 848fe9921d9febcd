// Beam search's selection over beams and vocabulary (beam_select.cu).
#pragma once

#include "common.cuh"

namespace tb {

struct BeamSelect {
    const void* logits;            // [groups * beams, logits_ld]
    const float* scores;           // [groups * beams]
    const uint8_t* finished;       // [groups * beams] or null
    float* next_scores;            // [groups, keep]
    uint32_t *tokens, *parents;    // [groups, keep]
    uint8_t* next_finished;        // [groups, keep] or null
    void* workspace;
    uint64_t workspace_bytes, logits_ld;
    uint32_t groups, beams, vocab, keep, end_token;
    int* d_status;                 // or null
};
constexpr uint32_t BEAM_MAX = 32, BEAM_MAX_KEEP = 64;
constexpr uint32_t BEAM_MAX_VOCAB = 1u << 26;
// Bytes of a workspace before the lists: the groups' tickets, zero between calls.  A fixed place, so that a call of other sizes finds no other call's lists there.
constexpr uint32_t BEAM_COUNTERS = 4096;
uint64_t beam_select_workspace_bytes(uint32_t groups, uint32_t beams, uint32_t vocab, uint32_t keep);
int launch_beam_select(const BeamSelect& b, int dtype, cudaStream_t stream);

}  // namespace tb
