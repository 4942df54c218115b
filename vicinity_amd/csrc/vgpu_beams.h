// The selection of beams: arguments of its two kernels.
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

namespace vgpu {

constexpr int BEAM_MAX_K = 256;
constexpr int BEAM_MAX_BEAMS = 1024;

struct BeamArgs {
    const void* logits = nullptr;
    int type = 0;                      // VGPU_F32, VGPU_F16 or VGPU_BF16
    int64_t st_row = 0, st_token = 0;  // strides in elements
    const float* scores = nullptr;     // of the rows, or null: 0
    int64_t st_score = 0;
    int rows = 0, vocab = 0, beams = 0, k = 0;
    int pieces = 0;                    // of 16 bytes, of each of 256 threads, in a slice of a row
    int slices = 0;                    // of a row
    // of each row and slice: largest logit, sum of exp(logit - it), and its k best tokens
    float* top = nullptr;
    double* sum = nullptr;
    uint2* best = nullptr;             // (logit as bits, token), descending; token ~0: none
    float* out_scores = nullptr;       // [rows / beams, k]
    int64_t *out_parents = nullptr, *out_tokens = nullptr;
};

// Sets pieces and slices.
void beam_plan(BeamArgs& a);
void launch_beams(const BeamArgs& a, hipStream_t s);

}  // namespace vgpu
