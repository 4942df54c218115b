// Selection of beams, the host side: argument checks and the workspace's layout.
#include "vgpu_beams.h"

#include "vgpu_runtime.h"

namespace vgpu {

namespace {

void need(bool ok, const char* msg, int code = VGPU_ERR_INVALID_PARAMETER) {
    if (!ok) throw Error(code, msg);
}

// The checked sizes, and how a row is cut.
BeamArgs sizes(int dtype, size_t rows, size_t vocab, size_t beams, size_t k) {
    need(dtype == VGPU_F32 || dtype == VGPU_F16 || dtype == VGPU_BF16, "dtype must be float32, float16 or bfloat16");
    need(beams > 0 && beams <= (size_t)BEAM_MAX_BEAMS, "beams must be in the range 1..=1024");
    need(vocab > 0 && vocab <= (size_t)1 << 30, "vocab must be in the range 1..=2^30");
    need(rows % beams == 0 && rows <= (size_t)1 << 24, "rows must be a multiple of beams, at most 2^24");
    // a launch's threads, 1024 to a group, are counted in 32 bits
    need(rows / beams < (size_t)1 << 22, "more than 2^22 - 1 groups in one call");
    need(k > 0 && k <= (size_t)BEAM_MAX_K && k <= beams * vocab, "k must be in the range 1..=256 and at most beams * vocab");
    BeamArgs a;
    a.type = dtype;
    a.rows = (int)rows, a.vocab = (int)vocab, a.beams = (int)beams, a.k = (int)k;
    beam_plan(a);
    // (and 256 to a slice)
    need((int64_t)a.rows * a.slices < 1 << 24 && (int64_t)a.beams * a.slices * a.k < (int64_t)1 << 31,
         "too many logits in one call");
    return a;
}

}  // namespace

size_t beams_workspace(int dtype, size_t rows, size_t vocab, size_t beams, size_t k) {
    const BeamArgs a = sizes(dtype, rows, vocab, beams, k);
    const size_t parts = (size_t)a.rows * a.slices;
    return parts * (sizeof(double) + a.k * sizeof(uint2) + sizeof(float));
}

void select_beams(const vgpu_beams& q, hipStream_t s) {
    BeamArgs a = sizes(q.dtype, q.rows, q.vocab, q.beams, q.k);
    if (!q.rows) return;
    need(q.logits && q.out_scores && q.out_parents && q.out_tokens, "null argument");
    const size_t item = q.dtype == VGPU_F32 ? 4 : 2;
    need((uintptr_t)q.logits % item == 0 && (uintptr_t)q.scores % 4 == 0, "inputs must be aligned to their dtype");
    need((uintptr_t)q.out_scores % 4 == 0 && ((uintptr_t)q.out_parents | (uintptr_t)q.out_tokens) % 8 == 0,
         "outputs must be aligned to their dtype");
    const size_t parts = (size_t)a.rows * a.slices;
    need(q.workspace && (uintptr_t)q.workspace % 16 == 0 &&
             q.workspace_bytes >= parts * (sizeof(double) + a.k * sizeof(uint2) + sizeof(float)),
         "the workspace is smaller than vgpu_beams_workspace says, or not aligned to 16 bytes");
    a.logits = q.logits;
    a.st_row = q.stride_row, a.st_token = q.stride_token;
    a.scores = q.scores, a.st_score = q.stride_score;
    a.sum = (double*)q.workspace;
    a.best = (uint2*)(a.sum + parts);
    a.top = (float*)(a.best + parts * a.k);
    a.out_scores = q.out_scores, a.out_parents = q.out_parents, a.out_tokens = q.out_tokens;
    launch_beams(a, s);
    VGPU_HIP(hipGetLastError());
}

}  // namespace vgpu
