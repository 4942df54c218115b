// Softmax attention over the 8-bit cache.
//
// For a row r (a query token and head) and slot j:  u_j = scale * log2(e) * q_r.k_j,
// o = sum 2^(u_j) v_j / sum 2^(u_j).  One pass over the tiles with a running
// reference m: the value scale s_b of a block goes into the exponent,
// p_j = 2^(u_j + log2 s_b - m), so o's accumulators add p_j * code directly in the
// matrix instruction, and the denominator adds p_j S / s_b.  S is a row's own power of
// two, near the largest scale that moved its m, so that l stays in float32's range for
// scales of any size; the result is S o / l.
//
// Products: codes are integers up to 127 or e4m3 numbers, both exact in half
// precision.  A query row is scaled by a power of two to a largest element of 2^14
// and split into 1 (bf16, f16: exact for elements down to 2^-28 of it) or 2 (f32: 22 bits)
// halves, so the scores are float32 sums of exact products.  p is rounded to half precision
// (2^-11), the matrix instruction's, for 16-bit queries, whose results are rounded to as many
// bits or fewer, and to two halves (2^-22) for float32 ones; p is held near 2^6 .. 2^14 at the
// top, so what is below 2^-30 of the largest rounds to zero.
// m only moves when a score exceeds it by 2^8: a step that costs a scaling of the
// accumulators, taken by a whole wave, nearly always in the first tile only.
//
// SH: rows of several sequences over slots that all of them hold (KvMembers), and over what
// each holds alone; every workgroup leaves partial results.
#pragma once

#include "vgpu_kv.h"
#include "vgpu_launch.h"

#include <climits>
#include <hip/hip_bf16.h>

namespace vgpu {

namespace {

typedef _Float16 half8 __attribute__((ext_vector_type(8)));
typedef _Float16 half2v __attribute__((ext_vector_type(2)));
typedef float floatx4 __attribute__((ext_vector_type(4)));
typedef unsigned int u32x4 __attribute__((ext_vector_type(4)));

constexpr float KV_TOP = 6.f;    // p of the reference is 2^KV_TOP
constexpr float KV_SLACK = 8.f;  // and may grow to 2^(KV_TOP + KV_SLACK)
// S / s_b at most, and log2 s_b at least log2 S less its logarithm.  So a scale of 0, which
// stands for codes of 0, takes part in the denominators without setting m beside values down
// to 2^-80 of those that the row has seen; codes of a smaller scale that is not 0 come out as
// if it were 2^-80 of theirs.
constexpr float KV_FAR = 80.f, KV_FAR_F = 0x1p80f;
// S before a scale above 0 moved m: below all of them (2^-109 and up)
constexpr int KV_FIRST = -125;
#define KV_NEG (-__builtin_huge_valf())
// m - KV_TOP of a row that has seen no slot: whatever it sees stands far above (the least float).
constexpr float KV_START = -0x1.fffffep127f;

// Two halves of 8 codes.
template <int CODE>
__device__ __forceinline__ half8 kv_half8(uint32_t w0, uint32_t w1) {
    u32x4 r;
    if (CODE == KV_INT8) {
        // 1024 + (code + 128) by its bits, less 1152
        const half2v off = {(_Float16)-1152.f, (_Float16)-1152.f};
        const uint32_t magic = 0x64646464u;
        r.x = __builtin_bit_cast(uint32_t, __builtin_bit_cast(half2v, __builtin_amdgcn_perm(magic, w0, 0x04010400u)) + off);
        r.y = __builtin_bit_cast(uint32_t, __builtin_bit_cast(half2v, __builtin_amdgcn_perm(magic, w0, 0x04030402u)) + off);
        r.z = __builtin_bit_cast(uint32_t, __builtin_bit_cast(half2v, __builtin_amdgcn_perm(magic, w1, 0x04010400u)) + off);
        r.w = __builtin_bit_cast(uint32_t, __builtin_bit_cast(half2v, __builtin_amdgcn_perm(magic, w1, 0x04030402u)) + off);
    } else {
        r.x = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(w0, 1.f, false));
        r.y = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(w0, 1.f, true));
        r.z = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(w1, 1.f, false));
        r.w = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(w1, 1.f, true));
    }
    return __builtin_bit_cast(half8, r);
}

__device__ __forceinline__ float kv_half_bits(uint32_t h, int type) {
    return type == KV_F16 ? (float)__builtin_bit_cast(_Float16, (uint16_t)h) : __uint_as_float(h << 16);
}

// A lane's dims of a row, x[s][e] = dim 32 s + 8 g + e (0 from D on); PARTS 2: float32,
// else one of the 16-bit types.  Rows of one aligned piece per 8 dims, or any strides.
template <int S, int PARTS>
__device__ __forceinline__ void kv_load_row(const KvTensor& t, int64_t row, int g, int D, float (&x)[S][8]) {
    if (t.vec) {
#pragma unroll
        for (int s = 0; s < S; s++) {
            const int64_t at = row + min(32 * s + 8 * g, D - 8);
            const bool in = 32 * s + 8 * g < D;
            if (PARTS > 1) {
                const float4* p = (const float4*)((const float*)t.p + at);
                const float4 a = p[0], b = p[1];
                x[s][0] = a.x, x[s][1] = a.y, x[s][2] = a.z, x[s][3] = a.w;
                x[s][4] = b.x, x[s][5] = b.y, x[s][6] = b.z, x[s][7] = b.w;
            } else {
                const uint4 a = *(const uint4*)((const uint16_t*)t.p + at);
                const uint32_t w[4] = {a.x, a.y, a.z, a.w};
#pragma unroll
                for (int e = 0; e < 8; e++) x[s][e] = kv_half_bits(w[e >> 1] >> (16 * (e & 1)) & 0xffffu, t.type);
            }
#pragma unroll
            for (int e = 0; e < 8; e++) x[s][e] = in ? x[s][e] : 0.f;
        }
        return;
    }
#pragma unroll
    for (int s = 0; s < S; s++)
#pragma unroll
        for (int e = 0; e < 8; e++) {
            const int d = 32 * s + 8 * g + e;
            const int64_t at = row + (int64_t)min(d, D - 1) * t.sd;
            const float v = PARTS > 1 ? ((const float*)t.p)[at] : kv_half_bits(((const uint16_t*)t.p)[at], t.type);
            x[s][e] = d < D ? v : 0.f;
        }
}

// Dims d .. d + 3 of a result row (those below D), rounded once.
template <int PARTS>
__device__ __forceinline__ void kv_store4(const KvAttend& a, size_t row, int d, int D, floatx4 v) {
    if (PARTS > 1) {
        float* at = (float*)a.out + row + d;
        if (a.vec_out && d < D) {
            *(floatx4*)at = v;
            return;
        }
#pragma unroll
        for (int e = 0; e < 4; e++)
            if (d + e < D) at[e] = v[e];
        return;
    }
    uint32_t w[2];
    if (a.q.type == KV_F16) {
#pragma unroll
        for (int e = 0; e < 2; e++) w[e] = __builtin_bit_cast(uint32_t, half2v{(_Float16)v[2 * e], (_Float16)v[2 * e + 1]});
    } else {
#pragma unroll
        for (int e = 0; e < 2; e++) {
            const __hip_bfloat16 x = __float2bfloat16(v[2 * e]), y = __float2bfloat16(v[2 * e + 1]);
            w[e] = (uint32_t)__builtin_bit_cast(uint16_t, x) | (uint32_t)__builtin_bit_cast(uint16_t, y) << 16;
        }
    }
    uint16_t* at = (uint16_t*)a.out + row + d;
    if (a.vec_out && d < D) {
        *(uint2*)at = make_uint2(w[0], w[1]);
        return;
    }
#pragma unroll
    for (int e = 0; e < 4; e++)
        if (d + e < D) at[e] = (uint16_t)(w[e >> 1] >> (16 * (e & 1)));
}

// Largest over the four lanes that hold one row's slots.
__device__ __forceinline__ float kv_max4(float v) {
    v = fmaxf(v, __shfl_xor(v, 16));
    return fmaxf(v, __shfl_xor(v, 32));
}
__device__ __forceinline__ float kv_sum4(float v) {
    v += __shfl_xor(v, 16);
    return v + __shfl_xor(v, 32);
}

// Slots lo .. hi - 1 that row `row` (of count * G) of a sequence may see.
__device__ __forceinline__ void kv_range(const KvAttend& a, int len, int count, int row, int& lo, int& hi) {
    const int p = len - count + kv_div(row, a.by_group);  // its own slot
    hi = a.causal ? max(p + 1, 0) : len;
    lo = a.window ? max(p + 1 - a.window, 0) : 0;
}

template <bool SH>
__device__ __forceinline__ int kv_job_rows(const KvBatch& b, const KvAttend& a, int i) {
    return SH ? b.count[i] : b.count[i] * a.G;
}

// The sequence of the lane's row row0 + (lane & 15) (the last one past the end) of an entry
// whose rows begin with those of sequence `first`.
__device__ __forceinline__ int kv_member(const KvMembers& mem, int first, int rows, int row0) {
    const int base = mem.row0[first];
    if (mem.row0[first + 1] - base >= rows) return first;
    const int lane = threadIdx.x & 63;
    const int lo = lane < mem.n ? mem.row0[lane] : INT_MAX, hi = lane + 64 < mem.n ? mem.row0[lane + 64] : INT_MAX;
    int mine = 0;
#pragma unroll
    for (int c = 0; c < 16; c++) {
        const int row = base + min(row0 + c, rows - 1);
        const int m = __popcll(__ballot(lo <= row)) + __popcll(__ballot(hi <= row)) - 1;
        mine = (lane & 15) == c ? m : mine;
    }
    return mine;
}

// The running state of a wave: NC column tiles of 16 rows.
template <int S, int CODE, int PARTS, int NC, bool SH>
struct KvWave {
    half8 q[NC][PARTS][S];
    float qs[NC];          // 2^-(the row's scaling) * scale * log2(e)
    int lo[NC], hi[NC];    // slots that the row sees
    int row[NC];
    int tok[SH ? NC : 1];  // the row's token in the call
    int row0, len, count;
    float t[NC], l[NC], bad[NC];  // t: m - KV_TOP
    float s[NC], low[NC];  // S; log2 S - KV_FAR
    floatx4 o[NC][2 * S];
};

template <int S, int CODE, int PARTS, int NC, bool SH>
__device__ __forceinline__ void kv_load_rows(KvWave<S, CODE, PARTS, NC, SH>& w, const KvDev& c, const KvBatch& b,
                                             const KvAttend& a, const KvMem<SH>& mem, int i, int h, int row0) {
    const int lane = threadIdx.x & 63, col = lane & 15, g = lane >> 4;
    const int rows = kv_job_rows<SH>(b, a, i), len = b.len[i];
    w.row0 = row0, w.len = len, w.count = b.count[i];
#pragma unroll
    for (int n = 0; n < NC; n++) {
        const int row = row0 + n * 16 + col;
        w.row[n] = row < rows ? row : -1;
        w.lo[n] = 0, w.hi[n] = 0;  // rows past the end see nothing
        w.t[n] = KV_START, w.l[n] = 0.f, w.bad[n] = 0.f;
        w.s[n] = __builtin_ldexpf(1.f, KV_FIRST), w.low[n] = (float)KV_FIRST - KV_FAR;
        float big = 0.f;
        // (a row past the end loads the last one's and is not used)
        const int real = min(row, rows - 1);
        int tok = b.tok0[i], mine = real;  // the sequence's first token, and the row in it
        if constexpr (SH) {
            const int m = kv_member(mem, b.aux[i], rows, row0 + n * 16);
            tok = mem.tok0[m], mine = real + mem.row0[b.aux[i]] - mem.row0[m];
            w.tok[n] = tok + kv_div(mine, a.by_group);
            if (row < rows) {
                kv_range(a, mem.len[m], mem.count[m], mine, w.lo[n], w.hi[n]);
                w.lo[n] = max(w.lo[n], b.tok0[i] * KV_TILE), w.hi[n] = min(w.hi[n], len);
            }
        } else {
            if (row < rows) kv_range(a, len, b.count[i], row, w.lo[n], w.hi[n]);
        }
        const int64_t base = (int64_t)(tok + kv_div(mine, a.by_group)) * a.q.st + (int64_t)(h * a.G + kv_mod(mine, a.by_group)) * a.q.sh;
        float x[S][8];
        kv_load_row<S, PARTS>(a.q, base, g, c.D, x);
#pragma unroll
        for (int s = 0; s < S; s++)
#pragma unroll
            for (int e = 0; e < 8; e++) big = fmaxf(big, fabsf(x[s][e]));
        big = kv_max4(big);
        int ex = 0;
        if (big > 0.f && big < __builtin_huge_valf()) (void)frexpf(big, &ex), ex -= 15;
        // An infinite element makes every score infinite or NaN, and the softmax of any of them
        // NaN: also where all are -inf, which the sums would take for a row that sees nothing.
        w.qs[n] = big < __builtin_huge_valf() ? ldexpf(a.scale2, ex) : __uint_as_float(0x7fc00000u);
#pragma unroll
        for (int s = 0; s < S; s++)
#pragma unroll
            for (int e = 0; e < 8; e++) {
                const float y = ldexpf(x[s][e], -ex);
                const _Float16 y0 = (_Float16)y;
                w.q[n][0][s][e] = y0;
                if (PARTS > 1) w.q[n][PARTS - 1][s][e] = (_Float16)(y - (float)y0);
            }
#pragma unroll
        for (int j = 0; j < 2 * S; j++) w.o[n][j] = floatx4{0.f, 0.f, 0.f, 0.f};
    }
}

// Four column tiles have no registers for their rows' numbers and slots: here they are worked
// out again, before they are needed (64 dims, 2048 tokens over 16384 slots: 372 us, 377 kept).
template <int S, int CODE, int PARTS, int NC, bool SH>
__device__ __forceinline__ void kv_rows_again(KvWave<S, CODE, PARTS, NC, SH>& w, const KvAttend& a, int n) {
    if (NC <= 2 || SH) return;  // (SH keeps them: a row's sequence would have to be found again)
    const int row = w.row0 + n * 16 + (threadIdx.x & 15);
    w.row[n] = row < w.count * a.G ? row : -1;
    w.lo[n] = w.hi[n] = 0;
    if (w.row[n] >= 0) kv_range(a, w.len, w.count, row, w.lo[n], w.hi[n]);
}

// What a wave needs to know of 64 tiles, one to a lane: refilled every 64 tiles, so no
// step waits for the block table or a scale.
struct KvTiles {
    uint32_t lo, hi;   // its offset in the pool
    float ks, lv, rv;  // key scale, log2 of the value scale and 1 by it (0 and NaN: -inf and inf)
    uint64_t bad;      // tiles whose value scale is NaN
};

// Tiles first, first + step, ... below last, for lanes 0, 1, ...
__device__ __forceinline__ KvTiles kv_tile_infos(const KvDev& c, const int* table, int h, int first, int step, int last) {
    const int t = first + (threadIdx.x & 63) * step;
    KvTiles r;
    const bool in = t < last;
    const int block = in ? table[t >> (c.shift - 5)] : 0;
    const size_t part = (size_t)block * c.H + h;
    const size_t at = kv_tile_offset(c, block, h, t & (c.B / KV_TILE - 1));
    r.lo = (uint32_t)at, r.hi = (uint32_t)(at >> 32);
    r.ks = in ? c.kscale[part] : 0.f;
    const float vs = in ? c.vscale[part] : 0.f;
    r.bad = __ballot(vs != vs);
    r.lv = vs > 0.f ? log2f(vs) : KV_NEG;
    r.rv = vs > 0.f ? 1.f / vs : -KV_NEG;
    return r;
}
__device__ __forceinline__ const uint8_t* kv_tile_of(const KvDev& c, const KvTiles& f, int lane) {
    const uint32_t lo = (uint32_t)__builtin_amdgcn_readlane((int)f.lo, lane);
    const uint32_t hi = (uint32_t)__builtin_amdgcn_readlane((int)f.hi, lane);
    return c.pool + ((size_t)hi << 32 | lo);
}
__device__ __forceinline__ float kv_lane(float v, int lane) {
    return __uint_as_float((uint32_t)__builtin_amdgcn_readlane((int)__float_as_uint(v), lane));
}

// Largest of 8, a NaN only if all are (fmaxf would quiet each operand first).
__device__ __forceinline__ float kv_max8(const float (&x)[8]) {
    float r;
    asm("v_max3_f32 %0, %1, %2, %3" : "=v"(r) : "v"(x[0]), "v"(x[1]), "v"(x[2]));
    asm("v_max3_f32 %0, %1, %2, %3" : "=v"(r) : "v"(r), "v"(x[3]), "v"(x[4]));
    asm("v_max3_f32 %0, %1, %2, %3" : "=v"(r) : "v"(r), "v"(x[5]), "v"(x[6]));
    asm("v_max_f32 %0, %1, %2" : "=v"(r) : "v"(r), "v"(x[7]));
    return r;
}

// A tile's base-2 scores above m - KV_TOP from its products u with the rows; m moves if one
// is too far above it.  inside: every row sees all 32 slots.
template <int S, int CODE, int PARTS, int NC, bool SH>
__device__ __forceinline__ void kv_reference(KvWave<S, CODE, PARTS, NC, SH>& w, const floatx4 (&u)[NC][2], float ks, float lv,
                                             bool bad, int slot0, bool inside, const KvAttend& a, int tok0, float* scores,
                                             int64_t score_row, float (&x)[NC][8]) {
    const int g = (threadIdx.x & 63) >> 4;
    bool over = false;
    if (inside && !scores) {
#pragma unroll
        for (int n = 0; n < NC; n++) {
            const float f = w.qs[n] * ks, base = fmaxf(lv, w.low[n]) - w.t[n];
#pragma unroll
            for (int j = 0; j < 8; j++) x[n][j] = __builtin_fmaf(u[n][j >> 2][j & 3], f, base);
        }
        if (bad)
#pragma unroll
            for (int n = 0; n < NC; n++) w.bad[n] = __uint_as_float(0x7fc00000u);
    } else {
#pragma unroll
        for (int n = 0; n < NC; n++) {
            const float f = w.qs[n] * ks, base = fmaxf(lv, w.low[n]) - w.t[n];
            bool any = inside;
#pragma unroll
            for (int j = 0; j < 8; j++) x[n][j] = u[n][j >> 2][j & 3] * f;
            if (!inside) {
                kv_rows_again(w, a, n);
                // slot0 + 4 g + off sees: lo <= slot < hi
                const int first = w.lo[n] - slot0 - 4 * g, count = w.hi[n] - w.lo[n];
#pragma unroll
                for (int j = 0; j < 8; j++) {
                    const bool see = (unsigned)((j >> 2) * 16 + (j & 3) - first) < (unsigned)count && count > 0;
                    x[n][j] = see ? x[n][j] : KV_NEG;
                    any |= see;
                }
                if (a.mask && any) {
                    any = false;
                    const uint8_t* mask = a.mask + (int64_t)(SH ? w.tok[n] : tok0 + kv_div(max(w.row[n], 0), a.by_group)) * a.mask_st;
                    uint8_t see[8];
#pragma unroll
                    for (int j = 0; j < 8; j++)  // (slots past the row's last are hidden already)
                        see[j] = mask[min(slot0 + 4 * g + (j >> 2) * 16 + (j & 3), w.hi[n] - 1) * a.mask_ss];
#pragma unroll
                    for (int j = 0; j < 8; j++) {
                        x[n][j] = see[j] ? x[n][j] : KV_NEG;
                        any |= see[j] && (unsigned)((j >> 2) * 16 + (j & 3) - first) < (unsigned)count;
                    }
                }
            }
            if (bad && any) w.bad[n] = __uint_as_float(0x7fc00000u);
            if (scores && w.row[n] >= 0) {
                float4* at = (float4*)(scores + (int64_t)w.row[n] * score_row + slot0);
                at[g] = make_float4(x[n][0], x[n][1], x[n][2], x[n][3]);
                at[4 + g] = make_float4(x[n][4], x[n][5], x[n][6], x[n][7]);
            }
#pragma unroll
            for (int j = 0; j < 8; j++) x[n][j] += base;
        }
    }
#pragma unroll
    for (int n = 0; n < NC; n++) over |= kv_max8(x[n]) > KV_TOP + KV_SLACK;
    if (__any(over)) {
#pragma unroll
        for (int n = 0; n < NC; n++) {
            const bool none = w.t[n] == KV_START;
            if (none) {
                const float f = w.qs[n] * ks, base = fmaxf(lv, w.low[n]);
#pragma unroll
                for (int j = 0; j < 8; j++)
                    x[n][j] = x[n][j] == KV_NEG ? KV_NEG : __builtin_fmaf(u[n][j >> 2][j & 3], f, base);
            }
            const float was = none ? 0.f : w.t[n], best = kv_max4(kv_max8(x[n])) + was - KV_TOP;
            const float now = fmaxf(w.t[n], best);
            const float down = none ? KV_NEG : w.t[n] - now, f1 = exp2f(down);
#pragma unroll
            for (int j = 0; j < 8; j++) x[n][j] += was - now;
            // S follows the scale that moved m, as far as l stays below 2^100
            int up = 0;
            if (now > w.t[n] && lv > w.low[n] + KV_FAR) {
                up = (int)ceilf(lv - (w.low[n] + KV_FAR));
                if (!none)
                    up = max(min(up, 100 - max(__builtin_amdgcn_frexp_expf(kv_max4(w.l[n])), 0) - (int)down), 0);
                w.s[n] = ldexpf(w.s[n], up), w.low[n] += (float)up;
            }
            w.t[n] = now;
            w.l[n] *= exp2f(down + (float)up);
#pragma unroll
            for (int j = 0; j < 2 * S; j++) w.o[n][j] *= f1;
        }
    }
}

// The probabilities of a tile in operand order (p1: their second halves), and the
// denominators' sums.
template <int S, int CODE, int PARTS, int NC, bool SH>
__device__ __forceinline__ void kv_exponents(KvWave<S, CODE, PARTS, NC, SH>& w, const float (&x)[NC][8], float rv,
                                             half8 (&p0)[NC], half8 (&p1)[NC]) {
#pragma unroll
    for (int n = 0; n < NC; n++) {
        float sum = 0.f;
#pragma unroll
        for (int j = 0; j < 8; j++) {
            const float p = __builtin_amdgcn_exp2f(x[n][j]);
            const _Float16 ph = (_Float16)p;
            p0[n][j] = ph;
            if (PARTS > 1) p1[n][j] = (_Float16)(p - (float)ph);
            sum += p;  // (the rounded ones' sum, by dot products, would cost the logarithm its float32)
        }
        w.l[n] = __builtin_fmaf(sum, fminf(rv * w.s[n], KV_FAR_F), w.l[n]);
    }
}

// Products of a tile's keys with the rows.
template <int S, int CODE, int PARTS, bool SH>
__device__ __forceinline__ void kv_scores(const KvWave<S, CODE, PARTS, 1, SH>& w, const uint4 (&kc)[S], floatx4 (&u)[1][2]) {
    u[0][0] = u[0][1] = floatx4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int o = 0; o < 2 * S; o++) {
        const uint4 r = kc[o >> 1];
        const half8 k = o & 1 ? kv_half8<CODE>(r.z, r.w) : kv_half8<CODE>(r.x, r.y);
#pragma unroll
        for (int p = 0; p < PARTS; p++)
            u[0][o / S] = __builtin_amdgcn_mfma_f32_16x16x32_f16(k, w.q[0][p][o % S], u[0][o / S], 0, 0, 0);
    }
}

template <int S, int CODE, int PARTS, bool SH>
__device__ __forceinline__ void kv_add_values(KvWave<S, CODE, PARTS, 1, SH>& w, const uint4 (&vc)[S], const half8& p0, const half8& p1) {
#pragma unroll
    for (int o = 0; o < 2 * S; o++) {
        const uint4 r = vc[o >> 1];
        const half8 v = o & 1 ? kv_half8<CODE>(r.z, r.w) : kv_half8<CODE>(r.x, r.y);
        w.o[0][o] = __builtin_amdgcn_mfma_f32_16x16x32_f16(v, p0, w.o[0][o], 0, 0, 0);
        if (PARTS > 1) w.o[0][o] = __builtin_amdgcn_mfma_f32_16x16x32_f16(v, p1, w.o[0][o], 0, 0, 0);
    }
}

// A half of a tile, 16 contiguous bytes of a lane at a time.  ONCE: no other workgroup reads
// it, so it passes the caches by.
template <int S, bool ONCE>
__device__ __forceinline__ void kv_fetch(uint4 (&k)[S], const uint8_t* half) {
    const u32x4* p = (const u32x4*)half + (threadIdx.x & 63);
#pragma unroll
    for (int s = 0; s < S; s++) k[s] = __builtin_bit_cast(uint4, ONCE ? __builtin_nontemporal_load(p + s * 64) : p[s * 64]);
}

// m of a row, -inf if it has seen no slot.
__device__ __forceinline__ float kv_reached(float t) { return t == KV_START ? KV_NEG : t + KV_TOP; }

// A part leaves its sums o and l, its m less log2 S, and log2 S: of several, l goes by the
// power of 2 that its m stands below the largest, mx, and o by that and by the power that its
// S stands below the largest.  A part without a score has m -inf and l 0, or l NaN where its
// scores were NaN.
__device__ __forceinline__ float kv_join_factor(float m, float l, float mx) {
    return m == KV_NEG ? 0.f * l : exp2f(m - mx);
}

// Index of a row in the outputs, and in the arrays of one head after the other.
__device__ __forceinline__ size_t kv_row(const KvDev& c, const KvBatch& b, const KvAttend& a, int i, int h, int row) {
    return (size_t)(b.tok0[i] + kv_div(row, a.by_group)) * c.H * a.G + h * a.G + kv_mod(row, a.by_group);
}
__device__ __forceinline__ size_t kv_head_row(const KvDev& c, const KvBatch& b, const KvAttend& a, int i, int h, int row) {
    return ((size_t)b.tok0[i] * c.H + (size_t)h * b.count[i]) * a.G + row;
}

// A finished row's logarithm.
__device__ __forceinline__ void kv_finish(const KvDev& c, const KvBatch& b, const KvAttend& a, int i, int h, int row,
                                          float m, float l) {
    const float lse2 = l == 0.f ? KV_NEG : m - KV_TOP + log2f(l);
    if (a.lse) a.lse[kv_row(c, b, a, i, h, row)] = lse2 * 0.69314718055994531f;
    if (a.lse2) a.lse2[kv_head_row(c, b, a, i, h, row)] = lse2;
}

// What a workgroup does: its sequence, split and first row (last splits first, they are
// the shorter ones of their rows, and last rows, which see most, before the first: the
// short work comes at the end), and the tiles t0 .. t1 - 1 that its rows see in its split.
struct KvJob {
    int i, h, split, row0, row1;
    int t0, t1;
    bool whole;  // no other split has tiles
    bool none;   // this one has none
};
__device__ __forceinline__ KvJob kv_job(const KvDev& c, const KvBatch& b, const KvAttend& a, int wg_rows) {
    KvJob j;
    j.h = kv_mod(blockIdx.x, c.by_heads);
    const int unit = kv_div(blockIdx.x, c.by_heads);
    j.i = kv_find(b, unit);
    const int u = unit - b.unit0[j.i], rows = b.count[j.i] * a.G, row_tiles = (rows + wg_rows - 1) / wg_rows;
    const int tile = row_tiles - 1 - u % row_tiles;
    j.split = b.splits[j.i] - 1 - u / row_tiles;
    j.row0 = tile * wg_rows, j.row1 = min(j.row0 + wg_rows, rows);
    int lo0, hi0, lo1, hi1;
    kv_range(a, b.len[j.i], b.count[j.i], j.row0, lo0, hi0);
    kv_range(a, b.len[j.i], b.count[j.i], j.row1 - 1, lo1, hi1);
    const int first = lo0 / KV_TILE, last = (hi1 + KV_TILE - 1) / KV_TILE;
    j.t0 = first + j.split * b.per[j.i], j.t1 = min(j.t0 + b.per[j.i], last);
    j.whole = first + b.per[j.i] >= last;
    j.none = j.split > 0 && j.t0 >= j.t1;
    return j;
}

// The same for an entry of shared slots: tiles b.tok0 .. of the slots up to b.len, for b.count
// rows; the splits go by the entry's tiles, and the rows of one sequence leave out what none
// of them sees.
__device__ __forceinline__ KvJob kv_shared_job(const KvDev& c, const KvBatch& b, const KvAttend& a, const KvMembers& mem, int wg_rows) {
    KvJob j;
    j.h = kv_mod(blockIdx.x, c.by_heads);
    const int unit = kv_div(blockIdx.x, c.by_heads);
    j.i = kv_find(b, unit);
    const int u = unit - b.unit0[j.i], rows = b.count[j.i], row_tiles = (rows + wg_rows - 1) / wg_rows;
    j.split = u / row_tiles;
    j.row0 = (u - j.split * row_tiles) * wg_rows, j.row1 = min(j.row0 + wg_rows, rows);
    j.t0 = b.tok0[j.i] + j.split * b.per[j.i];
    j.t1 = min(j.t0 + b.per[j.i], (b.len[j.i] + KV_TILE - 1) / KV_TILE);
    const int m = b.aux[j.i];
    if (mem.row0[m + 1] - mem.row0[m] >= rows) {
        int lo0, hi0, lo1, hi1;
        kv_range(a, mem.len[m], mem.count[m], j.row0, lo0, hi0);
        kv_range(a, mem.len[m], mem.count[m], j.row1 - 1, lo1, hi1);
        j.t0 = max(j.t0, lo0 / KV_TILE), j.t1 = min(j.t1, (hi1 + KV_TILE - 1) / KV_TILE);
    }
    j.whole = false, j.none = j.t0 >= j.t1;
    return j;
}

// A workgroup without a tile leaves rows that have seen nothing.
__device__ __forceinline__ void kv_no_part(const KvAttend& a, int wg_rows) {
    if ((int)threadIdx.x >= wg_rows) return;
    const size_t at = (size_t)blockIdx.x * wg_rows + threadIdx.x;
    a.part_ml[at] = make_float2(KV_NEG, 0.f), a.part_s[at] = KV_FIRST;
}

// Slots that all rows of a wave see.
template <int S, int CODE, int PARTS, int NC>
__device__ __forceinline__ void kv_all_see(const KvWave<S, CODE, PARTS, NC, true>& w, int& all_lo, int& all_hi) {
    all_lo = 0, all_hi = INT_MAX;
#pragma unroll
    for (int n = 0; n < NC; n++)
        if (w.row[n] >= 0) all_lo = max(all_lo, w.lo[n]), all_hi = min(all_hi, w.hi[n]);
#pragma unroll
    for (int o = 1; o < 16; o <<= 1) all_lo = max(all_lo, __shfl_xor(all_lo, o)), all_hi = min(all_hi, __shfl_xor(all_hi, o));
}

// Few rows: the four waves of a workgroup take the same 16 rows and every fourth tile,
// joined at the end.  The next tile's keys are loaded when this one's are used up, under
// its softmax and values, and its values under the next one's keys: one tile of registers.
// Bound by the cache's bytes: a tile's 64 Dp bytes against Dp / 8 matrix instructions of
// 16 cycles, Dp / 4 for float32 queries (61 sequences up to 8191 slots, 8 x 128: 349 MB in
// 63 us, 5.5 TB/s; 64 to 256 dims, 61 sequences of 4096: 5.6 to 6.3).
// ONCE: no row tile but this one reads the tiles (64 sequences of 4096, 8 x 128, one row tile:
// 86 us, by the caches 97; two row tiles 145 and 129).
template <int S, int CODE, int PARTS, bool ONCE, bool SH>
__global__ __launch_bounds__(256, S <= 4 ? 3 : 2) void kv_step_kernel(KvDev c, KvBatch b, KvAttend a, KvMem<SH> mem) {
    extern __shared__ __align__(16) float lds[];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int col = lane & 15, g = lane >> 4;
    KvJob sp;
    if constexpr (SH) sp = kv_shared_job(c, b, a, mem, 16);
    else sp = kv_job(c, b, a, 16);
    if (sp.none) {
        if (SH) kv_no_part(a, 16);
        return;
    }
    const int i = sp.i, h = sp.h, row0 = sp.row0, row1 = sp.row1;
    const int len = b.len[i], rows = kv_job_rows<SH>(b, a, i);

    const int* table = c.table + (size_t)b.seq[i] * c.W;
    const int64_t score_row = (int64_t)((len + KV_TILE - 1) / KV_TILE) * KV_TILE;
    float* scores = !SH && a.scores ? a.scores + (int64_t)b.aux[i] * KV_TILE * c.H + h * score_row * rows : nullptr;
    int all_lo, all_hi, x0, x1;  // slots that every row sees
    if constexpr (!SH) {
        kv_range(a, len, b.count[i], row0, x0, all_hi);
        kv_range(a, len, b.count[i], row1 - 1, all_lo, x1);
    }

    const int n = max((sp.t1 - sp.t0 - wave + 3) / 4, 0);  // tiles of this wave
    const int tw = sp.t0 + wave;
    KvTiles info = kv_tile_infos(c, table, h, tw, 4, sp.t1);
    const auto tile = [&](const KvTiles& f, int x) { return kv_tile_of(c, f, x & 63); };
    uint4 kc[S], vc[S];
    if (n > 0) kv_fetch<S, ONCE>(kc, tile(info, 0)), kv_fetch<S, ONCE>(vc, tile(info, 0) + kv_half(32 * S));
    KvWave<S, CODE, PARTS, 1, SH> w;
    kv_load_rows(w, c, b, a, mem, i, h, row0);
    if constexpr (SH) kv_all_see(w, all_lo, all_hi);
    for (int x = 0; x < n; x++) {
        const int t = tw + 4 * x, y = x & 63;
        const float ks = kv_lane(info.ks, y), lv = kv_lane(info.lv, y), rv = kv_lane(info.rv, y);
        const bool bad = info.bad >> y & 1;
        if (y == 63 && x + 1 < n) info = kv_tile_infos(c, table, h, t + 4, 4, sp.t1);
        const uint8_t* next = tile(info, x + 1 < n ? x + 1 : x);
        floatx4 u[1][2];
        kv_scores(w, kc, u);
        if (x + 1 < n) kv_fetch<S, ONCE>(kc, next);
        half8 p0[1], p1[1];
        const bool inside = t * KV_TILE >= all_lo && (t + 1) * KV_TILE <= all_hi && !a.mask;
        float z[1][8];
        kv_reference(w, u, ks, lv, bad, t * KV_TILE, inside, a, b.tok0[i], scores, score_row, z);
        kv_exponents(w, z, rv, p0, p1);
        kv_add_values(w, vc, p0[0], p1[0]);
        if (x + 1 < n) kv_fetch<S, ONCE>(vc, next + kv_half(32 * S));
    }
    w.l[0] = kv_sum4(w.l[0]), w.bad[0] = kv_sum4(w.bad[0]);

    // join the four waves: rows of [wave][row][32 S + 4] floats, then (m, l) and S
    constexpr int LDO = 32 * S + 4;
    float* ml = lds + 4 * 16 * LDO;
    const int r4 = wave * 16 + col;
#pragma unroll
    for (int j = 0; j < 2 * S; j++) *(floatx4*)(lds + r4 * LDO + 16 * j + 4 * g) = w.o[0][j] + w.bad[0];
    if (g == 0) ml[2 * r4] = kv_reached(w.t[0]) - (w.low[0] + KV_FAR), ml[2 * r4 + 1] = w.l[0], ml[128 + r4] = w.low[0] + KV_FAR;
    __syncthreads();
    for (int u = threadIdx.x; u < 16 * 8 * S; u += 256) {
        const int r = u / (8 * S), d = u % (8 * S) * 4;
        const int row = row0 + r;
        if (row >= rows) break;
        float mx = KV_NEG, top = KV_FIRST;
#pragma unroll
        for (int x = 0; x < 4; x++) mx = fmaxf(mx, ml[2 * (x * 16 + r)]), top = fmaxf(top, ml[128 + x * 16 + r]);
        floatx4 o = {0.f, 0.f, 0.f, 0.f};
        float l = 0.f;
#pragma unroll
        for (int x = 0; x < 4; x++) {
            const int rr = x * 16 + r;
            const float f = kv_join_factor(ml[2 * rr], ml[2 * rr + 1], mx);
            l += f * ml[2 * rr + 1];
            o += *(const floatx4*)(lds + rr * LDO + d) * ldexpf(f, (int)(ml[128 + rr] - top));
        }
        if (sp.whole) {
            const size_t at = kv_row(c, b, a, i, h, row);
            if (d == 0) kv_finish(c, b, a, i, h, row, mx, l);
            const float inv = l == 0.f ? 0.f : 1.f / l;
            kv_store4<PARTS>(a, at * c.D, d, c.D, o * inv * ldexpf(1.f, (int)top));
        } else {
            const size_t at = (size_t)blockIdx.x * 16 + r;
            if (d == 0) a.part_ml[at] = make_float2(mx, l), a.part_s[at] = top;
            *(floatx4*)(a.part_o + at * (32 * S) + d) = o;
        }
    }
}

// Many rows: the four waves of a workgroup take 4 * NC * 16 rows and every tile.  A tile's
// codes are converted once, a quarter by each wave, and shared as half-precision operands
// through LDS (three buffers, one barrier to a tile); an operand read feeds NC products.
// 2048 tokens over 32768 slots, 8 x 4 x 128: the vector unit is busy 63% of the time and
// the matrix unit 42%; over 16384 slots 980 TFLOP/s, 650 to 810 at other widths, and 400 to
// 560 in float32, which has two products for one.
template <int S, int CODE, int PARTS, int NC, bool SH>
__global__ __launch_bounds__(256, S == 8 ? 1 : 2) void kv_chunk_kernel(KvDev c, KvBatch b, KvAttend a, KvMem<SH> mem) {
    __shared__ half8 tiles[3][4 * S][64];  // operands of keys, then of values
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int g = lane >> 4;
    constexpr int WG_ROWS = 64 * NC;
    KvJob sp;
    if constexpr (SH) sp = kv_shared_job(c, b, a, mem, WG_ROWS);
    else sp = kv_job(c, b, a, WG_ROWS);
    if (sp.none) {
        if (SH) kv_no_part(a, WG_ROWS);
        return;
    }
    const int i = sp.i, h = sp.h, wg_row0 = sp.row0;
    const int len = b.len[i], rows = kv_job_rows<SH>(b, a, i);
    const int row0 = wg_row0 + wave * 16 * NC;

    const int n_tiles = max(sp.t1 - sp.t0, 0);
    KvTiles info = kv_tile_infos(c, c.table + (size_t)b.seq[i] * c.W, h, sp.t0, 1, sp.t1), ahead = info;
    constexpr int PIECES = (2 * S + 3) / 4;  // 16-byte pieces of a lane that a wave converts
    const auto fetch = [&](uint4(&to)[PIECES], const uint8_t* tile) {
        const uint4* p = (const uint4*)tile + lane;
#pragma unroll
        for (int x = 0; x < PIECES; x++)
            if ((x + 1) * 4 <= 2 * S || x * 4 + wave < 2 * S) to[x] = p[(x * 4 + wave) * 64];
    };
    const auto stage = [&](int buf, const uint4(&from)[PIECES]) {
#pragma unroll
        for (int x = 0; x < PIECES; x++)
            if ((x + 1) * 4 <= 2 * S || x * 4 + wave < 2 * S) {
                tiles[buf][2 * (x * 4 + wave)][lane] = kv_half8<CODE>(from[x].x, from[x].y);
                tiles[buf][2 * (x * 4 + wave) + 1][lane] = kv_half8<CODE>(from[x].z, from[x].w);
            }
    };
    // the first three tiles and the rows are on the way together
    uint4 next[PIECES];
    KvWave<S, CODE, PARTS, NC, SH> w;
    if (n_tiles > 0) {
        uint4 tile0[PIECES], tile1[PIECES];
        fetch(tile0, kv_tile_of(c, info, 0));
        fetch(tile1, kv_tile_of(c, info, min(n_tiles - 1, 1)));
        fetch(next, kv_tile_of(c, info, min(n_tiles - 1, 2)));
        kv_load_rows(w, c, b, a, mem, i, h, row0);
        stage(0, tile0);
        stage(1, tile1);
    } else {
        kv_load_rows(w, c, b, a, mem, i, h, row0);
    }
    int all_lo = 0, all_hi = 0, x0, x1;  // slots that every row of this wave sees
    if constexpr (SH) {
        kv_all_see(w, all_lo, all_hi);
    } else if (row0 < rows) {
        kv_range(a, len, b.count[i], row0, x0, all_hi);
        kv_range(a, len, b.count[i], min(row0 + 16 * NC, rows) - 1, all_lo, x1);
    }
    if (!SH && a.qop && sp.split == 0) {
#pragma unroll
        for (int n = 0; n < NC; n++) {
            const int tile = row0 / 16 + n;
            if (tile * 16 >= rows) continue;
            uint4* to = a.qop + ((size_t)b.aux[i] * c.H + (size_t)h * ((rows + 15) / 16) + tile) * (PARTS * S * 64);
#pragma unroll
            for (int x = 0; x < PARTS * S; x++) to[x * 64 + lane] = __builtin_bit_cast(uint4, w.q[n][x / S][x % S]);
            kv_rows_again(w, a, n);
            if (g == 0 && w.row[n] >= 0) a.qs[kv_head_row(c, b, a, i, h, w.row[n])] = w.qs[n];
        }
    }
    // Step t: the exponentials and values of tile t stand beside the keys' products of
    // tile t + 1, so the vector and the matrix unit have independent work; tile t + 2 goes
    // to LDS, t + 3 to registers.  (Two buffers, values one step later, freed LDS that no
    // wave could use and took 1311 us for 1218: two addresses to a step.)
    const auto products = [&](const half8(&k)[2 * S], floatx4(&u)[NC][2]) {
#pragma unroll
        for (int n = 0; n < NC; n++) u[n][0] = u[n][1] = floatx4{0.f, 0.f, 0.f, 0.f};
        // 2 NC sums in turn, so that no product waits for the one before it
#pragma unroll
        for (int s = 0; s < S; s++)
#pragma unroll
            for (int p = 0; p < PARTS; p++)
#pragma unroll
                for (int j = 0; j < 2; j++)
#pragma unroll
                    for (int n = 0; n < NC; n++)
                        u[n][j] = __builtin_amdgcn_mfma_f32_16x16x32_f16(k[j * S + s], w.q[n][p][s], u[n][j], 0, 0, 0);
    };
    floatx4 u[NC][2];
    __syncthreads();
    if (n_tiles > 0) {
        half8 kop[2 * S];
#pragma unroll
        for (int o = 0; o < 2 * S; o++) kop[o] = tiles[0][o][lane];
        products(kop, u);
    }
    int b0 = 0, b1 = 1, b2 = 2;  // buffers of tiles t, t + 1, t + 2
    for (int xt = 0; xt < n_tiles; xt++) {
        const int t = sp.t0 + xt, y = xt & 63;
        if (y == 0 && xt > 0) info = ahead;
        const bool inside = t * KV_TILE >= all_lo && (t + 1) * KV_TILE <= all_hi && !a.mask;
        const float rv = kv_lane(info.rv, y);
        float z[NC][8];
        half8 kop[2 * S], vop[2 * S];
#pragma unroll
        for (int o = 0; o < 2 * S; o++) kop[o] = tiles[b1][o][lane];
        kv_reference(w, u, kv_lane(info.ks, y), kv_lane(info.lv, y), info.bad >> y & 1, t * KV_TILE, inside, a, b.tok0[i],
                     nullptr, 0, z);
        if (y == 60) ahead = kv_tile_infos(c, c.table + (size_t)b.seq[i] * c.W, h, t + 4, 1, sp.t1);
        half8 p0[NC], p1[NC];
        // past the last tile this works on what lies there, and is not used
#pragma unroll
        for (int o = 0; o < 2 * S; o++) vop[o] = tiles[b0][2 * S + o][lane];
        // the loads first: their use waits behind the keys' products (two halves: no registers for it)
        if (PARTS == 1) __builtin_amdgcn_sched_barrier(0);
        // a wave among its products yields to one that prepares its own, so that the two waves of a
        // SIMD part company (2048 tokens over 32768 slots: 1248 us without, 1147 the other way round,
        // 1120 so; eight waves to a workgroup instead: 1168)
        __builtin_amdgcn_s_setprio(0);
        products(kop, u);
        kv_exponents(w, z, rv, p0, p1);
#pragma unroll
        for (int o = 0; o < 2 * S; o++) {
#pragma unroll
            for (int n = 0; n < NC; n++) {
                w.o[n][o] = __builtin_amdgcn_mfma_f32_16x16x32_f16(vop[o], p0[n], w.o[n][o], 0, 0, 0);
                if (PARTS > 1) w.o[n][o] = __builtin_amdgcn_mfma_f32_16x16x32_f16(vop[o], p1[n], w.o[n][o], 0, 0, 0);
            }
        }
        stage(b2, next);
        __builtin_amdgcn_s_setprio(1);
        if (xt + 3 < n_tiles) fetch(next, y + 3 < 64 ? kv_tile_of(c, info, y + 3) : kv_tile_of(c, ahead, y + 3 - 64));
        __syncthreads();
        const int tmp = b0;
        b0 = b1, b1 = b2, b2 = tmp;
    }
#pragma unroll
    for (int n = 0; n < NC; n++) {
        w.l[n] = kv_sum4(w.l[n]), w.bad[n] = kv_sum4(w.bad[n]);
        kv_rows_again(w, a, n);
        if (w.row[n] < 0) continue;
        const float power = w.low[n] + KV_FAR, m = kv_reached(w.t[n]) - power;
        if (sp.whole) {
            const size_t at = kv_row(c, b, a, i, h, w.row[n]);
            if (g == 0) kv_finish(c, b, a, i, h, w.row[n], m, w.l[n]);
            const float inv = w.l[n] == 0.f ? 0.f : 1.f / w.l[n];
#pragma unroll
            for (int j = 0; j < 2 * S; j++) kv_store4<PARTS>(a, at * c.D, 16 * j + 4 * g, c.D, w.o[n][j] * inv * w.s[n] + w.bad[n]);
        } else {
            const size_t at = (size_t)blockIdx.x * WG_ROWS + (w.row[n] - wg_row0);
            if (g == 0) a.part_ml[at] = make_float2(m, w.l[n]), a.part_s[at] = power;
#pragma unroll
            for (int j = 0; j < 2 * S; j++) *(floatx4*)(a.part_o + at * (32 * S) + 16 * j + 4 * g) = w.o[n][j] + w.bad[n];
        }
    }
}

}  // namespace

}  // namespace vgpu
