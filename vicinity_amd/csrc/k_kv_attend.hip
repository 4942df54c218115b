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
#include "vgpu_kv.h"
#include "vgpu_launch.h"

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

// The running state of a wave: NC column tiles of 16 rows.
template <int S, int CODE, int PARTS, int NC>
struct KvWave {
    half8 q[NC][PARTS][S];
    float qs[NC];          // 2^-(the row's scaling) * scale * log2(e)
    int lo[NC], hi[NC];    // slots that the row sees
    int row[NC];
    int row0, len, count;
    float t[NC], l[NC], bad[NC];  // t: m - KV_TOP
    float s[NC], low[NC];  // S; log2 S - KV_FAR
    floatx4 o[NC][2 * S];
};

template <int S, int CODE, int PARTS, int NC>
__device__ __forceinline__ void kv_load_rows(KvWave<S, CODE, PARTS, NC>& w, const KvDev& c, const KvBatch& b,
                                             const KvAttend& a, int i, int h, int row0) {
    const int lane = threadIdx.x & 63, col = lane & 15, g = lane >> 4;
    const int rows = b.count[i] * a.G, len = b.len[i];
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
        const int64_t base = (int64_t)(b.tok0[i] + kv_div(real, a.by_group)) * a.q.st + (int64_t)(h * a.G + kv_mod(real, a.by_group)) * a.q.sh;
        if (row < rows) kv_range(a, len, b.count[i], row, w.lo[n], w.hi[n]);
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
template <int S, int CODE, int PARTS, int NC>
__device__ __forceinline__ void kv_rows_again(KvWave<S, CODE, PARTS, NC>& w, const KvAttend& a, int n) {
    if (NC <= 2) return;
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
template <int S, int CODE, int PARTS, int NC>
__device__ __forceinline__ void kv_reference(KvWave<S, CODE, PARTS, NC>& w, const floatx4 (&u)[NC][2], float ks, float lv,
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
                    const uint8_t* mask = a.mask + (int64_t)(tok0 + kv_div(max(w.row[n], 0), a.by_group)) * a.mask_st;
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
template <int S, int CODE, int PARTS, int NC>
__device__ __forceinline__ void kv_exponents(KvWave<S, CODE, PARTS, NC>& w, const float (&x)[NC][8], float rv,
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
template <int S, int CODE, int PARTS>
__device__ __forceinline__ void kv_scores(const KvWave<S, CODE, PARTS, 1>& w, const uint4 (&kc)[S], floatx4 (&u)[1][2]) {
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

template <int S, int CODE, int PARTS>
__device__ __forceinline__ void kv_add_values(KvWave<S, CODE, PARTS, 1>& w, const uint4 (&vc)[S], const half8& p0, const half8& p1) {
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

// Few rows: the four waves of a workgroup take the same 16 rows and every fourth tile,
// joined at the end.  The next tile's keys are loaded when this one's are used up, under
// its softmax and values, and its values under the next one's keys: one tile of registers.
// Bound by the cache's bytes: a tile's 64 Dp bytes against Dp / 8 matrix instructions of
// 16 cycles, Dp / 4 for float32 queries (61 sequences up to 8191 slots, 8 x 128: 349 MB in
// 63 us, 5.5 TB/s; 64 to 256 dims, 61 sequences of 4096: 5.6 to 6.3).
// ONCE: no row tile but this one reads the tiles (64 sequences of 4096, 8 x 128, one row tile:
// 86 us, by the caches 97; two row tiles 145 and 129).
template <int S, int CODE, int PARTS, bool ONCE>
__global__ __launch_bounds__(256, S <= 4 ? 3 : 2) void kv_step_kernel(KvDev c, KvBatch b, KvAttend a) {
    extern __shared__ __align__(16) float lds[];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int col = lane & 15, g = lane >> 4;
    const KvJob sp = kv_job(c, b, a, 16);
    if (sp.none) return;
    const int i = sp.i, h = sp.h, row0 = sp.row0, row1 = sp.row1;
    const int len = b.len[i], rows = b.count[i] * a.G;

    const int* table = c.table + (size_t)b.seq[i] * c.W;
    const int64_t score_row = (int64_t)((len + KV_TILE - 1) / KV_TILE) * KV_TILE;
    float* scores = a.scores ? a.scores + (int64_t)b.aux[i] * KV_TILE * c.H + h * score_row * rows : nullptr;
    int all_lo, all_hi, x0, x1;  // slots that every row sees
    kv_range(a, len, b.count[i], row0, x0, all_hi);
    kv_range(a, len, b.count[i], row1 - 1, all_lo, x1);

    const int n = max((sp.t1 - sp.t0 - wave + 3) / 4, 0);  // tiles of this wave
    const int tw = sp.t0 + wave;
    KvTiles info = kv_tile_infos(c, table, h, tw, 4, sp.t1);
    const auto tile = [&](const KvTiles& f, int x) { return kv_tile_of(c, f, x & 63); };
    uint4 kc[S], vc[S];
    if (n > 0) kv_fetch<S, ONCE>(kc, tile(info, 0)), kv_fetch<S, ONCE>(vc, tile(info, 0) + kv_half(32 * S));
    KvWave<S, CODE, PARTS, 1> w;
    kv_load_rows(w, c, b, a, i, h, row0);
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
template <int S, int CODE, int PARTS, int NC>
__global__ __launch_bounds__(256, S == 8 ? 1 : 2) void kv_chunk_kernel(KvDev c, KvBatch b, KvAttend a) {
    __shared__ half8 tiles[3][4 * S][64];  // operands of keys, then of values
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int g = lane >> 4;
    constexpr int WG_ROWS = 64 * NC;
    const KvJob sp = kv_job(c, b, a, WG_ROWS);
    if (sp.none) return;
    const int i = sp.i, h = sp.h, wg_row0 = sp.row0;
    const int len = b.len[i], rows = b.count[i] * a.G;
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
    KvWave<S, CODE, PARTS, NC> w;
    if (n_tiles > 0) {
        uint4 tile0[PIECES], tile1[PIECES];
        fetch(tile0, kv_tile_of(c, info, 0));
        fetch(tile1, kv_tile_of(c, info, min(n_tiles - 1, 1)));
        fetch(next, kv_tile_of(c, info, min(n_tiles - 1, 2)));
        kv_load_rows(w, c, b, a, i, h, row0);
        stage(0, tile0);
        stage(1, tile1);
    } else {
        kv_load_rows(w, c, b, a, i, h, row0);
    }
    int all_lo = 0, all_hi = 0, x0, x1;  // slots that every row of this wave sees
    if (row0 < rows) {
        kv_range(a, len, b.count[i], row0, x0, all_hi);
        kv_range(a, len, b.count[i], min(row0 + 16 * NC, rows) - 1, all_lo, x1);
    }
    if (a.qop && sp.split == 0) {
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

// Joins the splits of rows whose tiles went to several workgroups; Dp / 4 threads read a
// partial row.  WIDE: a workgroup per row, its thread groups take splits in turn (steps of
// many splits and few rows); else a thread group per row (chunks of few splits and many
// rows).  unit0 counts row tiles here, aux is the first of the sequence's units.
template <bool WIDE>
__global__ __launch_bounds__(256) void kv_join_kernel(KvDev c, KvBatch b, KvAttend a, int wg_rows, int used_rows) {
    __shared__ floatx4 sh_o[256];
    __shared__ float sh_l[64];
    const int tid = threadIdx.x;
    const int width = c.Dp / 4, groups = 256 / width, grp = tid / width, d4 = tid % width;
    const int per_wg = WIDE ? 1 : groups, pieces = (used_rows + per_wg - 1) / per_wg;
    const int h = kv_mod(blockIdx.x, c.by_heads), piece = kv_div(blockIdx.x, c.by_heads) % pieces, unit = kv_div(blockIdx.x, c.by_heads) / pieces;
    const int i = kv_find(b, unit);
    const int rows = b.count[i] * a.G, u = unit - b.unit0[i];
    const int row0 = (b.unit0[i + 1] - b.unit0[i] - 1 - u) * wg_rows;
    const int r = WIDE ? piece : piece * groups + grp, row = row0 + r;
    int lo0, hi0, lo1, hi1;
    kv_range(a, b.len[i], b.count[i], row0, lo0, hi0);
    kv_range(a, b.len[i], b.count[i], min(row0 + wg_rows, rows) - 1, lo1, hi1);
    const int tiles = (hi1 + KV_TILE - 1) / KV_TILE - lo0 / KV_TILE;
    const int splits = (tiles + b.per[i] - 1) / b.per[i];
    if (splits <= 1) return;  // the one workgroup has written the rows
    if (WIDE ? row >= rows : (grp >= groups || r >= wg_rows || row >= rows)) return;
    const int row_tiles = b.unit0[i + 1] - b.unit0[i];
    const int64_t stride = -(int64_t)row_tiles * c.H * wg_rows;  // the first split's parts lie last
    const int64_t base = ((int64_t)(b.aux[i] + u + (b.splits[i] - 1) * row_tiles) * c.H + h) * wg_rows + r;
    float mx = KV_NEG, top = KV_FIRST;
    if (WIDE) {
        for (int s = tid & 63; s < splits; s += 64)
            mx = fmaxf(mx, a.part_ml[base + s * stride].x), top = fmaxf(top, a.part_s[base + s * stride]);
#pragma unroll
        for (int x = 32; x; x >>= 1) mx = fmaxf(mx, __shfl_xor(mx, x)), top = fmaxf(top, __shfl_xor(top, x));
    } else {
        for (int s = 0; s < splits; s++)
            mx = fmaxf(mx, a.part_ml[base + s * stride].x), top = fmaxf(top, a.part_s[base + s * stride]);
    }
    floatx4 o = {0.f, 0.f, 0.f, 0.f};
    float l = 0.f;
    if (grp < groups) {
#pragma unroll 4
        for (int s = WIDE ? grp : 0; s < splits; s += WIDE ? groups : 1) {
            const float2 ml = a.part_ml[base + s * stride];
            const float f = kv_join_factor(ml.x, ml.y, mx);
            l += f * ml.y;
            o += *(const floatx4*)(a.part_o + (base + s * stride) * c.Dp + d4 * 4) * ldexpf(f, (int)(a.part_s[base + s * stride] - top));
        }
    }
    if (WIDE) {
        if (grp < groups) {
            sh_o[tid] = o;
            if (d4 == 0) sh_l[grp] = l;
        }
        __syncthreads();
        if (tid >= width) return;
        for (int x = 1; x < groups; x++) o += sh_o[x * width + tid];
        l = sh_l[0];
        for (int x = 1; x < groups; x++) l += sh_l[x];
    }
    if (d4 == 0) kv_finish(c, b, a, i, h, row, mx, l);
    const size_t at = kv_row(c, b, a, i, h, row) * c.D;
    o = o * (l == 0.f ? 0.f : 1.f / l) * ldexpf(1.f, (int)top);
    if (a.q.type == KV_F32)
        kv_store4<2>(a, at, 4 * d4, c.D, o);
    else
        kv_store4<1>(a, at, 4 * d4, c.D, o);
}

// Weights from the kept scores of a step: four slots to a thread, bound by the scores' bytes.
__global__ __launch_bounds__(256) void kv_score_weights_kernel(KvDev c, KvBatch b, KvAttend a) {
    const int h = kv_mod(blockIdx.x, c.by_heads), unit = kv_div(blockIdx.x, c.by_heads);
    const int i = kv_find(b, unit);
    const int slot = (unit - b.unit0[i]) * KV_SCORE_SLOTS + threadIdx.x * 4;
    const int len = b.len[i], rows = b.count[i] * a.G;
    if (slot >= len) return;
    const int64_t score_row = (int64_t)((len + KV_TILE - 1) / KV_TILE) * KV_TILE;
    const float* scores = a.scores + (int64_t)b.aux[i] * KV_TILE * c.H + h * score_row * rows + slot;
    const float* lses = a.lse2 + kv_head_row(c, b, a, i, h, 0);
    floatx4 sum = {0.f, 0.f, 0.f, 0.f};
#pragma unroll 4
    for (int r = 0; r < rows; r++) {
        int lo, hi;
        kv_range(a, len, b.count[i], r, lo, hi);
        const float lse = lses[r];
        // scores exist for the tiles of the row's workgroup only; -inf: it sees nothing
        if (slot + 3 < lo || slot >= hi || lse == KV_NEG) continue;
        const floatx4 x = *(const floatx4*)(scores + (int64_t)r * score_row);
#pragma unroll
        for (int e = 0; e < 4; e++)
            if (slot + e >= lo && slot + e < hi) sum[e] += __builtin_amdgcn_exp2f(x[e] - lse);
    }
    const int block = c.table[(size_t)b.seq[i] * c.W + (slot >> c.shift)];
    float* w = c.weights + ((size_t)block * c.H + h) * c.B + (slot & (c.B - 1));
#pragma unroll
    for (int e = 0; e < 4; e++)
        if (slot + e < len) w[e] = a.decay == 0.f ? sum[e] : a.decay * w[e] + sum[e];
}

// Weights of calls with many rows, by a second pass over the keys:  w_j = sum_r
// 2^(u_rj - lse_r).  The attention left its query operands (a.qop) and each row's
// factor (a.qs) and logarithm.  A wave holds the operands of KV_WT tiles and goes over
// the rows of its chunk, 32 at a time through LDS, which the four waves share; the
// chunks' sums are added in their order by kv_chunk_weights_kernel.  Bound by waits, at the
// loads and the barrier of each 32 rows: prompts of 4001, 2036 and 604 tokens, 4 x 4 x 128,
// take 92 us, of which the vector unit is busy 42% and the matrix unit 19%.
constexpr int KV_WT = 1;              // 32-slot tiles of a wave
static_assert(KV_WEIGHT_SLOTS == 4 * KV_WT * KV_TILE, "four waves of KV_WT tiles");

template <int S, int CODE, int PARTS>
__global__ __launch_bounds__(256, 2) void kv_tile_weights_kernel(KvDev c, KvBatch b, KvAttend a) {
    extern __shared__ __align__(16) uint4 qbuf[];  // [2][2 row tiles][PARTS * S][64]
    constexpr int QT = PARTS * S * 64;             // 16-byte pieces of a row tile
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int g = lane >> 4, col = lane & 15;
    const int h = kv_mod(blockIdx.x, c.by_heads), chunk = kv_div(blockIdx.x, c.by_heads) % a.chunks, unit = kv_div(blockIdx.x, c.by_heads) / a.chunks;
    const int i = kv_find(b, unit);
    const int len = b.len[i], count = b.count[i], rows = count * a.G;
    const int slots0 = (unit - b.unit0[i]) * KV_WEIGHT_SLOTS;
    const int t0 = slots0 / KV_TILE + wave * KV_WT;
    const int* table = c.table + (size_t)b.seq[i] * c.W;
    const int per_block = c.shift - 5;
    // rows of the chunk that see a slot of the workgroup
    int r0 = chunk * a.chunk_rows, r1 = min(r0 + a.chunk_rows, rows);
    if (a.causal) {
        // token p sees slot0 from p = slot0 on: row (slot0 - (len - count)) * G
        const int tok = slots0 - (len - count);
        if (tok > 0) r0 = max(r0, (int)min((int64_t)tok * a.G, (int64_t)rows) / 32 * 32);
    }
    if (a.window) {
        const int64_t tok = (int64_t)min(slots0 + KV_WEIGHT_SLOTS, len) - 1 + a.window - (len - count);
        r1 = (int)min((int64_t)r1, max(tok, (int64_t)0) * a.G);
    }
    half8 k[KV_WT][2 * S];
    float ks[KV_WT];
#pragma unroll
    for (int x = 0; x < KV_WT; x++) {
        ks[x] = 0.f;
        const bool in = (t0 + x) * KV_TILE < len;
        const int t = in ? t0 + x : 0;  // a tile past the end: any that exists, unused
        const int block = __builtin_amdgcn_readfirstlane(table[t >> per_block]);
        ks[x] = c.kscale[(size_t)block * c.H + h];
        const uint4* p = (const uint4*)(c.pool + kv_tile_offset(c, block, h, t & ((1 << per_block) - 1))) + lane;
#pragma unroll
        for (int s = 0; s < S; s++) {
            const uint4 r = p[s * 64];
            k[x][2 * s] = kv_half8<CODE>(r.x, r.y);
            k[x][2 * s + 1] = kv_half8<CODE>(r.z, r.w);
        }
    }
    // Rows any_lo .. any_hi - 1 see some slot of the wave's tiles, all_lo .. all_hi - 1 every
    // one: token p sees slots p - window + 1 .. p, and row (p - len + count) G is its first.
    const auto first_row = [&](int64_t p) { return (int)min(max((p - (len - count)) * a.G, (int64_t)0), (int64_t)rows); };
    const int64_t slot_lo = t0 * KV_TILE, slot_hi = (t0 + KV_WT) * KV_TILE;
    const int any_lo = a.causal ? first_row(slot_lo) : 0, all_lo = a.causal ? first_row(slot_hi - 1) : 0;
    const int any_hi = a.window ? first_row(slot_hi - 1 + a.window) : rows, all_hi = a.window ? first_row(slot_lo + a.window) : rows;
    float sum[KV_WT][8] = {};
    const size_t row_base = kv_head_row(c, b, a, i, h, 0);
    const uint4* qop = a.qop + ((size_t)(b.aux[i]) * c.H + (size_t)h * ((rows + 15) / 16)) * QT;
    const int end = min(r1, rows);
    const int last_kib = (rows + 15) / 16 * PARTS * S - 1;  // of the head's operands
    float next_f[2], next_lse[2];  // of this lane's row in the two row tiles
    // straight to LDS, 1 KiB of a wave at a time
    const auto fetch = [&](int r, uint4* to) {
        for (int x = wave; x < 2 * PARTS * S; x += 4)
            __builtin_amdgcn_global_load_lds(
                (const __attribute__((address_space(1))) void*)(qop + (size_t)min(r / 16 * PARTS * S + x, last_kib) * 64 + lane),
                (__attribute__((address_space(3))) void*)(to + x * 64), 16, 0, 0);
#pragma unroll
        for (int y = 0; y < 2; y++) {
            const int row = r + 16 * y + col;
            next_f[y] = row < end ? a.qs[row_base + row] : 0.f;
            next_lse[y] = row < end ? a.lse2[row_base + row] : KV_NEG;
        }
    };
    if (r0 < r1) fetch(r0, qbuf);
    int buf = 0;
    for (int r = r0; r < r1; r += 32, buf ^= 1) {
        const uint4* to = qbuf + buf * 2 * QT;
        float fs[2], ls[2];
#pragma unroll
        for (int y = 0; y < 2; y++) {
            fs[y] = next_f[y];
            ls[y] = next_lse[y] == KV_NEG ? -KV_NEG : next_lse[y];  // sees nothing: every p is 0
        }
        __builtin_amdgcn_s_waitcnt(0x0f70);  // vmcnt(0): the loads to LDS have landed
        __syncthreads();
        if (r + 32 < r1) fetch(r + 32, qbuf + (buf ^ 1) * 2 * QT);
#pragma unroll
        for (int y = 0; y < 2; y++) {
            const int row0 = r + 16 * y, row = row0 + col;
            if (row0 >= end) break;
            if (row0 + 16 <= any_lo || row0 >= any_hi) continue;
            const bool real = row < end;
            const float f = fs[y], lse = ls[y];
            floatx4 u[KV_WT][2];
#pragma unroll
            for (int x = 0; x < KV_WT; x++) u[x][0] = u[x][1] = floatx4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int s = 0; s < S; s++)
#pragma unroll
                for (int p = 0; p < PARTS; p++) {
                    const half8 q = __builtin_bit_cast(half8, to[y * QT + (p * S + s) * 64 + lane]);
#pragma unroll
                    for (int x = 0; x < KV_WT; x++)
#pragma unroll
                        for (int j = 0; j < 2; j++)
                            u[x][j] = __builtin_amdgcn_mfma_f32_16x16x32_f16(k[x][j * S + s], q, u[x][j], 0, 0, 0);
                }
            const bool inside = !a.mask && row0 >= all_lo && min(row0 + 16, rows) <= all_hi;
            if (inside) {
#pragma unroll
                for (int x = 0; x < KV_WT; x++)
#pragma unroll
                    for (int j = 0; j < 8; j++)
                        sum[x][j] += __builtin_amdgcn_exp2f(__builtin_fmaf(u[x][j >> 2][j & 3], f * ks[x], -lse));
            } else {
                int lo = 0, hi = 0;
                if (real) kv_range(a, len, count, row, lo, hi);
#pragma unroll
                for (int x = 0; x < KV_WT; x++)
#pragma unroll
                    for (int j = 0; j < 8; j++) {
                        const int slot = (t0 + x) * KV_TILE + (j >> 2) * 16 + 4 * g + (j & 3);
                        bool see = slot >= lo && slot < hi;
                        if (see && a.mask) see = a.mask[(int64_t)(b.tok0[i] + kv_div(row, a.by_group)) * a.mask_st + slot * a.mask_ss] != 0;
                        sum[x][j] += see ? __builtin_amdgcn_exp2f(__builtin_fmaf(u[x][j >> 2][j & 3], f * ks[x], -lse)) : 0.f;
                    }
            }
        }
    }
#pragma unroll
    for (int x = 0; x < KV_WT; x++)
#pragma unroll
        for (int j = 0; j < 8; j++) {
            float v = sum[x][j];
#pragma unroll
            for (int y = 1; y < 16; y <<= 1) v += __shfl_xor(v, y);
            // partial sums of the chunk: [unit, H, chunk, slot of the workgroup]
            const int slot = (wave * KV_WT + x) * KV_TILE + (j >> 2) * 16 + 4 * g + (j & 3);
            if (col == j) a.wpart[(((size_t)unit * c.H + h) * a.chunks + chunk) * KV_WEIGHT_SLOTS + slot] = v;
        }
}

// A thread per slot: the chunks' sums, and the weight.
__global__ __launch_bounds__(KV_WEIGHT_SLOTS) void kv_chunk_weights_kernel(KvDev c, KvBatch b, KvAttend a) {
    const int h = kv_mod(blockIdx.x, c.by_heads), unit = kv_div(blockIdx.x, c.by_heads);
    const int i = kv_find(b, unit);
    const int slot = (unit - b.unit0[i]) * KV_WEIGHT_SLOTS + threadIdx.x;
    if (slot >= b.len[i]) return;
    float sum = 0.f;
    for (int x = 0; x < a.chunks; x++)
        sum += a.wpart[(((size_t)unit * c.H + h) * a.chunks + x) * KV_WEIGHT_SLOTS + threadIdx.x];
    const int block = c.table[(size_t)b.seq[i] * c.W + (slot >> c.shift)];
    float* w = c.weights + ((size_t)block * c.H + h) * c.B + (slot & (c.B - 1));
    *w = a.decay == 0.f ? sum : a.decay * *w + sum;
}

template <int S, int CODE, int PARTS>
void attend_s(const KvDev& c, const KvBatch& b, const KvAttend& a, hipStream_t s) {
    const dim3 grid((unsigned)b.unit0[b.n] * c.H);
    if (a.by_rows) {
        hipLaunchKernelGGL((kv_chunk_kernel<S, CODE, PARTS, kv_chunk_nc(S * 32, PARTS)>), grid, dim3(256), 0, s, c, b, a);
        return;
    }
    const size_t lds = (size_t)4 * 16 * (32 * S + 4 + 3) * 4;
    int most = 0;
    for (int i = 0; i < b.n; i++) most = b.count[i] * a.G > most ? b.count[i] * a.G : most;
    const auto kernel = most <= 16 ? kv_step_kernel<S, CODE, PARTS, true> : kv_step_kernel<S, CODE, PARTS, false>;
    if (lds > 65536) ensure_dyn_lds((const void*)kernel, lds);
    hipLaunchKernelGGL(kernel, grid, dim3(256), lds, s, c, b, a);
}

template <int S, int CODE, int PARTS>
void weights_s(const KvDev& c, const KvBatch& b, const KvAttend& a, hipStream_t s) {
    const size_t lds = (size_t)2 * 2 * PARTS * S * 1024;
    const auto kernel = kv_tile_weights_kernel<S, CODE, PARTS>;
    if (lds > 65536) ensure_dyn_lds((const void*)kernel, lds);
    hipLaunchKernelGGL(kernel, dim3((unsigned)b.unit0[b.n] * c.H * a.chunks), dim3(256), lds, s, c, b, a);
}

template <int CODE, int PARTS, bool WEIGHTS>
void by_dim(const KvDev& c, const KvBatch& b, const KvAttend& a, hipStream_t s) {
    switch (c.Dp / 32) {
#define KV_CASE(S)                                  \
    case S:                                         \
        if (WEIGHTS)                                \
            weights_s<S, CODE, PARTS>(c, b, a, s);  \
        else                                        \
            attend_s<S, CODE, PARTS>(c, b, a, s);   \
        break;
        KV_CASE(2)
        KV_CASE(3)
        KV_CASE(4)
        KV_CASE(6)
        KV_CASE(8)
#undef KV_CASE
    }
}

template <bool WEIGHTS>
void by_type(const KvDev& c, const KvBatch& b, const KvAttend& a, hipStream_t s) {
    const bool two = a.q.type == KV_F32;
    if (c.code == KV_INT8)
        two ? by_dim<KV_INT8, 2, WEIGHTS>(c, b, a, s) : by_dim<KV_INT8, 1, WEIGHTS>(c, b, a, s);
    else
        two ? by_dim<KV_FP8, 2, WEIGHTS>(c, b, a, s) : by_dim<KV_FP8, 1, WEIGHTS>(c, b, a, s);
}

}  // namespace

void launch_kv_attend(const KvDev& c, const KvBatch& b, const KvAttend& a, hipStream_t s) {
    if (!b.unit0[b.n]) return;
    by_type<false>(c, b, a, s);
    // the sequences with several splits, by row tiles
    const int wg_rows = kv_attend_rows(a, c.Dp);
    KvBatch j = b;
    int used = 1;
    for (int i = 0; i < b.n; i++) {
        const int rows = b.count[i] * a.G, tiles = b.splits[i] > 1 ? (rows + wg_rows - 1) / wg_rows : 0;
        j.aux[i] = b.unit0[i];
        j.unit0[i + 1] = j.unit0[i] + tiles;
        if (tiles && rows > used) used = rows < wg_rows ? rows : wg_rows;
    }
    if (!j.unit0[j.n]) return;
    if (a.by_rows) {
        const int per_wg = 256 / (c.Dp / 4);
        hipLaunchKernelGGL(kv_join_kernel<false>, dim3((unsigned)j.unit0[j.n] * c.H * ((used + per_wg - 1) / per_wg)),
                           dim3(256), 0, s, c, j, a, wg_rows, used);
    } else {
        hipLaunchKernelGGL(kv_join_kernel<true>, dim3((unsigned)j.unit0[j.n] * c.H * used), dim3(256), 0, s, c, j, a,
                           wg_rows, used);
    }
}

void launch_kv_weights(const KvDev& c, const KvBatch& b, const KvAttend& a, hipStream_t s) {
    if (!b.unit0[b.n]) return;
    const dim3 grid((unsigned)b.unit0[b.n] * c.H);
    if (!a.by_rows) {  // (a.scores is null where no row has a slot: none is read then)
        hipLaunchKernelGGL(kv_score_weights_kernel, grid, dim3(256), 0, s, c, b, a);
        return;
    }
    by_type<true>(c, b, a, s);
    hipLaunchKernelGGL(kv_chunk_weights_kernel, grid, dim3(KV_WEIGHT_SLOTS), 0, s, c, b, a);
}

}  // namespace vgpu
