// Softmax attention over the 8-bit cache: a sequence's rows by themselves (kv_attend.h), the
// join of split rows, and accumulated weights.
#include "kv_attend.h"

namespace vgpu {

namespace {

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
        hipLaunchKernelGGL((kv_chunk_kernel<S, CODE, PARTS, kv_chunk_nc(S * 32, PARTS), false>), grid, dim3(256), 0, s, c, b, a,
                           KvAlone{});
        return;
    }
    const size_t lds = (size_t)4 * 16 * (32 * S + 4 + 3) * 4;
    int most = 0;
    for (int i = 0; i < b.n; i++) most = b.count[i] * a.G > most ? b.count[i] * a.G : most;
    const auto kernel = most <= 16 ? kv_step_kernel<S, CODE, PARTS, true, false> : kv_step_kernel<S, CODE, PARTS, false, false>;
    if (lds > 65536) ensure_dyn_lds((const void*)kernel, lds);
    hipLaunchKernelGGL(kernel, grid, dim3(256), lds, s, c, b, a, KvAlone{});
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
