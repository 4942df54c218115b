// The attention memory: quantising append, reading back, the block table.
//
// append  s = amax * (1 / Z) per (block, head), codes round(x / s): two passes over the
//         new elements, the second from L2.  Bound by the bytes in and out.
// read    code * s.
// Rounding: codes are the cache's format; every value before them is float32.
#include "vgpu_kv.h"

#include <climits>
#include <hip/hip_bf16.h>
#include <hip/hip_fp16.h>

namespace vgpu {

namespace {

// Scales are 0 below this largest magnitude, so 1 / s stays finite.
constexpr float KV_TINY = 0x1p-100f;

__device__ __forceinline__ float to_f32(const void* p, int64_t i, int type) {
    if (type == KV_F32) return ((const float*)p)[i];
    if (type == KV_F16) return (float)((const _Float16*)p)[i];
    return __uint_as_float((uint32_t)((const uint16_t*)p)[i] << 16);
}

// dims 8 m .. 8 m + 7 of a row (0 from D on)
template <int T>
__device__ __forceinline__ void load8(const KvTensor& x, int64_t row, int m, int D, float* v) {
    if (x.vec) {
        if (T == KV_F32) {
            const float4* p = (const float4*)((const float*)x.p + row + 8 * m);
            const float4 a = p[0], b = p[1];
            v[0] = a.x, v[1] = a.y, v[2] = a.z, v[3] = a.w;
            v[4] = b.x, v[5] = b.y, v[6] = b.z, v[7] = b.w;
        } else {
            const uint4 a = *(const uint4*)((const uint16_t*)x.p + row + 8 * m);
            const uint32_t w[4] = {a.x, a.y, a.z, a.w};
#pragma unroll
            for (int e = 0; e < 8; e++) {
                const uint16_t h = (uint16_t)(w[e >> 1] >> (16 * (e & 1)));
                v[e] = T == KV_F16 ? (float)__builtin_bit_cast(_Float16, h) : __uint_as_float((uint32_t)h << 16);
            }
        }
    } else {
#pragma unroll
        for (int e = 0; e < 8; e++) {
            const int d = 8 * m + e;
            v[e] = d < D ? to_f32(x.p, row + d * x.sd, T) : 0.f;
        }
    }
}

__device__ __forceinline__ uint32_t encode4(float a, float b, float c, float d, int code) {
    if (code == KV_INT8) {
        const int i0 = (int)rintf(fminf(fmaxf(a, -127.f), 127.f)) + 128, i1 = (int)rintf(fminf(fmaxf(b, -127.f), 127.f)) + 128;
        const int i2 = (int)rintf(fminf(fmaxf(c, -127.f), 127.f)) + 128, i3 = (int)rintf(fminf(fmaxf(d, -127.f), 127.f)) + 128;
        return (uint32_t)i0 | (uint32_t)i1 << 8 | (uint32_t)i2 << 16 | (uint32_t)i3 << 24;
    }
    a = fminf(fmaxf(a, -448.f), 448.f), b = fminf(fmaxf(b, -448.f), 448.f);
    c = fminf(fmaxf(c, -448.f), 448.f), d = fminf(fmaxf(d, -448.f), 448.f);
    int w = __builtin_amdgcn_cvt_pk_fp8_f32(a, b, 0, false);
    w = __builtin_amdgcn_cvt_pk_fp8_f32(c, d, w, true);
    return (uint32_t)w;
}

__device__ __forceinline__ void decode4(uint32_t w, int code, float* v) {
    if (code == KV_INT8) {
#pragma unroll
        for (int e = 0; e < 4; e++) v[e] = (float)(int)((w >> (8 * e)) & 255u) - 128.f;
        return;
    }
    typedef float f2 __attribute__((ext_vector_type(2)));
    const f2 lo = __builtin_amdgcn_cvt_pk_f32_fp8((int)w, false), hi = __builtin_amdgcn_cvt_pk_f32_fp8((int)w, true);
    v[0] = lo.x, v[1] = lo.y, v[2] = hi.x, v[3] = hi.y;
}

__device__ __forceinline__ uint32_t zero_codes(int code) { return code == KV_INT8 ? 0x80808080u : 0u; }

__device__ __forceinline__ uint32_t rescale4(uint32_t w, float r, int code) {
    float v[4];
    decode4(w, code, v);
    return encode4(v[0] * r, v[1] * r, v[2] * r, v[3] * r, code);
}

__global__ __launch_bounds__(256) void kv_table_kernel(int* table, KvRuns r) {
    const int i = blockIdx.x;
    for (int j = threadIdx.x; j < r.count[i]; j += blockDim.x) table[r.at[i] + j] = r.block[i] + j;
}

// One workgroup: the keys or the values of one (block, head) that new tokens enter.
template <int T>
__global__ __launch_bounds__(256) void kv_append_kernel(KvDev c, KvBatch b, KvTensor k, KvTensor v,
                                                        const int* __restrict__ positions,
                                                        const float* __restrict__ weights) {
    __shared__ __align__(16) uint8_t image[KV_TILE * KV_MAX_DIM];
    __shared__ uint32_t red[4];
    const int tid = threadIdx.x;
    const bool vals = blockIdx.x & 1;
    const int h = (blockIdx.x >> 1) % c.H, unit = (blockIdx.x >> 1) / c.H;
    const int i = kv_find(b, unit);
    const int len0 = b.len[i], len1 = len0 + b.count[i];
    const int blk = (len0 >> c.shift) + unit - b.unit0[i];
    const int slot0 = blk << c.shift;
    const int held = max(len0 - slot0, 0), end = min(len1 - slot0, c.B);  // new slots held .. end - 1
    const int block = c.table[(size_t)b.seq[i] * c.W + blk];
    const size_t part = (size_t)block * c.H + h;
    const KvTensor& x = vals ? v : k;
    const int64_t tok0 = (int64_t)b.tok0[i] + slot0 - len0;  // token of slot 0 of the block
    const int S = c.Dp / 32;
    const int Md = (c.D + 7) / 8;

    // largest magnitude, as bits: infinities and NaN are above every number
    uint32_t big = 0;
    for (int u = tid; u < (end - held) * Md; u += 256) {
        const int r = held + u / Md, m = u % Md;
        float e[8];
        load8<T>(x, (tok0 + r) * x.st + (int64_t)h * x.sh, m, c.D, e);
#pragma unroll
        for (int j = 0; j < 8; j++) big = max(big, __float_as_uint(e[j]) & 0x7fffffffu);
    }
#pragma unroll
    for (int o = 32; o; o >>= 1) big = max(big, (uint32_t)__shfl_xor((int)big, o));
    if ((tid & 63) == 0) red[tid >> 6] = big;
    __syncthreads();
    big = max(max(red[0], red[1]), max(red[2], red[3]));
    const float rz = c.code == KV_INT8 ? 1.f / 127.f : 1.f / 448.f;
    const float amax = __uint_as_float(big);
    float* scale = (vals ? c.vscale : c.kscale) + part;
    const float s_old = held ? *scale : 0.f;
    float s = amax >= KV_TINY ? amax * rz : 0.f;
    s = s_old > s ? s_old : s;
    if (big >= 0x7f800000u || s_old != s_old) s = __uint_as_float(0x7fc00000u);
    const float inv = s > 0.f ? 1.f / s : 0.f;
    const float ratio = s > 0.f ? s_old / s : 0.f;
    const bool grown = held && s > s_old;  // (false for NaN: the old codes stay as they are)
    __syncthreads();
    if (tid == 0) *scale = s;

    uint8_t* base = c.pool + kv_tile_offset(c, block, h, 0) + (vals ? kv_half(c.Dp) : 0);
    for (int t = grown ? 0 : held / KV_TILE; t * KV_TILE < end; t++) {
        uint8_t* tile = base + (size_t)t * 2 * kv_half(c.Dp);
        const int r0 = t * KV_TILE;
        for (int u = tid; u < kv_half(c.Dp) / 16; u += 256) {
            uint4 w = {zero_codes(c.code), zero_codes(c.code), zero_codes(c.code), zero_codes(c.code)};
            if (r0 < held) {
                w = ((const uint4*)tile)[u];
                if (grown) {
                    w.x = rescale4(w.x, ratio, c.code), w.y = rescale4(w.y, ratio, c.code);
                    w.z = rescale4(w.z, ratio, c.code), w.w = rescale4(w.w, ratio, c.code);
                }
            }
            ((uint4*)image)[u] = w;
        }
        __syncthreads();
        const int lo = max(held - r0, 0), hi = min(end - r0, KV_TILE);
        for (int u = tid; u < (hi - lo) * Md; u += 256) {
            const int r = lo + u / Md, m = u % Md;
            float e[8];
            load8<T>(x, (tok0 + r0 + r) * x.st + (int64_t)h * x.sh, m, c.D, e);
            const uint32_t w0 = encode4(e[0] * inv, e[1] * inv, e[2] * inv, e[3] * inv, c.code);
            const uint32_t w1 = encode4(e[4] * inv, e[5] * inv, e[6] * inv, e[7] * inv, c.code);
            if (!vals) {
                *(uint2*)(image + kv_key_byte(r, m, S)) = make_uint2(w0, w1);
            } else {
#pragma unroll
                for (int j = 0; j < 8; j++)
                    image[kv_value_byte(r, 8 * m + j)] = (uint8_t)((j < 4 ? w0 : w1) >> (8 * (j & 3)));
            }
        }
        __syncthreads();
        for (int u = tid; u < kv_half(c.Dp) / 16; u += 256) ((uint4*)tile)[u] = ((const uint4*)image)[u];
        __syncthreads();
    }
    if (!vals) {
        for (int r = held + tid; r < end; r += 256) {
            const int64_t at = (tok0 + r) * c.H + h;
            c.positions[part * c.B + r] = positions ? positions[at] : b.aux[i] + slot0 + r - len0;
            c.weights[part * c.B + r] = weights ? weights[at] : 0.f;
        }
    }
}

__device__ __forceinline__ void store1(void* p, size_t i, float v, int type) {
    if (type == KV_F32)
        ((float*)p)[i] = v;
    else if (type == KV_F16)
        ((_Float16*)p)[i] = (_Float16)v;
    else
        ((__hip_bfloat16*)p)[i] = __float2bfloat16(v);
}

// N values of a row from dim d on (those below D), rounded once.
template <int T, int N>
__device__ __forceinline__ void store_row(void* p, size_t row, int d, int D, bool vec, const float* v) {
    if (vec && d + N <= D) {
        if (T == KV_F32) {
            float4* at = (float4*)((float*)p + row + d);
#pragma unroll
            for (int j = 0; j < N / 4; j++) at[j] = make_float4(v[4 * j], v[4 * j + 1], v[4 * j + 2], v[4 * j + 3]);
        } else {
            uint32_t w[N / 2];
#pragma unroll
            for (int j = 0; j < N / 2; j++) {
                uint16_t h[2];
                store1(h, 0, v[2 * j], T), store1(h, 1, v[2 * j + 1], T);
                w[j] = (uint32_t)h[0] | (uint32_t)h[1] << 16;
            }
#pragma unroll
            for (int j = 0; j < N / 8; j++)
                ((uint4*)((uint16_t*)p + row + d))[j] = make_uint4(w[4 * j], w[4 * j + 1], w[4 * j + 2], w[4 * j + 3]);
        }
        return;
    }
#pragma unroll
    for (int j = 0; j < N; j++)
        if (d + j < D) store1(p, row + d + j, v[j], T);
}

// The values of a tile, by one wave: a lane takes its 16 bytes of each piece, which are
// 8 dims each of one slot and two operands (keys), or two dims of 8 slots (values).
// row(slot): the element index of the slot's row in the outputs, or ~0.
template <int T, typename Row>
__device__ __forceinline__ void read_tile(const KvDev& c, const uint8_t* tile, float ks, float vs, void* ko, void* vo,
                                          bool vec, Row row) {
    const int lane = threadIdx.x & 63, g = lane >> 4, x = lane & 15;
    const int S = c.Dp / 32;
    const uint4* at = (const uint4*)tile + lane;
    if (ko) {
        const size_t rows[2] = {row(x), row(16 + x)};
        for (int p = 0; p < S; p++) {
            const uint4 w = at[p * 64];
#pragma unroll
            for (int o = 0; o < 2; o++) {
                const int j = (2 * p + o) / S, s = (2 * p + o) % S;
                const size_t r = j ? rows[1] : rows[0];
                float e[8];
                decode4(o ? w.z : w.x, c.code, e);
                decode4(o ? w.w : w.y, c.code, e + 4);
#pragma unroll
                for (int i = 0; i < 8; i++) e[i] *= ks;
                if (r != ~(size_t)0) store_row<T, 8>(ko, r, 32 * s + 8 * g, c.D, vec, e);
            }
        }
    }
    if (vo) {
        size_t rows[8];
#pragma unroll
        for (int i = 0; i < 8; i++) rows[i] = row((i >> 2) * 16 + 4 * g + (i & 3));
        for (int p = 0; p < S; p++) {
            const uint4 w = at[(S + p) * 64];
#pragma unroll
            for (int o = 0; o < 2; o++) {
                const int d = (2 * p + o) * 16 + x;
                float e[8];
                decode4(o ? w.z : w.x, c.code, e);
                decode4(o ? w.w : w.y, c.code, e + 4);
                if (d < c.D) {
#pragma unroll
                    for (int i = 0; i < 8; i++)
                        if (rows[i] != ~(size_t)0) store1(vo, rows[i] + d, e[i] * vs, T);
                }
            }
        }
    }
}

// One workgroup: 128 slots of one head, a tile to a wave.  Bound by the bytes written:
// no element passes through LDS, a key store is 32 contiguous bytes of a lane, a value
// store 64 bytes of 16 lanes.
template <int T>
__global__ __launch_bounds__(256) void kv_read_kernel(KvDev c, KvBatch b, KvReadOut o) {
    const int tid = threadIdx.x, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int h = blockIdx.x % c.H, unit = blockIdx.x / c.H;
    const int i = kv_find(b, unit);
    const int first = b.aux[i], last = first + b.count[i];
    const int group = (first / KV_READ + unit - b.unit0[i]) * KV_READ;
    const int* table = c.table + (size_t)b.seq[i] * c.W;
    const int64_t tok = (int64_t)b.tok0[i] - first;  // row of slot 0
    const int slot0 = group + wave * KV_TILE;
    if ((o.k || o.v) && slot0 < last && slot0 + KV_TILE > first) {
        const int block = __builtin_amdgcn_readfirstlane(table[slot0 >> c.shift]);
        const size_t part = (size_t)block * c.H + h;
        const uint8_t* tile = c.pool + kv_tile_offset(c, block, h, (slot0 & (c.B - 1)) / KV_TILE);
        read_tile<T>(c, tile, c.kscale[part], c.vscale[part], o.k, o.v, o.vec, [&](int r) -> size_t {
            const int slot = slot0 + r;
            return slot >= first && slot < last ? ((size_t)(tok + slot) * c.H + h) * c.D : ~(size_t)0;
        });
    }
    const int slot = group + tid;
    if (tid < KV_READ && slot >= first && slot < last && (o.positions || o.weights)) {
        const size_t at = (size_t)(tok + slot) * c.H + h;
        const size_t from = ((size_t)table[slot >> c.shift] * c.H + h) * c.B + (slot & (c.B - 1));
        if (o.positions) o.positions[at] = c.positions[from];
        if (o.weights) o.weights[at] = c.weights[from];
    }
}

// ---- eviction -----------------------------------------------------------------

// Weights by size, NaN above all: the order of the unsigned keys.
__device__ __forceinline__ uint32_t weight_key(float w) {
    if (w != w) return 0xffffffffu;
    const uint32_t u = __float_as_uint(w == 0.f ? 0.f : w);  // -0 and 0 are equal
    return (u & 0x80000000u) ? ~u : (u | 0x80000000u);
}

__device__ __forceinline__ size_t slot_at(const KvDev& c, const int* row, int h, int slot) {
    return ((size_t)row[slot >> c.shift] * c.H + h) * c.B + (slot & (c.B - 1));
}

// One workgroup: which slots of one (sequence, head) stay.  The key of the last one
// that does is found by its 8-bit digits, from the top; of the slots with that very
// key the lowest stay.
__global__ __launch_bounds__(1024) void kv_select_kernel(KvDev c, KvBatch b, KvEvict e) {
    __shared__ uint32_t hist[256];
    __shared__ uint32_t sh_prefix, sh_need;
    __shared__ uint32_t wsum[2][16];
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const int h = blockIdx.x % c.H, i = blockIdx.x / c.H;
    const int* row = c.table + (size_t)b.seq[i] * c.W;
    const int len = b.len[i], stay = b.count[i];
    int* kept = e.kept + ((size_t)i * c.H + h) * e.budget;
    int* gone = e.gone ? e.gone + ((size_t)i * c.H + h) * e.slots : nullptr;
    const int recent = stay < len ? min(e.recent, stay) : 0;
    const int old = len - recent, want = stay - recent;
    uint32_t prefix = 0, bits = 0, need = want;
    if (want > 0 && want < old) {
        for (int shift = 24; shift >= 0; shift -= 8) {
            for (int j = tid; j < 256; j += 1024) hist[j] = 0;
            __syncthreads();
            for (int j = tid; j < old; j += 1024) {
                const uint32_t key = weight_key(c.weights[slot_at(c, row, h, j)]);
                if ((key & bits) == prefix) atomicAdd(&hist[(key >> shift) & 255], 1u);
            }
            __syncthreads();
            if (tid == 0) {
                uint32_t left = need;
                int digit = 255;
                for (; digit > 0 && hist[digit] < left; digit--) left -= hist[digit];
                sh_prefix = prefix | (uint32_t)digit << shift;
                sh_need = left;
            }
            __syncthreads();
            prefix = sh_prefix, need = sh_need;
            bits |= 255u << shift;
        }
    }
    // prefix: the key of the last slot that stays, need: how many with that key do
    uint32_t done = 0, equal = 0;
    for (int j0 = 0; j0 < old; j0 += 1024) {
        const int j = j0 + tid;
        const bool in = j < old;
        const uint32_t key = in && want > 0 && want < old ? weight_key(c.weights[slot_at(c, row, h, j)]) : 0;
        const bool eq = in && want > 0 && want < old && key == prefix;
        const uint64_t eb = __ballot(eq);
        if (lane == 0) wsum[0][wave] = (uint32_t)__popcll(eb);
        __syncthreads();
        uint32_t before = equal, all = 0;
        for (int w = 0; w < 16; w++) {
            if (w < wave) before += wsum[0][w];
            all += wsum[0][w];
        }
        const uint32_t rank = before + (uint32_t)__popcll(eb & ((1ull << lane) - 1));
        const bool keep = in && (want >= old || (want > 0 && (key > prefix || (eq && rank < need))));
        const uint64_t kb = __ballot(keep);
        if (lane == 0) wsum[1][wave] = (uint32_t)__popcll(kb);
        __syncthreads();
        uint32_t at = done, kall = 0;
        for (int w = 0; w < 16; w++) {
            if (w < wave) at += wsum[1][w];
            kall += wsum[1][w];
        }
        at += (uint32_t)__popcll(kb & ((1ull << lane) - 1));
        if (keep) kept[at] = j;
        if (in && gone) gone[j] = keep ? -1 : j - (int)at;
        equal += all, done += kall;
        __syncthreads();
    }
    for (int j = tid; j < recent; j += 1024) {
        kept[want + j] = old + j;
        if (gone) gone[old + j] = -1;
    }
}

// One workgroup: one block of one head of the result.
__global__ __launch_bounds__(256) void kv_move_kernel(KvDev c, KvBatch b, KvEvict e) {
    __shared__ int from_block[256], from_slot[256];
    __shared__ float kr[256], vr[256];
    __shared__ float red[2][4];
    const int tid = threadIdx.x, lane = tid & 63;
    const int h = blockIdx.x % c.H, unit = blockIdx.x / c.H;
    const int i = kv_find(b, unit);
    const int blk = unit - b.unit0[i], slot0 = blk << c.shift;
    const int n = min(b.count[i] - slot0, c.B);
    const int* row = c.table + (size_t)b.seq[i] * c.W;
    const int* kept = e.kept + ((size_t)i * c.H + h) * e.budget + slot0;
    const int block = e.dst[(size_t)b.aux[i] * c.W + blk];
    const size_t part = (size_t)block * c.H + h;
    float ks = 0.f, vs = 0.f;
    if (tid < n) {
        const int slot = kept[tid];
        const int fb = row[slot >> c.shift];
        const size_t fp = (size_t)fb * c.H + h;
        from_block[tid] = fb;
        from_slot[tid] = slot & (c.B - 1);
        ks = c.kscale[fp], vs = c.vscale[fp];
        c.positions[part * c.B + tid] = c.positions[fp * c.B + (slot & (c.B - 1))];
        c.weights[part * c.B + tid] = c.weights[fp * c.B + (slot & (c.B - 1))];
    }
    // the largest scale, as bits (scales are not negative; NaN is above all)
    uint32_t kb = __float_as_uint(ks), vb = __float_as_uint(vs);
#pragma unroll
    for (int o = 32; o; o >>= 1) {
        kb = max(kb, (uint32_t)__shfl_xor((int)kb, o));
        vb = max(vb, (uint32_t)__shfl_xor((int)vb, o));
    }
    if (lane == 0) red[0][tid >> 6] = __uint_as_float(kb), red[1][tid >> 6] = __uint_as_float(vb);
    __syncthreads();
    for (int w = 0; w < 4; w++) {
        kb = max(kb, __float_as_uint(red[0][w]));
        vb = max(vb, __float_as_uint(red[1][w]));
    }
    const float kt = __uint_as_float(kb), vt = __uint_as_float(vb);
    if (tid < n) {
        kr[tid] = kt > 0.f ? ks / kt : 0.f;
        vr[tid] = vt > 0.f ? vs / vt : 0.f;
    }
    if (tid == 0) c.kscale[part] = kt, c.vscale[part] = vt;
    __syncthreads();
    const int S = c.Dp / 32, half = kv_half(c.Dp);
    const uint32_t zero = zero_codes(c.code);
    for (int t = 0; t * KV_TILE < n; t++) {
        uint8_t* tile = c.pool + kv_tile_offset(c, block, h, t);
        for (int u = tid; u < half / 8; u += 256) {  // keys: 8 dims of one slot
            const int p = u >> 7, l = (u & 127) >> 1, o = 2 * p + (u & 1);
            const int r = (o / S) * 16 + (l & 15), m = (o % S) * 4 + (l >> 4);
            const int q = t * KV_TILE + r;
            uint2 w = make_uint2(zero, zero);
            if (q < n) {
                const uint8_t* src = c.pool + kv_tile_offset(c, from_block[q], h, from_slot[q] / KV_TILE);
                w = *(const uint2*)(src + kv_key_byte(from_slot[q] & 31, m, S));
                if (kr[q] != 1.f && kt == kt) w.x = rescale4(w.x, kr[q], c.code), w.y = rescale4(w.y, kr[q], c.code);
            }
            ((uint2*)tile)[u] = w;
        }
        for (int u = tid; u < half / 8; u += 256) {  // values: 8 slots of one dim
            const int p = u >> 7, l = (u & 127) >> 1, d = (2 * p + (u & 1)) * 16 + (l & 15);
            uint32_t w[2] = {0, 0};
#pragma unroll
            for (int j = 0; j < 8; j++) {
                const int q = t * KV_TILE + (j >> 2) * 16 + (l >> 4) * 4 + (j & 3);
                uint32_t byte = zero & 255u;
                if (q < n) {
                    const uint8_t* src = c.pool + kv_tile_offset(c, from_block[q], h, from_slot[q] / KV_TILE) + half;
                    byte = src[kv_value_byte(from_slot[q] & 31, d)];
                    if (vr[q] != 1.f && vt == vt) byte = rescale4(byte, vr[q], c.code) & 255u;
                }
                w[j >> 2] |= byte << (8 * (j & 3));
            }
            ((uint2*)(tile + half))[u] = make_uint2(w[0], w[1]);
        }
    }
}

// One workgroup: 128 slots of one head; those that leave are written to their rows.
__global__ __launch_bounds__(256) void kv_dropped_kernel(KvDev c, KvBatch b, KvEvict e, int groups) {
    const int tid = threadIdx.x, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int h = blockIdx.x % c.H, g = blockIdx.x / c.H % groups, i = blockIdx.x / c.H / groups;
    const int len = b.len[i], group = g * KV_READ;
    const int* table = c.table + (size_t)b.seq[i] * c.W;
    const int* gone = e.gone + ((size_t)i * c.H + h) * e.slots;
    const int slot0 = group + wave * KV_TILE;
    if ((e.dk || e.dv) && slot0 < len) {
        const int block = __builtin_amdgcn_readfirstlane(table[slot0 >> c.shift]);
        const size_t part = (size_t)block * c.H + h;
        const uint8_t* tile = c.pool + kv_tile_offset(c, block, h, (slot0 & (c.B - 1)) / KV_TILE);
        read_tile<KV_F32>(c, tile, c.kscale[part], c.vscale[part], e.dk, e.dv, e.vec, [&](int r) -> size_t {
            const int to = slot0 + r < len ? gone[slot0 + r] : -1;
            return to >= 0 ? ((size_t)(b.tok0[i] + to) * c.H + h) * c.D : ~(size_t)0;
        });
    }
    const int slot = group + tid;
    if (e.dpos && tid < KV_READ && slot < len) {
        const int to = gone[slot];
        if (to >= 0)
            e.dpos[(size_t)(b.tok0[i] + to) * c.H + h] =
                c.positions[((size_t)table[slot >> c.shift] * c.H + h) * c.B + (slot & (c.B - 1))];
    }
}

// Rows past what a sequence lost: position -1 and zeros.
__global__ __launch_bounds__(256) void kv_dropped_rest_kernel(KvDev c, KvBatch b, KvEvict e) {
    const int i = blockIdx.y;
    const int n = b.len[i] - b.count[i];
    const size_t width = (size_t)c.H * c.D;
    for (int j = n + blockIdx.x; j < e.drop; j += gridDim.x) {
        const size_t row = (size_t)(b.tok0[i] + j);
        for (size_t u = threadIdx.x; u < width; u += 256) {
            if (e.dk) e.dk[row * width + u] = 0.f;
            if (e.dv) e.dv[row * width + u] = 0.f;
        }
        if (e.dpos)
            for (int u = threadIdx.x; u < c.H; u += 256) e.dpos[row * c.H + u] = -1;
    }
}

}  // namespace

void launch_kv_table(int* table, const KvRuns& r, hipStream_t s) {
    if (r.n > 0) hipLaunchKernelGGL(kv_table_kernel, dim3(r.n), dim3(256), 0, s, table, r);
}

void launch_kv_append(const KvDev& c, const KvBatch& b, const KvTensor& k, const KvTensor& v,
                      const int* positions, const float* weights, hipStream_t s) {
    const dim3 grid((unsigned)b.unit0[b.n] * c.H * 2);
    if (!grid.x) return;
    if (k.type == KV_F32)
        hipLaunchKernelGGL(kv_append_kernel<KV_F32>, grid, dim3(256), 0, s, c, b, k, v, positions, weights);
    else if (k.type == KV_F16)
        hipLaunchKernelGGL(kv_append_kernel<KV_F16>, grid, dim3(256), 0, s, c, b, k, v, positions, weights);
    else
        hipLaunchKernelGGL(kv_append_kernel<KV_BF16>, grid, dim3(256), 0, s, c, b, k, v, positions, weights);
}

void launch_kv_read(const KvDev& c, const KvBatch& b, const KvReadOut& o, hipStream_t s) {
    const dim3 grid((unsigned)b.unit0[b.n] * c.H);
    if (!grid.x) return;
    if (o.type == KV_F32)
        hipLaunchKernelGGL(kv_read_kernel<KV_F32>, grid, dim3(256), 0, s, c, b, o);
    else if (o.type == KV_F16)
        hipLaunchKernelGGL(kv_read_kernel<KV_F16>, grid, dim3(256), 0, s, c, b, o);
    else
        hipLaunchKernelGGL(kv_read_kernel<KV_BF16>, grid, dim3(256), 0, s, c, b, o);
}

void launch_kv_evict(const KvDev& c, const KvBatch& b, const KvEvict& e, hipStream_t s) {
    hipLaunchKernelGGL(kv_select_kernel, dim3(b.n * c.H), dim3(1024), 0, s, c, b, e);
    if (e.drop > 0) {
        int longest = 0, least = INT_MAX;  // slots, and rows that leave
        for (int i = 0; i < b.n; i++) {
            longest = b.len[i] > longest ? b.len[i] : longest;
            least = b.len[i] - b.count[i] < least ? b.len[i] - b.count[i] : least;
        }
        const int groups = (longest + KV_READ - 1) / KV_READ;
        if (groups)
            hipLaunchKernelGGL(kv_dropped_kernel, dim3((unsigned)b.n * c.H * groups), dim3(256), 0, s, c, b, e, groups);
        if (least < e.drop)
            hipLaunchKernelGGL(kv_dropped_rest_kernel, dim3(e.drop - least < 256 ? e.drop - least : 256, b.n), dim3(256),
                               0, s, c, b, e);
    }
    if (b.unit0[b.n])
        hipLaunchKernelGGL(kv_move_kernel, dim3((unsigned)b.unit0[b.n] * c.H), dim3(256), 0, s, c, b, e);
}

}  // namespace vgpu
