// The attention memory: quantising append, reading back, the block table.
//
// append  s = amax * (1 / Z) per (block, head), codes round(x * (1 / s)): the elements are
//         read once and stay in registers until s is known (long float32 rows: read twice).
// read    code * s.
// evict   the weight of the last slot that stays by a radix selection, the kept codes
//         gathered into new blocks under their largest scale.
// Each is bound by the bytes in and out; what the kernels reach stands at each.
// Rounding: codes are the cache's format; every value before them is float32.
#include "vgpu_kv.h"

#include <climits>
#include <hip/hip_bf16.h>
#include <hip/hip_fp16.h>

namespace vgpu {

namespace {

typedef float floatx4 __attribute__((ext_vector_type(4)));
typedef unsigned int u32x4 __attribute__((ext_vector_type(4)));

// Scales are 0 below this largest magnitude, so 1 / s stays finite.
constexpr float KV_TINY = 0x1p-100f;

// Eight elements as they lie in memory.
template <int T>
struct Eight {
    uint32_t w[T == KV_F32 ? 8 : 4];
    __device__ __forceinline__ float at(int e) const {
        if (T == KV_F32) return __uint_as_float(w[e]);
        const uint32_t h = w[e >> 1] >> (16 * (e & 1)) & 0xffffu;
        return T == KV_F16 ? (float)__builtin_bit_cast(_Float16, (uint16_t)h) : __uint_as_float(h << 16);
    }
};

// dims 8 m .. 8 m + 7 of a row (0 from D on)
template <int T>
__device__ __forceinline__ Eight<T> load8(const KvTensor& x, int64_t row, int m, int D) {
    Eight<T> r;
    constexpr int W = T == KV_F32 ? 8 : 4;
    if (x.vec) {
        const uint4* p = (const uint4*)((const uint8_t*)x.p + (row + 8 * m) * (T == KV_F32 ? 4 : 2));
#pragma unroll
        for (int j = 0; j < W / 4; j++) {
            const uint4 a = p[j];
            r.w[4 * j] = a.x, r.w[4 * j + 1] = a.y, r.w[4 * j + 2] = a.z, r.w[4 * j + 3] = a.w;
        }
    } else {
#pragma unroll
        for (int j = 0; j < W; j++) r.w[j] = 0;
#pragma unroll
        for (int e = 0; e < 8; e++) {
            const int d = 8 * m + e;
            if (d >= D) continue;
            if (T == KV_F32)
                r.w[e] = ((const uint32_t*)x.p)[row + d * x.sd];
            else
                r.w[e >> 1] |= (uint32_t)((const uint16_t*)x.p)[row + d * x.sd] << (16 * (e & 1));
        }
    }
    return r;
}

__device__ __forceinline__ uint32_t encode4(float a, float b, float c, float d, int code) {
    const float z = code == KV_INT8 ? 127.f : 448.f;
    // (a NaN becomes some number: its block's scale is NaN)
    a = __builtin_amdgcn_fmed3f(a, -z, z), b = __builtin_amdgcn_fmed3f(b, -z, z);
    c = __builtin_amdgcn_fmed3f(c, -z, z), d = __builtin_amdgcn_fmed3f(d, -z, z);
    if (code == KV_INT8) {
        // 1.5 * 2^23 + 128: the sum's last byte is the integer, ties to even, plus 128
        const float m = 12583040.f;
        const uint32_t lo = __builtin_amdgcn_perm(__float_as_uint(b + m), __float_as_uint(a + m), 0x0c0c0400u);
        const uint32_t hi = __builtin_amdgcn_perm(__float_as_uint(d + m), __float_as_uint(c + m), 0x04000c0cu);
        return lo | hi;
    }
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

// Byte l & 3 of each of the quad's four lanes, in their order.
__device__ __forceinline__ uint32_t quad_transpose(uint32_t w) {
    const uint32_t q = threadIdx.x & 3;
    const uint32_t a0 = (uint32_t)__builtin_amdgcn_mov_dpp((int)w, 0x00, 0xf, 0xf, true);
    const uint32_t a1 = (uint32_t)__builtin_amdgcn_mov_dpp((int)w, 0x55, 0xf, 0xf, true);
    const uint32_t a2 = (uint32_t)__builtin_amdgcn_mov_dpp((int)w, 0xaa, 0xf, 0xf, true);
    const uint32_t a3 = (uint32_t)__builtin_amdgcn_mov_dpp((int)w, 0xff, 0xf, 0xf, true);
    const uint32_t sel = q | (q + 4) << 8;  // byte q of the second operand, then of the first
    const uint32_t lo = __builtin_amdgcn_perm(a1, a0, sel), hi = __builtin_amdgcn_perm(a3, a2, sel);
    return __builtin_amdgcn_perm(hi, lo, 0x05040100u);
}

__global__ __launch_bounds__(256) void kv_table_kernel(int* table, KvRuns r) {
    const int i = blockIdx.x;
    for (int j = threadIdx.x; j < r.count[i]; j += blockDim.x) table[r.at[i] + j] = r.block[i] + j;
}

constexpr int KV_COLUMNS = 2048;  // of a workgroup that goes over table rows
__global__ __launch_bounds__(256) void kv_rows_kernel(const int* from, int* to, int W, KvRows r) {
    const int i = blockIdx.y;
    const int end = min(r.end[i], r.first[i] + ((int)blockIdx.x + 1) * KV_COLUMNS);
    for (int j = r.first[i] + blockIdx.x * KV_COLUMNS + threadIdx.x; j < end; j += 256)
        to[(size_t)r.to[i] * W + j] = from[(size_t)r.from[i] * W + j];
}

__global__ __launch_bounds__(256) void kv_rename_kernel(int* table, int W, KvRows r, const int* map, int above) {
    const int i = blockIdx.y;
    const int end = min(r.end[i], r.first[i] + ((int)blockIdx.x + 1) * KV_COLUMNS);
    for (int j = r.first[i] + blockIdx.x * KV_COLUMNS + threadIdx.x; j < end; j += 256) {
        int* at = table + (size_t)r.to[i] * W + j;
        if (*at >= above) *at = map[*at];
    }
}

// Blocks copied whole: a workgroup takes 16 KiB of a block's codes (a block is contiguous, and
// a multiple of 4 KiB) and its share of the positions and weights; the first of a block also takes
// the scales (10 blocks of 64 heads x 256 slots: all of these by the first workgroup 28 us, so 10).
// Stores pass the caches by, which leaves them to what is read (206 MB by themselves: 52 us,
// cached stores 78, 32 KiB to a workgroup 63).
__global__ __launch_bounds__(256) void kv_moves_kernel(KvDev from, KvDev to, KvMoves m, int pieces, int* map) {
    const int tid = threadIdx.x, unit = blockIdx.x / pieces, piece = blockIdx.x - unit * pieces;
    int lo = 0, hi = m.n;  // the run: unit0[lo] <= unit < unit0[lo + 1]
    while (hi - lo > 1) {
        const int mid = (lo + hi) / 2;
        if (m.unit0[mid] <= unit) lo = mid;
        else hi = mid;
    }
    const int src = m.src[lo] + unit - m.unit0[lo], dst = m.dst[lo] + unit - m.unit0[lo];
    const size_t bytes = (size_t)from.H * from.B * 2 * from.Dp;
    const u32x4* in = (const u32x4*)(from.pool + (size_t)src * bytes);
    u32x4* out = (u32x4*)(to.pool + (size_t)dst * bytes);
    const int at = piece * (KV_COPY * 256) + tid, end = (int)(bytes / 16);
    u32x4 x[KV_COPY];
#pragma unroll
    for (int j = 0; j < KV_COPY; j++)
        if (at + j * 256 < end) x[j] = in[at + j * 256];
#pragma unroll
    for (int j = 0; j < KV_COPY; j++)
        if (at + j * 256 < end) __builtin_nontemporal_store(x[j], out + at + j * 256);
    // (a head has a multiple of 32 slots)
    const int quads = from.H * from.B / 4, q1 = (int)((int64_t)quads * (piece + 1) / pieces);
    const uint4* pos_in = (const uint4*)from.positions + (size_t)src * quads;
    const uint4* wts_in = (const uint4*)from.weights + (size_t)src * quads;
    uint4* pos_out = (uint4*)to.positions + (size_t)dst * quads;
    uint4* wts_out = (uint4*)to.weights + (size_t)dst * quads;
    for (int j = (int)((int64_t)quads * piece / pieces) + tid; j < q1; j += 256) pos_out[j] = pos_in[j], wts_out[j] = wts_in[j];
    if (piece) return;
    if (map && tid == 0) map[src] = dst;
    for (int h = tid; h < from.H; h += 256) {
        to.kscale[(size_t)dst * from.H + h] = from.kscale[(size_t)src * from.H + h];
        to.vscale[(size_t)dst * from.H + h] = from.vscale[(size_t)src * from.H + h];
    }
}

// One workgroup: the keys or the values of one (block, head) that new tokens enter.  Each
// thread loads its pieces of 8 dims once and keeps them (HOLD of them; blocks with more are
// read a second time, from L2) until the scale is known; the codes are put in order in LDS
// and leave in 16-byte pieces.  A few tokens in a begun block that keeps its scale go to
// their bytes directly.  Bound by the bytes in and out, one workgroup's load, reduction and codes
// after another: 16384 tokens of 8 x 128 16-bit elements 33 us, 3.0 TB/s, float32 41 us, 4.1;
// of 8 x 256 in 256-slot blocks, read twice, 97 us, 2.1, and 115 us, 2.9.
// One token to each of 64 begun blocks that others hold too: 11.5 us, 7.8 MB in and 7.9 out.
constexpr int KV_HOLD = 8;
constexpr int KV_FEW = 4;

template <int T>
__global__ __launch_bounds__(256) void kv_append_kernel(KvDev c, KvBatch b, KvTensor k, KvTensor v,
                                                        const int* __restrict__ positions,
                                                        const float* __restrict__ weights) {
    extern __shared__ __align__(16) uint8_t image[];  // the block's codes: B * Dp bytes
    __shared__ uint32_t red[4];
    const int tid = threadIdx.x;
    const bool vals = blockIdx.x & 1;
    const int h = kv_mod(blockIdx.x >> 1, c.by_heads), unit = kv_div(blockIdx.x >> 1, c.by_heads);
    const int i = kv_find(b, unit);
    const int len0 = b.len[i], len1 = len0 + b.count[i];
    const int blk = (len0 >> c.shift) + unit - b.unit0[i];
    const int slot0 = blk << c.shift;
    const int held = max(len0 - slot0, 0), end = min(len1 - slot0, c.B);  // new slots held .. end - 1
    // a sequence that touches one block brings its number, and the table learns a new one here
    int* entry = c.table + (size_t)b.seq[i] * c.W + blk;
    const int block = __builtin_amdgcn_readfirstlane(b.splits[i] >= 0 ? b.splits[i] : *entry);
    // a begun block that others hold too is copied on the way: what it held comes from there
    const int source = blk == len0 >> c.shift && b.per[i] >= 0 ? b.per[i] : block;
    const bool copied = source != block;
    if (b.splits[i] >= 0 && (!held || copied) && h == 0 && !vals && tid == 0) *entry = block;
    const size_t part = (size_t)block * c.H + h, part0 = (size_t)source * c.H + h;
    const KvTensor& x = vals ? v : k;
    const int64_t tok0 = (int64_t)b.tok0[i] + slot0 - len0;  // token of slot 0 of the block
    // piece u: 8 dims m of the new slot r.  Values go by quads of slots, aligned in the block
    // (r may lie outside at its ends), so that a quad of lanes can exchange their codes.
    const int S = c.Dp / 32, Md = (c.D + 7) / 8;
    // u / Md of u < 256 Md, Md <= 32: the product's excess stays below 2^20
    const uint32_t inv_m = ((1u << 20) + Md - 1) / Md;
    const auto split = [&](int u, int& q, int& m) {
        q = (int)((uint32_t)u * inv_m >> 20);
        m = u - q * Md;
    };
    const int start = vals ? held & ~3 : held, units = (vals ? (end - start + 3 & ~3) : end - held) * Md;
    const auto piece = [&](int u, int& r, int& m) {
        int q;
        split(vals ? u >> 2 : u, q, m);
        r = start + (vals ? q * 4 + (u & 3) : q);
        return r >= held && r < end;
    };
    const auto load = [&](int u) {
        int r, m;
        return piece(u, r, m) ? load8<T>(x, (tok0 + r) * x.st + (int64_t)h * x.sh, m, c.D) : Eight<T>{};
    };
    float* scale = (vals ? c.vscale : c.kscale) + part;
    const float s_old = held ? (vals ? c.vscale : c.kscale)[part0] : 0.f;
    uint8_t* base = c.pool + kv_tile_offset(c, block, h, 0) + (vals ? kv_half(c.Dp) : 0);
    const uint8_t* base0 = c.pool + kv_tile_offset(c, source, h, 0) + (vals ? kv_half(c.Dp) : 0);
    const int half = kv_half(c.Dp);

    // largest magnitude, as bits: infinities and NaN are above every number
    uint32_t big = 0;
    Eight<T> e[KV_HOLD];
    const bool hold = units <= KV_HOLD * 256;
    const auto magnitude = [&](const Eight<T>& y) {
#pragma unroll
        for (int j = 0; j < 8; j++) big = max(big, __float_as_uint(y.at(j)) & 0x7fffffffu);
    };
    if (hold) {
#pragma unroll
        for (int z = 0; z < KV_HOLD; z++) {
            if (z * 256 + tid < units) e[z] = load(z * 256 + tid);
        }
#pragma unroll
        for (int z = 0; z < KV_HOLD; z++)
            if (z * 256 + tid < units) magnitude(e[z]);
    } else {
        for (int u = tid; u < units; u += 256) {
            e[0] = load(u);
            magnitude(e[0]);
        }
    }
#pragma unroll
    for (int o = 32; o; o >>= 1) big = max(big, (uint32_t)__shfl_xor((int)big, o));
    if ((tid & 63) == 0) red[tid >> 6] = big;
    __syncthreads();
    big = max(max(red[0], red[1]), max(red[2], red[3]));
    const float rz = c.code == KV_INT8 ? 1.f / 127.f : 1.f / 448.f;
    const float amax = __uint_as_float(big);
    float s = amax >= KV_TINY ? amax * rz : 0.f;
    s = s_old > s ? s_old : s;
    if (big >= 0x7f800000u || s_old != s_old) s = __uint_as_float(0x7fc00000u);
    const float inv = s > 0.f ? 1.f / s : 0.f;
    const float ratio = s > 0.f ? s_old / s : 0.f;
    const bool grown = held && s > s_old;  // (false for NaN: the old codes stay as they are)
    if (tid == 0 && !(s == s_old && held && !copied)) *scale = s;
    if (!vals) {
        if (copied)
            for (int r = tid; r < held; r += 256) {
                c.positions[part * c.B + r] = c.positions[part0 * c.B + r];
                c.weights[part * c.B + r] = c.weights[part0 * c.B + r];
            }
        for (int r = held + tid; r < end; r += 256) {
            const int64_t at = (tok0 + r) * c.H + h;
            c.positions[part * c.B + r] = positions ? positions[at] : b.aux[i] + slot0 + r - len0;
            c.weights[part * c.B + r] = weights ? weights[at] : 0.f;
        }
    }

    const bool direct = held % KV_TILE && !grown && !copied && end - held <= KV_FEW && held / KV_TILE == (end - 1) / KV_TILE;
    const int first = grown || copied ? 0 : held / KV_TILE, last = (end + KV_TILE - 1) / KV_TILE;  // tiles that change
    if (!direct) {
        for (int t = first; t < last; t++)
            for (int o = tid; o < half / 16; o += 256) {
                uint4 w = {zero_codes(c.code), zero_codes(c.code), zero_codes(c.code), zero_codes(c.code)};
                if (t * KV_TILE < held) {
                    w = ((const uint4*)(base0 + (size_t)t * 2 * half))[o];
                    if (grown) {
                        w.x = rescale4(w.x, ratio, c.code), w.y = rescale4(w.y, ratio, c.code);
                        w.z = rescale4(w.z, ratio, c.code), w.w = rescale4(w.w, ratio, c.code);
                    }
                }
                ((uint4*)(image + (t - first) * half))[o] = w;
            }
        __syncthreads();
    }
    const auto encode = [&](int u, const Eight<T>& y) {
        int r, m;
        (void)piece(u, r, m);
        const int t = r / KV_TILE;
        uint32_t w[2] = {encode4(y.at(0) * inv, y.at(1) * inv, y.at(2) * inv, y.at(3) * inv, c.code),
                         encode4(y.at(4) * inv, y.at(5) * inv, y.at(6) * inv, y.at(7) * inv, c.code)};
        uint8_t* to = direct ? base + (size_t)t * 2 * half : image + (t - first) * half;
        if (!vals) {
            *(uint2*)(to + kv_key_byte(r & 31, m, S)) = make_uint2(w[0], w[1]);
            return;
        }
        // four slots of dim 8 m + (lane of the quad), and of that + 4
        const int r0 = r & ~3, d = 8 * m + (u & 3);
#pragma unroll
        for (int j = 0; j < 2; j++) {
            const uint32_t four = quad_transpose(w[j]);
            uint8_t* at = to + kv_value_byte(r0 & 31, d + 4 * j);
            if (r0 >= held && r0 + 3 < end) {
                *(uint32_t*)at = four;
            } else {
#pragma unroll
                for (int z = 0; z < 4; z++)
                    if (r0 + z >= held && r0 + z < end) at[z] = (uint8_t)(four >> (8 * z));
            }
        }
    };
    if (hold) {
#pragma unroll
        for (int z = 0; z < KV_HOLD; z++)
            if (z * 256 + tid < units) encode(z * 256 + tid, e[z]);
    } else {
        for (int u = tid; u < units; u += 256) {
            e[0] = load(u);
            encode(u, e[0]);
        }
    }
    if (direct) return;
    __syncthreads();
    for (int t = first; t < last; t++)
        for (int o = tid; o < half / 16; o += 256)
            ((uint4*)(base + (size_t)t * 2 * half))[o] = ((const uint4*)(image + (t - first) * half))[o];
}

__device__ __forceinline__ void store1(void* p, size_t i, float v, int type) {
    if (type == KV_F32)
        ((float*)p)[i] = v;
    else if (type == KV_F16)
        ((_Float16*)p)[i] = (_Float16)v;
    else
        ((__hip_bfloat16*)p)[i] = __float2bfloat16(v);
}

// Four values of a row from dim d on (those below D), rounded once.
__device__ __forceinline__ void store_row(float* p, size_t row, int d, int D, bool vec, const float* v) {
    if (vec && d + 4 <= D) {
        __builtin_nontemporal_store(floatx4{v[0], v[1], v[2], v[3]}, (floatx4*)(p + row + d));
        return;
    }
#pragma unroll
    for (int j = 0; j < 4; j++)
        if (d + j < D) p[row + d + j] = v[j];
}

// Eight codes of a row from dim d on, in 16 bits.
template <int T>
__device__ __forceinline__ void store_row8(void* p, size_t row, int d, int D, bool vec, uint32_t c0, uint32_t c1, int code, float s) {
    float v[8];
    decode4(c0, code, v);
    decode4(c1, code, v + 4);
    uint16_t e[8];
#pragma unroll
    for (int j = 0; j < 8; j++) {
        // (the float32 product, and its rounding: one instruction for both would round once and
        // lose the sign of a zero)
        float x = v[j] * s;
        asm("" : "+v"(x));
        store1(e, j, x, T);
    }
    if (vec && d + 8 <= D) {
        u32x4 w;
#pragma unroll
        for (int j = 0; j < 4; j++) w[j] = (uint32_t)e[2 * j] | (uint32_t)e[2 * j + 1] << 16;
        u32x4* to = (u32x4*)((uint16_t*)p + row + d);
        // (rows of whole 128-byte lines leave past the caches)
        if (D % 64 == 0) __builtin_nontemporal_store(w, to);
        else *to = w;
        return;
    }
#pragma unroll
    for (int j = 0; j < 8; j++)
        if (d + j < D) ((uint16_t*)p)[row + d + j] = e[j];
}

// The values of a tile, by one wave: a lane takes its 16 bytes of each piece, which are
// 8 dims each of one slot and two operands (keys), or of 8 slots and two dims (values).
// row(slot): the element index of the slot's row in the outputs, or ~0.
template <int T, typename Row>
__device__ __forceinline__ void read_tile(const KvDev& c, const uint8_t* tile, float ks, float vs, void* ko, void* vo,
                                          bool vec, Row row) {
    const int lane = threadIdx.x & 63, g = lane >> 4, x = lane & 15;
    const int S = c.Dp / 32;
    const uint4* at = (const uint4*)tile + lane;
    const bool odd = lane & 1;
    if constexpr (T != KV_F32) {
        // A lane's two pieces of 8 dims, of 32 dims each of its slot, go out in two stores: of
        // the even lanes' slots, then of the odd ones'.  Eight lanes hold a slot's 64 dims: whole
        // 128-byte lines, but where the pieces are odd in number.
        const auto swap = [&](uint32_t first, uint32_t second, uint32_t (&to)[2]) {
            const uint32_t other = (uint32_t)__builtin_amdgcn_mov_dpp((int)(odd ? first : second), 0xb1, 0xf, 0xf, true);
            to[0] = odd ? other : first, to[1] = odd ? second : other;
        };
        if (ko) {
            const int r = x & ~1;
            const size_t rows[2][2] = {{row(r), row(r + 1)}, {row(16 + r), row(17 + r)}};
            for (int p = 0; p < S; p++) {
                const uint4 w = at[p * 64];
                uint32_t a[2], b[2];
                swap(w.x, w.z, a), swap(w.y, w.w, b);
                const int o = 2 * p + odd, j = o >= S, d = 32 * (o - (j ? S : 0)) + 8 * g;
#pragma unroll
                for (int y = 0; y < 2; y++) {
                    const size_t to = j ? rows[1][y] : rows[0][y];
                    if (to != ~(size_t)0) store_row8<T>(ko, to, d, c.D, vec, a[y], b[y], c.code, ks);
                }
            }
        }
        if (vo) {
            const int r = 4 * g + (x & 2);
            const size_t rows[2][2] = {{row(r), row(r + 1)}, {row(16 + r), row(17 + r)}};
            for (int p = 0; p < S; p += 2) {
                // as below, then a quad and the next exchange 4 dims, so that a lane has 8
                const bool far = lane & 4;
                uint32_t e[2][2][2];  // [piece][lower or upper slots][4 dims]
#pragma unroll
                for (int q = 0; q < 2; q++) {
                    const uint4 w = at[(S + min(p + q, S - 1)) * 64];
                    const uint32_t t[4] = {quad_transpose(w.x), quad_transpose(w.y), quad_transpose(w.z), quad_transpose(w.w)};
#pragma unroll
                    for (int u = 0; u < 2; u++) {
                        const int mine = (int)(far ? t[u] : t[2 + u]);
                        // (from 4 lanes on for quads 0 and 2, from 4 lanes before for 1 and 3)
                        const int up = __builtin_amdgcn_update_dpp(0, mine, 0x104, 0xf, 0x5, false);
                        const uint32_t other = (uint32_t)__builtin_amdgcn_update_dpp(up, mine, 0x114, 0xf, 0xa, false);
                        e[q][u][0] = far ? other : t[u], e[q][u][1] = far ? t[2 + u] : other;
                    }
                }
                const int piece = p + odd, d = 32 * piece + 4 * (x >> 2 & 2) + (far ? 16 : 0);
#pragma unroll
                for (int u = 0; u < 2; u++) {
                    uint32_t a[2], b[2];
                    swap(e[0][u][0], e[1][u][0], a), swap(e[0][u][1], e[1][u][1], b);
#pragma unroll
                    for (int y = 0; y < 2; y++)
                        if (rows[u][y] != ~(size_t)0 && piece < S)
                            store_row8<T>(vo, rows[u][y], d, c.D, vec, a[y], b[y], c.code, vs);
                }
            }
        }
        return;
    }
    // A lane's two pieces of 4 dims, of the lower and the upper 16 of 32 dims of its slot, go
    // out in two stores: of the even lanes' slots, then of the odd ones'.  Eight lanes hold a
    // slot's 32 dims, so that a store is of whole 128-byte lines.
    const auto emit = [&](void* out, uint32_t lower, uint32_t upper, float s, const size_t* r, int d) {
        const uint32_t other = (uint32_t)__builtin_amdgcn_mov_dpp((int)(odd ? lower : upper), 0xb1, 0xf, 0xf, true);
        const uint32_t two[2] = {odd ? other : lower, odd ? upper : other};
#pragma unroll
        for (int y = 0; y < 2; y++) {
            float e[4];
            decode4(two[y], c.code, e);
#pragma unroll
            for (int i = 0; i < 4; i++) e[i] *= s;
            if (r[y] != ~(size_t)0) store_row((float*)out, r[y], d + (odd ? 16 : 0), c.D, vec, e);
        }
    };
    if (ko) {
        size_t rows[2][2];
#pragma unroll
        for (int y = 0; y < 2; y++) rows[0][y] = row((x & ~1) + y), rows[1][y] = row(16 + (x & ~1) + y);
        for (int p = 0; p < S; p++) {
            const uint4 w = at[p * 64];
#pragma unroll
            for (int o = 0; o < 2; o++) {
                const int j = (2 * p + o) / S, s = (2 * p + o) % S;
                // dims 8 g .. + 3 and + 4 .. + 7 of lane group g become 4 g .. and 16 + 4 g ..
                const auto half = __builtin_amdgcn_permlane16_swap(o ? w.z : w.x, o ? w.w : w.y, false, false);
                const auto two = __builtin_amdgcn_permlane32_swap(half[0], half[1], false, false);
                emit(ko, two[0], two[1], ks, j ? rows[1] : rows[0], 32 * s + 4 * g);
            }
        }
    }
    if (vo) {
        // a quad of lanes exchanges bytes, so that a lane has 4 dims of slots 4 g + (x & 3)
        // and 16 above
        const int r = 4 * g + (x & 2);
        const size_t rows[2][2] = {{row(r), row(r + 1)}, {row(16 + r), row(17 + r)}};
        for (int p = 0; p < S; p++) {
            const uint4 w = at[(S + p) * 64];
            const int d = 32 * p + (x & ~3);
            emit(vo, quad_transpose(w.x), quad_transpose(w.z), vs, rows[0], d);
            emit(vo, quad_transpose(w.y), quad_transpose(w.w), vs, rows[1], d);
        }
    }
}

// One workgroup: 128 slots of one head, a tile's keys or values to a wave (both to one: 777
// slots of 5 x 80 11.1 us for 7.4: a wave alone on its SIMD waits for each result).  Bound by
// the bytes written: no element passes through LDS, and stores of whole lines leave the caches
// to the pool (nontemporal: 31 sequences moved in 41 us for 64 before them; 64-byte halves of
// lines stored so took 68 us of reading for 58).  110000 slots of 8 x 128 in bfloat16: 690 MB in
// 124 us, 5.5 TB/s; by 8 bytes to a lane, which left as halves of lines (810 MB), 173.
template <int T>
__global__ __launch_bounds__(512) void kv_read_kernel(KvDev c, KvBatch b, KvReadOut o) {
    const int tid = threadIdx.x, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int h = kv_mod(blockIdx.x, c.by_heads), unit = kv_div(blockIdx.x, c.by_heads);
    const int i = kv_find(b, unit);
    const int first = b.aux[i], last = first + b.count[i];
    const int group = (first / KV_READ + unit - b.unit0[i]) * KV_READ;
    const int* table = c.table + (size_t)b.seq[i] * c.W;
    const int64_t tok = (int64_t)b.tok0[i] - first;  // row of slot 0
    const int slot0 = group + wave * KV_TILE;
    const bool vals = threadIdx.y;
    if ((vals ? o.v : o.k) && slot0 < last && slot0 + KV_TILE > first) {
        const int block = __builtin_amdgcn_readfirstlane(table[slot0 >> c.shift]);
        const size_t part = (size_t)block * c.H + h;
        const uint8_t* tile = c.pool + kv_tile_offset(c, block, h, (slot0 & (c.B - 1)) / KV_TILE);
        read_tile<T>(c, tile, c.kscale[part], c.vscale[part], vals ? nullptr : o.k, vals ? o.v : nullptr, o.vec, [&](int r) -> size_t {
            const int slot = slot0 + r;
            return slot >= first && slot < last ? ((size_t)(tok + slot) * c.H + h) * c.D : ~(size_t)0;
        });
    }
    const int slot = group + tid;
    if (!vals && tid < KV_READ && slot >= first && slot < last && (o.positions || o.weights)) {
        const size_t at = (size_t)(tok + slot) * c.H + h;
        const size_t from = ((size_t)table[slot >> c.shift] * c.H + h) * c.B + (slot & (c.B - 1));
        if (o.positions) o.positions[at] = c.positions[from];
        if (o.weights) o.weights[at] = c.weights[from];
    }
}

// Positions and weights alone: 128 slots of every head to a workgroup, so that the outputs
// [token, head] leave in one piece.
__global__ __launch_bounds__(256) void kv_read_side_kernel(KvDev c, KvBatch b, KvReadOut o) {
    const int unit = blockIdx.x, i = kv_find(b, unit);
    const int first = b.aux[i], last = first + b.count[i];
    const int group = (first / KV_READ + unit - b.unit0[i]) * KV_READ;
    const int* table = c.table + (size_t)b.seq[i] * c.W;
    const size_t tok = (size_t)b.tok0[i];
    for (int u = threadIdx.x; u < KV_READ * c.H; u += 256) {
        const int r = kv_div(u, c.by_heads), h = u - r * c.H, slot = group + r;
        if (slot < first || slot >= last) continue;
        const size_t at = (tok + (slot - first)) * c.H + h;
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

// The weight of the last slot that stays is found by its key's digits of 11, 11 and 10
// bits, from the top: a histogram of the slots that share the digits so far, and the digit
// in which the count from above reaches what is needed.  Of the slots with that very key
// the lowest stay.
constexpr int KV_BINS = 2048;
__device__ __forceinline__ int digit_shift(int pass) { return pass == 0 ? 21 : pass == 1 ? 10 : 0; }
__device__ __forceinline__ uint32_t digit_bits(int pass) { return pass == 0 ? 0xffe00000u : pass == 1 ? 0xfffffc00u : ~0u; }
__device__ __forceinline__ uint32_t digit_of(uint32_t key, int pass) { return key >> digit_shift(pass) & (pass < 2 ? 2047u : 1023u); }

struct KvCut {
    uint32_t key, need;  // the digits so far; how many of the slots that share them stay
};
// By 1024 threads: adds the digit of a histogram (LDS or global).  scan: 18 words of LDS.
__device__ void find_digit(const uint32_t* hist, int pass, uint32_t* scan, KvCut& cut) {
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const int hi = KV_BINS - 1 - 2 * tid;  // this thread's two bins, from the top
    const uint32_t c0 = hist[hi], c1 = hist[hi - 1];
    uint32_t sum = c0 + c1;
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
        const uint32_t up = (uint32_t)__shfl_up((int)sum, o);
        if (lane >= o) sum += up;
    }
    if (lane == 63) scan[wave] = sum;
    __syncthreads();
    for (int w = 0; w < wave; w++) sum += scan[w];
    const uint32_t before = sum - c0 - c1;
    if (before < cut.need && sum >= cut.need) {  // one thread
        const bool first = before + c0 >= cut.need;
        scan[16] = (uint32_t)(first ? hi : hi - 1);
        scan[17] = cut.need - before - (first ? 0 : c0);
    }
    __syncthreads();
    cut.key |= scan[16] << digit_shift(pass);
    cut.need = scan[17];
    __syncthreads();
}

// One (sequence, head): the slots before `old` compete for `want` places.
struct KvSelect {
    const int* row;
    int h, old, want, recent;
    int *kept, *gone;
    bool compete;
};
__device__ __forceinline__ KvSelect select_job(const KvDev& c, const KvBatch& b, const KvEvict& e, int i, int h) {
    KvSelect j;
    j.row = c.table + (size_t)b.seq[i] * c.W;
    j.h = h;
    j.kept = e.kept + ((size_t)i * c.H + h) * e.budget;
    j.gone = e.gone ? e.gone + ((size_t)i * c.H + h) * e.slots : nullptr;
    j.recent = b.count[i] < b.len[i] ? min(e.recent, b.count[i]) : 0;
    j.old = b.len[i] - j.recent, j.want = b.count[i] - j.recent;
    j.compete = j.want > 0 && j.want < j.old;
    return j;
}

// Whether each of 1024 threads' slots stays, and its place: done and equal count what the
// slots before took and how many had the cut's key.
__device__ __forceinline__ void place_slots(const KvSelect& s, const KvCut& cut, uint32_t key, int j, bool in,
                                            uint32_t* scan, uint32_t& done, uint32_t& equal) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const bool eq = in && s.compete && key == cut.key;
    const bool above = in && (s.want >= s.old || (s.compete && key > cut.key));
    const uint64_t eb = __ballot(eq), ab = __ballot(above);
    if (lane == 0) scan[wave] = (uint32_t)__popcll(eb) | (uint32_t)__popcll(ab) << 16;
    __syncthreads();
    uint32_t e0 = equal, a0 = 0, all_e = 0, all_a = 0;
    for (int w = 0; w < 16; w++) {
        const uint32_t x = scan[w];
        if (w < wave) e0 += x & 0xffffu, a0 += x >> 16;
        all_e += x & 0xffffu, all_a += x >> 16;
    }
    const uint64_t below = (1ull << lane) - 1;
    e0 += (uint32_t)__popcll(eb & below), a0 += (uint32_t)__popcll(ab & below);
    // kept so far: those above the cut, and of the equal ones at most cut.need
    const uint32_t at = done - min(equal, cut.need) + a0 + min(e0, cut.need);
    const bool keep = above || (eq && e0 < cut.need);
    if (keep) s.kept[at] = j;
    if (in && s.gone) s.gone[j] = keep ? -1 : j - (int)at;
    done += all_a + min(equal + all_e, cut.need) - min(equal, cut.need);
    equal += all_e;
    __syncthreads();
}

// Up to 16384 slots: one workgroup, the keys in registers.
constexpr int KV_SELECT = 16;
__global__ __launch_bounds__(1024) void kv_select_kernel(KvDev c, KvBatch b, KvEvict e) {
    __shared__ uint32_t hist[KV_BINS];
    __shared__ uint32_t scan[18];
    const int tid = threadIdx.x;
    const KvSelect s = select_job(c, b, e, kv_div(blockIdx.x, c.by_heads), kv_mod(blockIdx.x, c.by_heads));
    uint32_t key[KV_SELECT];
#pragma unroll
    for (int x = 0; x < KV_SELECT; x++) {
        const int j = x * 1024 + tid;
        key[x] = s.compete && j < s.old ? weight_key(c.weights[slot_at(c, s.row, s.h, j)]) : 0;
    }
    KvCut cut = {0, (uint32_t)max(s.want, 0)};
    if (s.compete) {
        for (int pass = 0; pass < 3; pass++) {
            hist[tid] = hist[tid + 1024] = 0;
            __syncthreads();
            const uint32_t bits = pass ? digit_bits(pass - 1) : 0;
#pragma unroll
            for (int x = 0; x < KV_SELECT; x++)
                if (x * 1024 + tid < s.old && (key[x] & bits) == cut.key) atomicAdd(&hist[digit_of(key[x], pass)], 1u);
            __syncthreads();
            find_digit(hist, pass, scan, cut);
        }
    }
    uint32_t done = 0, equal = 0;
#pragma unroll
    for (int x = 0; x < KV_SELECT; x++)
        if (x * 1024 < s.old) place_slots(s, cut, key[x], x * 1024 + tid, x * 1024 + tid < s.old, scan, done, equal);
    for (int j = tid; j < s.recent; j += 1024) {
        s.kept[s.want + j] = s.old + j;
        if (s.gone) s.gone[s.old + j] = -1;
    }
}

// Longer sequences: 4096 slots to a workgroup and a launch for each step, e.hist (three
// histograms of each sequence and head, zero before) and e.counts between them.
constexpr int KV_LONG = 4096;
__device__ __forceinline__ KvCut long_cut(const KvDev& c, const KvEvict& e, const KvSelect& s, int i, int passes, uint32_t* scan) {
    KvCut cut = {0, (uint32_t)max(s.want, 0)};
    if (s.compete)
        for (int p = 0; p < passes; p++) find_digit(e.hist + (((size_t)i * c.H + s.h) * 3 + p) * KV_BINS, p, scan, cut);
    return cut;
}

__global__ __launch_bounds__(1024) void kv_long_hist_kernel(KvDev c, KvBatch b, KvEvict e, int groups, int pass) {
    __shared__ uint32_t hist[KV_BINS];
    __shared__ uint32_t scan[18];
    const int tid = threadIdx.x, h = kv_mod(blockIdx.x, c.by_heads), g = kv_div(blockIdx.x, c.by_heads) % groups, i = kv_div(blockIdx.x, c.by_heads) / groups;
    const KvSelect s = select_job(c, b, e, i, h);
    if (!s.compete || g * KV_LONG >= s.old) return;
    uint32_t key[4];
#pragma unroll
    for (int x = 0; x < 4; x++) {
        const int j = g * KV_LONG + x * 1024 + tid;
        key[x] = j < s.old ? weight_key(c.weights[slot_at(c, s.row, h, j)]) : 0;
    }
    const KvCut cut = long_cut(c, e, s, i, pass, scan);
    hist[tid] = hist[tid + 1024] = 0;
    __syncthreads();
    const uint32_t bits = pass ? digit_bits(pass - 1) : 0;
#pragma unroll
    for (int x = 0; x < 4; x++)
        if (g * KV_LONG + x * 1024 + tid < s.old && (key[x] & bits) == cut.key)
            atomicAdd(&hist[digit_of(key[x], pass)], 1u);
    __syncthreads();
    uint32_t* to = e.hist + (((size_t)i * c.H + h) * 3 + pass) * KV_BINS;
    for (int x = tid; x < KV_BINS; x += 1024)
        if (hist[x]) atomicAdd(&to[x], hist[x]);  // counts: the order does not matter
}

// place 0: how many of each group are above the cut and how many on it; 1: their places.
__global__ __launch_bounds__(1024) void kv_long_place_kernel(KvDev c, KvBatch b, KvEvict e, int groups, int place) {
    __shared__ uint32_t scan[18];
    __shared__ uint32_t sums[2];
    const int tid = threadIdx.x, h = kv_mod(blockIdx.x, c.by_heads), g = kv_div(blockIdx.x, c.by_heads) % groups, i = kv_div(blockIdx.x, c.by_heads) / groups;
    const KvSelect s = select_job(c, b, e, i, h);
    if (place && g == 0)
        for (int j = tid; j < s.recent; j += 1024) {
            s.kept[s.want + j] = s.old + j;
            if (s.gone) s.gone[s.old + j] = -1;
        }
    if (g * KV_LONG >= s.old) return;
    uint32_t key[4];
#pragma unroll
    for (int x = 0; x < 4; x++) {
        const int j = g * KV_LONG + x * 1024 + tid;
        key[x] = s.compete && j < s.old ? weight_key(c.weights[slot_at(c, s.row, h, j)]) : 0;
    }
    const KvCut cut = long_cut(c, e, s, i, 3, scan);
    uint2* counts = e.counts + ((size_t)i * c.H + h) * groups;
    if (tid < 2) sums[tid] = 0;
    __syncthreads();
    if (!place) {
        uint32_t above = 0, on = 0;
#pragma unroll
        for (int x = 0; x < 4; x++) {
            const bool in = g * KV_LONG + x * 1024 + tid < s.old;
            above += (uint32_t)__popcll(__ballot(in && (s.want >= s.old || (s.compete && key[x] > cut.key))));
            on += (uint32_t)__popcll(__ballot(in && s.compete && key[x] == cut.key));
        }
        if ((tid & 63) == 0) atomicAdd(&sums[0], above), atomicAdd(&sums[1], on);
        __syncthreads();
        if (tid == 0) counts[g] = make_uint2(sums[0], sums[1]);
        return;
    }
    uint32_t above = 0, on = 0;
    for (int x = tid; x < g; x += 1024) above += counts[x].x, on += counts[x].y;
    if (above) atomicAdd(&sums[0], above);
    if (on) atomicAdd(&sums[1], on);
    __syncthreads();
    uint32_t equal = sums[1], done = sums[0] + min(equal, cut.need);
#pragma unroll
    for (int x = 0; x < 4; x++) {
        const int j = g * KV_LONG + x * 1024 + tid;
        place_slots(s, cut, key[x], j, j < s.old, scan, done, equal);
    }
}

__global__ __launch_bounds__(256) void kv_zero_kernel(uint4* p, int n) {
    for (int i = blockIdx.x * 256 + threadIdx.x; i < n; i += gridDim.x * 256) p[i] = make_uint4(0, 0, 0, 0);
}

// One workgroup: the keys or the values of one block of one head of the result, gathered
// from L2, 8 bytes of a key or one byte of a value at a time.  (Source tiles brought to LDS
// whole: 72 us for 61, and 113 for 71 where one slot in six stays.)  31 sequences cut to 1024
// slots, 8 x 128: 119 MB come in, for lines hold slots that leave as well, and 56 go out in
// 41 us.
__global__ __launch_bounds__(256) void kv_move_kernel(KvDev c, KvBatch b, KvEvict e) {
    __shared__ const uint8_t* from[256];  // a slot's tile half
    __shared__ int slots[256];            // and its place there
    __shared__ float ratios[256];
    __shared__ uint32_t red[4];
    const int tid = threadIdx.x, lane = tid & 63;
    const bool vals = blockIdx.x & 1;
    const int h = kv_mod(blockIdx.x >> 1, c.by_heads), unit = kv_div(blockIdx.x >> 1, c.by_heads);
    const int i = kv_find(b, unit);
    const int blk = unit - b.unit0[i], slot0 = blk << c.shift;
    const int n = min(b.count[i] - slot0, c.B);
    const int* row = c.table + (size_t)b.seq[i] * c.W;
    const int* kept = e.kept + ((size_t)i * c.H + h) * e.budget + slot0;
    const int block = e.dst[(size_t)b.aux[i] * c.W + blk];
    const size_t part = (size_t)block * c.H + h;
    const int S = c.Dp / 32, half = kv_half(c.Dp);
    float s_old = 0.f;
    if (tid < n) {
        const int slot = kept[tid], in = slot & (c.B - 1), fb = row[slot >> c.shift];
        const size_t fp = (size_t)fb * c.H + h;
        from[tid] = c.pool + kv_tile_offset(c, fb, h, in / KV_TILE) + (vals ? half : 0);
        slots[tid] = in & 31;
        s_old = vals ? c.vscale[fp] : c.kscale[fp];
        if (vals)
            c.weights[part * c.B + tid] = c.weights[fp * c.B + in];
        else
            c.positions[part * c.B + tid] = c.positions[fp * c.B + in];
    }
    // the largest scale, as bits (scales are not negative; NaN is above all)
    uint32_t big = __float_as_uint(s_old);
#pragma unroll
    for (int o = 32; o; o >>= 1) big = max(big, (uint32_t)__shfl_xor((int)big, o));
    if (lane == 0) red[tid >> 6] = big;
    __syncthreads();
    big = max(max(red[0], red[1]), max(red[2], red[3]));
    const float s = __uint_as_float(big);
    if (tid < n) ratios[tid] = s != s ? 1.f : s > 0.f ? s_old / s : 0.f;  // NaN: the codes stay
    if (tid == 0) (vals ? c.vscale : c.kscale)[part] = s;
    __syncthreads();
    const uint32_t zero = zero_codes(c.code);
    uint8_t* base = c.pool + kv_tile_offset(c, block, h, 0) + (vals ? half : 0);
    const int tiles = (n + KV_TILE - 1) / KV_TILE;
    for (int x = tid; x < half / 8; x += 256)
    for (int t = 0; t < tiles; t++) {
        const int p = x >> 7, l = (x & 127) >> 1, o = 2 * p + (x & 1);
        uint32_t w[2] = {zero, zero};
        if (!vals) {  // 8 dims of one slot
            const int upper = o >= S, q = t * KV_TILE + upper * 16 + (l & 15), m = (o - upper * S) * 4 + (l >> 4);
            if (q < n) {
                const uint2 v = *(const uint2*)(from[q] + kv_key_byte(slots[q], m, S));
                w[0] = v.x, w[1] = v.y;
                if (ratios[q] != 1.f) w[0] = rescale4(w[0], ratios[q], c.code), w[1] = rescale4(w[1], ratios[q], c.code);
            }
        } else {  // 8 slots of one dim
            const int d = o * 16 + (l & 15), q0 = t * KV_TILE + (l >> 4) * 4;
            uint32_t bytes[8];
            float r[8];
#pragma unroll
            for (int j = 0; j < 8; j++) {
                const int q = min(q0 + (j >> 2) * 16 + (j & 3), n - 1);  // past the end: any slot, unused
                bytes[j] = from[q][kv_value_byte(slots[q], d)];
                r[j] = ratios[q];
            }
#pragma unroll
            for (int y = 0; y < 2; y++) {
                float v[4];
                decode4(bytes[4 * y] | bytes[4 * y + 1] << 8 | bytes[4 * y + 2] << 16 | bytes[4 * y + 3] << 24, c.code, v);
                // (a ratio of 1 keeps the code)
                w[y] = encode4(v[0] * r[4 * y], v[1] * r[4 * y + 1], v[2] * r[4 * y + 2], v[3] * r[4 * y + 3], c.code);
            }
        }
        *(uint2*)(base + (size_t)t * 2 * half + x * 8) = make_uint2(w[0], w[1]);
    }
}

// One workgroup: 128 slots of one head; those that leave are written to their rows.
__global__ __launch_bounds__(256) void kv_dropped_kernel(KvDev c, KvBatch b, KvEvict e, int groups) {
    const int tid = threadIdx.x, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int h = kv_mod(blockIdx.x, c.by_heads), g = kv_div(blockIdx.x, c.by_heads) % groups, i = kv_div(blockIdx.x, c.by_heads) / groups;
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

static dim3 rows_grid(const KvRows& r) {
    int most = 0;
    for (int i = 0; i < r.n; i++) most = r.end[i] - r.first[i] > most ? r.end[i] - r.first[i] : most;
    return dim3((unsigned)((most + KV_COLUMNS - 1) / KV_COLUMNS), (unsigned)r.n);
}

void launch_kv_rows(const KvDev& c, const int* from, int* to, const KvRows& r, hipStream_t s) {
    const dim3 grid = rows_grid(r);
    if (grid.x && grid.y) hipLaunchKernelGGL(kv_rows_kernel, grid, dim3(256), 0, s, from, to, c.W, r);
}

void launch_kv_rename(const KvDev& c, const KvRows& r, const int* map, int above, hipStream_t s) {
    const dim3 grid = rows_grid(r);
    if (grid.x && grid.y) hipLaunchKernelGGL(kv_rename_kernel, grid, dim3(256), 0, s, c.table, c.W, r, map, above);
}

void launch_kv_moves(const KvDev& from, const KvDev& to, const KvMoves& m, int* map, hipStream_t s) {
    if (!m.n) return;
    const int pieces = kv_move_pieces(from);
    hipLaunchKernelGGL(kv_moves_kernel, dim3((unsigned)(m.unit0[m.n] * pieces)), dim3(256), 0, s, from, to, m, pieces, map);
}

void launch_kv_append(const KvDev& c, const KvBatch& b, const KvTensor& k, const KvTensor& v,
                      const int* positions, const float* weights, hipStream_t s) {
    const dim3 grid((unsigned)b.unit0[b.n] * c.H * 2);
    const size_t lds = (size_t)c.B * c.Dp;  // at most 64 KiB
    if (!grid.x) return;
    if (k.type == KV_F32)
        hipLaunchKernelGGL(kv_append_kernel<KV_F32>, grid, dim3(256), lds, s, c, b, k, v, positions, weights);
    else if (k.type == KV_F16)
        hipLaunchKernelGGL(kv_append_kernel<KV_F16>, grid, dim3(256), lds, s, c, b, k, v, positions, weights);
    else
        hipLaunchKernelGGL(kv_append_kernel<KV_BF16>, grid, dim3(256), lds, s, c, b, k, v, positions, weights);
}

void launch_kv_read(const KvDev& c, const KvBatch& b, const KvReadOut& o, hipStream_t s) {
    const dim3 grid((unsigned)b.unit0[b.n] * c.H);
    if (!grid.x) return;
    if (!o.k && !o.v)
        hipLaunchKernelGGL(kv_read_side_kernel, dim3((unsigned)b.unit0[b.n]), dim3(256), 0, s, c, b, o);
    else if (o.type == KV_F32)
        hipLaunchKernelGGL(kv_read_kernel<KV_F32>, grid, dim3(256, 2), 0, s, c, b, o);
    else if (o.type == KV_F16)
        hipLaunchKernelGGL(kv_read_kernel<KV_F16>, grid, dim3(256, 2), 0, s, c, b, o);
    else
        hipLaunchKernelGGL(kv_read_kernel<KV_BF16>, grid, dim3(256, 2), 0, s, c, b, o);
}

void launch_kv_evict(const KvDev& c, const KvBatch& b, const KvEvict& e, hipStream_t s) {
    int longest = 0, least = INT_MAX;  // slots, and rows that leave
    for (int i = 0; i < b.n; i++) {
        longest = b.len[i] > longest ? b.len[i] : longest;
        least = b.len[i] - b.count[i] < least ? b.len[i] - b.count[i] : least;
    }
    if (longest <= KV_SELECT * 1024) {
        hipLaunchKernelGGL(kv_select_kernel, dim3(b.n * c.H), dim3(1024), 0, s, c, b, e);
    } else {
        const int groups = (longest + KV_LONG - 1) / KV_LONG;
        const dim3 grid((unsigned)b.n * c.H * groups);
        const int words = b.n * c.H * 3 * KV_BINS / 4;
        hipLaunchKernelGGL(kv_zero_kernel, dim3(words / 256 < 1024 ? (words + 255) / 256 : 1024), dim3(256), 0, s, (uint4*)e.hist, words);
        for (int pass = 0; pass < 3; pass++)
            hipLaunchKernelGGL(kv_long_hist_kernel, grid, dim3(1024), 0, s, c, b, e, groups, pass);
        for (int place = 0; place < 2; place++)
            hipLaunchKernelGGL(kv_long_place_kernel, grid, dim3(1024), 0, s, c, b, e, groups, place);
    }
    if (e.drop > 0) {
        const int groups = (longest + KV_READ - 1) / KV_READ;
        if (groups)
            hipLaunchKernelGGL(kv_dropped_kernel, dim3((unsigned)b.n * c.H * groups), dim3(256), 0, s, c, b, e, groups);
        if (least < e.drop)
            hipLaunchKernelGGL(kv_dropped_rest_kernel, dim3(e.drop - least < 256 ? e.drop - least : 256, b.n), dim3(256),
                               0, s, c, b, e);
    }
    if (b.unit0[b.n])
        hipLaunchKernelGGL(kv_move_kernel, dim3((unsigned)b.unit0[b.n] * c.H * 2), dim3(256), 0, s, c, b, e);
}

KvSelectSpace kv_select_space(const KvDev& c, int n, int longest) {
    KvSelectSpace r;
    if (longest > KV_SELECT * 1024) {
        r.hist = (size_t)n * c.H * 3 * KV_BINS;
        r.counts = (size_t)n * c.H * ((longest + KV_LONG - 1) / KV_LONG);
    }
    return r;
}

}  // namespace vgpu
