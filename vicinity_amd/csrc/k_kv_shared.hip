// Softmax attention of sequences that hold the same first blocks: the rows of all of them
// over the shared slots, read once, each over its own, and the join of the parts.
#include "kv_attend.h"

namespace vgpu {

namespace {

// Up to so many rows have a workgroup each in the join.
constexpr int64_t KV_WIDE_JOIN = 16384;

// A row's parts, of the shared slots and of its own, by Dp / 4 threads each: the sums o and l
// go by the power of 2 that a part's m stands below the largest.  WIDE: a workgroup per row,
// its thread groups take parts in turn; else a thread group per row.
template <bool WIDE>
__global__ __launch_bounds__(256) void kv_shared_join_kernel(KvDev c, KvAttend a, KvMembers mem, KvShares j) {
    __shared__ floatx4 sh_o[256];
    __shared__ float sh_l[64];
    const int tid = threadIdx.x;
    const int width = c.Dp / 4, groups = 256 / width, grp = tid / width, d4 = tid % width;
    const int h = kv_mod(blockIdx.x, c.by_heads), unit = kv_div(blockIdx.x, c.by_heads);
    const int row = WIDE ? unit : unit * groups + grp;
    if (!WIDE && (grp >= groups || row >= mem.row0[mem.n])) return;
    int m = 0, end = mem.n;
    while (end - m > 1) {
        const int mid = (m + end) / 2;
        if (mem.row0[mid] <= row) m = mid;
        else end = mid;
    }
    const int mine = row - mem.row0[m], s0 = j.splits[0][m], splits = s0 + j.splits[1][m];
    size_t first[2], step[2];
#pragma unroll
    for (int y = 0; y < 2; y++) {
        const int r = mine + (y ? 0 : j.row0[m]), tile = r / j.rows[y];
        first[y] = j.base[y] + ((size_t)(j.unit[y][m] + tile) * c.H + h) * j.rows[y] + (r - tile * j.rows[y]);
        step[y] = (size_t)j.tiles[y][m] * c.H * j.rows[y];
    }
    const auto part = [&](int s) { return s < s0 ? first[0] + s * step[0] : first[1] + (s - s0) * step[1]; };
    float mx = KV_NEG, top = KV_FIRST;
    if (WIDE) {
        for (int s = tid & 63; s < splits; s += 64) {
            const size_t at = part(s);
            mx = fmaxf(mx, a.part_ml[at].x), top = fmaxf(top, a.part_s[at]);
        }
#pragma unroll
        for (int x = 32; x; x >>= 1) mx = fmaxf(mx, __shfl_xor(mx, x)), top = fmaxf(top, __shfl_xor(top, x));
    } else {
        for (int s = 0; s < splits; s++) {
            const size_t at = part(s);
            mx = fmaxf(mx, a.part_ml[at].x), top = fmaxf(top, a.part_s[at]);
        }
    }
    floatx4 o = {0.f, 0.f, 0.f, 0.f};
    float l = 0.f;
    if (grp < groups) {
#pragma unroll 4
        for (int s = WIDE ? grp : 0; s < splits; s += WIDE ? groups : 1) {
            const size_t at = part(s);
            const float2 ml = a.part_ml[at];
            if (ml.x == KV_NEG && ml.y == 0.f) continue;  // has seen nothing (and left no o)
            const float f = kv_join_factor(ml.x, ml.y, mx);
            l += f * ml.y;
            o += *(const floatx4*)(a.part_o + at * c.Dp + d4 * 4) * ldexpf(f, (int)(a.part_s[at] - top));
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
    const int tok = kv_div(mine, a.by_group);
    const size_t out = (size_t)(mem.tok0[m] + tok) * c.H * a.G + (size_t)h * a.G + (mine - tok * a.G);
    if (d4 == 0 && a.lse) a.lse[out] = (l == 0.f ? KV_NEG : mx - KV_TOP + log2f(l)) * 0.69314718055994531f;
    o = o * (l == 0.f ? 0.f : 1.f / l) * ldexpf(1.f, (int)top);
    if (a.q.type == KV_F32)
        kv_store4<2>(a, out * c.D, 4 * d4, c.D, o);
    else
        kv_store4<1>(a, out * c.D, 4 * d4, c.D, o);
}

template <int S, int CODE, int PARTS>
void shared_s(const KvDev& c, const KvBatch& b, const KvAttend& a, const KvMembers& mem, hipStream_t s) {
    const dim3 grid((unsigned)b.unit0[b.n] * c.H);
    if (a.by_rows) {
        hipLaunchKernelGGL((kv_chunk_kernel<S, CODE, PARTS, kv_chunk_nc(S * 32, PARTS), true>), grid, dim3(256), 0, s, c, b, a, mem);
        return;
    }
    const size_t lds = (size_t)4 * 16 * (32 * S + 4 + 3) * 4;
    int most = 0;
    for (int i = 0; i < b.n; i++) most = b.count[i] > most ? b.count[i] : most;
    const auto kernel = most <= 16 ? kv_step_kernel<S, CODE, PARTS, true, true> : kv_step_kernel<S, CODE, PARTS, false, true>;
    if (lds > 65536) ensure_dyn_lds((const void*)kernel, lds);
    hipLaunchKernelGGL(kernel, grid, dim3(256), lds, s, c, b, a, mem);
}

template <int CODE, int PARTS>
void by_dim(const KvDev& c, const KvBatch& b, const KvAttend& a, const KvMembers& mem, hipStream_t s) {
    switch (c.Dp / 32) {
        case 2: return shared_s<2, CODE, PARTS>(c, b, a, mem, s);
        case 3: return shared_s<3, CODE, PARTS>(c, b, a, mem, s);
        case 4: return shared_s<4, CODE, PARTS>(c, b, a, mem, s);
        case 6: return shared_s<6, CODE, PARTS>(c, b, a, mem, s);
        case 8: return shared_s<8, CODE, PARTS>(c, b, a, mem, s);
    }
}

}  // namespace

void launch_kv_shared(const KvDev& c, const KvBatch& b, const KvAttend& a, const KvMembers& mem, hipStream_t s) {
    if (!b.unit0[b.n]) return;
    const bool two = a.q.type == KV_F32;
    if (c.code == KV_INT8)
        two ? by_dim<KV_INT8, 2>(c, b, a, mem, s) : by_dim<KV_INT8, 1>(c, b, a, mem, s);
    else
        two ? by_dim<KV_FP8, 2>(c, b, a, mem, s) : by_dim<KV_FP8, 1>(c, b, a, mem, s);
}

void launch_kv_shared_join(const KvDev& c, const KvAttend& a, const KvMembers& mem, const KvShares& j, hipStream_t s) {
    const int rows = mem.row0[mem.n], groups = 256 / (c.Dp / 4);
    if ((int64_t)rows * c.H <= KV_WIDE_JOIN)
        hipLaunchKernelGGL(kv_shared_join_kernel<true>, dim3((unsigned)(rows * c.H)), dim3(256), 0, s, c, a, mem, j);
    else
        hipLaunchKernelGGL(kv_shared_join_kernel<false>, dim3((unsigned)((rows + groups - 1) / groups * c.H)), dim3(256), 0, s, c, a, mem, j);
}

}  // namespace vgpu
