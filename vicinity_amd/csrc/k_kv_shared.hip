// Softmax attention of sequences that hold the same first blocks: the rows of all of them
// over the shared slots, read once, each over its own, and the join of the parts.
//
// Few rows (kv_step_kernel): 61 sequences of 32 query heads on 8 of 128 under 8192 shared slots
// 43 us (135 MB in; the vector unit 44% busy: 16 workgroups convert the same tiles for 16 rows
// each, three to a compute unit), 64 beams of 8 prompts of 3000 slots 18 us (48 MB; latency:
// some eight tiles to a workgroup).  Many (kv_chunk_kernel): 48 sequences of 64 query heads on 8 of 128
// over 65536 shared slots 137 us, 750 TFLOP/s (matrix unit 34% busy, vector unit 49%; 33 MB of
// partial rows).  One launch of both kernels' code for shared and own slots was slower (the
// first 60 us for 56 with the join, the last 159 to 205 for 145), as were two tiles of 16 rows
// to a workgroup of few (64 beams 32 us for 18).
#include "kv_attend.h"

namespace vgpu {

namespace {

// A row's parts, of the shared slots and of its own, by `share` groups of Dp / 4 threads, each of
// which takes parts in turn, four at a time: the sums o and l go by the power of 2 that a part's
// m stands below the largest, o also by the power of 2 that its S does.  Bound by latency: the
// parts of a row lie one launch's tiles apart (33 MB, 10.5 us; 3 MB 4.9).
__global__ __launch_bounds__(256) void kv_shared_join_kernel(KvDev c, KvAttend a, KvMembers mem, KvShares j, int share) {
    __shared__ floatx4 sh_o[256];
    __shared__ float sh_m[64], sh_l[64], sh_top[64];
    __shared__ int row0[KV_BATCH + 1];
    const int tid = threadIdx.x;
    const int width = c.Dp / 4, per_wg = 256 / width / share, grp = tid / width, d4 = tid % width;
    if (tid <= mem.n) row0[tid] = mem.row0[tid];
    __syncthreads();
    const int h = kv_mod(blockIdx.x, c.by_heads);
    const int row = kv_div(blockIdx.x, c.by_heads) * per_wg + grp / share, mine = grp % share;
    const bool used = grp < per_wg * share && row < row0[mem.n];
    int m = 0, end = mem.n;
    while (end - m > 1) {
        const int mid = (m + end) / 2;
        if (row0[mid] <= row) m = mid;
        else end = mid;
    }
    const int r0 = row - row0[m];  // its row among the sequence's
    float mx = KV_NEG, top = KV_FIRST, l = 0.f;
    floatx4 o = {0.f, 0.f, 0.f, 0.f};
    if (used) {
        const int s0 = j.splits[0][m], splits = s0 + j.splits[1][m];
        size_t first[2], step[2];
#pragma unroll
        for (int y = 0; y < 2; y++) {
            const int r = r0 + (y ? 0 : j.row0[m]), tile = r / j.rows[y];
            first[y] = j.base[y] + ((size_t)(j.unit[y][m] + tile) * c.H + h) * j.rows[y] + (r - tile * j.rows[y]);
            step[y] = (size_t)j.tiles[y][m] * c.H * j.rows[y];
        }
        for (int s = mine; s < splits; s += 4 * share) {
            float2 ml[4];
            float st[4];
            floatx4 po[4];
#pragma unroll
            for (int x = 0; x < 4; x++) {
                const int t = min(s + x * share, splits - 1);
                const size_t at = t < s0 ? first[0] + t * step[0] : first[1] + (t - s0) * step[1];
                ml[x] = a.part_ml[at], st[x] = a.part_s[at];
                po[x] = *(const floatx4*)(a.part_o + at * c.Dp + d4 * 4);
            }
            float now = mx, high = top;
#pragma unroll
            for (int x = 0; x < 4; x++) {
                // past the end, or without a slot (and then without an o)
                if (s + x * share >= splits || (ml[x].x == KV_NEG && ml[x].y == 0.f))
                    ml[x] = make_float2(KV_NEG, 0.f), st[x] = KV_FIRST, po[x] = floatx4{0.f, 0.f, 0.f, 0.f};
                now = fmaxf(now, ml[x].x), high = fmaxf(high, st[x]);
            }
            const float down = kv_join_factor(mx, l, now);
            l *= down, o *= ldexpf(down, (int)(top - high));
#pragma unroll
            for (int x = 0; x < 4; x++) {
                const float f = kv_join_factor(ml[x].x, ml[x].y, now);
                l += f * ml[x].y;
                o += po[x] * ldexpf(f, (int)(st[x] - high));
            }
            mx = now, top = high;
        }
    }
    if (share > 1) {
        sh_o[tid] = o;
        if (d4 == 0) sh_m[grp] = mx, sh_l[grp] = l, sh_top[grp] = top;
        __syncthreads();
        if (mine || !used) return;
        for (int x = 1; x < share; x++) mx = fmaxf(mx, sh_m[grp + x]), top = fmaxf(top, sh_top[grp + x]);
        o = floatx4{0.f, 0.f, 0.f, 0.f}, l = 0.f;
        for (int x = 0; x < share; x++) {
            const float f = kv_join_factor(sh_m[grp + x], sh_l[grp + x], mx);
            l += f * sh_l[grp + x];
            o += sh_o[tid + x * width] * ldexpf(f, (int)(sh_top[grp + x] - top));
        }
    }
    if (!used) return;
    const int tok = kv_div(r0, a.by_group);
    const size_t out = (size_t)(mem.tok0[m] + tok) * c.H * a.G + (size_t)h * a.G + (r0 - tok * a.G);
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
    if constexpr (kv_shared_many(S * 32, PARTS))
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
    int most = 1;  // (none, where all sequences are empty)
    for (int m = 0; m < mem.n; m++) most = j.splits[0][m] + j.splits[1][m] > most ? j.splits[0][m] + j.splits[1][m] : most;
    // A group of threads for every four parts, up to 768 workgroups (48 tokens of 64 query
    // heads, 22 parts each: 10 us with two, 14 with six; 512 rows in all of 25 parts: 8.5 and 6.4).
    const int rows = mem.row0[mem.n], groups = 256 / (c.Dp / 4);
    const int64_t room = 768ll * groups / ((int64_t)rows * c.H);
    int share = (most + 3) / 4 < groups ? (most + 3) / 4 : groups;
    if (share > room) share = room > 1 ? (int)room : 1;
    const int per_wg = groups / share;
    hipLaunchKernelGGL(kv_shared_join_kernel, dim3((unsigned)((rows + per_wg - 1) / per_wg * c.H)), dim3(256), 0, s, c, a, mem, j, share);
}

}  // namespace vgpu
