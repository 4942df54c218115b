// Selection of beams: of all continuations of a group's rows (beams) by a token, the k with
// the largest total = score[row] + logit[row, token] - log sum_t exp(logit[row, t]).
//
// A row is cut into slices that a workgroup holds in registers, so each logit is read once:
// the slice's largest logit and sum of exponentials, and its k best tokens.  Within a row the
// order is the logits' own, so no slice needs the row's sum for it.  A second kernel adds the
// slices' sums and takes the k best of a group's lists.
// The k-th largest of the threads' largest logits bounds the slice's k-th best from below,
// and few others reach it: those are put in order by counting.
// Differences and exponentials are float32, sums and totals float64: candidates of different
// beams lie close together, and their order is what the kernel answers.
#include <hip/hip_bf16.h>

#include "vgpu_beams.h"
#include "vgpu_kv.h"
#include "vgpu_launch.h"

namespace vgpu {

namespace {

#define BEAM_NEG (-__builtin_huge_valf())
constexpr float BEAM_LOG2E = 1.44269504088896341f;

// Floats by size as unsigned numbers, 0 and -0 alike (NaN: anywhere; its row is taken apart).
__device__ __forceinline__ uint32_t size_key(float x) {
    const uint32_t u = __float_as_uint(x + 0.f);
    return u & 0x80000000u ? ~u : u | 0x80000000u;
}
__device__ __forceinline__ float of_key(uint32_t k) {
    return __uint_as_float(k & 0x80000000u ? k & 0x7fffffffu : ~k);
}
__device__ __forceinline__ uint64_t size_key(double x) {
    const uint64_t u = (uint64_t)__double_as_longlong(x + 0.0);
    return u >> 63 ? ~u : u | 1ull << 63;
}

// What a score does to its row: 0 adds to the logits, 1 leaves every total -inf, 2 NaN.
__device__ __forceinline__ int score_kind(float s) {
    return s == BEAM_NEG ? 1 : s < __builtin_huge_valf() ? 0 : 2;
}
__device__ __forceinline__ float score_of(const BeamArgs& a, int row) { return a.scores ? a.scores[row * a.st_score] : 0.f; }

template <int T>
__device__ __forceinline__ float element(const uint4& r, int e) {
    const uint32_t w[4] = {r.x, r.y, r.z, r.w};
    if (T == KV_F32) return __uint_as_float(w[e]);
    const uint32_t h = w[e >> 1] >> (16 * (e & 1)) & 0xffffu;
    return T == KV_F16 ? (float)__builtin_bit_cast(_Float16, (uint16_t)h) : __uint_as_float(h << 16);
}

constexpr int BEAM_LIST = 1024;  // tokens that one slice puts in order

// One workgroup: one slice of one row.
template <int T, int N>
__global__ __launch_bounds__(256) void beam_slice_kernel(BeamArgs a) {
    constexpr int W = T == KV_F32 ? 4 : 8, SLICE = 256 * N * W;
    __shared__ __align__(16) uint32_t tops[256];
    __shared__ uint64_t list[BEAM_LIST];  // (key, ~token)
    __shared__ uint32_t count, shared_key, scan[4];
    __shared__ double sums[4];
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const int row = blockIdx.x / a.slices, slice = blockIdx.x - row * a.slices;
    if (score_kind(score_of(a, row))) return;  // its logits do not matter
    const size_t item = T == KV_F32 ? 4 : 2;
    const uint8_t* base = (const uint8_t*)a.logits + (int64_t)row * a.st_row * (int64_t)item;
    // Places of a row count from the 16-byte boundary before it.
    const int skew = a.st_token == 1 ? (int)((uintptr_t)base & 15) / (int)item : 0;
    const int first = slice * SLICE + tid * W - skew;  // token of the thread's first element
    const auto token = [&](int p, int e) { return first + p * (256 * W) + e; };
    uint4 x[N];
#pragma unroll
    for (int p = 0; p < N; p++) {
        const int t0 = token(p, 0);
        if (a.st_token == 1 && t0 >= 0 && t0 + W <= a.vocab) {
            x[p] = *(const uint4*)(base + (int64_t)t0 * (int64_t)item);
        } else {  // ends of the row, or elements apart: one by one, -inf outside
            uint32_t w[4] = {0, 0, 0, 0};
#pragma unroll
            for (int e = 0; e < W; e++) {
                const bool in = t0 + e >= 0 && t0 + e < a.vocab;
                const int64_t at = (int64_t)(t0 + e) * a.st_token;
                if (T == KV_F32)
                    w[e] = in ? ((const uint32_t*)base)[at] : 0xff800000u;
                else
                    w[e >> 1] |= (in ? (uint32_t)((const uint16_t*)base)[at] : T == KV_F16 ? 0xfc00u : 0xff80u) << (16 * (e & 1));
            }
            x[p] = make_uint4(w[0], w[1], w[2], w[3]);
        }
    }
    float top = BEAM_NEG;
#pragma unroll
    for (int p = 0; p < N; p++)
#pragma unroll
        for (int e = 0; e < W; e++) top = fmaxf(top, element<T>(x[p], e));
    const bool any = token(0, W - 1) >= 0 && token(0, 0) < a.vocab;  // has the thread a token?
    const uint32_t my = any ? size_key(top) : 0;
    tops[tid] = my;
    if (tid == 0) count = 0;
    __syncthreads();
    // the k-th largest of the threads' largest, and the slice's largest
    uint32_t rank = 0, big = 0;
#pragma unroll 4
    for (int j = 0; j < 256; j += 4) {
        const uint4 o = *(const uint4*)(tops + j);
        rank += (o.x > my || (o.x == my && j < tid)) + (o.y > my || (o.y == my && j + 1 < tid)) +
                (o.z > my || (o.z == my && j + 2 < tid)) + (o.w > my || (o.w == my && j + 3 < tid));
        big = max(max(big, max(o.x, o.y)), max(o.z, o.w));
    }
    if ((int)rank == a.k - 1) shared_key = my;
    __syncthreads();
    const uint32_t bound = shared_key;
    const float most = big ? of_key(big) : BEAM_NEG;
    if (my >= bound) {
#pragma unroll
        for (int p = 0; p < N; p++)
#pragma unroll
            for (int e = 0; e < W; e++) {
                const uint32_t key = size_key(element<T>(x[p], e));
                const int t = token(p, e);
                if (key >= bound && t >= 0 && t < a.vocab) {
                    const uint32_t at = atomicAdd(&count, 1u);
                    if (at < BEAM_LIST) list[at] = (uint64_t)key << 32 | (uint32_t)~t;
                }
            }
    }
    // (a row of -inf alone: exp(-inf - 0) = 0; NaN and +inf make the sum NaN)
    const float off = most == BEAM_NEG ? 0.f : most;
    float sum = 0.f;
#pragma unroll
    for (int p = 0; p < N; p++)
#pragma unroll
        for (int e = 0; e < W; e++) sum += __builtin_amdgcn_exp2f((element<T>(x[p], e) - off) * BEAM_LOG2E);
    double total = sum;
#pragma unroll
    for (int o = 32; o; o >>= 1) total += __shfl_xor(total, o);
    if (lane == 0) sums[wave] = total;
    __syncthreads();
    const size_t part = (size_t)row * a.slices + slice;
    if (tid == 0) a.top[part] = off, a.sum[part] = sums[0] + sums[1] + sums[2] + sums[3];
    uint2* best = a.best + part * a.k;
    uint32_t n = count;
    if (n > BEAM_LIST) {
        // Many reach the bound: the k-th best key itself, then the tokens above it and the first
        // of those that have it.  Every wave of the workgroup comes here.
        const auto reach = [&](uint32_t key) {  // how many of the slice's tokens are not below key
            uint32_t c = 0;
#pragma unroll
            for (int p = 0; p < N; p++)
#pragma unroll
                for (int e = 0; e < W; e++) {
                    const int t = token(p, e);
                    c += size_key(element<T>(x[p], e)) >= key && t >= 0 && t < a.vocab;
                }
#pragma unroll
            for (int o = 32; o; o >>= 1) c += (uint32_t)__shfl_xor((int)c, o);
            __syncthreads();
            if (lane == 0) scan[wave] = c;
            __syncthreads();
            return scan[0] + scan[1] + scan[2] + scan[3];
        };
        uint32_t lo = bound, hi = ~0u;  // reach(lo) >= k (NaN lie above every number)
        if (lo < hi && reach(lo + 1) < (uint32_t)a.k) hi = lo;
        while (lo < hi) {
            const uint32_t mid = lo + (hi - lo) / 2 + 1;
            if (reach(mid) >= (uint32_t)a.k) lo = mid;
            else hi = mid - 1;
        }
        __syncthreads();
        if (tid == 0) count = 0;
        __syncthreads();
#pragma unroll
        for (int p = 0; p < N; p++)
#pragma unroll
            for (int e = 0; e < W; e++) {
                const uint32_t key = size_key(element<T>(x[p], e));
                const int t = token(p, e);
                if (key > lo && t >= 0 && t < a.vocab) list[atomicAdd(&count, 1u)] = (uint64_t)key << 32 | (uint32_t)~t;
            }
        __syncthreads();
        n = count;  // below k
#pragma unroll
        for (int p = 0; p < N; p++) {
            if (n >= (uint32_t)a.k) break;
            uint32_t c = 0;
#pragma unroll
            for (int e = 0; e < W; e++) {
                const int t = token(p, e);
                c += size_key(element<T>(x[p], e)) == lo && t >= 0 && t < a.vocab;
            }
            uint32_t before = c;
#pragma unroll
            for (int o = 1; o < 64; o <<= 1) {
                const uint32_t up = (uint32_t)__shfl_up((int)before, o);
                if (lane >= o) before += up;
            }
            __syncthreads();
            if (lane == 63) scan[wave] = before;
            __syncthreads();
            before -= c;
            for (int w = 0; w < wave; w++) before += scan[w];
#pragma unroll
            for (int e = 0; e < W; e++) {
                const int t = token(p, e);
                if (size_key(element<T>(x[p], e)) == lo && t >= 0 && t < a.vocab) {
                    if (n + before < (uint32_t)a.k) list[n + before] = (uint64_t)lo << 32 | (uint32_t)~t;
                    before++;
                }
            }
            n = min(n + scan[0] + scan[1] + scan[2] + scan[3], (uint32_t)a.k);
        }
        __syncthreads();
    }
    for (uint32_t i = tid; i < n; i += 256) {
        const uint64_t mine = list[i];
        uint32_t place = 0;
#pragma unroll 4
        for (uint32_t j = 0; j < n; j++) place += list[j] > mine;
        if (place < (uint32_t)a.k) best[place] = make_uint2(__float_as_uint(of_key((uint32_t)(mine >> 32))), ~(uint32_t)mine);
    }
    for (int i = (int)n + tid; i < a.k; i += 256) best[i] = make_uint2(0, ~0u);
}

constexpr int BEAM_POOL = 2048;  // candidates that a group puts in order at once

// One workgroup: one group.  Threads go down the lists of the group's slices, L of them, from
// the top, several threads to a list (every 1024 / L-th entry each) or several lists to a thread.
__global__ __launch_bounds__(1024) void beam_group_kernel(BeamArgs a) {
    // total = (logit - largest) + lift, lift = score - log sum exp(logit - largest)
    __shared__ double lift[BEAM_MAX_BEAMS];
    __shared__ float largest[BEAM_MAX_BEAMS];
    __shared__ uint8_t kinds[BEAM_MAX_BEAMS];
    __shared__ __align__(16) uint32_t tops[256];
    __shared__ uint64_t key[BEAM_POOL];  // the total's order
    __shared__ uint64_t who[BEAM_POOL];  // beam << 32 | token
    __shared__ uint32_t count, bound32;
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const int row0 = blockIdx.x * a.beams;
    for (int b = wave; b < a.beams; b += 16) {
        const int row = row0 + b;
        int kind = score_kind(score_of(a, row));
        double total = 0.0;
        float most = BEAM_NEG;
        if (!kind) {
            const float* top = a.top + (size_t)row * a.slices;
            const double* sum = a.sum + (size_t)row * a.slices;
            // (slices of -inf alone have top 0 and sum 0)
            for (int j = lane; j < a.slices; j += 64) most = fmaxf(most, sum[j] == 0.0 ? BEAM_NEG : top[j]);
#pragma unroll
            for (int o = 32; o; o >>= 1) most = fmaxf(most, __shfl_xor(most, o));
            for (int j = lane; j < a.slices; j += 64)
                if (sum[j] != 0.0) total += sum[j] * exp2((double)(top[j] - most) * 1.4426950408889634);
#pragma unroll
            for (int o = 32; o; o >>= 1) total += __shfl_xor(total, o);
            kind = total == 0.0 ? 1 : total > 0.0 ? 0 : 2;
        }
        if (lane == 0) {
            lift[b] = kind ? 0.0 : (double)score_of(a, row) - log(total);
            largest[b] = most, kinds[b] = (uint8_t)kind;
        }
    }
    if (tid == 0) count = 0;
    __syncthreads();

    const int64_t L = (int64_t)a.beams * a.slices;
    const int per = L < 1024 ? 1024 / (int)L : 1;  // threads of a list
    const bool used = L >= 1024 || tid < per * (int)L;
    const int64_t list0 = L < 1024 ? tid % (int)L : tid;
    const int place0 = L < 1024 ? tid / (int)L : 0;
    struct Entry {
        uint64_t key, who;
        uint32_t key32;
    };
    // Entry `place` of a list: false where it ends.
    const auto entry = [&](int64_t l, int place, Entry& r) {
        const int b = (int)(l / a.slices), slice = (int)(l - (int64_t)b * a.slices);
        if (place >= a.k) return false;
        double total;
        uint32_t token;
        if (kinds[b]) {  // all totals alike: the first tokens, as one list
            if (slice || place >= a.vocab) return false;
            token = (uint32_t)place;
            total = kinds[b] == 1 ? -__builtin_huge_val() : __builtin_nan("");
        } else {
            const uint2 c = a.best[((size_t)(row0 + b) * a.slices + slice) * a.k + place];
            if (c.y == ~0u) return false;
            token = c.y;
            total = ((double)__uint_as_float(c.x) - (double)largest[b]) + lift[b];
        }
        r.key = total != total ? ~0ull : size_key(total);
        r.key32 = total != total ? ~0u : size_key((float)total);
        r.who = (uint64_t)b << 32 | token;
        return true;
    };
    // The k-th largest of 256 quads of threads' first entries, rounded to float32 (which keeps
    // the order), bounds the k-th best from below; 0 where there are not so many.
    uint32_t my = 0;
    Entry e;
    if (used)
        for (int64_t l = list0; l < L; l += 1024)
            if (entry(l, place0, e)) my = max(my, e.key32);
    my = max(my, (uint32_t)__shfl_xor((int)my, 1));
    my = max(my, (uint32_t)__shfl_xor((int)my, 2));
    if ((tid & 3) == 0) tops[tid >> 2] = my;
    __syncthreads();
    if (tid < 256) {
        const uint32_t mine = tops[tid];
        uint32_t rank = 0;
#pragma unroll 4
        for (int j = 0; j < 256; j += 4) {
            const uint4 o = *(const uint4*)(tops + j);
            rank += (o.x > mine || (o.x == mine && j < tid)) + (o.y > mine || (o.y == mine && j + 1 < tid)) +
                    (o.z > mine || (o.z == mine && j + 2 < tid)) + (o.w > mine || (o.w == mine && j + 3 < tid));
        }
        if ((int)rank == a.k - 1) bound32 = mine;
    }
    __syncthreads();
    const uint32_t least = bound32;
    uint64_t kth_key = 0, kth_who = ~0ull;  // of the pool, once it held k: what is behind cannot win

    // Put the pool's candidates in order: the k best stay, or go out.
    const auto order = [&](uint32_t n, bool out) {
        uint64_t k0[2], w0[2];
        uint32_t place[2] = {~0u, ~0u};
#pragma unroll
        for (int y = 0; y < 2; y++) {
            const uint32_t i = tid + 1024 * y;
            if (i >= n) continue;
            k0[y] = key[i], w0[y] = who[i];
            uint32_t c = 0;
#pragma unroll 4
            for (uint32_t j = 0; j < n; j++) c += key[j] > k0[y] || (key[j] == k0[y] && who[j] < w0[y]);
            place[y] = c;
        }
        __syncthreads();
#pragma unroll
        for (int y = 0; y < 2; y++) {
            if (place[y] >= (uint32_t)a.k) continue;
            if (out) {
                const size_t at = (size_t)blockIdx.x * a.k + place[y];
                const int64_t parent = row0 + (int64_t)(w0[y] >> 32);
                const uint64_t u = k0[y] >> 63 ? k0[y] & ~(1ull << 63) : ~k0[y];
                a.out_scores[at] = (float)__longlong_as_double((long long)u);
                a.out_parents[at] = parent;
                a.out_tokens[at] = (int64_t)(uint32_t)w0[y];
            } else {
                key[place[y]] = k0[y], who[place[y]] = w0[y];
            }
        }
        __syncthreads();
    };
    // Down the lists: each thread adds one candidate to the pool at a time.
    int64_t l = list0;
    int place = place0;
    bool more = used && l < L;
    while (true) {
        bool add = false;
        while (more && !add) {
            add = entry(l, place, e) && e.key32 >= least && !(e.key < kth_key || (e.key == kth_key && e.who > kth_who));
            if (add) {
                place += per;
            } else {  // the rest of the list is behind
                l += 1024, place = place0;
                more = per == 1 && l < L;
            }
        }
        if (add) {
            const uint32_t at = atomicAdd(&count, 1u);
            key[at] = e.key, who[at] = e.who;
        }
        if (!__syncthreads_or(add)) break;
        const uint32_t n = count;
        __syncthreads();
        if (n > BEAM_POOL - 1024) {
            order(n, false);
            const uint32_t kept = min(n, (uint32_t)a.k);
            if (kept == (uint32_t)a.k) kth_key = key[kept - 1], kth_who = who[kept - 1];
            if (tid == 0) count = kept;
            __syncthreads();
        }
    }
    order(count, true);
}

template <int T>
void slices_of(const BeamArgs& a, hipStream_t s) {
    const dim3 grid((unsigned)(a.rows * a.slices));
    if (a.pieces == 8)
        hipLaunchKernelGGL((beam_slice_kernel<T, 8>), grid, dim3(256), 0, s, a);
    else
        hipLaunchKernelGGL((beam_slice_kernel<T, 2>), grid, dim3(256), 0, s, a);
}

}  // namespace

void beam_plan(BeamArgs& a) {
    const int skew = a.type == KV_F32 ? 3 : 7;  // places before a row, at most
    for (int pieces : {8, 2}) {
        a.pieces = pieces;
        const int64_t slice = beam_slice(a);
        a.slices = (int)((a.vocab + skew + slice - 1) / slice);
        if ((int64_t)a.rows * a.slices >= 512) break;
    }
}

void launch_beams(const BeamArgs& a, hipStream_t s) {
    if (a.type == KV_F32)
        slices_of<KV_F32>(a, s);
    else if (a.type == KV_F16)
        slices_of<KV_F16>(a, s);
    else
        slices_of<KV_BF16>(a, s);
    hipLaunchKernelGGL(beam_group_kernel, dim3((unsigned)(a.rows / a.beams)), dim3(1024), 0, s, a);
}

}  // namespace vgpu
