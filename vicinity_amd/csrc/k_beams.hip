// Selection of beams: of all continuations of a group's rows (beams) by a token, the k with
// the largest total = score[row] + logit[row, token] - log sum_t exp(logit[row, t]).
//
// A row is cut into slices that a workgroup holds in registers, so each logit is read once:
// the slice's largest logit and sum of exponentials, and its k best tokens.  Within a row the
// order is the logits' own, so no slice needs the row's sum for it.  A second kernel adds the
// slices' sums and takes the k best of a group's lists.
// The largest logits of threads bound the slice's k-th best from below, and few others reach
// that: those are put in order by counting.
// Differences and exponentials are float32, all sums and totals float64: candidates of different
// beams lie close together, and their order is what the kernel answers (a thread's exponentials
// added in float32 first: 2 us less of 41 for 512 rows of 100003, and rows told apart no closer
// than 2^-17).
#include <hip/hip_bf16.h>

#include "vgpu_beams.h"
#include "vgpu_kv.h"
#include "vgpu_launch.h"

namespace vgpu {

namespace {

typedef unsigned int u32x4 __attribute__((ext_vector_type(4)));

#define BEAM_NEG (-__builtin_huge_valf())
constexpr float BEAM_LOWEST = -0x1.fffffep127f;  // of all numbers
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

// Largest element of a piece, a NaN only if all are (fmaxf would quiet each operand first).
template <int T>
__device__ __forceinline__ float piece_top(const uint4& r) {
    float x[T == KV_F32 ? 4 : 8], m;
#pragma unroll
    for (int e = 0; e < (T == KV_F32 ? 4 : 8); e++) x[e] = element<T>(r, e);
    asm("v_max3_f32 %0, %1, %2, %3" : "=v"(m) : "v"(x[0]), "v"(x[1]), "v"(x[2]));
    if (T == KV_F32) {
        asm("v_max_f32 %0, %1, %2" : "=v"(m) : "v"(m), "v"(x[3]));
    } else {
        asm("v_max3_f32 %0, %1, %2, %3" : "=v"(m) : "v"(m), "v"(x[3]), "v"(x[4 % (T == KV_F32 ? 4 : 8)]));
        asm("v_max3_f32 %0, %1, %2, %3" : "=v"(m) : "v"(m), "v"(x[5 % (T == KV_F32 ? 4 : 8)]), "v"(x[6 % (T == KV_F32 ? 4 : 8)]));
        asm("v_max_f32 %0, %1, %2" : "=v"(m) : "v"(m), "v"(x[7 % (T == KV_F32 ? 4 : 8)]));
    }
    return m;
}

constexpr int BEAM_LIST = 1024;   // tokens that one slice puts in order
constexpr int BEAM_PIECES = 512;  // pieces that are looked through for them

// One workgroup: one slice of one row, loaded at once.  Bound by the vector unit where rows are
// many: a conversion, a comparison, a difference, a product, an exponential (four times as
// long), a conversion to float64 and a sum for each logit (512 rows of 100003 in bfloat16: 32 us,
// 3.2 TB/s, the vector unit 52% busy and the loads before it not hidden; 4 rows of 32000 in float32:
// 6 us).  The hits counted by each thread before they are taken to LDS: 10 us more.
template <int T, int N>
__global__ __launch_bounds__(256, T == KV_F32 ? 6 : 7) void beam_slice_kernel(BeamArgs a) {
    constexpr int W = T == KV_F32 ? 4 : 8, HALF = (N + 1) / 2;
    __shared__ uint64_t list[BEAM_LIST];  // (key, ~token)
    __shared__ uint4 found[BEAM_PIECES];  // pieces with an element that reaches the bound
    __shared__ int found_at[BEAM_PIECES];
    __shared__ uint32_t count, pieces, scan[4], bounds[4];
    __shared__ float tops[4];
    __shared__ double sums[4];
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const int row = __builtin_amdgcn_readfirstlane(blockIdx.x / a.slices), slice = blockIdx.x - row * a.slices;
    if (score_kind(score_of(a, row))) return;  // its logits do not matter
    const size_t item = T == KV_F32 ? 4 : 2;
    typedef const __attribute__((address_space(1))) uint8_t* Bytes;
    const Bytes base = (Bytes)a.logits + (int64_t)row * a.st_row * (int64_t)item;
    // Places of a row count from the 16-byte boundary before it.
    const int skew = a.st_token == 1 ? (int)((uintptr_t)base & 15) / (int)item : 0;
    const int begin = slice * a.pieces * (256 * W) - skew, first = begin + tid * W;  // tokens at the slice's and the thread's first place
    const int np = min(a.pieces, (a.vocab - begin + 256 * W - 1) / (256 * W));  // pieces of a thread, 0 or less: none
    const auto token = [&](int p, int e) { return first + p * (256 * W) + e; };
    const bool apart = a.st_token != 1;
    const auto piece = [&](int t0) {
        return __builtin_bit_cast(uint4, *(const __attribute__((address_space(1))) u32x4*)(base + (int64_t)t0 * (int64_t)item));
    };
    const auto load = [&](int p) {
        const int t0 = token(p, 0);
        if (!apart && t0 >= 0 && t0 + W <= a.vocab) return piece(t0);
        constexpr uint32_t none = T == KV_F32 ? 0xff800000u : T == KV_F16 ? 0xfc00fc00u : 0xff80ff80u;  // -inf
        if (t0 >= a.vocab) return make_uint4(none, none, none, none);
        // ends of the row, or elements apart: one by one, those outside from an end
        uint32_t r[W], w[4] = {0, 0, 0, 0};
#pragma unroll
        for (int e = 0; e < W; e++) {
            const Bytes at = base + (int64_t)min(max(t0 + e, 0), a.vocab - 1) * a.st_token * (int64_t)item;
            r[e] = T == KV_F32 ? *(const __attribute__((address_space(1))) uint32_t*)at
                               : (uint32_t) * (const __attribute__((address_space(1))) uint16_t*)at;
        }
#pragma unroll
        for (int e = 0; e < W; e++) {
            const bool in = t0 + e >= 0 && t0 + e < a.vocab;
            if (T == KV_F32) w[e] = in ? r[e] : none;
            else w[e >> 1] |= (in ? r[e] : none >> 16) << (16 * (e & 1));
        }
        return make_uint4(w[0], w[1], w[2], w[3]);
    };
    // (the elements stay as they lie in memory: 148 registers and more, kept as floats)
    const auto keep = [](uint4(&r)[N]) {
#pragma unroll
        for (int p = 0; p < N; p++) asm volatile("" : "+v"(r[p].x), "+v"(r[p].y), "+v"(r[p].z), "+v"(r[p].w));
    };
    uint4 x[N];
    if (!apart && begin >= 0 && begin + np * (256 * W) <= a.vocab) {
#pragma unroll
        for (int p = 0; p < N; p++)
            if (p < np) x[p] = piece(token(p, 0));
    } else {
#pragma unroll
        for (int p = 0; p < N; p++)
            if (p < np) x[p] = load(p);
    }
    if (tid == 0) count = 0, pieces = 0;
    // the largest of each piece, and of each half of the pieces (NaN are passed over)
    float tp[N], th[2] = {BEAM_NEG, BEAM_NEG};
#pragma unroll
    for (int p = 0; p < N; p++) {
        tp[p] = p < np ? piece_top<T>(x[p]) : __builtin_nanf("");
        th[p / HALF] = fmaxf(th[p / HALF], tp[p]);
    }
    keep(x);
    float top = fmaxf(th[0], th[1]);
    // A lower bound of the slice's k-th best: each wave finds the largest number (the first BITS
    // bits of its key) that a quarter of k halves' largest reach, and the least of the four is
    // reached by k.  In a short slice the waves that have tokens take more.  0: no such number.
    {
        constexpr int BITS = T == KV_BF16 ? 16 : T == KV_F16 ? 19 : 18, SHIFT = 32 - BITS;
        const uint32_t k0 = token(0, 0) < a.vocab ? size_key(th[0]) >> SHIFT : 0;
        const uint32_t k1 = HALF < np && token(HALF, 0) < a.vocab ? size_key(th[1]) >> SHIFT : 0;
        const int used = min(max((a.vocab - begin + W - 1) / W, 0), 256);  // threads that have a token
        const auto most_of = [&](int r) {  // halves, with at most r of each wave
            return min(r, min(used, 64)) + min(r, min(max(used - 64, 0), 64)) + min(r, min(max(used - 128, 0), 64)) +
                   min(r, max(used - 192, 0));
        };
        int need = (a.k + 3) / 4;
        while (most_of(need) < a.k && need < 64) need++;
        const bool enough = most_of(need) >= a.k;
        need = min(need, min(max(used - 64 * wave, 0), 64));
        uint32_t key = 0;
#pragma unroll
        for (int bit = BITS - 1; bit >= 0; bit--) {
            const uint32_t more = key | 1u << bit;
            if (__popcll(__builtin_amdgcn_ballot_w64(k0 >= more)) + __popcll(__builtin_amdgcn_ballot_w64(k1 >= more)) >= need) key = more;
        }
#pragma unroll
        for (int o = 32; o; o >>= 1) top = fmaxf(top, __shfl_xor(top, o));
        if (lane == 0) bounds[wave] = enough ? key << SHIFT : 0, tops[wave] = top;
    }
    __syncthreads();
    const uint32_t bound = min(min(bounds[0], bounds[1]), min(bounds[2], bounds[3]));
    // No such number, or -inf (a grammar that leaves few tokens): all numbers are looked at, and the
    // first tokens of -inf fill up (40 tokens of 100003, 512 rows: 43 us for both kernels; the search
    // below, which took these slices before, 617).
    const uint32_t lowest = size_key(BEAM_LOWEST);
    const bool open = bound < lowest;
    const float least = open ? BEAM_LOWEST : of_key(bound);
    const float most = fmaxf(fmaxf(tops[0], tops[1]), fmaxf(tops[2], tops[3]));
    // Pieces that reach the bound go to LDS, where their elements are looked at side by side.
    uint32_t hits = 0;
#pragma unroll
    for (int p = 0; p < N; p++) hits += tp[p] >= least;
    if (hits) {
        uint32_t at = atomicAdd(&pieces, hits);
#pragma unroll
        for (int p = 0; p < N; p++)
            if (tp[p] >= least) {
                if (at < BEAM_PIECES) found[at] = x[p], found_at[at] = token(p, 0);
                at++;
            }
    }
    keep(x);
    // exp(x - off) as 2^(x log2 e - c), c = off log2 e rounded, and what that rounding did taken
    // back from the sum.  (A row of -inf alone: off 0, every term 0; NaN makes the sum NaN.)
    const float off = most == BEAM_NEG ? 0.f : most;
    const float c = off * BEAM_LOG2E, rest = __builtin_fmaf(off, BEAM_LOG2E, -c);
    const bool plain = fabsf(off) < 0x1p12f;  // then rest is below 2^-11
    double total = 0.0;
    if (plain) {
#pragma unroll
        for (int p = 0; p < N; p++)
            if (p < np)
#pragma unroll
            for (int e = 0; e < W; e++) total += (double)__builtin_amdgcn_exp2f(__builtin_fmaf(element<T>(x[p], e), BEAM_LOG2E, -c));
    } else {  // (c may not be finite; +inf makes the sum NaN)
#pragma unroll 1
        for (int p = 0; p < np; p++) {
            const uint4 r = load(p);
#pragma unroll
            for (int e = 0; e < W; e++) total += (double)__builtin_amdgcn_exp2f((element<T>(r, e) - off) * BEAM_LOG2E);
        }
    }
#pragma unroll
    for (int o = 32; o; o >>= 1) total += __shfl_xor(total, o);
    if (lane == 0) sums[wave] = total;
    __syncthreads();
    const size_t part = (size_t)row * a.slices + slice;
    if (tid == 0) {
        const double y = plain ? (double)rest * -0.6931471805599453 : 0.0;  // 2^-rest by its series
        a.top[part] = off, a.sum[part] = (sums[0] + sums[1] + sums[2] + sums[3]) * (1.0 + y + y * y * 0.5);
    }
    uint2* best = a.best + part * a.k;
    uint32_t n = pieces;
    if (n <= BEAM_PIECES) {
        for (uint32_t i = tid; i < n * W; i += 256) {
            const int t = found_at[i / W] + (int)(i & (W - 1));
            float v;
            if (T == KV_F32) v = ((const float*)found)[i];
            else if (T == KV_F16) v = (float)((const _Float16*)found)[i];
            else v = __uint_as_float((uint32_t)((const uint16_t*)found)[i] << 16);
            if (v >= least && t >= 0 && t < a.vocab) {
                const uint32_t at = atomicAdd(&count, 1u);
                if (at < BEAM_LIST) list[at] = (uint64_t)size_key(v) << 32 | (uint32_t)~t;
            }
        }
        __syncthreads();
        n = count;
    } else {
        n = BEAM_LIST + 1;
    }
    uint32_t tie = size_key(BEAM_NEG);  // tokens of this key go behind the list, the first ones, up to k
    if (n > BEAM_LIST) {
        // Many reach the bound: the k-th best key itself, then the tokens above it and the first
        // of those that have it.  Every wave of the workgroup comes here.
        // (the logits come from memory again: this is rare, and needs their registers)
        const uint32_t high = size_key(most);  // (keys above it are NaN, whose rows are taken apart)
        const auto reach = [&](uint32_t key) {  // how many of the slice's tokens are not below key
            uint32_t c = 0;
#pragma unroll 1
            for (int p = 0; p < np; p++) {
                const uint4 r = load(p);
#pragma unroll
                for (int e = 0; e < W; e++) {
                    const int t = token(p, e);
                    const uint32_t x = size_key(element<T>(r, e));
                    c += x >= key && x <= high && t >= 0 && t < a.vocab;
                }
            }
#pragma unroll
            for (int o = 32; o; o >>= 1) c += (uint32_t)__shfl_xor((int)c, o);
            __syncthreads();
            if (lane == 0) scan[wave] = c;
            __syncthreads();
            return scan[0] + scan[1] + scan[2] + scan[3];
        };
        // (more than BEAM_LIST tokens or BEAM_PIECES pieces reach lo)
        uint32_t lo = max(bound, lowest), hi = high;
        if (reach(hi) >= (uint32_t)a.k) lo = hi;  // (one value, for example)
        while (lo < hi) {
            const uint32_t mid = lo + (hi - lo) / 2 + 1;
            if (reach(mid) >= (uint32_t)a.k) lo = mid;
            else hi = mid - 1;
        }
        __syncthreads();
        if (tid == 0) count = 0;
        __syncthreads();
#pragma unroll 1
        for (int p = 0; p < np; p++) {
            const uint4 r = load(p);
#pragma unroll
            for (int e = 0; e < W; e++) {
                const uint32_t key = size_key(element<T>(r, e));
                const int t = token(p, e);
                if (key > lo && key <= high && t >= 0 && t < a.vocab) list[atomicAdd(&count, 1u)] = (uint64_t)key << 32 | (uint32_t)~t;
            }
        }
        __syncthreads();
        n = count;  // below k
        tie = lo;
    }
    if (n < (uint32_t)a.k) {
#pragma unroll 1
        for (int p = 0; p < np; p++) {
            if (n >= (uint32_t)a.k) break;
            const uint4 r = load(p);
            uint32_t c = 0;
#pragma unroll
            for (int e = 0; e < W; e++) {
                const int t = token(p, e);
                c += size_key(element<T>(r, e)) == tie && t >= 0 && t < a.vocab;
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
                if (size_key(element<T>(r, e)) == tie && t >= 0 && t < a.vocab) {
                    if (n + before < (uint32_t)a.k) list[n + before] = (uint64_t)tie << 32 | (uint32_t)~t;
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

constexpr int BEAM_POOL = 2048;     // candidates that a group puts in order at once
constexpr int BEAM_SAMPLES = 4096;  // keys of samples that are kept
constexpr int BEAM_BINS = 2048;

// One workgroup: one group, of L lists (one of each row and slice), k places each.
//
// Places 0, 1, 3, 7, ... of every list are its samples; a sample stands for the places from the
// one before it to its own.  Of the totals rounded to float32 (which keeps the order) the
// largest that samples for k places reach, found by two digits of 11 bits, bounds the k-th best
// from below; and as a list's places beyond its last sample that reaches it are fewer than
// those up to there, about 2 k candidates pass.
//
// Bound by latency: 64 groups of 8 rows, 16 results, 7 lists to a row: 9 us; 3 groups of 48
// rows, 96 results, 5 lists: 16; lists walked thread by thread until they end: 93.  Up to 256
// candidates go in order by counting, more by a bitonic sort (512: 7.5 us, by counting 27).
__global__ __launch_bounds__(1024) void beam_group_kernel(BeamArgs a) {
    // total = (logit - largest) + lift, lift = score - log sum exp(logit - largest)
    __shared__ double lift[BEAM_MAX_BEAMS];
    __shared__ float largest[BEAM_MAX_BEAMS];
    __shared__ uint8_t kinds[BEAM_MAX_BEAMS];
    __shared__ ulonglong2 pool[BEAM_POOL];  // the total's order; who: beam, logit's order, place
    __shared__ uint32_t sample[BEAM_SAMPLES];
    __shared__ uint32_t hist[BEAM_BINS];
    __shared__ uint32_t place[256];
    __shared__ uint32_t scan[18], count;
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const int row0 = blockIdx.x * a.beams;
    // Equal totals go by beam, then by logit (float64 may hold the totals of different ones as
    // equal), then by the place in the row's lists, where equal logits lie in their tokens' order.
    // A beam and a place have 32 bits together, for a group has fewer than 2^31 places.
    const int row_places = a.slices * a.k, place_bits = row_places > 1 ? 32 - __clz(row_places - 1) : 0;
    // 16 lanes to a row
    for (int b0 = 0; b0 < a.beams; b0 += 64) {
        const int b = min(b0 + (tid >> 4), a.beams - 1), row = row0 + b;
        int kind = score_kind(score_of(a, row));
        double total = 0.0;
        float most = BEAM_NEG;
        const float* top = a.top + (size_t)row * a.slices;
        const double* sum = a.sum + (size_t)row * a.slices;
        // (slices of -inf alone have top 0 and sum 0; rows of another kind have neither)
        if (!kind)
            for (int j = lane & 15; j < a.slices; j += 16) most = fmaxf(most, sum[j] == 0.0 ? BEAM_NEG : top[j]);
#pragma unroll
        for (int o = 8; o; o >>= 1) most = fmaxf(most, __shfl_xor(most, o));
        if (!kind)
            for (int j = lane & 15; j < a.slices; j += 16)
                if (sum[j] != 0.0) total += sum[j] * exp2((double)(top[j] - most) * 1.4426950408889634);
#pragma unroll
        for (int o = 8; o; o >>= 1) total += __shfl_xor(total, o);
        if (!kind) kind = total == 0.0 ? 1 : total > 0.0 ? 0 : 2;
        if ((lane & 15) == 0 && b0 + (tid >> 4) < a.beams) {
            lift[b] = kind ? 0.0 : (double)score_of(a, row) - log(total);
            largest[b] = most, kinds[b] = (uint8_t)kind;
        }
    }
    if (tid == 0) count = 0;
    for (int i = tid; i < BEAM_BINS; i += 1024) hist[i] = 0;
    __syncthreads();

    struct Entry {
        uint64_t key, who;
        uint32_t key32;
    };
    // Entry `at` of a list: false where it has none.
    const auto entry = [&](uint32_t l, int at, Entry& r) {
        const uint32_t b = l / (uint32_t)a.slices, slice = l - b * (uint32_t)a.slices;
        double total;
        uint32_t logit = 0;
        if (kinds[b]) {  // all totals alike: the first tokens, as one list
            if (slice || at >= a.vocab) return false;
            total = kinds[b] == 1 ? -__builtin_huge_val() : __builtin_nan("");
        } else {
            const uint2 c = a.best[((size_t)row0 * a.slices + l) * a.k + at];
            if (c.y == ~0u) return false;
            logit = ~size_key(__uint_as_float(c.x));
            total = ((double)__uint_as_float(c.x) - (double)largest[b]) + lift[b];
        }
        r.key = total != total ? ~0ull : size_key(total);
        r.key32 = total != total ? ~0u : size_key((float)total);
        r.who = ((uint64_t)b << 32 | logit) << place_bits | (slice * (uint32_t)a.k + (uint32_t)at);
        return true;
    };
    // The digit in which the samples' weights, from the top, reach `need`.
    const auto digit = [&](uint32_t& need) {
        const int hi = BEAM_BINS - 1 - 2 * tid;  // this thread's two bins, from the top
        const uint32_t c0 = hist[hi], c1 = hist[hi - 1];
        uint32_t sum = c0 + c1;
#pragma unroll
        for (int o = 1; o < 64; o <<= 1) {
            const uint32_t up = (uint32_t)__shfl_up((int)sum, o);
            if (lane >= o) sum += up;
        }
        if (lane == 63) scan[wave] = sum;
        if (tid == 0) scan[16] = ~0u;
        __syncthreads();
        for (int w = 0; w < wave; w++) sum += scan[w];
        const uint32_t before = sum - c0 - c1;
        if (before < need && sum >= need) {  // one thread at most
            const bool one = before + c0 >= need;
            scan[16] = (uint32_t)(one ? hi : hi - 1);
            scan[17] = need - before - (one ? 0 : c0);
        }
        hist[hi] = hist[hi - 1] = 0;
        __syncthreads();
        const uint32_t d = scan[16];
        need = scan[17];
        return d;
    };
    const uint32_t L = (uint32_t)a.beams * a.slices, places = L * (uint32_t)a.k;
    const bool few = places <= 256;  // put in order without a bound
    const int steps = 32 - __clz(a.k);  // samples of a list
    const auto each_sample = [&](auto&& f) {
        for (uint32_t i = tid; i < L * steps; i += 1024) {
            const int step = (int)(i / L);
            const int at = (1 << step) - 1;
            if (at < a.k) f(i, i - step * L, at, step ? 1u << (step - 1) : 1u);
        }
    };
    Entry e;
    const bool keep = L * steps <= BEAM_SAMPLES;
    uint32_t need = (uint32_t)a.k, least = 0;
    if (!few) {
        each_sample([&](uint32_t i, uint32_t l, int at, uint32_t weight) {
            const uint32_t k32 = entry(l, at, e) ? e.key32 : 0;
            if (keep) sample[i] = k32;
            if (k32) atomicAdd(&hist[k32 >> 21], weight);
        });
        __syncthreads();
        const uint32_t d0 = digit(need);
        if (d0 != ~0u) {
            each_sample([&](uint32_t i, uint32_t l, int at, uint32_t weight) {
                const uint32_t k32 = keep ? sample[i] : entry(l, at, e) ? e.key32 : 0;
                if (k32 && k32 >> 21 == d0) atomicAdd(&hist[k32 >> 10 & 2047u], weight);
            });
            __syncthreads();
            least = d0 << 21 | digit(need) << 10;
        }
    }

    // Put the pool's n candidates in order: the k best stay in front, or go out.
    const auto before = [](const ulonglong2& x, const ulonglong2& y) { return (x.x > y.x) | ((x.x == y.x) & (x.y < y.y)); };
    const auto order = [&](uint32_t n, bool out) {
        ulonglong2 mine;
        uint32_t to = ~0u;
        if (n <= 256) {
            // by counting, 4 threads to a candidate: first by the upper halves of the orders, and
            // in full where those are equal
            const uint32_t* upper = (const uint32_t*)pool + 1;
            const uint32_t i = tid & 255;
            if (tid < 256) place[tid] = 0;
            __syncthreads();
            if (i < n) {
                mine = pool[i];
                const uint32_t top = (uint32_t)(mine.x >> 32);
                uint32_t above = 0, equal = 0;
#pragma unroll 8
                for (uint32_t j = tid >> 8; j < n; j += 4) above += upper[4 * j] > top, equal += upper[4 * j] == top;
                if (equal > (i % 4 == tid >> 8 ? 1u : 0u))
                    for (uint32_t j = tid >> 8; j < n; j += 4) above += upper[4 * j] == top && before(pool[j], mine);
                if (above) atomicAdd(&place[i], above);
            }
            __syncthreads();
            if (tid < (int)n) to = place[tid];
        } else {
            uint32_t size = 512;
            while (size < n) size <<= 1;
            for (uint32_t i = n + tid; i < size; i += 1024) pool[i] = make_ulonglong2(0, ~0ull);
            for (uint32_t run = 2; run <= size; run <<= 1)
                for (uint32_t step = run >> 1; step; step >>= 1) {
                    __syncthreads();
                    for (uint32_t x = tid; x < size / 2; x += 1024) {
                        const uint32_t i = 2 * x - (x & (step - 1)), j = i + step;
                        const ulonglong2 p = pool[i], q = pool[j];
                        if (before(q, p) == !(i & run)) pool[i] = q, pool[j] = p;
                    }
                }
            __syncthreads();
            if (tid < a.k && tid < (int)n) mine = pool[tid], to = tid;
        }
        __syncthreads();
        if (to < (uint32_t)a.k) {
            if (out) {
                const size_t at = (size_t)blockIdx.x * a.k + to;
                const uint64_t u = mine.x >> 63 ? mine.x & ~(1ull << 63) : ~mine.x;
                a.out_scores[at] = (float)__longlong_as_double((long long)u);
                const int b = (int)(mine.y >> place_bits >> 32);
                const uint32_t spot = (uint32_t)mine.y & (uint32_t)((1ull << place_bits) - 1);
                a.out_parents[at] = row0 + b;
                a.out_tokens[at] = kinds[b] ? spot : a.best[(size_t)(row0 + b) * row_places + spot].y;
            } else {
                pool[to] = mine;
            }
        }
        __syncthreads();
    };
    // 16 lanes to a list, as far as the sample that does not reach the bound
    for (uint32_t l0 = 0; l0 < L; l0 += 64) {
        const uint32_t l = l0 + (tid >> 4);
        const int step = lane & 15;
        bool reaches = false;
        if (l < L && step < steps) {
            const int at = (1 << step) - 1;
            reaches = few || (keep ? sample[step * L + l] >= max(least, 1u) : entry(l, at, e) && e.key32 >= least);
        }
        const int reached = __popc((uint32_t)(__ballot(reaches) >> (lane & 48)) & 0xffffu);
        const int end = reached == steps ? a.k : (1 << reached) - 1;
        for (int at = step; at < end; at += 16)
            if (entry(l, at, e) && e.key32 >= least) {
                const uint32_t to = atomicAdd(&count, 1u);
                if (to < BEAM_POOL) pool[to] = make_ulonglong2(e.key, e.who);
            }
    }
    __syncthreads();
    if (count > BEAM_POOL) {
        // Many equal totals: 1024 entries at a time, beside the k best of those before.
        uint64_t kth_key = 0, kth_who = ~0ull;
        __syncthreads();
        if (tid == 0) count = 0;
        __syncthreads();
        for (uint32_t i0 = 0; i0 < places; i0 += 1024) {
            const uint32_t i = i0 + tid, l = i / (uint32_t)a.k;
            if (i < places && entry(l, (int)(i - l * a.k), e) && e.key32 >= least &&
                (e.key > kth_key || (e.key == kth_key && e.who < kth_who))) {
                const uint32_t at = atomicAdd(&count, 1u);
                pool[at] = make_ulonglong2(e.key, e.who);
            }
            __syncthreads();
            const uint32_t n = count;
            __syncthreads();
            if (n > BEAM_POOL - 1024) {
                order(n, false);
                const uint32_t kept = min(n, (uint32_t)a.k);
                if (kept == (uint32_t)a.k) kth_key = pool[kept - 1].x, kth_who = pool[kept - 1].y;
                if (tid == 0) count = kept;
                __syncthreads();
            }
        }
    }
    order(count, true);
}

template <int T>
void slices_of(const BeamArgs& a, hipStream_t s) {
    const dim3 grid((unsigned)(a.rows * a.slices));
    if (a.pieces > 2)
        hipLaunchKernelGGL((beam_slice_kernel<T, 8>), grid, dim3(256), 0, s, a);
    else
        hipLaunchKernelGGL((beam_slice_kernel<T, 2>), grid, dim3(256), 0, s, a);
}

}  // namespace

void beam_plan(BeamArgs& a) {
    const int skew = a.type == KV_F32 ? 3 : 7;  // places before a row, at most
    const int64_t piece = 256 * (a.type == KV_F32 ? 4 : 8), all = (a.vocab + skew + piece - 1) / piece;
    // Slices of at most 8 pieces, alike; of 2 where that leaves the card's workgroups idle.
    for (int most : {8, 2}) {
        a.slices = (int)((all + most - 1) / most);
        a.pieces = (int)((all + a.slices - 1) / a.slices);
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
