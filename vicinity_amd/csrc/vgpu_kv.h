// The attention memory's device layout and the launchers of its kernels.
//
// The pool is made of blocks of B slots; a block holds every head's part one
// after the other, and a part is B / 32 tiles of 32 slots.  A tile is 32 * Dp
// bytes of key codes, then 32 * Dp bytes of value codes, in the order in which the
// lanes of a wave take them as operands of the 16x16x32 matrix instruction, so every
// load of the attention is 16 contiguous bytes per lane and no element changes lanes
// between the two products.  Dp is the smallest of 64, 96, 128, 192 and 256 that holds
// the head dimension, for which the kernels are compiled; the rest is stored and read
// as zeros (dimension 32 takes the bytes of 64, 136 those of 192):
//
//   keys    operand (j, s) = slots 16 j .. 16 j + 15 x dims 32 s .. 32 s + 31;
//           lane 16 g + r holds slot 16 j + r, dims 32 s + 8 g .. + 7.
//   values  operand i = dims 16 i .. 16 i + 15 x the 32 slots;
//           lane 16 g + r holds dim 16 i + r, slots 4 g .. 4 g + 3 and
//           16 + 4 g .. 16 + 4 g + 3: the slots whose scores that lane gets from
//           the key products j = 0 and j = 1.
//
// Operands 2 p and 2 p + 1 (keys: number j * Dp / 32 + s) share 16 bytes of a lane.
// int8 codes are stored with 128 added; e4m3 codes as they are.
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

namespace vgpu {

constexpr int KV_TILE = 32;
constexpr int KV_MAX_DIM = 256;
// sequences of one launch: their batch description is a kernel argument
constexpr int KV_BATCH = 128;

enum KvCode { KV_INT8 = 0, KV_FP8 = 1 };
enum KvType { KV_F32 = 0, KV_F16 = 1, KV_BF16 = 2 };

// Division of numbers below 2^30 by a launch's constant d: with k = ceil(log2 d) and
// m = ceil(2^(30 + k) / d), x / d is x m >> 30 + k (the product's excess, below x 2^k,
// stays below 2^(30 + k)).
struct KvDiv {
    uint32_t m = 1u << 30;
    int shift = 30, d = 1;
    KvDiv() = default;
    explicit KvDiv(int by) : d(by) {
        int k = 0;
        while ((1ll << k) < by) k++;
        shift = 30 + k;
        m = (uint32_t)(((1ull << shift) + (uint64_t)by - 1) / (uint64_t)by);
    }
};

struct KvDev {
    uint8_t* pool = nullptr;
    float* kscale = nullptr;   // [block * H + head]
    float* vscale = nullptr;
    int* positions = nullptr;  // [(block * H + head) * B + slot]
    float* weights = nullptr;
    int* table = nullptr;      // [seq * W + i]: the block of the sequence's slots i * B ..
    int H = 0, D = 0, Dp = 0, B = 0, W = 0;
    int shift = 0;             // log2 B
    int code = KV_INT8;
    KvDiv by_heads;            // H
};

// n sequences of one launch.  Workgroups unit0[i] .. unit0[i + 1] - 1 (times what
// the kernel multiplies them by) belong to sequence i.
struct KvBatch {
    int n = 0;
    int seq[KV_BATCH];
    int len[KV_BATCH];    // slots in use (append: before it)
    int tok0[KV_BATCH];   // row of its first token in the call's tensors
    int count[KV_BATCH];  // its tokens
    int aux[KV_BATCH];    // append: position of the first token; read: first slot;
                          // evict: sequence that receives the result; attend: see there
    int splits[KV_BATCH]; // attend: parts that the tiles of its rows go to, of per[i] tiles;
                          // append: the one block it touches, or -1 (see the table)
    int per[KV_BATCH];
    int unit0[KV_BATCH + 1];
};

struct KvTensor {
    const void* p = nullptr;
    int64_t st = 0, sh = 0, sd = 0;  // strides in elements
    int type = KV_F32;
    bool vec = false;  // 8 dims of a row are one aligned 16- or 32-byte piece
};

// Bytes of a tile's key (or value) half.
__host__ __device__ inline int kv_half(int Dp) { return KV_TILE * Dp; }

#ifdef __HIPCC__
__device__ inline int kv_div(int x, const KvDiv& by) { return (int)((uint64_t)(uint32_t)x * by.m >> by.shift); }
__device__ inline int kv_mod(int x, const KvDiv& by) { return x - kv_div(x, by) * by.d; }
__device__ inline size_t kv_tile_offset(const KvDev& c, int block, int head, int tile) {
    const size_t part = (size_t)block * c.H + head;
    return (part * (size_t)(c.B / KV_TILE) + tile) * (size_t)(2 * kv_half(c.Dp));
}
// Byte of (slot r, dims 8 m .. 8 m + 7) in the key half.
__device__ inline int kv_key_byte(int r, int m, int S) {
    const int o = (r >> 4) * S + (m >> 2);
    return (o >> 1) * 1024 + ((m & 3) * 16 + (r & 15)) * 16 + (o & 1) * 8;
}
// Byte of (slot r, dim d) in the value half.
__device__ inline int kv_value_byte(int r, int d) {
    const int i = d >> 4;
    const int lane = ((r & 15) >> 2) * 16 + (d & 15);
    return (i >> 1) * 1024 + lane * 16 + (i & 1) * 8 + (r >> 4) * 4 + (r & 3);
}
// The batch entry of a workgroup: how many unit0 are not above it, less one.
__device__ inline int kv_find(const KvBatch& b, int unit) {
    if (b.n == 1) return 0;
    const int lane = threadIdx.x & 63;
    const int e0 = lane < b.n && b.unit0[lane] <= unit;
    const int e1 = lane + 64 < b.n && b.unit0[lane + 64] <= unit;
    return __builtin_amdgcn_readfirstlane(__popcll(__ballot(e0)) + __popcll(__ballot(e1)) - 1);
}
#endif

// Entries of the block table: runs of consecutive blocks.
struct KvRuns {
    static constexpr int MAX = 200;
    int n = 0;
    size_t at[MAX];
    int block[MAX], count[MAX];
};
void launch_kv_table(int* table, const KvRuns& r, hipStream_t s);

void launch_kv_append(const KvDev& c, const KvBatch& b, const KvTensor& k, const KvTensor& v,
                      const int* positions, const float* weights, hipStream_t s);

struct KvReadOut {
    void *k = nullptr, *v = nullptr;
    int* positions = nullptr;
    float* weights = nullptr;
    int type = KV_F32;
    bool vec = false;  // 8 dims of an output row are one aligned piece
};
// unit0 counts groups of KV_READ slots, from that of the first slot on.
constexpr int KV_READ = 128;
void launch_kv_read(const KvDev& c, const KvBatch& b, const KvReadOut& o, hipStream_t s);

// Eviction of the batch's sequences (count: the slots that stay, len above it).
struct KvEvict {
    int budget = 0, recent = 0, drop = 0;  // drop: rows of a sequence's dropped arrays (0: none)
    int* kept = nullptr;     // [n, H, budget] slots that stay, ascending
    int* gone = nullptr;     // [n, H, slots] a slot's row among those that leave, or -1; null without them
    int slots = 0;           // of the longest sequence
    bool vec = false;        // 8 dims of a dropped row are one aligned piece
    uint32_t* hist = nullptr;  // selection from long sequences (kv_select_space)
    uint2* counts = nullptr;
    const int* dst = nullptr;  // [seq * W + i] table with the new blocks of aux[i]
    int* dpos = nullptr;     // the caller's arrays, [n, drop, H] and [n, drop, H, D]
    float *dk = nullptr, *dv = nullptr;
};
// Elements of KvEvict's hist and counts for n sequences, the longest of them so long.
struct KvSelectSpace {
    size_t hist = 0, counts = 0;
};
KvSelectSpace kv_select_space(const KvDev& c, int n, int longest);
void launch_kv_evict(const KvDev& c, const KvBatch& b, const KvEvict& e, hipStream_t s);

struct KvAttend {
    KvTensor q;
    int G = 1;              // query heads per key/value head
    KvDiv by_group;         // G
    float scale2 = 0.f;     // scale * log2(e)
    int causal = 1, window = 0;
    const uint8_t* mask = nullptr;
    int64_t mask_st = 0, mask_ss = 0;
    int track = 0;
    float decay = 0.f;
    void* out = nullptr;       // [tokens, H * G, D] in q's type
    bool vec_out = false;      // 4 dims of its rows are one aligned piece
    float* lse = nullptr;      // [tokens, H * G]
    // tracked: base-2 lse of the rows, [sequence][head][row] (-inf: sees nothing)
    float* lse2 = nullptr;
    // tracked chunks: the query operands of 16-row tiles, [tile of the sequences before and of
    // the heads before][part][32-dim step][lane], and the factor of each row, as lse2
    uint4* qop = nullptr;
    float* qs = nullptr;
    float* wpart = nullptr;    // sums of `chunks` chunks of chunk_rows rows
    int chunks = 1, chunk_rows = 0;
    float* part_o = nullptr;   // split attention: partial rows [workgroup, rows, Dp]
    float2* part_ml = nullptr; // and their (max, sum), base 2
    float* part_s = nullptr;   // and the power of 2 that their sums are in
    float* scores = nullptr;   // tracked steps: base-2 scores [row, tile, 32] of each (sequence, head)
    int by_rows = 0;           // waves of a workgroup take different rows (else different tiles)
};
// 16-row tiles of a wave of the many-row kernel, by what its registers hold: Dp / 4
// accumulators and Dp * parts / 8 query operands for each (128 dims: 1431 us with two, 2311
// with four; in float32 924 with two, 1029 with one; 192 dims: 1087 with one, 2603 with two).
// 256 dims: one workgroup to a compute unit, by its LDS, with all the registers.
constexpr int kv_chunk_nc(int Dp, int parts) { return Dp * parts <= 64 ? 4 : Dp <= 128 || Dp * parts == 256 ? 2 : 1; }
// Rows that one workgroup takes.
inline int kv_attend_rows(const KvAttend& a, int Dp) {
    return a.by_rows ? 64 * kv_chunk_nc(Dp, a.q.type == KV_F32 ? 2 : 1) : 16;
}
// unit0 counts row tiles times splits of the sequences (of one head).
void launch_kv_attend(const KvDev& c, const KvBatch& b, const KvAttend& a, hipStream_t s);
// Slots of a workgroup that makes weights of kept scores, and of one that goes over the keys.
constexpr int KV_SCORE_SLOTS = 1024, KV_WEIGHT_SLOTS = 128;
// unit0 counts these.  aux: with scores the tiles of the score rows of the sequences
// before (of one head), without them the 16-row tiles of the sequences before.
void launch_kv_weights(const KvDev& c, const KvBatch& b, const KvAttend& a, hipStream_t s);

}  // namespace vgpu
