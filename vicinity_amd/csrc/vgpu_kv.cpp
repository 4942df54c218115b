// The attention memory's host side: argument checks, blocks and lengths, and the
// launches of one call.
#include <algorithm>
#include <climits>
#include <cmath>
#include <functional>

#include "vgpu_runtime.h"

namespace vgpu {

namespace {

// The message is put together only when the check fails.
#define need(ok, msg, ...)                                      \
    do {                                                        \
        if (!(ok)) refuse(msg, ##__VA_ARGS__);                  \
    } while (0)

[[noreturn]] void refuse(const std::string& msg, int code = VGPU_ERR_INVALID_PARAMETER) { throw Error(code, msg); }

size_t item_size(int type) { return type == KV_F32 ? 4 : 2; }

// Workgroups that a step is cut into where one round suffices: three for each of the 256
// compute units, which hold as many up to 128 dims; above, two fit, and the third ones follow.
constexpr int64_t kStepWorkgroups = 768;
// Workgroups of a call with many rows, two to a compute unit (at 256 dims one fits): with
// fewer, the tiles are split too, which costs a partial result for every row and split.
constexpr int64_t kChunkWorkgroups = 512;
// Workgroups of the second pass that makes weights: twelve to a compute unit, for its rows
// differ in length (8192: no faster).
constexpr int64_t kWeightWorkgroups = 3072;
// Workgroups of one launch: its threads, 256 to a workgroup, are counted in 32 bits.
constexpr int64_t kMaxWorkgroups = (1 << 24) - 1;
// Bytes of partial results of one launch.
constexpr int64_t kPartBytes = (int64_t)256 << 20;
// Calls of at most this many rows per head keep their scores for the weights; with more a
// second pass over the keys is cheaper (16 sequences of 4096, 8 x 128: 32 rows 70 and 93 us,
// 48 rows 91 and 96, 64 rows 116 and 102; measured in bfloat16 there, and taken for all).
constexpr int64_t kScoreRows = 48;
// The kernel of many rows takes over where its workgroups are filled to three quarters and
// have this many 32-slot tiles to do in all (16 sequences of 4096, 8 x 128, 128 rows: 65 us
// against 77 by row tiles of 16, 96 rows 67 and 58, 256 rows 106 and 139; 4 sequences of 1024,
// 256 rows: 29 and 16 us; measured in bfloat16 there, and taken for all).
constexpr int64_t kChunkTiles = 4096;

// Entries of one fork's row of the table that go as kernel arguments; more are copied on the GPU.
constexpr size_t kRowRuns = 64;

// Sequences that share so many slots are taken over them together.
constexpr int64_t kSharedSlots = 256;
// ... where that leaves so many bytes of a call unread, which the join of the parts costs: with
// sequences of more than 8 rows, and without (32 query heads on 8 of 128: 4 sequences of 512 slots,
// 3.1 MB, 15 us against 13; 8 query heads to one, 5 of 1312, 10.7 MB, 14.8 and 13.4; 8 or 4 of them,
// 8 of 1000 or 4 of 2048, 14 and 12.6 MB, alike; 4 x 4 of 1000, 25 MB, 15.8 and 17.2; 128 rows each:
// 4 sequences of 1376, 8.5 MB, 21.9 and 27.7).
constexpr int64_t kSharedBytes = (int64_t)8 << 20, kFewBytes = (int64_t)12 << 20;
// Sequences of at most 8 rows that need no splits when each is taken by itself, and then no join,
// have to share so many slots on average for each launch of some 96 of them (8 x 8 sequences of 32
// query heads on 8 of 128: 512 slots 16.6 us together and 13.7 apart, 800 17.5 and 16.6, 1000 17.8
// and 18.9, 1500 20.5 and 23.9; 32 x 4: 512 40 and 26, 1000 44 and 35, 2000 54 and 58); fewer where
// their workgroups are more than 512, and have more than one round to do (64 of 32 heads of 64 in
// float32: 512 slots 25 and 24, 1000 28 and 35; 65 of 32 of 192: 896 slots 44 and 81).
constexpr int64_t kCrowdedSlots = 1024, kCrowdedUnits = 512, kLaunchSeqs = 96;
// The kernel of many rows takes over shared slots from so many tiles of 16 rows on, from twice as
// many where its workgroups have 256 rows; they are a launch apart from the own slots then, with
// partial rows four times as many (8 heads, a token each, own slots 300; by 16 rows and by many:
// 128 dims in bfloat16, 32768 tiles 36 us and 50, 65536 67 and 59, 98304 82 and 67, 262144 216 and
// 109; 192 dims, 32768 47 and 57, 65536 81 and 77, 262144 287 and 176; 64 dims in float32, 24576 27
// and 40, 65536 56 and 51; 64 dims in bfloat16, 256 rows, 65536 51 and 54, 98304 59 and 64, 262144
// 163 and 91).
constexpr int64_t kSharedTiles = 65536;
// Tiles of a workgroup over shared slots, at least (32 beams of 8 prompts of 1000 slots, 8 x 4 x
// 128: with 2, 4, 8, 16 and 24 tiles 31, 30, 29, 30 and 31 us; 5 x 8 rows over 20000 slots of two
// heads 23, 23, 21, 19 and 20; more rows or slots: no difference).
constexpr int64_t kLeastTiles = 8;
// A sequence of more rows than this shares no tile of 16 rows with two others.  Where the tiles of
// such sequences are this many workgroups, taken apart, as if nothing were shared, they find in the
// caches what they read in common, and nobody joins their parts (8 x 128 in bfloat16: 32 sequences of
// 20 rows over 2048 shared slots 27 us apart, 32 together; 8 of 56 rows, 256 workgroups, 30 and 24).
constexpr int64_t kTileRows = 8;
constexpr int64_t kApartWorkgroups = kStepWorkgroups / 2;
// Rows that the kernel of many would not take one sequence at a time it takes together over so many
// shared slots, which pay for their parts (8 x 128: 32 of 40 rows over 8192 slots 101 us apart, 79
// together, 32 of 32 over 6560 a fifth faster together; 52 of 48 over 1792 49 and 69; 64 dims, 63 of
// 16 over 3328 86 and 112).
constexpr int64_t kLongSlots = 6144, kFullerSlots = 2560;  // (the second: see part_groups)
// Rows of the kernel of many have so many tiles of 16 to do where they leave sequences of fewer rows,
// which takes a launch more (28 sequences of which one has 684 rows over 1954 slots of 8 x 96, 34000
// tiles: 28 us together, 49 not; four of which one has 272 over 4672 of 32 x 64, 80000: 52 and 98; one
// of 8192 over 18400 of 8 x 128 beside 16 of 4, 2.4 million: 980 and 600).
constexpr int64_t kManyTiles = 131072;
// Levels of branches that are looked at for the best groups.
constexpr int kSharedDepth = 4;

// Rows that share slots: does the kernel of many rows suit them?  Not at 256 dims, nor at 128 in
// float32 (244 rows over 16384 slots of 8 heads: 95 us by 16 rows and 141 by many, 76 and 132; over
// 65536 slots the second 246 and 385): two operands' tiles and where each row's sequence lies are
// more than the registers hold.
bool many_shared(const KvDev& dev, int type, int64_t rows, int64_t tiles) {
    const int parts = type == KV_F32 ? 2 : 1;
    const int64_t wg = 64 * kv_chunk_nc(dev.Dp, parts);
    return kv_shared_many(dev.Dp, parts) && rows > wg * 3 / 4 && tiles >= (wg > 128 ? 2 : 1) * kSharedTiles;
}

// The row tiles of one launch's sequences, and the tiles that each goes over.
struct KvPlan {
    int n = 0, heads = 1;
    int64_t tiles[KV_BATCH], row_units[KV_BATCH];
    int64_t units = 0, work = 0;           // row tiles of all heads; their tiles
    int64_t groups = 0, split_units = 0;   // workgroups; those that leave partial results

    // A sequence of len slots whose last `count` tokens have G rows each, `rows` to a workgroup.
    void add(int64_t len, int64_t count, int64_t G, int64_t rows, bool causal, int64_t window) {
        row_units[n] = (count * G + rows - 1) / rows;
        units += row_units[n] * heads;
        tiles[n] = (len + KV_TILE - 1) / KV_TILE;
        if (window && causal) tiles[n] = std::min(tiles[n], (window + rows / G + 2 * KV_TILE) / KV_TILE + 1);
        // (the first tokens of a chunk see less than the last)
        const int64_t seen = causal && !window ? std::max<int64_t>(2 * len - count, 0) : 2 * KV_TILE * tiles[n];
        work += row_units[n] * heads * ((seen + 2 * KV_TILE - 1) / (2 * KV_TILE));
        n++;
    }

    // An entry of shared slots: count rows over so many tiles.
    void add_entry(int64_t count, int64_t over, int64_t rows) {
        row_units[n] = (count + rows - 1) / rows;
        units += row_units[n] * heads;
        tiles[n] = over;
        work += row_units[n] * heads * over;
        n++;
    }

    // Splits of at most `each` tiles: b's splits, per and unit0.  True if none is split.
    bool cut(KvBatch& b, int64_t each) {
        groups = split_units = 0;
        bool one = true;
        b.unit0[0] = 0;
        for (int j = 0; j < n; j++) {
            const int64_t splits = std::max<int64_t>((tiles[j] + each - 1) / each, 1);
            b.splits[j] = (int)splits;
            b.per[j] = (int)std::max<int64_t>((tiles[j] + splits - 1) / splits, 1);
            b.unit0[j + 1] = b.unit0[j] + (int)(row_units[j] * splits);
            groups += row_units[j] * splits * heads;
            one = one && splits == 1;
            if (splits > 1) split_units += row_units[j] * splits * heads;
        }
        return one;
    }

    // The same for entries of shared slots, which are whole rectangles: the least share that
    // keeps all workgroups on the card at once.
    void split_entries(KvBatch& b, bool by_rows, int64_t part_units) {
        const int64_t most = std::min(by_rows ? kChunkWorkgroups : kStepWorkgroups, part_units);
        int64_t lo = kLeastTiles, hi = std::max(lo, tiles_most());
        while (lo < hi) {
            const int64_t mid = (lo + hi) / 2;
            if (cut(b, mid), groups <= most) hi = mid;
            else lo = mid + 1;
        }
        // Some prefixes far above the others: in several rounds, as below (8 x 9 sequences of 4 rows over
        // 299 to 9339 shared slots of 8 x 128: 84 us in one round, 38 so; over 875 to 3500, where the
        // largest part is less than four shares, 22 and 27).
        const int64_t share = std::max<int64_t>((work + most - 1) / most, kLeastTiles);
        if (lo > 4 * share) lo = 2 * share;
        while (cut(b, lo), groups > part_units && lo < tiles_most()) lo += lo / 8 + 1;
    }
    int64_t tiles_most() const {
        int64_t most = 0;
        for (int j = 0; j < n; j++) most = std::max(most, tiles[j]);
        return most;
    }

    // As few tiles to a workgroup as keep all of them on the card at once; at most
    // part_units workgroups have room for partial results.
    void split(KvBatch& b, bool by_rows, int64_t part_units) {
        const int64_t target = by_rows ? kChunkWorkgroups : kStepWorkgroups;
        const int64_t share = std::max<int64_t>((work + target - 1) / target, by_rows ? 16 : 8);
        if (by_rows) {
            // whole unless that would leave one workgroup at work alone
            for (int64_t each = units >= 4 * target ? INT_MAX : share;; each += each / 8 + 1)
                if (cut(b, each + each / 4) || groups <= part_units) return;
        }
        for (int64_t each = share; each <= 2 * share; each += each / 8 + 1)
            if (cut(b, each) || groups <= std::min(target + target / 8, part_units)) return;
        // Many row tiles, or a few sequences far above the others, do not go in one round: no
        // workgroup takes more than its share of the work, in several (8 x 128; one sequence of
        // 131072 among 127 of 100: 65 us, whole 1031; 128 sequences of 512 to 8191: 140 and
        // 157; pieces of half a share 67 and 142).
        for (int64_t each = share;; each += each / 8 + 1)
            if (cut(b, each) || groups <= part_units) return;
    }
};

// A workspace that grows in large steps, where there is memory for them.
template <typename T>
void grow(DevBuf<T>& b, size_t count) {
    if (count <= b.n) return;
    const size_t step = b.n + b.n / 2;
    if (step > count) try {
        b.reserve(step);
        return;
    } catch (const Error& e) {
        if (e.code != VGPU_ERR_OUT_OF_MEMORY) throw;
    }
    b.reserve(count);
}

}  // namespace

void kv_plan_steps(const int64_t* lens, const int64_t* counts, int n, int heads, int group, int32_t* splits, int32_t* per) {
    KvPlan plan;
    KvBatch b;
    plan.heads = heads;
    for (int i = 0; i < n; i++) plan.add(lens[i], counts[i], group, 16, true, 0);
    plan.split(b, false, kPartBytes / (16 * (KV_MAX_DIM * 4 + 12)));
    for (int i = 0; i < n; i++) splits[i] = b.splits[i], per[i] = b.per[i];
}

KvCache::KvCache(const vgpu_kv_params& p) : params(p) {
    const auto cfg = [](bool ok, const char* msg) { need(ok, msg, VGPU_ERR_INVALID_CONFIG); };
    cfg(p.num_seqs > 0 && p.num_seqs <= (1u << 24), "num_seqs must be in the range 1..=2^24");
    cfg(p.num_heads > 0 && p.num_heads <= 4096, "num_heads must be in the range 1..=4096");
    cfg(p.head_dim > 0 && p.head_dim <= (size_t)KV_MAX_DIM, "head_dim must be in the range 1..=256");
    cfg(p.block_tokens == 32 || p.block_tokens == 64 || p.block_tokens == 128 || p.block_tokens == 256,
        "block_tokens must be 32, 64, 128 or 256");
    cfg(p.code == VGPU_KV_INT8 || p.code == VGPU_KV_FP8, "code must be 0 (int8) or 1 (fp8 e4m3)");
    cfg(p.num_blocks > 0 && p.num_blocks <= (size_t)1 << 30, "num_blocks must be in the range 1..=2^30");
    if (!params.max_blocks || params.max_blocks > p.num_blocks) params.max_blocks = p.num_blocks;
    // slots and score rows of a sequence are 32-bit numbers
    cfg(params.max_blocks <= (size_t)(INT_MAX / 2) / p.block_tokens, "a sequence's slots must stay below 2^30");
    VGPU_HIP(hipGetDevice(&device));
    dev.H = (int)p.num_heads;
    dev.by_heads = KvDiv(dev.H);
    dev.D = (int)p.head_dim;
    // padded dimensions the kernels are compiled for
    dev.Dp = dev.D <= 64 ? 64 : dev.D <= 96 ? 96 : dev.D <= 128 ? 128 : dev.D <= 192 ? 192 : 256;
    dev.B = (int)p.block_tokens;
    dev.shift = __builtin_ctz((unsigned)dev.B);
    dev.W = (int)params.max_blocks;
    dev.code = p.code;
    const size_t parts = p.num_blocks * p.num_heads, slots = parts * p.block_tokens;
    pool.reserve(slots * 2 * dev.Dp);
    kscale.reserve(parts);
    vscale.reserve(parts);
    positions.reserve(slots);
    weights.reserve(slots);
    table.reserve(p.num_seqs * params.max_blocks);
    dev.pool = pool.p, dev.kscale = kscale.p, dev.vscale = vscale.p;
    dev.positions = positions.p, dev.weights = weights.p, dev.table = table.p;
    shared_bytes = kSharedBytes;
    seqs.resize(p.num_seqs);
    seen.assign(p.num_seqs, 0);
    free_blocks.resize(p.num_blocks);
    for (size_t i = 0; i < p.num_blocks; i++) free_blocks[i] = (int)(p.num_blocks - 1 - i);
    holders.assign(p.num_blocks, 0);
}

KvCache::~KvCache() {
    // queued work still reads the buffers
    int cur = device;
    (void)hipGetDevice(&cur);
    if (cur != device) (void)hipSetDevice(device);
    (void)hipDeviceSynchronize();
    if (cur != device) (void)hipSetDevice(cur);
}

size_t KvCache::device_bytes() const {
    return pool.bytes() + kscale.bytes() + vscale.bytes() + weights.bytes() + positions.bytes() + table.bytes() +
           table2.bytes() + w_map.bytes() + w_kept.bytes() + w_gone.bytes() + w_part.bytes() + w_scores.bytes() + w_lse2.bytes() +
           w_ml.bytes() + w_power.bytes() + w_hist.bytes() + w_counts.bytes() + w_qop.bytes() + w_qs.bytes() + w_wpart.bytes();
}

void KvCache::check_call(hipStream_t s) {
    int cur = -1;
    VGPU_HIP(hipGetDevice(&cur));
    need(cur == device, "the cache's device (" + std::to_string(device) + ") must be current, not device " +
                            std::to_string(cur));
    hipStreamCaptureStatus st = hipStreamCaptureStatusNone;
    VGPU_HIP(hipStreamIsCapturing(s, &st));
    need(st == hipStreamCaptureStatusNone, "the cache's lengths cannot follow a captured stream", VGPU_ERR_UNSUPPORTED);
}

static void check_ids(const KvCache& c, std::vector<uint8_t>& seen, const int32_t* ids, size_t n) {
    std::string bad;
    size_t i = 0;
    for (; i < n && bad.empty(); i++) {
        if (ids[i] < 0 || (size_t)ids[i] >= c.seqs.size())
            bad = "sequence " + std::to_string(ids[i]) + " out of range [0, " + std::to_string(c.seqs.size()) + ")";
        else if (seen[ids[i]])
            bad = "sequence " + std::to_string(ids[i]) + " appears twice in the batch";
        else
            seen[ids[i]] = 1;
    }
    for (size_t j = 0; j < i; j++)
        if (ids[j] >= 0 && (size_t)ids[j] < c.seqs.size()) seen[ids[j]] = 0;
    need(bad.empty(), bad);
}

KvTensor KvCache::tensor(const vgpu_tensor3& t, const char* name) const {
    need(t.dtype == VGPU_F32 || t.dtype == VGPU_F16 || t.dtype == VGPU_BF16,
         std::string(name) + ": dtype must be float32, float16 or bfloat16");
    KvTensor x;
    x.p = t.data;
    x.type = t.dtype;
    x.st = t.stride_token, x.sh = t.stride_head, x.sd = t.stride_dim;
    const size_t item = item_size(t.dtype);
    need((uintptr_t)t.data % item == 0, std::string(name) + ": data must be aligned to its dtype");
    // 8 dims as one or two 16-byte loads
    const int64_t unit = 16 / (int64_t)item;
    x.vec = x.sd == 1 && dev.D % 8 == 0 && (uintptr_t)t.data % 16 == 0 && x.st % unit == 0 && x.sh % unit == 0;
    return x;
}

// One more entry of the table.
static void add_run(KvRuns& runs, size_t at, int block, int* tab, hipStream_t s) {
    if (runs.n && runs.at[runs.n - 1] + runs.count[runs.n - 1] == at &&
        runs.block[runs.n - 1] + runs.count[runs.n - 1] == block) {
        runs.count[runs.n - 1]++;
        return;
    }
    if (runs.n == KvRuns::MAX) {
        launch_kv_table(tab, runs, s);
        runs.n = 0;
    }
    runs.at[runs.n] = at, runs.block[runs.n] = block, runs.count[runs.n] = 1;
    runs.n++;
}

// Copies of blocks, gathered into launches.
struct KvCopies {
    const KvDev &from, &to;
    int* map;
    hipStream_t s;
    int64_t most;  // blocks of one launch
    KvMoves m;
    KvCopies(const KvDev& a, const KvDev& b, int* names, hipStream_t stream) : from(a), to(b), map(names), s(stream) {
        most = kMaxWorkgroups / kv_move_pieces(a);
        m.unit0[0] = 0;
    }
    void add(int src, int dst) {
        if (m.unit0[m.n] == most) flush();
        const int i = m.n - 1;
        if (m.n && m.src[i] + m.unit0[i + 1] - m.unit0[i] == src && m.dst[i] + m.unit0[i + 1] - m.unit0[i] == dst) {
            m.unit0[i + 1]++;
        } else {
            if (m.n == KvMoves::MAX) flush();
            m.src[m.n] = src, m.dst[m.n] = dst, m.unit0[m.n + 1] = m.unit0[m.n] + 1;
            m.n++;
        }
    }
    void flush() {
        launch_kv_moves(from, to, m, map, s);
        m.n = 0;
    }
};

int KvCache::take_block() {
    const int block = free_blocks.back();
    free_blocks.pop_back();
    holders[block] = 1;
    return block;
}

void KvCache::let_go(int block) {
    if (--holders[block] == 0) free_blocks.push_back(block);
    else shared_holds--;
}

void KvCache::take_blocks(std::vector<int>& out, size_t count, size_t row, int* tab, KvRuns& runs, hipStream_t s) {
    for (size_t j = 0; j < count; j++) {
        const int block = take_block();
        add_run(runs, row * (size_t)dev.W + out.size(), block, tab, s);
        out.push_back(block);
    }
}

void KvCache::release_blocks(std::vector<int>& blocks, size_t keep) {
    while (blocks.size() > keep) {
        let_go(blocks.back());
        blocks.pop_back();
    }
}

size_t KvCache::shared_blocks(const int32_t* ids, const int64_t* first, size_t n) {
    if (!shared_holds) return 0;
    // as own_blocks will find them: of the batch's holders of a block, the last one keeps it
    size_t count = 0;
    for (size_t i = 0; i < n; i++) {
        const std::vector<int>& b = seqs[ids[i]].blocks;
        for (size_t j = (size_t)first[i]; j < b.size(); j++)
            if (holders[b[j]] > 1) holders[b[j]]--, count++;
            else holders[b[j]] = -holders[b[j]];  // kept
    }
    // and back
    for (size_t i = n; i-- > 0;) {
        const std::vector<int>& b = seqs[ids[i]].blocks;
        for (size_t j = (size_t)first[i]; j < b.size(); j++)
            if (holders[b[j]] < 0) holders[b[j]] = -holders[b[j]];
            else holders[b[j]]++;
    }
    return count;
}

void KvCache::own_blocks(const int32_t* ids, const int64_t* first, size_t n, KvRuns& runs, hipStream_t s) {
    if (!shared_holds) return;
    KvCopies copies(dev, dev, nullptr, s);
    for (size_t i = 0; i < n; i++) {
        std::vector<int>& b = seqs[ids[i]].blocks;
        for (size_t j = (size_t)first[i]; j < b.size(); j++) {
            if (holders[b[j]] <= 1) continue;
            const int block = take_block();
            copies.add(b[j], block);
            add_run(runs, (size_t)ids[i] * (size_t)dev.W + j, block, table.p, s);
            let_go(b[j]);
            b[j] = block;
        }
    }
    copies.flush();
}

void KvCache::append(const int32_t* ids, const int64_t* counts, size_t n, const vgpu_tensor3& k, const vgpu_tensor3& v,
                     const int32_t* pos, const float* wts, hipStream_t s) {
    check_call(s);
    check_ids(*this, seen, ids, n);
    need(k.dtype == v.dtype, "k and v must have the same dtype");
    const KvTensor kt = tensor(k, "k"), vt = tensor(v, "v");
    int64_t tokens = 0;
    size_t want = 0;
    std::vector<int64_t> begun(n);  // the block that the first new token enters
    for (size_t i = 0; i < n; i++) {
        const Seq& q = seqs[ids[i]];
        begun[i] = counts[i] ? q.len >> dev.shift : (int64_t)q.blocks.size();
        need(counts[i] >= 0 && counts[i] <= INT_MAX / 2, "counts must not be negative, nor above 2^30");
        tokens += counts[i];
        need(tokens <= INT_MAX / 2, "more than 2^30 tokens in one call");
        const size_t total = blocks_of(q.len + counts[i]);
        need(total <= (size_t)dev.W, "sequence " + std::to_string(ids[i]) + " would need " + std::to_string(total) +
                                         " blocks, more than max_blocks (" + std::to_string(dev.W) + ")");
        need(pos || q.next + counts[i] <= INT_MAX, "positions must stay below 2^31");
        need((int64_t)(total - (q.len >> dev.shift)) * dev.H * 2 <= kMaxWorkgroups,
             "too many tokens of one sequence in one call");
        want += total - q.blocks.size();
    }
    need(!tokens || (k.data && v.data), "null argument");
    const size_t shared = shared_blocks(ids, begun.data(), n);
    want += shared;
    need(want <= free_blocks.size(),
         "the cache needs " + std::to_string(want) + " more blocks and has " + std::to_string(free_blocks.size()),
         VGPU_ERR_OUT_OF_MEMORY);
    for (size_t i = 0; i < n; i++) seqs[ids[i]].blocks.reserve(blocks_of(seqs[ids[i]].len + counts[i]));
    KvRuns runs;
    // Begun blocks that others hold too: the append itself copies them, but those that another
    // sequence of the call goes on in.
    std::vector<int> source(n, -1), kept;
    if (shared) {
        kept.reserve(n);
        for (size_t i = 0; i < n; i++) {
            Seq& q = seqs[ids[i]];
            if ((size_t)begun[i] >= q.blocks.size()) continue;
            int& block = q.blocks[(size_t)begun[i]];
            if (holders[block] > 1) {
                source[i] = block;
                block = take_block();
                let_go(source[i]);
            } else {
                kept.push_back(block);
            }
        }
        std::sort(kept.begin(), kept.end());
        KvCopies copies(dev, dev, nullptr, s);
        for (size_t i = 0; i < n; i++) {
            if (source[i] < 0) continue;
            const Seq& q = seqs[ids[i]];
            const int block = q.blocks[(size_t)begun[i]];
            const bool one = q.len % dev.B + counts[i] <= dev.B;  // the append writes the table too
            if (std::binary_search(kept.begin(), kept.end(), source[i])) {
                copies.add(source[i], block);
                add_run(runs, (size_t)ids[i] * (size_t)dev.W + (size_t)begun[i], block, table.p, s);
                source[i] = -1;
            } else if (!one) {
                add_run(runs, (size_t)ids[i] * (size_t)dev.W + (size_t)begun[i], block, table.p, s);
            }
        }
        copies.flush();
    }
    for (size_t i = 0; i < n; i++) {
        Seq& q = seqs[ids[i]];
        const size_t more = blocks_of(q.len + counts[i]) - q.blocks.size();
        // one block touched: the append itself writes the table
        if (more == 1 && q.len % dev.B == 0 && counts[i] <= dev.B) {
            q.blocks.push_back(take_block());
        } else {
            take_blocks(q.blocks, more, ids[i], table.p, runs, s);
        }
    }
    launch_kv_table(table.p, runs, s);
    int64_t tok = 0;
    for (size_t i = 0; i < n;) {
        KvBatch b;
        b.n = 0;
        b.unit0[0] = 0;
        for (; i < n && b.n < KV_BATCH; i++) {
            Seq& q = seqs[ids[i]];
            const int j = b.n;
            // blocks that the new tokens enter
            const int64_t first = q.len >> dev.shift;
            const int64_t touched = counts[i] ? (int64_t)blocks_of(q.len + counts[i]) - first : 0;
            if ((b.unit0[j] + touched) * dev.H * 2 > kMaxWorkgroups) break;
            b.seq[j] = ids[i];
            b.len[j] = (int)q.len;
            b.tok0[j] = (int)tok;
            b.count[j] = (int)counts[i];
            b.aux[j] = (int)q.next;
            b.splits[j] = touched == 1 ? q.blocks[first] : -1;
            b.per[j] = source[i];
            b.unit0[j + 1] = b.unit0[j] + (int)touched;
            b.n++;
            tok += counts[i];
            q.len += counts[i];
            q.next += counts[i];
        }
        launch_kv_append(dev, b, kt, vt, pos, wts, s);
    }
    VGPU_HIP(hipGetLastError());
}

void KvCache::read(const int32_t* ids, const int64_t* first, const int64_t* counts, size_t n, int dtype, void* k,
                   void* v, int32_t* pos, float* wts, hipStream_t s) {
    check_call(s);
    check_ids(*this, seen, ids, n);
    need(dtype == VGPU_F32 || dtype == VGPU_F16 || dtype == VGPU_BF16, "dtype must be float32, float16 or bfloat16");
    int64_t tok = 0;
    const auto count_of = [&](size_t i) { return counts ? counts[i] : seqs[ids[i]].len - first[i]; };
    for (size_t i = 0; i < n; i++) {
        const int64_t count = count_of(i);
        need(first[i] >= 0 && count >= 0 && first[i] <= seqs[ids[i]].len && count <= seqs[ids[i]].len - first[i],
             "slots outside sequence " + std::to_string(ids[i]) + " of length " + std::to_string(seqs[ids[i]].len));
        tok += count;
        need(tok <= INT_MAX / 2, "more than 2^30 tokens in one call");
        need((count / KV_READ + 2) * dev.H <= kMaxWorkgroups, "too many slots of one sequence in one call");
    }
    KvReadOut o;
    o.k = k, o.v = v, o.positions = pos, o.weights = wts, o.type = dtype;
    o.vec = dev.D % 8 == 0 && ((uintptr_t)k | (uintptr_t)v) % 16 == 0;
    tok = 0;
    for (size_t i = 0; i < n;) {
        KvBatch b;
        b.n = 0;
        b.unit0[0] = 0;
        for (; i < n && b.n < KV_BATCH; i++) {
            const int j = b.n;
            const int64_t count = count_of(i), last = first[i] + count;
            const int64_t groups = count ? (last + KV_READ - 1) / KV_READ - first[i] / KV_READ : 0;
            if ((b.unit0[j] + groups) * dev.H > kMaxWorkgroups) break;
            b.seq[j] = ids[i];
            b.len[j] = (int)seqs[ids[i]].len;
            b.tok0[j] = (int)tok;
            b.count[j] = (int)count;
            b.aux[j] = (int)first[i];
            b.unit0[j + 1] = b.unit0[j] + (int)groups;
            b.n++;
            tok += count;
        }
        if (k || v || pos || wts) launch_kv_read(dev, b, o, s);
    }
    VGPU_HIP(hipGetLastError());
}

void KvCache::truncate(const int32_t* ids, const int64_t* lengths, size_t n) {
    check_ids(*this, seen, ids, n);
    for (size_t i = 0; i < n; i++)
        need(lengths[i] >= 0 && lengths[i] <= seqs[ids[i]].len,
             "length " + std::to_string(lengths[i]) + " outside sequence " + std::to_string(ids[i]) + " of length " +
                 std::to_string(seqs[ids[i]].len));
    for (size_t i = 0; i < n; i++) {
        Seq& q = seqs[ids[i]];
        q.next = lengths[i] ? q.next - (q.len - lengths[i]) : 0;
        q.len = lengths[i];
        release_blocks(q.blocks, blocks_of(q.len));
    }
}

void KvCache::fork(const int32_t* ids, const int32_t* into, const int64_t* lengths, size_t n, bool copy, hipStream_t s) {
    check_call(s);
    check_ids(*this, seen, into, n);
    size_t want = 0;
    const auto slots = [&](size_t i) { return lengths ? lengths[i] : seqs[ids[i]].len; };
    for (size_t i = 0; i < n; i++) {
        need(ids[i] >= 0 && (size_t)ids[i] < seqs.size(),
             "sequence " + std::to_string(ids[i]) + " out of range [0, " + std::to_string(seqs.size()) + ")");
        need(slots(i) >= 0 && slots(i) <= seqs[ids[i]].len,
             "length " + std::to_string(slots(i)) + " outside sequence " + std::to_string(ids[i]) + " of length " +
                 std::to_string(seqs[ids[i]].len));
        if (copy) want += blocks_of(slots(i));
    }
    need(want <= free_blocks.size(),
         "the copies need " + std::to_string(want) + " free blocks, the cache has " + std::to_string(free_blocks.size()),
         VGPU_ERR_OUT_OF_MEMORY);
    // The table rows to be written: by runs where few entries differ, else row by row, through
    // the second table where one row is both read and written.
    std::vector<Fork>& next = forks;
    if (next.size() < n) next.resize(n);
    bool rows = false, crossed = false;
    for (size_t i = 0; i < n; i++) {
        const Seq& from = seqs[ids[i]];
        const std::vector<int>& old = seqs[into[i]].blocks;
        Fork& x = next[i];
        x.common = 0, x.row = false;
        x.q.len = slots(i);
        // (as truncate leaves it; whole, also where nothing is left of it, it goes on counting)
        x.q.next = x.q.len == from.len ? from.next : x.q.len ? from.next - (from.len - x.q.len) : 0;
        const size_t count = blocks_of(x.q.len);
        if (copy) {
            x.q.blocks.clear();
            x.q.blocks.reserve(count);
            continue;
        }
        x.q.blocks.assign(from.blocks.begin(), from.blocks.begin() + (ptrdiff_t)count);
        // where both hold a block they hold all before it
        size_t lo = 0, hi = std::min(count, old.size());
        while (lo < hi) {
            const size_t mid = (lo + hi) / 2;
            if (old[mid] == from.blocks[mid]) lo = mid + 1;
            else hi = mid;
        }
        x.common = lo;
        x.row = count - lo > kRowRuns;
        rows = rows || x.row;
    }
    if (rows) {
        for (size_t i = 0; i < n; i++) seen[into[i]] = 1;
        for (size_t i = 0; i < n; i++) crossed = crossed || (next[i].row && seen[ids[i]] && ids[i] != into[i]);
        for (size_t i = 0; i < n; i++) seen[into[i]] = 0;
        if (crossed) table2.reserve(table.n);
    }
    const auto copy_rows = [&](const int* from, int* to, bool back) {
        KvRows r;
        for (size_t i = 0; i < n; i++) {
            if (!next[i].row) continue;
            if (r.n == KV_BATCH) {
                launch_kv_rows(dev, from, to, r, s);
                r.n = 0;
            }
            r.from[r.n] = back ? into[i] : ids[i], r.to[r.n] = into[i];
            r.first[r.n] = (int)next[i].common, r.end[r.n] = (int)next[i].q.blocks.size();
            r.n++;
        }
        launch_kv_rows(dev, from, to, r, s);
    };
    if (rows) copy_rows(table.p, crossed ? table2.p : table.p, false);
    if (crossed) copy_rows(table2.p, table.p, true);
    KvRuns runs;
    if (copy) {
        KvCopies copies(dev, dev, nullptr, s);
        for (size_t i = 0; i < n; i++) {
            const size_t count = blocks_of(next[i].q.len);
            take_blocks(next[i].q.blocks, count, into[i], table.p, runs, s);
            for (size_t j = 0; j < count; j++) copies.add(seqs[ids[i]].blocks[j], next[i].q.blocks[j]);
        }
        copies.flush();
    } else {
        for (size_t i = 0; i < n; i++) {
            const std::vector<int>& b = next[i].q.blocks;
            for (size_t j = next[i].common; j < b.size(); j++) {
                holders[b[j]]++, shared_holds++;
                if (!next[i].row) add_run(runs, (size_t)into[i] * (size_t)dev.W + j, b[j], table.p, s);
            }
        }
    }
    launch_kv_table(table.p, runs, s);
    // what the sequences held, beyond what they keep
    for (size_t i = 0; i < n; i++) {
        Seq& q = seqs[into[i]];
        release_blocks(q.blocks, next[i].common);
        std::swap(q, next[i].q);
    }
    VGPU_HIP(hipGetLastError());
}

size_t KvCache::compact(size_t num_blocks, hipStream_t s) {
    check_call(s);
    const size_t old_blocks = params.num_blocks, used = old_blocks - free_blocks.size();
    if (!num_blocks) num_blocks = old_blocks;
    need(num_blocks <= (size_t)1 << 30, "num_blocks must be in the range 1..=2^30");
    need(num_blocks >= used, "the cache holds " + std::to_string(used) + " blocks, more than num_blocks (" +
                                 std::to_string(num_blocks) + ")");
    const bool other = num_blocks != old_blocks;
    // old numbers of the blocks 0 .. used - 1, and the new number of each old one
    std::vector<int> to(old_blocks, -1), from(used, -1);
    size_t moved = 0;
    if (other) {  // in the order of the sequences
        for (const Seq& q : seqs)
            for (int b : q.blocks)
                if (to[b] < 0) to[b] = (int)moved, from[moved++] = b;
    } else {  // those behind fill the gaps
        size_t gap = 0;
        for (size_t b = used; b < old_blocks; b++) {
            if (!holders[b]) continue;
            while (holders[gap]) gap++;
            to[b] = (int)gap, from[gap++] = (int)b, moved++;
        }
        if (!moved) return 0;
    }
    std::vector<int> fresh_free, fresh_holders(num_blocks, 0);
    fresh_free.reserve(num_blocks);
    DevBuf<uint8_t> new_pool;
    DevBuf<float> new_k, new_v, new_w;
    DevBuf<int> new_pos;
    KvDev now = dev;
    if (other) {
        const size_t parts = num_blocks * params.num_heads, count = parts * params.block_tokens;
        new_pool.reserve(count * 2 * dev.Dp);
        new_k.reserve(parts), new_v.reserve(parts);
        new_pos.reserve(count), new_w.reserve(count);
        now.pool = new_pool.p, now.kscale = new_k.p, now.vscale = new_v.p;
        now.positions = new_pos.p, now.weights = new_w.p;
    }
    w_map.reserve(old_blocks);
    const int above = other ? 0 : (int)used;  // blocks from here on have new numbers
    KvCopies copies(dev, now, w_map.p, s);
    for (size_t b = 0; b < used; b++)
        if (from[b] >= 0) copies.add(from[b], (int)b);
    copies.flush();
    KvRows r;
    for (size_t i = 0; i < seqs.size(); i++) {
        std::vector<int>& b = seqs[i].blocks;
        size_t first = b.size(), end = 0;
        for (size_t j = 0; j < b.size(); j++)
            if (b[j] >= above) first = std::min(first, j), end = j + 1;
        if (first >= end) continue;
        if (r.n == KV_BATCH) {
            launch_kv_rename(dev, r, w_map.p, above, s);
            r.n = 0;
        }
        r.to[r.n] = r.from[r.n] = (int)i, r.first[r.n] = (int)first, r.end[r.n] = (int)end;
        r.n++;
        for (size_t j = first; j < end; j++)
            if (b[j] >= above) b[j] = to[b[j]];
    }
    launch_kv_rename(dev, r, w_map.p, above, s);
    for (size_t b = 0; b < used; b++) fresh_holders[b] = holders[from[b] >= 0 ? (size_t)from[b] : b];
    for (size_t b = num_blocks; b > used; b--) fresh_free.push_back((int)b - 1);
    holders.swap(fresh_holders);
    free_blocks.swap(fresh_free);
    if (other) {
        pool.swap(new_pool), kscale.swap(new_k), vscale.swap(new_v), positions.swap(new_pos), weights.swap(new_w);
        dev = now;
        params.num_blocks = num_blocks;
    }
    VGPU_HIP(hipGetLastError());
    return moved;
}

void KvCache::evict(const int32_t* ids, const int32_t* into, size_t n, size_t budget, size_t recent,
                    size_t num_dropped, int32_t* dpos, float* dk, float* dv, hipStream_t s) {
    check_call(s);
    check_ids(*this, seen, ids, n);
    need(budget <= (size_t)INT_MAX / 2, "budget must not exceed 2^30");
    need(recent <= budget, "recent must not exceed budget");
    const bool drops = dpos || dk || dv;
    need(!drops || num_dropped <= (size_t)INT_MAX / 2, "num_dropped must not exceed 2^30");
    if (into) {
        std::vector<int32_t> both(ids, ids + n);
        both.insert(both.end(), into, into + n);
        check_ids(*this, seen, both.data(), both.size());
        for (size_t i = 0; i < n; i++)
            need(seqs[into[i]].len == 0, "sequence " + std::to_string(into[i]) + " is not empty");
    }
    const auto stays = [&](size_t i) { return std::min<int64_t>(seqs[ids[i]].len, (int64_t)budget); };
    // Does the pool hold the new blocks, given what comes back on the way?
    std::vector<int> gone;  // blocks that the sequences before have let go
    if (!into) {
        size_t all = 0;
        for (size_t i = 0; i < n; i++) all += seqs[ids[i]].blocks.size();
        gone.reserve(all);
    }
    std::string bad;
    int code = VGPU_ERR_INVALID_PARAMETER;
    size_t have = free_blocks.size();
    for (size_t i = 0; i < n && bad.empty(); i++) {
        const Seq& q = seqs[ids[i]];
        if (drops && q.len - stays(i) > (int64_t)num_dropped)
            bad = "num_dropped is below what leaves sequence " + std::to_string(ids[i]);
        if (!into && q.len <= (int64_t)budget) continue;
        const size_t take = blocks_of(stays(i));
        if ((int64_t)take * dev.H * 2 > kMaxWorkgroups) bad = "too many slots of one sequence in one call";
        if (take > have && bad.empty()) {
            bad = "the cut sequences need " + std::to_string(take) + " free blocks and find " + std::to_string(have);
            code = VGPU_ERR_OUT_OF_MEMORY;
        }
        have -= take;
        if (into) continue;
        for (int block : q.blocks) {
            if (--holders[block] == 0) have++;
            gone.push_back(block);
        }
    }
    for (int block : gone) holders[block]++;
    need(bad.empty(), bad, code);
    const int drop = drops ? (int)num_dropped : 0;
    need((int64_t)dev.H * drop <= INT_MAX / KV_BATCH && (int64_t)n * drop <= INT_MAX,
         "too many dropped slots in one call");
    int64_t longest = 0;
    for (size_t i = 0; i < n; i++) longest = std::max(longest, seqs[ids[i]].len);
    // sequences of one launch, which has a grid for the longest of them
    const int64_t grid = (longest / KV_READ + 1) * dev.H;
    need(grid <= kMaxWorkgroups, "too many slots of one sequence in one call");
    const size_t group = std::min<size_t>({n, (size_t)KV_BATCH, (size_t)(kMaxWorkgroups / grid)});
    if (!into) table2.reserve(table.n);
    const size_t most = std::max<size_t>(std::min<size_t>(budget, (size_t)longest), 1);  // slots that stay
    grow(w_kept, group * dev.H * most);
    if (drop) grow(w_gone, group * dev.H * (size_t)longest);
    const KvSelectSpace space = kv_select_space(dev, (int)group, (int)longest);
    grow(w_hist, space.hist);
    grow(w_counts, space.counts);
    std::vector<std::vector<int>> fresh(n);
    for (size_t i = 0; i < n; i++) fresh[i].reserve(blocks_of(stays(i)));
    if (into)
        for (size_t i = 0; i < n; i++) seqs[into[i]].blocks.reserve(blocks_of(stays(i)));
    else
        free_blocks.reserve(params.num_blocks);

    KvEvict e;
    e.budget = (int)most, e.recent = (int)std::min(recent, most), e.drop = drop;
    e.kept = w_kept.p, e.gone = drop ? w_gone.p : nullptr;
    e.dst = into ? table.p : table2.p;
    e.dpos = dpos, e.dk = dk, e.dv = dv;
    e.slots = (int)longest;
    e.hist = w_hist.p, e.counts = w_counts.p;
    e.vec = dev.D % 8 == 0 && ((uintptr_t)dk | (uintptr_t)dv) % 16 == 0;
    for (size_t i0 = 0; i0 < n;) {
        KvBatch b;
        KvRuns runs;
        b.n = 0;
        b.unit0[0] = 0;
        size_t i = i0;
        for (; i < n && b.n < (int)group; i++) {
            Seq& q = seqs[ids[i]];
            const int64_t stay = stays(i);
            const bool cut = into || q.len > stay;
            const size_t take = cut ? blocks_of(stay) : 0;
            if (take > free_blocks.size()) break;  // the blocks of those before come back first
            if ((int64_t)(b.unit0[b.n] + take) * dev.H * 2 > kMaxWorkgroups) break;
            const int j = b.n++;
            b.seq[j] = ids[i];
            b.len[j] = (int)q.len;
            b.count[j] = (int)stay;
            b.tok0[j] = (int)(i * (size_t)drop);
            b.aux[j] = into ? into[i] : ids[i];
            b.unit0[j + 1] = b.unit0[j] + (int)take;
            take_blocks(fresh[i], take, b.aux[j], into ? table.p : table2.p, runs, s);
        }
        launch_kv_table(into ? table.p : table2.p, runs, s);
        launch_kv_evict(dev, b, e, s);
        // the sequences' new state
        for (size_t x = i0; x < i; x++) {
            Seq& q = seqs[ids[x]];
            const int64_t stay = stays(x);
            if (into) {
                Seq& r = seqs[into[x]];
                r.blocks.assign(fresh[x].begin(), fresh[x].end());
                r.len = stay;
                r.next = q.next;
            } else if (q.len > stay) {
                KvRuns back;
                release_blocks(q.blocks, 0);
                for (size_t y = 0; y < fresh[x].size(); y++) {
                    const size_t at = (size_t)ids[x] * dev.W + y;
                    if (back.n && back.block[back.n - 1] + back.count[back.n - 1] == fresh[x][y]) {
                        back.count[back.n - 1]++;
                    } else {
                        if (back.n == KvRuns::MAX) {
                            launch_kv_table(table.p, back, s);
                            back.n = 0;
                        }
                        back.at[back.n] = at, back.block[back.n] = fresh[x][y], back.count[back.n] = 1;
                        back.n++;
                    }
                }
                launch_kv_table(table.p, back, s);
                q.blocks.assign(fresh[x].begin(), fresh[x].end());
                q.len = stay;
            }
        }
        i0 = i;
    }
    VGPU_HIP(hipGetLastError());
}

// Of sequences members[0..m), which hold the same blocks before block `from`, those that are to
// be taken together over the slots that they share, so that the most slots are read once for
// several; groups is given them, with the slots.
void KvCache::find_groups(const int32_t* ids, const int64_t* counts, const KvAttend& a, std::vector<uint32_t>& members,
                          size_t from, int depth, std::vector<Group>& groups, int64_t& saved) const {
    saved = 0;
    // leading blocks that all hold, and the slots of them that some row sees
    const std::vector<int>& one = seqs[ids[members[0]]].blocks;
    size_t common = one.size();
    int64_t slots = INT64_MAX, low = INT64_MAX;
    for (uint32_t i : members) {
        const Seq& q = seqs[ids[i]];
        size_t lo = from, hi = std::min(common, q.blocks.size());
        while (lo < hi) {
            const size_t mid = (lo + hi) / 2;
            if (q.blocks[mid] == one[mid]) lo = mid + 1;
            else hi = mid;
        }
        common = std::min(common, lo);
        slots = std::min(slots, q.len);
        low = std::min(low, a.window ? std::max<int64_t>(q.len - counts[i] + 1 - a.window, 0) : 0);
    }
    slots = std::min(slots, (int64_t)common << dev.shift) / KV_TILE * KV_TILE;
    low = low / KV_TILE * KV_TILE;
    const int64_t together = slots - low >= kSharedSlots ? (slots - low) * (int64_t)(members.size() - 1) : 0;
    // or apart where they part
    std::vector<Group> apart;
    int64_t apart_saved = 0;
    if (depth < kSharedDepth && members.size() > 2) {
        std::vector<uint32_t> by(members);
        const auto next = [&](uint32_t i) { return common < seqs[ids[i]].blocks.size() ? seqs[ids[i]].blocks[common] : -1; };
        std::stable_sort(by.begin(), by.end(), [&](uint32_t x, uint32_t y) { return next(x) < next(y); });
        for (size_t x = 0, y; x < by.size(); x = y) {
            for (y = x + 1; y < by.size() && next(by[y]) == next(by[x]);) y++;
            if (y - x < 2 || next(by[x]) < 0 || y - x == by.size()) continue;
            std::vector<uint32_t> part(by.begin() + (ptrdiff_t)x, by.begin() + (ptrdiff_t)y);
            int64_t more = 0;
            find_groups(ids, counts, a, part, common, depth + 1, apart, more);
            apart_saved += more;
        }
    }
    if (apart_saved > together) {
        saved = apart_saved;
        groups.insert(groups.end(), std::make_move_iterator(apart.begin()), std::make_move_iterator(apart.end()));
    } else if (together) {
        saved = together;
        groups.push_back(Group{members, low, slots});
    }
}

// Takes sequences out of the groups that are faster each by itself; true if there are such in the call.
bool KvCache::part_groups(const int32_t* ids, const int64_t* counts, size_t n, const KvAttend& a, std::vector<Group>& groups) const {
    const auto tiles_of = [](int64_t rows, int64_t wg) { return (rows + wg - 1) / wg; };
    const bool can_many = kv_shared_many(dev.Dp, a.q.type == KV_F32 ? 2 : 1);
    const int64_t chunk_rows = 64 * kv_chunk_nc(dev.Dp, a.q.type == KV_F32 ? 2 : 1);
    // The rows of a sequence: few, more, or those that the kernel of many takes (as for the rest).
    enum { FEW, MORE, MANY };
    int64_t chunk_tiles = 0, other_tiles = 0;  // of its workgroups
    for (size_t i = 0; i < n; i++)
        (counts[i] * a.G > chunk_rows * 3 / 4 ? chunk_tiles : other_tiles) +=
            tiles_of(counts[i] * a.G, chunk_rows) * dev.H * tiles_of(seqs[ids[i]].len, KV_TILE);
    const bool chunks = chunk_tiles >= kChunkTiles;
    // (taken apart beside one with many rows, those of few would go by the kernel of many as well)
    const bool steps = !chunk_tiles || chunk_tiles + other_tiles < kChunkTiles;
    const auto kind_of = [&](uint32_t i) {
        const int64_t rows = counts[i] * a.G;
        return rows <= kTileRows ? FEW : chunks && rows > chunk_rows * 3 / 4 ? MANY : MORE;
    };
    int64_t units[3] = {0, 0, 0};           // workgroups of 16 rows
    int64_t many_tiles = 0, by_many = 0;    // of MANY: tiles, sequences
    for (size_t i = 0; i < n; i++) {
        const int64_t own = tiles_of(counts[i] * a.G, 16) * dev.H;
        units[kind_of((uint32_t)i)] += own;
        if (kind_of((uint32_t)i) == MANY) by_many++, many_tiles += own * tiles_of(seqs[ids[i]].len, KV_TILE);
    }
    const bool has_many = by_many > 0;
    int64_t few = 0, few_slots = 0, others = 0, saved = 0, most = 0, most_slots = 0, tiles = 0;  // of the groups
    for (const Group& x : groups) {
        int64_t rows = 0;
        for (uint32_t i : x.members) rows += counts[i] * a.G;
        most = std::max(most, rows), most_slots = std::max(most_slots, x.slots - x.low);
        tiles += tiles_of(rows, 16) * dev.H * ((x.slots - x.low) / KV_TILE);
        saved += (x.slots - x.low) * (int64_t)(x.members.size() - 1);
        for (uint32_t i : x.members)
            if (kind_of(i) == FEW) few++, few_slots += x.slots - x.low;
            else others++, by_many -= kind_of(i) == MANY;
    }
    bool some = by_many > 0;  // not in any group
    // Beside rows of the kernel of many, where those are nearly all, less than 512 slots are not worth the
    // parts (39 sequences of 8 x 192 over 296 slots, a third with up to 1472 rows: 44 us apart, 116;
    // 39 of 32 x 128 in float32 over 475, a third with up to 147 rows: 162 and 50).
    if (!steps && most_slots < 512 && units[MANY] >= 8 * units[FEW]) {
        groups.clear();
        return true;
    }
    const bool whole = steps && whole_steps(ids, counts, n, a);
    // Those of few rows go one way, and those of more with them where they are the more, for each way
    // has launches of its own (32 sequences of 5 tokens and 32 of one, 4 x 8 x 128 over 2048 shared
    // slots: 32 us either way, 43 one each).
    const bool more_apart = whole && units[MORE] > kApartWorkgroups && units[MORE] >= 2 * units[FEW];
    const int64_t launches = tiles_of((int64_t)n, kLaunchSeqs), all = units[FEW] + units[MORE] + units[MANY];
    const int64_t least = kCrowdedSlots * launches * std::min(all, kCrowdedUnits * launches) / std::max<int64_t>(all, 1);
    const bool few_apart = (whole && few_slots < few * least) || (steps && !others && saved * dev.H * 2 * dev.Dp < kFewBytes);
    // Rows of the kernel of many stay together where that saves a third of its time, or a quarter over slots
    // that pay for the parts, by how full its workgroups and their last round are (11 sequences of 136
    // rows over 2394 slots of 32 x 96 188 us apart and 127; 12 of 266 over 16224 of 2 x 128 137 and 91, 38
    // of 204 over 8768 of 4 x 128 359 and 203, 80 of 268 over 960 of 8 x 128 204 and 315; 8 of 512
    // over 8192 164 and 244).  At the widths where it takes one sequence only it is slow, and four
    // times as many workgroups stay (9 of 560 rows over 3360 slots of 4 x 256 247 us, 181 by 16 rows
    // together; 10 of 688 over 1696 of 8 x 256 a third faster apart).
    double rounds = 1.;
    if (has_many) {
        KvPlan plan;
        KvBatch b;
        plan.heads = dev.H;
        for (size_t i = 0; i < n && plan.n < KV_BATCH; i++)
            if (kind_of((uint32_t)i) == MANY) plan.add(seqs[ids[i]].len, counts[i], a.G, chunk_rows, a.causal, a.window);
        plan.split(b, true, kPartBytes / (chunk_rows * ((int64_t)dev.Dp * 4 + 12)));
        if (plan.groups) rounds = (double)(tiles_of(plan.groups, kChunkWorkgroups) * kChunkWorkgroups) / (double)plan.groups;
    }
    const bool many_apart = units[MORE] + units[MANY] > (can_many ? 1 : 4) * kApartWorkgroups &&
                            (units[FEW] + units[MORE] == 0 || many_tiles >= kManyTiles);
    const bool many = many_shared(dev, a.q.type, most, tiles);
    for (Group& x : groups) {
        int64_t rows = 0, alone = 0;  // of the group; workgroups of many rows of its sequences
        for (uint32_t i : x.members) rows += counts[i] * a.G, alone += tiles_of(counts[i] * a.G, chunk_rows);
        const bool far = many && x.slots - x.low >= kLongSlots;
        const double gain = (double)alone * rounds / (double)tiles_of(rows, chunk_rows);
        const bool fuller = (many || !can_many) && gain >= (x.slots - x.low >= kFullerSlots ? 4. / 3 : 1.5);
        const auto apart = [&](uint32_t i) {
            const auto kind = kind_of(i);
            return kind == MANY ? many_apart && !fuller : (more_apart && !far) || (kind == FEW && few_apart);
        };
        const auto end = std::remove_if(x.members.begin(), x.members.end(), apart);
        some = some || end != x.members.end();
        x.members.erase(end, x.members.end());
    }
    return some;
}

// Makes groups of one of the sequences that are in none, where they are the fewer: a launch of both
// takes less than one after the other (8 x 11 beams of prompts of 211 to 6393 slots, of which
// two are too short to share, 4 x 8 x 128: 72 us by two ways, 49 each by itself).
void KvCache::add_singles(const int32_t* ids, const int64_t* counts, size_t n, const KvAttend& a, std::vector<Group>& groups) const {
    const auto units_of = [&](size_t i) { return (counts[i] * a.G + 15) / 16; };
    std::vector<uint8_t> in(n, 0);
    int64_t together = 0, alone = 0;
    for (const Group& x : groups)
        for (uint32_t i : x.members)
            if (x.members.size() > 1) in[i] = 1, together += units_of(i);
    for (size_t i = 0; i < n; i++)
        if (!in[i]) alone += units_of(i);
    if (alone > together) return;
    for (size_t i = 0; i < n; i++)
        if (!in[i] && counts[i]) groups.push_back(Group{{(uint32_t)i}, 0, 0});
}

// Whether steps of 16 rows, each sequence by itself, need no splits.
bool KvCache::whole_steps(const int32_t* ids, const int64_t* counts, size_t n, const KvAttend& a) const {
    std::vector<std::pair<int64_t, int64_t>> order(n);  // length, tokens
    for (size_t i = 0; i < n; i++) order[i] = {seqs[ids[i]].len, counts[i]};
    std::sort(order.begin(), order.end(), std::greater<>());
    for (size_t i = 0; i < n;) {
        KvPlan plan;
        KvBatch b;
        plan.heads = dev.H;
        for (; i < n && plan.n < KV_BATCH; i++) plan.add(order[i].first, order[i].second, a.G, 16, a.causal, a.window);
        plan.split(b, false, kPartBytes / (16 * ((int64_t)dev.Dp * 4 + 12)));
        if (plan.split_units) return false;
    }
    return true;
}

void KvCache::attend_shared(const int32_t* ids, const int64_t* counts, const std::vector<int64_t>& tok0, size_t n,
                            KvAttend a, std::vector<size_t>& rest, hipStream_t s) {
    // sequences whose first block others hold too, by that block
    std::vector<std::pair<int, uint32_t>> roots;
    if (!a.track && shared_holds)
        for (size_t i = 0; i < n; i++) {
            const std::vector<int>& b = seqs[ids[i]].blocks;
            if (counts[i] && !b.empty() && holders[b[0]] > 1) roots.push_back({b[0], (uint32_t)i});
        }
    std::vector<Group> groups;
    int64_t saved_slots = 0;
    if (roots.size() > 1) {
        std::sort(roots.begin(), roots.end());
        for (size_t x = 0, y; x < roots.size(); x = y) {
            std::vector<uint32_t> members;
            for (y = x; y < roots.size() && roots[y].first == roots[x].first; y++) members.push_back(roots[y].second);
            int64_t saved;
            if (members.size() > 1) find_groups(ids, counts, a, members, 0, 0, groups, saved), saved_slots += saved;
        }
    }
    const int parts = a.q.type == KV_F32 ? 2 : 1;
    const int64_t chunk_rows = 64 * kv_chunk_nc(dev.Dp, parts);
    bool some = false;
    if (!groups.empty() && shared_bytes) {  // (0: tests of shared slots, for any rows)
        some = part_groups(ids, counts, n, a, groups);
        saved_slots = 0;
        for (const Group& x : groups)
            if (x.members.size() > 1) saved_slots += (x.slots - x.low) * (int64_t)(x.members.size() - 1);
    }
    groups.erase(std::remove_if(groups.begin(), groups.end(), [](const Group& x) { return x.members.size() < 2; }), groups.end());
    if (saved_slots * dev.H * 2 * dev.Dp < shared_bytes) groups.clear();
    if (!groups.empty() && !some) add_singles(ids, counts, n, a, groups);
    // Groups in pieces of as many sequences as one launch takes: each has an entry of its own and
    // the piece one more, and every row leaves partial results of both.
    const int64_t row_bytes = (int64_t)dev.Dp * 4 + 12, room = kPartBytes / 2 / row_bytes / dev.H;
    const auto rows_of = [&](uint32_t i) { return (counts[i] * a.G + chunk_rows - 1) / chunk_rows * chunk_rows; };
    struct Piece {
        const Group* group;
        size_t first, end;  // of its members
        int64_t rows;
    };
    std::vector<Piece> pieces;
    for (const Group& x : groups) {
        Piece p{&x, 0, 0, 0};
        for (size_t j = 0; j <= x.members.size(); j++) {
            const int64_t more = j < x.members.size() ? rows_of(x.members[j]) : 0;
            if (j < x.members.size() && j - p.first < (size_t)KV_BATCH - 1 && p.rows + more <= room) {
                p.rows += more, p.end = j + 1;
                continue;
            }
            if (p.end - p.first > 1 || (p.end > p.first && !x.slots)) pieces.push_back(p);
            p = Piece{&x, j, j, 0};
            if (more && more <= room) p.rows = more, p.end = j + 1;
            else p.first = p.end = j + 1;  // too many rows for any launch
        }
    }
    std::vector<uint8_t> done(n, 0);
    for (size_t x = 0; x < pieces.size();) {
        struct Entry {
            int seq, first, rows, members;
            int64_t t0, end;
        };
        std::vector<Entry> entries[2];  // shared slots, own slots
        KvMembers mem;
        KvShares shares;
        int64_t used = 0;
        mem.row0[0] = 0;
        for (; x < pieces.size(); x++) {
            const Piece& p = pieces[x];
            const size_t many = p.end - p.first;
            if (mem.n && (mem.n + many + entries[0].size() + 1 > (size_t)KV_BATCH || used + p.rows > room)) break;
            used += p.rows;
            const int first = mem.n;
            for (size_t j = p.first; j < p.end; j++) {
                const uint32_t i = p.group->members[j];
                const Seq& q = seqs[ids[i]];
                const int m = mem.n++, count = (int)(counts[i] * a.G);
                mem.tok0[m] = (int)tok0[i], mem.len[m] = (int)q.len, mem.count[m] = (int)counts[i];
                mem.row0[m + 1] = mem.row0[m] + count;
                shares.row0[m] = mem.row0[m] - mem.row0[first];
                for (int z = 0; z < 2; z++) shares.unit[z][m] = shares.tiles[z][m] = shares.splits[z][m] = 0;
                const int64_t low = a.window ? std::max<int64_t>(q.len - counts[i] + 1 - a.window, 0) : 0;
                const int64_t t0 = std::max(p.group->slots, low) / KV_TILE;
                if (t0 * KV_TILE < q.len) entries[1].push_back({ids[i], m, count, 1, t0, q.len});
                done[i] = 1;
            }
            if (p.group->slots)
                entries[0].push_back({ids[p.group->members[p.first]], first, mem.row0[mem.n] - mem.row0[first], (int)many,
                                      p.group->low / KV_TILE, p.group->slots});
        }
        // the kernel that suits the rows, for each kind of slots; one launch where it is the same
        bool by_rows[2];
        for (int y = 0; y < 2; y++) {
            int64_t most = 0, tiles = 0;
            for (const Entry& e : entries[y]) {
                most = std::max<int64_t>(most, e.rows);
                tiles += (e.rows + 15) / 16 * dev.H * ((e.end + KV_TILE - 1) / KV_TILE - e.t0);
            }
            by_rows[y] = many_shared(dev, a.q.type, most, tiles);
        }
        const int launches = by_rows[0] == by_rows[1] ? 1 : 2;
        KvBatch b[2];
        int64_t base[2] = {0, 0}, all_rows = 0;
        for (int y = 0; y < launches; y++) {
            const int wg = by_rows[y] ? (int)chunk_rows : 16, z1 = launches == 1 ? 2 : y + 1;
            KvPlan plan;
            plan.heads = dev.H;
            b[y].n = 0, b[y].unit0[0] = 0;
            for (int z = y; z < z1; z++)
                for (const Entry& e : entries[z]) {
                    const int j = b[y].n++;
                    b[y].seq[j] = e.seq, b[y].aux[j] = e.first, b[y].count[j] = e.rows;
                    b[y].tok0[j] = (int)e.t0, b[y].len[j] = (int)e.end;
                    plan.add_entry(e.rows, (e.end + KV_TILE - 1) / KV_TILE - e.t0, wg);
                }
            plan.split_entries(b[y], by_rows[y], kPartBytes / 2 / (wg * row_bytes));
            base[y] = all_rows;
            all_rows += plan.groups * wg;
            int j = 0;
            for (int z = y; z < z1; z++) {
                shares.rows[z] = wg, shares.base[z] = (size_t)base[y];
                for (const Entry& e : entries[z]) {
                    for (int m = e.first; m < e.first + e.members; m++) {
                        shares.unit[z][m] = b[y].unit0[j], shares.splits[z][m] = b[y].splits[j];
                        shares.tiles[z][m] = (e.rows + wg - 1) / wg;
                    }
                    j++;
                }
            }
        }
        grow(w_part, (size_t)all_rows * dev.Dp);
        grow(w_ml, (size_t)all_rows);
        grow(w_power, (size_t)all_rows);
        for (int y = 0; y < launches; y++) {
            a.by_rows = by_rows[y];
            a.part_o = w_part.p + base[y] * dev.Dp, a.part_ml = w_ml.p + base[y], a.part_s = w_power.p + base[y];
            launch_kv_shared(dev, b[y], a, mem, s);
        }
        a.part_o = w_part.p, a.part_ml = w_ml.p, a.part_s = w_power.p;
        launch_kv_shared_join(dev, a, mem, shares, s);
    }
    for (size_t i = 0; i < n; i++)
        if (!done[i]) rest.push_back(i);
}

void KvCache::attend(const int32_t* ids, const int64_t* counts, size_t n, const vgpu_kv_query& q, hipStream_t s) {
    check_call(s);
    check_ids(*this, seen, ids, n);
    need(q.num_q_heads > 0 && q.num_q_heads % (size_t)dev.H == 0 && q.num_q_heads <= 65536,
         "num_q_heads must be a multiple of the cache's heads (" + std::to_string(dev.H) + ")");
    need(std::isfinite(q.scale), "scale must be finite");
    need(!q.track || std::isfinite(q.decay), "decay must be finite");
    KvAttend a;
    a.q = tensor(q.q, "q");
    a.G = (int)(q.num_q_heads / (size_t)dev.H);
    a.by_group = KvDiv(a.G);
    a.scale2 = q.scale * 1.44269504088896341f;
    a.causal = q.causal != 0;
    a.window = (int)std::min<size_t>(q.window, (size_t)INT_MAX / 2);
    a.mask = q.mask;
    a.mask_st = q.mask_stride_token, a.mask_ss = q.mask_stride_slot;
    a.track = q.track != 0;
    a.decay = q.decay;
    a.out = q.out;
    a.lse = q.lse;
    a.vec_out = dev.D % 4 == 0 && (uintptr_t)q.out % (4 * item_size(a.q.type)) == 0;
    const int parts = a.q.type == KV_F32 ? 2 : 1;
    const int64_t chunk_rows = 64 * kv_chunk_nc(dev.Dp, parts);
    int64_t tokens = 0, longest = 0;
    std::vector<int64_t> tok0(n);
    for (size_t i = 0; i < n; i++) {
        need(counts[i] >= 0 && counts[i] <= INT_MAX / 2, "counts must not be negative, nor above 2^30");
        tok0[i] = tokens;
        tokens += counts[i];
        need(tokens * (int64_t)q.num_q_heads <= INT_MAX / 2, "more than 2^30 query rows in one call");
        longest = std::max(longest, seqs[ids[i]].len);
    }
    need(!q.mask || (int64_t)q.mask_slots >= longest, "a mask row must cover the longest sequence (" +
                                                          std::to_string(longest) + " slots)");
    need(!tokens || (q.q.data && q.out), "null argument");
    need((uintptr_t)q.out % item_size(a.q.type) == 0 && (uintptr_t)q.lse % 4 == 0, "outputs must be aligned to their dtype");

    // The sequences that share their first blocks with others of the call, and the rest.
    std::vector<size_t> order;
    attend_shared(ids, counts, tok0, n, a, order, s);
    if (order.empty() && n) {
        VGPU_HIP(hipGetLastError());
        return;
    }
    int64_t most = 0, chunk_tiles = 0, step_units = 0;
    for (size_t i : order) {
        most = std::max(most, counts[i] * a.G);
        step_units += (counts[i] * a.G + 15) / 16 * dev.H;
        chunk_tiles += (counts[i] * a.G + chunk_rows - 1) / chunk_rows * dev.H * ((seqs[ids[i]].len + KV_TILE - 1) / KV_TILE);
    }
    // Many rows: each wave has its own; few: the waves share them and split the tiles.
    a.by_rows = a.track ? most > kScoreRows : most > chunk_rows * 3 / 4 && chunk_tiles >= kChunkTiles;
    const bool keep_scores = a.track && !a.by_rows;
    if (a.track) {
        // weights are written to every slot: the blocks have to be the sequences' own
        const std::vector<int64_t> all(n, 0);
        const size_t want = shared_blocks(ids, all.data(), n);
        need(want <= free_blocks.size(),
             "weights of shared blocks need " + std::to_string(want) + " more blocks, the cache has " +
                 std::to_string(free_blocks.size()), VGPU_ERR_OUT_OF_MEMORY);
        KvRuns runs;
        own_blocks(ids, all.data(), n, runs, s);
        launch_kv_table(table.p, runs, s);
        grow(w_lse2, (size_t)tokens * q.num_q_heads);
        a.lse2 = w_lse2.p;
        if (!keep_scores) {
            grow(w_qs, (size_t)tokens * q.num_q_heads);
            a.qs = w_qs.p;
        }
    }
    const int rows = kv_attend_rows(a, dev.Dp);
    // Where a workgroup's work depends on its sequence, the short sequences come first: the
    // light rows of the longest end the launch.  Steps that may have more workgroups than
    // are on the card at once begin with the longest.
    if (a.by_rows)
        std::stable_sort(order.begin(), order.end(), [&](size_t x, size_t y) { return seqs[ids[x]].len < seqs[ids[y]].len; });
    else if (step_units > kStepWorkgroups / 2)
        std::stable_sort(order.begin(), order.end(), [&](size_t x, size_t y) { return seqs[ids[x]].len > seqs[ids[y]].len; });
    // Where several launches add weights, all of them are checked and their workspaces grown
    // before the first, so that a call that fails has added none.
    const size_t rest = order.size();
    for (int dry = a.track && rest > KV_BATCH; dry >= 0; dry--)
    for (size_t i0 = 0; i0 < rest; i0 += KV_BATCH) {
        KvBatch b;
        b.n = 0;
        b.unit0[0] = 0;
        KvPlan plan;
        plan.heads = dev.H;
        int64_t score_tiles = 0, row_tiles = 0;
        for (size_t x = i0; x < std::min(rest, i0 + KV_BATCH); x++) {
            const size_t i = order[x];
            const int64_t len = seqs[ids[i]].len;
            const int j = b.n++;
            b.seq[j] = ids[i];
            b.len[j] = (int)len;
            b.tok0[j] = (int)tok0[i];
            b.count[j] = (int)counts[i];
            need(score_tiles <= INT_MAX / 2, "too many scores in one call");
            b.aux[j] = (int)(keep_scores ? score_tiles : row_tiles);
            if (keep_scores) score_tiles += (len + KV_TILE - 1) / KV_TILE * counts[i] * a.G;
            row_tiles += (counts[i] * a.G + 15) / 16;
            plan.add(len, counts[i], a.G, rows, a.causal, a.window);
        }
        need(plan.units <= kMaxWorkgroups, "too many query rows in one call");
        if (plan.units) {
            plan.split(b, a.by_rows, kPartBytes / (rows * ((int64_t)dev.Dp * 4 + 12)));
            const int64_t groups = plan.groups;
            a.part_o = nullptr, a.part_ml = nullptr, a.part_s = nullptr, a.scores = nullptr;
            if (plan.split_units) {
                grow(w_part, (size_t)(groups * rows) * dev.Dp);
                grow(w_ml, (size_t)(groups * rows));
                grow(w_power, (size_t)(groups * rows));
                a.part_o = w_part.p, a.part_ml = w_ml.p, a.part_s = w_power.p;
            }
            if (keep_scores) {
                grow(w_scores, (size_t)score_tiles * KV_TILE * dev.H);
                a.scores = w_scores.p;
            }
            if (a.track && !keep_scores) {
                grow(w_qop, (size_t)row_tiles * dev.H * parts * (dev.Dp / 32) * 64);
                a.qop = w_qop.p;
            }
            if (!dry) launch_kv_attend(dev, b, a, s);
        }
        if (a.track) {
            const int per = keep_scores ? KV_SCORE_SLOTS : KV_WEIGHT_SLOTS;
            for (int j = 0; j < b.n; j++) b.unit0[j + 1] = b.unit0[j] + (b.len[j] + per - 1) / per;
            if (!keep_scores) {
                // chunks of at least 256 rows, until there are workgroups enough
                const int64_t groups = std::max<int64_t>((int64_t)b.unit0[b.n] * dev.H, 1);
                const int64_t chunks = std::min((most + 255) / 256, (kWeightWorkgroups + groups - 1) / groups);
                a.chunk_rows = (int)(((most + chunks - 1) / chunks + 31) / 32 * 32);
                a.chunks = (int)((most + a.chunk_rows - 1) / a.chunk_rows);
                grow(w_wpart, (size_t)(groups * a.chunks * KV_WEIGHT_SLOTS));
                a.wpart = w_wpart.p;
            }
            if (!dry) launch_kv_weights(dev, b, a, s);
        }
    }
    VGPU_HIP(hipGetLastError());
}

}  // namespace vgpu
