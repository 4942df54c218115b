// The attention memory's host side: argument checks, blocks and lengths, and the
// launches of one call.
#include <algorithm>
#include <climits>
#include <cmath>

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
    seqs.resize(p.num_seqs);
    seen.assign(p.num_seqs, 0);
    free_blocks.resize(p.num_blocks);
    for (size_t i = 0; i < p.num_blocks; i++) free_blocks[i] = (int)(p.num_blocks - 1 - i);
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
           table2.bytes() + w_kept.bytes() + w_gone.bytes() + w_part.bytes() + w_scores.bytes() + w_lse2.bytes() +
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

void KvCache::take_blocks(std::vector<int>& out, size_t count, size_t row, int* tab, KvRuns& runs, hipStream_t s) {
    for (size_t j = 0; j < count; j++) {
        const int block = free_blocks.back();
        const size_t at = row * (size_t)dev.W + out.size();
        if (runs.n && runs.at[runs.n - 1] + runs.count[runs.n - 1] == at &&
            runs.block[runs.n - 1] + runs.count[runs.n - 1] == block) {
            runs.count[runs.n - 1]++;
        } else {
            if (runs.n == KvRuns::MAX) {
                launch_kv_table(tab, runs, s);
                runs.n = 0;
            }
            runs.at[runs.n] = at, runs.block[runs.n] = block, runs.count[runs.n] = 1;
            runs.n++;
        }
        out.push_back(block);
        free_blocks.pop_back();
    }
}

void KvCache::release_blocks(std::vector<int>& blocks, size_t keep) {
    while (blocks.size() > keep) {
        free_blocks.push_back(blocks.back());
        blocks.pop_back();
    }
}

void KvCache::append(const int32_t* ids, const int64_t* counts, size_t n, const vgpu_tensor3& k, const vgpu_tensor3& v,
                     const int32_t* pos, const float* wts, hipStream_t s) {
    check_call(s);
    check_ids(*this, seen, ids, n);
    need(k.dtype == v.dtype, "k and v must have the same dtype");
    const KvTensor kt = tensor(k, "k"), vt = tensor(v, "v");
    int64_t tokens = 0;
    size_t want = 0;
    for (size_t i = 0; i < n; i++) {
        const Seq& q = seqs[ids[i]];
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
    need(want <= free_blocks.size(),
         "the cache needs " + std::to_string(want) + " more blocks and has " + std::to_string(free_blocks.size()),
         VGPU_ERR_OUT_OF_MEMORY);
    for (size_t i = 0; i < n; i++) seqs[ids[i]].blocks.reserve(blocks_of(seqs[ids[i]].len + counts[i]));
    KvRuns runs;
    for (size_t i = 0; i < n; i++) {
        Seq& q = seqs[ids[i]];
        const size_t more = blocks_of(q.len + counts[i]) - q.blocks.size();
        // one block touched: the append itself writes the table
        if (more == 1 && q.len % dev.B == 0 && counts[i] <= dev.B) {
            q.blocks.push_back(free_blocks.back());
            free_blocks.pop_back();
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
    // does the pool hold the new blocks, given what comes back on the way?
    size_t have = free_blocks.size();
    for (size_t i = 0; i < n; i++) {
        const Seq& q = seqs[ids[i]];
        need(!drops || q.len - stays(i) <= (int64_t)num_dropped,
             "num_dropped is below what leaves sequence " + std::to_string(ids[i]));
        if (!into && q.len <= (int64_t)budget) continue;
        const size_t take = blocks_of(stays(i));
        need((int64_t)take * dev.H * 2 <= kMaxWorkgroups, "too many slots of one sequence in one call");
        need(take <= have, "the cut sequences need " + std::to_string(take) + " free blocks and find " +
                               std::to_string(have), VGPU_ERR_OUT_OF_MEMORY);
        have -= take;
        if (!into) have += q.blocks.size();
    }
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
    int64_t tokens = 0, longest = 0, most = 0, chunk_tiles = 0, step_units = 0;
    for (size_t i = 0; i < n; i++) {
        need(counts[i] >= 0 && counts[i] <= INT_MAX / 2, "counts must not be negative, nor above 2^30");
        tokens += counts[i];
        need(tokens * (int64_t)q.num_q_heads <= INT_MAX / 2, "more than 2^30 query rows in one call");
        longest = std::max(longest, seqs[ids[i]].len);
        most = std::max(most, counts[i] * a.G);
        step_units += (counts[i] * a.G + 15) / 16 * dev.H;
        chunk_tiles += (counts[i] * a.G + chunk_rows - 1) / chunk_rows * dev.H * ((seqs[ids[i]].len + KV_TILE - 1) / KV_TILE);
    }
    need(!q.mask || (int64_t)q.mask_slots >= longest, "a mask row must cover the longest sequence (" +
                                                          std::to_string(longest) + " slots)");
    need(!tokens || (q.q.data && q.out), "null argument");
    need((uintptr_t)q.out % item_size(a.q.type) == 0 && (uintptr_t)q.lse % 4 == 0, "outputs must be aligned to their dtype");

    // Many rows: each wave has its own; few: the waves share them and split the tiles.
    a.by_rows = a.track ? most > kScoreRows : most > chunk_rows * 3 / 4 && chunk_tiles >= kChunkTiles;
    const bool keep_scores = a.track && !a.by_rows;
    if (a.track) {
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
    std::vector<size_t> order(n);
    std::vector<int64_t> tok0(n);
    int64_t tok = 0;
    for (size_t i = 0; i < n; i++) order[i] = i, tok0[i] = tok, tok += counts[i];
    if (a.by_rows)
        std::stable_sort(order.begin(), order.end(), [&](size_t x, size_t y) { return seqs[ids[x]].len < seqs[ids[y]].len; });
    else if (step_units > kStepWorkgroups / 2)
        std::stable_sort(order.begin(), order.end(), [&](size_t x, size_t y) { return seqs[ids[x]].len > seqs[ids[y]].len; });
    // Where several launches add weights, all of them are checked and their workspaces grown
    // before the first, so that a call that fails has added none.
    for (int dry = a.track && n > KV_BATCH; dry >= 0; dry--)
    for (size_t i0 = 0; i0 < n; i0 += KV_BATCH) {
        KvBatch b;
        b.n = 0;
        b.unit0[0] = 0;
        KvPlan plan;
        plan.heads = dev.H;
        int64_t score_tiles = 0, row_tiles = 0;
        for (size_t x = i0; x < std::min(n, i0 + KV_BATCH); x++) {
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
