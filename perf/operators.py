"""The attention memory's operators, as cases that can be timed.

A KVCache holds the keys and values of a model's tokens in 8 bits, with one
scale for each block of tokens and head.  Three operators work on it:

  append  new tokens are quantised into the cache (a block's scale only grows;
          the codes that it holds already are rounded again when it does);
  attend  softmax attention of the newest tokens over the cached ones, also
          with the weight that each cached token received;
  evict   each head keeps its newest tokens and those of largest accumulated
          weight; the others leave the cache as float32 values (for a vector
          index, which searches them by the same inner product).

The state that append and evict leave behind is returned as the values that the
8-bit codes stand for, through KVCache.read.

Keys have a few dimensions of large magnitude, queries lean towards some
cached keys, accumulated weights are heavy-tailed with many equal ones.
"""

from __future__ import annotations

import math
import random

import torch

DEV = "cuda:0"
own = False  # True: the calls of vicinity_amd; False: elementary torch operations

ZMAX = {"int8": 127.0, "fp8": 448.0}
TINY = 2.0 ** -100  # a block whose largest magnitude is below this is stored as zeros
DTYPES = {"bfloat16": torch.bfloat16, "float16": torch.float16, "float32": torch.float32}


def listed():
    return [
        # one generated token of each of a serving batch's conversations joins its cache
        dict(name="append_step", kind="append", n=61, longest=3500, new=1, heads=8, dim=128,
             block=64, code="int8", dtype="bfloat16"),
        # four prompts of different lengths enter empty caches
        dict(name="append_prompts", kind="append", n=4, longest=0, new=8191, heads=8, dim=128,
             block=64, code="fp8", dtype="bfloat16"),
        # a chunk of one long document joins what is there, float32 keys, an odd head dimension
        dict(name="append_chunk_odd", kind="append", n=1, longest=1001, new=777, heads=5, dim=80,
             block=32, code="int8", dtype="float32"),
        # the first tokens of one short conversation: latency
        dict(name="attend_short", kind="attend", n=1, longest=37, queries=1, heads=4, group=4,
             dim=64, code="int8", dtype="bfloat16", block=64, window=0, masked=False, track=False),
        # a serving batch's decode step, ragged lengths, shared heads
        dict(name="attend_batch", kind="attend", n=61, longest=8191, queries=1, heads=8, group=4,
             dim=128, code="int8", dtype="bfloat16", block=64, window=0, masked=False,
             track=False),
        # one token over a long document, with the weights that eviction needs
        dict(name="attend_long_weights", kind="attend", n=1, longest=131_071, queries=1, heads=8,
             group=8, dim=128, code="fp8", dtype="bfloat16", block=128, window=0, masked=False,
             track=True),
        # float32 queries, a head each, odd dimension, a few drafted tokens at once, a window
        # and a mask of the documents that the user may see
        dict(name="attend_draft_masked", kind="attend", n=7, longest=5003, queries=5, heads=12,
             group=1, dim=80, code="int8", dtype="float32", block=32, window=2048, masked=True,
             track=False),
        # a chunk of a long document attends to all that came before it
        dict(name="attend_chunk", kind="attend", n=1, longest=32_768, queries=2048, heads=8,
             group=4, dim=128, code="int8", dtype="bfloat16", block=64, window=0, masked=False,
             track=False),
        # whole prompts, with the weights that each of their tokens received
        dict(name="attend_prompts_weights", kind="attend", n=3, longest=4001, queries=4001,
             heads=4, group=4, dim=128, code="fp8", dtype="float16", block=64, window=0,
             masked=False, track=True),
        # a serving batch's caches are cut to their budget
        dict(name="evict_batch", kind="evict", n=31, longest=4096, budget=1024, recent=128,
             heads=8, dim=128, block=64, code="int8", dropped=False),
        # a long document is cut down and what leaves it goes to the vector index
        dict(name="evict_long_dropped", kind="evict", n=1, longest=100_003, budget=16_384,
             recent=1000, heads=8, dim=128, block=128, code="fp8", dropped=True),
    ]


def _log_int(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    """One more case of the listed ones' ranges."""
    kind = rng.choice(["append", "append", "attend", "attend", "attend", "attend", "evict"])
    case = dict(kind=kind, heads=rng.choice([1, 2, 4, 5, 8, 8, 12]),
                dim=rng.choice([40, 64, 64, 80, 96, 128, 128, 128, 192, 256]),
                block=rng.choice([32, 64, 64, 128]), code=rng.choice(["int8", "fp8"]))
    if kind == "append":
        case["dtype"] = rng.choice(["bfloat16", "bfloat16", "float16", "float32"])
        case["n"] = _log_int(rng, 1, 64)
        case["longest"] = rng.choice([0, _log_int(rng, 1, 8192)])
        case["new"] = 1 if rng.random() < 0.4 else _log_int(rng, 2, max(2, 8192 // case["n"]))
        return case
    if kind == "evict":
        case["n"] = _log_int(rng, 1, 48)
        case["longest"] = _log_int(rng, 64, max(64, min(100_000, 131_072 // case["n"])))
        case["budget"] = max(2, int(case["longest"] * rng.uniform(0.05, 0.7)))
        case["recent"] = int(case["budget"] * rng.choice([0.0, 0.1, 0.5]))
        case["dropped"] = rng.random() < 0.5
        return case
    case["dtype"] = rng.choice(["bfloat16", "bfloat16", "float16", "float32"])
    case["group"] = rng.choice([1, 1, 2, 3, 4, 4, 7, 8, 16])
    case["track"] = rng.random() < 0.3
    case["masked"] = rng.random() < 0.25
    form = rng.choice(["step", "step", "draft", "chunk"])
    if form == "chunk":
        case["n"] = rng.choice([1, 1, 2, 3])
        case["queries"] = _log_int(rng, 17, 2048 // case["n"])
        case["longest"] = case["queries"] + rng.choice([0, _log_int(rng, 1, 16_384)])
    else:
        case["n"] = _log_int(rng, 1, 64)
        case["queries"] = 1 if form == "step" else rng.randint(2, 16)
        case["longest"] = _log_int(rng, 16, max(16, min(131_072, 262_144 // case["n"])))
    case["window"] = rng.choice([0, 0, 0, _log_int(rng, 1, max(1, case["longest"]))])
    return case


# ---- inputs ---------------------------------------------------------------


def _gen(seed, part):
    return torch.Generator(device=DEV).manual_seed(seed * 1000 + part)


def _lens(case):
    """Cached tokens of each sequence before the call: the longest one and others spread
    below it (a plain function of the case)."""
    n, longest = case["n"], case["longest"]
    if longest == 0:
        return [0] * n
    rng = random.Random(f"lens {n} {longest}")
    lens = [longest] + [_log_int(rng, max(1, longest // 16), longest) for _ in range(n - 1)]
    if case["kind"] == "attend" and case["queries"] < longest:  # otherwise whole prompts
        lens = [max(x, case["queries"]) for x in lens]
    return lens


def _new(case):
    """Tokens that an append case adds to each sequence."""
    if case["new"] == 1:
        return [1] * case["n"]
    rng = random.Random(f"new {case['n']} {case['new']}")
    return [case["new"]] + [_log_int(rng, max(1, case["new"] // 4), case["new"])
                            for _ in range(case["n"] - 1)]


def _queries(case):
    lens = _lens(case)
    return lens if case["queries"] == case["longest"] else [case["queries"]] * case["n"]


def _tokens(t, heads, dim, seed, part, dtype):
    """Keys and values [t, heads, dim]: a head's keys have an offset and a few large
    dimensions."""
    g = _gen(seed, part)
    gain = torch.ones((heads, dim), device=DEV)
    gain[:, :: max(1, dim // 3)] = 4.0
    off = torch.randn((heads, dim), generator=_gen(seed, 7), device=DEV) * 0.5
    k = torch.randn((t, heads, dim), generator=g, device=DEV).mul_(gain).add_(off * gain)
    v = torch.randn((t, heads, dim), generator=g, device=DEV)
    return k.to(dtype), v.to(dtype)


def _weights(t, heads, seed):
    """Accumulated weights [t, heads]: heavy-tailed, a sixth of them equal to another one."""
    g = _gen(seed, 11)
    w = torch.randn((t, heads), generator=g, device=DEV).mul_(2.0).exp_()
    coarse = torch.rand((t, heads), generator=g, device=DEV) < 1 / 6
    return torch.where(coarse, (w * 4).round() / 4, w)


def _inputs(case, seed):
    """What the caller holds, on the GPU: cached tokens (as they were before quantisation)
    and the call's own tensors."""
    dtype = DTYPES[case.get("dtype", "bfloat16")]
    h, d = case["heads"], case["dim"]
    lens = _lens(case)
    k, v = _tokens(sum(lens), h, d, seed, 1, dtype)
    out = {"lens": lens, "k": k, "v": v}
    if case["kind"] == "append":
        out["new"] = _new(case)
        nk, nv = _tokens(sum(out["new"]), h, d, seed, 2, dtype)
        # some of the new keys are larger than what their block held
        out["new_k"], out["new_v"] = nk * 1.25, nv
    elif case["kind"] == "evict":
        out["weights"] = _weights(sum(lens), h, seed)
    else:
        counts = _queries(case)
        rows, heads_q = sum(counts), h * case["group"]
        g = _gen(seed, 3)
        q = torch.randn((rows, heads_q, d), generator=g, device=DEV)
        # each query row leans towards one cached key of its sequence
        start = torch.tensor([sum(lens[:i]) for i in range(len(lens))], device=DEV)
        seq = torch.repeat_interleave(torch.arange(len(lens), device=DEV),
                                      torch.tensor(counts, device=DEV))
        size = torch.tensor(lens, device=DEV)[seq]
        pick = start[seq] + (torch.rand((rows,), generator=g, device=DEV) * size).long()
        near = k[pick].float().repeat_interleave(case["group"], dim=1)
        out["counts"] = counts
        out["q"] = (0.3 * q + 0.1 * near).to(dtype)
        if case["masked"]:
            # documents of 16 tokens that a user may see, one in eight of them not
            spans = (max(lens) + 15) // 16
            see = torch.rand((rows, spans), generator=g, device=DEV) >= 0.125
            out["mask"] = see.repeat_interleave(16, dim=1)[:, :max(lens)].contiguous()
    return out


def prepare(case, seed):
    x = _inputs(case, seed)
    lens = x["lens"]
    state = {"case": case, "x": x}
    if own:
        import vicinity_amd as va

        extra = x["new"] if case["kind"] == "append" else [0] * case["n"]
        blocks = sum(-(-(a + b) // case["block"]) for a, b in zip(lens, extra))
        if case["kind"] == "evict":
            blocks += case["n"] * -(-case["budget"] // case["block"])
        seqs = case["n"] * (2 if case["kind"] == "evict" else 1)
        cache = va.KVCache(seqs, case["heads"], case["dim"], blocks, block_tokens=case["block"],
                           code=case["code"])
        if sum(lens):
            cache.append(x["k"], x["v"], seqs=range(case["n"]), counts=lens,
                         weights=x.get("weights"))
        state["cache"] = cache
    else:
        held, at = [], 0
        for n in lens:
            kc, ks = _grow(None, None, x["k"][at:at + n], case)
            vc, vs = _grow(None, None, x["v"][at:at + n], case)
            held.append((kc, ks, vc, vs))
            at += n
        state["held"] = held
    # the caller keeps what it still needs; the cached tokens live in the cache alone
    if case["kind"] != "evict":
        x.pop("weights", None)
    x.pop("k")
    x.pop("v")
    return state


# ---- the plain forms --------------------------------------------------------


def _encode(x, code):
    if code == "int8":
        return x.round().clamp(-127.0, 127.0).to(torch.int8)
    return x.clamp(-448.0, 448.0).to(torch.float8_e4m3fn)


def _blocks(x, block):
    """[t, ...] padded with zeros to whole blocks: [blocks, block, ...]."""
    pad = -x.shape[0] % block
    if pad:
        x = torch.cat([x, x.new_zeros((pad,) + x.shape[1:])])
    return x.view((-1, block) + x.shape[1:])


def _grow(codes, scales, x, case):
    """One sequence's codes [t, h, d] and scales [blocks, h] after x [m, h, d] joins it."""
    block, z = case["block"], ZMAX[case["code"]]
    held = 0 if codes is None else codes.shape[0]
    first = held // block * block
    x = x.float()
    m = x.shape[0]
    lead = x.new_zeros((held - first,) + x.shape[1:])
    xb = _blocks(torch.cat([lead, x]), block)
    amax = xb.abs().amax(dim=(1, 3))
    s = torch.where(amax >= TINY, amax / z, torch.zeros_like(amax))
    if held > first:
        s[0] = torch.maximum(s[0], scales[-1])
    inv = torch.where(s > 0, 1.0 / s, torch.zeros_like(s))
    new = _encode(xb * inv[:, None, :, None], case["code"])
    new = new.view((-1,) + x.shape[1:])[held - first:held - first + m]
    if held == 0:
        return new, s
    if held > first:
        ratio = torch.where(s[0] > 0, scales[-1] / s[0], torch.zeros_like(s[0]))
        tail = _encode(codes[first:].float() * ratio[None, :, None], case["code"])
        keep = scales[:-1]
    else:
        tail, keep = codes[first:], scales
    return _cat([codes[:first], tail, new]), torch.cat([keep, s])


def _cat(parts):
    if parts[0].dtype == torch.int8:
        return torch.cat(parts)
    return torch.cat([p.view(torch.uint8) for p in parts]).view(parts[0].dtype)


def _values(codes, scales, block):
    per_slot = scales.repeat_interleave(block, dim=0)[:codes.shape[0]]
    return codes.float() * per_slot[:, :, None]


def _plain_append(state):
    case, x = state["case"], state["x"]
    k, v, at = [], [], 0
    for (kc, ks, vc, vs), n, m in zip(state["held"], x["lens"], x["new"]):
        first = n // case["block"] * case["block"]
        for out, codes, scales, new in ((k, kc, ks, x["new_k"]), (v, vc, vs, x["new_v"])):
            c, s = _grow(codes if n else None, scales, new[at:at + m], case)
            out.append(_values(c, s, case["block"])[first:])
        at += m
    return {"k": torch.cat(k), "v": torch.cat(v)}


def _plain_attend(state):
    case, x = state["case"], state["x"]
    g, d = case["group"], case["dim"]
    outs, lses, ws, at = [], [], [], 0
    for (kc, ks, vc, vs), n, m in zip(state["held"], x["lens"], x["counts"]):
        k = _values(kc, ks, case["block"])
        v = _values(vc, vs, case["block"])
        q = x["q"][at:at + m].float()
        slot = torch.arange(n, device=DEV)
        last = n - m + torch.arange(m, device=DEV)
        see = slot[None, :] <= last[:, None]
        if case["window"]:
            see &= slot[None, :] > last[:, None] - case["window"]
        if case["masked"]:
            see &= x["mask"][at:at + m, :n]
        # [heads, m * g, d] x [heads, d, n]
        qh = q.view(m, case["heads"], g, d).transpose(0, 1).reshape(case["heads"], m * g, d)
        kt, vh = k.permute(1, 2, 0).contiguous(), v.transpose(0, 1).contiguous()
        s = torch.bmm(qh, kt) * (1.0 / math.sqrt(d))
        s = s.view(-1, m, g, n).masked_fill_(~see[None, :, None, :], -math.inf)
        top = s.amax(dim=3, keepdim=True)
        top = torch.where(top == -math.inf, torch.zeros_like(top), top)
        p = torch.exp(s - top)
        total = p.sum(dim=3, keepdim=True)
        lse = (top + torch.log(total))[..., 0].transpose(0, 1).reshape(m, -1)
        p = p / torch.where(total == 0, torch.ones_like(total), total)
        o = torch.bmm(p.view(-1, m * g, n), vh).view(-1, m, g, d)
        o = o.transpose(0, 1).reshape(m, -1, d)
        w = p.sum(dim=(1, 2)).T
        outs.append(o.to(x["q"].dtype))
        lses.append(lse)
        ws.append(w)
        at += m
    out = {"out": torch.cat(outs), "lse": torch.cat(lses)}
    if case["track"]:
        out["weights"] = torch.cat(ws)
    return out


def _kept(w, budget, recent):
    """Slots that stay, ascending, and those that leave, of one sequence: w [n, h]."""
    n = w.shape[0]
    if n <= budget:
        every = torch.arange(n, device=DEV)[:, None].expand(n, w.shape[1])
        return every, every[:0]
    old = n - recent
    order = torch.sort(w[:old], dim=0, descending=True, stable=True).indices
    best = order[:budget - recent].sort(dim=0).values
    gone = order[budget - recent:].sort(dim=0).values
    tail = torch.arange(old, n, device=DEV)[:, None].expand(recent, w.shape[1])
    return torch.cat([best, tail]), gone


def _plain_evict(state):
    case, x = state["case"], state["x"]
    block = case["block"]
    out = {"k": [], "v": [], "positions": [], "weights": []}
    drop = {"k": [], "v": [], "positions": []}
    at = 0
    most = max(max(x["lens"]) - case["budget"], 0)
    for (kc, ks, vc, vs), n in zip(state["held"], x["lens"]):
        w = x["weights"][at:at + n]
        at += n
        stay, gone = _kept(w, case["budget"], case["recent"])
        heads = torch.arange(case["heads"], device=DEV)[None, :]
        for name, codes, scales in (("k", kc, ks), ("v", vc, vs)):
            c = codes.float()[stay, heads]
            s = scales[stay // block, heads]
            top = _blocks(s, block).amax(dim=1)
            if n <= case["budget"]:
                top = scales
            per_slot = top.repeat_interleave(block, dim=0)[:stay.shape[0]]
            ratio = torch.where(per_slot > 0, s / per_slot, torch.zeros_like(s))
            moved = _encode(c * ratio[:, :, None], case["code"]).float()
            out[name].append(moved * per_slot[:, :, None])
            if case["dropped"]:
                part = codes.float()[gone, heads] * scales[gone // block, heads][:, :, None]
                full = torch.zeros((most,) + part.shape[1:], device=DEV)
                full[:part.shape[0]] = part
                drop[name].append(full)
        out["positions"].append(stay.to(torch.int32))
        out["weights"].append(w[stay, heads])
        if case["dropped"]:
            full = torch.full((most, case["heads"]), -1, dtype=torch.int32, device=DEV)
            full[:gone.shape[0]] = gone.to(torch.int32)
            drop["positions"].append(full)
    res = {name: torch.cat(parts) for name, parts in out.items()}
    if case["dropped"]:
        res["dropped"] = {name: torch.stack(parts) for name, parts in drop.items()}
    return res


# ---- one pass ---------------------------------------------------------------


def run(state):
    case, x = state["case"], state["x"]
    if not own:
        return {"append": _plain_append, "attend": _plain_attend,
                "evict": _plain_evict}[case["kind"]](state)
    cache, n = state["cache"], case["n"]
    if case["kind"] == "append":
        cache.append(x["new_k"], x["new_v"], counts=x["new"])
        first = [a // case["block"] * case["block"] for a in x["lens"]]
        held = cache.read(first=first, fields=("k", "v"))
        cache.truncate(x["lens"])  # as a program does whose drafted tokens were refused
        return held
    if case["kind"] == "attend":
        # decay 0: the weights of this call alone
        out, lse = cache.attend(x["q"], counts=x["counts"], window=case["window"],
                                mask=x.get("mask"), decay=0.0 if case["track"] else None,
                                return_lse=True)
        res = {"out": out, "lse": lse}
        if case["track"]:
            res["weights"] = cache.read(fields=("weights",))["weights"]
        return res
    # the cut copy goes to sequences of its own; the long ones stay for other branches
    gone = cache.evict(case["budget"], case["recent"], seqs=range(n), into=range(n, 2 * n),
                       dropped=case["dropped"])
    res = cache.read(seqs=range(n, 2 * n))
    if case["dropped"]:
        res["dropped"] = gone
    cache.truncate([0] * n, seqs=range(n, 2 * n))
    return res


def work(case):
    lens, h, d = _lens(case), case["heads"], case["dim"]
    if case["kind"] == "append":
        new = _new(case)
        item = DTYPES[case["dtype"]].itemsize
        tail = sum(a % case["block"] for a in lens)  # what the touched blocks held
        touched = sum(new) + tail
        return {"bytes": 2 * h * d * (sum(new) * (item + 1) + tail + 4 * touched), "flops": 0}
    if case["kind"] == "evict":
        kept = sum(min(a, case["budget"]) for a in lens)
        gone = (sum(lens) - kept) if case["dropped"] else 0
        pad = (case["n"] * max(max(lens) - case["budget"], 0)) if case["dropped"] else 0
        return {"bytes": h * (4 * sum(lens) + kept * (2 * d * (1 + 1 + 4) + 16)
                              + gone * 2 * d + pad * (8 * d + 4)), "flops": 0}
    counts = _queries(case)
    item = DTYPES[case["dtype"]].itemsize
    heads_q = h * case["group"]
    seen, cached = 0, 0
    for n, m in zip(lens, counts):
        win = case["window"] or n
        full = [min(win, n - m + 1 + i) for i in (0, m - 1)]
        # visible slots summed over the call's tokens, and the slots that any of them sees
        if full[0] == full[1]:
            seen += m * full[0]
        else:
            seen += sum(min(win, n - m + 1 + i) for i in range(m))
        cached += min(n, win + m - 1)
    rows = sum(counts)
    nbytes = 2 * cached * h * d + rows * heads_q * (2 * d * item + 4)
    if case["masked"]:
        nbytes += seen
    if case["track"]:
        nbytes += 4 * sum(lens) * h * 2  # written, and read back
    return {"bytes": nbytes, "flops": 4 * seen * heads_q * d}


# ---- 64-bit references --------------------------------------------------------


def exact(case, seed):
    """The definitions in float64.  The stored codes and scales are part of the cache's
    format, which rounds in float32: they are made here slot block by slot block."""
    x = _inputs(case, seed)
    caches, at = [], 0
    for n in x["lens"]:
        caches.append([_Store(case, x[name][at:at + n]) for name in ("k", "v")])
        at += n
    if case["kind"] == "append":
        res, at = {"k": [], "v": []}, 0
        for pair, n, m in zip(caches, x["lens"], x["new"]):
            for store, name in zip(pair, ("k", "v")):
                store.add(x["new_" + name][at:at + m])
                res[name].append(store.read(n // case["block"] * case["block"]))
            at += m
        return {name: torch.cat(parts) for name, parts in res.items()}
    if case["kind"] == "attend":
        return _exact_attend(case, x, caches)
    return _exact_evict(case, x, caches)


class _Store:
    """One sequence's keys or values: a list of blocks, each (codes as float64, scale)."""

    def __init__(self, case, x):
        self.case, self.blocks, self.n = case, [], 0
        if x.shape[0]:
            self.add(x)

    def _code(self, y):
        if self.case["code"] == "int8":
            return torch.clamp(torch.round(y), -127, 127).double()
        return torch.clamp(y, -448, 448).to(torch.float8_e4m3fn).double()

    def add(self, x):
        b, z = self.case["block"], ZMAX[self.case["code"]]
        done = 0
        while done < x.shape[0]:
            room = b - self.n % b
            part = x[done:done + room].float()
            big = part.abs().amax(dim=2).amax(dim=0)
            s = torch.where(big >= TINY, big / z, big * 0)
            old = None
            if room < b:
                old, s_old = self.blocks.pop()
                s = torch.maximum(s, s_old)
                r = torch.where(s > 0, s_old / s, s * 0)
                old = self._code(old.float() * r[None, :, None])
            inv = torch.where(s > 0, torch.ones_like(s) / s, s * 0)
            c = self._code(part * inv[None, :, None])
            self.blocks.append((c if old is None else torch.cat([old, c]), s))
            done += part.shape[0]
            self.n += part.shape[0]

    def parts(self):
        """Codes [n, h, d] and each slot's scale [n, h]."""
        codes = torch.cat([c for c, _ in self.blocks])
        scale = torch.cat([s.double()[None].expand(c.shape[0], -1) for c, s in self.blocks])
        return codes, scale

    def read(self, first=0):
        codes, scale = self.parts()
        return (codes * scale[:, :, None])[first:]


def _exact_attend(case, x, caches):
    g, d = case["group"], case["dim"]
    if work(case)["flops"] > 2e12:
        return None
    outs, lses, ws, at = [], [], [], 0
    for (ks, vs), n, m in zip(caches, x["lens"], x["counts"]):
        k, v = ks.read(), vs.read()
        o = torch.zeros((m, case["heads"] * g, d), dtype=torch.float64, device=DEV)
        lse = torch.zeros((m, case["heads"] * g), dtype=torch.float64, device=DEV)
        w = torch.zeros((n, case["heads"]), dtype=torch.float64, device=DEV)
        slot = torch.arange(n, device=DEV)
        for head in range(case["heads"] * g):
            kv = head // g
            kt, vh = k[:, kv].T.contiguous(), v[:, kv].contiguous()
            for r0 in range(0, m, 1024):
                r1 = min(m, r0 + 1024)
                s = torch.mm(x["q"][at + r0:at + r1, head].double().contiguous(), kt) / math.sqrt(d)
                end = n - m + 1 + torch.arange(r0, r1, device=DEV)[:, None]
                hide = slot >= end
                if case["window"]:
                    hide = hide | (slot < end - case["window"])
                if case["masked"]:
                    hide = hide | ~x["mask"][at + r0:at + r1, :n]
                s[hide] = -math.inf
                z = torch.logsumexp(s, dim=1)
                p = torch.exp(s - torch.where(z == -math.inf, torch.zeros_like(z), z)[:, None])
                o[r0:r1, head] = torch.mm(p, vh)
                lse[r0:r1, head] = z
                w[:, kv] += p.sum(dim=0)
        outs.append(o)
        lses.append(lse)
        ws.append(w)
        at += m
    res = {"out": torch.cat(outs), "lse": torch.cat(lses)}
    if case["track"]:
        res["weights"] = torch.cat(ws)
    return res


def _exact_evict(case, x, caches):
    b, budget, recent, heads = case["block"], case["budget"], case["recent"], case["heads"]
    most = max(max(x["lens"]) - budget, 0)
    res = {name: [] for name in ("k", "v", "positions", "weights")}
    drop = {name: [] for name in ("k", "v", "positions")}
    at = 0
    for pair, n in zip(caches, x["lens"]):
        w = x["weights"][at:at + n]
        at += n
        cut = n > budget
        keep = torch.ones((n, heads), dtype=torch.bool, device=DEV)
        if cut:
            keep[:n - recent] = False
            # rank of a slot: how many come before it by (weight descending, slot ascending)
            order = torch.argsort(w[:n - recent].double().neg(), dim=0, stable=True)
            keep.scatter_(0, order[:budget - recent], True)
        size = min(n, budget)
        stay = torch.stack([keep[:, h].nonzero()[:, 0] for h in range(heads)], dim=1)
        gone = torch.stack([(~keep[:, h]).nonzero()[:, 0] for h in range(heads)], dim=1)
        for name, store in zip(("k", "v"), pair):
            codes, scale = store.parts()
            values = torch.empty((size, heads, case["dim"]), dtype=torch.float64, device=DEV)
            left = torch.zeros((most, heads, case["dim"]), dtype=torch.float64, device=DEV)
            for h in range(heads):
                s_old = scale[stay[:, h], h].float()
                for j in range(0, size, b):
                    part = s_old[j:j + b]
                    top = part.max()
                    c = codes[stay[j:j + b, h], h].float() * (part / top)[:, None]
                    if cut:
                        values[j:j + b, h] = store._code(c) * top.double()
                    else:
                        values[j:j + b, h] = codes[j:j + b, h] * scale[j:j + b, h, None]
                left[:n - size, h] = codes[gone[:, h], h] * scale[gone[:, h], h, None]
            res[name].append(values)
            drop[name].append(left)
        res["positions"].append(stay.to(torch.int32))
        res["weights"].append(torch.gather(w, 0, stay).double())
        at_drop = torch.full((most, heads), -1, dtype=torch.int32, device=DEV)
        at_drop[:n - size] = gone.to(torch.int32)
        drop["positions"].append(at_drop)
    out = {name: torch.cat(parts) for name, parts in res.items()}
    if case["dropped"]:
        out["dropped"] = {name: torch.stack(parts) for name, parts in drop.items()}
    return out
