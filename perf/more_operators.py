"""Operators for many continuations of one text, as cases that can be timed.

Sampling several answers and beam search work on sequences of a KVCache that begin
alike.  Three operators serve them:

  fork    sequences that continue others hold the same blocks; a block is copied when
          one of its holders writes into it, or at once (copy); blocks that nobody
          holds any more are free, and compact moves the used ones together;
  attend  softmax attention over sequences that share a prefix, read once for all;
  select  the best candidates of beams x vocabulary, with the rows that they continue.

The state that fork and compact leave behind is returned as the values that the 8-bit
codes stand for, through KVCache.read.
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
        # a step of beam search over a serving batch: every beam is replaced by the
        # continuation of one that was chosen, and one token joins it
        dict(name="fork_beams_step", kind="fork", prompts=8, width=8, prefix=3500, tail=75, new=1,
             heads=8, dim=128, block=64, code="int8", dtype="bfloat16"),
        # several users ask about one document, each a question of their own
        dict(name="fork_document_questions", kind="fork", prompts=1, width=5, prefix=50_001,
             tail=0, new=333, heads=8, dim=80, block=128, code="fp8", dtype="float32"),
        # a short conversation is copied as a whole
        dict(name="copy_short", kind="copy", n=1, longest=777, heads=5, dim=80, block=32,
             code="int8", compact=False),
        # long conversations are copied, the old ones leave, and what is left moves together
        dict(name="copy_compact", kind="copy", n=7, longest=30_011, heads=8, dim=128, block=64,
             code="fp8", compact=True),
        # four answers to one short prompt: latency
        dict(name="attend_samples", kind="attend", prompts=1, width=4, prefix=1500, own=60,
             queries=1, heads=4, group=4, dim=64, code="int8", dtype="bfloat16", block=64,
             window=0, masked=False),
        # the step of beam search over a serving batch
        dict(name="attend_beams", kind="attend", prompts=8, width=8, prefix=3500, own=75,
             queries=1, heads=8, group=4, dim=128, code="int8", dtype="bfloat16", block=64,
             window=0, masked=False),
        # a batch of conversations under one long instruction, each with a history of its own
        dict(name="attend_instruction", kind="attend", prompts=1, width=61, prefix=8192, own=2000,
             queries=1, heads=8, group=4, dim=128, code="int8", dtype="bfloat16", block=64,
             window=0, masked=False),
        # many answers about one long document
        dict(name="attend_document", kind="attend", prompts=1, width=48, prefix=65_536, own=500,
             queries=1, heads=8, group=8, dim=128, code="fp8", dtype="float16", block=128,
             window=0, masked=False),
        # float32 queries, a head each, an odd dimension, drafted tokens in two batches, a
        # window and a mask of the documents that the user may see
        dict(name="attend_draft_masked", kind="attend", prompts=2, width=9, prefix=4001, own=333,
             queries=5, heads=12, group=1, dim=80, code="int8", dtype="float32", block=32,
             window=2048, masked=True),
        # the first words of one prompt's beams: latency
        dict(name="select_one_prompt", kind="select", prompts=1, beams=4, vocab=32_000, k=8,
             dtype="float32", masked=False),
        # a serving batch, rows that begin at odd addresses
        dict(name="select_batch", kind="select", prompts=64, beams=8, vocab=100_003, k=16,
             dtype="bfloat16", masked=False),
        # wide beams under a grammar that forbids most tokens
        dict(name="select_wide_masked", kind="select", prompts=3, beams=48, vocab=65_536, k=96,
             dtype="float16", masked=True),
    ]


def _log_int(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    """One more case of the listed ones' ranges."""
    kind = rng.choice(["fork", "fork", "copy", "attend", "attend", "attend", "select", "select"])
    if kind == "select":
        prompts = _log_int(rng, 1, 64)
        beams = _log_int(rng, 1, max(1, min(64, 512 // prompts)))
        vocab = _log_int(rng, 100, min(150_000, 50_000_000 // (prompts * beams)))
        return dict(kind=kind, prompts=prompts, beams=beams, vocab=vocab,
                    k=rng.randint(1, min(128, beams * 4)), masked=rng.random() < 0.3,
                    dtype=rng.choice(["bfloat16", "bfloat16", "float16", "float32"]))
    case = dict(kind=kind, heads=rng.choice([1, 2, 4, 5, 8, 8, 12]),
                dim=rng.choice([40, 64, 64, 80, 96, 128, 128, 128, 192, 256]),
                block=rng.choice([32, 64, 64, 128]), code=rng.choice(["int8", "fp8"]))
    if kind == "copy":
        case["n"] = _log_int(rng, 1, 32)
        case["longest"] = _log_int(rng, 16, max(16, 200_000 // case["n"] // max(1, case["dim"] // 64)))
        case["compact"] = rng.random() < 0.5
        return _bounded(case, "longest")
    case["dtype"] = rng.choice(["bfloat16", "bfloat16", "float16", "float32"])
    case["prompts"] = rng.choice([1, 1, 2, _log_int(rng, 1, 8)])
    case["width"] = _log_int(rng, 2, 64 // case["prompts"])
    seqs = case["prompts"] * case["width"]
    if kind == "fork":
        case["prefix"] = _log_int(rng, 1, 50_000 // case["prompts"])
        case["tail"] = rng.choice([0, _log_int(rng, 1, 200)])
        case["new"] = 1 if rng.random() < 0.5 else _log_int(rng, 2, max(2, 4096 // seqs))
        return case
    case["prefix"] = _log_int(rng, 32, 65_536 // case["prompts"])
    case["group"] = rng.choice([1, 1, 2, 3, 4, 4, 7, 8])
    case["queries"] = rng.choice([1, 1, 1, rng.randint(2, 16), _log_int(rng, 17, max(17, 1024 // seqs))])
    case["own"] = max(case["queries"], _log_int(rng, 1, 2000))
    case["masked"] = rng.random() < 0.2
    case["window"] = rng.choice([0, 0, 0, _log_int(rng, 1, case["prefix"])])
    return _bounded(case, "prefix")


def _bounded(case, length):
    """The case, made shorter until it costs no more than the largest listed ones."""
    while work(case)["flops"] > 1e11 or work(case)["bytes"] > 9e8:
        case[length] = case[length] * 3 // 4
    return case


# ---- inputs ---------------------------------------------------------------


def _gen(seed, part):
    return torch.Generator(device=DEV).manual_seed(seed * 1000 + part)


def _spread(text, n, lo, longest):
    """n lengths from lo to longest, the longest one first (a plain function of its arguments)."""
    rng = random.Random(f"{text} {n} {lo} {longest}")
    return [longest] + [_log_int(rng, lo, longest) for _ in range(n - 1)]


def _prefixes(case):
    return _spread("prefix", case["prompts"], max(1, case["prefix"] // 4), case["prefix"])


def _own(case):
    """Tokens of its own of every sequence, prompt after prompt."""
    n = case["prompts"] * case["width"]
    if case["kind"] == "fork":
        return _spread("tail", n, max(1, case["tail"] // 4), case["tail"]) if case["tail"] else [0] * n
    return _spread("own", n, max(case["queries"], case["own"] // 8), case["own"])


def _new(case):
    n = case["prompts"] * case["width"]
    return [1] * n if case["new"] == 1 else _spread("new", n, max(1, case["new"] // 4), case["new"])


def _parents(case):
    """The beams that were chosen, each prompt's of its own; some more than once, some not."""
    p, w = case["prompts"], case["width"]
    rng = random.Random(f"parents {p} {w}")
    return [i * w + rng.randrange(w) for i in range(p) for _ in range(w)]


def _lens(case):
    return _spread("copy", case["n"], max(1, case["longest"] // 8), case["longest"])


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


def _inputs(case, seed):
    """What the caller holds, on the GPU: tokens as they were before quantisation, and the
    call's own tensors."""
    if case["kind"] == "select":
        return _logits(case, seed)
    dtype = DTYPES[case.get("dtype", "bfloat16")]
    h, d = case["heads"], case["dim"]
    if case["kind"] == "copy":
        lens = _lens(case)
        k, v = _tokens(sum(lens), h, d, seed, 1, dtype)
        w = torch.randn((sum(lens), h), generator=_gen(seed, 11), device=DEV).exp_()
        return {"lens": lens, "k": k, "v": v, "weights": w}
    x = {"prefix": _prefixes(case), "own": _own(case)}
    x["k"], x["v"] = _tokens(sum(x["prefix"]), h, d, seed, 1, dtype)
    x["own_k"], x["own_v"] = _tokens(sum(x["own"]), h, d, seed, 2, dtype)
    if case["kind"] == "fork":
        x["new"] = _new(case)
        nk, nv = _tokens(sum(x["new"]), h, d, seed, 4, dtype)
        # some of the new keys are larger than what their block held
        x["new_k"], x["new_v"] = nk * 1.25, nv
        x["parents"] = _parents(case)
        return x
    n, m, heads_q = len(x["own"]), case["queries"], h * case["group"]
    g = _gen(seed, 3)
    q = torch.randn((n * m, heads_q, d), generator=g, device=DEV)
    # each query row leans towards one key of its prompt
    start, size = [], []
    for p, length in enumerate(x["prefix"]):
        start += [sum(x["prefix"][:p])] * (case["width"] * m)
        size += [length] * (case["width"] * m)
    start, size = torch.tensor(start, device=DEV), torch.tensor(size, device=DEV)
    pick = start + (torch.rand((n * m,), generator=g, device=DEV) * size).long()
    near = x["k"][pick].float().repeat_interleave(case["group"], dim=1)
    x["q"] = (0.3 * q + 0.1 * near).to(dtype)
    if case["masked"]:
        # documents of 16 tokens that a user may see, one in eight of them not
        longest = max(_totals(case))
        see = torch.rand((n * m, (longest + 15) // 16), generator=g, device=DEV) >= 0.125
        x["mask"] = see.repeat_interleave(16, dim=1)[:, :longest].contiguous()
    return x


def _totals(case):
    w = case["width"]
    return [_prefixes(case)[i // w] + t for i, t in enumerate(_own(case))]


def _logits(case, seed):
    rows, vocab = case["prompts"] * case["beams"], case["vocab"]
    g = _gen(seed, 1)
    logits = torch.randn((rows, vocab), generator=g, device=DEV).mul_(2.5)
    # a few dozen likely tokens that the beams of a prompt have in common, more or less likely
    some = min(40, vocab)
    likely = torch.randint(0, vocab, (case["prompts"], some), generator=g, device=DEV)
    likely = likely.repeat_interleave(case["beams"], dim=0)
    lift = 8.0 + 4.0 * torch.rand((rows, some), generator=g, device=DEV)
    logits.scatter_(1, likely, lift)
    if case["masked"]:
        logits[torch.rand((rows, vocab), generator=g, device=DEV) < 0.9] = -math.inf
        logits[:, 0] = 0.0  # the end is always allowed
    scores = torch.rand((rows,), generator=g, device=DEV).mul_(-12.0)
    return {"logits": logits.to(DTYPES[case["dtype"]]), "scores": scores}


def prepare(case, seed):
    x = _inputs(case, seed)
    state = {"case": case, "x": x}
    if case["kind"] == "select":
        return state
    if own:
        state["cache"] = _fill(case, x, state)
    else:
        state["held"] = _hold(case, x)
    for name in ("k", "v", "own_k", "own_v", "weights"):
        if name in x:
            del x[name]
    return state


def _blocks_of(tokens, block):
    return -(-tokens // block)


def _fill(case, x, state):
    """The cache that the program has: prompts, and beams that continue them."""
    import vicinity_amd as va

    b = case["block"]
    if case["kind"] == "copy":
        n = case["n"]
        blocks = 2 * sum(_blocks_of(t, b) for t in x["lens"])
        cache = va.KVCache(2 * n, case["heads"], case["dim"], blocks, block_tokens=b, code=case["code"])
        cache.append(x["k"], x["v"], seqs=range(n), counts=x["lens"], weights=x["weights"])
        state["from"] = 0
        return cache
    n, p, w = len(x["own"]), case["prompts"], case["width"]
    more = x.get("new", [0] * n)
    # per sequence: its own tokens' blocks, a block that it no longer shares, and its child's
    blocks = sum(_blocks_of(t, b) for t in x["prefix"])
    blocks += sum(_blocks_of(a, b) + _blocks_of(c, b) + 3 for a, c in zip(x["own"], more))
    cache = va.KVCache(2 * n + p, case["heads"], case["dim"], blocks, block_tokens=b,
                       code=case["code"])
    prompts = range(2 * n, 2 * n + p)
    cache.append(x["k"], x["v"], seqs=prompts, counts=x["prefix"])
    cache.fork([2 * n + i // w for i in range(n)], range(n))
    if sum(x["own"]):
        cache.append(x["own_k"], x["own_v"], seqs=range(n), counts=x["own"])
    return cache


def _hold(case, x):
    """The same for the plain forms: each sequence's codes and scales."""
    held, at = [], 0
    if case["kind"] == "copy":
        for t in x["lens"]:
            w = x["weights"][at:at + t].clone()
            held.append(_grow(None, None, x["k"][at:at + t], case)
                        + _grow(None, None, x["v"][at:at + t], case) + (w,))
            at += t
        return held
    prompts = []
    for t in x["prefix"]:
        prompts.append(_grow(None, None, x["k"][at:at + t], case)
                       + _grow(None, None, x["v"][at:at + t], case))
        at += t
    at = 0
    for i, t in enumerate(x["own"]):
        kc, ks, vc, vs = prompts[i // case["width"]]
        if t:
            kc, ks = _grow(kc, ks, x["own_k"][at:at + t], case)
            vc, vs = _grow(vc, vs, x["own_v"][at:at + t], case)
        held.append((kc, ks, vc, vs))
        at += t
    return held


# ---- the plain forms --------------------------------------------------------


def _encode(x, code):
    if code == "int8":
        return x.round().clamp(-127.0, 127.0).to(torch.int8)
    return x.clamp(-448.0, 448.0).to(torch.float8_e4m3fn)


def _grow(codes, scales, x, case):
    """One sequence's codes [t, h, d] and scales [blocks, h] after x [m, h, d] joins it."""
    block, z = case["block"], ZMAX[case["code"]]
    held = 0 if codes is None else codes.shape[0]
    first = held // block * block
    x = x.float()
    m = x.shape[0]
    xb = torch.cat([x.new_zeros((held - first,) + x.shape[1:]), x])
    pad = -xb.shape[0] % block
    xb = torch.cat([xb, x.new_zeros((pad,) + x.shape[1:])]).view((-1, block) + x.shape[1:])
    amax = xb.abs().amax(dim=(1, 3))
    s = torch.where(amax >= TINY, amax / z, torch.zeros_like(amax))
    if held > first:
        s[0] = torch.maximum(s[0], scales[-1])
    inv = torch.where(s > 0, 1.0 / s, torch.zeros_like(s))
    new = _encode(xb * inv[:, None, :, None], case["code"])
    new = new.view((-1,) + x.shape[1:])[held - first:held - first + m]
    if held == 0:
        return new, s
    tail, keep = codes[first:], scales
    if held > first:
        ratio = torch.where(s[0] > 0, scales[-1] / s[0], torch.zeros_like(s[0]))
        tail, keep = _encode(tail.float() * ratio[None, :, None], case["code"]), scales[:-1]
    return _cat([codes[:first], tail, new]), torch.cat([keep, s])


def _cat(parts):
    if parts[0].dtype == torch.int8:
        return torch.cat(parts)
    return torch.cat([p.view(torch.uint8) for p in parts]).view(parts[0].dtype)


def _values(codes, scales, block):
    per_slot = scales.repeat_interleave(block, dim=0)[:codes.shape[0]]
    return codes.float() * per_slot[:, :, None]


def _plain_fork(state):
    """Each child is a copy of its parent's codes, which its new tokens then join."""
    case, x = state["case"], state["x"]
    out, at = {"k": [], "v": [], "positions": []}, 0
    for parent, m in zip(x["parents"], x["new"]):
        kc, ks, vc, vs = (t.clone() for t in state["held"][parent])
        first = kc.shape[0] // case["block"] * case["block"]
        kc, ks = _grow(kc, ks, x["new_k"][at:at + m], case)
        vc, vs = _grow(vc, vs, x["new_v"][at:at + m], case)
        out["k"].append(_values(kc, ks, case["block"])[first:])
        out["v"].append(_values(vc, vs, case["block"])[first:])
        slots = torch.arange(first, kc.shape[0], dtype=torch.int32, device=DEV)
        out["positions"].append(slots[:, None].expand(-1, case["heads"]))
        at += m
    return {name: torch.cat(parts) for name, parts in out.items()}


def _plain_copy(state):
    case = state["case"]
    out = {"k": [], "v": [], "positions": [], "weights": []}
    for held in state["held"]:
        kc, ks, vc, vs, w = (t.clone() for t in held)
        if case["compact"]:  # and once more, to where they stay
            kc, ks, vc, vs, w = (t.clone() for t in (kc, ks, vc, vs, w))
        out["k"].append(_values(kc, ks, case["block"]).to(torch.bfloat16))
        out["v"].append(_values(vc, vs, case["block"]).to(torch.bfloat16))
        slots = torch.arange(kc.shape[0], dtype=torch.int32, device=DEV)
        out["positions"].append(slots[:, None].expand(-1, case["heads"]))
        out["weights"].append(w)
    return {name: torch.cat(parts) for name, parts in out.items()}


def _plain_attend(state):
    case, x = state["case"], state["x"]
    g, d, m = case["group"], case["dim"], case["queries"]
    outs, lses = [], []
    for i, (kc, ks, vc, vs) in enumerate(state["held"]):
        n = kc.shape[0]
        k, v = _values(kc, ks, case["block"]), _values(vc, vs, case["block"])
        q = x["q"][i * m:i * m + m].float()
        slot = torch.arange(n, device=DEV)
        last = n - m + torch.arange(m, device=DEV)
        see = slot[None, :] <= last[:, None]
        if case["window"]:
            see &= slot[None, :] > last[:, None] - case["window"]
        if case["masked"]:
            see &= x["mask"][i * m:i * m + m, :n]
        # [heads, m * g, d] x [heads, d, n]
        qh = q.view(m, case["heads"], g, d).transpose(0, 1).reshape(case["heads"], m * g, d)
        kt, vh = k.permute(1, 2, 0).contiguous(), v.transpose(0, 1).contiguous()
        s = torch.bmm(qh, kt) * (1.0 / math.sqrt(d))
        s = s.view(-1, m, g, n).masked_fill_(~see[None, :, None, :], -math.inf)
        top = s.amax(dim=3, keepdim=True)
        top = torch.where(top == -math.inf, torch.zeros_like(top), top)
        p = torch.exp(s - top)
        total = p.sum(dim=3, keepdim=True)
        lses.append((top + torch.log(total))[..., 0].transpose(0, 1).reshape(m, -1))
        p = p / torch.where(total == 0, torch.ones_like(total), total)
        o = torch.bmm(p.view(-1, m * g, n), vh).view(-1, m, g, d)
        outs.append(o.transpose(0, 1).reshape(m, -1, d).to(x["q"].dtype))
    return {"out": torch.cat(outs), "lse": torch.cat(lses)}


def _plain_select(state):
    """Totals in 64 bits: candidates of different beams lie close together."""
    case, x = state["case"], state["x"]
    p, b, v = case["prompts"], case["beams"], case["vocab"]
    scores, parents, tokens = [], [], []
    for i in range(p):
        logits = x["logits"][i * b:i * b + b].double()
        top = logits.amax(dim=1, keepdim=True)
        lse = top + torch.log(torch.exp(logits - top).sum(dim=1, keepdim=True))
        total = (x["scores"][i * b:i * b + b, None].double() + (logits - lse)).view(-1)
        best, order = torch.sort(total, descending=True, stable=True)
        pick = order[:case["k"]]
        scores.append(best[:case["k"]].float())
        parents.append(i * b + pick // v)
        tokens.append(pick % v)
    return {"scores": torch.stack(scores), "parents": torch.stack(parents),
            "tokens": torch.stack(tokens)}


# ---- one pass ---------------------------------------------------------------


def run(state):
    case, x = state["case"], state["x"]
    kind = case["kind"]
    if not own:
        return {"fork": _plain_fork, "copy": _plain_copy, "attend": _plain_attend,
                "select": _plain_select}[kind](state)
    if kind == "select":
        import vicinity_amd as va

        scores, parents, tokens = va.select_beams(x["logits"], x["scores"], case["beams"], case["k"])
        return {"scores": scores, "parents": parents, "tokens": tokens}
    cache = state["cache"]
    if kind == "fork":
        n = len(x["new"])
        children = range(n, 2 * n)
        cache.fork(x["parents"], children)
        cache.append(x["new_k"], x["new_v"], seqs=children, counts=x["new"])
        at = _totals(case)
        first = [at[p] // case["block"] * case["block"] for p in x["parents"]]
        res = cache.read(seqs=children, first=first, fields=("k", "v", "positions"))
        cache.truncate([0] * n, seqs=children)  # the beams stay, as if the step were refused
        return res
    if kind == "copy":
        n, at = case["n"], state["from"]
        old, new = range(at, at + n), range(n - at, 2 * n - at)
        cache.fork(old, new, copy=True)
        if case["compact"]:
            cache.truncate([0] * n, seqs=old)
            cache.compact()
            state["from"] = n - at
            return cache.read(seqs=new, dtype=torch.bfloat16)
        res = cache.read(seqs=new, dtype=torch.bfloat16)
        cache.truncate([0] * n, seqs=new)
        return res
    n = len(x["own"])
    out, lse = cache.attend(x["q"], seqs=range(n), counts=[case["queries"]] * n,
                            window=case["window"], mask=x.get("mask"), return_lse=True)
    return {"out": out, "lse": lse}


def work(case):
    if case["kind"] == "select":
        rows = case["prompts"] * case["beams"]
        # a difference, an exponential, a sum and a comparison for each logit
        return {"bytes": rows * (case["vocab"] * DTYPES[case["dtype"]].itemsize + 4)
                + case["prompts"] * case["k"] * 20, "flops": 4 * rows * case["vocab"]}
    h, d, b = case["heads"], case["dim"], case["block"]
    if case["kind"] == "copy":
        # codes, scales, positions and weights in and out, and what is read back
        n = sum(_lens(case))
        return {"bytes": n * h * (2 * d * (1 + 1 + 2) + 24), "flops": 0}
    totals = _totals(case)
    item = DTYPES[case["dtype"]].itemsize
    if case["kind"] == "fork":
        # a chosen beam's last block goes in once, and out once for each of its children
        parents = _parents(case)
        chosen, new = sum(totals[i] % b for i in set(parents)), sum(_new(case))
        tails = sum(totals[i] % b for i in parents)
        return {"bytes": 2 * h * d * (chosen + tails + new * (item + 1) + 4 * (tails + new))
                + 4 * h * (tails + new), "flops": 0}
    m, w = case["queries"], case["width"]
    seen, cached = 0, 0
    for p, prefix in enumerate(_prefixes(case)):
        read = 0  # of the prefix, by the one that sees most of it
        for n in totals[p * w:p * w + w]:
            win = case["window"] or n
            seen += sum(min(win, n - m + 1 + i) for i in range(m))
            lo = max(n - m + 1 - win, 0)
            read = max(read, prefix - lo)
            cached += n - max(lo, prefix)
        cached += max(read, 0)
    heads_q = h * case["group"]
    nbytes = 2 * cached * h * d + len(totals) * m * heads_q * (2 * d * item + 4)
    if case["masked"]:
        nbytes += seen
    return {"bytes": nbytes, "flops": 4 * seen * heads_q * d}


# ---- 64-bit references --------------------------------------------------------


def exact(case, seed):
    """The definitions in float64.  The stored codes and scales are part of the cache's
    format, which rounds in float32: they are made here slot block by slot block."""
    x = _inputs(case, seed)
    kind = case["kind"]
    if kind == "select":
        return _exact_select(case, x)
    if kind == "copy":
        res, at = {"k": [], "v": [], "positions": []}, 0
        for n in x["lens"]:
            for name in ("k", "v"):
                st = _Store(case)
                st.add(x[name][at:at + n])
                res[name].append(st.read())
            res["positions"].append(_slots(0, n, case["heads"]))
            at += n
        out = {name: torch.cat(parts) for name, parts in res.items()}
        out["weights"] = x["weights"].double()
        return out
    prompts, at = [], 0
    for n in x["prefix"]:
        pair = _Store(case), _Store(case)
        pair[0].add(x["k"][at:at + n])
        pair[1].add(x["v"][at:at + n])
        prompts.append(pair)
        at += n
    ends = [sum(x["own"][:i]) for i in range(len(x["own"]) + 1)]

    def beam(i):
        pair = [st.twin() for st in prompts[i // case["width"]]]
        for st, name in zip(pair, ("own_k", "own_v")):
            st.add(x[name][ends[i]:ends[i + 1]])
        return pair

    if kind == "attend":
        return _exact_attend(case, x, beam)
    res, at = {"k": [], "v": [], "positions": []}, 0
    for parent, m in zip(x["parents"], x["new"]):
        pair = beam(parent)
        first = pair[0].n // case["block"] * case["block"]
        for st, name in zip(pair, ("k", "v")):
            st.add(x["new_" + name][at:at + m])
            res[name].append(st.read(first))
        res["positions"].append(_slots(first, pair[0].n, case["heads"]))
        at += m
    return {name: torch.cat(parts) for name, parts in res.items()}


def _slots(first, end, heads):
    return torch.tensor(range(first, end), dtype=torch.int32, device=DEV)[:, None].repeat(1, heads)


class _Store:
    """One sequence's keys or values: a list of blocks, each (codes as float64, scale)."""

    def __init__(self, case):
        self.case, self.blocks, self.n = case, [], 0
        self.done = None  # the values of the first blocks, which twins share

    def twin(self):
        other = _Store(self.case)
        other.blocks, other.n = list(self.blocks), self.n
        full = self.n // self.case["block"]
        if self.done is None:
            self.done = self._join(self.blocks[:full]) if full else None
        other.done = self.done
        return other

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

    @staticmethod
    def _join(blocks):
        return torch.cat([c * s.double()[None, :, None] for c, s in blocks])

    def read(self, first=0):
        skip = first // self.case["block"]
        if skip or self.done is None:
            return self._join(self.blocks[skip:])[first - skip * self.case["block"]:]
        rest = self.blocks[self.done.shape[0] // self.case["block"]:]
        return torch.cat([self.done, self._join(rest)]) if rest else self.done


def _exact_attend(case, x, beam):
    g, d, m = case["group"], case["dim"], case["queries"]
    if work(case)["flops"] > 2e12:
        return None
    outs, lses = [], []
    for i in range(len(x["own"])):
        k, v = (st.read() for st in beam(i))
        n = k.shape[0]
        q = x["q"][i * m:i * m + m].double()
        end = n - m + 1 + torch.arange(m, device=DEV)[:, None]
        slot = torch.arange(n, device=DEV)
        hide = slot >= end
        if case["window"]:
            hide = hide | (slot < end - case["window"])
        if case["masked"]:
            hide = hide | ~x["mask"][i * m:i * m + m, :n]
        out = torch.zeros((m, case["heads"] * g, d), dtype=torch.float64, device=DEV)
        lse = torch.zeros((m, case["heads"] * g), dtype=torch.float64, device=DEV)
        rows = hide.repeat_interleave(g, dim=0)
        for head in range(case["heads"]):
            qh = q[:, head * g:head * g + g].reshape(m * g, d)
            s = torch.mm(qh, k[:, head].T.contiguous()) / math.sqrt(d)
            s[rows] = -math.inf
            z = torch.logsumexp(s, dim=1)
            p = torch.exp(s - torch.where(z == -math.inf, torch.zeros_like(z), z)[:, None])
            out[:, head * g:head * g + g] = torch.mm(p, v[:, head].contiguous()).view(m, g, d)
            lse[:, head * g:head * g + g] = z.view(m, g)
        outs.append(out)
        lses.append(lse)
    return {"out": torch.cat(outs), "lse": torch.cat(lses)}


def _exact_select(case, x):
    """The k best one after the other: the largest total, of equal ones the first."""
    p, b, v = case["prompts"], case["beams"], case["vocab"]
    logits = x["logits"].double()
    logp = logits - torch.logsumexp(logits, dim=1, keepdim=True)
    total = (logp + x["scores"].double()[:, None]).view(p, b * v)
    scores = torch.empty((p, case["k"]), dtype=torch.float64, device=DEV)
    at = torch.empty((p, case["k"]), dtype=torch.int64, device=DEV)
    place = torch.arange(b * v, device=DEV)
    for j in range(case["k"]):
        best = total.amax(dim=1, keepdim=True)
        first = torch.where(total == best, place, b * v).amin(dim=1, keepdim=True)
        scores[:, j:j + 1], at[:, j:j + 1] = best, first
        total.scatter_(1, first, -math.inf)
    base = torch.arange(p, device=DEV)[:, None] * b
    return {"scores": scores, "parents": base + at // v, "tokens": at % v}
