"""Measured cases of the paged-cache operators: rotary positions written into the pages of a KV
cache, attention of new tokens over those pages, and the bookkeeping of the pages themselves.

Each case is one pass a decoder layer (or the scheduler between two steps) makes. ``run`` computes
it in plain torch operations, or through ``inference_performance_lab.kernels.extension`` where
``own`` is true; ``exact`` computes the same outputs in 64 bits from the definitions.

Head layouts: 28 query and 4 key heads of 128 are those of the served 7B architecture; the others
are generic.
"""

from __future__ import annotations

import math
import random

import torch

own = False

# --------------------------------------------------------------------------------------------
# cases


def listed() -> list[dict]:
    return [
        # Rotary positions of one decode step: 64 sequences, one token each, q rotated in place,
        # k rotated into the cache together with v. A launch this small is all latency.
        dict(name="rotary_decode", op="rotary", tokens=64, heads=28, kv_heads=4, dim=128, rot=128, neox=True,
             append=True, max_pos=32768, page=16, pages=512),
        # The same for a prefill step of 8192 tokens.
        dict(name="rotary_chunk", op="rotary", tokens=8192, heads=28, kv_heads=4, dim=128, rot=128, neox=True,
             append=True, max_pos=32768, page=16, pages=1024),
        # Interleaved pairs on half of the head, both tensors in place, an odd token count.
        dict(name="rotary_partial", op="rotary", tokens=2049, heads=32, kv_heads=8, dim=64, rot=32, neox=False,
             append=False, max_pos=8192, page=16, pages=16),
        # A single sequence decoding: the smallest attention call of an interactive session.
        dict(name="attention_decode_one", op="attention", decodes=1, chunks=0, new=1, lo=1027, hi=1027, heads=28,
             kv_heads=4, dim=128, page=16, window=0),
        # A full decode batch with contexts from one token to 8192: HBM-bound on the cache.
        dict(name="attention_decode_batch", op="attention", decodes=64, chunks=0, new=1, lo=1, hi=8192, heads=28,
             kv_heads=4, dim=128, page=16, window=0),
        # Four whole prompts of ragged, odd lengths.
        dict(name="attention_prompts", op="attention", decodes=0, chunks=4, new=2011, lo=1, hi=2011, heads=28,
             kv_heads=4, dim=128, page=16, window=0),
        # The last chunk of a long prompt: the largest call, bound by the matrix products.
        dict(name="attention_chunk_long", op="attention", decodes=0, chunks=1, new=2048, lo=16384, hi=16384, heads=28,
             kv_heads=4, dim=128, page=64, window=0),
        # A step that mixes 16 decoding sequences with one chunk of a prompt; heads of 64, a
        # sliding window.
        dict(name="attention_mixed", op="attention", decodes=16, chunks=1, new=509, lo=700, hi=4099, heads=32,
             kv_heads=8, dim=64, page=32, window=1024),
        # Between two steps of parallel sampling: four sequences end, four continue a common
        # prompt, each gets room for new tokens.
        dict(name="pages_turnover_small", op="turnover", rows=16, parents=2, children=4, tokens=519, grow=3, width=64,
             layers=2, kv_heads=4, dim=128, page=16, pages=512),
        # The same for a beam step over many sequences of long prompts, every layer's cache.
        dict(name="pages_turnover_large", op="turnover", rows=256, parents=16, children=96, tokens=2043, grow=17,
             width=144, layers=28, kv_heads=4, dim=128, page=64, pages=900),
        # Compaction after a few sequences of a small pool ended.
        dict(name="pages_compact_small", op="compact", rows=8, width=32, layers=2, kv_heads=4, dim=128, page=16,
             pages=256, live=100, moves=9),
        # Compaction of a fragmented pool over every layer's cache.
        dict(name="pages_compact_large", op="compact", rows=64, width=64, layers=28, kv_heads=4, dim=128, page=16,
             pages=2048, live=1500, moves=411),
    ]


def _log(rng: random.Random, lo: int, hi: int) -> int:
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 1)))))))


def draw(rng: random.Random) -> dict:
    kind = rng.choice(["rotary", "decode", "decode", "chunk", "chunk", "turnover", "compact"])
    heads, kv_heads, dim = rng.choice([(28, 4, 128), (32, 8, 128), (32, 8, 64), (16, 16, 64), (12, 2, 64), (16, 1, 96),
                                       (40, 8, 80)])
    page = rng.choice([16, 16, 32, 48, 64, 128])
    if kind == "rotary":
        tokens = _log(rng, 1, 8192)
        rot = rng.choice([dim, dim, dim // 2, 16])
        return dict(op="rotary", tokens=tokens, heads=heads, kv_heads=kv_heads, dim=dim, rot=rot,
                    neox=rng.random() < 0.6, append=rng.random() < 0.6, max_pos=_log(rng, 2048, 32768), page=page,
                    pages=tokens // page + 1 + _log(rng, 1, 256))
    if kind == "decode":
        hi = _log(rng, 1, 8192)
        return dict(op="attention", decodes=_log(rng, 1, 64), chunks=0, new=1, lo=_log(rng, 1, hi), hi=hi, heads=heads,
                    kv_heads=kv_heads, dim=dim, page=page, window=rng.choice([0, 0, 0, 127, 1000]))
    if kind == "chunk":
        chunks = rng.choice([1, 1, 2, 3])
        new = _log(rng, 2, 2048 // chunks)
        hi = _log(rng, new, 12000 // chunks)
        return dict(op="attention", decodes=rng.choice([0, 0, 1, 7]), chunks=chunks, new=new, lo=_log(rng, new, hi),
                    hi=hi, heads=min(heads, 32), kv_heads=kv_heads if heads <= 32 else 8, dim=dim, page=page,
                    window=rng.choice([0, 0, 0, 255, 1024]))
    layers = _log(rng, 1, 28)
    kv_heads = min(kv_heads, 8)
    if kind == "turnover":
        parents = _log(rng, 1, 16)
        children = _log(rng, 1, 96)
        tokens = _log(rng, 1, 2043)
        grow = _log(rng, 1, 64)
        per_row = -(-tokens // page)
        more = -(-(tokens + grow) // page) - tokens // page
        return dict(op="turnover", rows=parents + children + rng.randint(0, 64), parents=parents, children=children,
                    tokens=tokens, grow=grow, width=per_row + -(-grow // page) + rng.randint(1, 33), layers=min(layers, 12),
                    kv_heads=min(kv_heads, 4), dim=min(dim, 96), page=page,
                    pages=parents * per_row + children * (more + 1) + rng.randint(0, 300))
    pages = _log(rng, 16, 2048)
    live = rng.randint(1, pages - 1)
    moves = rng.randint(0, min(live, pages - live))
    width = rng.randint(1, 64)
    return dict(op="compact", rows=-(-live // width) + rng.randint(0, 8), width=width, layers=min(layers, 14),
                kv_heads=min(kv_heads, 4), dim=min(dim, 96), page=min(page, 32), pages=pages, live=live, moves=moves)


def _spread(i: int, lo: int, hi: int) -> int:
    """The i-th of a ragged set of lengths in lo..hi; the first is hi."""
    return hi - int((hi - lo + 1) * ((i * 0.6180339887498949) % 1.0))


def _lengths(case: dict) -> tuple[list[int], list[int]]:
    """New tokens and total length of every sequence: the decoding ones, then the chunks."""
    new = [1] * case["decodes"] + [_spread(i, max(1, case["new"] // 2), case["new"]) for i in range(case["chunks"])]
    total = [_spread(i, case["lo"], case["hi"]) for i in range(len(new))]
    return new, [max(n, t) for n, t in zip(new, total)]


# --------------------------------------------------------------------------------------------
# what a user's program has in hand before the call


def _cos_sin_table(rot: int, max_pos: int) -> torch.Tensor:
    frequency = 10000.0 ** (-torch.arange(0, rot, 2, dtype=torch.float64, device="cuda") / rot)
    angle = torch.arange(max_pos, dtype=torch.float64, device="cuda")[:, None] * frequency
    return torch.cat([angle.cos(), angle.sin()], dim=1).float()


def _ints(values, dtype=torch.int32) -> torch.Tensor:
    return torch.tensor(values, dtype=dtype, device="cuda")


def prepare(case: dict, seed: int) -> dict:
    g = torch.Generator(device="cuda").manual_seed(seed)

    def normal(*shape):
        return torch.randn(*shape, generator=g, device="cuda", dtype=torch.bfloat16)

    def shuffled(n):
        return torch.randperm(n, generator=g, device="cuda")

    s = {"case": case}
    page = case["page"]
    if case["op"] == "rotary":
        tokens, heads, kv_heads, dim = case["tokens"], case["heads"], case["kv_heads"], case["dim"]
        # q, k and v are views of one projection's output, as a decoder layer splits it.
        qkv = normal(tokens, heads + 2 * kv_heads, dim)
        s["q"], s["k"], s["v"] = qkv.split([heads, kv_heads, kv_heads], dim=1)
        s["positions"] = torch.randint(0, case["max_pos"], (tokens,), generator=g, device="cuda")
        s["table"] = _cos_sin_table(case["rot"], case["max_pos"])
        if case["append"]:
            s["kc"], s["vc"] = normal(2, case["pages"], page, kv_heads, dim).unbind(0)
            s["slots"] = shuffled(case["pages"] * page)[:tokens].contiguous()
            # Padding tokens of a captured batch are not written.
            s["slots"][::37] = -1
    elif case["op"] == "attention":
        new, total = _lengths(case)
        counts = [-(-t // page) for t in total]
        pages = sum(counts) + 7
        width = max(counts) + 1
        order = shuffled(pages)
        at = torch.arange(width, device="cuda")[None, :]
        count = _ints(counts, torch.int64)[:, None]
        first = torch.cumsum(count, 0) - count
        # Entries past a sequence's pages are not page numbers.
        s["tables"] = torch.where(at < count, order[torch.where(at < count, first + at, 0)], -1).int()
        s["kc"], s["vc"] = normal(2, pages, page, case["kv_heads"], case["dim"]).unbind(0)
        s["q"] = normal(sum(new), case["heads"], case["dim"]) * 1.5
        s["starts"] = _ints([sum(new[:i]) for i in range(len(new) + 1)])
        s["lens"] = _ints(total)
        s["max_new"], s["max_len"] = max(new), max(total)
        s["scale"] = case["dim"] ** -0.5
    else:
        layers, kv_heads, dim, pages = case["layers"], case["kv_heads"], case["dim"], case["pages"]
        store = normal(2 * layers, pages, page, kv_heads, dim)
        s["store"], s["caches"] = store, list(store.unbind(0))
        order = shuffled(pages)
        tables = torch.full((case["rows"], case["width"]), -1, device="cuda", dtype=torch.int64)
        if case["op"] == "turnover":
            parents, children, tokens = case["parents"], case["children"], case["tokens"]
            per_row = -(-tokens // page)
            rows = shuffled(case["rows"])
            s["parents"] = rows[:parents].repeat(-(-children // parents))[:children].int()
            s["children"] = rows[parents : parents + children].int()
            s["grown"] = s["children"]
            s["grown_lens"] = torch.full((children,), tokens + case["grow"], device="cuda", dtype=torch.int32)
            tables[rows[:parents], :per_row] = order[: parents * per_row].view(parents, per_row)
            # The sequences that end hold a page of their own each where the pool has one left.
            spare = min(children, pages - parents * per_row)
            tables[rows[parents : parents + spare], 0] = order[parents * per_row : parents * per_row + spare]
            lens = torch.zeros(case["rows"], device="cuda", dtype=torch.int64)
            lens[rows[:parents]] = tokens
            lens[rows[parents : parents + spare]] = 1
            s["lens"] = lens.int()
        else:
            # `moves` live pages lie above the first `live` ones, at random.
            live, moves, width = case["live"], case["moves"], case["width"]
            held = torch.cat([shuffled(live)[: live - moves], live + shuffled(pages - live)[:moves]])
            held = held[shuffled(live)]
            tables.view(-1)[:live] = held
        s["tables"] = tables.int()
        refs = torch.zeros(pages + 1, device="cuda", dtype=torch.int64)
        refs.index_add_(0, torch.where(tables < 0, pages, tables).view(-1), torch.ones_like(tables).view(-1))
        s["refs"] = refs[:pages].int()
    return s


# --------------------------------------------------------------------------------------------
# one pass


def _extension():
    import sys
    from pathlib import Path

    package = str(Path(__file__).resolve().parents[1] / "inference-performance-lab_b200")
    if package not in sys.path:
        sys.path.insert(0, package)
    from inference_performance_lab.kernels import extension

    return extension


_ops = None


def run(state: dict):
    global _ops
    if own and _ops is None:
        _ops = _extension()
    return _PASSES[state["case"]["op"]](state)


def _pass_rotary(s: dict):
    c = s["case"]
    if own:
        if c["append"]:
            _ops.rotary_embedding_cache(s["positions"], s["q"], s["k"], s["v"], s["table"], s["kc"], s["vc"], s["slots"],
                                        c["neox"])
        else:
            _ops.rotary_embedding(s["positions"], s["q"], s["k"], s["table"], c["neox"])
    else:
        cos, sin = s["table"][s["positions"]][:, None, :].chunk(2, dim=-1)
        q, k = _rotate(s["q"], cos, sin, c), _rotate(s["k"], cos, sin, c)
        s["q"].copy_(q)
        if c["append"]:
            # A token without a slot writes token 1's values to token 1's slot once more.
            keep = torch.where(s["slots"] >= 0, torch.arange(c["tokens"], device="cuda"), 1 if c["tokens"] > 1 else 0)
            if c["tokens"] > 1:
                slots = s["slots"][keep]
                page, offset = slots // c["page"], slots % c["page"]
                s["kc"][page, offset] = k[keep]
                s["vc"][page, offset] = s["v"][keep]
        else:
            s["k"].copy_(k)
    if c["append"]:
        return {"q": s["q"], "key_cache": s["kc"], "value_cache": s["vc"]}
    return {"q": s["q"], "k": s["k"]}


def _rotate(x, cos, sin, c):
    rot, x32 = c["rot"], x.float()
    head, rest = x32[..., :rot], x32[..., rot:]
    if c["neox"]:
        a, b = head.chunk(2, dim=-1)
        turned = torch.cat([a * cos - b * sin, b * cos + a * sin], dim=-1)
    else:
        a, b = head[..., 0::2], head[..., 1::2]
        turned = torch.stack([a * cos - b * sin, b * cos + a * sin], dim=-1).flatten(-2)
    return torch.cat([turned, rest], dim=-1).to(x.dtype)


def _pass_attention(s: dict):
    c = s["case"]
    if own:
        return _ops.paged_attention(s["q"], s["kc"], s["vc"], s["tables"], s["starts"], s["lens"], s["max_new"],
                                    s["max_len"], s["scale"], c["window"])
    group, page = c["heads"] // c["kv_heads"], c["page"]
    pages = -(-s["max_len"] // page)
    starts, lens = s["starts"].long(), s["lens"].long()
    count = starts[1:] - starts[:-1]
    batch = lens.numel()
    at = torch.arange(s["max_new"], device="cuda")
    valid = at < count[:, None]  # [batch, new]
    token = torch.where(valid, starts[:-1, None] + at, 0)
    q = s["q"][token].float().view(batch, -1, c["kv_heads"], group, c["dim"]).permute(0, 2, 1, 3, 4)
    table = s["tables"][:, :pages].long().clamp(min=0)
    keys = s["kc"][table].view(batch, pages * page, c["kv_heads"], c["dim"]).permute(0, 2, 1, 3).float()
    values = s["vc"][table].view(batch, pages * page, c["kv_heads"], c["dim"]).permute(0, 2, 1, 3).float()
    scores = q.flatten(2, 3) @ keys.transpose(-1, -2) * s["scale"]  # [batch, kv, new * group, keys]
    position = (lens - count)[:, None] + at
    key = torch.arange(pages * page, device="cuda")
    seen = (key <= position[..., None]) & (key < lens[:, None, None])
    if c["window"] > 0:
        seen &= key > position[..., None] - c["window"]
    seen = seen[:, None, :, None, :].expand(-1, -1, -1, group, -1).flatten(2, 3)
    scores = scores.masked_fill_(~seen, float("-inf"))
    top = scores.amax(-1, keepdim=True).clamp(min=torch.finfo(torch.float32).min)
    weights = scores.sub_(top).exp_()
    out = (weights @ values) / weights.sum(-1, keepdim=True).clamp(min=torch.finfo(torch.float32).tiny)
    out = out.view(batch, c["kv_heads"], s["max_new"], group, c["dim"]).permute(0, 2, 1, 3, 4).flatten(2, 3)
    return out[valid].to(s["q"].dtype)


def _pass_turnover(s: dict):
    c = s["case"]
    page = c["page"]
    if own:
        _ops.release_sequences(s["tables"], s["lens"], s["refs"], s["children"])
        short = _ops.fork_sequences(s["caches"], s["tables"], s["lens"], s["refs"], s["parents"], s["children"])
        lacking = _ops.reserve_pages(s["tables"], s["lens"], s["refs"], s["grown"], s["grown_lens"], page)
        return {"tables": s["tables"], "lens": s["lens"], "refs": s["refs"], "status": [short, lacking], "store": s["store"]}
    tables, lens, refs = s["tables"], s["lens"], s["refs"]
    parents, children = s["parents"].long(), s["children"].long()
    # Release: each page held by an ending sequence loses one reference.
    gone = tables[children].long()
    refs.scatter_add_(0, gone.clamp(min=0).view(-1), torch.where(gone >= 0, -1, 0).int().view(-1))
    tables[children] = -1
    lens[children] = 0
    # Fork: whole pages are shared, a page that is partly filled is copied to the lowest free one.
    length = lens[parents].long()
    whole = length // page
    at = torch.arange(c["width"], device="cuda")
    shared = torch.where(at < whole[:, None], tables[parents], -1)
    refs.scatter_add_(0, shared.long().clamp(min=0).view(-1), (shared >= 0).int().view(-1))
    partly = length % page > 0  # of all the parents or of none: they are of one length
    rank = torch.cumsum(partly, 0) - 1
    free = torch.argsort((refs != 0).int(), stable=True)
    fresh = free[rank.clamp(min=0)]
    source = tables[parents, whole.clamp(max=c["width"] - 1)].long()
    tables[children] = torch.where(partly[:, None] & (at == whole[:, None]), fresh[:, None].int(), shared)
    source, target = torch.where(partly, source, 0), torch.where(partly, fresh, 0)
    s["store"][:, target] = s["store"][:, source]
    refs.scatter_add_(0, target, partly.int())
    lens[children] = length.int()
    # Reserve: the pages that the new lengths reach, each the lowest that is free.
    grown, wanted = s["grown"].long(), s["grown_lens"].long()
    have, need = -(-lens[grown].long() // page), -(-wanted // page)
    more = (at >= have[:, None]) & (at < need[:, None])
    rank = (torch.cumsum(more.view(-1), 0) - 1).view_as(more)
    free = torch.argsort((refs != 0).int(), stable=True)
    fresh = free[rank.clamp(min=0, max=c["pages"] - 1)]
    tables[grown] = torch.where(more, fresh.int(), tables[grown])
    refs.scatter_add_(0, fresh.view(-1), more.int().view(-1))
    lens[grown] = torch.maximum(lens[grown], s["grown_lens"])
    zero = torch.zeros(1, device="cuda", dtype=torch.int32)
    return {"tables": tables, "lens": lens, "refs": refs, "status": [zero, zero], "store": s["store"]}


def _pass_compact(s: dict):
    if own:
        tables, refs, live = _ops.compact_pages(s["caches"], s["tables"], s["refs"])
        return {"tables": tables, "refs": refs, "live": live, "store": s["store"]}
    held = s["refs"] > 0
    live = held.sum()
    number = torch.arange(held.numel(), device="cuda")
    above, hole = held & (number >= live), ~held & (number < live)
    # The k-th live page past the first `live` ones goes to the k-th hole below; the others stay.
    by_hole = torch.argsort((~hole).int(), stable=True)
    place = torch.where(above, by_hole[(torch.cumsum(above, 0) - 1).clamp(min=0)], number)
    moves = s["case"]["moves"]
    source, target = torch.argsort((~above).int(), stable=True)[:moves], by_hole[:moves]
    s["store"][:, target] = s["store"][:, source]
    tables = torch.where(s["tables"] >= 0, place[s["tables"].long().clamp(min=0)].int(), s["tables"])
    refs = torch.where(above, 0, s["refs"])
    refs[target] = s["refs"][source]
    return {"tables": tables, "refs": refs, "live": live.int().view(1), "store": s["store"]}


_PASSES = {"rotary": _pass_rotary, "attention": _pass_attention, "turnover": _pass_turnover, "compact": _pass_compact}


# --------------------------------------------------------------------------------------------
# what a pass cannot do without


def _visible(new: int, total: int, window: int) -> int:
    """Sum over a sequence's new tokens of the keys each one sees."""
    seen = [min(p + 1, window) if window else p + 1 for p in (total - new, total - 1)]
    if window and total - new + 1 < window < total:
        short = window - (total - new) - 1
        return (seen[0] + window - 1) * short // 2 + window * (new - short)
    return (seen[0] + seen[1]) * new // 2


def work(case: dict) -> dict:
    page = case["page"]
    if case["op"] == "rotary":
        tokens, heads, kv_heads, dim, rot = (case[k] for k in ("tokens", "heads", "kv_heads", "dim", "rot"))
        table = min(tokens, case["max_pos"]) * rot * 4 + tokens * 8
        if case["append"]:
            written = tokens - -(-tokens // 37)
            moved = tokens * heads * 2 * rot * 2 + written * (4 * kv_heads * dim * 2 + 8)
        else:
            moved = tokens * (heads + kv_heads) * 2 * rot * 2
        return {"bytes": table + moved, "flops": 3 * tokens * (heads + kv_heads) * rot}
    if case["op"] == "attention":
        new, total = _lengths(case)
        heads, kv_heads, dim, window = (case[k] for k in ("heads", "kv_heads", "dim", "window"))
        keys = sum(min(t, window + n - 1) if window else t for n, t in zip(new, total))
        seen = sum(_visible(n, t, window) for n, t in zip(new, total))
        return {"bytes": keys * kv_heads * dim * 4 + sum(new) * heads * dim * 4 + -(-keys // page) * 4,
                "flops": 4 * seen * heads * dim}
    token_bytes = 2 * case["layers"] * case["kv_heads"] * case["dim"] * 2
    if case["op"] == "turnover":
        tokens, children = case["tokens"], case["children"]
        entries = tokens // page
        grown = -(-(tokens + case["grow"]) // page) - -(-tokens // page)
        tables = children * (entries * 4 * 4 + (1 + grown) * 8 + 16)
        return {"bytes": 2 * children * (tokens % page) * token_bytes + tables, "flops": 0}
    return {"bytes": 2 * case["moves"] * page * token_bytes + 8 * (case["rows"] * case["width"] + case["pages"]), "flops": 0}


# --------------------------------------------------------------------------------------------
# the definitions in 64 bits


def exact(case: dict, seed: int):
    s = prepare(case, seed)
    if case["op"] == "rotary":
        return _exact_rotary(case, s)
    if case["op"] == "attention":
        return _exact_attention(case, s)
    return None  # whole numbers and copies


def _exact_rotary(case: dict, s: dict):
    half = case["rot"] // 2
    table = s["table"][s["positions"]].double()
    turn = torch.complex(table[:, :half], table[:, half:])[:, None, :]

    def rotated(x):
        y = x.double()
        i = torch.arange(half, device="cuda")
        re, im = (i, i + half) if case["neox"] else (2 * i, 2 * i + 1)
        z = torch.complex(y[..., re], y[..., im]) * turn
        y[..., re], y[..., im] = z.real, z.imag
        return y

    if not case["append"]:
        return {"q": rotated(s["q"]), "k": rotated(s["k"])}
    kept = s["slots"] >= 0
    caches = []
    for cache, rows in ((s["kc"], rotated(s["k"])), (s["vc"], s["v"].double())):
        flat = cache.double().flatten(0, 1)
        flat[s["slots"][kept]] = rows[kept]
        caches.append(flat.view(cache.shape))
    return {"q": rotated(s["q"]), "key_cache": caches[0], "value_cache": caches[1]}


def _exact_attention(case: dict, s: dict):
    new, total = _lengths(case)
    group, page, window = case["heads"] // case["kv_heads"], case["page"], case["window"]
    out, first = [], 0
    for row, (n, t) in enumerate(zip(new, total)):
        pages = s["tables"][row, : -(-t // page)].long()
        q = s["q"][first : first + n].double()
        first += n
        result = torch.empty_like(q)
        for head in range(case["kv_heads"]):
            keys = s["kc"][pages, :, head].flatten(0, 1)[:t].double()
            values = s["vc"][pages, :, head].flatten(0, 1)[:t].double()
            behind = torch.arange(t - n, t, device="cuda")[:, None] - torch.arange(t, device="cuda")
            hidden = behind < 0
            if window:
                hidden |= behind >= window
            mine = slice(head * group, (head + 1) * group)
            logits = torch.einsum("ngd,td->gnt", q[:, mine], keys) * s["scale"]
            logits[:, hidden] = -torch.inf
            result[:, mine] = torch.einsum("gnt,td->ngd", torch.softmax(logits, -1), values)
        out.append(result)
    return torch.cat(out)
