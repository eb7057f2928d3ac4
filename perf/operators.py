"""Measured cases of the serving operators: rotary positions, the paged K/V cache and the attention over it.

Four operators, all head_dim 64 and bf16 like the rest of the framework:

``rope``    rotation of Q and K by positions with one to three axes, forward and backward
``append``  new K and V, K rotated, into the pages of a cache, and the rotated Q beside them
``paged``   attention of new tokens (one to thousands a sequence) over a paged cache
``prefix``  the same for a batch whose sequences share one long prefix

``own`` chooses between the plain torch forms and the framework's calls.
"""
import math

import numpy as np
import torch

own = False

D = 64
BF16 = torch.bfloat16


# ------------------------------------------------------------------ the cases

def listed():
    return [
        # One decode step of a small batch: a few hundred rows, all latency.
        dict(name="rope_step", op="rope", tokens=16, hq=8, hk=2, rot=64, axes=1, pairs=0, train=0, max_pos=8192),
        # A training batch of images and video: time, height and width positions, both directions.
        dict(name="rope_train_3axes", op="rope", tokens=30011, hq=16, hk=16, rot=64, axes=3, pairs=0, train=1, max_pos=8192),
        # The cache update of one decode step.
        dict(name="append_step", op="append", batch=48, new_lo=1, new_hi=1, ctx_lo=60, ctx_hi=700, hq=32, hk=8, page=16,
             rot=64, axes=1, pairs=0, ragged=0, max_pos=8192),
        # Prompts of odd lengths entering the cache, with image positions.
        dict(name="append_prompts", op="append", batch=12, new_lo=301, new_hi=4099, ctx_lo=0, ctx_hi=300, hq=16, hk=4, page=64,
             rot=64, axes=3, pairs=0, ragged=1, max_pos=8192),
        # One user, short context, one token: the least that a step can cost.
        dict(name="decode_one", op="paged", batch=1, new_lo=1, new_hi=1, ctx_lo=776, ctx_hi=776, hq=8, hk=2, page=16, ragged=0,
             causal=1, lse=0),
        # A serving batch in its decode phase, contexts of very different lengths.
        dict(name="decode_batch", op="paged", batch=64, new_lo=1, new_hi=1, ctx_lo=100, ctx_hi=4095, hq=32, hk=8, page=16,
             ragged=0, causal=1, lse=0),
        # Few users with very long contexts, a K/V head for each query head.
        dict(name="decode_long", op="paged", batch=4, new_lo=1, new_hi=1, ctx_lo=39999, ctx_hi=130001, hq=16, hk=16, page=64,
             ragged=0, causal=1, lse=1),
        # Several drafted tokens a sequence checked at once, six query heads a K/V head.
        dict(name="verify_drafts", op="paged", batch=24, new_lo=5, new_hi=5, ctx_lo=200, ctx_hi=3001, hq=24, hk=4, page=32,
             ragged=0, causal=1, lse=0),
        # Chunks of prompts over what is cached already: work of the matrix units.
        dict(name="prompt_chunks", op="paged", batch=6, new_lo=513, new_hi=2048, ctx_lo=0, ctx_hi=8191, hq=16, hk=4, page=64,
             ragged=1, causal=1, lse=1),
        # A handful of requests under one system prompt.
        dict(name="prefix_few", op="prefix", batch=6, new_lo=1, new_hi=1, prefix=1000, ctx_lo=0, ctx_hi=60, hq=8, hk=2, page=16,
             ragged=0, lse=0),
        # A serving batch under one long prompt.
        dict(name="prefix_batch", op="prefix", batch=64, new_lo=1, new_hi=1, prefix=8192, ctx_lo=31, ctx_hi=511, hq=32, hk=8,
             page=32, ragged=0, lse=0),
        # Many samples drawn from one document.
        dict(name="prefix_wide", op="prefix", batch=192, new_lo=1, new_hi=1, prefix=24577, ctx_lo=15, ctx_hi=1023, hq=32, hk=4,
             page=64, ragged=0, lse=1),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    heads = [(8, 8), (8, 2), (16, 16), (16, 4), (24, 4), (24, 8), (32, 8), (32, 4), (32, 32), (12, 1), (10, 2)]
    most_bytes, most_flops, most_cells = 1.6e9, 1.18e11, 1.0e9  # the largest listed ones', and 4 GB of plain scores
    while True:
        op = rng.choice(["rope", "append", "paged", "paged", "prefix"])
        hq, hk = rng.choice(heads)
        page = rng.choice([8, 16, 32, 64, 128])
        if op == "rope":
            c = dict(op=op, tokens=_log_int(rng, 1, 30000), hq=hq, hk=hk, rot=rng.choice([32, 64, 64]), axes=rng.choice([1, 2, 3]),
                     pairs=rng.choice([0, 1]), train=rng.choice([0, 1]), max_pos=8192)
        elif op == "append":
            new = rng.choice([1, 1, _log_int(rng, 2, 4000)])
            ctx = _log_int(rng, 1, 2000)
            c = dict(op=op, batch=_log_int(rng, 1, 200), new_lo=max(1, new // 5), new_hi=new, ctx_lo=ctx // 4, ctx_hi=ctx, hq=hq,
                     hk=hk, page=page, rot=rng.choice([32, 64, 64]), axes=rng.choice([1, 2, 3]), pairs=rng.choice([0, 1]),
                     ragged=int(new > 1), max_pos=8192)
        elif op == "paged":
            new = rng.choice([1, 1, rng.randint(2, 12), _log_int(rng, 13, 2000)])
            ctx = _log_int(rng, 1, 130000)
            ragged = int(new > 12) or rng.choice([0, 1])
            c = dict(op=op, batch=_log_int(rng, 1, 200), new_lo=max(1, new // 4) if ragged else new, new_hi=new, ctx_lo=ctx // 6,
                     ctx_hi=ctx, hq=hq, hk=hk, page=page, ragged=ragged, causal=rng.choice([1, 1, 0]), lse=rng.choice([0, 1]))
        else:
            new = rng.choice([1, 1, 1, rng.randint(2, 6)])
            ctx = _log_int(rng, 1, 1500)
            c = dict(op=op, batch=_log_int(rng, 2, 200), new_lo=new, new_hi=new, prefix=_log_int(rng, 100, 32000), ctx_lo=ctx // 5,
                     ctx_hi=ctx, hq=hq, hk=hk, page=page, ragged=rng.choice([0, 1]), lse=rng.choice([0, 1]))
        w = work(c)
        cells = 0 if op in ("rope", "append") else c["batch"] * c["new_hi"] * hq * (c["ctx_hi"] + c["new_hi"] + c.get("prefix", 0))
        if w["bytes"] <= most_bytes and w["flops"] <= most_flops and cells <= most_cells:
            return c


def _lengths(case):
    """(new tokens, keys with the new ones) of every sequence: part of the case, the same for every seed."""
    r = np.random.default_rng(case["batch"] * 1000003 + case["ctx_hi"] * 31 + case["new_hi"])
    n = case["batch"]
    new = r.integers(case["new_lo"], case["new_hi"] + 1, n)
    lo, hi = case["ctx_lo"] + 1, case["ctx_hi"] + 1
    ctx = np.floor(np.exp(r.uniform(np.log(lo), np.log(hi), n))).astype(np.int64) - 1 if hi > 8 * lo else r.integers(lo, hi + 1, n) - 1
    ctx[r.integers(0, n)] = case["ctx_hi"]
    return new, ctx + new


def work(case):
    hq, hk = case["hq"], case["hk"]
    if case["op"] == "rope":
        t, n = case["tokens"], 1 + case["train"]
        # Q and K read and written once a direction, the positions, and the table's rows that they name (at most all of it).
        rows = min(t, case["max_pos"])
        return {"bytes": n * (4 * t * (hq + hk) * D + 4 * t * case["axes"] + 4 * rows * case["rot"]),
                "flops": n * 3 * t * (hq + hk) * case["rot"]}
    new, keys = _lengths(case)
    t, total = int(new.sum()), int(keys.sum())
    if case["op"] == "append":
        return {"bytes": 4 * t * (hq + 2 * hk) * D + 4 * t * case["axes"] + 4 * min(t, case["max_pos"]) * case["rot"]
                + 4 * int((-(-keys // case["page"]) - (keys - new) // case["page"]).sum()),
                "flops": 3 * t * (hq + hk) * case["rot"]}
    out = 4 * t * hq * D + 4 * t * hq * case["lse"]
    pairs = int((new * keys - (new * (new - 1) // 2 if case.get("causal", 1) else 0)).sum())
    if case["op"] == "prefix":
        total += case["prefix"]
        pairs += t * case["prefix"]
    return {"bytes": out + 4 * total * hk * D + 4 * (total // case["page"]), "flops": 4 * pairs * hq * D}


# ------------------------------------------------------------------ inputs

def _sections(case):
    """Rotated pairs of each axis, in order: an even share, what is over to the last ones."""
    n, a = case["rot"] // 2, case["axes"]
    return tuple(n // a + (1 if i >= a - n % a else 0) for i in range(a))


def prepare(case, seed):
    dev = torch.device("cuda")
    g = torch.Generator(device=dev)
    g.manual_seed(seed)

    def normal(*shape, by=1.0):
        return (torch.randn(*shape, generator=g, device=dev) * by).to(BF16)

    s = dict(case, sections=_sections(case) if "axes" in case else None)
    if "axes" in case:
        # cos and sin of every position, made once in 64 bits.
        n = case["rot"] // 2
        angle = torch.arange(case["max_pos"], device=dev, dtype=torch.float64)[:, None] * (
            10000.0 ** (-torch.arange(n, device=dev, dtype=torch.float64) / n))
        s["table"] = torch.cat([angle.cos(), angle.sin()], 1).float().contiguous()
    if case["op"] == "rope":
        t = case["tokens"]
        s["q"], s["k"] = normal(t, case["hq"], D), normal(t, case["hk"], D)
        s["positions"] = torch.randint(0, case["max_pos"], (case["axes"], t), generator=g, device=dev, dtype=torch.int32)
        if case["train"]:
            s["dq"], s["dk"] = normal(t, case["hq"], D), normal(t, case["hk"], D)
        return s
    new, keys = _lengths(case)
    b, t, page, hk = case["batch"], int(new.sum()), case["page"], case["hk"]
    need = -(-int(keys.max()) // page)
    extra = -(-case.get("prefix", 0) // page)
    pages = torch.randperm(b * need + extra, generator=g, device=dev).to(torch.int32)
    s["page_table"] = pages[: b * need].view(b, need)
    if extra:
        s["prefix_pages"] = pages[b * need:].contiguous()
    s["k_cache"], s["v_cache"] = normal(b * need + extra, page, hk, D), normal(b * need + extra, page, hk, D)
    s["keys"] = torch.tensor(keys, device=dev, dtype=torch.int32)
    s["max_new"] = int(new.max())
    if case["ragged"]:
        s["starts"] = torch.tensor(np.concatenate([[0], np.cumsum(new)]), device=dev, dtype=torch.int32)
        lead = (t,)
    else:
        s["starts"] = None
        lead = (b, int(new.max()))
    # Queries a little sharper than keys: scores with a standard deviation of 1.5.
    s["q"] = normal(*lead, case["hq"], D, by=1.5)
    if case["op"] == "append":
        s["k"], s["v"] = normal(*lead, hk, D), normal(*lead, hk, D)
        s["positions"] = None
        if case["axes"] > 1:
            s["positions"] = torch.randint(0, case["max_pos"], (case["axes"], *lead), generator=g, device=dev, dtype=torch.int32)
    return s


# ------------------------------------------------------------------ the plain forms

def _rotate(x, table, positions, sections, pairs, sign):
    """x [..., heads, 64] by positions [axes, ...], 32 bits, not rounded."""
    n = table.shape[1] // 2
    j = torch.arange(n, device=x.device)
    bounds = torch.tensor(np.cumsum(sections), device=x.device)
    at = positions.long()[torch.bucketize(j, bounds, right=True)].movedim(0, -1)
    cos, sin = table[at, j].unsqueeze(-2), table[at, j + n].unsqueeze(-2) * sign
    x = x.float()
    a, b = (x[..., 0:2 * n:2], x[..., 1:2 * n:2]) if pairs else (x[..., :n], x[..., n:2 * n])
    u, w = a * cos - b * sin, a * sin + b * cos
    y = torch.stack([u, w], -1).flatten(-2) if pairs else torch.cat([u, w], -1)
    return torch.cat([y, x[..., 2 * n:]], -1)


def _places(s):
    """For each new token its sequence, its number there and its place in the cache."""
    keys = s["keys"].long()
    if s["starts"] is None:
        b, n = s["q"].shape[:2]
        seq, i = torch.arange(b, device=keys.device)[:, None], torch.arange(n, device=keys.device)[None, :]
        return seq, i, keys[:, None] - n + i
    starts = s["starts"].long()
    t = torch.arange(s["q"].shape[0], device=keys.device)
    seq = torch.bucketize(t, starts[1:], right=True)
    i = t - starts[seq]
    return seq, i, keys[seq] - (starts[seq + 1] - starts[seq]) + i


def _plain_rope(s):
    f = (s["table"], s["positions"], s["sections"], s["pairs"])
    out = [_rotate(s["q"], *f, 1.0).to(BF16), _rotate(s["k"], *f, 1.0).to(BF16)]
    if s["train"]:
        out += [_rotate(s["dq"], *f, -1.0).to(BF16), _rotate(s["dk"], *f, -1.0).to(BF16)]
    return out


def _plain_append(s):
    seq, i, place = _places(s)
    p = s["positions"] if s["positions"] is not None else place.expand(1, *s["q"].shape[:-2])
    page = s["page_table"][seq, place // s["page"]].long()
    q = _rotate(s["q"], s["table"], p, s["sections"], s["pairs"], 1.0).to(BF16)
    s["k_cache"][page, place % s["page"]] = _rotate(s["k"], s["table"], p, s["sections"], s["pairs"], 1.0).to(BF16)
    s["v_cache"][page, place % s["page"]] = s["v"]
    return [q, s["k_cache"], s["v_cache"]]


def _plain_attention(s):
    hq, hk = s["hq"], s["hk"]
    seq, i, place = _places(s)
    q = s["q"]
    if s["starts"] is not None:  # padded to the longest
        b, n = s["batch"], s["max_new"]
        full = torch.zeros(b, n, hq, D, device=q.device)
        full[seq, i] = q.float()
        last = torch.full((b, n), -1, device=q.device, dtype=torch.long)
        last[seq, i] = place
    else:
        full, last = q.float(), place
    b, n = full.shape[:2]
    full = full.view(b, n, hk, hq // hk, D) * (D ** -0.5)
    k = s["k_cache"][s["page_table"].long()].flatten(1, 2).float()
    v = s["v_cache"][s["page_table"].long()].flatten(1, 2).float()
    j = torch.arange(k.shape[1], device=q.device)
    if s.get("causal", 1):
        seen = j <= last[..., None]
    else:
        seen = (j < s["keys"].long()[:, None, None]) & (last[..., None] >= 0)
    scores = torch.einsum("bnhgd,bkhd->bhgnk", full, k).masked_fill_(~seen[:, None, None], -math.inf)
    top = scores.amax(-1, keepdim=True)
    if s["op"] == "prefix":  # its keys once for all
        pk = s["k_cache"][s["prefix_pages"].long()].flatten(0, 1)[: s["prefix"]].float()
        pv = s["v_cache"][s["prefix_pages"].long()].flatten(0, 1)[: s["prefix"]].float()
        first = torch.einsum("bnhgd,khd->bhgnk", full, pk)
        top = torch.maximum(top, first.amax(-1, keepdim=True))
    top = top.clamp_min(-1e30)
    p = torch.exp(scores.sub_(top))
    total = p.sum(-1, keepdim=True)
    o = torch.einsum("bhgnk,bkhd->bhgnd", p, v)
    if s["op"] == "prefix":
        p = torch.exp(first.sub_(top))
        total = total + p.sum(-1, keepdim=True)
        o = o + torch.einsum("bhgnk,khd->bhgnd", p, pv)
    o = torch.where(total > 0, o / total, 0.0).permute(0, 3, 1, 2, 4).reshape(b, n, hq, D)
    out = [(o if s["starts"] is None else o[seq, i]).to(BF16)]
    if s["lse"]:
        lse = (top + total.log()).view(b, hq, n)
        out.append(lse if s["starts"] is None else lse[seq, :, i].t().contiguous())
    return out


# ------------------------------------------------------------------ the framework's calls

def _own_rope(s):
    import fmha_native_b200 as fm
    f = dict(sections=s["sections"], interleaved=bool(s["pairs"]))
    out = list(fm.rope(s["q"], s["k"], s["table"], s["positions"], **f))
    if s["train"]:
        out += fm.rope_bwd(s["dq"], s["dk"], s["table"], s["positions"], **f)
    return out


def _own_append(s):
    import fmha_native_b200 as fm
    q = fm.paged_append(s["k"], s["v"], s["k_cache"], s["v_cache"], s["page_table"], s["keys"], q=s["q"], cos_sin=s["table"],
                        positions=s["positions"], sections=s["sections"], interleaved=bool(s["pairs"]), cu_seqlens_q=s["starts"])
    return [q, s["k_cache"], s["v_cache"]]


def _own_attention(s):
    import fmha_native_b200 as fm
    if s["op"] == "prefix":
        out = fm.prefix_fwd(s["q"], s["k_cache"], s["v_cache"], s["prefix_pages"], s["prefix"], s["page_table"], s["keys"],
                            return_lse=bool(s["lse"]), cu_seqlens_q=s["starts"], max_seqlen_q=s["max_new"])
    else:
        out = fm.paged_fwd(s["q"], s["k_cache"], s["v_cache"], s["page_table"], s["keys"], causal=bool(s["causal"]),
                           return_lse=bool(s["lse"]), cu_seqlens_q=s["starts"], max_seqlen_q=s["max_new"])
    return list(out) if s["lse"] else [out]


def run(state):
    if own:
        f = {"rope": _own_rope, "append": _own_append}.get(state["op"], _own_attention)
    else:
        f = {"rope": _plain_rope, "append": _plain_append}.get(state["op"], _plain_attention)
    return f(state)


# ------------------------------------------------------------------ 64 bits

def exact(case, seed):
    s = prepare(case, seed)
    f64 = torch.float64

    def turn(x, positions, sign):
        # pair by pair: (a, b) -> (a cos - b sin, a sin + b cos)
        y, n = x.to(f64).clone(), s["rot"] // 2
        axis = [a for a, m in enumerate(s["sections"]) for _ in range(m)]
        for j in range(n):
            lo, hi = (2 * j, 2 * j + 1) if s["pairs"] else (j, j + n)
            row = s["table"][positions[axis[j]].long()]
            c, d = row[..., j].to(f64)[..., None], sign * row[..., j + n].to(f64)[..., None]
            a, b = x[..., lo].to(f64), x[..., hi].to(f64)
            y[..., lo], y[..., hi] = a * c - b * d, a * d + b * c
        return y

    if s["op"] == "rope":
        out = [turn(s["q"], s["positions"], 1.0), turn(s["k"], s["positions"], 1.0)]
        return out + [turn(s["dq"], s["positions"], -1.0), turn(s["dk"], s["positions"], -1.0)] if s["train"] else out
    new, keys = _lengths(case)
    page, lead = s["page"], s["q"].shape[:-2]
    q = s["q"].flatten(0, len(lead) - 1)
    begin = np.concatenate([[0], np.cumsum(new)])
    if s["op"] == "append":
        place = torch.cat([torch.arange(int(l - n), int(l), device=q.device) for n, l in zip(new, keys)])
        seq = torch.cat([torch.full((int(n),), b, device=q.device) for b, n in enumerate(new)])
        p = s["positions"].flatten(1) if s["positions"] is not None else place[None]
        at = s["page_table"].long()[seq, place // page] * page + place % page
        kc, vc = s["k_cache"].to(f64), s["v_cache"].to(f64)
        kc.view(-1, s["hk"], D)[at] = turn(s["k"].flatten(0, len(lead) - 1), p, 1.0)
        vc.view(-1, s["hk"], D)[at] = s["v"].flatten(0, len(lead) - 1).to(f64)
        return [turn(q, p, 1.0).view(s["q"].shape), kc, vc]
    if work(case)["flops"] > 4e11:
        return None
    group = s["hq"] // s["hk"]
    o = torch.zeros(q.shape, device=q.device, dtype=f64)
    lse = torch.zeros(q.shape[0], s["hq"], device=q.device, dtype=f64)
    if s["op"] == "prefix":
        pk = s["k_cache"][s["prefix_pages"].long()].flatten(0, 1)[: s["prefix"]]
        pv = s["v_cache"][s["prefix_pages"].long()].flatten(0, 1)[: s["prefix"]]
    for b in range(len(new)):
        n, length, row = int(new[b]), int(keys[b]), int(begin[b])
        own_pages = s["page_table"][b, : -(-length // page)].long()
        k, v = s["k_cache"][own_pages].flatten(0, 1)[:length], s["v_cache"][own_pages].flatten(0, 1)[:length]
        ahead = 0
        if s["op"] == "prefix":
            k, v, ahead = torch.cat([pk, k]), torch.cat([pv, v]), s["prefix"]
        last = ahead + length - n + torch.arange(n, device=q.device)
        seen = torch.arange(ahead + length, device=q.device)[None] <= last[:, None]
        for h in range(s["hk"]):
            x = q[row:row + n, h * group:(h + 1) * group].to(f64)
            z = torch.einsum("ngd,kd->gnk", x, k[:, h].to(f64)) / math.sqrt(D)
            if s.get("causal", 1):
                z.masked_fill_(~seen, -math.inf)
            m = z.amax(-1, keepdim=True)
            z = z.sub_(m).exp_()
            total = z.sum(-1, keepdim=True)
            o[row:row + n, h * group:(h + 1) * group] = (torch.einsum("gnk,kd->gnd", z, v[:, h].to(f64)) / total).transpose(0, 1)
            lse[row:row + n, h * group:(h + 1) * group] = (m + total.log()).squeeze(-1).t()
    out = [o.view(s["q"].shape)]
    if s["lse"]:
        out.append(lse.t().contiguous() if s["ragged"] else lse.view(*lead, s["hq"]).transpose(1, 2).contiguous())
    return out
