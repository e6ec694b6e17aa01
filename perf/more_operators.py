"""Workloads of the 8-bit KV cache, its attention, the paged tables and the scaled rotary positions.

Four operators in the order in which a step uses them: rotary positions of a fused QKV projection (half or interleaved
layout, part of a head, scaled for long contexts; with its gradient), block tables and slot maps made from request
lengths, the write of K and V into an 8-bit paged cache, and the decode attention that reads it. Every case is a dict
of plain values; ``prepare`` makes its inputs, ``run`` takes one pass (the plain form in elementary torch operations,
or the framework's kernels when ``own`` is set) and ``exact`` gives the result in 64 bits.

8-bit cache: ``k`` and ``v`` are ``[pages, heads, page, hd]`` bytes, ``scale`` is ``[pages, heads, page / 16, 2]``
fp32 (k, v). The 16 tokens of a block share one scale per head. With ``r`` the largest number of 8 significant bits
that is not above 127 / max|x|, a channel is kept as the byte ``rint(x r) + 128`` and the scale as fp32(1 / r); it
stands for ``scale (byte - 128)``. A write that holds a block's first token starts the block anew; any other keeps the
smaller of the old and the new ``r``, and where that shrinks it, the block's other tokens are requantised,
``rint(n r' / r)``.
"""

from __future__ import annotations

import math
import random

import torch

own = False

BLOCK = 16
LEAST, MOST = 2.0 ** -100, 2.0 ** 126   # range of a block's largest magnitude
HEADS = [(12, 2, 128), (14, 2, 64), (16, 2, 128), (16, 8, 128), (32, 8, 128), (28, 4, 128), (32, 4, 128),
         (24, 2, 128), (8, 8, 64), (4, 2, 64)]
LARGEST_KV = 8 * 131072 * 2 * 128       # channels of K in the longest listed attention case
LARGEST_WRITE = 32768 * 8 * 128         # channels of K in the largest listed write
LARGEST_ROTARY = 16384 * 48 * 128       # channels of the fused projection in the largest listed rotary case
LARGEST_MAP = 256 * 8192                # tokens of the largest listed map


# ── cases ────────────────────────────────────────────────────────────────────

def listed():
    return [
        # one decode step of 64 rows of the 12-head model, its context stretched fourfold: latency
        {"name": "rotary_decode_64", "op": "rotary", "tokens": 64, "q_heads": 12, "heads": 2, "hd": 128, "rot": 128,
         "interleaved": False, "scaling": "yarn", "norm": False, "grad": False, "longest": 131072, "theta": 1e4},
        # a training micro-batch of the 8B model (32 / 8 heads), forward and backward
        {"name": "rotary_train_16k", "op": "rotary", "tokens": 16384, "q_heads": 32, "heads": 8, "hd": 128, "rot": 128,
         "interleaved": False, "scaling": "llama3", "norm": False, "grad": True, "longest": 8192, "theta": 5e5},
        # a ragged micro-batch of a model with QK-norm: the norms' weights have gradients too
        {"name": "rotary_norm_5003", "op": "rotary", "tokens": 5003, "q_heads": 16, "heads": 8, "hd": 128, "rot": 128,
         "interleaved": False, "scaling": "yarn", "norm": True, "grad": True, "longest": 5003, "theta": 1e6},
        # head width 64, half of it rotated, interleaved pairs
        {"name": "rotary_part_777", "op": "rotary", "tokens": 777, "q_heads": 14, "heads": 2, "hd": 64, "rot": 32,
         "interleaved": True, "scaling": "linear", "norm": False, "grad": True, "longest": 777, "theta": 1e6},
        # the prompts of 16 requests admitted together
        {"name": "paging_admit_16", "op": "paging", "rows": 16, "slots": 64, "page": 64, "start": 0, "shortest": 1,
         "longest": 2000, "lens": 1},
        # 256 interrupted rollouts of up to 8192 tokens resumed after a weight update
        {"name": "paging_resume_256", "op": "paging", "rows": 256, "slots": 256, "page": 64, "start": 300,
         "shortest": 512, "longest": 8192, "lens": 2},
        # one new token of each of 64 running rows, appended to blocks that hold others
        {"name": "write_decode_64", "op": "write", "tokens": 64, "heads": 2, "hd": 128, "page": 64, "append": True},
        # a prefill chunk of 32768 prompt tokens, 8 KV heads; its own attention takes the values back
        {"name": "write_prefill_32k", "op": "write", "tokens": 32768, "heads": 8, "hd": 128, "page": 64,
         "append": False},
        # one interactive request with a short context: latency
        {"name": "attn_1x700", "op": "attn", "rows": 1, "q_heads": 12, "heads": 2, "hd": 128, "page": 64,
         "shortest": 700, "longest": 700, "lens": 3, "empty": False},
        # head width 64, seven query heads to a KV head, pages of 16, idle rows of length zero
        {"name": "attn_33_hd64_p16", "op": "attn", "rows": 33, "q_heads": 14, "heads": 2, "hd": 64, "page": 16,
         "shortest": 1, "longest": 5001, "lens": 4, "empty": True},
        # a rollout batch in mid flight: 64 ragged rows up to 8k tokens
        {"name": "attn_64_ragged_8k", "op": "attn", "rows": 64, "q_heads": 12, "heads": 2, "hd": 128, "page": 64,
         "shortest": 1, "longest": 8192, "lens": 5, "empty": False},
        # the 128k recipe's tail: 8 rows at full length
        {"name": "attn_8x128k", "op": "attn", "rows": 8, "q_heads": 16, "heads": 2, "hd": 128, "page": 64,
         "shortest": 131072, "longest": 131072, "lens": 6, "empty": False},
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 0.49)))))))


def draw(rng):
    op = rng.choice(["rotary", "rotary", "paging", "write", "attn", "attn"])
    if op == "rotary":
        q_heads, heads, hd = rng.choice(HEADS)
        tokens = _log_int(rng, 1, LARGEST_ROTARY // ((q_heads + 2 * heads) * hd))
        return {"op": op, "tokens": tokens, "q_heads": q_heads, "heads": heads, "hd": hd,
                "rot": rng.choice([hd, hd, hd // 2, hd // 4, 3 * hd // 4]), "interleaved": rng.random() < 0.4,
                "scaling": rng.choice(["none", "linear", "llama3", "yarn"]), "norm": rng.random() < 0.4,
                "grad": rng.random() < 0.6, "longest": _log_int(rng, 1, 1 << 20), "theta": rng.choice([1e4, 5e5, 1e6])}
    if op == "paging":
        rows = _log_int(rng, 1, 300)
        longest = _log_int(rng, 1, LARGEST_MAP // rows)
        return {"op": op, "rows": rows, "slots": rows + rng.randrange(1, 40), "page": rng.choice([16, 32, 64, 128]),
                "start": rng.choice([0, _log_int(rng, 1, 4000)]), "shortest": rng.randrange(0, longest + 1),
                "longest": longest, "lens": rng.randrange(1 << 30)}
    if op == "write":
        _, heads, hd = rng.choice(HEADS)
        append = rng.random() < 0.5
        most = 600 if append else min(40000, LARGEST_WRITE // (heads * hd))
        return {"op": op, "tokens": _log_int(rng, 1, most), "heads": heads, "hd": hd,
                "page": rng.choice([16, 32, 64, 128]), "append": append}
    q_heads, heads, hd = rng.choice(HEADS)
    rows = _log_int(rng, 1, 300)
    longest = _log_int(rng, 1, min(131072, LARGEST_KV // (heads * hd * rows)))
    return {"op": op, "rows": rows, "q_heads": q_heads, "heads": heads, "hd": hd, "page": rng.choice([16, 32, 64, 128]),
            "shortest": rng.randrange(1, longest + 1), "longest": longest, "lens": rng.randrange(1 << 30),
            "empty": rng.random() < 0.3}


def lengths(case):
    rng = random.Random(case["lens"])
    lens = [rng.randint(case["shortest"], case["longest"]) for _ in range(case["rows"])]
    if case.get("empty") and len(lens) > 2:
        lens[1] = 0
        lens[-1] = 0
    return lens


def work(case):
    op = case["op"]
    if op == "rotary":
        T, hd = case["tokens"], case["hd"]
        qk, v = (case["q_heads"] + case["heads"]) * hd, case["heads"] * hd
        passes = 4 * T * (qk + v) + 4 * T  # the projection read, q, k and v written, positions
        flops = 3 * T * (case["q_heads"] + case["heads"]) * case["rot"]
        if case["grad"]:
            passes += 4 * T * (qk + v) + 4 * T + (2 * T * qk if case["norm"] else 0)
            flops *= 2
        return {"bytes": passes, "flops": flops + (6 * T * qk if case["norm"] else 0)}
    if op == "paging":
        lens, page = lengths(case), case["page"]
        pages = sum(_pages(case["start"] + n, page) - _pages(case["start"], page) for n in lens)
        return {"bytes": 12 * sum(lens) + 8 * pages + 20 * case["rows"], "flops": 0}
    if op == "write":
        rows = case["tokens"] * case["heads"] * 2
        held = rows * (BLOCK + 1) // 2 if case["append"] else rows  # tokens whose values are returned, on average
        return {"bytes": rows * (2 * case["hd"] + 8) + 3 * held * case["hd"], "flops": 4 * rows * case["hd"]}
    tokens = sum(lengths(case))
    row = 2 * case["hd"] + 8 / BLOCK
    return {"bytes": int(tokens * case["heads"] * row) + 4 * case["rows"] * case["q_heads"] * case["hd"]
            + 4 * (tokens // case["page"] + 2 * case["rows"]),
            "flops": 4 * tokens * case["q_heads"] * case["hd"]}


# ── inputs ───────────────────────────────────────────────────────────────────

def _pages(tokens, page):
    return -(-tokens // page)


def _channels(T, heads, hd, g):
    """K or V as projections give them: channels of different spread, a few of them large, bf16."""
    spread = torch.exp(0.4 * torch.randn(heads, hd, generator=g, device="cuda"))
    spread = torch.where(torch.rand(heads, hd, generator=g, device="cuda") < 0.03, 4.0 * spread, spread)
    return (torch.randn(T, heads, hd, generator=g, device="cuda") * spread).bfloat16()


def _steps(amax):
    """``r`` of a block whose largest magnitude is ``amax`` (fp32)."""
    q = 127.0 / amax.clamp(LEAST, MOST)
    return (q.view(torch.int32) & -65536).view(torch.float32)  # eight significant bits, towards zero


def _pack_blocks(x):
    """Bytes ``[n, heads, 16, hd]`` and scales ``[n, heads]`` of whole blocks ``x [n, 16, heads, hd]``."""
    f = x.float().transpose(1, 2)
    r = _steps(f.abs().amax((-1, -2)))
    n = torch.round(f.clamp(-MOST, MOST) * r[..., None, None])
    return (n + 128).to(torch.uint8), 1.0 / r


def _empty_cache(pages, heads, page, hd):
    return {"k": torch.zeros(pages, heads, page, hd, dtype=torch.uint8, device="cuda"),
            "v": torch.zeros(pages, heads, page, hd, dtype=torch.uint8, device="cuda"),
            "scale": torch.zeros(pages, heads, page // BLOCK, 2, device="cuda")}


def _filled_cache(pages, heads, page, hd, g):
    c = _empty_cache(pages, heads, page, hd)
    step = max(1, (1 << 25) // (page * heads * hd))
    for key, kv in (("k", 0), ("v", 1)):
        for s in range(0, pages, step):
            e = min(pages, s + step)
            x = _channels((e - s) * page, heads, hd, g).view(-1, BLOCK, heads, hd)
            b, a = _pack_blocks(x)
            c[key][s:e] = b.view(e - s, page // BLOCK, heads, BLOCK, hd).transpose(1, 2).reshape(e - s, heads, page, hd)
            c["scale"][s:e, :, :, kv] = a.view(e - s, page // BLOCK, heads).transpose(1, 2)
    return c


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    rng = random.Random(seed)
    op, st = case["op"], {"case": case}
    if op == "rotary":
        T, hd, q_heads, heads = case["tokens"], case["hd"], case["q_heads"], case["heads"]
        st["qkv"] = torch.randn(T, (q_heads + 2 * heads) * hd, generator=g, device="cuda").bfloat16()
        if case["grad"]:  # packed documents
            at = torch.arange(T, device="cuda")
            cut = rng.randrange(T)
            st["positions"] = (torch.where(at < cut, at, at - cut) % case["longest"]).int()
        else:  # one new token to a row
            st["positions"] = torch.randint(case["longest"], (T,), generator=g, device="cuda").int()
        st["q_norm"] = st["k_norm"] = None
        if case["norm"]:
            st["q_norm"] = (1 + 0.2 * torch.randn(hd, generator=g, device="cuda")).bfloat16()
            st["k_norm"] = (1 + 0.2 * torch.randn(hd, generator=g, device="cuda")).bfloat16()
        if case["grad"]:
            for key, n in (("gq", q_heads), ("gk", heads), ("gv", heads)):
                st[key] = torch.randn(T, n, hd, generator=g, device="cuda").bfloat16()
        if own:
            st["rope"] = _own_rope(case)
    elif op == "paging":
        lens, page, rows, start = lengths(case), case["page"], case["rows"], case["start"]
        i32 = dict(dtype=torch.int32, device="cuda")
        have, width = _pages(start, page), _pages(start + case["longest"], page)
        need = [_pages(start + n, page) for n in lens]
        ids = torch.randperm(case["slots"] * width + 1, generator=g, device="cuda").int()
        st["block_table"] = torch.zeros(case["slots"], width, **i32)
        st["block_table"][:, :have] = ids[:case["slots"] * have].view(case["slots"], have)
        st["pages"] = ids[case["slots"] * have:][:sum(need) - have * rows].contiguous()
        st["rows"] = torch.randperm(case["slots"], generator=g, device="cuda")[:rows].int()
        st["have"], st["need"] = torch.full((rows,), have, **i32), torch.tensor(need, **i32)
        st["start"], st["lens"] = torch.full((rows,), start, **i32), torch.tensor(lens, **i32)
        st["total"] = sum(lens)
    elif op == "write":
        T, heads, hd, page = case["tokens"], case["heads"], case["hd"], case["page"]
        st["k"], st["v"] = _channels(T, heads, hd, g), _channels(T, heads, hd, g)
        if case["append"]:
            c = st["cache"] = _filled_cache(T + 1, heads, page, hd, g)
            places = random.Random(T)  # places within the pages: the case's, dealt to the rows by the seed
            off = torch.tensor([places.randrange(page) for _ in range(T)], device="cuda")
            off = off[torch.randperm(T, generator=g, device="cuda")]
            st["slots"] = (torch.randperm(T, generator=g, device="cuda") + 1) * page + off
            first = st["slots"] // BLOCK * BLOCK  # the tokens that each block now holds
            at = first[:, None] + torch.arange(BLOCK, device="cuda")
            st["held"] = at[at <= st["slots"][:, None]]
        else:
            pages = _pages(T, page) + 8
            st["cache"] = _empty_cache(pages, heads, page, hd)
            cut = rng.randrange(T)  # two prompts, each on pages of its own
            at = torch.arange(T, device="cuda")
            at = torch.where(at < cut, at, at - cut + _pages(cut, page) * page)
            order = torch.randperm(pages, generator=g, device="cuda")
            st["slots"] = order[at // page] * page + at % page
    else:
        lens, heads, hd, page = lengths(case), case["heads"], case["hd"], case["page"]
        need = [_pages(n, page) for n in lens]
        pages = sum(need) + 1
        st["cache"] = _filled_cache(pages, heads, page, hd, g)
        order = torch.randperm(pages, generator=g, device="cuda").int()
        bt = torch.zeros(case["rows"], max(need + [1]), dtype=torch.int32, device="cuda")
        at = 0
        for i, n in enumerate(need):
            bt[i, :n] = order[at:at + n]
            at += n
        st["block_table"], st["seq_lens"] = bt, torch.tensor(lens, dtype=torch.int32, device="cuda")
        st["q"] = torch.randn(case["rows"], case["q_heads"], hd, generator=g, device="cuda").bfloat16()
    if own and op in ("write", "attn"):
        from meshy_b200.ops.kv8 import KV8Cache

        st["own_cache"] = KV8Cache(**st["cache"])
    return st


SCALING = {
    "none": None,
    "linear": {"rope_type": "linear", "factor": 4.0},
    "llama3": {"rope_type": "llama3", "factor": 8.0, "low_freq_factor": 1.0, "high_freq_factor": 4.0,
               "original_max_position_embeddings": 8192},
    "yarn": {"rope_type": "yarn", "factor": 4.0, "original_max_position_embeddings": 32768},
}


def _own_rope(case):
    from meshy_b200.ops.rotary import Rope

    return Rope(case["hd"], theta=case["theta"], rotary_dim=case["rot"], interleaved=case["interleaved"],
                scaling=SCALING[case["scaling"]])


# ── one pass ─────────────────────────────────────────────────────────────────

def run(st):
    op = st["case"]["op"]
    if own:
        return {"rotary": _own_rotary, "paging": _own_paging, "write": _own_write, "attn": _own_attn}[op](st)
    return {"rotary": _plain_rotary, "paging": _plain_paging, "write": _plain_write, "attn": _plain_attn}[op](st)


def _own_rotary(st):
    from meshy_b200.ops.rotary import qkv_rotary

    c = st["case"]
    if not c["grad"]:
        with torch.no_grad():
            return qkv_rotary(st["qkv"], st["positions"], st["rope"], c["q_heads"], c["heads"], st["q_norm"],
                              st["k_norm"], 1e-6)
    leaves = [x.detach().requires_grad_() for x in (st["qkv"], st["q_norm"], st["k_norm"]) if x is not None]
    out = qkv_rotary(leaves[0], st["positions"], st["rope"], c["q_heads"], c["heads"], *(leaves[1:] or (None, None)),
                     1e-6)
    return (*(x.detach() for x in out), *torch.autograd.grad(out, leaves, (st["gq"], st["gk"], st["gv"])))


def _own_paging(st):
    from meshy_b200.ops.paging import assign_pages, token_maps

    assign_pages(st["block_table"], st["rows"], st["have"], st["need"], st["pages"])
    return st["block_table"], *token_maps(st["block_table"], st["rows"], st["start"], st["lens"], st["total"],
                                          st["case"]["page"])


def _own_write(st):
    from meshy_b200.ops.kv8 import kv8_read, kv8_write

    if st["case"]["append"]:
        kv8_write(st["k"], st["v"], st["own_cache"], st["slots"])
        return kv8_read(st["own_cache"], st["held"])
    return kv8_write(st["k"], st["v"], st["own_cache"], st["slots"], keep=True)


def _own_attn(st):
    from meshy_b200.ops.kv8 import paged_attention_kv8

    return paged_attention_kv8(st["q"], st["own_cache"], st["block_table"], st["seq_lens"])


def _frequencies(case):
    """Radians per position ``[rot / 2]`` in 64 bits, and the factor of the rotated channels."""
    s, rot = SCALING[case["scaling"]], case["rot"]
    i = torch.arange(0, rot, 2, dtype=torch.float64, device="cuda")
    f = case["theta"] ** (-i / rot)
    if s is None:
        return f, 1.0
    if s["rope_type"] == "linear":
        return f / s["factor"], 1.0
    n = s["original_max_position_embeddings"]
    if s["rope_type"] == "llama3":
        turns = n * f / (2 * math.pi)  # over the original context
        mix = (turns - s["low_freq_factor"]) / (s["high_freq_factor"] - s["low_freq_factor"])
        return f / s["factor"] + mix.clamp(0, 1) * (f - f / s["factor"]), 1.0

    def channel(turns):
        return rot * math.log(n / (turns * 2 * math.pi)) / (2 * math.log(case["theta"]))

    low, high = max(math.floor(channel(32.0)), 0), min(math.ceil(channel(1.0)), rot - 1)
    ramp = ((i / 2 - low) / max(high - low, 1e-3)).clamp(0, 1)
    return f / s["factor"] * ramp + f * (1 - ramp), 0.1 * math.log(s["factor"]) + 1.0


def _halves(x, case):
    """The two members of each rotated pair of ``x [.., hd]`` and the rest."""
    rot = case["rot"]
    r = x[..., :rot]
    a, b = (r[..., 0::2], r[..., 1::2]) if case["interleaved"] else (r[..., :rot // 2], r[..., rot // 2:])
    return a, b, x[..., rot:]


def _joined(a, b, rest, case):
    r = torch.stack((a, b), -1).flatten(-2) if case["interleaved"] else torch.cat((a, b), -1)
    return torch.cat((r, rest), -1)


def _rotate(x, cos, sin, case):
    a, b, rest = _halves(x, case)
    return _joined(a * cos - b * sin, b * cos + a * sin, rest, case)


def _plain_rotary(st):
    c = st["case"]
    T, hd, q_heads, heads = c["tokens"], c["hd"], c["q_heads"], c["heads"]
    f, m = _frequencies(c)
    w = st["positions"].double()[:, None, None] * f
    cos, sin = (m * torch.cos(w)).float(), (m * torch.sin(w)).float()
    x = st["qkv"].view(T, -1, hd)
    qk, v = x[:, :q_heads + heads].float(), x[:, q_heads + heads:]
    weight = None
    if c["norm"]:
        weight = torch.cat((st["q_norm"].float().expand(q_heads, hd), st["k_norm"].float().expand(heads, hd)))
        rstd = torch.rsqrt((qk * qk).mean(-1, keepdim=True) + 1e-6)
        y = _rotate(qk * rstd * weight, cos, sin, c).bfloat16()
    else:
        y = _rotate(qk, cos, sin, c).bfloat16()
    out = (y[:, :q_heads].contiguous(), y[:, q_heads:].contiguous(), v.contiguous())
    if not c["grad"]:
        return out
    g = _rotate(torch.cat((st["gq"], st["gk"]), 1).float(), cos, -sin, c)
    grads = ()
    if c["norm"]:
        unit = qk * rstd
        by_head = (g * unit).sum(0)
        grads = (by_head[:q_heads].sum(0).bfloat16(), by_head[q_heads:].sum(0).bfloat16())
        g = g * weight
        g = rstd * (g - unit * (g * unit).mean(-1, keepdim=True))
    return (*out, torch.cat((g.bfloat16(), st["gv"]), 1).view(T, -1), *grads)


def _plain_paging(st):
    bt, page = st["block_table"], st["case"]["page"]
    rows, more = st["rows"].long(), (st["need"] - st["have"]).long()
    n = rows.numel()
    each = torch.repeat_interleave(torch.arange(n, device="cuda"), more)
    col = torch.arange(each.numel(), device="cuda") - (torch.cumsum(more, 0) - more)[each] + st["have"].long()[each]
    bt[rows[each], col] = st["pages"]
    lens = st["lens"].long()
    ends = torch.cumsum(lens, 0)
    row = torch.repeat_interleave(torch.arange(n, device="cuda"), lens)
    pos = torch.arange(row.numel(), device="cuda") - (ends - lens)[row] + st["start"].long()[row]
    slots = bt[rows[row], pos // page].long() * page + pos % page
    return bt, pos.int(), slots, torch.cat((torch.zeros_like(ends[:1]), ends)).int()


def _plain_write(st):
    c, slots = st["cache"], st["slots"]
    page = c["k"].shape[2]
    block, place = slots // BLOCK, slots % BLOCK
    per = page // BLOCK
    which, mine = torch.unique(block, return_inverse=True)
    pg, bl = which // per, which % per
    T, heads, hd = st["k"].shape
    anew = torch.zeros(which.numel(), dtype=torch.int32, device="cuda")
    anew = anew.scatter_reduce(0, mine, (place == 0).int(), "amax").bool()[:, None]
    for key, kv in (("k", 0), ("v", 1)):
        x = st[key].float()
        top = torch.zeros(which.numel(), heads, device="cuda")
        top = top.scatter_reduce(0, mine[:, None].expand(T, heads), x.abs().amax(-1), "amax")
        r, old = _steps(top), c["scale"][pg, :, bl, kv]
        r_old = torch.where(old > 0, 1.0 / old, math.inf).bfloat16().float()
        r = torch.where(anew, r, torch.minimum(r, r_old))
        blocks = c[key].view(-1, heads, per, BLOCK, hd)
        n = blocks[pg, :, bl].float() - 128
        again = (~anew & (r < r_old))[..., None, None]
        n = torch.where(again, torch.round(n * r[..., None, None] / r_old[..., None, None]), n)
        n[mine, :, place] = torch.round(x.clamp(-MOST, MOST) * r[mine][..., None])
        blocks[pg, :, bl] = (n + 128).to(torch.uint8)
        c["scale"][pg, :, bl, kv] = 1.0 / r
    return _plain_read(c, st["held"] if st["case"]["append"] else slots)


def _plain_read(c, slots):
    page = c["k"].shape[2]
    pg, off = slots // page, slots % page
    a = c["scale"][pg, :, off // BLOCK]
    return tuple(((c[key][pg, :, off].float() - 128) * a[..., kv, None]).bfloat16() for key, kv in (("k", 0), ("v", 1)))


def _plain_attn(st):
    q, c, bt, lens = st["q"], st["cache"], st["block_table"].long(), st["seq_lens"]
    rows, q_heads, hd = q.shape
    heads, page = c["k"].shape[1], c["k"].shape[2]
    n = bt.shape[1] * page

    def values(key, kv):  # [rows, heads, n, hd]
        x = c[key][bt].float().sub_(128).unflatten(3, (page // BLOCK, BLOCK))
        return x.mul_(c["scale"][bt][..., kv, None, None]).transpose(1, 2).reshape(rows, heads, n, hd)

    s = torch.matmul(q.float().view(rows, heads, -1, hd), values("k", 0).transpose(-1, -2)) / math.sqrt(hd)
    keep = (torch.arange(n, device="cuda") < lens[:, None])[:, None, None]
    s = torch.where(keep, s, -math.inf)
    top = s.amax(-1, keepdim=True)
    p = torch.exp(s - torch.where(top > -math.inf, top, 0.0))
    o = torch.matmul(p, values("v", 1)) / p.sum(-1, keepdim=True).clamp(min=1e-30)
    return o.reshape(rows, q_heads, hd).bfloat16()


# ── the definition in 64 bits ────────────────────────────────────────────────

def exact(case, seed):
    st = prepare(case, seed)
    of = {"rotary": _exact_rotary, "paging": _exact_paging, "write": _exact_write, "attn": _exact_attn}
    return of[case["op"]](st)


def _exact_rotary(st):
    """Channels as complex numbers, turned by the angle; the gradient is the conjugate turn."""
    c = st["case"]
    T, hd, q_heads, heads, rot = c["tokens"], c["hd"], c["q_heads"], c["heads"], c["rot"]
    s = SCALING[c["scaling"]]
    f = []
    m = 0.1 * math.log(s["factor"]) + 1 if s and s["rope_type"] == "yarn" else 1.0
    for i in range(rot // 2):
        w = c["theta"] ** (-2 * i / rot)
        if s and s["rope_type"] == "linear":
            w /= s["factor"]
        elif s and s["rope_type"] == "llama3":
            n, lo, hi = s["original_max_position_embeddings"], s["low_freq_factor"], s["high_freq_factor"]
            length = 2 * math.pi / w
            if length > n / lo:
                w /= s["factor"]
            elif length >= n / hi:
                mix = (n / length - lo) / (hi - lo)
                w = (1 - mix) * w / s["factor"] + mix * w
        elif s:
            n = s["original_max_position_embeddings"]
            lo, hi = (rot * math.log(n / (b * 2 * math.pi)) / (2 * math.log(c["theta"])) for b in (32.0, 1.0))
            lo, hi = max(math.floor(lo), 0), min(math.ceil(hi), rot - 1)
            mix = min(max((i - lo) / (hi - lo if hi > lo else 1e-3), 0.0), 1.0)
            w = w * (1 - mix) + w / s["factor"] * mix
        f.append(w)
    turn = torch.polar(torch.tensor(m, dtype=torch.float64, device="cuda"),
                       st["positions"].double()[:, None] * torch.tensor(f, dtype=torch.float64, device="cuda"))[:, None]
    ch = torch.arange(rot, device="cuda")
    first, second = (ch[0::2], ch[1::2]) if c["interleaved"] else (ch[:rot // 2], ch[rot // 2:])

    def turned(x, by):
        z = torch.complex(x[..., first], x[..., second]) * by
        y = x.clone()
        y[..., first], y[..., second] = z.real, z.imag
        return y

    x = st["qkv"].double().view(T, -1, hd)
    parts = list(x.split([q_heads, heads, heads], 1))
    norms = [st["q_norm"], st["k_norm"]]
    out, back, weights = [], [], []
    for j in range(2):
        y = parts[j]
        if c["norm"]:
            size = (y.pow(2).mean(-1, keepdim=True) + 1e-6).sqrt()
            y = y / size * norms[j].double()
        out.append(turned(y, turn))
        if c["grad"]:
            g = turned(st["gq" if j == 0 else "gk"].double(), turn.conj())
            if c["norm"]:
                u = parts[j] / size
                weights.append((g * u).sum((0, 1)))
                g = g * norms[j].double()
                g = (g - u * (g * u).mean(-1, keepdim=True)) / size
            back.append(g)
    out.append(parts[2])
    if not c["grad"]:
        return tuple(out)
    back.append(st["gv"].double())
    return (*out, torch.cat(back, 1).view(T, -1), *weights)


def _exact_paging(st):
    """Row by row, on the host."""
    bt, page = st["block_table"].tolist(), st["case"]["page"]
    pages = iter(st["pages"].tolist())
    pos, slots, cu = [], [], [0]
    for row, have, need, start, n in zip(*(st[k].tolist() for k in ("rows", "have", "need", "start", "lens"))):
        for j in range(have, need):
            bt[row][j] = next(pages)
        at = range(start, start + n)
        pos.extend(at)
        slots.extend(bt[row][p // page] * page + p % page for p in at)
        cu.append(cu[-1] + n)
    i32 = dict(dtype=torch.int32, device="cuda")
    return (torch.tensor(bt, **i32), torch.tensor(pos, **i32), torch.tensor(slots, dtype=torch.int64, device="cuda"),
            torch.tensor(cu, **i32))


def _exact_write(st):
    """Block by block for appended tokens, prompt blocks by their running number otherwise; scales are fp32 numbers by
    the format's definition, everything else is in 64 bits."""
    c, slots, T = st["cache"], st["slots"], st["case"]["tokens"]
    page, hd = c["k"].shape[2], st["case"]["hd"]

    def steps(amax):
        m, e = torch.frexp(127.0 / amax.clamp(LEAST, MOST))
        return torch.ldexp(torch.floor(m * 256) / 256, e)

    def scale(r):
        return (1.0 / r).float().double()

    out = []
    for key, kv in (("k", 0), ("v", 1)):
        x = st[key].double()
        if not st["case"]["append"]:
            block = slots // BLOCK
            number = torch.cumsum(torch.cat((block.new_zeros(1), (block[1:] != block[:-1]).long())), 0)
            top = torch.zeros(int(number[-1]) + 1, x.shape[1], dtype=torch.float64, device="cuda")
            top.index_reduce_(0, number, x.abs().amax(-1), "amax")
            r = steps(top)[number][..., None]
            out.append((x * r).round() * scale(r))
            continue
        pg, off = slots // page, slots % page
        old = c["scale"][pg, :, off // BLOCK, kv].double()
        m, e = torch.frexp(1.0 / old)
        r_old = torch.ldexp(torch.round(m * 256) / 256, e)
        r = steps(x.abs().amax(-1))
        r = torch.where((off % BLOCK == 0)[:, None], r, torch.minimum(r, r_old))
        first = off // BLOCK * BLOCK
        rows = torch.arange(BLOCK, device="cuda")
        n = c[key][pg[:, None], :, first[:, None] + rows].double() - 128  # [T, 16, heads, hd]
        n = (n * r[:, None, :, None] / r_old[:, None, :, None]).round()
        n[torch.arange(T, device="cuda"), off % BLOCK] = (x * r[..., None]).round()
        n = n * scale(r)[:, None, :, None]
        out.append(n[(rows <= (off % BLOCK)[:, None])].view(-1, x.shape[1], hd))
    return tuple(out)


def _exact_attn(st):
    q, c = st["q"].double(), st["cache"]
    rows, q_heads, hd = q.shape
    heads, page = c["k"].shape[1], c["k"].shape[2]
    out = torch.zeros(rows, q_heads, hd, dtype=torch.float64, device="cuda")
    for i, n in enumerate(st["seq_lens"].tolist()):
        if n == 0:
            continue
        t = torch.arange(n, device="cuda")
        pg, off = st["block_table"][i, t // page].long(), t % page
        for h in range(heads):
            k, v = ((c[key][pg, h, off].double() - 128) * c["scale"][pg, h, off // BLOCK, kv].double()[:, None]
                    for key, kv in (("k", 0), ("v", 1)))
            mine = slice(h * (q_heads // heads), (h + 1) * (q_heads // heads))
            out[i, mine] = torch.softmax(q[i, mine] @ k.T / math.sqrt(hd), dim=-1) @ v
    return out
