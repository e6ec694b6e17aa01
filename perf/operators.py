"""Workloads of the 4-bit KV cache and of the logit controls of the rollout engine.

Four operators of a decode step: the cache write (with its read-back), paged attention over the 4-bit cache, the
token state of admitted requests, and the controls (penalties, biases, token masks) applied to the logits. Every
case is a dict of plain values; ``prepare`` makes its inputs, ``run`` takes one pass (the plain form in elementary
torch operations, or the framework's kernels when ``own`` is set) and ``exact`` gives the result in 64 bits.

4-bit cache: one row is one head of one token. Its ``hd`` channels form groups of 64; a group keeps a scale ``a`` and
a base ``z`` in fp16 and a nibble ``n`` per channel, which stands for ``a n + z``. The 32-bit word ``w`` of a row holds
channels ``64 (w mod G) + 8 (w div G) + 0..7`` (``G = hd / 64``), the lowest channel in the lowest nibble. ``k`` and ``v``
are ``[pages, heads, page, hd / 2]`` bytes, ``scale`` is ``[pages, heads, page, 2 (k, v), G, 2 (a, z)]``.
"""

from __future__ import annotations

import math
import random

import torch

own = False

GROUP = 64
HALF_MAX = 65504.0
HEADS = [(12, 2, 128), (14, 2, 64), (16, 2, 128), (16, 8, 128), (32, 8, 128), (28, 4, 128), (32, 4, 128),
         (24, 2, 128), (8, 8, 64), (4, 2, 64)]
VOCABS = [151936, 130560, 128256, 152064, 2048, 32001, 100003]
LARGEST_KV = 8 * 131072 * 2 * 128      # channels of K in the longest listed attention case
LARGEST_WRITE = 32768 * 8 * 128        # channels of K in the largest listed write
LARGEST_LOGITS = 256 * 128256
LARGEST_TOKENS = 64 * 16384


# ── cases ────────────────────────────────────────────────────────────────────

def listed():
    return [
        # one new token of each of 64 running rows, one layer of the 12-head model
        {"name": "write_decode_64", "op": "write", "tokens": 64, "heads": 2, "hd": 128, "page": 64},
        # a prefill chunk of 32768 prompt tokens, 8 KV heads
        {"name": "write_prefill_32k", "op": "write", "tokens": 32768, "heads": 8, "hd": 128, "page": 64},
        # one interactive request with a short context: latency
        {"name": "attn_1x700", "op": "attn", "rows": 1, "q_heads": 12, "heads": 2, "hd": 128, "page": 64,
         "shortest": 700, "longest": 700, "lens": 1, "empty": False},
        # a rollout batch in mid flight: 64 ragged rows up to 8k tokens
        {"name": "attn_64_ragged_8k", "op": "attn", "rows": 64, "q_heads": 12, "heads": 2, "hd": 128, "page": 64,
         "shortest": 1, "longest": 8192, "lens": 2, "empty": False},
        # many short rows, 8 KV heads
        {"name": "attn_256x1500", "op": "attn", "rows": 256, "q_heads": 32, "heads": 8, "hd": 128, "page": 64,
         "shortest": 900, "longest": 1500, "lens": 3, "empty": False},
        # head width 64, seven query heads to a KV head, pages of 16, idle rows of length zero
        {"name": "attn_33_hd64_p16", "op": "attn", "rows": 33, "q_heads": 14, "heads": 2, "hd": 64, "page": 16,
         "shortest": 1, "longest": 5001, "lens": 4, "empty": True},
        # the 128k recipe's tail: 8 rows at full length
        {"name": "attn_8x128k", "op": "attn", "rows": 8, "q_heads": 16, "heads": 2, "hd": 128, "page": 64,
         "shortest": 131072, "longest": 131072, "lens": 5, "empty": False},
        # prompts of 16 requests admitted together
        {"name": "tokens_admit_16", "op": "tokens", "rows": 16, "slots": 64, "vocab": 151936, "shortest": 1,
         "longest": 2000, "generated": 0.0, "lens": 6},
        # 64 partial rollouts resumed after a weight update, most of their tokens generated
        {"name": "tokens_resume_64", "op": "tokens", "rows": 64, "slots": 64, "vocab": 151936, "shortest": 512,
         "longest": 16384, "generated": 0.9, "lens": 7},
        # one row: latency
        {"name": "logits_1", "op": "logits", "rows": 1, "slots": 4, "vocab": 130560, "dtype": "float32",
         "history": 4096, "bias": 32, "masked": 0.0},
        # a rollout batch; every other row under a token mask
        {"name": "logits_64", "op": "logits", "rows": 64, "slots": 64, "vocab": 151936, "dtype": "float32",
         "history": 4096, "bias": 16, "masked": 0.5},
        # the largest batch, bf16 logits
        {"name": "logits_256_bf16", "op": "logits", "rows": 256, "slots": 256, "vocab": 128256, "dtype": "bfloat16",
         "history": 2048, "bias": 8, "masked": 0.25},
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 0.49)))))))


def draw(rng):
    op = rng.choice(["write", "attn", "attn", "tokens", "logits"])
    seed = rng.randrange(1 << 30)
    if op == "write":
        _, heads, hd = rng.choice(HEADS)
        return {"op": op, "tokens": _log_int(rng, 1, min(40000, LARGEST_WRITE // (heads * hd))), "heads": heads, "hd": hd,
                "page": rng.choice([16, 32, 64, 128])}
    if op == "attn":
        q_heads, heads, hd = rng.choice(HEADS)
        rows = _log_int(rng, 1, 300)
        longest = _log_int(rng, 1, min(131072, LARGEST_KV // (rows * heads * hd)))
        shortest = rng.choice([1, max(1, longest // 2), longest])
        return {"op": op, "rows": rows, "q_heads": q_heads, "heads": heads, "hd": hd, "page": rng.choice([16, 32, 64, 128]),
                "shortest": shortest, "longest": longest, "lens": seed, "empty": rng.random() < 0.3}
    vocab = rng.choice(VOCABS)
    if op == "tokens":
        rows = _log_int(rng, 1, 64)
        longest = _log_int(rng, 1, min(32768, LARGEST_TOKENS // rows))
        return {"op": op, "rows": rows, "slots": rows + rng.randrange(8), "vocab": vocab, "shortest": rng.choice([0, 1, longest]),
                "longest": longest, "generated": rng.choice([0.0, 0.5, 0.9, 1.0]), "lens": seed}
    rows = _log_int(rng, 1, min(256, LARGEST_LOGITS // vocab))
    return {"op": op, "rows": rows, "slots": rows + rng.randrange(8), "vocab": vocab,
            "dtype": rng.choice(["float32", "float32", "bfloat16"]), "history": _log_int(rng, 1, 8192),
            "bias": rng.choice([0, 1, 8, 64, 300]), "masked": rng.choice([0.0, 0.25, 0.5, 1.0])}


def lengths(case):
    """The rows' lengths: part of the case, so that :func:`work` knows them."""
    rng = random.Random(case["lens"])
    out = [rng.randint(case["shortest"], case["longest"]) for _ in range(case["rows"])]
    if case["op"] == "attn" and case["rows"] > 1:
        out[rng.randrange(case["rows"])] = case["longest"]
        if case["empty"]:
            out[rng.randrange(case["rows"])] = 0
    return out


def work(case):
    op = case["op"]
    if op in ("write", "attn"):
        hd, heads = case["hd"], case["heads"]
        row = hd + 8 * (hd // GROUP)  # K and V nibbles and their fp16 pairs
        if op == "write":
            n = case["tokens"] * heads
            return {"bytes": n * (4 * hd + row + 4 * hd) + 8 * case["tokens"], "flops": 8 * n * 2 * hd}
        total = sum(lengths(case))
        return {"bytes": total * heads * row + 4 * case["rows"] * case["q_heads"] * hd,
                "flops": 4 * total * case["q_heads"] * hd}
    rows, V = case["rows"], case["vocab"]
    words = (V + 31) // 32
    if op == "tokens":
        return {"bytes": 8 * sum(lengths(case)) + rows * (4 * V + 4 * words), "flops": sum(lengths(case))}
    item = 4 if case["dtype"] == "float32" else 2
    seen = V * (1.0 - math.exp(-case["history"] / V * 4.0)) / 4.0  # about this many distinct tokens in a history
    return {"bytes": int(rows * (V * (item + 4) + 4 * words * (1 + case["masked"]) + 4 * seen + 8 * case["bias"])),
            "flops": 4 * rows * V}


# ── inputs ───────────────────────────────────────────────────────────────────

def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _channels(n, heads, hd, g):
    """K-like or V-like rows: channels of unequal spread, a few with an offset (as a QKV bias gives)."""
    spread = torch.exp(0.5 * torch.randn(heads, hd, generator=g, device="cuda"))
    offset = 3.0 * torch.randn(heads, hd, generator=g, device="cuda") * (torch.rand(heads, hd, generator=g, device="cuda") < 0.1)
    return (torch.randn(n, heads, hd, generator=g, device="cuda") * spread + offset).bfloat16()


def _pack(x):
    """``x [n, heads, hd]`` bf16 to ``(bytes [n, heads, hd / 2], pairs [n, heads, G, 2])``."""
    n, heads, hd = x.shape
    G = hd // GROUP
    xf = x.float().clamp(-HALF_MAX, HALF_MAX).view(n, heads, G, GROUP)
    lo = xf.amin(-1, keepdim=True)
    hi = xf.amax(-1, keepdim=True)
    a = ((hi - lo) / 15.0).half()
    z = lo.half()
    af = a.float()
    q = torch.round((xf - z.float()) / torch.where(af > 0, af, torch.ones_like(af)))
    q = torch.where(af > 0, q, torch.zeros_like(q)).clamp(0, 15).to(torch.uint8)
    words = q.view(n, heads, G, 8, 8).transpose(2, 3).reshape(n, heads, hd)  # word u G + grp, nibble by nibble
    return words[..., 0::2] | (words[..., 1::2] << 4), torch.stack([a.squeeze(-1), z.squeeze(-1)], -1)


def _unpack(b, pairs, dtype):
    """Inverse of :func:`_pack`: the values ``[n, heads, hd]`` that the nibbles stand for, in ``dtype``."""
    n, heads, half = b.shape
    hd = 2 * half
    G = hd // GROUP
    nib = torch.stack([b & 15, b >> 4], -1).reshape(n, heads, 8, G, 8).transpose(2, 3).reshape(n, heads, G, GROUP)
    return (nib.to(dtype) * pairs[..., :1].to(dtype) + pairs[..., 1:].to(dtype)).reshape(n, heads, hd)


def _empty_cache(pages, heads, page, hd):
    return {"k": torch.zeros(pages, heads, page, hd // 2, dtype=torch.uint8, device="cuda"),
            "v": torch.zeros(pages, heads, page, hd // 2, dtype=torch.uint8, device="cuda"),
            "scale": torch.zeros(pages, heads, page, 2, hd // GROUP, 2, dtype=torch.float16, device="cuda")}


def _tokens(n, V, g):
    """Token ids with few frequent and many rare ones."""
    u = torch.rand(n, generator=g, device="cuda")
    rank = (V * u.pow(3)).long().clamp(max=V - 1)
    return (rank * 7919 + 13) % V


def _bits(x):
    """``x [rows, V]`` bool to ``[rows, ceil(V / 32)]`` int32 words, entry ``v`` at bit ``v mod 32``."""
    rows, V = x.shape
    W = (V + 31) // 32
    pad = torch.zeros(rows, W * 32, dtype=torch.bool, device=x.device)
    pad[:, :V] = x
    out = torch.zeros(rows, W, dtype=torch.int32, device=x.device)
    pad = pad.view(rows, W, 32)
    for i in range(32):
        out |= pad[:, :, i].int() << i
    return out


def _unbits(words, V):
    sh = torch.arange(32, dtype=torch.int32, device=words.device)
    return ((words.unsqueeze(-1) >> sh) & 1).bool().reshape(words.shape[0], -1)[:, :V]


def prepare(case, seed):
    g = _gen(seed)
    st = {"case": case}
    op = case["op"]
    if op == "write":
        T, heads, hd, page = case["tokens"], case["heads"], case["hd"], case["page"]
        # K and V as they leave the fused projection: strided views of one row block
        slab = torch.cat([_channels(T, heads, hd, g), _channels(T, heads, hd, g)], 1)
        st["k"], st["v"] = slab[:, :heads], slab[:, heads:]
        pages = -(-T // page) + 2
        per_row = T <= 512  # decode: one token each on many pages; prefill: whole pages
        if per_row:
            st["slots"] = torch.randperm(pages * page, generator=g, device="cuda")[:T]
        else:
            order = torch.randperm(pages, generator=g, device="cuda")
            t = torch.arange(T, device="cuda")
            st["slots"] = order[t // page] * page + t % page
        st["cache"] = _empty_cache(pages, heads, page, hd)
    elif op == "attn":
        heads, hd, page = case["heads"], case["hd"], case["page"]
        lens = lengths(case)
        need = [-(-n // page) for n in lens]
        pages = sum(need) + 1
        st["cache"] = c = _empty_cache(pages, heads, page, hd)
        step = max(1, (1 << 25) // (page * heads * hd))
        for key, kv in (("k", 0), ("v", 1)):
            for s in range(0, pages, step):
                e = min(pages, s + step)
                b, pairs = _pack(_channels((e - s) * page, heads, hd, g))
                c[key][s:e] = b.view(e - s, page, heads, hd // 2).transpose(1, 2)
                c["scale"][s:e, :, :, kv] = pairs.view(e - s, page, heads, -1, 2).transpose(1, 2)
        order = torch.randperm(pages, generator=g, device="cuda").int()
        bt = torch.zeros(case["rows"], max(need + [1]), dtype=torch.int32, device="cuda")
        at = 0
        for i, n in enumerate(need):
            bt[i, :n] = order[at:at + n]
            at += n
        st["block_table"] = bt
        st["lens"] = lens
        st["seq_lens"] = torch.tensor(lens, dtype=torch.int32, device="cuda")
        st["q"] = torch.randn(case["rows"], case["q_heads"], hd, generator=g, device="cuda").bfloat16()
    else:
        rows, slots, V = case["rows"], case["slots"], case["vocab"]
        W = (V + 31) // 32
        st["slots"] = torch.randperm(slots, generator=g, device="cuda")[:rows]
        if op == "tokens":
            lens = lengths(case)
            st["tokens"] = _tokens(sum(lens), V, g)
            cu = [0]
            for n in lens:
                cu.append(cu[-1] + n)
            st["cu"] = torch.tensor(cu, dtype=torch.int32, device="cuda")
            st["n_prompt"] = torch.tensor([n - int(n * case["generated"]) for n in lens], dtype=torch.int32, device="cuda")
            st["lens"] = lens
            st["seen"] = torch.zeros(slots, W, dtype=torch.int32, device="cuda")
            st["counts"] = torch.zeros(slots, V, dtype=torch.int32, device="cuda")
            ctl = {}
        else:
            st["logits"] = (3.0 * torch.randn(rows, V, generator=g, device="cuda")).to(getattr(torch, case["dtype"]))
            counts = torch.zeros(slots, V, dtype=torch.int32, device="cuda")
            seen = torch.zeros(slots, V, dtype=torch.bool, device="cuda")
            hist = _tokens(slots * case["history"], V, g).view(slots, -1)
            seen.scatter_(1, hist, True)
            half = hist[:, hist.shape[1] // 2:]  # the first half is the prompt
            counts.scatter_add_(1, half, torch.ones_like(half, dtype=torch.int32))
            st["seen"], st["counts"] = _bits(seen), counts
            K = case["bias"]
            st["bias_ids"] = torch.full((slots, K), -1, dtype=torch.int32, device="cuda")
            st["bias_vals"] = torch.zeros(slots, K, device="cuda")
            if K:
                strip = V // K
                ids = torch.arange(K, device="cuda") * strip + torch.randint(strip, (slots, K), generator=g, device="cuda")
                keep = torch.rand(slots, K, generator=g, device="cuda") < 0.8
                st["bias_ids"] = torch.where(keep, ids, -torch.ones_like(ids)).int()
                st["bias_vals"] = 4.0 * torch.randn(slots, K, generator=g, device="cuda")

            def some(values):
                return torch.tensor(values, device="cuda")[torch.randint(len(values), (slots,), generator=g, device="cuda")]

            st["repetition"], st["frequency"], st["presence"] = some([1.0, 1.1, 1.3, 0.9]), some([0.0, 0.2, 0.5]), some([0.0, 0.3, -0.1])
            st["mask_on"] = (torch.arange(slots, device="cuda") < round(case["masked"] * slots)).int()
            st["mask_on"] = st["mask_on"][torch.randperm(slots, generator=g, device="cuda")]
            allowed = torch.rand(slots, V, generator=g, device="cuda") < 0.2
            st["mask"] = _bits(allowed)
            ctl = {k: st[k] for k in ("repetition", "frequency", "presence", "bias_ids", "bias_vals", "mask", "mask_on")}
        if own:
            from meshy_b200.ops.controls import LogitControls

            c = LogitControls.create(slots, V, device="cuda", max_bias=case.get("bias", 0))
            for k, v in dict(ctl, seen=st["seen"], counts=st["counts"]).items():
                getattr(c, k).copy_(v)
            st["ctl"] = c
    if own and op in ("write", "attn"):
        from meshy_b200.ops.kv4 import KV4Cache

        st["own_cache"] = KV4Cache(**st["cache"])
    return st


# ── one pass ─────────────────────────────────────────────────────────────────

def run(st):
    op = st["case"]["op"]
    if own:
        return {"write": _own_write, "attn": _own_attn, "tokens": _own_tokens, "logits": _own_logits}[op](st)
    return {"write": _plain_write, "attn": _plain_attn, "tokens": _plain_tokens, "logits": _plain_logits}[op](st)


def _own_write(st):
    from meshy_b200.ops.kv4 import kv4_read, kv4_write

    kv4_write(st["k"], st["v"], st["own_cache"], st["slots"])
    return kv4_read(st["own_cache"], st["slots"])


def _own_attn(st):
    from meshy_b200.ops.kv4 import paged_attention_kv4

    return paged_attention_kv4(st["q"], st["own_cache"], st["block_table"], st["seq_lens"])


def _own_tokens(st):
    from meshy_b200.ops.controls import load_tokens

    load_tokens(st["ctl"], st["slots"], st["tokens"], st["cu"], st["n_prompt"])
    return st["ctl"].seen, st["ctl"].counts


def _own_logits(st):
    from meshy_b200.ops.controls import apply_logit_controls

    out = torch.empty(st["logits"].shape, dtype=torch.float32, device="cuda")
    return apply_logit_controls(st["logits"], st["ctl"], st["slots"], out=out)


def _plain_write(st):
    c, slots = st["cache"], st["slots"]
    page = c["k"].shape[2]
    pg, off = slots // page, slots % page
    out = []
    for key, kv, x in (("k", 0, st["k"]), ("v", 1, st["v"])):
        b, pairs = _pack(x)
        c[key][pg, :, off] = b
        c["scale"][pg, :, off, kv] = pairs
        out.append(_unpack(c[key][pg, :, off], c["scale"][pg, :, off, kv], torch.float32).bfloat16())
    return tuple(out)


def _plain_attn(st):
    q, c, bt = st["q"], st["cache"], st["block_table"]
    rows, q_heads, hd = q.shape
    heads, page = c["k"].shape[1], c["k"].shape[2]
    rep = q_heads // heads
    out = torch.zeros(rows, q_heads, hd, device="cuda")
    for i, n in enumerate(st["lens"]):
        if n == 0:
            continue
        pg = bt[i, : -(-n // page)].long()

        def rows_of(key, kv):
            x = _unpack(c[key][pg].transpose(1, 2).reshape(-1, heads, hd // 2),
                        c["scale"][pg][:, :, :, kv].transpose(1, 2).reshape(-1, heads, hd // GROUP, 2), torch.float32)
            return x[:n].transpose(0, 1)  # [heads, n, hd]

        s = torch.matmul(q[i].float().view(heads, rep, hd), rows_of("k", 0).transpose(1, 2)) / math.sqrt(hd)
        p = torch.exp(s - s.amax(-1, keepdim=True))
        o = torch.matmul(p, rows_of("v", 1)) / p.sum(-1, keepdim=True)
        out[i] = o.reshape(q_heads, hd)
    return out.bfloat16()


def _plain_tokens(st):
    V, slots, tokens = st["case"]["vocab"], st["slots"], st["tokens"]
    lens = torch.tensor(st["lens"], device="cuda")
    row = torch.repeat_interleave(torch.arange(len(st["lens"]), device="cuda"), lens)
    gen = torch.arange(tokens.numel(), device="cuda") - st["cu"][row] >= st["n_prompt"][row]
    seen = torch.zeros(slots.numel(), V, dtype=torch.bool, device="cuda")
    seen[row, tokens] = True
    counts = torch.zeros(slots.numel(), V, dtype=torch.int32, device="cuda")
    counts.index_put_((row, tokens), gen.int(), accumulate=True)
    st["seen"][slots] = _bits(seen)
    st["counts"][slots] = counts
    return st["seen"], st["counts"]


def _plain_logits(st):
    z = st["logits"].float()
    V, slots = z.shape[1], st["slots"]
    seen = _unbits(st["seen"][slots], V)
    c = st["counts"][slots].float()
    r = st["repetition"][slots, None]
    z = torch.where(seen, torch.where(z > 0, z / r, z * r), z)
    z = z - st["frequency"][slots, None] * c - st["presence"][slots, None] * (c > 0).float()
    if st["bias_ids"].shape[1]:
        ids = st["bias_ids"][slots].long()
        z.scatter_add_(1, ids.clamp(min=0), torch.where(ids >= 0, st["bias_vals"][slots], 0.0))
    banned = (st["mask_on"][slots, None] != 0) & ~_unbits(st["mask"][slots], V)
    return torch.where(banned, torch.full_like(z, -math.inf), z)


# ── the definition in 64 bits ────────────────────────────────────────────────

def exact(case, seed):
    st = prepare(case, seed)
    op = case["op"]
    if op == "write":
        return tuple(_exact_quantised(st[k]) for k in ("k", "v"))
    if op == "attn":
        return _exact_attn(st)
    if op == "tokens":
        seen = st["seen"].clone()
        counts = st["counts"].clone()
        V = case["vocab"]
        at = 0
        for i, n in enumerate(st["lens"]):
            toks = st["tokens"][at:at + n]
            at += n
            slot = int(st["slots"][i])
            seen[slot] = _bits((torch.bincount(toks, minlength=V) > 0)[None])[0]
            counts[slot] = torch.bincount(toks[int(st["n_prompt"][i]):], minlength=V).int()
        return seen, counts
    out = torch.empty(st["logits"].shape, dtype=torch.float64, device="cuda")
    V = case["vocab"]
    for i in range(case["rows"]):
        s = int(st["slots"][i])
        z = st["logits"][i].double()
        c = st["counts"][s].double()
        r = float(st["repetition"][s])
        hit = _unbits(st["seen"][s][None], V)[0]
        z = torch.where(hit, z * torch.where(z > 0, 1.0 / r, r), z)
        z = z - float(st["frequency"][s]) * c - float(st["presence"][s]) * (c > 0)
        for j in range(case["bias"]):
            v = st["bias_ids"][s, j].long().clamp(min=0)
            z[v] += torch.where(st["bias_ids"][s, j] >= 0, st["bias_vals"][s, j].double(), 0.0)
        if int(st["mask_on"][s]):
            z[~_unbits(st["mask"][s][None], V)[0]] = -math.inf
        out[i] = z
    return out


def _exact_quantised(x):
    """The values the cache holds for ``x``; scale and base are fp16 numbers by the format's definition (the scale
    rounded to fp16 from the fp32 quotient), everything else is in 64 bits."""
    d = x.double().clamp(-HALF_MAX, HALF_MAX).unflatten(-1, (-1, GROUP))
    lo, hi = d.amin(-1, keepdim=True), d.amax(-1, keepdim=True)
    a = ((hi - lo) / 15.0).float().half().double()
    z = lo.half().double()
    n = ((d - z) / a).round().nan_to_num(0.0).clamp(0, 15)
    return (a * n + z).flatten(-2)


def _exact_attn(st):
    q, c = st["q"].double(), st["cache"]
    rows, q_heads, hd = q.shape
    heads, page = c["k"].shape[1], c["k"].shape[2]
    G = hd // GROUP
    out = torch.zeros(rows, q_heads, hd, dtype=torch.float64, device="cuda")
    word = torch.arange(hd, device="cuda")
    at = ((word % GROUP) // 8 * G + word // GROUP) * 8 + word % 8  # nibble of each channel within its row
    for i, n in enumerate(st["lens"]):
        if n == 0:
            continue
        t = torch.arange(n, device="cuda")
        pg, off = st["block_table"][i, t // page].long(), t % page
        for h in range(heads):
            val = []
            for key, kv in (("k", 0), ("v", 1)):
                b = c[key][pg, h, off].long()[:, at // 2]
                nib = (b >> (4 * (at % 2))) & 15
                pair = c["scale"][pg, h, off, kv].double()[:, word // GROUP]
                val.append(pair[..., 0] * nib + pair[..., 1])
            mine = slice(h * (q_heads // heads), (h + 1) * (q_heads // heads))
            p = torch.softmax(q[i, mine] @ val[0].T / math.sqrt(hd), dim=-1)
            out[i, mine] = p @ val[1]
    return out
