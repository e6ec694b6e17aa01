"""Plain-PyTorch definitions of every hot op.

These are the numerical oracle for the CUDA kernels (tests compare each
kernel with the function of the same name here, computed in fp32) and the
implementation used when tensors live on the CPU (the CPU
``gloo`` tests).  They favour clarity over speed.
"""

from __future__ import annotations

import math

import torch
import torch.nn.functional as F


# ── normalisation ────────────────────────────────────────────────────────────

def rmsnorm(x: torch.Tensor, w: torch.Tensor, eps: float) -> torch.Tensor:
    xf = x.float()
    y = xf * torch.rsqrt(xf.pow(2).mean(-1, keepdim=True) + eps)
    return (y * w.float()).to(x.dtype)


# ── rotary embedding (rotate-half pairing) ───────────────────────────────────

def rope_cos_sin(positions: torch.Tensor, head_dim: int, theta: float) -> tuple[torch.Tensor, torch.Tensor]:
    """cos/sin tables ``[T, head_dim/2]`` (fp32) for integer ``positions``."""
    # HF convention, fp32 throughout: inv_freq = 1 / theta^(arange(0, hd, 2) / hd)
    # built on the positions' device so the op can run inside CUDA graph capture
    dev = positions.device
    ar = torch.arange(0, head_dim, 2, dtype=torch.int64, device=dev).float() / head_dim
    inv = 1.0 / torch.pow(torch.full((), float(theta), device=dev), ar)
    ang = positions.float().unsqueeze(-1) * inv
    return torch.cos(ang), torch.sin(ang)


def apply_rope(x: torch.Tensor, cos: torch.Tensor, sin: torch.Tensor) -> torch.Tensor:
    """Rotate ``x [T, H, hd]``: pairs ``(i, i + hd/2)``."""
    half = x.shape[-1] // 2
    xf = x.float()
    x1, x2 = xf[..., :half], xf[..., half:]
    c = cos.unsqueeze(1)
    s = sin.unsqueeze(1)
    out = torch.cat([x1 * c - x2 * s, x2 * c + x1 * s], dim=-1)
    return out.to(x.dtype)


def rotary_angles(positions: torch.Tensor, rope) -> tuple[torch.Tensor, torch.Tensor]:
    """cos/sin ``[T, rotary_dim / 2]`` (fp64) of a :class:`.rotary.Rope`, its factor included."""
    f = torch.tensor(rope.frequencies(), dtype=torch.float64, device=positions.device)
    w = positions.double().unsqueeze(-1) * f
    return torch.cos(w) * rope.factor, torch.sin(w) * rope.factor


def apply_rotary(x: torch.Tensor, cos: torch.Tensor, sin: torch.Tensor, rope) -> torch.Tensor:
    """``x [T, H, hd]`` turned as ``rope`` says."""
    rot = rope.rotary_dim
    r, rest = x[..., :rot], x[..., rot:]
    a, b = (r[..., 0::2], r[..., 1::2]) if rope.interleaved else r.chunk(2, -1)
    c, s = cos.unsqueeze(1), sin.unsqueeze(1)
    pair = (a * c - b * s, b * c + a * s)
    return torch.cat([torch.stack(pair, -1).flatten(-2) if rope.interleaved else torch.cat(pair, -1), rest], -1)


def qkv_rotary(qkv, positions, rope, n_heads, n_kv, q_norm=None, k_norm=None, eps: float = 1e-6):
    """See :func:`.rotary.qkv_rotary`; in fp32 (fp64 for fp64 inputs), rounded once."""
    q, k, v = qkv.view(qkv.shape[0], -1, rope.head_dim).split([n_heads, n_kv, n_kv], 1)
    cos, sin = rotary_angles(positions, rope)

    def turned(x, w):
        y = x if x.dtype == torch.float64 else x.float()
        if w is not None:
            y = y * torch.rsqrt(y.pow(2).mean(-1, keepdim=True) + eps) * w.to(y.dtype)
        return apply_rotary(y, cos.to(y.dtype), sin.to(y.dtype), rope).to(x.dtype)

    return turned(q, q_norm), turned(k, k_norm), v.contiguous()


# ── SwiGLU with the block-interleaved fused gate/up weight ───────────────────

def deinterleave_w13(h: torch.Tensor, block: int) -> tuple[torch.Tensor, torch.Tensor]:
    """Split ``h [.., 2F]`` laid out ``[g0 u0 g1 u1 ...]`` (blocks of ``block``)."""
    shp = h.shape[:-1]
    two_f = h.shape[-1]
    hb = h.reshape(*shp, two_f // (2 * block), 2, block)
    g = hb[..., 0, :].reshape(*shp, two_f // 2)
    u = hb[..., 1, :].reshape(*shp, two_f // 2)
    return g, u


def interleave_w13(w_gate: torch.Tensor, w_up: torch.Tensor, block: int) -> torch.Tensor:
    """Inverse of :func:`deinterleave_w13` for weights ``[F, D]`` → ``[2F, D]``."""
    F_, D = w_gate.shape
    if F_ % block:
        raise ValueError(f"ffn dim {F_} is not a multiple of the interleave block {block}")
    g = w_gate.reshape(F_ // block, 1, block, D)
    u = w_up.reshape(F_ // block, 1, block, D)
    return torch.cat([g, u], dim=1).reshape(2 * F_, D)


def split_w13(w13: torch.Tensor, block: int) -> tuple[torch.Tensor, torch.Tensor]:
    two_f, D = w13.shape
    wb = w13.reshape(two_f // (2 * block), 2, block, D)
    return wb[:, 0].reshape(two_f // 2, D), wb[:, 1].reshape(two_f // 2, D)


def swiglu(h: torch.Tensor, block: int) -> torch.Tensor:
    g, u = deinterleave_w13(h.float(), block)
    return (F.silu(g) * u).to(h.dtype)


# ── attention ────────────────────────────────────────────────────────────────

def attention_chunks(q, k, v, cu_q, cu_k, q_off, scale: float | None = None) -> torch.Tensor:
    """Causal GQA attention of query chunks against separate key documents: chunk ``d`` holds queries
    ``cu_q[d]..`` at key positions ``q_off[d]..`` of keys ``cu_k[d]..cu_k[d+1]`` (fp32 oracle)."""
    T, Hq, hd = q.shape
    rep = Hq // k.shape[1]
    scale = scale if scale is not None else 1.0 / math.sqrt(hd)
    out = torch.zeros(T, Hq, hd, dtype=torch.float32, device=q.device)
    cq, ck, qo = cu_q.tolist(), cu_k.tolist(), q_off.tolist()
    for d in range(len(cq) - 1):
        s, e, ks, ke = cq[d], cq[d + 1], ck[d], ck[d + 1]
        if e <= s:
            continue
        qd = q[s:e].float().transpose(0, 1)
        kd = k[ks:ke].float().transpose(0, 1).repeat_interleave(rep, 0)
        vd = v[ks:ke].float().transpose(0, 1).repeat_interleave(rep, 0)
        sc = torch.matmul(qd, kd.transpose(1, 2)) * scale
        qpos = torch.arange(e - s, device=q.device).unsqueeze(1) + qo[d]
        kpos = torch.arange(ke - ks, device=q.device).unsqueeze(0)
        sc = sc.masked_fill(kpos > qpos, float("-inf"))
        out[s:e] = torch.matmul(torch.softmax(sc, -1), vd).transpose(0, 1)
    return out


def attention_varlen(
    q: torch.Tensor,          # [T, Hq, hd]
    k: torch.Tensor,          # [T, Hkv, hd]
    v: torch.Tensor,          # [T, Hkv, hd]
    cu_seqlens: torch.Tensor,  # [n_docs+1] int32
    scale: float | None = None,
    causal: bool = True,
) -> tuple[torch.Tensor, torch.Tensor]:
    """Causal GQA attention over packed documents; returns ``(out, lse [Hq, T])``."""
    T, Hq, hd = q.shape
    Hkv = k.shape[1]
    rep = Hq // Hkv
    scale = scale if scale is not None else 1.0 / math.sqrt(hd)
    out = torch.zeros(T, Hq, hd, dtype=torch.float32, device=q.device)
    lse = torch.full((Hq, T), float("-inf"), dtype=torch.float32, device=q.device)
    cu = cu_seqlens.tolist()
    for i in range(len(cu) - 1):
        s, e = cu[i], cu[i + 1]
        if e <= s:
            continue
        qd = q[s:e].float().transpose(0, 1)                       # [Hq, L, hd]
        kd = k[s:e].float().transpose(0, 1).repeat_interleave(rep, 0)
        vd = v[s:e].float().transpose(0, 1).repeat_interleave(rep, 0)
        sc = torch.matmul(qd, kd.transpose(1, 2)) * scale          # [Hq, L, L]
        if causal:
            L = e - s
            m = torch.ones(L, L, dtype=torch.bool, device=q.device).triu(1)
            sc = sc.masked_fill(m, float("-inf"))
        l = torch.logsumexp(sc, dim=-1)                             # [Hq, L]
        p = torch.exp(sc - l.unsqueeze(-1))
        out[s:e] = torch.matmul(p, vd).transpose(0, 1)
        lse[:, s:e] = l
    return out.to(q.dtype), lse


def attention_decode_paged(
    q: torch.Tensor,            # [B, Hq, hd]
    k_cache: torch.Tensor,      # [n_pages, Hkv, page, hd]
    v_cache: torch.Tensor,
    block_table: torch.Tensor,  # [B, max_pages] int32
    seq_lens: torch.Tensor,     # [B] int32 (tokens in cache incl. current)
    scale: float | None = None,
) -> torch.Tensor:
    B, Hq, hd = q.shape
    Hkv, page = k_cache.shape[1], k_cache.shape[2]
    rep = Hq // Hkv
    scale = scale if scale is not None else 1.0 / math.sqrt(hd)
    out = torch.zeros(B, Hq, hd, dtype=torch.float32, device=q.device)
    for b in range(B):
        L = int(seq_lens[b])
        npg = (L + page - 1) // page
        pages = block_table[b, :npg].long()
        kk = k_cache[pages].permute(1, 0, 2, 3).reshape(Hkv, npg * page, hd)[:, :L].float()
        vv = v_cache[pages].permute(1, 0, 2, 3).reshape(Hkv, npg * page, hd)[:, :L].float()
        kk = kk.repeat_interleave(rep, 0)
        vv = vv.repeat_interleave(rep, 0)
        sc = torch.einsum("hd,hld->hl", q[b].float(), kk) * scale
        p = torch.softmax(sc, dim=-1)
        out[b] = torch.einsum("hl,hld->hd", p, vv)
    return out.to(q.dtype)


# ── 4-bit KV cache ───────────────────────────────────────────────────────────

KV4_GROUP = 64
_HALF_MAX = 65504.0


def kv4_quantize(x: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor]:
    """``x [T, H, hd]`` to nibble bytes ``[T, H, hd / 2]`` uint8 and ``(a, z)`` pairs ``[T, H, hd / 64, 2]`` fp16
    (:mod:`.kv4` describes the format)."""
    T, H, hd = x.shape
    G = hd // KV4_GROUP
    xf = x.float().clamp(-_HALF_MAX, _HALF_MAX).reshape(T, H, G, KV4_GROUP)
    lo, hi = xf.amin(-1, keepdim=True), xf.amax(-1, keepdim=True)
    a, z = ((hi - lo) / 15.0).half(), lo.half()
    af = a.float()
    n = torch.where(af > 0, ((xf - z.float()) / torch.where(af > 0, af, 1.0)).round(), 0.0).clamp(0, 15)
    n = n.to(torch.uint8).view(T, H, G, 8, 8).transpose(2, 3).reshape(T, H, hd)  # word u G + group, then nibble
    return n[..., 0::2] | (n[..., 1::2] << 4), torch.cat([a, z], -1)


def kv4_dequantize(b: torch.Tensor, pairs: torch.Tensor, dtype=torch.float32) -> torch.Tensor:
    """Values ``[T, H, hd]`` of :func:`kv4_quantize`'s output."""
    T, H, half = b.shape
    G = 2 * half // KV4_GROUP
    n = torch.stack([b & 15, b >> 4], -1).reshape(T, H, 8, G, 8).transpose(2, 3).reshape(T, H, G, KV4_GROUP)
    return (n.to(dtype) * pairs[..., :1].to(dtype) + pairs[..., 1:].to(dtype)).reshape(T, H, 2 * half)


def _kv4_slots(cache, slots):
    page = cache.k.shape[2]
    ok = (slots >= 0) & (slots < cache.k.shape[0] * page)
    s = slots.clamp(0, cache.k.shape[0] * page - 1).long()
    return ok, s // page, s % page


def kv4_write(k, v, cache, slots) -> None:
    ok, pg, off = _kv4_slots(cache, slots)
    for x, data, kv in ((k, cache.k, 0), (v, cache.v, 1)):
        b, pairs = kv4_quantize(x[ok])
        data[pg[ok], :, off[ok]] = b
        cache.scale[pg[ok], :, off[ok], kv] = pairs


def kv4_read(cache, slots, dtype=torch.float32):
    ok, pg, off = _kv4_slots(cache, slots)
    return tuple(torch.where(ok[:, None, None], kv4_dequantize(data[pg, :, off], cache.scale[pg, :, off, kv]), 0.0).to(dtype)
                 for data, kv in ((cache.k, 0), (cache.v, 1)))


def attention_decode_kv4(q, cache, block_table, seq_lens, scale: float | None = None) -> torch.Tensor:
    """:func:`attention_decode_paged` over the values of a 4-bit cache. Tokens of pages outside the cache or past the
    block table do not count; a row without tokens gives zeros."""
    return _attention_decode_read(kv4_read, q, cache, block_table, seq_lens, scale)


def _attention_decode_read(read, q, cache, block_table, seq_lens, scale):
    B, Hq, hd = q.shape
    pages, Hkv, page = cache.k.shape[:3]
    scale = scale if scale is not None else 1.0 / math.sqrt(hd)
    out = torch.zeros(B, Hq, hd, dtype=torch.float32, device=q.device)
    for b in range(B):
        t = torch.arange(max(0, min(int(seq_lens[b]), block_table.shape[1] * page)), device=q.device)
        pg = block_table[b, t // page].long()
        there = (pg >= 0) & (pg < pages)
        if not bool(there.any()):
            continue
        k, v = read(cache, (pg * page + t % page)[there])
        qb = q[b].float().view(Hkv, Hq // Hkv, hd)
        p = torch.softmax(torch.einsum("grd,lgd->grl", qb, k) * scale, dim=-1)
        out[b] = torch.einsum("grl,lgd->grd", p, v).reshape(Hq, hd)
    return out.to(q.dtype)


# ── 8-bit KV cache ───────────────────────────────────────────────────────────

KV8_BLOCK = 16
_KV8_LEAST, _KV8_MOST = 2.0 ** -100, 2.0 ** 126


def kv8_steps(amax: torch.Tensor) -> torch.Tensor:
    """Steps per unit ``r`` (fp32) of blocks with these largest magnitudes (:mod:`.kv8` describes the format)."""
    q = 127.0 / amax.float().clamp(_KV8_LEAST, _KV8_MOST)
    return torch.where(q.isnan(), q, (q.view(torch.int32) & -65536).view(torch.float32))


def kv8_write(k, v, cache, slots) -> None:
    pages, Hkv, page, hd = cache.k.shape
    ok = (slots >= 0) & (slots < pages * page)
    slots = slots[ok].long()
    which, mine = torch.unique(slots // KV8_BLOCK, return_inverse=True)
    per, place = page // KV8_BLOCK, slots % KV8_BLOCK
    for i in range(which.numel()):
        pg, bl = int(which[i]) // per, int(which[i]) % per
        at = place[mine == i]
        for x, data, kv in ((k, cache.k, 0), (v, cache.v, 1)):
            x = x[ok][mine == i].float()  # [rows, Hkv, hd]
            block = data[pg, :, bl * KV8_BLOCK:(bl + 1) * KV8_BLOCK]
            r = kv8_steps(x.abs().amax((0, 2)))
            if not bool((at == 0).any()):
                old = cache.scale[pg, :, bl, kv]
                r_old = torch.where(old == 0, torch.inf, 1.0 / old).bfloat16().float()
                r = torch.minimum(r, r_old)
                n = (block.float() - 128) * r[:, None, None] / r_old[:, None, None]
                block.copy_(torch.where((r < r_old)[:, None, None], (n.round() + 128).nan_to_num(0).to(torch.uint8), block))
            n = (x.clamp(-_KV8_MOST, _KV8_MOST) * r[:, None]).round().nan_to_num(0) + 128
            block[:, at] = n.to(torch.uint8).transpose(0, 1)
            cache.scale[pg, :, bl, kv] = 1.0 / r


def kv8_read(cache, slots, dtype=torch.float32):
    page = cache.k.shape[2]
    ok, pg, off = _kv4_slots(cache, slots)
    a = cache.scale[pg, :, off // KV8_BLOCK]
    return tuple(torch.where(ok[:, None, None], (data[pg, :, off].float() - 128) * a[..., kv, None], 0.0).to(dtype)
                 for data, kv in ((cache.k, 0), (cache.v, 1)))


def attention_decode_kv8(q, cache, block_table, seq_lens, scale: float | None = None) -> torch.Tensor:
    """:func:`attention_decode_paged` over the values of an 8-bit cache. Tokens of pages outside the cache or past the
    block table do not count; a row without tokens gives zeros."""
    return _attention_decode_read(kv8_read, q, cache, block_table, seq_lens, scale)


# ── paged tables ─────────────────────────────────────────────────────────────

def assign_pages(block_table, rows, have, need, pages) -> None:
    """See :func:`.paging.assign_pages`."""
    at, R, M = 0, *block_table.shape
    for row, h, n in zip(rows.tolist(), have.tolist(), need.tolist()):
        h = max(h, 0)
        got = pages[at:at + max(0, n - h)]
        at += max(0, n - h)
        if 0 <= row < R and h < M:
            got = got[:M - h]
            block_table[row, h:h + got.numel()] = got


def token_maps(block_table, rows, start, lens, total: int, page: int):
    """See :func:`.paging.token_maps`."""
    R, M = block_table.shape
    dev = block_table.device
    positions = torch.zeros(total, dtype=torch.int32, device=dev)
    slots = torch.full((total,), -1, dtype=torch.int64, device=dev)
    cu = [0]
    for row, s, n in zip(rows.tolist(), start.tolist(), lens.tolist()):
        n = max(n, 0)
        at, p = cu[-1], torch.arange(s, s + max(0, min(n, total - cu[-1])), dtype=torch.int64, device=dev)
        cu.append(at + n)
        positions[at:at + p.numel()] = p.int()
        if 0 <= row < R and M:
            pg = block_table[row].long()[(p // page).clamp(0, M - 1)]
            there = (p >= 0) & (p < M * page) & (p < 1 << 31) & (pg >= 0)
            slots[at:at + p.numel()] = torch.where(there, pg * page + p % page, -1)
    return positions, slots, torch.tensor(cu, dtype=torch.int64, device=dev).clamp(max=(1 << 31) - 1).int()


# ── logit controls ───────────────────────────────────────────────────────────

def _unpack_bits(words: torch.Tensor, n: int) -> torch.Tensor:
    sh = torch.arange(32, dtype=torch.int32, device=words.device)
    return ((words.unsqueeze(-1) >> sh) & 1).bool().flatten(-2)[..., :n]


def _set_bit(words: torch.Tensor, v: int) -> None:
    bit = v % 32
    words[v // 32] |= -(1 << 31) if bit == 31 else 1 << bit


def load_tokens(ctl, slots, tokens, cu_tokens, n_prompt) -> None:
    """Token state of admitted requests (see :mod:`.controls`)."""
    cu = cu_tokens.tolist()
    for i, slot in enumerate(slots.tolist()):
        if not 0 <= slot < ctl.counts.shape[0]:
            continue
        ctl.seen[slot] = 0
        ctl.counts[slot] = 0
        for j, v in enumerate(tokens[cu[i]:cu[i + 1]].tolist()):
            if 0 <= v < ctl.vocab:
                _set_bit(ctl.seen[slot], v)
                ctl.counts[slot, v] += j >= int(n_prompt[i])


def apply_logit_controls(logits, ctl, slots, new_tokens=None, done=None, out=None) -> torch.Tensor:
    """Penalties, biases and token masks on ``logits [B, V]`` (see :mod:`.controls`)."""
    out = torch.empty(logits.shape, dtype=torch.float32, device=logits.device) if out is None else out
    rows = []
    for b, s in enumerate(slots.tolist()):
        z = logits[b].float()
        if 0 <= s < ctl.counts.shape[0]:
            tok = int(new_tokens[b]) if new_tokens is not None and (done is None or int(done[b]) == 0) else -1
            if 0 <= tok < ctl.vocab:
                ctl.counts[s, tok] += 1
                _set_bit(ctl.seen[s], tok)
            c = ctl.counts[s].float()
            r = ctl.repetition[s]
            z = torch.where(_unpack_bits(ctl.seen[s], ctl.vocab), torch.where(z > 0, z / r, z * r), z)
            z = z - ctl.frequency[s] * c - torch.where(c > 0, ctl.presence[s], 0.0)
            ids = ctl.bias_ids[s].long()
            use = (ids >= 0) & (ids < ctl.vocab)
            z = z.index_add(0, ids[use], ctl.bias_vals[s][use])
            if int(ctl.mask_on[s]):
                z = z.masked_fill(~_unpack_bits(ctl.mask[s], ctl.vocab), float("-inf"))
        rows.append(z)
    for b, z in enumerate(rows):  # after every read: the two may share memory
        out[b] = z
    return out


# ── LM head + log-softmax + entropy ──────────────────────────────────────────

def lm_head_logprobs(
    h: torch.Tensor,       # [T, D]
    w: torch.Tensor,       # [V, D]
    labels: torch.Tensor,  # [T] long
    with_entropy: bool = True,
    chunk: int = 1024,
) -> tuple[torch.Tensor, torch.Tensor | None]:
    """``lp[t] = z[t, y_t] - logsumexp(z[t])`` and entropy, chunked over tokens."""
    lps, ents = [], []
    for s in range(0, h.shape[0], chunk):
        z = (h[s:s + chunk].float() @ w.float().t())
        lse = torch.logsumexp(z, dim=-1)
        lps.append(z.gather(-1, labels[s:s + chunk].long().unsqueeze(-1)).squeeze(-1) - lse)
        if with_entropy:
            p = torch.softmax(z, dim=-1)
            ents.append(lse - (p * z).sum(-1))
    lp = torch.cat(lps) if lps else h.new_zeros(0, dtype=torch.float32)
    ent = (torch.cat(ents) if ents else h.new_zeros(0, dtype=torch.float32)) if with_entropy else None
    return lp, ent


# ── sampling ────────────────────────────────────────────────────────────────

def sample_with_logprob(logits: torch.Tensor, temperature: float, generator=None,
                        top_k: int = -1, top_p: float = 1.0) -> tuple[torch.Tensor, torch.Tensor]:
    """Multinomial sample from ``softmax(logits / T)`` (+ top-k / top-p filter).

    Returns the token and its log-probability under the *filtered, tempered*
    distribution, which is what the rollout reports as the behaviour policy.
    """
    z = logits.float()
    if temperature <= 0:
        tok = z.argmax(-1)
        return tok, torch.zeros_like(tok, dtype=torch.float32)
    z = z / temperature
    if top_k > 0:
        kth = torch.topk(z, top_k, dim=-1).values[..., -1:]
        z = z.masked_fill(z < kth, float("-inf"))
    if top_p < 1.0:
        sz, idx = torch.sort(z, dim=-1, descending=True)
        cp = torch.softmax(sz, -1).cumsum(-1)
        drop = (cp - torch.softmax(sz, -1)) > top_p
        sz = sz.masked_fill(drop, float("-inf"))
        z = torch.full_like(z, float("-inf")).scatter(-1, idx, sz)
    logp = torch.log_softmax(z, dim=-1)
    tok = torch.multinomial(logp.exp(), 1, generator=generator).squeeze(-1)
    return tok, logp.gather(-1, tok.unsqueeze(-1)).squeeze(-1)


# ── PPO clipped loss (token level) ──────────────────────────────────────────

def ppo_token_terms(new_lp, old_lp, adv_tok, mask, eps_low, eps_high):
    """Per-token ``-min(r A, clip(r) A) * mask`` and the ratio."""
    ratio = torch.exp(new_lp - old_lp)
    pg = -torch.minimum(ratio * adv_tok, ratio.clamp(1 - eps_low, 1 + eps_high) * adv_tok)
    return pg * mask, ratio


# ── optimiser ───────────────────────────────────────────────────────────────

def adamw_(param, grad, exp_avg, exp_avg_sq, *, lr, beta1, beta2, eps, weight_decay, step, grad_scale=1.0):
    """Decoupled-weight-decay Adam on fp32 tensors, in place."""
    g = grad * grad_scale
    exp_avg.mul_(beta1).add_(g, alpha=1 - beta1)
    exp_avg_sq.mul_(beta2).addcmul_(g, g, value=1 - beta2)
    bc1 = 1 - beta1 ** step
    bc2 = 1 - beta2 ** step
    param.mul_(1 - lr * weight_decay)
    denom = (exp_avg_sq / bc2).sqrt_().add_(eps)
    param.addcdiv_(exp_avg, denom, value=-lr / bc1)


__all__ = [n for n in dir() if not n.startswith("_") and n not in ("math", "torch", "F", "annotations")]
