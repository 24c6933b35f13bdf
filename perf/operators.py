"""Cases, plain forms and 64-bit definitions of the sequence operators.

Three operators work on packed token rows and on a paged key-value cache:

  attention_packed   attention of sequences of different lengths packed one behind the other,
                     grouped heads, full or causal (a prompt, an image, a chunk behind a prefix)
  rope_append        rotates the new queries and keys by their positions and appends the keys and
                     values to the paged cache
  attention_paged    attention of one new token per sequence over the paged cache

A case is a dict of plain values; `run` is one pass of its operator on what `prepare` made. With
`own` false `run` computes the plain form in elementary torch operations and 32 bits.
"""
import os
import random
import sys

import torch

own = False

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
DTYPES = {"f16": torch.float16, "bf16": torch.bfloat16}
DEV = "cuda:0"


def _package():
    path = os.path.join(ROOT, "dinov3-loom_b200")
    if path not in sys.path:
        sys.path.insert(0, path)
    import dinov3_b200

    return dinov3_b200


# ---- the cases -----------------------------------------------------------------------------------
def _prompt(name, n, lo, hi, q_heads, kv_heads, dim, dtype, causal, cached=0, fused=False):
    """n sequences of lo..hi new tokens each, behind up to `cached` earlier keys."""
    return {"name": name, "op": "prompt", "n": n, "lo": lo, "hi": hi, "q_heads": q_heads, "kv_heads": kv_heads, "dim": dim, "dtype": dtype,
            "causal": causal, "cached": cached, "fused": fused}


def _append(name, n, lo, hi, q_heads, kv_heads, dim, dtype, page, cached):
    """lo..hi new tokens for each of n sequences that hold up to `cached` tokens."""
    return {"name": name, "op": "append", "n": n, "lo": lo, "hi": hi, "q_heads": q_heads, "kv_heads": kv_heads, "dim": dim, "dtype": dtype,
            "page": page, "cached": cached}


def _decode(name, n, lo, hi, q_heads, kv_heads, dim, dtype, page):
    """One new token for each of n sequences of lo..hi cached tokens."""
    return {"name": name, "op": "decode", "n": n, "lo": lo, "hi": hi, "q_heads": q_heads, "kv_heads": kv_heads, "dim": dim, "dtype": dtype,
            "page": page}


def listed():
    return [
        # a single short prompt on a small decoder: latency
        _prompt("prompt short", 1, 37, 37, 8, 2, 64, "bf16", True),
        # a batch of images at the model's own size, read from the fused QKV rows
        _prompt("prompt images", 64, 201, 201, 6, 6, 64, "f16", False, fused=True),
        # a serving step's prompts, of very different lengths
        _prompt("prompt ragged", 24, 1, 2048, 32, 8, 128, "bf16", True),
        # the next chunk of long prompts, whose first part is cached already
        _prompt("prompt chunk", 4, 300, 512, 32, 8, 128, "f16", True, cached=4096),
        # one long document
        _prompt("prompt long", 1, 16384, 16384, 32, 8, 128, "bf16", True),
        # one user's next token on a small decoder: latency
        _append("append one", 1, 1, 1, 8, 2, 64, "f16", 16, 130),
        # a serving step of one token for each of 64 users
        _append("append tokens", 64, 1, 1, 32, 8, 128, "bf16", 16, 1000),
        # the prompts of a serving step, pages that are no power of two
        _append("append prompts", 16, 1, 4096, 32, 8, 128, "f16", 48, 0),
        # one user's next token on a small decoder: latency
        _decode("decode one", 1, 130, 130, 8, 2, 64, "f16", 16),
        # captions: one query per image over the 201 tokens of each of 256 images, three pages each
        _decode("decode images", 256, 201, 201, 6, 6, 64, "f16", 67),
        # a serving step of 64 users with contexts of very different lengths
        _decode("decode ragged", 64, 1, 4096, 32, 8, 128, "bf16", 16),
        # one user with a long document: the cache's length has to be split
        _decode("decode long", 1, 131072, 131072, 32, 8, 128, "f16", 64),
    ]


def _log_int(rng, lo, hi):
    return min(hi, max(lo, int(round(lo * (hi / lo) ** rng.random()))))


def draw(rng):
    kv_heads = rng.choice([1, 2, 3, 4, 6, 8])
    group = rng.choice([1, 2, 3, 4, 5, 7, 8])
    dim, dtype = rng.choice([64, 128]), rng.choice(["f16", "bf16"])
    page = rng.choice([8, 16, 16, 32, 48, 64, 67, 128])
    op = rng.choice(["prompt", "append", "decode"])
    n = _log_int(rng, 1, 64)
    heads = (group * kv_heads, kv_heads, dim, dtype)
    if op == "prompt":
        hi = _log_int(rng, 1, 8192)
        lo = rng.choice([1, hi, _log_int(rng, 1, hi)])
        cached = rng.choice([0, 0, _log_int(rng, 1, 4096)])
        while n * heads[0] * hi * (hi + cached) > 1 << 32:  # scores of the padded batch
            n, hi = max(1, n // 2), (hi + 1) // 2 if n == 1 else hi
        c = _prompt("", n, min(lo, hi), hi, *heads, rng.random() < 0.6, cached, cached == 0 and rng.random() < 0.5)
    elif op == "append":
        hi = rng.choice([1, _log_int(rng, 1, 4096)])
        while n * hi > 1 << 15:
            n = max(1, n // 2)
        c = _append("", n, rng.choice([1, hi]), hi, *heads, page, _log_int(rng, 1, 1024))
    else:
        hi = _log_int(rng, 1, 65536)
        while n * hi > 1 << 17:
            n = max(1, n // 2)
        c = _decode("", n, rng.choice([1, hi, _log_int(rng, 1, hi)]), hi, *heads, page)
    del c["name"]
    return c


def _lengths(case, lo, hi, tag):
    """The case's sequence lengths, spread over the logarithm of lo..hi; the longest is hi."""
    rng = random.Random("%s %d %d %d" % (tag, case["n"], lo, hi))
    got = [hi] + [_log_int(rng, lo, hi) for _ in range(case["n"] - 1)]
    rng.shuffle(got)
    return got


def _new_and_total(case):
    """Each sequence's new tokens, and its tokens with those it held before."""
    new = _lengths(case, case["lo"], case["hi"], "new")
    held = _lengths(case, 1, case["cached"], "held") if case["cached"] else [0] * case["n"]
    return new, [a + b for a, b in zip(new, held)]


def work(case):
    hq, hkv, d = case["q_heads"], case["kv_heads"], case["dim"]
    if case["op"] == "prompt":
        new, total = _new_and_total(case)
        pairs = sum(a * b - (a * (a - 1) // 2 if case["causal"] else 0) for a, b in zip(new, total))
        return {"bytes": 2 * d * (2 * hq * sum(new) + 2 * hkv * sum(total)), "flops": 4 * d * hq * pairs}
    if case["op"] == "append":
        new, _ = _new_and_total(case)
        t = sum(new)
        return {"bytes": 2 * 2 * d * t * (hq + 2 * hkv) + 4 * d * t, "flops": 3 * d * t * (hq + hkv)}
    t = sum(_lengths(case, case["lo"], case["hi"], "new"))
    return {"bytes": 2 * d * (2 * hkv * t + 2 * hq * case["n"]), "flops": 4 * d * hq * t}


# ---- what a user's program has in hand -----------------------------------------------------------
def _cu(lengths):
    cu = [0]
    for x in lengths:
        cu.append(cu[-1] + x)
    return torch.tensor(cu, dtype=torch.int32, device=DEV)


def _paged(case, totals, gen, dtype):
    """A shuffled page table over a pool of random pages, with a few pages nobody holds; entries
    behind a sequence's last page are -1."""
    page, hkv, d = case["page"], case["kv_heads"], case["dim"]
    counts = [-(-t // page) for t in totals]
    pool = sum(counts) + 3
    order = torch.randperm(pool, generator=gen, device=DEV).to(torch.int32)
    wide = max(counts)
    col = torch.arange(wide, device=DEV)
    cu = _cu(counts)
    table = order[(cu[:-1, None] + col).clamp(max=pool - 1).long()]
    table = torch.where(col < torch.tensor(counts, device=DEV)[:, None], table, -1).contiguous()
    k = torch.randn(pool, hkv, page, d, generator=gen, device=DEV, dtype=dtype)
    v = torch.randn(pool, hkv, page, d, generator=gen, device=DEV, dtype=dtype)
    return table, k, v


def prepare(case, seed):
    gen = torch.Generator(device=DEV)
    gen.manual_seed(seed)
    dtype, hq, hkv, d = DTYPES[case["dtype"]], case["q_heads"], case["kv_heads"], case["dim"]

    def rows(n, heads, scale=1.0):
        return torch.randn(n, heads, d, generator=gen, device=DEV, dtype=dtype) * scale

    s = {"op": case["op"], "scale": d ** -0.5}
    if case["op"] == "decode":
        lengths = _lengths(case, case["lo"], case["hi"], "new")
        s["q"] = rows(case["n"], hq, 2.0)
        s["table"], s["k"], s["v"] = _paged(case, lengths, gen, dtype)
        s["lens"] = torch.tensor(lengths, dtype=torch.int32, device=DEV)
        s["max_len"] = max(lengths)
        return s
    new, total = _new_and_total(case)
    s["cu_q"] = _cu(new)
    if case["op"] == "append":
        s["q"], s["new_k"], s["new_v"] = rows(sum(new), hq), rows(sum(new), hkv), rows(sum(new), hkv)
        s["table"], s["k"], s["v"] = _paged(case, total, gen, dtype)
        s["lens"] = torch.tensor(total, dtype=torch.int32, device=DEV)
        s["one"] = case["hi"] == 1
        # the rotation's tables over the positions that the program allows for
        angle = torch.arange(max(total) + 64, device=DEV, dtype=torch.float64)[:, None] * 10000.0 ** (-torch.arange(0, d, 2, device=DEV, dtype=torch.float64) / d)
        s["cos"], s["sin"] = angle.cos().float(), angle.sin().float()
        return s
    s["causal"], s["max_q"], s["max_k"] = case["causal"], max(new), max(total)
    if case["fused"]:
        qkv = rows(sum(new), hq + 2 * hkv)
        s["q"], s["new_k"], s["new_v"] = qkv[:, :hq], qkv[:, hq:hq + hkv], qkv[:, hq + hkv:]
        s["cu_k"] = s["cu_q"]
    else:
        s["q"], s["new_k"], s["new_v"] = rows(sum(new), hq, 2.0), rows(sum(total), hkv), rows(sum(total), hkv)
        s["cu_k"] = _cu(total) if case["cached"] else s["cu_q"]
    return s


# ---- one pass ------------------------------------------------------------------------------------
def run(s):
    if own:
        dv = _package()
        if s["op"] == "prompt":
            return dv.attention_packed(s["q"], s["new_k"], s["new_v"], s["cu_q"], s["cu_k"], causal=s["causal"], scale=s["scale"])
        if s["op"] == "append":
            q = dv.rope_append(s["q"], s["new_k"], s["new_v"], s["k"], s["v"], s["table"], s["lens"], s["cos"], s["sin"], cu_new=None if s["one"] else s["cu_q"])
            return q, s["k"], s["v"]
        return dv.attention_paged(s["q"], s["k"], s["v"], s["table"], s["lens"], max_len=s["max_len"], scale=s["scale"])
    return {"prompt": _plain_packed, "append": _plain_append, "decode": _plain_paged}[s["op"]](s)


def _token_places(cu, n):
    """Sequence and index within it of each of n packed rows."""
    t = torch.arange(n, device=DEV)
    seq = torch.searchsorted(cu, t.to(torch.int32), right=True) - 1
    return seq, t - cu[seq]


def _plain_softmax_product(scores, allowed, values):
    """softmax over the allowed scores (changed in place) times the values; 0 where none is."""
    scores.masked_fill_(~allowed, float("-inf"))
    top = scores.amax(-1, keepdim=True).clamp(min=torch.finfo(torch.float32).min)
    scores.sub_(top).exp_()
    total = scores.sum(-1, keepdim=True)
    return scores.flatten(2, -2) @ values / total.clamp(min=1e-37).flatten(2, -2)


def _plain_packed(s):
    q, k, v, cu_q, cu_k = s["q"], s["new_k"], s["new_v"], s["cu_q"], s["cu_k"]
    (total_q, hq, d), hkv, n, lq, lk = q.shape, k.shape[1], cu_q.numel() - 1, s["max_q"], s["max_k"]
    group = hq // hkv
    at_q, at_k = torch.arange(lq, device=DEV), torch.arange(lk, device=DEV)
    len_q, len_k = cu_q.diff(), cu_k.diff()
    pq = q[(cu_q[:-1, None] + at_q).clamp(max=total_q - 1).long()].float() * s["scale"]
    rows_k = (cu_k[:-1, None] + at_k).clamp(max=k.shape[0] - 1).long()
    pq = pq.view(n, lq, hkv, group, d).permute(0, 2, 3, 1, 4).reshape(n, hkv, group * lq, d)
    allowed = (at_k < len_k[:, None])[:, None, :]
    if s["causal"]:
        allowed = allowed & (at_k <= at_q[:, None] + (len_k - len_q)[:, None, None])
    scores = (pq @ k[rows_k].float().permute(0, 2, 3, 1)).view(n, hkv, group, lq, lk)
    out = _plain_softmax_product(scores, allowed[:, None, None], v[rows_k].float().permute(0, 2, 1, 3))
    seq, pos = _token_places(cu_q, total_q)
    return out.view(n, hkv, group, lq, d)[seq, :, :, pos].reshape(total_q, hq, d).to(q.dtype)


def _plain_rotated(x, cos, sin):
    half = cos.shape[-1]
    a, b = x[..., :half].float(), x[..., half:].float()
    cos, sin = cos[:, None], sin[:, None]
    return torch.cat([a * cos - b * sin, b * cos + a * sin], -1).to(x.dtype)


def _plain_append(s):
    q, table, page = s["q"], s["table"], s["k"].shape[2]
    seq, index = _token_places(s["cu_q"], q.shape[0])
    pos = s["lens"][seq] - s["cu_q"].diff()[seq] + index
    cos, sin = s["cos"][pos], s["sin"][pos]
    at, slot = table[seq, pos // page].long(), (pos % page).long()
    s["k"][at, :, slot] = _plain_rotated(s["new_k"], cos, sin)
    s["v"][at, :, slot] = s["new_v"]
    return _plain_rotated(q, cos, sin), s["k"], s["v"]


def _plain_paged(s):
    q, table, lens = s["q"], s["table"].clamp(min=0).long(), s["lens"]
    (n, hq, d), (_, hkv, page, _) = q.shape, s["k"].shape
    k, v = (s[x][table].permute(0, 2, 1, 3, 4).reshape(n, hkv, -1, d).float() for x in ("k", "v"))
    scores = (q.float() * s["scale"]).view(n, hkv, hq // hkv, d) @ k.transpose(2, 3)
    allowed = torch.arange(k.shape[2], device=DEV) < lens[:, None]
    return _plain_softmax_product(scores, allowed[:, None, None], v).view(n, hq, d).to(q.dtype)


# ---- the definitions in 64 bits ------------------------------------------------------------------
def _exact_rows(q, k, v, scale, visible):
    """Attention of one sequence: q [a, hq, d], k and v [b, hkv, d]; row i sees visible[i] keys."""
    a, hq, d = q.shape
    b, hkv, _ = k.shape
    out = torch.zeros(a, hq, d, dtype=torch.float64, device=DEV)
    hidden = torch.arange(b, device=DEV)[None, :] >= visible[:, None]
    for h in range(hq):
        g = h // (hq // hkv)
        w = torch.einsum("id,jd->ij", q[:, h].double(), k[:, g].double()).mul_(scale).masked_fill_(hidden, -1e300)
        w = torch.softmax(w, 1).masked_fill_(hidden, 0.0)
        out[:, h] = w @ v[:, g].double()
    return out


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "prompt":
        new, total = _new_and_total(case)
        out, tq, tk = [], 0, 0
        for a, b in zip(new, total):
            visible = torch.full((a,), b, device=DEV)
            if case["causal"]:
                visible = torch.arange(a, device=DEV) + (b - a + 1)
            out.append(_exact_rows(s["q"][tq:tq + a], s["new_k"][tk:tk + b], s["new_v"][tk:tk + b], s["scale"], visible))
            tq, tk = tq + a, tk + b
        return torch.cat(out)
    page, hkv, d = case["page"], case["kv_heads"], case["dim"]
    if case["op"] == "decode":
        out = []
        for i, b in enumerate(_lengths(case, case["lo"], case["hi"], "new")):
            ids = s["table"][i, : -(-b // page)].long()
            k, v = (s[x][ids].transpose(1, 2).reshape(-1, hkv, d)[:b] for x in ("k", "v"))
            out.append(_exact_rows(s["q"][i:i + 1], k, v, s["scale"], torch.tensor([b], device=DEV)))
        return torch.cat(out)
    new, total = _new_and_total(case)
    turn = torch.complex(s["cos"].double(), s["sin"].double())

    def turned(x, first):
        z = torch.complex(*x.double().chunk(2, -1)) * turn[first:first + x.shape[0], None]
        return torch.cat([z.real, z.imag], -1)

    q, k, v, t = [], s["k"].double(), s["v"].double(), 0
    for i, (a, b) in enumerate(zip(new, total)):
        q.append(turned(s["q"][t:t + a], b - a))
        pos = torch.arange(b - a, b, device=DEV)
        ids = s["table"][i].long()[pos // page]
        k[ids, :, pos % page] = turned(s["new_k"][t:t + a], b - a)
        v[ids, :, pos % page] = s["new_v"][t:t + a].double()
        t += a
    return torch.cat(q), k, v
