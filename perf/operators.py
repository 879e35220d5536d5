"""Attention over whole prompts and over a paged key-value cache: the three operators, their plain forms and the cases they are measured on.

    append    writes the keys and values of new tokens into the pages of their sequences (optionally rotating q and k by position)
    decode    attention of one new token per sequence over its pages
    prefill   attention of whole prompts, packed one after the other, causal or not

`run` computes the plain form (elementary torch operations in 32 bits) or, with `own` set, calls nemotron_infer_b200.ops.
"""
import math
import random

import torch

own = False

DEV = "cuda"
BF = torch.bfloat16
E4M3 = torch.float8_e4m3fn

# The model's attention: 40 query heads over 8 key-value heads of 128, a default context of 2048 tokens.
Q_HEADS, KV_HEADS, HEAD = 40, 8, 128


def listed():
    return [
        # ---- append ----
        # one decode step of a small batch: 32 new tokens, latency only
        _append("append step 32 sequences", batch=32, new=1, prefix=500, page=64, rot=128),
        # a pack of prompts of different lengths, q / k / v as views of one projection's output, rows of padding behind the last
        _append("append ragged prompts", batch=9, new=1100, prefix=0, page=32, rot=64, interleaved=True, strided=True, pad=37, ragged=True),
        # a long prompt into an 8-bit cache, no rotation (the model has none)
        _append("append prompt 16384 e4m3", batch=1, new=16384, prefix=0, page=64, rot=0, cache="e4m3"),
        # ---- decode ----
        # one sequence at a short context: the latency of a single user's step
        _decode("decode 1 x 512", batch=1, length=512, page=64),
        # one sequence at a very long context: the whole GPU on one cache
        _decode("decode 1 x 131071", batch=1, length=131071, page=64),
        # a server's batch, every length between a few tokens and the limit, 8-bit cache
        _decode("decode ragged 64 e4m3", batch=64, length=8192, page=16, ragged=True, cache="e4m3"),
        # a full batch at long context: bandwidth
        _decode("decode 192 x 4000", batch=192, length=4000, page=64),
        # other head layout: one key-value head per query head, 64 wide
        _decode("decode 33 x 1500 heads of 64", batch=33, length=1500, page=32, ragged=True, q_heads=16, kv_heads=16, head=64),
        # ---- prefill ----
        # one short prompt
        _prefill("prefill 1 x 200", batch=1, length=200),
        # a pack of prompts of different lengths, views of one projection's output, padding behind the last
        _prefill("prefill ragged 24", batch=24, length=2048, ragged=True, strided=True, pad=50),
        # the next chunk of prompts whose first part is cached already, heads of 64
        _prefill("prefill chunk after prefix", batch=4, length=1000, prefix=5000, q_heads=32, kv_heads=4, head=64, ragged=True),
        # one long prompt
        _prefill("prefill 1 x 16384", batch=1, length=16384),
    ]


def _append(name, batch, new, prefix, page, rot, q_heads=Q_HEADS, kv_heads=KV_HEADS, head=HEAD, cache="bf16", interleaved=False, strided=False,
            pad=0, ragged=False, lens=1):
    return dict(name=name, op="append", batch=batch, new=new, prefix=prefix, page=page, rot=rot, q_heads=q_heads, kv_heads=kv_heads, head=head,
                cache=cache, interleaved=interleaved, strided=strided, pad=pad, ragged=ragged, lens=lens)


def _decode(name, batch, length, page, q_heads=Q_HEADS, kv_heads=KV_HEADS, head=HEAD, cache="bf16", ragged=False, lens=1):
    return dict(name=name, op="decode", batch=batch, length=length, page=page, q_heads=q_heads, kv_heads=kv_heads, head=head, cache=cache,
                ragged=ragged, lens=lens)


def _prefill(name, batch, length, prefix=0, q_heads=Q_HEADS, kv_heads=KV_HEADS, head=HEAD, causal=True, strided=False, pad=0, ragged=False, lens=1):
    return dict(name=name, op="prefill", batch=batch, length=length, prefix=prefix, q_heads=q_heads, kv_heads=kv_heads, head=head, causal=causal,
                strided=strided, pad=pad, ragged=ragged, lens=lens)


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 1)))))))


def draw(rng):
    op = rng.choice(["append", "decode", "decode", "prefill", "prefill"])
    ratio = rng.choice([1, 2, 4, 5, 8, 16])
    kv_heads = rng.choice([1, 2, 3, 4, 8])
    head = rng.choice([64, 128, 128])
    heads = dict(q_heads=kv_heads * ratio, kv_heads=kv_heads, head=head)
    if heads["q_heads"] > 64:
        heads.update(q_heads=5 * kv_heads)
    page = rng.choice([8, 16, 32, 64, 128])
    cache = rng.choice(["bf16", "bf16", "e4m3"])
    lens = rng.randrange(1 << 20)
    if op == "append":
        batch = _log(rng, 1, 200)
        new = 1 if rng.random() < 0.3 else _log(rng, 1, 16384 // batch)
        c = _append("", batch=batch, new=new, prefix=rng.choice([0, _log(rng, 1, 1000)]), page=page, rot=rng.choice([0, 32, 64, head]), cache=cache,
                    interleaved=rng.random() < 0.5, strided=rng.random() < 0.5, pad=rng.choice([0, rng.randrange(1, 60)]), ragged=new > 1 and rng.random() < 0.7,
                    lens=lens, **heads)
    elif op == "decode":
        batch = _log(rng, 1, 192)
        c = _decode("", batch=batch, length=_log(rng, 1, min(131071, 768000 // batch)), page=page, cache=cache, ragged=rng.random() < 0.6, lens=lens, **heads)
    else:
        batch = _log(rng, 1, 32)
        c = _prefill("", batch=batch, length=_log(rng, 1, int(16384 / math.sqrt(batch))), prefix=rng.choice([0, 0, _log(rng, 1, 4000 // batch + 1)]),
                     causal=rng.random() < 0.75, strided=rng.random() < 0.5, pad=rng.choice([0, rng.randrange(1, 90)]), ragged=rng.random() < 0.6, lens=lens, **heads)
        cost = lambda k: work(k)["flops"]
        while cost(c) > cost(_prefill("", batch=1, length=16384)):
            c["length"] = max(1, c["length"] * 3 // 4)
    del c["name"]
    return c


def _lengths(case, most, salt):
    """One length per sequence: all `most`, or spread over the logarithm of 1 .. most with the longest among them."""
    b = case["batch"]
    if not case.get("ragged") or most <= 1:
        return [most] * b
    rng = random.Random(case["lens"] * 31 + salt)
    ls = [_log(rng, 1, most) for _ in range(b)]
    ls[rng.randrange(b)] = most
    return ls


def _seq(case):
    """(new tokens, tokens in the cache after them) of every sequence."""
    if case["op"] == "decode":
        ls = _lengths(case, case["length"], 1)
        return [1] * case["batch"], ls
    new = _lengths(case, case["new"] if case["op"] == "append" else case["length"], 1)
    pre = _lengths(case, case["prefix"], 2) if case["prefix"] else [0] * case["batch"]
    return new, [n + p for n, p in zip(new, pre)]


def work(case):
    new, total = _seq(case)
    hq, hk, d = case["q_heads"], case["kv_heads"], case["head"]
    t = sum(new)
    if case["op"] == "append":
        cb = 1 if case["cache"] == "e4m3" else 2
        nbytes = t * hk * d * 2 * (2 + cb)
        flops = 0
        if case["rot"]:
            nbytes += t * hq * d * 4 + t * case["rot"] * 4
            flops = t * (hq + hk) * case["rot"] * 3
        return {"bytes": nbytes, "flops": flops}
    if case["op"] == "decode":
        cb = 1 if case["cache"] == "e4m3" else 2
        return {"bytes": sum(total) * hk * d * 2 * cb + case["batch"] * hq * d * 4, "flops": 4 * hq * d * sum(total)}
    pairs = sum(n * m - (n * (n - 1) // 2 if case["causal"] else 0) for n, m in zip(new, total))
    return {"bytes": t * hq * d * 4 + sum(total) * hk * d * 4, "flops": 4 * d * hq * pairs}


# ---------------------------------------------------------------------------------------------------------------------
# inputs
# ---------------------------------------------------------------------------------------------------------------------
def _randn(g, *shape):
    return torch.randn(*shape, generator=g, device=DEV)


def _cu(lens):
    out = [0]
    for n in lens:
        out.append(out[-1] + n)
    return torch.tensor(out, dtype=torch.int32, device=DEV)


def _pages(case, total, g):
    """A page table whose pages are scattered over the cache, with a few pages nobody uses."""
    p = case["page"]
    need = [(n + p - 1) // p for n in total]
    num = sum(need) + 3
    perm = torch.randperm(num, generator=g, device=DEV).to(torch.int32)
    table = torch.zeros(len(total), max(max(need), 1), dtype=torch.int32, device=DEV)
    at = 0
    for b, n in enumerate(need):
        table[b, :n] = perm[at:at + n]
        at += n
    return table, num


def _cache(case, num, g):
    shape = (num, case["kv_heads"], case["page"], case["head"])
    k, v = _randn(g, *shape), _randn(g, *shape) + 0.25
    if case["cache"] == "e4m3":
        ks, vs = torch.full((1,), 0.02, device=DEV), torch.full((1,), 0.03, device=DEV)
        return (k / ks).clamp(-448, 448).to(E4M3), (v / vs).clamp(-448, 448).to(E4M3), ks, vs
    return k.to(BF), v.to(BF), None, None


def _qkv(case, t_q, t_k, g):
    hq, hk, d = case["q_heads"], case["kv_heads"], case["head"]
    if case["strided"] and t_q == t_k:
        x = _randn(g, t_q, hq + 2 * hk, d)
        x[:, hq + hk:] += 0.25
        x = x.to(BF)
        return x[:, :hq], x[:, hq:hq + hk], x[:, hq + hk:]
    return _randn(g, t_q, hq, d).to(BF), _randn(g, t_k, hk, d).to(BF), (_randn(g, t_k, hk, d) + 0.25).to(BF)


def _rope_rows(positions, rot):
    """cos | sin of position * 10000^(-2 i / rot), i < rot / 2: the rows a model computes once."""
    inv = 10000.0 ** (-torch.arange(0, rot, 2, dtype=torch.float64, device=DEV) / rot)
    a = torch.arange(positions, dtype=torch.float64, device=DEV)[:, None] * inv
    return torch.cat([a.cos(), a.sin()], dim=1).float()


def prepare(case, seed):
    g = torch.Generator(device=DEV)
    g.manual_seed(int(seed))
    new, total = _seq(case)
    s = dict(case=case, scale=1.0 / math.sqrt(case["head"]), new=new, total=total)
    if case["op"] == "prefill":
        t, m = sum(new), sum(total)
        s["q"], s["k"], s["v"] = _qkv(case, t + case["pad"], m + case["pad"], g)
        s["cu"] = _cu(new)
        s["cu_k"] = _cu(total) if total != new else None
        # rows of padding stay as they are: the result goes into a buffer of the program's own
        s["out"] = torch.zeros(t + case["pad"], case["q_heads"], case["head"], dtype=BF, device=DEV)
        return s
    s["table"], num = _pages(case, total, g)
    s["k_cache"], s["v_cache"], s["k_scale"], s["v_scale"] = _cache(case, num, g)
    s["lens"] = torch.tensor(total, dtype=torch.int32, device=DEV)
    if case["op"] == "decode":
        s["q"] = _randn(g, case["batch"], case["q_heads"], case["head"]).to(BF)
        if own:
            from nemotron_infer_b200 import ops
            s["workspace"] = ops.sdpa_decode_paged_workspace(case["batch"], case["q_heads"], case["kv_heads"], case["head"], DEV)
        return s
    t = sum(new)
    s["q"], s["k"], s["v"] = _qkv(case, t + case["pad"], t + case["pad"], g)
    s["cu"] = _cu(new) if max(new) > 1 or case["pad"] else None
    if case["rot"]:
        s["rope"] = _rope_rows(max(total), case["rot"])
        s["q_out"] = torch.zeros(t + case["pad"], case["q_heads"], case["head"], dtype=BF, device=DEV)
    return s


# ---------------------------------------------------------------------------------------------------------------------
# one pass
# ---------------------------------------------------------------------------------------------------------------------
def run(s):
    op = s["case"]["op"]
    if own:
        from nemotron_infer_b200 import ops
        if op == "prefill":
            return ops.sdpa_prefill(s["q"], s["k"], s["v"], s["cu"], s["cu_k"], causal=s["case"]["causal"], out=s["out"])
        if op == "decode":
            return ops.sdpa_decode_paged(s["q"], s["k_cache"], s["v_cache"], s["table"], s["lens"], k_scale=s["k_scale"], v_scale=s["v_scale"],
                                         workspace=s["workspace"])
        if s["case"]["rot"]:
            q = ops.kv_append_paged(s["k"], s["v"], s["k_cache"], s["v_cache"], s["table"], s["lens"], s["cu"], q=s["q"], rope=s["rope"],
                                    interleaved=s["case"]["interleaved"], k_scale=s["k_scale"], v_scale=s["v_scale"], q_out=s["q_out"])
            return {"q": q, "k_cache": s["k_cache"], "v_cache": s["v_cache"]}
        ops.kv_append_paged(s["k"], s["v"], s["k_cache"], s["v_cache"], s["table"], s["lens"], s["cu"], k_scale=s["k_scale"], v_scale=s["v_scale"])
        return {"k_cache": s["k_cache"], "v_cache": s["v_cache"]}
    return {"append": _plain_append, "decode": _plain_decode, "prefill": _plain_prefill}[op](s)


def _rotate(x, cos, sin, interleaved):
    """x [T, H, D] in 32 bits; cos, sin [T, rot / 2]: the first rot entries of every head are turned in pairs."""
    r = cos.shape[1]
    cos, sin = cos[:, None], sin[:, None]
    y = x.clone()
    if interleaved:
        a, b = x[..., 0:2 * r:2], x[..., 1:2 * r:2]
        y[..., 0:2 * r:2], y[..., 1:2 * r:2] = a * cos - b * sin, b * cos + a * sin
    else:
        a, b = x[..., :r], x[..., r:2 * r]
        y[..., :r], y[..., r:2 * r] = a * cos - b * sin, b * cos + a * sin
    return y


def _plain_append(s):
    case = s["case"]
    t = sum(s["new"])
    page = case["page"]
    tok = torch.arange(t, device=DEV)
    cu = s["cu"].long() if s["cu"] is not None else torch.arange(case["batch"] + 1, device=DEV)
    seq = torch.searchsorted(cu, tok, right=True) - 1
    pos = s["lens"].long()[seq] - (cu[seq + 1] - tok)
    slot_page, slot = s["table"][seq, pos // page].long(), pos % page
    k, v = s["k"][:t].float(), s["v"][:t].float()
    if case["rot"]:
        half = case["rot"] // 2
        cos, sin = s["rope"][pos, :half], s["rope"][pos, half:]
        k = _rotate(k, cos, sin, case["interleaved"])
        s["q_out"][:t] = _rotate(s["q"][:t].float(), cos, sin, case["interleaved"]).to(BF)
    if case["cache"] == "e4m3":
        k, v = (k / s["k_scale"]).clamp(-448, 448).to(E4M3), (v / s["v_scale"]).clamp(-448, 448).to(E4M3)
        s["k_cache"].view(torch.uint8)[slot_page, :, slot] = k.view(torch.uint8)
        s["v_cache"].view(torch.uint8)[slot_page, :, slot] = v.view(torch.uint8)
    else:
        s["k_cache"][slot_page, :, slot] = k.to(BF)
        s["v_cache"][slot_page, :, slot] = v.to(BF)
    out = {"k_cache": s["k_cache"], "v_cache": s["v_cache"]}
    if case["rot"]:
        out["q"] = s["q_out"]
    return out


def _plain_decode(s):
    """A few sequences at a time: their pages gathered, scores, softmax with the masked places left out, weighted sum."""
    case = s["case"]
    hq, hk, d, page = case["q_heads"], case["kv_heads"], case["head"], case["page"]
    out = torch.empty(case["batch"], hq, d, dtype=BF, device=DEV)
    width = s["table"].shape[1] * page
    step = max(1, (1 << 28) // (width * hk * d))
    cache_k, cache_v = (c.view(torch.uint8) if case["cache"] == "e4m3" else c for c in (s["k_cache"], s["v_cache"]))
    for b in range(0, case["batch"], step):
        rows = s["table"][b:b + step].long()
        n = rows.shape[0]
        k, v = (c[rows].view(s["k_cache"].dtype).float().permute(0, 2, 1, 3, 4).reshape(n, hk, width, d) for c in (cache_k, cache_v))
        if case["cache"] == "e4m3":
            k, v = k * s["k_scale"], v * s["v_scale"]
        keep = (torch.arange(width, device=DEV) < s["lens"][b:b + step, None])[:, None, None]
        q = s["q"][b:b + step].float().view(n, hk, hq // hk, d)
        x = (q @ k.transpose(-1, -2) * s["scale"]).masked_fill(~keep, -math.inf)
        top = x.amax(-1, keepdim=True)
        p = torch.exp(x - torch.where(top == -math.inf, 0.0, top))
        o = (p @ torch.where(keep.transpose(-1, -2), v, 0.0)) / p.sum(-1, keepdim=True).clamp_min(1e-30)
        out[b:b + step] = o.reshape(n, hq, d).to(BF)
    return out


def _plain_prefill(s):
    """Sequence by sequence, a block of queries at a time against the keys that the last of them sees."""
    case = s["case"]
    hq, hk, d = case["q_heads"], case["kv_heads"], case["head"]
    at = at_k = 0
    for n, m in zip(s["new"], s["total"]):
        k = s["k"][at_k:at_k + m].float().permute(1, 2, 0)[:, None]
        v = s["v"][at_k:at_k + m].float().permute(1, 0, 2)[:, None]
        q = s["q"][at:at + n].float().permute(1, 0, 2).reshape(hk, hq // hk, n, d)
        step = max(1, (1 << 28) // (m * hq))
        for i in range(0, n, step):
            e = min(n, i + step)
            sees = m - n + e if case["causal"] else m
            x = q[:, :, i:e] @ k[..., :sees] * s["scale"]
            if case["causal"]:
                late = torch.arange(sees, device=DEV)[None, :] > torch.arange(i, e, device=DEV)[:, None] + (m - n)
                x.masked_fill_(late, -math.inf)
            top = x.amax(-1, keepdim=True)
            p = torch.exp(x - top)
            o = (p @ v[..., :sees, :]) / p.sum(-1, keepdim=True)
            s["out"][at + i:at + e] = o.reshape(hq, e - i, d).transpose(0, 1).to(BF)
        at, at_k = at + n, at_k + m
    return s["out"]


# ---------------------------------------------------------------------------------------------------------------------
# 64 bits
# ---------------------------------------------------------------------------------------------------------------------
def exact(case, seed):
    s = prepare(case, seed)
    return {"append": _exact_append, "decode": _exact_decode, "prefill": _exact_prefill}[case["op"]](s)


def _exact_append(s):
    """Token by token position along each sequence; a rotation is a product with e^(i angle) of the table's own cosines and sines."""
    case = s["case"]
    rot = case["rot"]
    ks = s["k_scale"].double() if s["k_scale"] is not None else 1.0
    vs = s["v_scale"].double() if s["v_scale"] is not None else 1.0
    kc, vc = s["k_cache"].double(), s["v_cache"].double()
    qo = s["q_out"].double() if rot else None

    def turn(x, pos):
        x = x.double().clone()
        if rot:
            rows = s["rope"][pos].double()
            unit = torch.complex(rows[:, :rot // 2], rows[:, rot // 2:])[:, None]
            if case["interleaved"]:
                z = torch.complex(x[..., 0:rot:2].contiguous(), x[..., 1:rot:2].contiguous()) * unit
                x[..., 0:rot:2], x[..., 1:rot:2] = z.real, z.imag
            else:
                z = torch.complex(x[..., :rot // 2].contiguous(), x[..., rot // 2:rot].contiguous()) * unit
                x[..., :rot // 2], x[..., rot // 2:rot] = z.real, z.imag
        return x

    at = 0
    for b, (n, m) in enumerate(zip(s["new"], s["total"])):
        pos = torch.arange(m - n, m, device=DEV)
        k = turn(s["k"][at:at + n], pos) / ks
        v = s["v"][at:at + n].double() / vs
        if case["cache"] == "e4m3":
            k, v = k.clamp(-448, 448), v.clamp(-448, 448)
        rows = s["table"][b].long()[torch.div(pos, case["page"], rounding_mode="floor")]
        kc[rows, :, pos % case["page"]] = k
        vc[rows, :, pos % case["page"]] = v
        if rot:
            qo[at:at + n] = turn(s["q"][at:at + n], pos)
        at += n
    out = {"k_cache": kc, "v_cache": vc}
    if rot:
        out["q"] = qo
    return out


def _softmax64(x):
    return torch.exp(x - torch.logsumexp(x, dim=-1, keepdim=True))


def _exact_decode(s):
    case = s["case"]
    hq, hk, d = case["q_heads"], case["kv_heads"], case["head"]
    out = torch.zeros(case["batch"], hq, d, dtype=torch.float64, device=DEV)
    for b, n in enumerate(s["total"]):
        pages = s["table"][b, :(n + case["page"] - 1) // case["page"]].tolist()
        for h in range(hk):
            k = torch.cat([s["k_cache"][p, h].double() for p in pages])[:n] if len(pages) < 8 else _rows64(s["k_cache"], pages, h)[:n]
            v = torch.cat([s["v_cache"][p, h].double() for p in pages])[:n] if len(pages) < 8 else _rows64(s["v_cache"], pages, h)[:n]
            if s["k_scale"] is not None:
                k, v = k * s["k_scale"].double(), v * s["v_scale"].double()
            g = hq // hk
            w = _softmax64(torch.einsum("gd,nd->gn", s["q"][b, h * g:(h + 1) * g].double(), k) / math.sqrt(d))
            out[b, h * g:(h + 1) * g] = torch.einsum("gn,nd->gd", w, v)
    return out


def _rows64(cache, pages, h):
    at = torch.tensor(pages, device=DEV)
    raw = cache[:, h].view(torch.uint8)[at] if cache.dtype == E4M3 else cache[at, h]
    return (raw.view(E4M3) if cache.dtype == E4M3 else raw).double().flatten(0, 1)


def _exact_prefill(s):
    case = s["case"]
    hq, hk, d = case["q_heads"], case["kv_heads"], case["head"]
    out = s["out"].double()
    at = at_k = 0
    for n, m in zip(s["new"], s["total"]):
        for h in range(hq):
            q = s["q"][at:at + n, h].double()
            k, v = (s[c][at_k:at_k + m, h // (hq // hk)].double() for c in "kv")
            for i in range(0, n, 4096):
                e = min(n, i + 4096)
                sees = min(m, m - n + e) if case["causal"] else m
                x = torch.einsum("id,jd->ij", q[i:e], k[:sees]) / math.sqrt(d)
                if case["causal"]:
                    x += torch.full_like(x, -math.inf).triu(m - n + i + 1)
                out[at + i:at + e, h] = _softmax64(x) @ v[:sees]
        at, at_k = at + n, at_k + m
    return out
