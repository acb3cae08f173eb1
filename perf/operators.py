"""Cases that measure the operators between a model's q/k/v projections and its output projection:
rotary positions, the paged key/value cache (written, quantised, read back) and attention over it.

Each operator has its plain form here, in elementary torch operations in 32 bits, its definition in
64 bits (``exact``), and the call of ``compressai_b200.attention`` that a user's program makes."""
import math

import torch

own = False
DEV = "cuda"
DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16}


# ---------------------------------------------------------------------------------------- cases
def _attn(name, **kw):
    # seqs sequences; the longest holds `ctx` tokens, `new` of them new (the queries); the others are
    # shorter by up to the share `ragged`. int8: the cache holds 8-bit values and fp32 scales.
    case = dict(name=name, op="attention", seqs=1, new=1, ctx=1024, hq=16, hkv=2, d=256, dtype="bf16", int8=False,
                page=64, ragged=0.0, causal=True, window=0)
    case.update(kw)
    return case


def listed():
    return [
        # one user's chat turn, one token a step, the stack's attention shape: latency only
        _attn("decode one sequence", ctx=701),
        # a serving batch in its decode step, lengths all over the place
        _attn("decode batch", seqs=64, ctx=8000, ragged=0.9),
        # few long documents in 8 bits: bandwidth of the quantised cache, work split along the length
        _attn("decode long int8", seqs=4, ctx=100003, hq=32, hkv=8, d=128, int8=True, ragged=0.4, page=32),
        # drafted tokens checked together, sliding-window layers
        _attn("verify drafts window", seqs=9, new=5, ctx=3001, d=128, dtype="fp16", window=1024, ragged=0.5, page=16),
        # a scheduler's chunk: pieces of three prompts over what their caches hold already
        _attn("chunk ragged", seqs=3, new=611, ctx=8191, hq=32, hkv=8, d=128, ragged=0.5),
        # the same over a quantised cache, with the stack's shape
        _attn("chunk int8", seqs=2, new=257, ctx=16385, int8=True, ragged=0.3),
        # a whole prompt at once, the stack's shape: tensor-core bound
        _attn("prefill", new=8192, ctx=8192, page=128),
        # many short prompts with small heads, every token sees its whole prompt
        _attn("short prompts", seqs=24, new=301, ctx=301, hq=12, hkv=12, d=64, dtype="fp16", ragged=0.8, causal=False),
        # rotary of one token, a quarter of the head (the stack's): latency only
        dict(name="rotary one token", op="rotary", tokens=1, hq=16, hkv=2, d=256, rot=64, dtype="bf16",
             interleaved=False, inverse=False, scaled=False),
        # rotary of a long prompt's gradient, neighbours paired, frequencies stretched
        dict(name="rotary prompt back", op="rotary", tokens=8191, hq=32, hkv=8, d=128, rot=128, dtype="fp16",
             interleaved=True, inverse=True, scaled=True),
        # the decode step's cache write of a batch, rotary of q and k fused
        dict(name="write decode", op="write", seqs=32, new=1, ctx=4000, hq=16, hkv=2, d=256, rot=64, dtype="bf16",
             int8=False, page=64, ragged=0.9, interleaved=False),
        # prompts written into an 8-bit cache with rotary, then read back
        dict(name="write prompts int8", op="write", seqs=5, new=3001, ctx=3001, hq=32, hkv=8, d=128, rot=128,
             dtype="bf16", int8=True, page=16, ragged=0.5, interleaved=True),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["decode", "decode", "chunk", "chunk", "rotary", "write"])
    hkv, g, d = rng.choice([1, 2, 4, 8]), rng.choice([1, 2, 4, 5, 8]), rng.choice([64, 96, 128, 256])
    both = dict(hq=hkv * g, hkv=hkv, d=d, dtype=rng.choice(["bf16", "fp16"]))
    paged = dict(page=rng.choice([16, 32, 64, 128]), ragged=round(rng.uniform(0, 0.95), 2), int8=rng.random() < 0.4)
    if kind == "rotary":
        rot = rng.choice([d, d // 2, d // 4])
        return dict(op="rotary", tokens=_log(rng, 1, 8000), rot=rot, interleaved=rng.random() < 0.5,
                    inverse=rng.random() < 0.3, scaled=rng.random() < 0.5, **both)
    if kind == "write":
        new = rng.choice([1, _log(rng, 2, 4000)])
        seqs = max(1, min(_log(rng, 1, 64), 12000 // new))
        # a quantised write is read back whole: prompts that start empty, short ones where it is one token
        ctx = new if paged["int8"] else new + _log(rng, 1, 6000)
        return dict(op="write", seqs=seqs, new=new, ctx=ctx, rot=rng.choice([d, d // 2]), interleaved=rng.random() < 0.5,
                    **both, **paged)
    if kind == "decode":
        ctx = _log(rng, 1, 60000)
        seqs = max(1, min(_log(rng, 1, 64), 300_000_000 // (ctx * hkv * d)))
        return dict(op="attention", seqs=seqs, new=1, ctx=ctx, causal=True, window=rng.choice([0, 0, 512]), **both, **paged)
    new = _log(rng, 2, 3000)
    ctx = new + rng.choice([0, _log(rng, 1, 12000)])
    seqs = max(1, min(_log(rng, 1, 24), 250_000_000 // (new * ctx * hkv * g)))
    return dict(op="attention", seqs=seqs, new=new, ctx=ctx, causal=rng.random() < 0.8,
                window=rng.choice([0, 0, 1024]), **both, **paged)


def _lengths(case):
    """(new tokens, all tokens) of each sequence: the first has the case's, the others less by up to `ragged`."""
    news, lens = [], []
    for b in range(case["seqs"]):
        u = (b * 0.6180339887498949) % 1.0 * case["ragged"]
        new = max(1, int(case["new"] * (1 - u)))
        old = int((case["ctx"] - case["new"]) * (1 - u))
        news.append(new)
        lens.append(old + new)
    return news, lens


def work(case):
    d = case["d"]
    if case["op"] == "rotary":
        n = case["tokens"] * (case["hq"] + case["hkv"])
        return {"bytes": n * d * 4 + 4 * case["tokens"], "flops": 3 * n * case["rot"]}
    news, lens = _lengths(case)
    row = d + 4 if case["int8"] else 2 * d
    T = sum(news)
    if case["op"] == "write":
        moved = T * (case["hq"] * d * 4 + 2 * case["hkv"] * (2 * d + row))
        if case["int8"]:  # read back
            moved += T * 2 * case["hkv"] * (row + 2 * d)
        return {"bytes": moved, "flops": 3 * T * (case["hq"] + case["hkv"]) * case["rot"]}
    keys = pairs = 0
    for n, l in zip(news, lens):
        w = case["window"] or l
        keys += min(l, w + n - 1)
        if case["causal"]:
            full = max(0, min(n, l - w))  # rows that see a whole window
            pairs += full * w + sum(range(l - n + 1, l - full + 1))
        else:
            pairs += sum(l - max(0, l - n + i - w + 1) for i in range(n))
    return {"bytes": 4 * T * case["hq"] * d + 2 * keys * case["hkv"] * row, "flops": 4 * pairs * case["hq"] * d}


# --------------------------------------------------------------------------------------- inputs
def _frequencies(rot, scaled):
    f = 10000.0 ** (-torch.arange(0, rot, 2, dtype=torch.float64) / rot)
    if not scaled:
        return f.float().to(DEV), 1.0
    # context stretched eightfold: slow pairs interpolated, fast ones kept, a ramp between
    turns = 4096 * f / (2 * math.pi)
    keep = ((turns - 1) / (32 - 1)).clamp(0, 1)
    return (f * keep + f / 8 * (1 - keep)).float().to(DEV), 0.1 * math.log(8) + 1


def prepare(case, seed):
    g = torch.Generator(device=DEV).manual_seed(seed)
    dt, d, hq, hkv = DTYPES[case["dtype"]], case["d"], case["hq"], case["hkv"]
    s = {"case": case}
    if case["op"] == "rotary":
        T = case["tokens"]
        qkv = torch.randn(T, (hq + 2 * hkv) * d, generator=g, device=DEV).to(dt)  # as one projection leaves it
        s["q"] = qkv[:, : hq * d].unflatten(1, (hq, d))
        s["k"] = qkv[:, hq * d:(hq + hkv) * d].unflatten(1, (hkv, d))
        first = int(torch.randint(0, 30000, (1,), generator=g, device=DEV))
        s["positions"] = torch.arange(first, first + T, device=DEV, dtype=torch.int32)
        s["inv_freq"], s["factor"] = _frequencies(case["rot"], case["scaled"])
        return s
    news, lens = _lengths(case)
    T, P = sum(news), case["page"]
    qkv = torch.randn(T, (hq + 2 * hkv) * d, generator=g, device=DEV).to(dt)
    s["q"] = qkv[:, : hq * d].unflatten(1, (hq, d))
    s["k"] = qkv[:, hq * d:(hq + hkv) * d].unflatten(1, (hkv, d))
    s["v"] = qkv[:, (hq + hkv) * d:].unflatten(1, (hkv, d))
    starts = [0]
    for n in news:
        starts.append(starts[-1] + n)
    s["starts"] = torch.tensor(starts, dtype=torch.int32, device=DEV)
    s["lens"] = torch.tensor(lens, dtype=torch.int32, device=DEV)
    s["max_new"], s["max_len"], s["total"] = max(news), max(lens), T
    # pages in no order, some of the pool free; the table is wider than any sequence needs
    need = [-(-l // P) for l in lens]
    pages = sum(need) + 3
    perm = torch.randperm(pages, generator=g, device=DEV).to(torch.int32)
    row = torch.repeat_interleave(torch.arange(len(need), device=DEV), torch.tensor(need, device=DEV))
    col = torch.cat([torch.arange(n, device=DEV) for n in need])
    s["table"] = torch.full((len(lens), max(need) + 2), -1, dtype=torch.int32, device=DEV)
    s["table"][row, col] = perm[: row.numel()]
    if case["op"] == "write":
        s["inv_freq"], s["factor"] = _frequencies(case["rot"], False)
        kind = torch.int8 if case["int8"] else dt
        s["k_pages"], s["v_pages"] = (torch.zeros(pages, hkv, P, d, dtype=kind, device=DEV) for _ in range(2))
        s["k_scale"], s["v_scale"] = ((torch.zeros(pages, hkv, P, device=DEV) if case["int8"] else None) for _ in range(2))
        return s
    # what no sequence has written yet is whatever was in memory: NaN here
    fresh = torch.ones(pages, P, dtype=torch.bool, device=DEV)
    fresh[perm[: row.numel()].long()] = torch.arange(P, device=DEV) + col[:, None] * P >= s["lens"][row][:, None]
    s["q"] = 1.5 * s["q"]
    for name in ("k", "v"):
        x = torch.randn(pages, hkv, P, d, generator=g, device=DEV).to(dt)
        if case["int8"]:
            amax = x.abs().amax(-1, keepdim=True).float()
            s[name + "_pages"] = torch.round(x.float() * (127 / amax)).clamp(-127, 127).to(torch.int8)
            s[name + "_scale"] = (amax[..., 0] / 127).masked_fill(fresh[:, None], float("nan"))
        else:
            s[name + "_pages"] = x.masked_fill(fresh[:, None, :, None], float("nan"))
            s[name + "_scale"] = None
    del s["k"], s["v"]
    return s


# ---------------------------------------------------------------------------------- plain forms
def _rotate(x, positions, inv_freq, interleaved, factor, inverse):
    """x [T, H, D] in 32 bits with the first 2 * len(inv_freq) values of each head turned."""
    r = 2 * inv_freq.numel()
    t = positions.float()[:, None, None] * inv_freq
    c, n = torch.cos(t) * factor, torch.sin(t) * factor
    if inverse:
        n = -n
    x = x.float()
    a, b = (x[..., 0:r:2], x[..., 1:r:2]) if interleaved else (x[..., : r // 2], x[..., r // 2: r])
    a, b = a * c - b * n, b * c + a * n
    y = torch.stack([a, b], -1).flatten(-2) if interleaved else torch.cat([a, b], -1)
    return torch.cat([y, x[..., r:]], -1)


def _tokens(s):
    """Of each new token: its sequence, its place among the sequence's new ones, its position."""
    t = torch.arange(s["total"], device=DEV)
    b = (t[:, None] >= s["starts"][None, 1:]).sum(1)
    i = t - s["starts"][b]
    return b, i, s["lens"][b] - (s["starts"][b + 1] - s["starts"][b]) + i


def _plain_write(s):
    case, P = s["case"], s["case"]["page"]
    b, i, pos = _tokens(s)
    rot = (pos, s["inv_freq"], case["interleaved"], s["factor"], False)
    q, k, v = _rotate(s["q"], *rot), _rotate(s["k"], *rot), s["v"].float()
    page, off = s["table"][b, pos // P].long(), pos % P
    out = [q.to(s["q"].dtype)]
    for x, pool, scale in ((k, s["k_pages"], s["k_scale"]), (v, s["v_pages"], s["v_scale"])):
        if scale is None:
            pool[page, :, off] = x.to(pool.dtype)
            out.append(pool)
            continue
        amax = x.abs().amax(-1)
        pool[page, :, off] = torch.round(x * (127 / amax)[..., None]).clamp(-127, 127).to(torch.int8)
        scale[page, :, off] = amax / 127
        out.append((pool[page, :, off].float() * scale[page, :, off][..., None]).to(s["q"].dtype))
    return out


def _plain_attention(s):
    case, P = s["case"], s["case"]["page"]
    hq, hkv, d = case["hq"], case["hkv"], case["d"]
    B, Q, L = case["seqs"], s["max_new"], s["max_len"]
    l = torch.arange(L, device=DEV)
    page, off = s["table"][:, l // P].long(), (l % P).expand(B, L)
    there = l < s["lens"][:, None]
    k, v = s["k_pages"][page, :, off].float(), s["v_pages"][page, :, off].float()  # [B, L, hkv, d]
    if case["int8"]:
        k = k * s["k_scale"][page, :, off][..., None]
        v = v * s["v_scale"][page, :, off][..., None]
    k, v = (torch.where(there[:, :, None, None], x, torch.zeros((), device=DEV)) for x in (k, v))
    b, i, pos = _tokens(s)
    q = torch.zeros(B, Q, hq, d, device=DEV)
    q[b, i] = s["q"].float()
    new = s["starts"][1:] - s["starts"][:-1]
    at = (s["lens"] - new)[:, None] + torch.arange(Q, device=DEV)  # position of each row [B, Q]
    sees = there[:, None, :].expand(B, Q, L)
    if case["causal"]:
        sees = sees & (l <= at[..., None])
    if case["window"]:
        sees = sees & (l > at[..., None] - case["window"])
    q = q.view(B, Q, hkv, hq // hkv, d).permute(0, 2, 3, 1, 4)  # [B, hkv, g, Q, d]
    k, v = k.permute(0, 2, 3, 1)[:, :, None], v.permute(0, 2, 1, 3)[:, :, None]
    x = torch.matmul(q, k) * d ** -0.5
    x = x.masked_fill(~sees[:, None, None], float("-inf"))
    top = x.amax(-1, keepdim=True)
    p = torch.exp(x - torch.where(top == float("-inf"), torch.zeros_like(top), top))
    del x
    total = p.sum(-1, keepdim=True)
    o = torch.matmul(p, v) / torch.where(total == 0, torch.ones_like(total), total)
    return o.permute(0, 3, 1, 2, 4).reshape(B, Q, hq, d)[b, i].to(s["q"].dtype)


def _plain(s):
    case = s["case"]
    if case["op"] == "rotary":
        rot = (s["positions"], s["inv_freq"], case["interleaved"], s["factor"], case["inverse"])
        return [_rotate(x, *rot).to(x.dtype) for x in (s["q"], s["k"])]
    return _plain_write(s) if case["op"] == "write" else _plain_attention(s)


def run(s):
    if not own:
        return _plain(s)
    from compressai_b200 import attention as A
    case = s["case"]
    if case["op"] == "rotary":
        return list(A.rotary(s["q"], s["k"], s["positions"], s["inv_freq"], interleaved=case["interleaved"],
                             factor=s["factor"], inverse=case["inverse"]))
    if case["op"] == "write":
        q = A.cache_write(s["k"], s["v"], s["k_pages"], s["v_pages"], s["table"], s["lens"], s["starts"],
                          k_scale=s["k_scale"], v_scale=s["v_scale"], q=s["q"], inv_freq=s["inv_freq"],
                          interleaved=case["interleaved"], factor=s["factor"])
        if not case["int8"]:
            return [q, s["k_pages"], s["v_pages"]]
        return [q, *A.cache_read(s["k_pages"], s["v_pages"], s["table"], s["starts"], s["total"], k_scale=s["k_scale"],
                                 v_scale=s["v_scale"], dtype=s["q"].dtype)]
    return A.paged_attention(s["q"], s["k_pages"], s["v_pages"], s["table"], s["lens"], s["starts"], k_scale=s["k_scale"],
                             v_scale=s["v_scale"], causal=case["causal"], window=case["window"], max_new=s["max_new"],
                             max_len=s["max_len"])


# ------------------------------------------------------------------------------- 64 bits
def _turn64(x, pos, f, interleaved, factor, sign):
    x = x.double().clone()
    n = f.numel()
    for i in range(n):
        a, b = (2 * i, 2 * i + 1) if interleaved else (i, i + n)
        t = pos.double() * f[i].double()
        c, w = (torch.cos(t) * factor)[:, None], (sign * torch.sin(t) * factor)[:, None]
        u, v = x[..., a].clone(), x[..., b].clone()
        x[..., a], x[..., b] = u * c - v * w, u * w + v * c
    return x


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "rotary":
        return [_turn64(x, s["positions"], s["inv_freq"], case["interleaved"], s["factor"], -1 if case["inverse"] else 1)
                for x in (s["q"], s["k"])]
    news, lens = _lengths(case)
    P, table = case["page"], s["table"].tolist()
    if case["op"] == "write":
        pos = torch.cat([torch.arange(l - n, l, device=DEV) for n, l in zip(news, lens)])
        q, k = (_turn64(x, pos, s["inv_freq"], case["interleaved"], s["factor"], 1) for x in (s["q"], s["k"]))
        v = s["v"].double()
        if case["int8"]:
            steps = [x.abs().amax(-1, keepdim=True) / 127 for x in (k, v)]
            return [q] + [torch.round(x / w) * w for x, w in zip((k, v), steps)]
        pools = [p.double() for p in (s["k_pages"], s["v_pages"])]
        slot = torch.tensor([table[b][p // P] * P + p % P for b, (n, l) in enumerate(zip(news, lens)) for p in range(l - n, l)],
                            device=DEV)
        for pool, x in zip(pools, (k, v)):
            for h in range(case["hkv"]):
                pool[slot // P, h, slot % P] = x[:, h]
        return [q, *pools]
    outs, at, g = [], 0, case["hq"] // case["hkv"]
    for b, (n, l) in enumerate(zip(news, lens)):
        ids = torch.tensor(table[b][: -(-l // P)], device=DEV)
        rows = torch.arange(l - n, l, device=DEV)
        keys = torch.arange(l, device=DEV)
        hidden = torch.zeros(n, l, dtype=torch.bool, device=DEV)
        if case["causal"]:
            hidden |= keys[None] > rows[:, None]
        if case["window"]:
            hidden |= keys[None] <= rows[:, None] - case["window"]
        o = torch.zeros(n, case["hq"], case["d"], dtype=torch.float64, device=DEV)
        for h in range(case["hq"]):
            k, v = (s[x + "_pages"][ids, h // g].reshape(-1, case["d"])[:l].double() for x in "kv")
            if case["int8"]:
                k, v = (y * s[x + "_scale"][ids, h // g].reshape(-1, 1)[:l].double() for x, y in (("k", k), ("v", v)))
            x = (s["q"][at:at + n, h].double() @ k.T / math.sqrt(case["d"])).masked_fill(hidden, -math.inf)
            o[:, h] = torch.softmax(x, -1) @ v
        outs.append(o)
        at += n
    return torch.cat(outs)
