"""Workloads of the paged key-value cache: appending rotated keys and values to it, attention of one new token per
sequence over it, and attention of prompt chunks over it, each in a plain form (elementary torch operations in 32 bits)
and as calls of the library.

A cache is a pool of pages of `page` token rows, [pages, page, kv_heads, dim] bf16 (or [pages, kv_heads, page, dim] with
"head_major"), one pool for keys and one for values; row i of `page_table` lists the pages of sequence i. Pages are dealt
out in random order, and rows that no sequence owns hold NaN: nobody may read them."""
import math
import os
import random
import sys

import torch

own = False

HERE = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


# ---------------------------------------------------------------- cases ----

def _append(name, rows, seqs, dtype, dim, kv, group, page, norm=False, interleaved=False, rotary=0, far=0, pad=0, head_major=False, qkv=False):
    return {"name": name, "op": "append", "rows": rows, "seqs": seqs, "dtype": dtype, "dim": dim, "kv": kv, "group": group, "page": page,
            "norm": norm, "interleaved": interleaved, "rotary": rotary or dim, "far": far, "pad": pad, "head_major": head_major, "qkv": qkv}


def _decode(name, rows, least, most, dtype, dim, kv, group, page, window=0, softcap=0.0, slopes=False, prefix=0, lse=False, head_major=False):
    return {"name": name, "op": "decode", "rows": rows, "least": least, "most": most, "dtype": dtype, "dim": dim, "kv": kv, "group": group,
            "page": page, "window": window, "softcap": softcap, "slopes": slopes, "prefix": prefix, "lse": lse, "head_major": head_major}


def _prefill(name, seqs, chunk, past, dim, kv, group, page, window=0, softcap=0.0, slopes=False, prefix=0, lse=False, head_major=False):
    return {"name": name, "op": "prefill", "seqs": seqs, "chunk": chunk, "past": past, "dtype": "bf16", "dim": dim, "kv": kv, "group": group,
            "page": page, "window": window, "softcap": softcap, "slopes": slopes, "prefix": prefix, "lse": lse, "head_major": head_major}


def listed():
    return [
        # one new token of one conversation, the 26-layer decoder's heads: latency alone
        _append("append 1 token f32", 1, 1, "f32", 256, 4, 2, 16, norm=True, far=4096, qkv=True),
        # one new token for each of 64 conversations (four slots empty), bf16 rows far into long contexts
        _append("append 64 tokens bf16", 64, 64, "bf16", 128, 8, 4, 64, far=131072, pad=4, head_major=True),
        # a prompt chunk of several conversations at once, the 62-layer decoder's heads
        _append("append 8190 tokens bf16", 8190, 6, "bf16", 128, 16, 2, 32, norm=True, far=1024, qkv=True),
        # one conversation after a short prompt, the 26-layer decoder's heads: latency alone
        _decode("decode 1 x 1279 f32", 1, 1279, 1279, "f32", 256, 4, 2, 16),
        # a serving batch of mixed lengths, the 62-layer decoder's heads
        _decode("decode 32 x 4608 bf16", 32, 257, 4608, "bf16", 128, 16, 2, 32, lse=True),
        # capped scores in a sliding block, f32 activations, odd page size and some empty slots
        _decode("decode 48 x 3001 f32 capped window", 48, 0, 3001, "f32", 128, 4, 8, 24, window=1024, softcap=50.0),
        # few long documents, many query heads for each key head, a bias that falls with distance
        _decode("decode 4 x 120001 bf16 slopes", 4, 30000, 120001, "bf16", 128, 8, 12, 64, slopes=True, lse=True),
        # a short prompt on the 26-layer decoder's heads, scores capped
        _prefill("prefill 1 x 1024 capped", 1, 1024, 0, 256, 4, 2, 16, softcap=50.0),
        # a long prompt on the 62-layer decoder's heads
        _prefill("prefill 1 x 8192", 1, 8192, 0, 128, 16, 2, 64, lse=True),
        # chunks of several conversations packed behind one another, sliding block, a prefix that all see
        _prefill("prefill 7 x 1500 past 3000 window prefix", 7, 1500, 3000, 128, 8, 4, 32, window=1024, prefix=64),
        # drafts of a few tokens checked against long contexts: few rows, long axis
        _prefill("prefill 4 x 9 past 40000 slopes", 4, 9, 40000, 128, 4, 4, 16, slopes=True),
        # documents of odd lengths packed behind one another, narrow heads
        _prefill("prefill 12 x 777 heads of 64", 12, 777, 0, 64, 6, 3, 24),
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 0.49)))))))


def draw(rng):
    op = rng.choice(["append", "decode", "prefill"])
    dim = rng.choice([64, 128, 128, 256])
    kv = rng.choice([1, 2, 3, 4, 8, 16])
    group = rng.choice([1, 2, 3, 4, 5, 7, 8, 12, 16])
    page = rng.choice([1, 8, 16, 16, 24, 32, 64, 100, 128])
    major = rng.random() < 0.25
    mask = {"window": rng.choice([0, 0, _log(rng, 1, 4096)]), "softcap": rng.choice([0.0, 0.0, 30.0, 50.0]), "slopes": rng.random() < 0.3,
            "prefix": rng.choice([0, 0, 0, _log(rng, 1, 600)]), "lse": rng.random() < 0.5, "head_major": major}
    if op == "append":
        rows = _log(rng, 1, 8000)
        while rows * kv * (group + 2) * dim > 8190 * 16 * 4 * 128:
            rows //= 2
        rows = max(rows, 1)
        c = _append("", rows, rng.randint(1, min(rows, 64)), rng.choice(["f32", "bf16"]), dim, kv, group, page, norm=rng.random() < 0.5,
                    interleaved=rng.random() < 0.3, rotary=rng.choice([dim, dim, dim // 2]), far=_log(rng, 1, 200000), pad=rng.choice([0, 0, min(rows - 1, 5)]),
                    head_major=major, qkv=rng.random() < 0.5)
    elif op == "decode":
        rows, most = _log(rng, 1, 200), _log(rng, 1, 60000)
        while rows * most * kv * dim * (1 + group / 8) > 4 * 100000 * 8 * 128:
            rows, most = max(1, rows // 2), max(1, most * 2 // 3)
        c = _decode("", rows, rng.choice([0, 1, most // 2]), most, rng.choice(["f32", "bf16"]), dim, kv, group, page, **mask)
    else:
        seqs, chunk, past = _log(rng, 1, 16), _log(rng, 1, 6000), rng.choice([0, 0, _log(rng, 1, 40000)])
        while seqs * chunk * (past + chunk) * kv * group * dim > 0.4 * 8192 * 8192 * 32 * 128 or seqs * (past + chunk) * kv * dim > 300e6:
            seqs, chunk, past = max(1, seqs // 2), max(1, chunk * 2 // 3), past * 2 // 3
        c = _prefill("", seqs, chunk, past, dim, kv, group, page, **mask)
    del c["name"]
    return c


def _lengths(case):
    """(new tokens, length with them) of each sequence. They follow from the case alone; the longest comes first."""
    r = random.Random(7)
    if case["op"] == "append":
        live, n = case["rows"] - case["pad"], case["seqs"]
        cuts = sorted(r.sample(range(1, live), min(n, live) - 1)) if min(n, live) > 1 else []
        new = [b - a for a, b in zip([0] + cuts, cuts + [live])]
        new += [0] * (n - len(new))
        return [(m, m + (case["far"] if i == 0 else r.randint(0, case["far"]))) for i, m in enumerate(new)]
    if case["op"] == "decode":
        lens = [case["most"]] + [r.randint(case["least"], case["most"]) for _ in range(case["rows"] - 1)]
        if case["least"] == 0 and len(lens) > 2:
            lens[1] = 0
        return [(1, n) for n in lens]
    new = [case["chunk"]] + [r.randint((case["chunk"] + 3) // 4, case["chunk"]) for _ in range(case["seqs"] - 1)]
    return [(m, m + (case["past"] if i == 0 else r.randint(0, case["past"]))) for i, m in enumerate(new)]


def _visible(case, new, length):
    """How many (query, key) pairs of one sequence the mask leaves, and how many of its keys some query sees."""
    w, p = case["window"], min(case["prefix"], length)
    pairs, first = 0, length
    for q in range(max(0, length - new), length):
        lo = max(0, q - w + 1) if w else 0
        pairs += (q + 1 - lo) + max(0, p - (q + 1)) + min(p, lo)
        first = min(first, lo)
    return pairs, (length - first) + min(p, first) if length else 0


def work(case):
    size = 4 if case["dtype"] == "f32" else 2
    D, Hkv, Hq = case["dim"], case["kv"], case["kv"] * case["group"]
    lens = _lengths(case)
    if case["op"] == "append":
        live = case["rows"] - case["pad"]
        return {"bytes": live * D * (Hq * 2 * size + 2 * Hkv * (size + 2)) + live * 8 + 4 * D,
                "flops": live * D * (Hq + Hkv) * (3 + 4 * case["norm"])}
    both = [_visible(case, n, m) for n, m in lens]
    tokens = sum(n for n, _ in lens)
    return {"bytes": tokens * Hq * D * 2 * size + sum(k for _, k in both) * Hkv * D * 4 + (4 * tokens * Hq if case["lse"] else 0),
            "flops": 4 * D * Hq * sum(p for p, _ in both)}


# --------------------------------------------------------------- inputs ----

def prepare(case, seed):
    dev = torch.device("cuda")
    g = torch.Generator(device=dev).manual_seed(seed)
    rnd = lambda *s: torch.randn(*s, device=dev, generator=g)  # noqa: E731
    dtype = torch.float32 if case["dtype"] == "f32" else torch.bfloat16
    D, Hkv, Hq, ps = case["dim"], case["kv"], case["kv"] * case["group"], case["page"]
    lens = _lengths(case)
    S = len(lens)
    per = max(1, max((m + ps - 1) // ps for _, m in lens))
    # pages: sequences that are appended to bring only the pages of their new rows; the others all of theirs
    first = [(m - n) // ps if case["op"] == "append" else 0 for n, m in lens]
    held = [[i for i in range(f, (m + ps - 1) // ps) if n > 0] for f, (n, m) in zip(first, lens)]
    pages = sum(len(h) for h in held) + 3
    order = torch.randperm(pages, device=dev, generator=g).to(torch.int32)
    at = 0
    rows_i, cols_i = [], []
    for i, h in enumerate(held):
        rows_i += [i] * len(h)
        cols_i += h
        at += len(h)
    table = torch.full((S, per), -1, dtype=torch.int32, device=dev)
    table[torch.tensor(rows_i, dtype=torch.long, device=dev), torch.tensor(cols_i, dtype=torch.long, device=dev)] = order[:at]
    shape = (pages, Hkv, ps, D) if case["head_major"] else (pages, ps, Hkv, D)
    kpool, vpool = (rnd(*shape).to(torch.bfloat16) for _ in range(2))
    s = {"case": dict(case), "table": table, "k": kpool, "v": vpool, "D": D, "Hq": Hq, "Hkv": Hkv, "ps": ps}
    if case["op"] == "append":
        live, rows = case["rows"] - case["pad"], case["rows"]
        seq = torch.cat([torch.full((n,), i) for i, (n, _) in enumerate(lens)]).to(torch.int32)
        pos = torch.cat([torch.arange(m - n, m) for n, m in lens]).to(torch.int32)
        s["row_seq"] = torch.cat([seq, torch.full((rows - live,), -1, dtype=torch.int32)]).to(dev)
        s["row_pos"] = torch.cat([pos, torch.zeros(rows - live, dtype=torch.int32)]).to(dev)
        if case["qkv"]:  # one projection's output, as it comes
            s["qkv"] = rnd(rows, (Hq + 2 * Hkv) * D).to(dtype)
            s["xq"], s["xk"], s["xv"] = s["qkv"].split([Hq * D, Hkv * D, Hkv * D], 1)
        else:
            s["xq"], s["xk"], s["xv"] = (rnd(rows, h * D).to(dtype) for h in (Hq, Hkv, Hkv))
        s["q_out"] = torch.zeros(rows, Hq * D, dtype=dtype, device=dev)
        s["inv_freq"] = 10000.0 ** (-2.0 * torch.arange(case["rotary"] // 2, device=dev, dtype=torch.float64) / D)
        s["nq"], s["nk"] = (1 + 0.1 * rnd(D) if case["norm"] else None for _ in range(2))
    else:
        owned = torch.zeros(pages * ps, dtype=torch.bool, device=dev)
        for i, (_, m) in enumerate(lens):
            if m:
                p = torch.arange(m, device=dev)
                owned[table[i, p // ps].long() * ps + p % ps] = True
        owned = owned.view(pages, 1, ps, 1) if case["head_major"] else owned.view(pages, ps, 1, 1)
        for pool in (kpool, vpool):
            pool.masked_fill_(~owned, float("nan"))
        s["new"] = [n for n, _ in lens]
        s["total"] = sum(s["new"])
        s["q"] = rnd(s["total"], Hq, D).to(dtype)
        s["kv_lens"] = torch.tensor([m for _, m in lens], dtype=torch.int32, device=dev)
        s["q_start"] = torch.tensor([0] + s["new"], dtype=torch.int32, device=dev).cumsum(0).to(torch.int32)
        s["most_new"], s["most"] = max(s["new"]), max(m for _, m in lens)
        s["slopes"] = torch.exp2(-8.0 * torch.arange(1, Hq + 1, device=dev, dtype=torch.float32) / Hq) if case["slopes"] else None
        s["prefix"] = s["kv_lens"].clamp(max=case["prefix"]) if case["prefix"] else None
        s["out"] = torch.empty(s["total"], Hq, D, dtype=dtype, device=dev)
        s["lse"] = torch.empty(s["total"], Hq, dtype=torch.float32, device=dev) if case["lse"] else None
    if own:
        _handles(s)
    return s


def _handles(s):
    """What a serving program keeps beside its tensors: the cache's description, options and workspace."""
    path = os.path.join(HERE, "go-inference_b200")
    if path not in sys.path:
        sys.path.insert(0, path)
    import lthn
    c = s["case"]
    D, ps, Hkv = s["D"], s["ps"], s["Hkv"]
    strides = {"row_stride": D, "head_stride": ps * D} if c["head_major"] else {}
    s["lthn"] = lthn
    s["cache"] = lthn.PagedKV(s["k"], s["v"], s["table"], pages=s["k"].shape[0], page_size=ps, kv_heads=Hkv, head_dim=D, seqs=s["table"].shape[0],
                              table_stride=s["table"].shape[1], page_stride=ps * Hkv * D, **strides)
    s["dt"] = lthn.F32 if c["dtype"] == "f32" else lthn.BF16
    if c["op"] == "append":
        s["rope"] = lthn.rope_params(inv_freq=s["inv_freq"], rotary_dim=c["rotary"], interleaved=c["interleaved"], q_norm=s["nq"], k_norm=s["nk"], eps=1e-6)
        return
    s["options"] = lthn.attn_options(softcap=c["softcap"], slopes=s["slopes"], window=c["window"], prefix_lens=s["prefix"])
    if c["op"] == "decode":
        need = lthn.paged_sdpa_decode_workspace(s["cache"], s["total"], s["Hq"], s["dt"])
    else:
        need = lthn.paged_prefill_attention_workspace(s["cache"], len(s["new"]), s["total"], s["Hq"], s["most"])
    s["work"] = torch.empty(max(need, 16), dtype=torch.uint8, device=s["q"].device)


# ------------------------------------------------------------- one pass ----

def run(s):
    c = s["case"]
    if own:
        m, st = s["lthn"], torch.cuda.current_stream().cuda_stream
        if c["op"] == "append":
            m.paged_kv_append(s["cache"], s["xk"], s["xv"], s["row_seq"], s["row_pos"], c["rows"], s["dt"], rope=s["rope"], q=s["xq"], q_heads=s["Hq"],
                              q_out=s["q_out"], out_dtype=s["dt"], q_stride=s["xq"].stride(0), k_stride=s["xk"].stride(0), v_stride=s["xv"].stride(0), stream=st)
            return {"q": s["q_out"], "k": s["k"], "v": s["v"]}
        if c["op"] == "decode":
            m.paged_sdpa_decode(s["cache"], s["q"], s["dt"], s["kv_lens"], s["total"], s["Hq"], s["out"], s["work"], options=s["options"], lse=s["lse"], stream=st)
        else:
            m.paged_prefill_attention(s["cache"], s["q"], s["q_start"], s["kv_lens"], len(s["new"]), s["total"], s["Hq"], s["out"], s["work"],
                                      max_ctx=s["most"], options=s["options"], lse=s["lse"], stream=st)
        return {"out": s["out"], "lse": s["lse"]}
    return _plain_append(s) if c["op"] == "append" else _plain_attention(s)


def _plain_append(s):
    c, D, ps = s["case"], s["D"], s["ps"]
    live = (s["row_seq"] >= 0).nonzero()[:, 0]
    seq, pos = s["row_seq"][live].long(), s["row_pos"][live].long()
    angle = pos.double()[:, None] * s["inv_freq"][None]
    cos, sin = torch.cos(angle).float()[:, None], torch.sin(angle).float()[:, None]

    def turned(x, w):
        x = x[live].float().view(len(live), -1, D)
        if w is not None:
            x = x / torch.sqrt((x * x).mean(-1, keepdim=True) + 1e-6) * w
        h = c["rotary"] // 2
        y = x.clone()
        if c["interleaved"]:
            a, b = x[..., 0:2 * h:2], x[..., 1:2 * h:2]
            y[..., 0:2 * h:2], y[..., 1:2 * h:2] = a * cos - b * sin, a * sin + b * cos
        else:
            a, b = x[..., :h], x[..., D // 2:D // 2 + h]
            y[..., :h], y[..., D // 2:D // 2 + h] = a * cos - b * sin, a * sin + b * cos
        return y

    s["q_out"][live] = turned(s["xq"], s["nq"]).flatten(1).to(s["q_out"].dtype)
    page, off = s["table"][seq, pos // ps].long(), pos % ps
    for pool, x in ((s["k"], turned(s["xk"], s["nk"])), (s["v"], s["xv"][live].float().view(len(live), -1, D))):
        if c["head_major"]:
            pool[page, :, off] = x.to(pool.dtype)
        else:
            pool[page, off] = x.to(pool.dtype)
    return {"q": s["q_out"], "k": s["k"], "v": s["v"]}


def _plain_attention(s):
    """Every sequence padded to the longest: scores [sequences, key heads, queries of a key head, new tokens, keys]."""
    c, D, Hkv, G, ps = s["case"], s["D"], s["Hkv"], s["case"]["group"], s["ps"]
    S, N, L = len(s["new"]), s["most_new"], s["most"]
    dev = s["q"].device
    lens, start = s["kv_lens"].long(), s["q_start"].long()
    new = start[1:] - start[:-1]
    tok = torch.arange(N, device=dev)[None]
    real = tok < new[:, None]                                     # [S, N]
    at = (start[:-1, None] + tok).clamp(max=s["total"] - 1)
    q = s["q"][at].float().view(S, N, Hkv, G, D).permute(0, 2, 3, 1, 4).reshape(S, Hkv, G * N, D)
    key = torch.arange(L, device=dev)
    page = s["table"][:, key // ps].long().clamp(min=0)           # [S, L]
    inside = key[None] < lens[:, None]
    k, v = ((p[page, :, key % ps] if c["head_major"] else p[page, key % ps]).float().masked_fill_(~inside[:, :, None, None], 0.0).permute(0, 2, 1, 3)
            for p in (s["k"], s["v"]))                            # [S, Hkv, L, D]
    x = torch.matmul(q, k.transpose(2, 3)).mul_(1.0 / math.sqrt(D)).view(S, Hkv, G, N, L)
    if c["softcap"]:
        x = x.div_(c["softcap"]).tanh_().mul_(c["softcap"])
    where = lens[:, None] - new[:, None] + tok                    # [S, N] position of each query
    gap = where[:, :, None] - key                                 # [S, N, L]
    if c["slopes"]:
        x -= s["slopes"].view(1, Hkv, G, 1, 1) * gap.abs().float()[:, None, None]
    seen = gap >= 0
    if c["window"]:
        seen &= gap < c["window"]
    if c["prefix"]:
        seen |= (key[None] < s["prefix"].long()[:, None])[:, None]
    seen &= inside[:, None]
    x.masked_fill_(~seen[:, None, None], float("-inf"))
    top = x.amax(-1, keepdim=True)
    some = top > float("-inf")
    x = x.sub_(torch.where(some, top, 0.0)).exp_()
    total = x.sum(-1, keepdim=True)
    o = torch.matmul(x.view(S, Hkv, G * N, L), v).view(S, Hkv, G, N, D) / torch.where(some, total, 1.0)
    lse = torch.where(some, top + torch.log(total), float("-inf"))
    s["out"][at[real]] = o.permute(0, 3, 1, 2, 4).reshape(S, N, Hkv * G, D)[real].to(s["out"].dtype)
    if s["lse"] is not None:
        s["lse"][at[real]] = lse.permute(0, 3, 1, 2, 4).reshape(S, N, Hkv * G)[real]
    return {"out": s["out"], "lse": s["lse"]}


# ------------------------------------------------------------ in 64 bits ----

def exact(case, seed):
    s = prepare(case, seed)
    return _exact_append(s) if case["op"] == "append" else _exact_attention(s)


def _exact_append(s):
    c, D, ps = s["case"], s["D"], s["ps"]
    q_out, pools = s["q_out"].double(), [s["k"].double(), s["v"].double()]
    seq, pos = s["row_seq"].cpu(), s["row_pos"].cpu()
    live = [i for i in range(c["rows"]) if seq[i] >= 0]
    pick = torch.tensor(live, device=q_out.device)
    theta = torch.outer(s["row_pos"].double()[pick], s["inv_freq"])
    turn = torch.polar(torch.ones_like(theta), theta)             # e^(i theta)

    def rotate(x, w):
        x = x.double()[pick].reshape(len(live), -1, D)
        if w is not None:
            x = w.double() * x * torch.rsqrt(x.square().sum(-1, keepdim=True) / D + 1e-6)
        h = turn.shape[1]
        idx = torch.arange(h, device=x.device)
        lo, hi = (2 * idx, 2 * idx + 1) if c["interleaved"] else (idx, idx + D // 2)
        z = torch.complex(x[..., lo], x[..., hi]) * turn[:, None]
        x[..., lo], x[..., hi] = z.real, z.imag
        return x

    q_out[pick] = rotate(s["xq"], s["nq"]).reshape(len(live), -1)
    page = s["table"].cpu()[seq[live].long(), pos[live].long() // ps].long().to(pick.device)
    slot = (pos[live].long() % ps).to(pick.device)
    new = [rotate(s["xk"], s["nk"]), s["xv"].double()[pick].reshape(len(live), -1, D)]
    for pool, x in zip(pools, new):
        rows = pool.transpose(1, 2) if c["head_major"] else pool   # [pages, page, kv, D]
        rows[page, slot] = x
    return {"q": q_out, "k": pools[0], "v": pools[1]}


def _exact_attention(s):
    c, D, Hkv, G, ps = s["case"], s["D"], s["Hkv"], s["case"]["group"], s["ps"]
    out = torch.zeros(s["total"], s["Hq"], D, dtype=torch.float64, device=s["q"].device)
    lse = torch.full((s["total"], s["Hq"]), -math.inf, dtype=torch.float64, device=out.device)
    pools = [p.transpose(1, 2) if c["head_major"] else p for p in (s["k"], s["v"])]
    row = 0
    for i, length in enumerate(s["kv_lens"].tolist()):
        n = s["new"][i]
        j = torch.arange(length, device=out.device)
        rows = s["table"][i].long()[j // ps], j % ps
        pos = torch.arange(length - n, length, device=out.device)[:, None]
        ok = j[None] <= pos
        if c["window"]:
            ok &= j[None] > pos - c["window"]
        if c["prefix"]:
            ok |= j[None] < min(c["prefix"], length)
        for h in range(Hkv if length else 0):
            k, v = (p[rows[0], rows[1], h].double() for p in pools)
            for a in range(h * G, (h + 1) * G):
                t = s["q"][row:row + n, a].double() @ k.T / math.sqrt(D)
                if c["softcap"]:
                    t = c["softcap"] * torch.tanh(t / c["softcap"])
                if c["slopes"]:
                    t = t - s["slopes"][a].double() * (pos - j[None]).abs()
                t = torch.where(ok, t, -math.inf)
                lse[row:row + n, a] = torch.logsumexp(t, 1)
                out[row:row + n, a] = torch.where(ok.any(1)[:, None], torch.softmax(t, 1), 0.0) @ v
        row += n
    return {"out": out, "lse": lse if c["lse"] else None}
