"""Performance cases of the operators between a layer's q|k|v projection and
its output projection, over a paged KV cache, each one call through the public
entry points.

Kinds of case (field ``kind``):

* ``plan``  one mi355x_kv_plan call: the block tables, slots, positions and
            row offsets of a step, from the requests' lengths.
* ``rope``  one mi355x_qk_norm_rope call: bias, the norm of each query and key
            head, the rotation, and the store of keys and values into pages.
* ``attn``  one mi355x_paged_attention call: the new tokens of every request
            against all its cached ones.

The lengths of a case come from the case alone (``lens`` seeds them), the
values from the seed.  Queries and keys are as norms and rotations leave them:
N(0, 1) per value, queries twice that, so that the scores of a row spread over
about ten binades of weights; a few channels are larger, as in trained models.
Pages are a random permutation of the pool.
"""
import math
import os
import random
import sys

import torch

own = False

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
DTYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
# ggml's type ids
TYPE_IDS = {"f32": 0, "f16": 1, "bf16": 30}
EPS = 1e-6


def listed():
    return [
        # every step of 64 requests that decode together
        {"name": "plan decode 64", "kind": "plan", "B": 64, "added_lo": 1, "added_hi": 1, "cached_lo": 0,
         "cached_hi": 8191, "page": 16, "lens": 1},
        # a step of many prompts' chunks, lengths odd
        {"name": "plan chunks 256", "kind": "plan", "B": 256, "added_lo": 1, "added_hi": 512, "cached_lo": 0,
         "cached_hi": 4096, "page": 64, "lens": 2},
        # one token of the 3B shape: q|k|v from the GEMV in f32, biases, no norms
        {"name": "rope token 3B", "kind": "rope", "T": 1, "heads": 16, "kv_heads": 2, "hd": 128, "rot": 128,
         "pairs": False, "in": "f32", "type": "f16", "bias": True, "norm": False, "page": 16, "hnd": False, "pad": 0,
         "pos": 32768},
        # a few tokens with norms, half of each head rotated in adjacent pairs, rows apart
        {"name": "rope norm 37", "kind": "rope", "T": 37, "heads": 14, "kv_heads": 2, "hd": 64, "rot": 32,
         "pairs": True, "in": "bf16", "type": "bf16", "bias": False, "norm": True, "page": 8, "hnd": True, "pad": 24,
         "pos": 1000000},
        # a large chunk with norms
        {"name": "rope chunk 8192", "kind": "rope", "T": 8192, "heads": 32, "kv_heads": 8, "hd": 128, "rot": 128,
         "pairs": False, "in": "bf16", "type": "bf16", "bias": False, "norm": True, "page": 64, "hnd": False, "pad": 0,
         "pos": 131072},
        # the last token of a 512-token prompt and 128 generated ones, the 3B shape; f32 for the next GEMV
        {"name": "attn token 3B", "kind": "attn", "B": 1, "heads": 16, "kv_heads": 2, "hd": 128, "type": "f16",
         "out": "f32", "page": 16, "hnd": False, "q_lo": 1, "q_hi": 1, "kv_lo": 640, "kv_hi": 640, "window": 0,
         "cap": 0.0, "lens": 3},
        # 64 requests of very different lengths decoding together
        {"name": "attn decode 64 ragged", "kind": "attn", "B": 64, "heads": 32, "kv_heads": 8, "hd": 128,
         "type": "bf16", "out": "bf16", "page": 16, "hnd": False, "q_lo": 1, "q_hi": 1, "kv_lo": 1, "kv_hi": 8192,
         "window": 0, "cap": 0.0, "lens": 4},
        # one request on a very long context
        {"name": "attn decode 131072", "kind": "attn", "B": 1, "heads": 32, "kv_heads": 8, "hd": 128, "type": "f16",
         "out": "f16", "page": 64, "hnd": False, "q_lo": 1, "q_hi": 1, "kv_lo": 131072, "kv_hi": 131072, "window": 0,
         "cap": 0.0, "lens": 5},
        # four drafted tokens and the one before them, 16 requests
        {"name": "attn drafts 16x5", "kind": "attn", "B": 16, "heads": 16, "kv_heads": 2, "hd": 128, "type": "bf16",
         "out": "bf16", "page": 32, "hnd": True, "q_lo": 5, "q_hi": 5, "kv_lo": 500, "kv_hi": 6000, "window": 0,
         "cap": 0.0, "lens": 6},
        # a 512-row micro-batch in the middle of a long prompt, the 3B shape
        {"name": "attn chunk 512", "kind": "attn", "B": 1, "heads": 16, "kv_heads": 2, "hd": 128, "type": "f16",
         "out": "f32", "page": 16, "hnd": False, "q_lo": 512, "q_hi": 512, "kv_lo": 4608, "kv_hi": 4608, "window": 0,
         "cap": 0.0, "lens": 7},
        # chunks and single tokens together, a head for each query head, a sliding window and capped scores
        {"name": "attn mixed window cap", "kind": "attn", "B": 24, "heads": 8, "kv_heads": 8, "hd": 64,
         "type": "bf16", "out": "bf16", "page": 8, "hnd": True, "q_lo": 1, "q_hi": 400, "kv_lo": 1, "kv_hi": 5000,
         "window": 1000, "cap": 30.0, "lens": 8},
        # a whole long prompt at once
        {"name": "attn prompt 8192", "kind": "attn", "B": 1, "heads": 32, "kv_heads": 8, "hd": 128, "type": "bf16",
         "out": "bf16", "page": 64, "hnd": False, "q_lo": 8192, "q_hi": 8192, "kv_lo": 8192, "kv_hi": 8192,
         "window": 0, "cap": 0.0, "lens": 9},
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _cost(case):
    w = work(case)
    return max(w["bytes"], w["flops"] / 50)


def draw(rng: random.Random):
    kind = rng.choices(["attn", "rope", "plan"], [7, 3, 2])[0]
    page = rng.choice([8, 16, 16, 32, 64, 256])
    lens = rng.randint(100, 10**6)
    if kind == "plan":
        hi = _log_int(rng, 1, 512)
        return {"kind": "plan", "B": _log_int(rng, 1, 256), "added_lo": rng.choice([0, 1, hi]), "added_hi": hi,
                "cached_lo": 0, "cached_hi": _log_int(rng, 1, 8191), "page": page, "lens": lens}
    kv_heads = rng.choice([1, 2, 4, 8])
    heads = kv_heads * rng.choice([1, 2, 4, 7, 8])
    hd = rng.choice([64, 96, 128, 128, 128, 256])
    t = rng.choice(["f16", "bf16"])
    if kind == "rope":
        most = 8192 * 48 * 128 // ((heads + 2 * kv_heads) * hd)
        return {"kind": "rope", "T": _log_int(rng, 1, min(8192, most)), "heads": heads, "kv_heads": kv_heads, "hd": hd,
                "rot": hd if rng.random() < 0.7 else hd // 2, "pairs": rng.random() < 0.3,
                "in": rng.choice(["f32", t]), "type": t, "bias": rng.random() < 0.4, "norm": rng.random() < 0.6,
                "page": page, "hnd": rng.random() < 0.3, "pad": rng.choice([0, 0, 8, 40]),
                "pos": _log_int(rng, 1, 1000000)}
    most = max(_cost(c) for c in listed())
    while True:
        form = rng.choice(["token", "token", "drafts", "chunk", "mixed"])
        B = _log_int(rng, 1, 4 if form == "chunk" else 64)
        kv_hi = _log_int(rng, 16, 131072 if form == "token" else 16384)
        q_lo, q_hi = {"token": (1, 1), "drafts": (2, 8), "chunk": (1, 8192), "mixed": (1, 600)}[form]
        if form == "drafts":
            q_lo = q_hi = rng.randint(2, 8)
        if form == "chunk":
            q_lo = q_hi = _log_int(rng, 9, 8192)
        q_lo, q_hi = min(q_lo, kv_hi), min(q_hi, kv_hi)
        kv_lo = rng.choice([q_lo, kv_hi])
        c = {"kind": "attn", "B": B, "heads": heads, "kv_heads": kv_heads, "hd": hd, "type": t,
             "out": rng.choice([t, t, "f32"]), "page": page, "hnd": rng.random() < 0.3, "q_lo": q_lo, "q_hi": q_hi,
             "kv_lo": kv_lo, "kv_hi": kv_hi, "window": rng.choice([0, 0, 0, 100, 1000]),
             "cap": rng.choice([0.0, 0.0, 0.0, 30.0]), "lens": lens}
        # the plain form's padded scores and keys have to fit beside the state
        if _cost(c) <= most and B * q_hi * heads * kv_hi <= 2**31 and B * kv_hi * kv_heads * hd <= 2**30:
            return c


# ---- lengths: from the case alone ---------------------------------------------


def _ints(rng, lo, hi, n):
    return [rng.randint(lo, hi) for _ in range(n)]


def _attn_lens(c):
    """(new tokens, all tokens) of each request."""
    rng = random.Random(c["lens"])
    q = _ints(rng, c["q_lo"], c["q_hi"], c["B"])
    kv = [max(a, b) for a, b in zip(q, _ints(rng, c["kv_lo"], c["kv_hi"], c["B"]))]
    return q, kv


def _plan_lens(c):
    """(cached tokens, new tokens) of each request."""
    rng = random.Random(c["lens"])
    cached = _ints(rng, c["cached_lo"], c["cached_hi"], c["B"])
    return cached, _ints(rng, c["added_lo"], c["added_hi"], c["B"])


def _pages(n, page):
    return -(-n // page)


# ---- inputs ------------------------------------------------------------------


def _rand(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed * 1000003 + 29)
    return g


def _int32(v):
    return torch.tensor(v, dtype=torch.int32, device="cuda")


def _normal(shape, g, dtype):
    return torch.randn(shape, generator=g, device="cuda").to(dtype)


def _pool(n_pages, c, g):
    """Pages of keys or values, [page][token][head][value] or (hnd) [page][head][token][value]."""
    inner = (c["kv_heads"], c["page"]) if c["hnd"] else (c["page"], c["kv_heads"])
    out = torch.empty((n_pages, *inner, c["hd"]), dtype=DTYPES[c["type"]], device="cuda")
    flat, step = out.view(-1), 1 << 26
    for at in range(0, flat.numel(), step):
        n = min(step, flat.numel() - at)
        flat[at:at + n] = torch.randn(n, generator=g, device="cuda").to(flat.dtype)
    return out


def prepare(case, seed):
    c = case
    g = _rand(seed)
    s = {"case": c}
    if c["kind"] == "plan":
        cached, added = _plan_lens(c)
        P = c["page"]
        cols = max(1, _pages(max(a + b for a, b in zip(cached, added)), P))
        held = [_pages(n, P) for n in cached]
        fresh = sum(_pages(a + b, P) - h for a, b, h in zip(cached, added, held))
        # pages of a pool in random order: those that the requests hold, then the free ones
        order = torch.randperm(sum(held) + fresh + 17, generator=g, device="cuda").to(torch.int32)
        table = torch.full((c["B"], cols), -1, dtype=torch.int32, device="cuda")
        have = torch.arange(cols, device="cuda")[None, :] < _int32(held)[:, None]
        table[have] = order[:sum(held)]
        # eleven entries of the free list are used up, at most six stay over; the rows are padded by three
        s.update(cached=_int32(cached), added=_int32(added), table=table, rows=sum(added) + 3,
                 free=torch.cat([order[:11], order[sum(held):]]).contiguous(), head=_int32([11]))
    elif c["kind"] == "rope":
        T, hd, dt = c["T"], c["hd"], DTYPES[c["in"]]
        width = (c["heads"] + 2 * c["kv_heads"]) * hd
        # q|k|v of a token side by side, as one projection gives them
        s["qkv"] = (1.5 * torch.randn((T, width + c["pad"]), generator=g, device="cuda")).to(dt)
        for name, heads in (("q", c["heads"]), ("k", c["kv_heads"])):
            s[name + "_norm"] = 1 + 0.2 * torch.randn(hd, generator=g, device="cuda") if c["norm"] else None
            s[name + "_bias"] = torch.randn(heads * hd, generator=g, device="cuda") if c["bias"] else None
        s["v_bias"] = torch.randn(c["kv_heads"] * hd, generator=g, device="cuda") if c["bias"] else None
        n_pages = _pages(T, c["page"]) + 2
        s["k_pool"], s["v_pool"] = _pool(n_pages, c, g), _pool(n_pages, c, g)
        s["slots"] = torch.randperm(n_pages * c["page"], generator=g, device="cuda")[:T].contiguous()
        s["positions"] = torch.randint(0, c["pos"], (T,), generator=g, device="cuda").to(torch.int32)
        i = torch.arange(c["rot"] // 2, device="cuda", dtype=torch.float64)
        s["inv_freq"] = (1e6 ** (-2 * i / c["rot"])).to(torch.float32)
    else:
        q_len, kv_len = _attn_lens(c)
        P, n = c["page"], [_pages(k, c["page"]) for k in kv_len]
        n_pages = sum(n) + 5
        s["k_pool"], s["v_pool"] = _pool(n_pages, c, g), _pool(n_pages, c, g)
        s["table"] = torch.full((c["B"], max(n)), -1, dtype=torch.int32, device="cuda")
        have = torch.arange(max(n), device="cuda")[None, :] < _int32(n)[:, None]
        s["table"][have] = torch.randperm(n_pages, generator=g, device="cuda")[:sum(n)].to(torch.int32)
        wide = 1 + 2 * (torch.rand(c["hd"], generator=g, device="cuda") < 0.02)
        s["q"] = (2 * wide * torch.randn((sum(q_len), c["heads"], c["hd"]), generator=g, device="cuda")).to(
            DTYPES[c["type"]])
        s["q_lens"], s["kv_lens"] = _int32(q_len), _int32(kv_len)
        s["row_offsets"] = _int32([sum(q_len[:b]) for b in range(c["B"] + 1)])
        s["most_rows"] = max(q_len)
    torch.cuda.synchronize()
    return s


# ---- the framework's calls -----------------------------------------------------

_ctx = []


def _context():
    """The binding and one context, as a program keeps them."""
    if not _ctx:
        sys.path.insert(0, os.path.join(ROOT, "xdna.cpp_amd"))
        import mi355x

        _ctx.extend((mi355x, mi355x.Context(0)))
    return _ctx


def _kv_pool(m, s):
    c, k = s["case"], s["k_pool"]
    st = k.stride()
    return m.KvPool(type=TYPE_IDS[c["type"]], n_kv_heads=c["kv_heads"], head_dim=c["hd"], page_tokens=c["page"],
                    n_pages=k.shape[0], k=k.data_ptr(), v=s["v_pool"].data_ptr(), page_stride=st[0],
                    token_stride=st[2 if c["hnd"] else 1], head_stride=st[1 if c["hnd"] else 2])


def _ptr(t):
    return None if t is None else t.data_ptr()


def _call(s):
    """What a program sets up once for its buffers: the call and its outputs."""
    m, ctx = _context()
    c = s["case"]
    if c["kind"] == "plan":
        B, rows = c["B"], s["rows"]
        o = {"row_offsets": torch.empty(B + 1, dtype=torch.int32, device="cuda"),
             "kv_lens": torch.empty(B, dtype=torch.int32, device="cuda"),
             "positions": torch.empty(rows, dtype=torch.int32, device="cuda"),
             "slots": torch.empty(rows, dtype=torch.int64, device="cuda"),
             "head": torch.empty(1, dtype=torch.int32, device="cuda"),
             "status": torch.empty(1, dtype=torch.int32, device="cuda"), "table": s["table"]}
        a = m.KvPlanArgs(n_seqs=B, page_tokens=c["page"], table_cols=s["table"].shape[1],
                         table_stride=s["table"].stride(0), n_free=s["free"].numel(), n_rows=rows,
                         cached=_ptr(s["cached"]), added=_ptr(s["added"]), block_table=_ptr(s["table"]),
                         free_pages=_ptr(s["free"]), free_head=_ptr(s["head"]), free_head_out=_ptr(o["head"]),
                         row_offsets=_ptr(o["row_offsets"]), kv_lens=_ptr(o["kv_lens"]),
                         positions=_ptr(o["positions"]), slots=_ptr(o["slots"]), status=_ptr(o["status"]))
        call = ctx.kv_plan
    elif c["kind"] == "rope":
        T, hd, hq, hk = c["T"], c["hd"], c["heads"], c["kv_heads"]
        qkv, es = s["qkv"], s["qkv"].element_size()
        s["keep"] = _kv_pool(m, s)
        o = {"q": torch.empty((T, hq, hd), dtype=DTYPES[c["type"]], device="cuda"), "k_pool": s["k_pool"],
             "v_pool": s["v_pool"]}
        a = m.QkNormRopeArgs(n_rows=T, n_heads=hq, n_kv_heads=hk, head_dim=hd, rot_dim=c["rot"],
                             rope_mode=m.ROPE_PAIRS if c["pairs"] else m.ROPE_HALVES, in_type=TYPE_IDS[c["in"]],
                             out_type=TYPE_IDS[c["type"]], q=_ptr(qkv), k=_ptr(qkv) + hq * hd * es,
                             v=_ptr(qkv) + (hq + hk) * hd * es, q_stride=qkv.stride(0), k_stride=qkv.stride(0),
                             v_stride=qkv.stride(0), q_bias=_ptr(s["q_bias"]), k_bias=_ptr(s["k_bias"]),
                             v_bias=_ptr(s["v_bias"]), q_norm=_ptr(s["q_norm"]), k_norm=_ptr(s["k_norm"]), eps=EPS,
                             positions=_ptr(s["positions"]), inv_freq=_ptr(s["inv_freq"]), q_out=_ptr(o["q"]),
                             q_out_stride=hq * hd, pool=m.pointer(s["keep"]), slots=_ptr(s["slots"]))
        call = ctx.qk_norm_rope
    else:
        rows = s["q"].shape[0]
        out = torch.empty(s["q"].shape, dtype=DTYPES[c["out"]], device="cuda")
        s["keep"] = _kv_pool(m, s)
        s["ws"] = torch.zeros(ctx.paged_attention_workspace(c["heads"], c["kv_heads"], c["hd"]), dtype=torch.uint8,
                              device="cuda")
        a = m.PagedAttentionArgs(n_rows=rows, n_seqs=c["B"], n_heads=c["heads"], max_added=s["most_rows"],
                                 q=_ptr(s["q"]), q_stride=s["q"].stride(0), pool=m.pointer(s["keep"]),
                                 row_offsets=_ptr(s["row_offsets"]), kv_lens=_ptr(s["kv_lens"]),
                                 block_table=_ptr(s["table"]), table_cols=s["table"].shape[1],
                                 table_stride=s["table"].stride(0), scale=c["hd"] ** -0.5, softcap=c["cap"],
                                 window=c["window"], causal=1, out=_ptr(out), out_type=TYPE_IDS[c["out"]],
                                 out_stride=out.stride(0), workspace=_ptr(s["ws"]), workspace_bytes=s["ws"].numel())
        call, o = ctx.paged_attention, out
    torch.cuda.synchronize()
    return call, a, o


# ---- the plain forms ---------------------------------------------------------


def _plain_plan(s):
    c, P = s["case"], s["case"]["page"]
    cached, added = s["cached"].long(), s["added"].long()
    kv = cached + added
    ends = torch.cumsum(added, 0)
    row_offsets = torch.cat([torch.zeros_like(ends[:1]), ends])
    held, need = (cached + P - 1) // P, (kv + P - 1) // P
    took = torch.cumsum(need - held, 0)
    first = s["head"].long() + took - (need - held)
    col = torch.arange(s["table"].shape[1], device="cuda")[None, :]
    fresh = (col >= held[:, None]) & (col < need[:, None])
    at = (first[:, None] + col - held[:, None]).clamp(0, s["free"].numel() - 1)
    table = torch.where(fresh, s["free"][at], s["table"])
    row = torch.arange(s["rows"], device="cuda")
    b = torch.searchsorted(ends, row, right=True)
    real = b < c["B"]
    b = b.clamp(max=c["B"] - 1)
    pos = cached[b] + row - row_offsets[b]
    pos = torch.where(real, pos, 0)
    page = table[b, (pos // P).clamp(max=table.shape[1] - 1)].long()
    return {"row_offsets": row_offsets.int(), "kv_lens": kv.int(), "positions": pos.int(),
            "slots": torch.where(real, page * P + pos % P, -1), "head": (s["head"] + took[-1:]).int(),
            "status": torch.zeros(1, dtype=torch.int32, device="cuda"), "table": table}


def _heads(s, first, heads, bias, norm):
    """Head vectors in f32, with bias and norm: [T, heads, hd]."""
    c = s["case"]
    x = s["qkv"][:, first * c["hd"]:(first + heads) * c["hd"]].float()
    if bias is not None:
        x = x + bias
    x = x.reshape(c["T"], heads, c["hd"])
    if norm is not None:
        x = x / torch.sqrt((x * x).mean(-1, keepdim=True) + EPS) * norm
    return x


def _rotate(c, x, cos, sin):
    r = c["rot"]
    if c["pairs"]:
        a, b = x[..., 0:r:2], x[..., 1:r:2]
        turned = torch.stack([a * cos - b * sin, b * cos + a * sin], -1).flatten(-2)
    else:
        a, b = x[..., :r // 2], x[..., r // 2:r]
        turned = torch.cat([a * cos - b * sin, b * cos + a * sin], -1)
    return torch.cat([turned, x[..., r:]], -1)


def _plain_rope(s):
    c, hq, hk = s["case"], s["case"]["heads"], s["case"]["kv_heads"]
    angle = s["positions"].double()[:, None, None] * s["inv_freq"].double()
    cos, sin = torch.cos(angle).float(), torch.sin(angle).float()
    q = _rotate(c, _heads(s, 0, hq, s["q_bias"], s["q_norm"]), cos, sin)
    k = _rotate(c, _heads(s, hq, hk, s["k_bias"], s["k_norm"]), cos, sin)
    v = _heads(s, hq + hk, hk, s["v_bias"], None)
    page, at = s["slots"] // c["page"], s["slots"] % c["page"]
    dt = DTYPES[c["type"]]
    for pool, x in ((s["k_pool"], k), (s["v_pool"], v)):
        (pool.transpose(1, 2) if c["hnd"] else pool)[page, at] = x.to(dt)
    return {"q": q.to(dt), "k_pool": s["k_pool"], "v_pool": s["v_pool"]}


def _plain_attn(s):
    c = s["case"]
    B, hk, hd, m = c["B"], c["kv_heads"], c["hd"], s["most_rows"]
    G = c["heads"] // hk
    rows = s["row_offsets"][:-1, None].long() + torch.arange(m, device="cuda")  # [B, m]
    real = torch.arange(m, device="cuda") < s["q_lens"][:, None]
    q = s["q"][torch.where(real, rows, 0)].float().reshape(B, m, hk, G, hd).permute(0, 2, 1, 3, 4)
    table = s["table"].clamp(min=0).long()

    def gathered(pool):
        x = (pool.transpose(1, 2) if c["hnd"] else pool)[table]  # [B, cols, page, hk, hd]
        return x.reshape(B, -1, hk, hd).transpose(1, 2).float().contiguous()  # [B, hk, n, hd]

    score = q.reshape(B, hk, m * G, hd) @ gathered(s["k_pool"]).transpose(2, 3).contiguous()
    score *= hd ** -0.5
    if c["cap"]:
        score = c["cap"] * torch.tanh(score / c["cap"])
    n = score.shape[-1]
    key = torch.arange(n, device="cuda")
    pos = (s["kv_lens"] - s["q_lens"])[:, None] + torch.arange(m, device="cuda")  # [B, m]
    seen = key <= pos[..., None]
    if c["window"]:
        seen &= key > pos[..., None] - c["window"]
    hidden = ~seen.repeat_interleave(G, 1)[:, None]
    score.masked_fill_(hidden, float("-inf"))
    score -= score.amax(-1, keepdim=True)
    p = torch.exp_(score)
    total = p.sum(-1, keepdim=True)
    o = (p @ gathered(s["v_pool"])) / total
    o = o.reshape(B, hk, m, G, hd).permute(0, 2, 1, 3, 4).reshape(B, m, c["heads"], hd)
    return o[real].to(DTYPES[c["out"]])


_PLAIN = {"plan": _plain_plan, "rope": _plain_rope, "attn": _plain_attn}


def run(state):
    if own:
        if "call" not in state:
            state["call"] = _call(state)
        call, args, out = state["call"]
        call(args)
        return out
    return _PLAIN[state["case"]["kind"]](state)


# ---- what a pass cannot do without --------------------------------------------


def work(case):
    c = case
    if c["kind"] == "plan":
        cached, added = _plan_lens(c)
        P, T = c["page"], sum(added)
        fresh = sum(_pages(a + b, P) - _pages(a, P) for a, b in zip(cached, added))
        partly = sum(1 for a, b in zip(cached, added) if a % P and b)
        return {"bytes": 16 * c["B"] + 12 + 8 * fresh + 4 * partly + 12 * (T + 3), "flops": 4 * c["B"] + 3 * T}
    if c["kind"] == "rope":
        T, n = c["T"], (c["heads"] + 2 * c["kv_heads"]) * c["hd"]
        turned = (c["heads"] + c["kv_heads"]) * c["rot"]
        fixed = (4 * n if c["bias"] else 0) + (8 * c["hd"] if c["norm"] else 0) + 2 * c["rot"]
        flops = 3 * turned + (n if c["bias"] else 0) + (4 * (c["heads"] + c["kv_heads"]) * c["hd"] if c["norm"] else 0)
        return {"bytes": T * (n * ((4 if c["in"] == "f32" else 2) + 2) + 12) + fixed, "flops": T * flops}
    q_len, kv_len = _attn_lens(c)
    w = c["window"] or 1 << 60
    pairs = keys = 0
    for q, kv in zip(q_len, kv_len):
        full = max(0, min(q, kv - w))  # rows whose window is full
        first = kv - q + 1  # tokens that the first row would see without a window
        short = q - full
        pairs += full * w + (short * (2 * first + short - 1) // 2 if short else 0)
        keys += kv - max(0, first - w)
    row = c["heads"] * c["hd"]
    return {"bytes": keys * c["kv_heads"] * c["hd"] * 4 + sum(q_len) * row * (2 + (4 if c["out"] == "f32" else 2))
            + 4 * sum(_pages(k, c["page"]) for k in kv_len) + 8 * c["B"], "flops": 4 * row * pairs}


# ---- 64-bit results ------------------------------------------------------------


def exact(case, seed):
    c = case
    if c["kind"] == "plan":
        return None  # whole numbers
    s = prepare(c, seed)
    hd, hk = c["hd"], c["kv_heads"]
    if c["kind"] == "rope":
        T, hq, r = c["T"], c["heads"], c["rot"]
        x = s["qkv"][:, :(hq + 2 * hk) * hd].double().view(T, hq + 2 * hk, hd)
        if c["bias"]:
            x = x + torch.cat([s["q_bias"], s["k_bias"], s["v_bias"]]).double().view(hq + 2 * hk, hd)
        if c["norm"]:
            w = torch.cat([s["q_norm"].expand(hq, hd), s["k_norm"].expand(hk, hd)]).double()
            ms = x[:, :hq + hk].square().sum(-1, keepdim=True) / hd
            x = torch.cat([x[:, :hq + hk] * (ms + EPS).rsqrt() * w, x[:, hq + hk:]], 1)
        # each turned pair is a complex number times e^(i angle)
        lo = torch.arange(0, r, 2, device="cuda") if c["pairs"] else torch.arange(r // 2, device="cuda")
        hi = lo + (1 if c["pairs"] else r // 2)
        angle = s["positions"].double().view(T, 1, 1) * s["inv_freq"].double()
        z = torch.complex(x[:, :hq + hk, lo], x[:, :hq + hk, hi]) * torch.polar(torch.ones_like(angle), angle)
        x = x.clone()
        x[:, :hq + hk, lo], x[:, :hq + hk, hi] = z.real, z.imag
        out = {"q": x[:, :hq]}
        for name, part in (("k_pool", x[:, hq:hq + hk]), ("v_pool", x[:, hq + hk:])):
            pool = s[name].double()
            flat = pool.transpose(1, 2).contiguous() if c["hnd"] else pool
            flat.view(-1, hk, hd)[s["slots"]] = part
            out[name] = flat.transpose(1, 2).contiguous() if c["hnd"] else flat
        return out
    q_len, kv_len = _attn_lens(c)
    G = c["heads"] // hk
    out = torch.zeros(s["q"].shape, dtype=torch.float64, device="cuda")
    first = 0
    for b in range(c["B"]):
        nq, n = q_len[b], kv_len[b]
        pages = s["table"][b, :_pages(n, c["page"])].long()
        for h in range(hk):
            k, v = ((p[pages, h] if c["hnd"] else p[pages, :, h]).reshape(-1, hd)[:n].double()
                    for p in (s["k_pool"], s["v_pool"]))
            for r0 in range(0, nq, 2048):
                m = min(2048, nq - r0)
                pos = n - nq + r0 + torch.arange(m, device="cuda")[:, None]
                key = torch.arange(n, device="cuda")[None, :]
                seen = (key <= pos) & (key > pos - (c["window"] or 1 << 60))
                for j in range(G):
                    sc = (s["q"][first + r0:first + r0 + m, h * G + j].double() @ k.T.contiguous()) / math.sqrt(hd)
                    if c["cap"]:
                        sc = torch.tanh(sc / c["cap"]) * c["cap"]
                    weight = torch.softmax(sc.masked_fill(~seen, -math.inf), -1)
                    out[first + r0:first + r0 + m, h * G + j] = weight @ v
        first += nq
    return out
