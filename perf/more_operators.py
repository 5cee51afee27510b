"""Performance cases of the operators of a layer in 8-bit integers and of what a
model's logits are read for, each one call through the public entry points.

Kinds of case (field ``kind``):

* ``norm``     one mi355x_norm_q8 call: the residual's addition, the
               root-mean-square norm, and the row in 8 bits with its scale.
* ``swiglu``   one mi355x_swiglu_q8 call: silu(gate) * up in 8 bits with a scale
               for each row.
* ``matmul``   one mi355x_matmul_q8 call: rows of 8-bit integers times a weight
               of 8-bit integers, a scale for each row and each output channel.
* ``logprobs`` one mi355x_logprobs call: log probabilities of given tokens, the
               entropy and the most likely tokens of each row of logits.

8-bit codes are whole numbers, -127 to 127, and returned as they are: round to
nearest, ties to even, of the exact quotient, so they are equal or wrong.
"""
import math
import os
import random
import sys

import torch

own = False

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
DTYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
BYTES = {"f32": 4, "f16": 2, "bf16": 2}
# ggml's type ids
TYPE_IDS = {"f32": 0, "f16": 1, "bf16": 30}
EPS = 1e-6


def listed():
    return [
        # the norm before a layer's q|k|v product, one token of the 3B shape, the residual stream in f32
        {"name": "norm token 3B", "kind": "norm", "T": 1, "n": 2048, "type": "f32", "res": "f32", "norm": True,
         "pad": 0},
        # a step of decoding requests and a short chunk, rows apart, a product's f16 output onto an f32 residual
        {"name": "norm 131 rows", "kind": "norm", "T": 131, "n": 5120, "type": "f16", "res": "f32", "norm": True,
         "pad": 24},
        # a long prompt's rows
        {"name": "norm chunk 8192", "kind": "norm", "T": 8192, "n": 8192, "type": "bf16", "res": "bf16",
         "norm": True, "pad": 0},
        # the gate of one token of the 3B shape, gate|up from one product
        {"name": "swiglu token 3B", "kind": "swiglu", "T": 1, "n": 11008, "type": "f32", "pad": 0},
        # the gate of a prompt's chunk
        {"name": "swiglu chunk 4096", "kind": "swiglu", "T": 4096, "n": 14336, "type": "bf16", "pad": 0},
        # gate|up of one token of the 3B shape
        {"name": "matmul token 3B", "kind": "matmul", "M": 1, "N": 22016, "K": 2048, "out": "f32", "bias": False},
        # requests that decode together, each with drafted tokens
        {"name": "matmul 37 rows", "kind": "matmul", "M": 37, "N": 17408, "K": 5120, "out": "bf16", "bias": False},
        # q|k|v of a short chunk of the 3B shape, with its biases
        {"name": "matmul qkv 201", "kind": "matmul", "M": 201, "N": 2560, "K": 2048, "out": "f16", "bias": True},
        # a 512-row micro-batch
        {"name": "matmul chunk 512", "kind": "matmul", "M": 512, "N": 4096, "K": 14336, "out": "f32", "bias": False},
        # a long prompt
        {"name": "matmul chunk 8192", "kind": "matmul", "M": 8192, "N": 8192, "K": 8192, "out": "bf16",
         "bias": False},
        # the sampled token and its alternatives, one request, logits as the vocabulary projection leaves them
        {"name": "logprobs token", "kind": "logprobs", "T": 1, "V": 151936, "type": "f32", "tokens": 1, "top": 20,
         "scale": 1.0},
        # scoring a prompt
        {"name": "logprobs prompt 2048", "kind": "logprobs", "T": 2048, "V": 151936, "type": "bf16", "tokens": 1,
         "top": 5, "scale": 1.0},
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _cost(case):
    w = work(case)
    return max(w["bytes"], w["flops"] / 50)


def draw(rng: random.Random):
    kind = rng.choices(["matmul", "norm", "swiglu", "logprobs"], [5, 3, 2, 3])[0]
    most = {k: max(_cost(c) for c in listed() if c["kind"] == k) for k in ("matmul", "norm", "swiglu", "logprobs")}
    t = rng.choice(["f32", "f16", "bf16"])
    while True:
        if kind == "norm":
            # any width; most are the multiples of 64 that models have
            n = _log_int(rng, 64, 16384)
            c = {"kind": "norm", "T": _log_int(rng, 1, 8192), "n": n if rng.random() < 0.3 else -(-n // 64) * 64,
                 "type": t, "res": rng.choice(["", t, "f32"]), "norm": rng.random() < 0.8,
                 "pad": rng.choice([0, 0, 8, 24, 3])}
        elif kind == "swiglu":
            n = _log_int(rng, 64, 32768)
            c = {"kind": "swiglu", "T": _log_int(rng, 1, 8192), "n": n if rng.random() < 0.3 else -(-n // 64) * 64,
                 "type": t, "pad": rng.choice([0, 0, 8, 24, 3])}
        elif kind == "matmul":
            N = _log_int(rng, 16, 32768)
            c = {"kind": "matmul", "M": _log_int(rng, 1, 8192), "N": N if rng.random() < 0.3 else -(-N // 64) * 64,
                 "K": _log_int(rng, 4, 1024) * 16, "out": t, "bias": rng.random() < 0.3}
        else:
            c = {"kind": "logprobs", "T": _log_int(rng, 1, 2048), "V": _log_int(rng, 1000, 262144), "type": t,
                 "tokens": rng.choice([1, 1, 1, 4]), "top": rng.choice([0, 1, 5, 20, 64]),
                 "scale": rng.choice([1.0, 1.0, 1.25, 0.7])}
        if _cost(c) <= most[kind]:
            return c


# ---- inputs ------------------------------------------------------------------


def _rand(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed * 1000003 + 31)
    return g


def _normal(shape, g):
    return torch.randn(shape, generator=g, device="cuda")


def _codes(rows, cols, g):
    """Rows of normal values in 8 bits: the largest of some thousands lies four deviations out."""
    return (_normal((rows, cols), g) * 32).round_().clamp_(-127, 127).to(torch.int8)


def prepare(case, seed):
    c = case
    g = _rand(seed)
    s = {"case": c}
    if c["kind"] == "norm":
        # a few channels are much larger, as in trained models' residual streams
        wide = 1 + 20 * (torch.rand(c["n"], generator=g, device="cuda") < 0.005)
        shape = (c["T"], c["n"] + c["pad"])
        s["x"] = (0.5 * _normal(shape, g)).to(DTYPES[c["type"]])
        s["residual"] = None
        if c["res"]:
            s["residual"] = _normal(shape, g)
            s["residual"][:, :c["n"]] *= wide
            s["residual"] = s["residual"].to(DTYPES[c["res"]])
        s["norm"] = (1 + 0.3 * _normal((c["n"],), g)) / wide.sqrt() if c["norm"] else None
    elif c["kind"] == "swiglu":
        # gate and up of a row side by side, as one product gives them
        s["gu"] = (1.5 * _normal((c["T"], 2 * c["n"] + c["pad"]), g)).to(DTYPES[c["type"]])
    elif c["kind"] == "matmul":
        s["x"], s["w"] = _codes(c["M"], c["K"], g), _codes(c["N"], c["K"], g)
        s["x_scales"] = torch.exp(0.5 * _normal((c["M"],), g)) * (4 / 127)
        s["w_scales"] = torch.exp(0.2 * _normal((c["N"],), g)) * (0.08 / 127)
        s["bias"] = _normal((c["N"],), g) if c["bias"] else None
    else:
        T, V = c["T"], c["V"]
        x = torch.empty((T, V), dtype=DTYPES[c["type"]], device="cuda")
        for at in range(0, T, 256):
            x[at:at + 256] = (2.5 * _normal((min(256, T - at), V), g)).to(x.dtype)
        # a few tokens of each row are likely
        likely = torch.randint(0, V, (T, 12), generator=g, device="cuda")
        x.scatter_(1, likely, (12 + 3 * _normal((T, 12), g)).to(x.dtype))
        s["logits"] = x
        s["tokens"] = torch.where(torch.rand((T, c["tokens"]), generator=g, device="cuda") < 0.7,
                                  likely[:, :c["tokens"]],
                                  torch.randint(0, V, (T, c["tokens"]), generator=g, device="cuda")).to(torch.int32)
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


def _ptr(t):
    return None if t is None else t.data_ptr()


def _call(s):
    """What a program sets up once for its buffers: the call and its outputs."""
    m, ctx = _context()
    c = s["case"]

    def empty(*shape, dtype=torch.float32):
        return torch.empty(shape, dtype=dtype, device="cuda")

    if c["kind"] == "norm":
        T, n, x, r = c["T"], c["n"], s["x"], s["residual"]
        o = {"codes": empty(T, n, dtype=torch.int8), "scales": empty(T)}
        if r is not None:
            o["residual"] = torch.empty((T, n), dtype=r.dtype, device="cuda")
        a = m.NormQ8Args(n_rows=T, n=n, type=TYPE_IDS[c["type"]], x=_ptr(x), x_stride=x.stride(0),
                         residual_type=TYPE_IDS[c["res"] or c["type"]], residual=_ptr(r),
                         residual_stride=0 if r is None else r.stride(0), residual_out=_ptr(o.get("residual")),
                         residual_out_stride=n, norm=_ptr(s["norm"]), eps=EPS, q=_ptr(o["codes"]), q_stride=n,
                         scales=_ptr(o["scales"]))
        call = ctx.norm_q8
    elif c["kind"] == "swiglu":
        T, n, gu = c["T"], c["n"], s["gu"]
        o = {"codes": empty(T, n, dtype=torch.int8), "scales": empty(T)}
        a = m.SwigluQ8Args(n_rows=T, n=n, type=TYPE_IDS[c["type"]], gate=_ptr(gu), gate_stride=gu.stride(0),
                           up=_ptr(gu) + n * gu.element_size(), up_stride=gu.stride(0), q=_ptr(o["codes"]),
                           q_stride=n, scales=_ptr(o["scales"]))
        call = ctx.swiglu_q8
    elif c["kind"] == "matmul":
        M, N, K = c["M"], c["N"], c["K"]
        o = {"out": empty(M, N, dtype=DTYPES[c["out"]])}
        s["ws"] = torch.zeros(ctx.matmul_q8_workspace(), dtype=torch.uint8, device="cuda")
        a = m.MatmulQ8Args(n_rows=M, n_out=N, k=K, x=_ptr(s["x"]), x_stride=K, x_scales=_ptr(s["x_scales"]),
                           w=_ptr(s["w"]), w_stride=K, w_scales=_ptr(s["w_scales"]), bias=_ptr(s["bias"]),
                           out=_ptr(o["out"]), out_type=TYPE_IDS[c["out"]], out_stride=N, workspace=_ptr(s["ws"]),
                           workspace_bytes=s["ws"].numel())
        call = ctx.matmul_q8
    else:
        T, V, x, k, top = c["T"], c["V"], s["logits"], c["tokens"], c["top"]
        o = {"logprobs": empty(T, k), "entropy": empty(T), "top": empty(T, top, dtype=torch.int32),
             "top_logprobs": empty(T, top)}
        s["ws"] = torch.zeros(ctx.logprobs_workspace(), dtype=torch.uint8, device="cuda")
        a = m.LogprobsArgs(n_rows=T, n_vocab=V, type=TYPE_IDS[c["type"]], logits=_ptr(x), stride=x.stride(0),
                           scale=c["scale"], n_tokens=k, tokens=_ptr(s["tokens"]), token_logprobs=_ptr(o["logprobs"]),
                           entropy=_ptr(o["entropy"]), n_top=top, top_tokens=_ptr(o["top"]),
                           top_logprobs=_ptr(o["top_logprobs"]), workspace=_ptr(s["ws"]),
                           workspace_bytes=s["ws"].numel())
        call = ctx.logprobs
    torch.cuda.synchronize()
    return call, a, o


# ---- the plain forms ---------------------------------------------------------


def _quantized(t):
    """Rows of 64-bit values in 8 bits (a value may lie next to a border), and the largest magnitude of each."""
    most = t.abs().amax(1, keepdim=True)
    return torch.round(t * 127 / torch.where(most > 0, most, 1)).to(torch.int8), most[:, 0]


def _plain_norm(s):
    c, n = s["case"], s["case"]["n"]
    h, o = s["x"][:, :n], {}
    if s["residual"] is not None:
        h = (h.float() + s["residual"][:, :n].float()).to(s["residual"].dtype)
        o["residual"] = h
    t = h.double()
    r = torch.ones((), dtype=torch.float64, device="cuda")
    if s["norm"] is not None:
        r = 1 / torch.sqrt((t * t).mean(1) + EPS)
        t = t * s["norm"].double()
    o["codes"], most = _quantized(t)
    o["scales"] = (most * r / 127).float()
    return o


def _plain_swiglu(s):
    n = s["case"]["n"]
    g, u = s["gu"][:, :n].double(), s["gu"][:, n:2 * n].double()
    codes, most = _quantized(g / (1 + torch.exp(-g)) * u)
    return {"codes": codes, "scales": (most / 127).float()}


def _plain_matmul(s):
    # products of 8-bit integers are exact in f32, their sum to its rounding
    y = s["x"].float() @ s["w"].float().T
    y = y * s["w_scales"] * s["x_scales"][:, None]
    if s["bias"] is not None:
        y = y + s["bias"]
    return {"out": y.to(DTYPES[s["case"]["out"]])}


def _plain_logprobs(s):
    c = s["case"]
    x = s["logits"].float()
    z = c["scale"] * (x - x.amax(1, keepdim=True))
    e = torch.exp(z)
    total = e.sum(1, keepdim=True)
    log_total = torch.log(total)
    o = {"logprobs": torch.gather(z, 1, s["tokens"].long()) - log_total,
         "entropy": (log_total - (e * z).sum(1, keepdim=True) / total)[:, 0]}
    del e
    # equal logits: the lowest token first
    order = torch.sort(x, dim=1, descending=True, stable=True).indices[:, :c["top"]]
    o["top"] = order.to(torch.int32)
    o["top_logprobs"] = torch.gather(z, 1, order) - log_total
    return o


_PLAIN = {"norm": _plain_norm, "swiglu": _plain_swiglu, "matmul": _plain_matmul, "logprobs": _plain_logprobs}


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
    if c["kind"] == "norm":
        moved = BYTES[c["type"]] + (2 * BYTES[c["res"]] if c["res"] else 0) + 1
        ops = 2 + (1 if c["res"] else 0) + (3 if c["norm"] else 0)
        return {"bytes": c["T"] * (c["n"] * moved + 4) + (4 * c["n"] if c["norm"] else 0),
                "flops": c["T"] * c["n"] * ops}
    if c["kind"] == "swiglu":
        return {"bytes": c["T"] * (c["n"] * (2 * BYTES[c["type"]] + 1) + 4), "flops": 6 * c["T"] * c["n"]}
    if c["kind"] == "matmul":
        M, N, K = c["M"], c["N"], c["K"]
        return {"bytes": (M + N) * (K + 4) + M * N * BYTES[c["out"]] + (4 * N if c["bias"] else 0),
                "flops": 2 * M * N * K}
    T, V = c["T"], c["V"]
    return {"bytes": T * (V * BYTES[c["type"]] + 8 * c["tokens"] + 8 * c["top"] + 4), "flops": 6 * T * V}


# ---- 64-bit results ------------------------------------------------------------


def exact(case, seed):
    c = case
    s = prepare(c, seed)
    if c["kind"] == "norm":
        n = c["n"]
        out = {"codes": None}
        h = s["x"][:, :n].double()
        if c["res"]:
            h = h + s["residual"][:, :n].double()
            out["residual"] = h
            h = h.float().to(DTYPES[c["res"]]).double()  # the norm is that of the stored residual
        peak = h
        if c["norm"]:
            peak = h * s["norm"].double() * (h.square().sum(1, keepdim=True) / n + EPS).rsqrt()
        out["scales"] = peak.abs().max(1).values / 127
        return out
    if c["kind"] == "swiglu":
        g, u = s["gu"].double()[:, :2 * c["n"]].split(c["n"], 1)
        return {"codes": None, "scales": (g * torch.sigmoid(g) * u).abs().max(1).values / 127}
    if c["kind"] == "matmul":
        y = (s["w"].double() * s["w_scales"].double()[:, None]) @ (s["x"].double() * s["x_scales"].double()[:, None]).T
        if c["bias"]:
            y += s["bias"].double()[:, None]
        return {"out": y.T.contiguous()}
    rows = []
    for at in range(0, c["T"], 128):
        x = s["logits"][at:at + 128].double() * c["scale"]
        lse = torch.logsumexp(x, 1, keepdim=True)
        lp = x - lse
        given = lp.gather(1, s["tokens"][at:at + 128].long())
        rows.append((given, -(lp.exp() * lp).sum(1), lp.topk(c["top"], 1).values))
    given, entropy, best = (torch.cat(v) for v in zip(*rows))
    return {"logprobs": given, "entropy": entropy, "top": None, "top_logprobs": best}
