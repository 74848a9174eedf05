"""The decode-step operators on quantised weights, as measured work.

Three operators, in the order in which one step of a language model served
from 4-bit weights meets them:

- ``norm``   residual addition + root-mean-square norm; the result either in
             the input's type (``ops.rmsnorm``) or as MX e4m3 bytes with one
             E8M0 scale per 32 elements (``ops.rmsnorm_mx``), laid out as
             ``gemm_mx`` / ``gemm_mx_w4`` / ``gemv_mx_w4`` read them;
- ``gemv``   a few tokens times MX e2m1 weights (32-element groups, E8M0
             scales): activations in bf16/fp16 (``ops.gemv_w4``) or in MX
             e4m3 (``ops.gemv_mx_w4``);
- ``sample`` temperature, top-k, top-p, min-p and the draw of one token for
             each row from a given uniform number (``ops.sample``).
"""

import math

import numpy as np
import torch

own = False

E2M1 = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)
DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
EPS = 1e-6


def listed():
    return [
        # one token enters a layer: latency is all that counts
        {"name": "norm_one_token", "op": "norm", "rows": 1, "k": 4096, "dtype": "bf16", "residual": True, "mx": True},
        # a prompt of ordinary length
        {"name": "norm_prompt", "op": "norm", "rows": 2048, "k": 4096, "dtype": "bf16", "residual": True, "mx": True},
        # a full batch of prompts at a wide model: pure bandwidth
        {"name": "norm_batch", "op": "norm", "rows": 16384, "k": 8192, "dtype": "bf16", "residual": True, "mx": True},
        # odd width and row count, the result kept in 16 bits
        {"name": "norm_odd_width", "op": "norm", "rows": 777, "k": 5003, "dtype": "fp16", "residual": True, "mx": False},
        # single-stream decoding: a square projection for one token
        {"name": "gemv_one_token", "op": "gemv", "m": 1, "n": 4096, "k": 4096, "act": "bf16", "bf16_out": False},
        # a few sequences, odd output count, K that ends inside a scale tile
        {"name": "gemv_odd", "op": "gemv", "m": 5, "n": 5001, "k": 2112, "act": "fp16", "bf16_out": False},
        # a small serving batch on 8-bit activations
        {"name": "gemv_mx_batch", "op": "gemv", "m": 16, "n": 8192, "k": 8192, "act": "mx", "bf16_out": False},
        # the output head for one token: the largest stream of weights
        {"name": "gemv_head", "op": "gemv", "m": 1, "n": 100000, "k": 8192, "act": "bf16", "bf16_out": False},
        # the largest batch that is still bound by the weights
        {"name": "gemv_mx_wide", "op": "gemv", "m": 64, "n": 28000, "k": 8192, "act": "mx", "bf16_out": True},
        # one user's next token with the usual filters
        {"name": "sample_one", "op": "sample", "rows": 1, "vocab": 32000, "dtype": "bf16", "pad": 0, "params": "usual"},
        # a small batch over an odd vocabulary in a padded buffer, no filter
        {"name": "sample_free", "op": "sample", "rows": 24, "vocab": 50001, "dtype": "fp32", "pad": 47, "params": "free"},
        # a large serving batch, every request with settings of its own
        {"name": "sample_batch", "op": "sample", "rows": 256, "vocab": 131072, "dtype": "bf16", "pad": 0, "params": "mixed"},
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["norm", "gemv", "sample"])
    if op == "norm":
        mx = rng.random() < 0.6
        k = 64 * _log_int(rng, 4, 128) if mx else _log_int(rng, 256, 8192)
        return {"op": op, "rows": _log_int(rng, 1, 8192), "k": k, "dtype": rng.choice(["bf16", "bf16", "fp16", "fp32"]),
                "residual": rng.random() < 0.7, "mx": mx}
    if op == "gemv":
        return {"op": op, "m": _log_int(rng, 1, 64), "n": _log_int(rng, 500, 28000), "k": 64 * _log_int(rng, 8, 128),
                "act": rng.choice(["bf16", "fp16", "mx"]), "bf16_out": rng.random() < 0.3}
    return {"op": op, "rows": _log_int(rng, 1, 256), "vocab": _log_int(rng, 8000, 131072), "dtype": rng.choice(["bf16", "fp16", "fp32"]),
            "pad": rng.choice([0, 0, 7, 64]), "params": rng.choice(["usual", "free", "mixed", "nucleus", "minp"])}


# ---- inputs ----------------------------------------------------------------

def _tiles(k):
    return (k + 127) // 128


def _prepare_norm(c, g):
    dt = DTYPES[c["dtype"]]
    shape = (c["rows"], c["k"])
    # a residual stream: most channels near one, a few far larger
    loud = torch.where(torch.rand(c["k"], generator=g, device="cuda") < 0.01, 20.0, 1.0)
    x = (torch.randn(shape, generator=g, device="cuda") * 0.7).to(dt)
    res = (torch.randn(shape, generator=g, device="cuda") * loud).to(dt) if c["residual"] else None
    weight = (1.0 + 0.2 * torch.randn(c["k"], generator=g, device="cuda")).to(dt)
    return {"op": "norm", "mx": c["mx"], "x": x, "residual": res, "weight": weight}


def _e2m1_codes():
    """For each of 256 equally likely draws the code that a normal weight,
    scaled by its group's largest, is rounded to."""
    p = (torch.arange(256, dtype=torch.float64) + 0.5) / 256
    v = torch.erfinv(2 * p - 1) * math.sqrt(2.0) * 1.9
    near = (v.abs()[:, None] - torch.tensor(E2M1, dtype=torch.float64)).abs().argmin(dim=1)
    return (near + 8 * (v < 0)).to(torch.uint8)


def _prepare_gemv(c, g):
    m, n, k = c["m"], c["n"], c["k"]
    codes = _e2m1_codes().cuda()
    lo = torch.randint(0, 256, (n, k // 2), generator=g, device="cuda", dtype=torch.uint8)
    w = codes[lo.int()]
    lo = torch.randint(0, 256, (n, k // 2), generator=g, device="cuda", dtype=torch.uint8)
    w |= codes[lo.int()] << 4
    sw = torch.randint(117, 122, (_tiles(k), n, 4), generator=g, device="cuda", dtype=torch.uint8)
    s = {"op": "gemv", "act": c["act"], "bf16_out": c["bf16_out"], "w": w, "sw": sw}
    x = torch.randn((m, k), generator=g, device="cuda")
    if c["act"] == "mx":
        s["q"] = (x * 120.0).clamp(-448, 448).to(torch.float8_e4m3fn).view(torch.uint8)
        s["sq"] = torch.randint(118, 122, (_tiles(k), m, 4), generator=g, device="cuda", dtype=torch.uint8)
    else:
        s["x"] = x.to(DTYPES[c["act"]])
    return s


def _prepare_sample(c, g):
    rows, vocab = c["rows"], c["vocab"]
    buf = torch.randn((rows, vocab + c["pad"]), generator=g, device="cuda") * 2.2
    # the few tokens that the text allows, falling off with their rank
    top = 14.0 - 1.3 * torch.arange(1, 257, device="cuda", dtype=torch.float32).log()
    top = top + 0.5 * torch.randn((rows, 256), generator=g, device="cuda")
    # each in a stretch of the vocabulary of its own, so that no two meet
    room = vocab // 256
    at = torch.randint(0, room, (rows, 256), generator=g, device="cuda")
    at += room * torch.randperm(256, generator=g, device="cuda")
    buf.scatter_(1, at, top)
    if c["pad"]:  # what pads the buffer would win if it were read
        buf[:, vocab:] = 100.0
    logits = buf.to(DTYPES[c["dtype"]])[:, :vocab]
    u = torch.rand(rows, generator=g, device="cuda")
    kinds = {  # temperature, top_k, top_p, min_p
        "usual": [(0.8, 50, 0.95, 0.0)],
        "free": [(1.0, 0, 1.0, 0.0)],
        "nucleus": [(1.0, 0, 0.9, 0.0)],
        "minp": [(1.2, 0, 1.0, 0.05)],
        "mixed": [(0.8, 50, 0.95, 0.0), (1.0, 0, 1.0, 0.0), (0.7, 0, 0.9, 0.0), (0.0, 0, 1.0, 0.0),
                  (1.3, 0, 1.0, 0.05), (1.0, 200, 1.0, 0.0), (0.6, 20, 0.8, 0.02), (1.0, 0, 0.95, 0.0)],
    }[c["params"]]
    if c["params"] == "mixed":
        row = [kinds[i % len(kinds)] for i in range(rows)]
        t, k, p, q = zip(*row)
        params = {"temperature": torch.tensor(t, device="cuda"), "top_k": torch.tensor(k, device="cuda", dtype=torch.int32),
                  "top_p": torch.tensor(p, device="cuda"), "min_p": torch.tensor(q, device="cuda")}
    else:
        t, k, p, q = kinds[0]
        params = {"temperature": t, "top_k": k, "top_p": p, "min_p": q}
    return {"op": "sample", "logits": logits, "u": u, "params": params}


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed * 7919 + 11)
    return {"norm": _prepare_norm, "gemv": _prepare_gemv, "sample": _prepare_sample}[case["op"]](case, g)


# ---- one pass --------------------------------------------------------------

def run(state):
    if own:
        return _run_own(state)
    return {"norm": _plain_norm, "gemv": _plain_gemv, "sample": _plain_sample}[state["op"]](state)


def _run_own(s):
    from lambdipy_amd import ops

    if s["op"] == "norm" and s["mx"]:
        out = ops.rmsnorm_mx(s["x"], s["weight"], residual=s["residual"], eps=EPS)
        return (out[0].view(torch.float8_e4m3fn), out[1].view(torch.float8_e8m0fnu)) + tuple(out[2:])
    if s["op"] == "norm":
        out = ops.rmsnorm(s["x"], s["weight"], residual=s["residual"], eps=EPS)
        return out if s["residual"] is not None else (out,)
    if s["op"] == "gemv" and s["act"] == "mx":
        return ops.gemv_mx_w4(s["q"], s["sq"], s["w"], s["sw"], bf16_out=s["bf16_out"])
    if s["op"] == "gemv":
        return ops.gemv_w4(s["x"], s["w"], s["sw"], bf16_out=s["bf16_out"])
    return ops.sample(s["logits"], s["u"], **s["params"])


def _plain_norm(s):
    h = s["x"].float()
    more = ()
    if s["residual"] is not None:
        h = h + s["residual"].float()
        more = (h.to(s["x"].dtype),)
    y = h * torch.rsqrt((h * h).mean(dim=1, keepdim=True) + EPS) * s["weight"].float()
    if not s["mx"]:
        return (y.to(s["x"].dtype),) + more
    rows, k = y.shape
    blocks = y.view(rows, k // 32, 32)
    amax = blocks.abs().amax(dim=2)
    e = torch.frexp(amax)[1] - 9
    e = e + (torch.ldexp(amax, -e) > 448.0)
    e = torch.where(amax > 0, e, torch.zeros_like(e)).clamp(-127, 127)
    q = torch.ldexp(blocks, -e.unsqueeze(2)).view(rows, k // 64, 4, 16)[:, :, [0, 2, 1, 3]]
    sc = torch.nn.functional.pad(e + 127, (0, 4 * _tiles(k) - k // 32), value=127)
    sc = sc.view(rows, _tiles(k), 4).transpose(0, 1).contiguous().to(torch.uint8)
    return (q.reshape(rows, k).to(torch.float8_e4m3fn), sc.view(torch.float8_e8m0fnu)) + more


def _scales(sc, k):
    """Tile-major E8M0 bytes [ceil(k/128), rows, 4] -> factors [rows, k/32, 1]."""
    s = sc.transpose(0, 1).reshape(sc.shape[1], -1)[:, : k // 32]
    return torch.exp2(s.float() - 127.0).unsqueeze(2)


def _plain_gemv(s):
    n, half = s["w"].shape
    k = 2 * half
    lut = torch.tensor(E2M1 + tuple(-v for v in E2M1), device="cuda")
    w = torch.stack([lut[(s["w"] & 15).int()], lut[(s["w"] >> 4).int()]], dim=2)
    w = (w.view(n, k // 32, 32) * _scales(s["sw"], k)).view(n, k)
    if s["act"] == "mx":
        m = s["q"].shape[0]
        x = s["q"].view(torch.float8_e4m3fn).float().view(m, k // 64, 4, 16)[:, :, [0, 2, 1, 3]]
        x = (x.reshape(m, k // 32, 32) * _scales(s["sq"], k)).view(m, k)
    else:
        x = s["x"].float()
    y = x @ w.t()
    return y.to(torch.bfloat16) if s["bf16_out"] else y


def _column(v, like, dtype):
    return (v.to(dtype) if torch.is_tensor(v) else torch.full((like.shape[0],), v, device="cuda", dtype=dtype)).unsqueeze(1)


def _plain_sample(s):
    # 64 bits: a sum over the whole vocabulary decides which side of a
    # border a token is on
    x = s["logits"].double()
    t = _column(s["params"]["temperature"], x, torch.float64)
    k = _column(s["params"]["top_k"], x, torch.int64)
    p = _column(s["params"]["top_p"], x, torch.float64)
    q = _column(s["params"]["min_p"], x, torch.float64)
    x, at = torch.sort(x, dim=1, descending=True, stable=True)
    w = torch.exp((x - x[:, :1]) / torch.where(t > 0, t, 1.0))
    rank = torch.arange(x.shape[1], device="cuda").unsqueeze(0)
    first = rank == 0
    w = torch.where((k <= 0) | (rank < k), w, 0.0)
    before = w.cumsum(dim=1) - w
    keep = ((p >= 1) | (before < p * w.sum(dim=1, keepdim=True))) & (w >= q) & (t > 0) | first
    c = torch.where(keep, w, 0.0).cumsum(dim=1)
    pos = (c <= s["u"].double().unsqueeze(1) * c[:, -1:]).sum(dim=1, keepdim=True)
    return at.gather(1, torch.minimum(pos, keep.sum(dim=1, keepdim=True) - 1)).squeeze(1)


# ---- 64 bits ---------------------------------------------------------------

def exact(case, seed):
    s = prepare(case, seed)
    return {"norm": _exact_norm, "gemv": _exact_gemv, "sample": _exact_sample}[s["op"]](s)


def _exact_norm(s):
    h = s["x"].to(torch.float64)
    if s["residual"] is not None:
        h += s["residual"].to(torch.float64)
    k = h.shape[1]
    y = (h / (h.pow(2).sum(dim=1) / k + EPS).sqrt()[:, None]) * s["weight"].to(torch.float64)
    more = (h,) if s["residual"] is not None else ()
    if not s["mx"]:
        return (y,) + more
    # the smallest power of two that brings a group's largest to 448 at most
    top = torch.stack([g.abs().max(dim=1).values for g in y.split(32, dim=1)])
    e = torch.ceil(torch.log2(top.clamp_min(1e-300) / 448.0))
    e = torch.where(top > 0, e, 0.0).clamp(-127, 127)  # [k/32, rows]
    f = torch.exp2(e)
    q = torch.empty_like(y)
    for b in range(k // 32):
        base, half = 64 * (b // 2), b % 2
        v = y[:, 32 * b: 32 * b + 32] / f[b][:, None]
        q[:, base + 16 * half: base + 16 * half + 16] = v[:, :16]
        q[:, base + 32 + 16 * half: base + 48 + 16 * half] = v[:, 16:]
    sc = torch.ones(_tiles(k), y.shape[0], 4, dtype=torch.float64, device=y.device)
    for b in range(k // 32):
        sc[b // 4, :, b % 4] = f[b]
    return (q, sc) + more


def _exact_gemv(s):
    n, half = s["w"].shape
    blocks = half // 16
    mag = torch.tensor(E2M1, dtype=torch.float64, device="cuda")
    if s["act"] == "mx":
        q = s["q"].view(torch.float8_e4m3fn).to(torch.float64)
        x = torch.empty_like(q)
        for b in range(blocks):
            f = torch.exp2(s["sq"][b // 4, :, b % 4].to(torch.float64) - 127)[:, None]
            base, h = 64 * (b // 2), b % 2
            x[:, 32 * b: 32 * b + 16] = q[:, base + 16 * h: base + 16 * h + 16] * f
            x[:, 32 * b + 16: 32 * b + 32] = q[:, base + 32 + 16 * h: base + 48 + 16 * h] * f
    else:
        x = s["x"].to(torch.float64)
    out = []
    for r in range(0, n, 4096):  # rows of weights at a time
        codes = s["w"][r: r + 4096]
        w = torch.empty(codes.shape[0], 2 * half, dtype=torch.float64, device="cuda")
        for nib in (0, 1):
            c = (codes >> (4 * nib)) & 15
            w[:, nib::2] = mag[(c & 7).long()] * (1.0 - 2.0 * (c >> 3).double())
        f = s["sw"][:, r: r + 4096].permute(1, 0, 2).flatten(1)[:, :blocks].double() - 127
        w *= torch.pow(2.0, f).repeat_interleave(32, dim=1)
        out.append((w @ x.t()).t())
    return torch.cat(out, dim=1)


def _exact_sample(s):
    x = s["logits"].double().cpu().numpy()
    u = s["u"].double().cpu().numpy()
    tokens = np.empty(x.shape[0], dtype=np.int64)

    def of(name, i):
        v = s["params"][name]
        return v[i].item() if torch.is_tensor(v) else v

    for i, row in enumerate(x):
        t, k, p, q = (of(name, i) for name in ("temperature", "top_k", "top_p", "min_p"))
        order = np.argsort(-row, kind="stable")
        if t <= 0:
            tokens[i] = order[0]
            continue
        if k > 0:
            order = order[:k]
        w = np.exp((row[order] - row[order[0]]) / t)
        if p < 1:  # the shortest prefix that holds a share p
            total = np.cumsum(w)
            order = order[: max(1, int(np.searchsorted(total, p * total[-1], side="left")) + 1)]
            w = w[: order.size]
        w = w[: max(1, int((w >= q).sum()))]
        total = np.cumsum(w)
        at = int(np.searchsorted(total, u[i] * total[-1], side="right"))
        tokens[i] = order[min(at, w.size - 1)]
    return torch.from_numpy(tokens)


# ---- what a pass cannot do without ------------------------------------------

def work(case):
    size = {"bf16": 2, "fp16": 2, "fp32": 4}
    if case["op"] == "norm":
        b, (r, k) = size[case["dtype"]], (case["rows"], case["k"])
        out = r * k + r * k // 32 if case["mx"] else r * k * b
        return {"bytes": r * k * b * (3 if case["residual"] else 1) + k * b + out, "flops": 6 * r * k}
    if case["op"] == "gemv":
        m, n, k = case["m"], case["n"], case["k"]
        act = m * k + m * k // 32 if case["act"] == "mx" else m * k * 2
        return {"bytes": n * k // 2 + n * k // 32 + act + m * n * (2 if case["bf16_out"] else 4), "flops": 2 * m * n * k}
    r, v = case["rows"], case["vocab"]
    return {"bytes": r * v * size[case["dtype"]] + 12 * r, "flops": 4 * r * v}
