"""The decode-step operators against plain 64-bit implementations.

u(t) below is half a step of a type, the most that one rounding is off
relative to the value: bf16 2^-8, fp16 2^-11, f32 2^-24, e4m3 2^-4.
"""

import pytest
import torch

from lambdipy_amd import ops

gpu = pytest.mark.gpu
built = pytest.mark.skipif(not ops.extension_available(),
                           reason="extension not built")
DEV = "cuda"
TYPES = [torch.bfloat16, torch.float16, torch.float32]


def _u(dtype):
    return torch.finfo(dtype).eps / 2


def _gen(seed):
    return torch.Generator(device="cpu").manual_seed(seed)


def _randn(shape, seed, dtype=torch.float32, scale=1.0):
    return (torch.randn(*shape, generator=_gen(seed)) * scale).to(dtype).to(DEV)


# ---- residual + RMS norm ---------------------------------------------------

# f32 arithmetic of a norm, relative to y: the sum of squares of n <= 2^17
# non-negative terms is added in chains of at most 8 * 17 within a thread and
# 22 steps across the workgroup, each off by u, the squares by 3u (two of
# them h's): its root by half of (158 + 3)u; division, rsqrt (2 ulp) and two
# products by at most 8u more. 90 u = 5.4e-6.
NORM_REL = 90 * 2.0 ** -24


def _norm64(x, weight, residual, eps):
    h = x.double()
    if residual is not None:
        h = h + residual.double()
    y = h / torch.sqrt((h * h).mean(dim=-1, keepdim=True) + eps)
    return y * weight.double(), h


def _near(got, want, rel, dtype):
    """|got - want| within rel of want, or half the type's smallest step."""
    small = torch.finfo(dtype).smallest_normal * torch.finfo(dtype).eps / 2
    err = (got.double() - want).abs()
    return bool((err <= rel * want.abs() + small).all())


NORM_SHAPES = [(1, 1), (3, 7), (1, 64), (5, 63), (2, 2048), (3, 2049),
               (2, 4096), (1, 5003), (4, 8192), (2, 8200), (1, 32768),
               (2, 33001), (1, 100001), (0, 128), (300, 130)]


@gpu
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows,k", NORM_SHAPES)
@pytest.mark.parametrize("residual", [False, True])
def test_rmsnorm(rows, k, dtype, residual):
    x = _randn((rows, k), 1, dtype, 3.0)
    w = _randn((k,), 2, dtype)
    r = _randn((rows, k), 3, dtype) if residual else None
    out = ops.rmsnorm(x, w, residual=r, eps=1e-5)
    y64, h64 = _norm64(x, w, r, 1e-5)
    y = out[0] if residual else out
    assert y.dtype == dtype and y.shape == x.shape
    assert _near(y, y64, _u(dtype) + NORM_REL, dtype)
    if residual:
        assert out[1].dtype == dtype and out[1].shape == x.shape
        assert _near(out[1], h64, _u(dtype) + 2.0 ** -24, dtype)


def _mx_rows(sc, k):
    """Tile-major scale bytes -> [rows, k/32]."""
    return sc.permute(1, 0, 2).flatten(1)[:, : k // 32]


def _mx_values(q, sc):
    rows, k = q.shape
    d = q.view(torch.float8_e4m3fn).double().view(rows, k // 64, 4, 16)
    d = d[:, :, [0, 2, 1, 3]].reshape(rows, k // 32, 32)
    return (d * torch.exp2(_mx_rows(sc, k).double() - 127).unsqueeze(2)).view(rows, k)


@gpu
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows,k", [(1, 64), (3, 128), (7, 192), (2, 2048),
                                    (5, 2112), (33, 4096), (2, 8192),
                                    (3, 8256), (2, 32832), (0, 64)])
@pytest.mark.parametrize("residual", [False, True])
def test_rmsnorm_mx(rows, k, dtype, residual):
    x = _randn((rows, k), 4, dtype, 2.0)
    # blocks whose largest elements differ by many powers of two
    w = (_randn((k,), 5) * torch.exp2(torch.arange(k, device=DEV) // 32 % 11 - 5.0))
    r = _randn((rows, k), 6, dtype) if residual else None
    out = ops.rmsnorm_mx(x, w, residual=r, eps=1e-5)
    q, sc = out[:2]
    y64, h64 = _norm64(x, w, r, 1e-5)
    assert q.shape == (rows, k) and q.dtype == torch.uint8
    assert sc.shape == ((k + 127) // 128, rows, 4) and sc.dtype == torch.uint8
    if residual:
        assert _near(out[2], h64, _u(dtype) + 2.0 ** -24, dtype)
    if rows == 0:
        return
    pad = sc.permute(1, 0, 2).reshape(rows, -1)[:, k // 32:]
    assert bool((pad == 127).all())
    s = torch.exp2(_mx_rows(sc, k).double() - 127)
    amax = y64.view(rows, k // 32, 32).abs().amax(dim=2)
    # the largest fills (224, 448] of its scale, up to y's own f32 error
    assert bool((amax <= 448 * s * (1 + NORM_REL)).all())
    assert bool((amax > 224 * s * (1 - NORM_REL)).all())
    # e4m3: half a step of the value, or of its smallest numbers (2^-9)
    step = (s * 2.0 ** -10).repeat_interleave(32, dim=1)
    err = (_mx_values(q, sc) - y64).abs()
    assert bool((err <= torch.maximum(2.0 ** -4 * y64.abs(), step)
                 + 2 * NORM_REL * y64.abs()).all())


@gpu
def test_rmsnorm_mx_equals_quantize_of_the_plain_norm():
    # f32 in and out: the same y goes through both quantisers
    x = _randn((37, 1088), 7)
    w = _randn((1088,), 8)
    y = ops.rmsnorm(x, w)
    q, sc = ops.rmsnorm_mx(x, w)
    q2, sc2 = ops.quantize_mx(y)
    assert torch.equal(q, q2)
    assert torch.equal(_mx_rows(sc, 1088), _mx_rows(sc2, 1088))


@gpu
def test_rmsnorm_mx_feeds_the_mx_products():
    # f32 in and out, so that both ways hand the same bytes to the products
    x, w = _randn((256, 512), 9), _randn((512,), 10)
    wq, ws = ops.quantize_mx(_randn((256, 512), 11))
    w4, s4 = ops.quantize_mx_fp4(_randn((256, 512), 11))
    q, sc = ops.rmsnorm_mx(x, w)
    q2, sc2 = ops.quantize_mx(ops.rmsnorm(x, w))
    assert torch.equal(ops.gemm_mx(q, sc, wq, ws), ops.gemm_mx(q2, sc2, wq, ws))
    assert torch.equal(ops.gemm_mx_w4(q, sc, w4, s4),
                       ops.gemm_mx_w4(q2, sc2, w4, s4))


@gpu
@pytest.mark.parametrize("mx", [False, True])
def test_rmsnorm_strided_and_shaped(mx):
    k = 320
    op = ops.rmsnorm_mx if mx else ops.rmsnorm
    wide = _randn((6, 2 * k + 3), 12, torch.bfloat16)
    w = _randn((k,), 13, torch.bfloat16)
    other = _randn((k, 6), 14, torch.bfloat16).t()  # columns apart
    for x in (wide[:, :k], wide[:, 3:3 + k], wide[::2, k:2 * k],
              wide[0, :k].expand(4, k)):
        r = other[: x.shape[0]]
        got = op(x, w, residual=r)
        want = op(x.contiguous().clone(), w, residual=r.contiguous())
        assert all(torch.equal(a, b) for a, b in zip(got, want))
    x3 = wide[:, :k].reshape(2, 3, k)
    got, want = op(x3, w, residual=x3), op(wide[:, :k], w, residual=wide[:, :k])
    assert got[-1].shape == (2, 3, k)
    assert all(torch.equal(a.flatten(), b.flatten()) for a, b in zip(got, want))
    one = op(wide[1, :k], w)
    want = op(wide[1:2, :k], w)
    a, b = (one[0], want[0]) if mx else (one, want)
    assert torch.equal(a.flatten(), b.flatten())


@gpu
def test_rmsnorm_odd_values():
    w = torch.ones(64, device=DEV)
    # a row of zeros stays zero; its blocks have scale 1
    z = torch.zeros(2, 64, device=DEV)
    assert torch.equal(ops.rmsnorm(z, w), z)
    q, sc = ops.rmsnorm_mx(z, w)
    assert int(q.sum()) == 0 and bool((sc == 127).all())
    # NaN and infinities reach their own row only
    x = _randn((3, 64), 15)
    want = ops.rmsnorm(x, w)
    bad = x.clone()
    bad[0, 5] = float("nan")
    bad[2, 40] = float("inf")
    y = ops.rmsnorm(bad, w)
    assert bool(y[0].isnan().all()) and torch.equal(y[1], want[1])
    assert bool(y[2, 40].isnan()) and float(y[2].nan_to_num(0).abs().sum()) == 0
    q, sc = ops.rmsnorm_mx(bad, w)
    v = q.view(torch.float8_e4m3fn).float()
    assert bool(v[0].isnan().all()) and not bool(v[1].isnan().any())
    assert int(v[2].isnan().sum()) == 1
    # an infinite weight gives the payload's NaN, its neighbours stay finite
    wi = w.clone()
    wi[3] = float("inf")
    v = ops.rmsnorm_mx(x, wi)[0].view(torch.float8_e4m3fn).float()
    assert int(v.isnan().sum()) == 3
    # blocks so small that the scale ends at its lowest
    tiny = torch.full((64,), 2.0 ** -130, device=DEV)
    q, sc = ops.rmsnorm_mx(x, tiny)
    assert bool((sc[0, :, :2] == 0).all())
    y64 = _norm64(x, tiny, None, 1e-6)[0]
    err = (_mx_values(q, sc) - y64).abs()
    assert bool((err <= torch.clamp(2.0 ** -4 * y64.abs(), min=2.0 ** -137) * 1.001).all())


@gpu
def test_rmsnorm_on_another_stream_and_in_a_graph():
    x = _randn((9, 4096), 16, torch.bfloat16)
    r = _randn((9, 4096), 17, torch.bfloat16)
    w = _randn((4096,), 18, torch.bfloat16)
    want = ops.rmsnorm_mx(x, w, residual=r)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        got = ops.rmsnorm_mx(x, w, residual=r)
    s.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        out = ops.rmsnorm_mx(x, w, residual=r)
    for k in range(3):
        x.copy_(_randn((9, 4096), 30 + k, torch.bfloat16))
        g.replay()
        want = ops.rmsnorm_mx(x, w, residual=r)
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(out, want))


@built
def test_rmsnorm_refuses():
    x, w = torch.zeros(2, 64), torch.ones(64)
    for op in (ops.rmsnorm, ops.rmsnorm_mx):
        for bad, why in (
                (lambda: op(x, torch.ones(65)), "weight must be"),
                (lambda: op(x, torch.ones(1, 64)), "weight must be"),
                (lambda: op(x, w.half()), "x's type or f32"),
                (lambda: op(x.long(), w), "supports bf16"),
                (lambda: op(x.double(), w), "supports bf16"),
                (lambda: op(x, w, residual=torch.zeros(1, 64)), "residual must"),
                (lambda: op(x, w, residual=x.half()), "residual must"),
                (lambda: op(x, w, eps=-1.0), "eps"),
                (lambda: op(x, w, eps=float("nan")), "eps"),
                (lambda: op(x, w), "on the ROCm device")):
            with pytest.raises(RuntimeError, match=why):
                bad()
        with pytest.raises(RuntimeError, match="no backward"):
            op(x, w.clone().requires_grad_())
    with pytest.raises(RuntimeError, match="K >= 1"):
        ops.rmsnorm(torch.zeros(2, 0), torch.zeros(0))
    with pytest.raises(RuntimeError, match="K%64"):
        ops.rmsnorm_mx(torch.zeros(2, 65), torch.ones(65))


# ---- 4-bit weights ---------------------------------------------------------

E2M1 = torch.tensor([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0] * 2,
                    dtype=torch.float64) * torch.tensor([1.0] * 8 + [-1.0] * 8)


def _fp4_values(w4, sc):
    n, k = w4.shape[0], 2 * w4.shape[1]
    lut = E2M1.to(w4.device)
    v = torch.stack([lut[(w4 & 15).long()], lut[(w4 >> 4).long()]], dim=2)
    s = torch.exp2(_mx_rows(sc, k).double() - 127).unsqueeze(2)
    return (v.view(n, k // 32, 32) * s).view(n, k)


def _weights(n, k, seed, lo=110, hi=140):
    """Random nibbles and scales; the bytes that pad the last tile are NaN."""
    w4 = torch.randint(0, 256, (n, k // 2), generator=_gen(seed), dtype=torch.uint8)
    sc = torch.randint(lo, hi, ((k + 127) // 128, n, 4), generator=_gen(seed + 1),
                       dtype=torch.uint8)
    if k % 128:
        sc[-1, :, 2:] = 255
    return w4.to(DEV), sc.to(DEV)


def _mx_acts(m, k, seed, lo=118, hi=136):
    q = (_randn((m, k), seed) * 100).clamp(-448, 448).to(torch.float8_e4m3fn)
    sc = torch.randint(lo, hi, ((k + 127) // 128, m, 4), generator=_gen(seed + 1),
                       dtype=torch.uint8)
    if k % 128:
        sc[-1, :, 2:] = 255
    return q.view(torch.uint8), sc.to(DEV)


def _product_ok(got, x64, w64):
    """Every product is exact in f32; k of them are summed in f32 in some
    order: off by at most k u of the sum of their magnitudes (and fp16's
    blocks by one more rounding each). bf16 results: half a step more."""
    want, mag = x64 @ w64.t(), x64.abs() @ w64.abs().t()
    tol = (x64.shape[1] + 64) * 2.0 ** -24 * mag
    if got.dtype == torch.bfloat16:
        tol = tol + 2.0 ** -8 * (want.abs() + tol)
    return bool(((got.double() - want).abs() <= tol).all())


GEMV_SHAPES = [(1, 1, 64), (1, 16, 128), (1, 17, 192), (2, 1000, 1024),
               (5, 333, 2112), (15, 31, 320), (16, 64, 4096), (17, 100, 640),
               (31, 257, 1088), (33, 129, 2048), (64, 64, 8192), (65, 50, 448),
               (130, 40, 576), (0, 8, 64), (3, 0, 64)]


@gpu
@pytest.mark.parametrize("m,n,k", GEMV_SHAPES)
@pytest.mark.parametrize("act", ["bf16", "fp16", "mx"])
@pytest.mark.parametrize("bf16_out", [False, True])
def test_gemv_4bit(m, n, k, act, bf16_out):
    w4, sw = _weights(n, k, 20)
    if act == "mx":
        q, sq = _mx_acts(m, k, 21)
        got = ops.gemv_mx_w4(q, sq, w4, sw, bf16_out=bf16_out)
        x64 = _mx_values(q, sq)
    else:
        x = _randn((m, k), 21, torch.bfloat16 if act == "bf16" else torch.float16, 4.0)
        got = ops.gemv_w4(x, w4, sw, bf16_out=bf16_out)
        x64 = x.double()
    assert got.shape == (m, n)
    assert got.dtype == (torch.bfloat16 if bf16_out else torch.float32)
    if m and n:
        assert _product_ok(got, x64, _fp4_values(w4, sw))


@gpu
def test_gemv_4bit_reads_what_the_quantisers_write():
    x = _randn((7, 1088), 22, torch.bfloat16)
    w4, sw = ops.quantize_mx_fp4(_randn((130, 1088), 23) * 0.02)
    w64 = _fp4_values(w4, sw)
    assert _product_ok(ops.gemv_w4(x, w4, sw), x.double(), w64)
    q, sq = ops.quantize_mx(x.float())
    assert _product_ok(ops.gemv_mx_w4(q, sq, w4, sw), _mx_values(q, sq), w64)


@gpu
@pytest.mark.parametrize("act", ["bf16", "fp16", "mx"])
def test_gemv_4bit_picks_out_single_weights(act):
    # one-hot rows give back the dequantised weights, bit for bit: any mix-up
    # of k between the two operands shows
    k, n = 256, 48
    w4, sw = _weights(n, k, 24)
    for k0 in range(0, k, 64):
        x = torch.zeros(64, k, device=DEV)
        x[torch.arange(64), k0 + torch.arange(64)] = 1.0
        if act == "mx":
            got = ops.gemv_mx_w4(*ops.quantize_mx(x), w4, sw)
        else:
            t = torch.bfloat16 if act == "bf16" else torch.float16
            got = ops.gemv_w4(x.to(t), w4, sw)
        want = _fp4_values(w4, sw)[:, k0:k0 + 64].t()
        assert torch.equal(got.double(), want)


@gpu
@pytest.mark.parametrize("act", ["bf16", "fp16", "mx"])
def test_gemv_4bit_far_scales(act):
    # weights near the ends of f32's exponents
    n, k = 32, 256
    x = torch.ones(3, k, device=DEV)
    for byte in (4, 60, 200, 240):
        w4, sw = _weights(n, k, 25)
        sw.fill_(byte)
        if act == "mx":
            got = ops.gemv_mx_w4(*ops.quantize_mx(x), w4, sw)
        else:
            t = torch.bfloat16 if act == "bf16" else torch.float16
            got = ops.gemv_w4(x.to(t), w4, sw)
        assert _product_ok(got, x.double(), _fp4_values(w4, sw))


@gpu
def test_gemv_4bit_nan_and_inf_stay_in_their_row():
    w4, sw = _weights(40, 256, 26)
    for dtype in (torch.bfloat16, torch.float16):
        x = _randn((20, 256), 27, dtype)
        want = ops.gemv_w4(x, w4, sw)
        bad = x.clone()
        bad[3, 17] = float("nan")
        bad[18, 200] = float("inf")
        got = ops.gemv_w4(bad, w4, sw)
        assert bool(got[3].isnan().all())
        assert not bool(got[18].isfinite().any())
        keep = [i for i in range(20) if i not in (3, 18)]
        assert torch.equal(got[keep], want[keep])


@gpu
def test_gemv_4bit_shapes_strides_and_repeats():
    w4, sw = _weights(70, 320, 28)
    wide = _randn((6, 643), 29, torch.float16)
    for x in (wide[:, :320], wide[:, 3:323], wide[::2, 320:640],
              wide[0, :320].expand(4, 320), _randn((320, 5), 30, torch.float16).t()):
        got = ops.gemv_w4(x, w4, sw)
        want = ops.gemv_w4(x.contiguous().clone(), w4, sw)
        assert torch.equal(got, want)
    x = wide[:, :320]
    assert torch.equal(ops.gemv_w4(x.reshape(2, 3, 320), w4, sw).view(6, 70),
                       ops.gemv_w4(x, w4, sw))
    assert torch.equal(ops.gemv_w4(x[1], w4, sw), ops.gemv_w4(x[1:2], w4, sw)[0])
    # a row's result does not depend on its neighbours
    assert torch.equal(ops.gemv_w4(x[:1], w4, sw), ops.gemv_w4(x, w4, sw)[:1])
    # weights that start anywhere in a buffer
    buf = torch.zeros(w4.numel() + 5, dtype=torch.uint8, device=DEV)
    off = buf[5:].view(w4.shape)
    off.copy_(w4)
    assert torch.equal(ops.gemv_w4(x, off, sw), ops.gemv_w4(x, w4, sw))


@gpu
def test_gemv_4bit_past_2_to_31_bytes():
    # the last rows of 2.2 GB of weights
    n, k = 270001, 16384
    w4 = torch.zeros(n, k // 2, dtype=torch.uint8, device=DEV)
    sw = torch.full((k // 128, n, 4), 127, dtype=torch.uint8, device=DEV)
    tail, st = _weights(64, k, 31)
    w4[-64:], sw[:, -64:] = tail, st
    x = _randn((2, k), 32, torch.bfloat16)
    got = ops.gemv_w4(x, w4, sw)
    assert _product_ok(got[:, -64:], x.double(), _fp4_values(tail, st))
    assert float(got[:, :-64].abs().max()) == 0


@gpu
def test_gemv_4bit_in_a_graph():
    w4, sw = _weights(500, 1024, 33)
    x = _randn((4, 1024), 34, torch.bfloat16)
    ops.gemv_w4(x, w4, sw)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        out = ops.gemv_w4(x, w4, sw)
    for i in range(3):
        x.copy_(_randn((4, 1024), 40 + i, torch.bfloat16))
        g.replay()
        want = ops.gemv_w4(x, w4, sw)
        torch.cuda.synchronize()
        assert torch.equal(out, want)


@built
def test_gemv_4bit_refuses():
    u8 = torch.uint8
    x = torch.zeros(2, 128, dtype=torch.bfloat16)
    w4, sw = torch.zeros(8, 64, dtype=u8), torch.zeros(1, 8, 4, dtype=u8)
    q, sq = torch.zeros(2, 128, dtype=u8), torch.zeros(1, 2, 4, dtype=u8)
    for bad, why in (
            (lambda: ops.gemv_w4(x.float(), w4, sw), "bf16 and fp16"),
            (lambda: ops.gemv_w4(x, w4.int(), sw), "byte tensors"),
            (lambda: ops.gemv_w4(x, w4, sw.int()), "byte tensors"),
            (lambda: ops.gemv_w4(x[:, :64], w4, sw), "fp4 nibbles"),
            (lambda: ops.gemv_w4(x[:, :96], w4[:, :48].contiguous(), sw), "K%64"),
            (lambda: ops.gemv_w4(x, w4.view(2, 4, 64), sw), "fp4 nibbles"),
            (lambda: ops.gemv_w4(x, w4, sw[:, :4]), "scale shapes"),
            (lambda: ops.gemv_w4(x, w4.t().contiguous().t(), sw), "contiguous"),
            (lambda: ops.gemv_w4(x, w4, sw), "on the ROCm device"),
            (lambda: ops.gemv_w4(x[:, :0], w4[:, :0], sw[:0]), "K%64"),
            (lambda: ops.gemv_w4(torch.tensor(1.0).bfloat16(), w4, sw), "expects x"),
            (lambda: ops.gemv_w4(x.clone().requires_grad_(), w4, sw), "no backward"),
            (lambda: ops.gemv_mx_w4(x, sq, w4, sw), "byte tensors"),
            (lambda: ops.gemv_mx_w4(q[0], sq, w4, sw), "expects A"),
            (lambda: ops.gemv_mx_w4(q, sq[:, :1], w4, sw), "scale shapes"),
            (lambda: ops.gemv_mx_w4(q.t().contiguous().t(), sq, w4, sw), "contiguous"),
            (lambda: ops.gemv_mx_w4(q, sq, w4, sw), "on the ROCm device")):
        with pytest.raises(RuntimeError, match=why):
            bad()


# ---- sampling --------------------------------------------------------------

def _sample64(logits, u, temperature=1.0, top_k=0, top_p=1.0, min_p=0.0):
    """The definition, row by row in 64 bits, and for each row how near a
    border decided: the smallest distance of a running weight from a border,
    relative to the row's weight."""
    rows = logits.shape[0]

    def of(v, i):
        return v[i].item() if torch.is_tensor(v) else v

    out, near = [], []
    for i in range(rows):
        x = logits[i].double().cpu()
        x = torch.where(x.isnan(), -torch.inf, x)
        t, k, p, q = (of(v, i) for v in (temperature, top_k, top_p, min_p))
        s, at = torch.sort(x, descending=True, stable=True)
        if s[0] == -torch.inf or not t > 0:
            out.append(-1 if s[0] == -torch.inf else int(at[0]))
            near.append(1.0)
            continue
        w = torch.where(s == s[0], 1.0, torch.exp((s - s[0]) / t))
        if k >= 1:
            w = w[:k]
        c = w.cumsum(0)
        n, gap = len(w), 1.0
        if p < 1:
            n = min(n, int((c - w < p * c[-1]).sum()))
            gap = float((c - p * c[-1]).abs().min() / c[-1])
        if q > 0:
            gap = min(gap, float((w - q)[w != 1.0].abs().min()) if bool((w != 1.0).any()) else 1.0)
        n = max(1, min(n, int((w >= q).sum())))
        c = c[:n]
        want = float(of(u, i)) * float(c[-1])
        out.append(int(at[min(int((c <= want).sum()), n - 1)]))
        near.append(min(gap, float((c - want).abs().min() / c[-1])))
    return torch.tensor(out), torch.tensor(near)


# A weight is off by half of 2^-45 and 2^-44 of itself: over V <= 2^17 of them
# (1 or more in all) a running weight by less than 2^17 * 2^-46 + 2^-44 of the
# row's. A row whose border is nearer than twice that may go to either side.
SAMPLE_NEAR = 2 * (2.0 ** -29 + 2.0 ** -44)


def _same_tokens(got, logits, u, **settings):
    want, near = _sample64(logits, u, **settings)
    far = near > SAMPLE_NEAR
    return bool((got.cpu().flatten()[far] == want[far]).all()) and bool(far.any())


SETTINGS = [dict(), dict(temperature=0.0), dict(temperature=0.3), dict(temperature=5.0),
            dict(top_k=1), dict(top_k=7), dict(top_k=1000), dict(top_k=10 ** 9),
            dict(top_p=0.0), dict(top_p=0.5), dict(top_p=0.97), dict(min_p=0.02),
            dict(min_p=1.0), dict(temperature=0.7, top_k=40, top_p=0.9, min_p=0.01),
            dict(temperature=1.4, top_k=3000, top_p=0.99)]


def _uniform(rows, seed):
    return torch.rand(rows, generator=_gen(seed)).to(DEV)


@gpu
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("settings", SETTINGS)
@pytest.mark.parametrize("rows,v", [(1, 1), (2, 2), (5, 63), (3, 1000), (4, 4097),
                                    (7, 50001), (2, 131072)])
def test_sample(rows, v, dtype, settings):
    x = _randn((rows, v), 50 + v, dtype, 2.5)
    u = _uniform(rows, 51)
    got = ops.sample(x, u, **settings)
    assert got.dtype == torch.int64 and got.shape == (rows,)
    assert _same_tokens(got, x, u, **settings)


@gpu
@pytest.mark.parametrize("dtype", TYPES)
def test_sample_settings_of_each_row(dtype):
    rows, v = 60, 9001
    x = _randn((rows, v), 52, dtype, 3.0)
    g = _gen(53)
    st = dict(temperature=torch.rand(rows, generator=g) * 2 * (torch.rand(rows, generator=g) > 0.2),
              top_k=torch.randint(-1, 300, (rows,), generator=g),
              top_p=0.5 + torch.rand(rows, generator=g).double(),
              min_p=torch.rand(rows, generator=g) * 0.1)
    st = {k: t.to(DEV) for k, t in st.items()}
    u = _uniform(rows, 54)
    got = ops.sample(x, u, **st)
    assert _same_tokens(got, x, u, **st)
    assert torch.equal(got, ops.sample(x, u.double(), **dict(st, top_k=st["top_k"].int())))
    # alone or among others, a row gives the same
    for i in (0, 17, 59):
        one = ops.sample(x[i:i + 1], u[i:i + 1], **{k: t[i:i + 1] for k, t in st.items()})
        assert int(one) == int(got[i])


@gpu
@pytest.mark.parametrize("v", [100, 5000, 70000])
@pytest.mark.parametrize("settings", [dict(), dict(top_k=30), dict(top_k=5000), dict(top_p=0.4),
                                      dict(top_k=4999, top_p=0.8), dict(min_p=0.5)])
def test_sample_ties(v, settings):
    # all equal; two values; a few values: the lowest indices are kept
    one = torch.full((v,), 1.5)
    two = torch.where(torch.arange(v) % 3 == 0, 2.0, 1.0)
    few = (torch.arange(v) * 7919 % 5).float()
    zero = torch.where(torch.arange(v) % 2 == 0, 0.0, -0.0)
    x = torch.stack([one, two, few, zero] * 4).to(DEV)
    u = torch.linspace(0.013, 0.987, 16).to(DEV)
    got = ops.sample(x, u, **settings)
    assert _same_tokens(got, x, u, **settings)


@gpu
@pytest.mark.parametrize("settings", [dict(), dict(top_k=50), dict(top_p=0.9), dict(temperature=0.0),
                                      dict(temperature=1e-3), dict(temperature=1e4, top_p=0.3)])
def test_sample_masked_and_extreme_rows(settings):
    v = 20000
    x = _randn((10, v), 55, scale=3.0)
    inf = float("inf")
    x[0] = -inf                                   # nothing left
    x[1] = -inf
    x[1, 777] = -5.0                              # one left
    x[2, :19000] = torch.finfo(torch.float32).min  # the type's lowest value
    x[3, ::2] = float("nan")
    x[4, 11] = x[4, 19999] = inf                  # two infinite
    x[5] = torch.finfo(torch.float32).min
    x[6, 5], x[6, 6] = 3e38, -3e38                # a range past f32's
    x[7] = float("nan")
    x[8, :] = -inf
    x[8, 100:400] = torch.randn(300, generator=_gen(56)).to(DEV)
    x[9] = x[9] * 1e-30                           # all but equal
    u = torch.linspace(0.05, 0.95, 10).to(DEV)
    got = ops.sample(x, u, **settings)
    assert _same_tokens(got, x, u, **settings)
    assert got[0] == -1 and got[7] == -1 and got[1] == 777


@gpu
def test_sample_draws_by_weight():
    # the ends of u, and the shares of a small row over a grid of it
    w = torch.tensor([0.1, 0.4, 0.2, 0.3])
    n = 1000
    u = ((torch.arange(n) + 0.5) / n).to(DEV)
    got = ops.sample(w.log().expand(n, 4).to(DEV), u)
    share = torch.bincount(got.cpu(), minlength=4) / n
    assert bool(((share - w).abs() <= 1.01 / n).all())
    x = w.log().expand(4, 4).contiguous().to(DEV)
    ends = torch.tensor([0.0, 1.0 - 2.0 ** -24, 1.0, 0.39], device=DEV)
    assert ops.sample(x, ends).tolist() == [1, 0, 0, 1]


@gpu
def test_sample_strided_shaped_and_elsewhere():
    v = 5003
    buf = _randn((6, v + 40), 57, torch.bfloat16, 3.0)
    buf[:, v:] = 100.0
    u = _uniform(6, 58)
    x = buf[:, :v]
    want = ops.sample(x.contiguous(), u, top_p=0.9)
    assert torch.equal(ops.sample(x, u, top_p=0.9), want)
    assert torch.equal(ops.sample(x.reshape(2, 3, v), u.view(2, 3), top_p=0.9).flatten(), want)
    assert ops.sample(x[4], u[4], top_p=0.9).shape == () and \
        int(ops.sample(x[4], u[4], top_p=0.9)) == int(want[4])
    cols = x.t().contiguous().t()  # tokens apart, rows together
    assert torch.equal(ops.sample(cols, u, top_p=0.9), want)
    for off in range(1, 9):  # rows that start anywhere
        y = torch.empty(6 * v + off, dtype=torch.bfloat16, device=DEV)[off:].view(6, v)
        y.copy_(x)
        assert torch.equal(ops.sample(y, u, top_p=0.9), want)
    assert ops.sample(x[:0], u[:0]).shape == (0,)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        got = ops.sample(x, u, top_p=0.9)
    s.synchronize()
    assert torch.equal(got, want)


@gpu
def test_sample_in_two_graphs():
    x = _randn((9, 30000), 59, torch.bfloat16, 3.0)
    u = _uniform(9, 60)
    ops.sample(x, u, top_p=0.9)
    graphs, outs = [], []
    for st in (dict(top_p=0.9), dict(top_k=20)):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(ops.sample(x, u, **st))
        graphs.append(g)
    for i in range(3):
        x.copy_(_randn((9, 30000), 61 + i, torch.bfloat16, 3.0))
        u.copy_(_uniform(9, 70 + i))
        for g in graphs:
            g.replay()
        want = [ops.sample(x, u, top_p=0.9), ops.sample(x, u, top_k=20)]
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(outs, want))


@gpu
def test_sample_a_long_row():
    # more chunks than a wave has lanes, and bins that no list holds
    v = 3_000_001
    x = _randn((1, v), 62, torch.float32, 2.0)
    for st in (dict(), dict(top_k=100000), dict(top_p=0.99), dict(temperature=0.0)):
        u = _uniform(1, 63)
        got = ops.sample(x, u, **st)
        want, _ = _sample64(x, u, **st)
        assert int(got) == int(want)


@built
def test_sample_refuses():
    x, u = torch.zeros(3, 10), torch.zeros(3)
    for bad, why in (
            (lambda: ops.sample(x.long(), u), "supports bf16"),
            (lambda: ops.sample(x, u[:2]), "u must have one value"),
            (lambda: ops.sample(x, u.half()), "f32 or f64"),
            (lambda: ops.sample(x, u.view(3, 1)), "one value for each row"),
            (lambda: ops.sample(x, u, temperature=-1.0), "temperature must be"),
            (lambda: ops.sample(x, u, temperature=float("nan")), "temperature must be"),
            (lambda: ops.sample(x, u, temperature=float("inf")), "temperature must be"),
            (lambda: ops.sample(x, u, top_k=-1), "top_k must be"),
            (lambda: ops.sample(x, u, top_p=1.5), "top_p must be"),
            (lambda: ops.sample(x, u, min_p=-0.1), "min_p must be"),
            (lambda: ops.sample(x, u, top_k=torch.zeros(3)), "int32 or int64"),
            (lambda: ops.sample(x, u, top_p=torch.zeros(3).int()), "f32 or f64"),
            (lambda: ops.sample(x, u, top_p=torch.zeros(2)), "one value for each row"),
            (lambda: ops.sample(torch.zeros(3, 0), u), "V >= 1"),
            (lambda: ops.sample(torch.tensor(1.0), u), "expects logits"),
            (lambda: ops.sample(x, u), "on the ROCm device")):
        with pytest.raises(RuntimeError, match=why):
            bad()


@gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("v", [300, 65535, 65537, 70000, 140001])
@pytest.mark.parametrize("settings", [dict(), dict(top_k=30), dict(top_k=5000), dict(top_p=0.4),
                                      dict(top_k=4999, top_p=0.8), dict(min_p=0.5),
                                      dict(temperature=0.0)])
def test_sample_ties_of_16_bits(dtype, v, settings):
    # more equal logits than 16 bits count, on both sides of zero
    one = torch.full((v,), 1.5)
    low = torch.full((v,), -3.0)
    low[v // 2] = -2.0
    few = (torch.arange(v) * 7919 % 5).float() - 4.0
    zero = torch.where(torch.arange(v) % 2 == 0, 0.0, -0.0)
    x = torch.stack([one, low, few, zero] * 4).to(dtype).to(DEV)
    u = torch.linspace(0.013, 0.987, 16).to(DEV)
    got = ops.sample(x, u, **settings)
    assert _same_tokens(got, x, u, **settings)


@gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("settings", [dict(), dict(top_k=50), dict(top_p=0.9), dict(temperature=0.0),
                                      dict(temperature=1e-3), dict(temperature=1e4, top_p=0.3)])
def test_sample_masked_rows_of_16_bits(dtype, settings):
    v = 20001
    x = _randn((10, v), 65, scale=3.0).to(dtype)
    inf, least = float("inf"), torch.finfo(dtype).min
    x[0] = -inf
    x[1] = -inf
    x[1, 777] = -5.0
    x[2, :19000] = least
    x[3, ::2] = float("nan")
    x[3, 1::4] = -torch.tensor(float("nan"))
    x[4, 11] = x[4, 19999] = inf
    x[5] = least
    x[6, 5], x[6, 6] = torch.finfo(dtype).max, least
    x[7] = float("nan")
    x[8, :] = -inf
    x[8, 100:400] = torch.randn(300, generator=_gen(66)).to(dtype).to(DEV)
    x[9] = x[9] * 2.0 ** -14
    u = torch.linspace(0.05, 0.95, 10).to(DEV)
    got = ops.sample(x, u, **settings)
    assert _same_tokens(got, x, u, **settings)
    assert got[0] == -1 and got[7] == -1 and got[1] == 777


@gpu
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows,k", [(1, 64), (37, 64), (3, 128), (70, 128), (9, 192),
                                    (5, 256), (33, 320), (131, 512), (3, 576), (2, 16384),
                                    (2, 16448)])
def test_rmsnorm_narrow_rows_and_neighbours(rows, k, dtype):
    # several rows to a wave: each has its own sum and its own scale tile
    x = _randn((rows, k), 80, dtype) * torch.exp2(
        torch.arange(rows, device=DEV) % 9 - 4.0).to(dtype).unsqueeze(1)
    w = _randn((k,), 81, dtype)
    y = ops.rmsnorm(x, w)
    assert _near(y, _norm64(x, w, None, 1e-6)[0], _u(dtype) + NORM_REL, dtype)
    q, sc = ops.rmsnorm_mx(x, w)
    one = [ops.rmsnorm_mx(x[i:i + 1], w) for i in range(rows)]
    assert torch.equal(q, torch.cat([o[0] for o in one]))
    assert torch.equal(sc, torch.cat([o[1] for o in one], dim=1))
    y64 = _norm64(x, w, None, 1e-6)[0]
    s = torch.exp2(_mx_rows(sc, k).double() - 127).repeat_interleave(32, dim=1)
    err = (_mx_values(q, sc) - y64).abs()
    assert bool((err <= torch.maximum(2.0 ** -4 * y64.abs(), s * 2.0 ** -10)
                 + 2 * NORM_REL * y64.abs()).all())
    assert bool((sc.permute(1, 0, 2).flatten(1)[:, k // 32:] == 127).all())


# ---- a run of them together ------------------------------------------------

class _Decoder:
    """Two MLP layers and a head on 4-bit weights, as a decode step runs them."""

    def __init__(self, k, hidden, vocab, dtype, seed):
        self.dtype = dtype
        self.norms = [(1 + 0.1 * _randn((k,), seed + i)).to(dtype) for i in range(3)]

        def weights(n, k, s):
            return ops.quantize_mx_fp4(_randn((n, k), s, scale=k ** -0.5))

        self.layers = [(weights(hidden, k, seed + 10 + i), weights(k, hidden, seed + 20 + i))
                       for i in range(2)]
        self.head = weights(vocab, k, seed + 30)

    def step(self, x, u, seen=None):
        note = (lambda *t: None) if seen is None else (lambda *t: seen.append(t))
        h = None
        for (up, down), w in zip(self.layers, self.norms):
            out = ops.rmsnorm_mx(x, w, residual=h)
            q, sc = out[:2]
            note("norm_mx", x, w, h, out)
            h = x if h is None else out[2]
            a = ops.gemv_mx_w4(q, sc, *up, bf16_out=True)
            note("mx", (q, sc), up, a)
            a = torch.relu(a)
            x = ops.gemv_w4(a, *down, bf16_out=True).to(self.dtype)
            note("w4", a, down, x)
        before = h
        y, h = ops.rmsnorm(x, self.norms[2], residual=before)
        note("norm", x, self.norms[2], before, (y, h))
        logits = ops.gemv_w4(y, *self.head)
        note("w4", y, self.head, logits)
        token = ops.sample(logits * 4, u, temperature=0.9, top_k=40, top_p=0.95)
        note("sample", logits * 4, u, token)
        return token, logits


@gpu
@pytest.mark.parametrize("rows", [1, 5, 33])
def test_decode_step(rows):
    # each operator against 64 bits on what the one before it gave
    net = _Decoder(512, 1088, 5003, torch.bfloat16, 100)
    x, u = _randn((rows, 512), 140, torch.bfloat16), _uniform(rows, 141)
    seen = []
    token, _ = net.step(x, u, seen)
    assert token.shape == (rows,) and bool(((0 <= token) & (token < 5003)).all())
    for kind, *t in seen:
        if kind == "norm_mx":
            y64, h64 = _norm64(t[0], t[1], t[2], 1e-6)
            q, sc = t[3][:2]
            s = torch.exp2(_mx_rows(sc, q.shape[1]).double() - 127).repeat_interleave(32, 1)
            err = (_mx_values(q, sc) - y64).abs()
            assert bool((err <= torch.maximum(2.0 ** -4 * y64.abs(), s * 2.0 ** -10)
                         + 2 * NORM_REL * y64.abs()).all())
            if t[2] is not None:
                assert _near(t[3][2], h64, 2.0 ** -8 + 2.0 ** -24, torch.bfloat16)
        elif kind == "norm":
            y64, h64 = _norm64(t[0], t[1], t[2], 1e-6)
            assert _near(t[3][0], y64, 2.0 ** -8 + NORM_REL, torch.bfloat16)
            assert _near(t[3][1], h64, 2.0 ** -8 + 2.0 ** -24, torch.bfloat16)
        elif kind == "mx":
            assert _product_ok(t[2], _mx_values(*t[0]), _fp4_values(*t[1]))
        elif kind == "w4":
            assert _product_ok(t[2], t[0].double(), _fp4_values(*t[1]))
        else:
            assert _same_tokens(t[2], t[0], t[1], temperature=0.9, top_k=40, top_p=0.95)


@gpu
def test_decode_step_captured_and_on_two_streams():
    net = _Decoder(512, 1088, 5003, torch.bfloat16, 200)
    x, u = _randn((6, 512), 240, torch.bfloat16), _uniform(6, 241)
    net.step(x, u)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        token, logits = net.step(x, u)
    for i in range(4):
        x.copy_(_randn((6, 512), 250 + i, torch.bfloat16))
        u.copy_(_uniform(6, 260 + i))
        g.replay()
        want = net.step(x, u)
        torch.cuda.synchronize()
        assert torch.equal(token, want[0]) and torch.equal(logits, want[1])
    streams = [torch.cuda.Stream() for _ in range(2)]
    xs = [_randn((6, 512), 270 + i, torch.bfloat16) for i in range(2)]
    want = [net.step(v, u) for v in xs]
    torch.cuda.synchronize()
    got = [[], []]
    for _ in range(5):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                got[i].append(net.step(xs[i], u))
    torch.cuda.synchronize()
    for i in range(2):
        assert all(torch.equal(t, want[i][0]) and torch.equal(v, want[i][1]) for t, v in got[i])


# As SAMPLE_NEAR for 2^19 + 1 logits, whose weights are held in steps of 2^-42
LONG_NEAR = 2 * (2.0 ** 19.1 * 2.0 ** -43 + 2.0 ** -44)


@gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("v", [524288, 524289])
def test_sample_the_longest_16_bit_rows(dtype, v):
    # up to 2^19 by the counts of values, above as f32
    x = _randn((2, v), 83, dtype, 2.0)
    x[0, v - 1] = 40.0
    for st in (dict(top_k=20), dict(temperature=0.0), dict(top_p=0.5)):
        u = _uniform(2, 84)
        got = ops.sample(x, u, **st).cpu()
        want, near = _sample64(x, u, **st)
        far = near > LONG_NEAR
        assert torch.equal(got[far], want[far]) and int(got[0]) == v - 1


@gpu
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("mask", [-torch.inf, "lowest", -1e4, 0.0, -0.0, torch.nan])
@pytest.mark.parametrize("settings", [
    {}, dict(top_k=50), dict(top_k=120000), dict(top_p=0.9), dict(min_p=0.05),
    dict(top_k=40, top_p=0.5, temperature=0.7), dict(temperature=0.0)])
def test_sample_rows_that_are_mostly_masked(dtype, mask, settings):
    v = 131075
    x = _randn((6, v), 85, dtype, 2.0)
    if mask == 0.0:
        x = x.abs()  # the masked are the lowest
    m = torch.finfo(dtype).min if mask == "lowest" else mask
    gen = torch.Generator(device="cuda").manual_seed(86)
    there = torch.rand((6, v), generator=gen, device="cuda")
    x[0] = torch.where(there[0] < 0.9, m, x[0])
    x[1] = torch.where(there[1] < 0.5, m, x[1])
    x[2] = torch.where(there[2] < 0.9999, m, x[2])
    x[3] = m  # every one
    x[4, 17:] = m
    x[5] = torch.where(there[5] < 0.6, m, -m if mask == 0.0 else x[5])
    u = _uniform(6, 87)
    _same_tokens(ops.sample(x, u, **settings), x, u, **settings)


@gpu
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("v", [1, 7, 9, 8191, 32773, 65543, 140009])
def test_sample_greedy_takes_the_first_of_the_highest(dtype, v):
    # rows that begin at every offset from a 16-byte boundary
    buf = _randn((9, v + 9), 88, dtype)
    x = torch.as_strided(buf, (8, v), (v + 10, 1), 1)
    top = x.float().max().item() * 2 + 1
    for i in range(8):
        for at in ((i * 131) % v, v // 2, v - 1, (i * 7919 + 5) % v):
            x[i, at] = top
    x[6] = 0.0
    x[6, 3::5] = -0.0
    x[7] = -0.0
    if v > 9:
        x[7, 9:] = 0.0
    want = [(r == r.max()).nonzero()[0].item() for r in x.cpu().float()]
    assert ops.sample(x, _uniform(8, 89), temperature=0.0).tolist() == want


@gpu
@pytest.mark.parametrize("act", ["bf16", "fp16", "mx"])
@pytest.mark.parametrize("m,n,k", [
    (2, 4200, 1088), (5, 4099, 192), (9, 4200, 320), (16, 8300, 448), (20, 4200, 320),
    (20, 8300, 2112), (32, 16501, 576), (33, 8300, 320), (40, 4200, 640), (64, 16333, 1088),
    (64, 16500, 448), (61, 33001, 64), (130, 4200, 320)])
def test_gemv_4bit_every_tile(m, n, k, act):
    # widths at which each tile of the rule is taken, by four and eight waves
    w4, sw = _weights(n, k, 90)
    w64 = _fp4_values(w4, sw)
    if act == "mx":
        q, sq = _mx_acts(m, k, 91)
        got, x64 = ops.gemv_mx_w4(q, sq, w4, sw), _mx_values(q, sq)
    else:
        x = _randn((m, k), 91, torch.bfloat16 if act == "bf16" else torch.float16)
        got, x64 = ops.gemv_w4(x, w4, sw), x.double()
    assert _product_ok(got, x64, w64)


@gpu
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("residual", [False, True])
@pytest.mark.parametrize("rows,k", [(777, 5003), (1030, 4096), (600, 5120), (600, 7171),
                                    (4200, 1003), (2600, 5122), (513, 8192), (9, 5004)])
def test_rmsnorm_more_rows_than_fit_at_once(rows, k, dtype, residual):
    # two steps a thread, and ragged ends of every length
    test_rmsnorm(rows, k, dtype, residual)
    test_rmsnorm(5, k + 1, dtype, residual)


@gpu
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("residual", [False, True])
@pytest.mark.parametrize("rows,k", [(1030, 4096), (600, 5120), (600, 7232), (4200, 1024)])
def test_rmsnorm_mx_more_rows_than_fit_at_once(rows, k, dtype, residual):
    test_rmsnorm_mx(rows, k, dtype, residual)


@gpu
@pytest.mark.parametrize("m", [1, 7, 64, 200, 256])
@pytest.mark.parametrize("bias", [False, True])
def test_linear_w4_of_any_batch(m, bias):
    from lambdipy_amd.shims.lpx_torch import LinearW4

    w, b = _randn((512, 384), 95, scale=0.05), _randn((512,), 96) if bias else None
    lin, x = LinearW4(w, b), _randn((m, 384), 97)
    got = lin(x)
    qa, sa = ops.quantize_mx(x)
    if m % 256:  # whole tiles go through the scaled MFMA, which sums less exactly
        assert _product_ok(got if b is None else lin.__class__(w)(x), _mx_values(qa, sa),
                           _fp4_values(lin.wq4, lin.wsc4))
        y = ops.gemv_mx_w4(qa, sa, lin.wq4, lin.wsc4)
    else:
        y = ops.gemm_mx_w4(qa, sa, lin.wq4, lin.wsc4)
    assert got.dtype == torch.float32
    assert torch.equal(got, y if b is None else y + b)


@gpu
@pytest.mark.parametrize("act", ["bf16", "fp16", "mx"])
@pytest.mark.parametrize("m,n,k", [(1, 1000, 8192), (1, 15, 2112), (3, 600, 64), (16, 2000, 4160),
                                   (9, 600, 8192), (30, 500, 6144), (64, 65, 1088)])
def test_gemv_4bit_few_tiles(m, n, k, act):
    # sixteen ways along k
    test_gemv_4bit_every_tile(m, n, k, act)
