"""The decode-step operators at the ends of what they take."""

import pytest
import torch
import torch.autograd.forward_ad as fwAD

from lambdipy_amd import ops
from tests.test_decode_ops_gpu import (DEV, TYPES, _fp4_values, _gen, _mx_values, _randn,
                                       _sample64, _uniform, _weights, built, gpu)

INF, NAN = float("inf"), float("nan")


# ---- residual + RMS norm -----------------------------------------------------

@gpu
@pytest.mark.parametrize("rows,k", [(1, 64), (5, 4096)])
def test_rmsnorm_mx_results_have_memory_of_their_own(rows, k):
    # keeping or saving one of them does not keep or save the others
    x = _randn((rows, k), 290, torch.bfloat16)
    out = ops.rmsnorm_mx(x, _randn((k,), 291), residual=x)
    assert [t.untyped_storage().nbytes() for t in out] == [t.nbytes for t in out]
    assert len({t.untyped_storage().data_ptr() for t in out}) == 3
    assert all(t.storage_offset() == 0 and t.is_contiguous() for t in out)


@built
def test_a_tangent_is_refused_and_not_lost():
    x, w = torch.zeros(2, 64), torch.ones(64)
    w4, sw = torch.zeros(8, 32, dtype=torch.uint8), torch.zeros(1, 8, 4, dtype=torch.uint8)

    def refused(why, *calls):
        for call in calls:
            with pytest.raises(RuntimeError, match=why):
                call()

    with fwAD.dual_level(), torch.no_grad():
        dx, dw = fwAD.make_dual(x, x), fwAD.make_dual(w, w)
        db = fwAD.make_dual(x.bfloat16(), x.bfloat16())
        refused("forward-mode", lambda: ops.gemv_w4(db, w4, sw))
        for op in (ops.rmsnorm, ops.rmsnorm_mx):
            refused("forward-mode", lambda: op(dx, w), lambda: op(x, dw),
                    lambda: op(x, w, residual=dx))
            # what carries none, or where none is asked for, goes on to the device
            refused("on the ROCm device", lambda: op(fwAD.unpack_dual(dx).primal, w),
                    lambda: op(x, w))
            with fwAD._set_fwd_grad_enabled(False):
                refused("on the ROCm device", lambda: op(dx, w))
    refused("forward-mode", lambda: torch.func.jvp(lambda v: ops.rmsnorm(v, w), (x,), (x,)))


# ---- 4-bit weights: scales at their ends -------------------------------------

@gpu
@pytest.mark.parametrize("act", ["bf16", "fp16", "mx"])
@pytest.mark.parametrize("byte", [0, 1, 2, 3, 4, 127, 250, 251, 252])
def test_gemv_4bit_weights_are_exact_at_scale(act, byte):
    # one-hot rows give back the dequantised weights, and with x shrunk or
    # grown they give the same weights at the other end of the exponents
    n, k = 40, 64
    w4, sw = _weights(n, k, 330)
    sw.fill_(byte)
    want = _fp4_values(w4, sw).t()
    eye = torch.eye(k, device=DEV)
    if act == "mx":
        got = ops.gemv_mx_w4(*ops.quantize_mx(eye), w4, sw)
    else:
        got = ops.gemv_w4(eye.to(torch.bfloat16 if act == "bf16" else torch.float16), w4, sw)
    assert torch.equal(got.double(), want)
    if act == "bf16":
        s = 2.0 ** min(max(127 - byte, -120), 120)
        assert torch.equal(ops.gemv_w4((eye * s).bfloat16(), w4, sw).double(), want * s)


@gpu
@pytest.mark.parametrize("byte", [3, 4, 9, 10, 127, 245, 246])
def test_gemv_4bit_activations_are_exact_at_scale(byte):
    # every finite e4m3 value at that scale, by a weight that brings it back
    v = torch.tensor([i for i in range(256) if i & 127 != 127], dtype=torch.uint8, device=DEV)
    q = torch.zeros(len(v), 64, dtype=torch.uint8, device=DEV)
    q[:, 0] = v
    sq = torch.full((1, len(v), 4), byte, dtype=torch.uint8, device=DEV)
    w4 = torch.zeros(3, 32, dtype=torch.uint8, device=DEV)
    w4[:, 0] = 2  # 1.0
    for other in (127, 254 - byte):
        sw = torch.full((1, 3, 4), other, dtype=torch.uint8, device=DEV)
        want = _mx_values(q, sq)[:, :1] * 2.0 ** (other - 127)
        assert torch.equal(ops.gemv_mx_w4(q, sq, w4, sw).double(), want.expand(-1, 3))


@gpu
@pytest.mark.parametrize("act", ["bf16", "fp16", "mx"])
def test_gemv_4bit_a_scale_of_255_is_nan(act):
    n, k = 40, 320
    w4, sw = _weights(n, k, 331)
    x = _randn((5, k), 332)

    def product(sw, bad_row=None):
        if act != "mx":
            return ops.gemv_w4(x.to(torch.bfloat16 if act == "bf16" else torch.float16), w4, sw)
        q, sq = ops.quantize_mx(x)
        if bad_row is not None:
            sq[2, bad_row, 1] = 255
        return ops.gemv_mx_w4(q, sq, w4, sw)

    want = product(sw)
    bad = sw.clone()
    bad[1, 7, 2] = 255
    got = product(bad)
    assert bool(got[:, 7].isnan().all())
    keep = [i for i in range(n) if i != 7]
    assert torch.equal(got[:, keep], want[:, keep])
    if act == "mx":
        got = product(sw, bad_row=3)
        assert bool(got[3].isnan().all())
        assert torch.equal(got[[0, 1, 2, 4]], want[[0, 1, 2, 4]])


# ---- more rows than one launch has threads for -------------------------------
# A grid holds fewer than 2^32 threads.

@gpu
@pytest.mark.parametrize("dtype,k,rows", [
    (torch.float16, 1, 2 ** 29 + 5),     # eight threads a row
    (torch.bfloat16, 520, 2 ** 25 + 3)])  # 128
def test_rmsnorm_past_a_grid(dtype, k, rows):
    some = _randn((7, k), 320, dtype)
    w = _randn((k,), 321, dtype)
    want = ops.rmsnorm(some, w)
    if k == 1:
        y = ops.rmsnorm(some.repeat(rows // 7 + 1, 1)[:rows], w)
        whole = rows // 7 * 7
        assert bool((y[:whole].view(-1, 7) == want.view(1, 7)).all())
        assert torch.equal(y[whole:], want[:rows - whole])
    else:  # one row for all, so that only the result takes memory
        y = ops.rmsnorm(some[:1].expand(rows, k), w)
        for at in range(0, rows, 2 ** 22):
            assert bool((y[at:at + 2 ** 22] == want[:1]).all())


@gpu
def test_rmsnorm_mx_past_a_grid():
    k, rows = 576, 2 ** 25 + 3
    x, w = _randn((1, k), 322, torch.bfloat16), _randn((k,), 323)
    q1, sc1 = ops.rmsnorm_mx(x, w)
    q, sc = ops.rmsnorm_mx(x.expand(rows, k), w)
    for at in range(0, rows, 2 ** 22):
        assert bool((q[at:at + 2 ** 22] == q1).all())
        assert bool((sc[:, at:at + 2 ** 22] == sc1).all())


@gpu
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("of_each_row", [False, True])
def test_sample_past_a_grid(dtype, of_each_row):
    rows = 2 ** 22 + 5  # 1024 threads each
    w = torch.tensor([0.125, 0.5, 0.0625, 0.3125], dtype=torch.float64)
    logits = w.log().to(dtype).to(DEV).expand(rows, 4)
    u = _uniform(rows, 324)
    settings = dict(temperature=0.0)
    want = torch.ones(rows, dtype=torch.int64)
    if of_each_row:
        settings = dict(temperature=torch.ones(rows, device=DEV),
                        top_k=torch.arange(rows, dtype=torch.int32, device=DEV) % 4 + 1)
        # in falling order: 1, 3, 0, 2
        c = torch.exp(logits[0].double().cpu()[[1, 3, 0, 2]]).cumsum(0)
        draw = u.double().cpu() * c[torch.arange(rows) % 4]
        want = torch.tensor([1, 3, 0, 2])[(c.unsqueeze(0) <= draw.unsqueeze(1)).sum(1)]
        sure = ((c.unsqueeze(0) - draw.unsqueeze(1)).abs() > 1e-12).all(dim=1)
    got = ops.sample(logits, u, **settings).cpu()
    differ = got != want
    assert not bool((differ & sure if of_each_row else differ).any())


@built
def test_gemv_4bit_refuses_more_weights_than_a_grid_has_threads_for():
    n = 2 ** 28 - 63
    w4 = torch.empty(n, 32, dtype=torch.uint8, device="meta")
    sw = torch.empty(1, n, 4, dtype=torch.uint8, device="meta")
    with pytest.raises(RuntimeError, match="too large"):
        ops.gemv_w4(torch.zeros(1, 64, dtype=torch.bfloat16), w4, sw)
    with pytest.raises(RuntimeError, match="too large"):
        ops.gemv_mx_w4(torch.zeros(1, 64, dtype=torch.uint8),
                       torch.zeros(1, 1, 4, dtype=torch.uint8), w4, sw)

@built
def test_sample_refuses_a_part_of_a_logit():
    # top_k counts logits: 2.5 of them was taken as 2, 0.5 as all
    x, u = torch.zeros(3, 10), torch.zeros(3)
    for k in (2.5, 0.5, 1e9 + 0.25):
        with pytest.raises(RuntimeError, match="top_k must be a whole number"):
            ops.sample(x, u, top_k=k)
    for k in (0, 2, 2.0, True, 10 ** 12):
        with pytest.raises(RuntimeError, match="on the ROCm device"):
            ops.sample(x, u, top_k=k)


# ---- sampling: NaN beside infinities ----------------------------------------

# how a row is sampled: f32 in one workgroup or as chunks; 16 bits by the count
# of each value, or as f32 because one value is there more than 65535 times
SAMPLE_FORMS = [("whole", torch.float32, 3001), ("chunks", torch.float32, 50001),
                ("many chunks", torch.float32, 400003),
                ("bf16", torch.bfloat16, 30001), ("fp16", torch.float16, 30001),
                ("bf16 kept whole", torch.bfloat16, 140001),
                ("fp16 kept whole", torch.float16, 140001)]


def _finite_row(dtype, v, seed):
    x = _randn((v,), seed, dtype)
    if dtype != torch.float32 and v > 65536:
        x[torch.arange(70000) * 2] = 1.0
        x[1::2] = x[1::2].clamp(-4, -0.5)
    return x


def _mids(n):
    """One u in the middle of each of n equal shares."""
    return ((torch.arange(n) + 0.5) / n).to(DEV)


def _every_third(v, n, start):
    return [start + i * (v // (3 * n)) for i in range(n)]


@gpu
@pytest.mark.parametrize("form,dtype,v", SAMPLE_FORMS)
@pytest.mark.parametrize("infs,nans", [(2, 1), (3, 40), (100, 300)])
def test_sample_infinities_share_a_row_beside_nan(form, dtype, v, infs, nans):
    row = _finite_row(dtype, v, 300)
    at_inf, at_nan = _every_third(v, infs, 7), _every_third(v, nans, v // 2)
    row[at_nan] = NAN
    row[at_inf] = INF
    for settings, n in ((dict(), infs), (dict(temperature=0.1), infs),
                        (dict(top_k=2), 2), (dict(top_k=infs + 1), infs),
                        (dict(top_k=infs + nans + 5), infs),
                        (dict(top_p=(infs - 0.5) / infs), infs),
                        (dict(top_p=1.5 / infs), 2), (dict(min_p=0.5), infs),
                        (dict(top_k=infs + nans, top_p=0.999, min_p=0.1), infs)):
        u = _mids(n)
        got = ops.sample(row.expand(n, v), u, **settings)
        assert got.tolist() == at_inf[:n], settings


@gpu
@pytest.mark.parametrize("form,dtype,v", SAMPLE_FORMS)
def test_sample_at_endless_temperatures(form, dtype, v):
    # all that a token can be drawn from is alike; with +inf that alone
    row = _finite_row(dtype, v, 301)
    row[_every_third(v, 50, 11)] = NAN
    row[_every_third(v, 30, v // 2)] = -INF
    order = torch.sort(torch.where(row.isnan(), -INF, row.float()).cpu(), descending=True,
                       stable=True).indices
    n = v - 80
    u = torch.tensor([0.25 / n, 0.3, 0.77, 1 - 0.25 / n], dtype=torch.float64, device=DEV)
    want = order[(u.cpu() * n).long()].tolist()
    top = row.clone()
    top[3], top[v - 2] = INF, INF
    for t in (INF, 1e300):
        t = torch.full((4,), t, dtype=torch.float64, device=DEV)
        assert ops.sample(row.expand(4, v), u, temperature=t).tolist() == want
        assert ops.sample(top.expand(4, v), u, temperature=t).tolist() == [3, 3, v - 2, v - 2]
        assert ops.sample(top.expand(4, v), u, temperature=t, top_k=2,
                          top_p=0.9).tolist() == [3, 3, v - 2, v - 2]


@gpu
@pytest.mark.parametrize("form,dtype,v", SAMPLE_FORMS)
@pytest.mark.parametrize("t", [1e-10, 1e-30, 5e-324])
def test_sample_near_zero_temperature_beside_nan(form, dtype, v, t):
    row = _finite_row(dtype, v, 302)
    row[_every_third(v, 70, 5)] = NAN
    top = _every_third(v, 5, v // 2)
    row[top] = 60.0
    for settings in (dict(), dict(top_k=9), dict(top_p=0.999), dict(min_p=0.5)):
        got = ops.sample(row.expand(5, v), _mids(5), temperature=t, **settings)
        assert got.tolist() == top, settings


# ---- sampling: rows that are mostly masked -----------------------------------

# A weight is held in steps of 2^-45 and off by half of one and by 2^-44 of
# itself, so a running weight over V logits (in all 1 or more) by less than
# V * 2^-46 + 2^-44 of the row's; a border that is nearer than twice that may
# be decided either way.
def _near_of(v):
    return 2 * (v * 2.0 ** -46 + 2.0 ** -44)


def _masked_rows(dtype, mask, v, seed):
    """Rows of which a part, nearly all or all is at one value."""
    x = _randn((6, v), seed, dtype, 2.0)
    if mask == 0.0:
        x = x.abs()  # the masked are the lowest
    m = torch.finfo(dtype).min if mask == "lowest" else mask
    there = torch.rand((6, v), generator=_gen(seed + 1)).to(DEV)
    x[0] = torch.where(there[0] < 0.9, m, x[0])
    x[1] = torch.where(there[1] < 0.5, m, x[1])
    x[2] = torch.where(there[2] < 0.9999, m, x[2])
    x[3] = m
    x[4, 17:] = m
    x[5] = torch.where(there[5] < 0.6, m, -m if mask == 0.0 else x[5])
    return x


@gpu
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("mask", [-INF, "lowest", -1e4, 0.0, -0.0, NAN])
@pytest.mark.parametrize("settings", [
    {}, dict(top_k=50), dict(top_k=120000), dict(top_p=0.9), dict(min_p=0.05),
    dict(top_k=40, top_p=0.5, temperature=0.7), dict(temperature=0.0)])
@pytest.mark.parametrize("v", [5003, 131075])
def test_sample_tokens_of_rows_that_are_mostly_masked(dtype, mask, settings, v):
    x = _masked_rows(dtype, mask, v, 310)
    u = _uniform(6, 312)
    got = ops.sample(x, u, **settings).cpu()
    want, near = _sample64(x, u, **settings)
    # Where all that can be kept is equal, every weight is 1 on both sides, its
    # sums are whole numbers, and the borders are the same products rounded the
    # same (times 2^45): nothing is near.
    k = settings.get("top_k", 0) or v
    top = x.float().nan_to_num(nan=-INF, posinf=INF, neginf=-INF).topk(min(k, v), dim=1).values
    sure = (near > _near_of(v)) | (top == top[:, :1]).all(dim=1).cpu()
    assert int(sure.sum()) >= 5  # one row may lie at a border by chance
    assert got[sure].tolist() == want[sure].tolist()
