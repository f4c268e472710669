"""GPU tests of dropout, the residual norm, the token mix and the tail of the time
mix against plain implementations in 64 bits.

Tolerances.  u(t) = finfo(t).eps / 2 bounds the relative error of one rounding to
type t, U32 = 2^-24 that of one in fp32.  A sum of n terms taken in fp32 in any order
is off by at most n U32 sum|terms|; each term adds a few roundings of its own (counted
as up to 16).  A result is off by the error of its sums carried through the formula,
plus its one rounding u(t) |result| at the store.
"""
from __future__ import annotations

import numpy as np
import pytest
import torch

from philox_oracle import kept, threshold
from test_block_gpu import DTYPES, U32, check, rnd, top_of_group, u, values64

pytestmark = pytest.mark.gpu

PARAMS = [torch.float32, torch.bfloat16, torch.float16]


def mask(shape, p, seed, offset=0):
    n = int(np.prod(shape))
    return torch.from_numpy(kept(n, p, seed, offset)).view(shape).cuda()


def factor(p, scale=1.0):
    """What a kept value is multiplied with."""
    t = threshold(p)
    return 0.0 if t == 65536 else scale * 65536 / (65536 - t)


def drop64(x, p, seed, offset=0, scale=1.0):
    """scale dropout(x) in 64 bits; what is dropped is 0 whatever it was."""
    x = x.double()
    return torch.where(mask(x.shape, p, seed, offset), x * factor(p, scale), 0.0) if threshold(p) else x * scale


# -------------------------------------------------------------------- dropout

@pytest.mark.parametrize("dt", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("shape", [(1,), (7,), (8,), (3, 33), (257, 96), (2, 5, 1003), (65, 2048)])
def test_dropout(cuda, dt, shape):
    """The factor rounds to fp32, the product to fp32 and to the type."""
    from swiftrwkv_b200 import block as B
    t = DTYPES[dt]
    x = rnd(shape, 200, t)
    for p, seed, offset in ((0.1, 0, 0), (0.5, 2**64 - 1, 3), (0.37, 12345678901234567890, 2**64 - 1), (0.0, 4, 0),
                            (1e-6, 5, 0), (1.0, 6, 0), (0.999999, 7, 0), (2**-16, 8, 1)):
        y = B.dropoutForward(x, p, seed, offset)
        want = drop64(x, p, seed, offset)
        assert torch.equal(y == 0, want == 0)
        check(y, want, want.abs() * (u(t) + 3 * U32), (p, seed))
        if p == 0.0:
            assert torch.equal(y, x)
        state = torch.tensor([seed - 2**64 if seed >= 2**63 else seed, 5], device="cuda")
        assert torch.equal(B.dropoutForward(x, p, state, (offset - 5) % 2**64), y)


def test_dropout_draws_anew_by_seed_offset_and_place(cuda):
    """Means within five standard deviations; two draws agree where they have to by chance."""
    from swiftrwkv_b200 import block as B
    x = torch.ones(1 << 20, device="cuda")
    for p in (0.1, 0.5, 0.9):
        draws = [B.dropoutForward(x, p, s, o) != 0 for s, o in ((1, 0), (2, 0), (1, 1), (1 << 32, 0), (1, 1 << 32))]
        q = 1 - threshold(p) / 65536
        sd = (q * (1 - q) / x.numel()) ** 0.5
        for k, a in enumerate(draws):
            assert abs(float(a.double().mean()) - q) < 5 * sd
            assert abs(float(a[::2].double().mean()) - float(a[1::2].double().mean())) < 10 * sd
            for b in draws[:k]:
                both = q * q
                assert abs(float((a & b).double().mean()) - both) < 5 * (both * (1 - both) / x.numel()) ** 0.5


def test_dropout_of_infinities_nan_views_and_its_gradient(cuda):
    from swiftrwkv_b200 import block as B
    x = torch.full((64, 64), float("nan"), device="cuda")
    x[::2] = float("inf")
    y = B.dropoutForward(x, 0.5, 3)
    m = mask(x.shape, 0.5, 3)
    assert (y[~m] == 0).all() and not torch.isfinite(y[m]).any()
    assert not B.dropoutForward(x, 1.0, 3).any()
    base = rnd((40, 50), 201, torch.bfloat16)
    assert torch.equal(B.dropoutForward(base.t(), 0.3, 9), B.dropoutForward(base.t().contiguous(), 0.3, 9))
    flat = rnd((1001,), 202, torch.float16)
    assert torch.equal(B.dropoutForward(flat[1:], 0.3, 9), B.dropoutForward(flat[1:].clone(), 0.3, 9))
    assert B.dropoutForward(base[:0], 0.3, 9).shape == (0, 50)
    for seed in (11, torch.tensor([11, 4], device="cuda")):
        x = rnd((33, 40), 203).requires_grad_(True)
        dy = rnd((33, 40), 204)
        y = B.dropout(x, 0.25, seed, 2)
        y.backward(dy.t().contiguous().t())
        o = 2 if isinstance(seed, int) else 6
        assert torch.equal(y.detach(), B.dropoutForward(x.detach(), 0.25, 11, o))
        assert torch.equal(x.grad, B.dropoutForward(dy, 0.25, 11, o))
    seed = torch.tensor([11, 4], device="cuda")
    y = B.dropout(x, 0.25, seed)
    seed += 1
    with pytest.raises(RuntimeError, match="inplace"):
        y.sum().backward()


def test_dropout_may_write_over_its_input(cuda):
    from swiftrwkv_b200 import _lib, block as B
    x = rnd((12345,), 205, torch.bfloat16)
    want, buf = B.dropoutForward(x, 0.2, 1), x.clone()
    _lib.call("rwkv_dropout", _lib.BF16, buf.data_ptr(), 0.2, 1, 0, None, buf.data_ptr(), buf.numel(),
              torch.cuda.current_stream().cuda_stream)
    assert torch.equal(buf, want)


def test_dropout_past_32_bits(cuda):
    """Places past 2^32: the block's number and the offsets of memory."""
    from swiftrwkv_b200 import block as B
    rows, D = (1 << 17) + 3, 1 << 15
    x = torch.ones(rows, D, device="cuda", dtype=torch.float16)
    y = B.dropoutForward(x, 0.5, 77, 1)
    for row in (0, 1 << 16, (1 << 17) - 1, 1 << 17, rows - 1):
        want = torch.from_numpy(kept(D, 0.5, 77, 1, first=row * D)).cuda()
        assert torch.equal(y[row] == 2, want) and torch.equal(y[row] == 0, ~want)


def test_dropout_of_flat_tensors_past_31_bits(cuda):
    """Dropout is by place, whatever the shape: a flat tensor of more than 2^31 - 1 elements is as
    good as rows; more than 2^40 are refused (nothing is copied)."""
    from swiftrwkv_b200 import block as B
    x = torch.ones((1 << 31) + 24, device="cuda", dtype=torch.float16)
    y = B.dropoutForward(x, 0.5, 78, 1)
    assert torch.equal(y, B.dropoutForward(x.view(8, -1), 0.5, 78, 1).view(-1))
    assert torch.equal(B.dropout(x[:1], 0.5, 78, 1), y[:1])
    with pytest.raises(ValueError, match="2\\^40"):
        B.dropoutForward(x[:1].expand((1 << 40) + 1), 0.5, 78)


# -------------------------------------------------------------- residual norm

# on both sides of each length at which the kernels change their threads
RNORM_SIZES = [(1, 8), (3, 64), (9, 72), (5, 136), (6, 256), (5, 264), (5, 512), (5, 520), (1, 2048), (33, 768), (4, 776),
               (3, 1024), (2, 1032), (4, 1536), (3, 1544), (2, 2056), (7, 2560), (3, 2568), (2, 4104), (5, 6144), (1003, 128),
               (700, 40)]


def rnorm64(x, branch, w, b, eps, p, seed, scale):
    """Sum, norm, statistics in 64 bits, and the bounds of their errors before the store."""
    q = drop64(branch, p, seed, scale=scale)
    s = x.double() + q
    es = 3 * U32 * q.abs() + U32 * s.abs()
    mean = s.mean(-1, keepdim=True)
    dev = s - mean
    var = (dev ** 2).mean(-1, keepdim=True)
    rstd = 1 / torch.sqrt(var + eps)
    y = dev * rstd * w.double() + b.double()
    n = (x.shape[-1] + 16) * U32
    em = n * s.abs().mean(-1, keepdim=True) + es.mean(-1, keepdim=True)
    ed = em + es + U32 * dev.abs()
    evar = (2 * dev.abs() * ed + ed ** 2).mean(-1, keepdim=True) + n * (dev ** 2).mean(-1, keepdim=True)
    er = 0.5 * evar * rstd ** 2 * 1.01 + 8 * U32                        # relative
    ey = w.double().abs() * rstd * (ed + dev.abs() * (er + 4 * U32)) + 2 * U32 * (y.abs() + b.double().abs())
    return (s, es), (y, ey * 1.01), (mean[..., 0], em[..., 0]), (rstd[..., 0], (rstd * er)[..., 0])


@pytest.mark.parametrize("dt", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("rows,D", RNORM_SIZES)
def test_residual_norm_forward(cuda, dt, rows, D):
    from swiftrwkv_b200 import block as B
    t = DTYPES[dt]
    x, branch = (rnd((rows, D), 210) * 2 + 0.5).to(t), rnd((rows, D), 211, t)
    w, b = rnd((D,), 212) * 0.2 + 1, rnd((D,), 213) * 0.2
    for p, scale in ((0.0, 1.0), (0.3, 1.0), (0.0, 0.7), (0.15, -0.3), (1.0, 2.0)):
        s, y, mean, rstd, ck = B.residualNormForward(x, branch, w, b, 1e-5, scale, p, 21, checkpoint=True)
        (s64, es), (y64, ey), (m64, em), (r64, er) = rnorm64(x, branch, w, b, 1e-5, p, 21, scale)
        check(s, s64, es + u(t) * (s64.abs() + es), "s")
        check(y, y64, ey + u(t) * (y64.abs() + ey), "y")
        check(mean, m64, em + U32 * m64.abs(), "mean")
        check(rstd, r64, er + U32 * r64, "rstd")
        # the checkpoint is that of the fp32 sum, es off
        top = top_of_group(s64)
        check(B.checkpoint8Values(ck, dtype=torch.float32), s64, top * (1 + 4 * U32) / 127.5 + es + U32 * s64.abs(), "ck")
        again = B.residualNormForward(x, branch, w, b, 1e-5, scale, p, 21)
        assert again[4] is None and all(torch.equal(a, c) for a, c in zip(again, (s, y, mean, rstd)))


@pytest.mark.parametrize("dt", ["f32", "bf16", "f16"])
def test_residual_norm_of_whole_numbers(cuda, dt):
    """Sums that are exact in every type: s and the checkpoint are their definitions."""
    from swiftrwkv_b200 import block as B
    t = DTYPES[dt]
    g = torch.Generator(device="cuda").manual_seed(1)
    for D in (40, 2048):
        x, branch = (torch.randint(-60, 61, (9, D), generator=g, device="cuda").to(t) for _ in range(2))
        w, b = torch.ones(D, device="cuda"), torch.zeros(D, device="cuda")
        s, _, _, _, ck = B.residualNormForward(x, branch, w, b, p=0.5, seed=3, checkpoint=True)
        want = x.double() + drop64(branch, 0.5, 3)
        assert torch.equal(s.double(), want)
        assert torch.equal(B.checkpoint8Values(ck, dtype=torch.float32).double(), values64(want))


@pytest.mark.parametrize("D", [8, 40, 64, 96, 128, 256, 512, 768, 776, 1024, 1536, 2048, 2560, 4096, 6144])
def test_residual_norm_far_from_zero(cuda, D):
    """Constant sums give the bias exactly, also at 1000.1 (their mean is exact); a row at
    1000 with spread 1 keeps the accuracy of the fp32 mean, 1000 2^-24 per rounding, 8 of
    them, as the layer norm's; an outlier anywhere costs at most the pivot's cancelling."""
    from swiftrwkv_b200 import block as B
    x = torch.full((6, D), 1000.1, device="cuda")
    x[1] = -3.0e-5
    x[2:4] = 1000.0 + rnd((2, D), 330)
    x[4:] = rnd((2, D), 331)
    x[4, 0], x[5, D - 1] = 1e4, -1e4           # an outlier in the pivot's vector, and at the end
    zero, w, b = torch.zeros_like(x), rnd((D,), 332), rnd((D,), 333)
    s, y, mean, rstd, _ = B.residualNormForward(x, zero, w, b)
    assert torch.equal(s, x) and torch.equal(mean[:2], x[:2, 0]) and torch.equal(y[:2], b.expand(2, D))
    dev = x.double() - x.double().mean(1, keepdim=True)
    r64 = 1 / torch.sqrt((dev ** 2).mean(1, keepdim=True) + 1e-5)
    y64 = dev * r64 * w.double() + b.double()
    tol = 8 * 1000 * U32 * (w.double().abs() * r64 + 1) * (1 + (y64 - b.double()).abs())
    check(y[2:4], y64[2:4], tol[2:4], "far")
    # sums of squares that cancel 32-fold at most (7 bits of 24 with the sums' own n 2^-24)
    n = (D + 16) * U32
    rel = 32 * n + 8 * U32
    tol = (w.double() * dev * r64).abs() * rel + w.double().abs() * r64 * n * x.double().abs().mean(1, keepdim=True) + 4 * U32 * (y64.abs() + b.double().abs())
    check(y[4:], y64[4:], tol[4:], "outlier")


def outlier_rows(D, VE):
    """Rows of spread 1 with values of 1000 and 30: at the start, in the whole first vectors, in the first
    vector of each 32 (as far as they are few), and with them at the end."""
    x = rnd((8, D), 337)
    heads = torch.arange(D, device="cuda") // VE % 32 == 0
    x[0, 0] = 1000.0
    x[1, :4] = 1000.0 + x[1, :4]
    x[2, :8] = 1000.0 + x[2, :8]
    x[3, :8] = -30.0
    x[4] = torch.where(heads, 1000.0 + x[4], x[4])
    x[5, :8] += torch.tensor([1000.0, -700.0, 300.0, 20.0, 1000.0, 5.0, 400.0, -30.0], device="cuda")
    x[6, -8:] = 1000.0
    x[7, 0], x[7, -1] = 1e4, -1e4
    return x


@pytest.mark.parametrize("dt", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("D", [72, 264, 520, 776, 1032, 1280, 1536, 2056, 2560, 4096, 6144])
def test_residual_norm_of_rows_with_outliers(cuda, dt, D):
    """The statistics are those of a sum around the mean, wherever the row's outliers are.  A term
    passes at most 28 additions (64 threads: 20 in its own, 1 for a pair's halves, 5 in the warp, 2
    between warps; 512 threads: 6, 1, 5 and 16): a sum of squares is off by 30 U32 (each square 2 U32 by
    its difference), by at most 4 times that where it is taken from another point than the mean; rstd by
    half of it and 2 roundings in the variance, 2 in the root and the quotient.  The mean: 32 U32 mean|s|."""
    from swiftrwkv_b200 import block as B
    t = DTYPES[dt]
    x = outlier_rows(D, 4 if dt == "f32" else 8).to(t)
    zero, w, b = torch.zeros_like(x), rnd((D,), 338), rnd((D,), 339)
    s, y, mean, rstd, _ = B.residualNormForward(x, zero, w, b)
    assert torch.equal(s, x)
    s64, w64, b64 = x.double(), w.double(), b.double()
    m64 = s64.mean(1, keepdim=True)
    dev = s64 - m64
    r64 = 1 / torch.sqrt((dev ** 2).mean(1, keepdim=True) + 1e-5)
    em = 32 * U32 * s64.abs().mean(1, keepdim=True)
    er = (4 * 32 / 2 + 4) * U32
    check(mean, m64[:, 0], em[:, 0] + U32 * m64[:, 0].abs(), "mean")
    check(rstd, r64[:, 0], er * r64[:, 0], "rstd")
    # where the outliers are at the start and large: no cancelling is left
    check(rstd[[0, 1, 2, 4]], r64[[0, 1, 2, 4], 0], (32 / 2 + 4) * U32 * r64[[0, 1, 2, 4], 0], "rstd of large outliers")
    y64 = dev * r64 * w64 + b64
    tol = w64.abs() * r64 * (em + U32 * dev.abs() + dev.abs() * (er + 4 * U32)) + 2 * U32 * (y64.abs() + b64.abs())
    check(y, y64, tol + u(t) * (y64.abs() + tol), "y")
    for i in range(8):  # a row's results are its own, whatever lies beside it
        alone = B.residualNormForward(x[i], zero[i], w, b, checkpoint=True)
        assert all(torch.equal(a, c[i]) for a, c in zip(alone, (s, y, mean, rstd)))


@pytest.mark.parametrize("D", [776, 1280, 2560, 6144])
def test_residual_norm_of_the_largest_outliers(cuda, D):
    """One value of 2^63: its square is within fp32, the sum of the others' squared distances to
    their vector's mean is not."""
    from swiftrwkv_b200 import block as B
    x = rnd((2, D), 346)
    x[0, 0] = 2.0 ** 63
    one, zero = torch.ones(D, device="cuda"), torch.zeros(D, device="cuda")
    _, y, mean, rstd, _ = B.residualNormForward(x, torch.zeros_like(x), one, zero)
    dev = x.double() - x.double().mean(1, keepdim=True)
    r64 = 1 / torch.sqrt((dev ** 2).mean(1) + 1e-5)
    check(rstd[0], r64[0], 20 * U32 * r64[0], "rstd")
    check(y[0, 0], (dev[0, 0] * r64[0]), 64 * U32 * (dev[0, 0] * r64[0]).abs(), "y")


@pytest.mark.parametrize("D", [64, 256, 512, 768, 1024, 1536, 2048, 2560, 4096, 6144])
def test_residual_norm_mean_near_zero(cuda, D):
    """Means much smaller than their rows' values: each of the D additions rounds by at most U32
    of a partial sum, which for random signs is sqrt(D) at most: in the root mean square over rows
    below sqrt(D) sqrt(D) U32 / D = U32."""
    from swiftrwkv_b200 import block as B
    x = rnd((512, D), 334)
    _, _, mean, _, _ = B.residualNormForward(x, torch.zeros_like(x), torch.ones(D, device="cuda"), torch.zeros(D, device="cuda"))
    off = mean.double() - x.double().mean(1)
    assert float(off.square().mean().sqrt()) < U32


@pytest.mark.parametrize("kept_", [False, True])
@pytest.mark.parametrize("dt", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("D", [8, 40, 72, 136, 264, 520, 776, 2056])
def test_residual_norm_backward_of_huge_constant_rows(cuda, dt, kept_, D):
    """Rows of one value, 2^121 (2^13 in fp16), with a rstd of 2^10 (2^118): their h is 0, while
    mean rstd, which zeros beyond a row's end would give, is beyond fp32.  g rounds
    once, its sum D times, dx a few times more and once at the store."""
    from swiftrwkv_b200 import block as B
    t = DTYPES[dt]
    top, inv, dy_unit, w_unit = (2.0**13, 2.0**118, 2.0**-14, 2.0**-104) if dt == "f16" else (2.0**121, 2.0**10, 2.0**-10, 1.0)
    x, w, dy = torch.full((37, D), top, device="cuda", dtype=t), rnd((D,), 335, scale=w_unit), rnd((37, D), 336, t, dy_unit)
    mean, rstd = torch.full((37,), top, device="cuda"), torch.full((37,), inv, device="cuda")
    s = x
    if kept_:
        assert torch.equal(values64(x), x.double())
        s = B.residualNormForward(x, torch.zeros_like(x), w, torch.zeros_like(w), checkpoint=True)[4]
    for p in (0.0, 0.25):
        dx, dbranch, dw, db = B.residualNormBackward(dy, s, w, mean, rstd, scale=0.5, p=p, seed=9)
        g = dy.double() * w.double()
        want = inv * (g - g.mean(1, keepdim=True))
        tol = inv * (4 * U32 * g.abs() + (D + 16) * U32 * g.abs().mean(1, keepdim=True))
        check(dx, want, tol + u(t) * want.abs(), p)
        check(dbranch, drop64(want, p, 9, scale=0.5), tol + (u(t) + 3 * U32) * want.abs(), p)
        assert not dw.any()
        check(db, dy.double().sum(0), (37 + 16) * U32 * dy.double().abs().sum(0), p)


@pytest.mark.parametrize("kept_", [False, True])
@pytest.mark.parametrize("dt", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("rows,D", RNORM_SIZES)
def test_residual_norm_backward(cuda, dt, kept_, rows, D):
    from swiftrwkv_b200 import block as B
    t = DTYPES[dt]
    s = (rnd((rows, D), 214) * 2 + 0.5).to(t)
    w, b = rnd((D,), 215) * 0.2 + 1, rnd((D,), 216)
    dy, dres = rnd((rows, D), 217, t), rnd((rows, D), 218, t)
    _, mean, rstd, ck = B.layerNormForward(s, w, b, checkpoint=True)
    sv = values64(s) if kept_ else s.double()
    m, r = mean.double()[:, None], rstd.double()[:, None]
    h = (sv - m) * r
    g = dy.double() * w.double()
    along, mg = (g * h).mean(1, keepdim=True), g.mean(1, keepdim=True)
    n = (D + 16) * U32
    hd = 3 * U32 * r * (sv.abs() + m.abs())                           # error of h
    for p, scale, res in ((0.3, 1.0, dres), (0.0, 0.5, None), (0.1, -0.75, dres)):
        dx, dbr, dw, db = B.residualNormBackward(dy, ck if kept_ else s, w, mean, rstd, res, scale, p, 31, 7)
        want = r * (g - mg - h * along) + (0 if res is None else res.double())
        tol = r * (g.abs() * 4 * U32 + n * g.abs().mean(1, keepdim=True) +
                   h.abs() * (n * (g * h).abs().mean(1, keepdim=True) + (g.abs() * hd).mean(1, keepdim=True)) +
                   hd * along.abs()) + 8 * U32 * (r * (g.abs() + mg.abs() + (h * along).abs()) + dres.double().abs())
        tol = tol * 1.01
        check(dx, want, tol + u(t) * (want.abs() + tol), "dx")
        f, m8 = abs(factor(p, scale)), mask(dy.shape, p, 31, 7)
        wantb = drop64(want, p, 31, 7, scale)
        tolb = torch.where(m8, f * tol, 0.0) + 3 * U32 * wantb.abs()
        check(dbr, wantb, tolb + u(t) * (wantb.abs() + tolb), "dbranch")
        assert not dbr[~m8].any()
        k = (rows + 16) * U32
        check(dw, (dy.double() * h).sum(0), k * (dy.double() * h).abs().sum(0) + (dy.double().abs() * hd).sum(0) + 1e-38, "dw")
        check(db, dy.double().sum(0), k * dy.double().abs().sum(0) + 1e-38, "db")
        again = B.residualNormBackward(dy, ck if kept_ else s, w, mean, rstd, res, scale, p, 31, 7)
        assert all(torch.equal(a, c) for a, c in zip(again, (dx, dbr, dw, db)))      # deterministic
        dx2, dbr2, none, _ = B.residualNormBackward(dy, ck if kept_ else s, w, mean, rstd, res, scale, p, 31, 7, params=False)
        assert none is None and torch.equal(dx2, dx) and torch.equal(dbr2, dbr)
    dx, dbr, dw, db = B.residualNormBackward(dy, ck if kept_ else s, w, mean, rstd, dres)
    assert dbr is dx
    for a, c in zip((dx, dw, db), B.layerNormBackward(dy, ck if kept_ else s, w, mean, rstd, dres)):
        assert torch.equal(a, c)


def test_residual_norm_of_more_rows_than_blocks(cuda):
    for D in (40, 128, 256, 768, 776, 2560):
        test_residual_norm_forward(cuda, "bf16", 3001, D)
        test_residual_norm_backward(cuda, "bf16", False, 3001, D)
        test_residual_norm_backward(cuda, "f16", True, 2999, D)
    test_residual_norm_backward(cuda, "f32", True, 2999, 384)


def test_residual_norm_of_16_bit_rows_past_6144(cuda):
    for D in (6152, 8200, 12288):
        test_residual_norm_forward(cuda, "bf16", 5, D)
        test_residual_norm_backward(cuda, "f16", True, 5, D)
        test_residual_norm_backward(cuda, "bf16", False, 301, D)


@pytest.mark.parametrize("dt", ["f32", "bf16"])
@pytest.mark.parametrize("D", [96, 2056, 2560, 6144])
def test_residual_norm_may_write_over_its_inputs(cuda, dt, D):
    """sum over x and y over branch, and the other way round; dx over dy and
    dbranch over dres, and the other way round (rwkv_cuda.h)."""
    from swiftrwkv_b200 import _lib, block as B
    t, rows = DTYPES[dt], 1301
    code, st = B._DT[t], torch.cuda.current_stream().cuda_stream
    x, branch, dy, dres = (rnd((rows, D), 220 + i, t) for i in range(4))
    w, b = rnd((D,), 224) * 0.2 + 1, rnd((D,), 225)
    s, y, mean, rstd, _ = B.residualNormForward(x, branch, w, b, scale=0.5, p=0.2, seed=4)
    dx, dbr, _, _ = B.residualNormBackward(dy, s, w, mean, rstd, dres, 0.5, 0.2, 4)
    for swap in (False, True):
        a, c = x.clone(), branch.clone()
        o1, o2 = (c, a) if swap else (a, c)
        _lib.call("rwkv_residual_norm_forward", code, a.data_ptr(), c.data_ptr(), 0.5, 0.2, 4, 0, None, _lib.F32,
                  w.data_ptr(), b.data_ptr(), 1e-5, o1.data_ptr(), o2.data_ptr(), None, None, None, None, rows, D, st)
        assert torch.equal(o1, s) and torch.equal(o2, y)
        a, c = dy.clone(), dres.clone()
        o1, o2 = (c, a) if swap else (a, c)
        _lib.call("rwkv_residual_norm_backward", code, a.data_ptr(), s.data_ptr(), None, None, _lib.F32, w.data_ptr(),
                  mean.data_ptr(), rstd.data_ptr(), c.data_ptr(), 0.5, 0.2, 4, 0, None, o1.data_ptr(), o2.data_ptr(), None,
                  None, rows, D, None, 0, st)
        assert torch.equal(o1, dx) and torch.equal(o2, dbr)


def test_residual_norm_gradient_matches_differences(cuda):
    """Against central differences of the forward in fp32: 1e-2 of the largest
    gradient at a step of 2^-6, as the layer norm's."""
    from swiftrwkv_b200 import block as B
    x, br, w, b = rnd((4, 24), 226), rnd((4, 24), 227), rnd((24,), 228) * 0.2 + 1, rnd((24,), 229)
    dy, ds = rnd((4, 24), 230), rnd((4, 24), 231)

    def f():
        s, y, _, _, _ = B.residualNormForward(x, br, w, b, scale=0.5, p=0.3, seed=8)
        return (y.double() * dy.double()).sum() + (s.double() * ds.double()).sum()
    s, _, mean, rstd, _ = B.residualNormForward(x, br, w, b, scale=0.5, p=0.3, seed=8)
    grads = B.residualNormBackward(dy, s, w, mean, rstd, ds, 0.5, 0.3, 8)
    for p, g in zip((x, br, w, b), grads):
        flat, gf = p.view(-1), g.reshape(-1)
        for i in range(0, flat.numel(), 5):
            keep = float(flat[i])
            flat[i] = keep + 2.0 ** -6
            up = f()
            flat[i] = keep - 2.0 ** -6
            dn = f()
            flat[i] = keep
            assert abs(float(up - dn) * 2 ** 5 - float(gf[i])) < 1e-2 * float(g.abs().max())


@pytest.mark.parametrize("checkpoint", [False, True])
def test_residual_norm_differentiable(cuda, checkpoint):
    from swiftrwkv_b200 import block as B
    t, state = torch.bfloat16, torch.tensor([5, 6], device="cuda")
    x, br, ds, dy = (rnd((2, 9, 64), 232 + i, t) for i in range(4))
    w, b = rnd((64,), 236, t), rnd((64,), 237, t)
    s, y, mean, rstd, ck = B.residualNormForward(x, br, w, b, 1e-5, 0.5, 0.2, 5, 10, checkpoint)
    want = B.residualNormBackward(dy, ck if checkpoint else s, w, mean, rstd, ds, 0.5, 0.2, 5, 10)
    for seed, offset in ((5, 10), (state, 4)):
        leaves = [v.clone().requires_grad_(True) for v in (x, br, w, b)]
        s2, y2 = B.residualNorm(*leaves, 1e-5, 0.5, 0.2, seed, offset, checkpoint)
        assert torch.equal(s2, s) and torch.equal(y2, y)
        torch.autograd.backward([s2, y2], [ds, dy])
        assert all(torch.equal(v.grad, g) and v.grad.dtype == v.dtype for v, g in zip(leaves, want))
    # only one of the outputs is used; nothing dropped
    x1, b1 = x.clone().requires_grad_(True), br.clone().requires_grad_(True)
    B.residualNorm(x1, b1, w, b)[0].backward(ds)
    assert torch.equal(x1.grad, ds) and torch.equal(b1.grad, ds)
    x1 = x.clone().requires_grad_(True)
    B.residualNorm(x1, br, w, b)[1].backward(dy)
    s1, _, m1, r1, _ = B.residualNormForward(x, br, w, b)
    assert torch.equal(x1.grad, B.layerNormBackward(dy, s1, w, m1, r1)[0])


@pytest.mark.parametrize("checkpoint", [False, True])
@pytest.mark.parametrize("scale,p", [(1.0, 0.0), (0.5, 0.0), (0.5, 0.2)])
def test_residual_norm_whose_norm_is_not_used(cuda, checkpoint, scale, p):
    """Without a gradient of y that of s passes as it is, whatever the row and the weights hold."""
    from swiftrwkv_b200 import block as B
    x, br, ds = (rnd((6, 96), 348 + i) for i in range(3))
    w, b = rnd((96,), 351), rnd((96,), 352)
    x[1, 5], x[3, 7], w[2] = float("inf"), float("nan"), float("inf")
    leaves = [v.clone().requires_grad_(True) for v in (x, br, w, b)]
    B.residualNorm(*leaves, scale=scale, p=p, seed=6, checkpoint=checkpoint)[0].backward(ds)
    want = drop64(ds, p, 6, scale=scale)
    assert torch.equal(leaves[0].grad, ds)
    check(leaves[1].grad, want, 4 * U32 * want.abs(), "dbranch")
    assert not leaves[2].grad.any() and not leaves[3].grad.any()


@pytest.mark.parametrize("dt", ["f32", "bf16"])
@pytest.mark.parametrize("D", [40, 128, 256, 512, 776, 2560, 6144])
def test_residual_norm_seeds_on_the_device(cuda, dt, D):
    """A seed tensor draws what its values draw, in each of the kernels."""
    from swiftrwkv_b200 import block as B
    t = DTYPES[dt]
    x, br, dy, dres = (rnd((37, D), 590 + i, t) for i in range(4))
    w, b = rnd((D,), 594), rnd((D,), 595)
    seed, state = 0xFEDCBA9876543210, torch.tensor([0xFEDCBA9876543210 - 2**64, 2**40], device="cuda")
    for checkpoint in (False, True):
        got = [B.residualNormForward(x, br, w, b, p=0.4, seed=s, offset=o, checkpoint=checkpoint)
               for s, o in ((seed, 2**40 + 3), (state, 3))]
        assert all(torch.equal(a, c) for a, c in zip(got[0][:4], got[1][:4]))
        kept_ = got[0][4] if checkpoint else got[0][0]
        back = [B.residualNormBackward(dy, kept_, w, *got[0][2:4], dres, 0.5, 0.4, s, o) for s, o in ((seed, 2**40 + 3), (state, 3))]
        assert all(torch.equal(a, c) for a, c in zip(*back))
        assert torch.equal(back[0][1] == 0, ~mask(dy.shape, 0.4, seed, 2**40 + 3))


def test_calls_of_two_lengths_on_two_threads(cuda):
    """A kernel's shared-memory limit does not follow the call's length."""
    import threading
    from swiftrwkv_b200 import block as B
    wrong = []

    def work(D, seed):
        s = torch.cuda.Stream()
        with torch.cuda.stream(s):
            x, dy = rnd((64, D), seed, torch.bfloat16), rnd((64, D), seed + 1, torch.bfloat16)
            w, b = torch.ones(D, device="cuda"), torch.zeros(D, device="cuda")
            first = None
            for _ in range(60):
                v, _, mean, rstd, _ = B.residualNormForward(x, dy, w, b, p=0.1, seed=seed)
                got = B.residualNormBackward(dy, v, w, mean, rstd, p=0.1, seed=seed)
                if first is None:
                    first = got
                elif not all(torch.equal(a, c) for a, c in zip(first, got)):
                    wrong.append(D)
        s.synchronize()

    def guarded(*a):
        try:
            work(*a)
        except Exception as e:  # noqa: BLE001
            wrong.append(e)
    threads = [threading.Thread(target=guarded, args=a) for a in ((776, 600), (2560, 602))]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not wrong


def test_residual_norm_empty_rows_views_and_types(cuda):
    from swiftrwkv_b200 import block as B
    w, b = rnd((64,), 240, torch.float16), rnd((64,), 241, torch.float16)
    x = rnd((0, 64), 242, torch.bfloat16)
    s, y, mean, rstd, ck = B.residualNormForward(x, x, w, b, p=0.1, checkpoint=True)
    assert s.shape == y.shape == (0, 64) and mean.shape == rstd.shape == (0,) and ck.codes.shape == (0, 64)
    dx, dbr, dw, db = B.residualNormBackward(x, s, w, mean, rstd, p=0.1)
    assert dx.shape == dbr.shape == (0, 64) and not dw.any() and not db.any()
    base, br = rnd((64, 70), 243), rnd((64 * 33 + 1,), 244)[1:].view(33, 64)     # strided; off a 16-byte boundary
    got = B.residualNormForward(base.t()[:33], br, w.float(), b.float(), p=0.1, seed=2)
    want = B.residualNormForward(base.t()[:33].contiguous(), br.clone(), w.float(), b.float(), p=0.1, seed=2)
    assert all(torch.equal(a, c) for a, c in zip(got[:4], want))
    one = B.residualNormForward(base[:, 0].contiguous(), base[:, 1].contiguous(), w, b)      # [D]
    assert one[0].shape == (64,) and one[2].shape == ()
    for wd in PARAMS:      # weights of every type beside activations of every type
        for xd in DTYPES.values():
            a, c = rnd((5, 64), 245, xd), rnd((5, 64), 246, xd)
            y1 = B.residualNormForward(a, c, w.to(wd), b.to(wd))[1]
            y2 = B.residualNormForward(a, c, w.to(wd).float(), b.to(wd).float())[1]
            assert torch.equal(y1, y2)


def test_residual_norm_of_infinities_and_nan(cuda):
    """They stay in their rows; dropped ones are gone."""
    from swiftrwkv_b200 import block as B
    x, br = rnd((6, 96), 247, torch.bfloat16), rnd((6, 96), 248, torch.bfloat16)
    m = mask(br.shape, 0.5, 12)
    br[~m] = float("nan")
    want = B.residualNormForward(x, torch.where(m, br, 0.0), torch.ones(96, device="cuda"), torch.zeros(96, device="cuda"),
                                 p=0.5, seed=12, checkpoint=True)
    got = B.residualNormForward(x, br, torch.ones(96, device="cuda"), torch.zeros(96, device="cuda"), p=0.5, seed=12,
                                checkpoint=True)
    assert all(torch.equal(a, c) for a, c in zip(got[:4], want[:4])) and torch.equal(got[4].codes, want[4].codes)
    x[3, 7] = float("inf")
    x[4, 40] = float("nan")
    s, y, _, _, ck = B.residualNormForward(x, br, torch.ones(96, device="cuda"), torch.zeros(96, device="cuda"), p=0.5, seed=12,
                                           checkpoint=True)
    assert torch.isfinite(y[[0, 1, 2, 5]]).all() and torch.isnan(y[4]).all() and torch.isnan(y[3]).any()
    v = B.checkpoint8Values(ck)
    assert torch.isnan(v[3, :32]).all() and torch.isfinite(v[3, 32:]).all() and torch.isnan(v[4, 32:64]).all()


# ------------------------------------------------------------------ token mix

def mix64(x, mix, prev, lengths):
    """(y, last, the tokens before, which tokens are real [B, T, 1]) in 64 bits; what is not real reads as 0."""
    B, T, D = x.shape
    n = torch.full((B,), T, device=x.device) if lengths is None else lengths.long().clamp(0, T)
    real = (torch.arange(T, device=x.device)[None] < n[:, None])[..., None]
    x = torch.where(real, x.double(), 0.0)
    first = torch.zeros(B, D, device=x.device, dtype=torch.float64) if prev is None else prev.double()
    before = torch.where(real, torch.cat((first[:, None], x[:, :-1]), 1), 0.0)
    y = torch.stack([x + (before - x) * m for m in mix.double()])
    last = torch.where(n[:, None] > 0, x[torch.arange(B, device=x.device), (n - 1).clamp(min=0)], first)
    return y, last, before, real


def lengths_of(kind, B, T, seed=0):
    """None, or lengths with an empty sequence, one of a single token and a whole one;
    "outside": past the ends too."""
    if kind is None:
        return None
    g = torch.Generator(device="cuda").manual_seed(seed)
    n = torch.randint(0, T + 1, (B,), generator=g, device="cuda", dtype=torch.int32)
    for i, v in enumerate((0, 1, T)):
        if i < B:
            n[i] = min(v, T)
    if kind == "outside":
        n[0], n[-1] = -5, T + 9
    return n


MIX_SIZES = [(1, 1, 8), (1, 5, 64), (64, 1, 264), (3, 2, 128), (4, 37, 96), (2, 130, 768), (5, 9, 1032), (1, 700, 256), (7, 3, 8200)]


@pytest.mark.parametrize("dt", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("J", [1, 2, 3, 4, 5, 6])
@pytest.mark.parametrize("given", [False, True])
@pytest.mark.parametrize("ragged", [None, "ragged", "outside"])
def test_token_mix(cuda, dt, J, given, ragged):
    """Forward: the difference, its product and the sum, each rounded to fp32.
    Backward: sums of J terms to a token, of all tokens to a weight."""
    from swiftrwkv_b200 import block as B
    t = DTYPES[dt]
    for k, (b, T, D) in enumerate(MIX_SIZES):
        x = rnd((b, T, D), 250 + k, t)
        wd = PARAMS[k % 3]
        mix = torch.rand(J, D, generator=torch.Generator(device="cuda").manual_seed(k), device="cuda").to(wd)
        prev = rnd((b, D), 260 + k, t) if given else None
        n = lengths_of(ragged, b, T, k)
        y64, last64, before, real = mix64(x, mix, prev, n)
        if n is not None:
            x[~real.expand_as(x)] = float("nan")     # not read
        y, last = B.tokenMixForward(x, mix, prev, n)
        m = mix.double()[:, None, None]
        x64 = torch.where(real, x.double(), 0.0)
        d = before - x64
        tol = 2 * U32 * (d.abs() * m.abs()) + U32 * y64.abs()
        check(y, torch.where(real, y64, 0.0), tol * 1.01 + u(t) * (y64.abs() + tol), "y")
        assert not y[~real.expand_as(y)].any() and torch.equal(last.double(), last64)
        # backward
        dys = [rnd((b, T, D), 270 + 7 * k + j, t) for j in range(J)]
        if J > 1:
            dys[1] = None
        dlast = rnd((b, D), 290 + k, t) if k % 2 else None
        dy64 = torch.stack([torch.where(real, v.double(), 0.0) if v is not None else torch.zeros_like(x64) for v in dys])
        for v in dys:
            if v is not None and n is not None:
                v[~real.expand_as(v)] = float("inf")  # not read
        dx, dmix, dprev = B.tokenMixBackward(dys, x, mix, prev, n, dlast)
        grid = torch.zeros(b, T + 1, D, device="cuda", dtype=torch.float64)
        mag = torch.zeros_like(grid)
        for j in range(J):
            for own, part in ((1, (1 - m[j]) * dy64[j]), (0, m[j] * dy64[j])):
                grid[:, own:T + own] += part
                mag[:, own:T + own] += part.abs()
        if dlast is not None:
            at = real[..., 0].sum(1)
            grid[torch.arange(b), at] += dlast.double()
            mag[torch.arange(b), at] += dlast.double().abs()
        tol = (2 * J + 6) * U32 * mag
        check(dx, grid[:, 1:], (tol * 1.01 + u(t) * (grid.abs() + tol))[:, 1:], "dx")
        assert not dx[~real.expand_as(dx)].any()
        if given:
            check(dprev, grid[:, 0], (tol * 1.01 + u(t) * (grid.abs() + tol))[:, 0], "dprev")
        else:
            assert dprev is None
        terms = dy64 * d
        want, tol = terms.sum((1, 2)), (b * T + 16) * U32 * terms.abs().sum((1, 2))
        check(dmix, want, tol + u(wd) * (want.abs() + tol) + 1e-38, "dmix")
        again = B.tokenMixBackward(dys, x, mix, prev, n, dlast)
        assert torch.equal(again[0], dx) and torch.equal(again[1], dmix)             # deterministic
        bare = B.tokenMixBackward(dys, x, mix, prev, n, dlast, params=False)
        assert bare[1] is None and torch.equal(bare[0], dx)
        if J == 1 or n is not None:
            continue
        whole = torch.stack([v if v is not None else torch.zeros_like(x) for v in dys])
        assert all(a is c or torch.equal(a, c) for a, c in zip(B.tokenMixBackward(whole, x, mix, prev, n, dlast), again))


@pytest.mark.parametrize("dt", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("J", [1, 2, 6])
@pytest.mark.parametrize("b,T,D", [(4, 5, 64), (5, 301, 768)])
def test_token_mix_of_infinities_and_nan_in_padded_batches(cuda, dt, J, b, T, D):
    """Tokens from a sequence's length on take no part: neither an infinity in its last token nor
    weights of infinity and NaN make anything of them but zeros."""
    from swiftrwkv_b200 import block as B
    t = DTYPES[dt]
    x, prev, mix = rnd((b, T, D), 353, t), rnd((b, D), 354, t), torch.rand(J, D, generator=torch.Generator(device="cuda").manual_seed(5), device="cuda")
    n = lengths_of("ragged", b, T, 3)
    n[3] = 3
    dys, dlast = [rnd((b, T, D), 355 + j, t).abs() + 1 for j in range(J)], rnd((b, D), 361, t)
    _, _, before, real = mix64(x, mix, prev, n)
    # the last token of sequence 3 holds infinities; all weights are finite
    x[3, 2, :8] = float("inf")
    dx, dmix, dprev = B.tokenMixBackward(dys, x, mix, prev, n, dlast)
    want = torch.stack([torch.where(real, dy.double() * (before - x.double()), 0.0).sum((0, 1)) for dy in dys])
    assert torch.equal(dmix[:, :8], torch.full((J, 8), -float("inf"), device="cuda"))
    lim = torch.stack([torch.where(real, dy.double() * (before - x.double()), 0.0).abs().sum((0, 1)) for dy in dys])
    check(dmix[:, 8:], want[:, 8:], (b * T + 16) * U32 * lim[:, 8:], "dmix")
    assert torch.isfinite(dx).all() and torch.isfinite(dprev).all()
    x[3, 2, :8] = 1.0
    mix[:, 0], mix[0, D - 1] = float("inf"), float("nan")
    y, last = B.tokenMixForward(x, mix, prev, n)
    assert not y[~real.expand_as(y)].any() and torch.isfinite(last).all()
    assert torch.isnan(y[0][real[..., 0]][:, D - 1]).all() and torch.isfinite(y[..., 1:D - 1]).all()
    dx, _, dprev = B.tokenMixBackward(dys, x, mix, prev, n, dlast)
    assert not dx[~real.expand_as(dx)].any() and torch.isfinite(dx[..., 1:D - 1]).all()
    assert torch.equal(dprev[0], dlast[0])                # an empty sequence's
    # no token follows the last one: its gradient is (1 - m) dy and dlast, which the infinite weights turn to -inf
    assert torch.equal(dx[3, 2, 0], torch.tensor(-float("inf"), device="cuda", dtype=t))


@pytest.mark.parametrize("dt", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("J", [1, 4, 6])
@pytest.mark.parametrize("given", [False, True])
@pytest.mark.parametrize("ragged", [None, "ragged"])
def test_token_mix_of_training_batches(cuda, monkeypatch, dt, J, given, ragged):
    """Past the size at which a thread of the forward takes four tokens, and where a thread of the
    backward walks over many, with ends of sequences among them."""
    monkeypatch.setitem(globals(), "MIX_SIZES", [(9, 301, 2560), (1500, 3, 2048)])
    test_token_mix(cuda, dt, J, given, ragged)


def test_token_mix_continues_a_sequence(cuda):
    """Split anywhere, with last as the next part's prev: the whole's results; token by token too."""
    from swiftrwkv_b200 import block as B
    x, mix, prev = rnd((3, 41, 64), 300, torch.bfloat16), torch.rand(6, 64, device="cuda"), rnd((3, 64), 301, torch.bfloat16)
    y, last = B.tokenMixForward(x, mix, prev)
    assert torch.equal(last, x[:, -1])
    for cuts in ([0, 1, 17, 40, 41], list(range(42))):
        carry, parts = prev, []
        for a, c in zip(cuts, cuts[1:]):
            part, carry = B.tokenMixForward(x[:, a:c], mix, carry)
            parts.append(part)
        assert torch.equal(torch.cat(parts, 2), y) and torch.equal(carry, last)


def test_token_mix_gradient_matches_differences(cuda):
    """y and last are linear in x, prev and mix each: differences of any step are the
    derivative, up to the forward's roundings (three per y, of at most 4 |x| |dy| each)
    divided by the step of 1."""
    from swiftrwkv_b200 import block as B
    x, mix, prev = rnd((2, 7, 8), 302), torch.rand(3, 8, device="cuda"), rnd((2, 8), 303)
    n = torch.tensor([7, 4], device="cuda", dtype=torch.int32)
    dys, dlast = rnd((3, 2, 7, 8), 304), rnd((2, 8), 305)

    def f():
        y, last = B.tokenMixForward(x, mix, prev, n)
        return (y.double() * dys.double()).sum() + (last.double() * dlast.double()).sum()
    grads = B.tokenMixBackward(dys, x, mix, prev, n, dlast)
    lim = 3 * U32 * 4 * (1 + float(x.abs().max())) * float(dys.abs().sum()) + 1e-6
    for p, g in zip((x, mix, prev), grads):
        flat, gf = p.view(-1), g.reshape(-1)
        for i in range(0, flat.numel(), 3):
            keep = float(flat[i])
            flat[i] = keep + 1
            up = f()
            flat[i] = keep - 1
            dn = f()
            flat[i] = keep
            assert abs(float(up - dn) / 2 - float(gf[i])) < lim


def test_token_mix_differentiable(cuda):
    from swiftrwkv_b200 import block as B
    x, prev, mix = rnd((3, 10, 64), 306, torch.bfloat16), rnd((3, 64), 307, torch.bfloat16), rnd((4, 64), 308)
    n = torch.tensor([10, 0, 6], device="cuda", dtype=torch.int32)
    dys, dlast = [rnd(x.shape, 309 + j, torch.bfloat16) for j in range(4)], rnd((3, 64), 315, torch.bfloat16)
    for p in (prev, None):
        for lengths in (n, None):
            want = B.tokenMixBackward([dys[0], None, dys[2], None], x, mix, p, lengths, dlast)
            leaves = [v if v is None else v.clone().requires_grad_(True) for v in (x, mix, p)]
            ys, last = B.tokenMix(*leaves, lengths)
            fwd, last2 = B.tokenMixForward(x, mix, p, lengths)
            assert len(ys) == 4 and all(torch.equal(a, c) for a, c in zip(ys, fwd)) and torch.equal(last, last2)
            torch.autograd.backward([ys[0], ys[2], last], [dys[0], dys[2].transpose(0, 1).contiguous().transpose(0, 1), dlast])
            assert all(v is None or torch.equal(v.grad, g) for v, g in zip(leaves, want))
    xs = x.clone().requires_grad_(True)
    ys, last = B.tokenMix(xs, mix)
    last.backward(dlast)                                  # no y is used
    assert torch.equal(xs.grad[:, -1], dlast) and not xs.grad[:, :-1].any()
    with torch.no_grad():
        assert not B.tokenMix(xs, mix)[0][0].requires_grad


def test_token_mix_empty_batches_and_views(cuda):
    from swiftrwkv_b200 import block as B
    mix = torch.rand(6, 64, device="cuda")
    for shape in ((0, 5, 64), (3, 0, 64)):
        x = rnd(shape, 316, torch.bfloat16)
        prev = rnd((shape[0], 64), 317, torch.bfloat16)
        y, last = B.tokenMixForward(x, mix, prev)
        assert y.shape == (6, *shape) and torch.equal(last, prev)
        assert not B.tokenMixForward(x, mix)[1].any()
        dx, dmix, dprev = B.tokenMixBackward(y, x, mix, prev, dlast=prev)
        assert dx.shape == shape and not dmix.any() and torch.equal(dprev, prev)
        assert not B.tokenMixBackward([None] * 6, x, mix, prev)[2].any()
    base = rnd((9, 4, 64), 318)
    x, mix2 = base.transpose(0, 1), rnd((64 * 6 + 1,), 319)[1:].view(6, 64)          # strided; off a 16-byte boundary
    got, want = B.tokenMixForward(x, mix2), B.tokenMixForward(x.contiguous(), mix2.clone())
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    got = B.tokenMixBackward(x.expand(6, *x.shape), x, mix2)
    want = B.tokenMixBackward([x.contiguous()] * 6, x.contiguous(), mix2.clone())
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    every = rnd((8,), 320).to(torch.int32).abs()
    assert torch.equal(B.tokenMixForward(x, mix, lengths=every[::2])[0],
                       B.tokenMixForward(x.contiguous(), mix, lengths=every[::2].contiguous())[0])
    with pytest.raises(ValueError, match="lengths"):
        B.tokenMixForward(x, mix, lengths=torch.ones(4, device="cuda", dtype=torch.int64))
    with pytest.raises(ValueError, match="prev"):
        B.tokenMixForward(x, mix, prev=rnd((4, 56), 321))
    with pytest.raises(ValueError, match="multiple of 8"):
        B.tokenMixForward(rnd((2, 3, 12), 322), rnd((2, 12), 323))


def test_token_mix_past_32_bits(cuda):
    """Offsets past 2^32 elements in one sequence: first and last tokens, and what a NULL gradient leaves."""
    from swiftrwkv_b200 import block as B
    T, D = (1 << 21) + 5, 2048
    x = torch.zeros(1, T, D, device="cuda", dtype=torch.bfloat16)
    x[0, -3:] = rnd((3, D), 324, torch.bfloat16)
    x[0, :2] = rnd((2, D), 325, torch.bfloat16)
    mix = torch.rand(1, D, device="cuda")
    y, last = B.tokenMixForward(x, mix)
    assert torch.equal(last[0], x[0, -1])
    for at in (0, T - 3):
        part, _ = B.tokenMixForward(x[:, at:at + 3], mix, x[:, at - 1] if at else None)
        assert torch.equal(y[0, 0, at:at + 3], part[0, 0])
    del y
    dx, dmix, _ = B.tokenMixBackward([x], x, mix, dlast=last)
    part, pm, _ = B.tokenMixBackward([x[:, -3:].contiguous()], x[:, -3:].contiguous(), mix, x[:, -4], dlast=last)
    head, hm, _ = B.tokenMixBackward([x[:, :3].contiguous()], x[:, :3].contiguous(), mix)
    assert torch.equal(dx[:, -3:], part) and torch.equal(dx[:, :2], head[:, :2])
    # the tokens in between add nothing: dmix is the two ends', up to the order of six terms
    lim = 6 * U32 * (x[0, -3:].double() ** 2).sum(0).max() * 2 + 6 * U32 * (x[0, :2].double() ** 2).sum(0).max() * 2
    check(dmix, (pm + hm).double(), 4 * lim, "dmix")


# ------------------------------------------------------ tail of the time mix

TAIL_SIZES = [(1, 1, 64), (3, 2, 64), (1, 32, 64), (7, 1, 32), (5, 3, 32), (2, 5, 128), (3, 3, 256), (33, 12, 64), (301, 4, 64),
              (1003, 2, 32), (2, 160, 64)]


def tail64(a, r, k, v, g, rk, w, b, eps, dout=None):
    """Outputs and gradients in 64 bits with the bounds of their errors before the store."""
    rows, (H, S) = a.shape[0], rk.shape
    a, r, k, v, g = (t.double().view(rows, H, S) for t in (a, r, k, v, g))
    rk, w, b = (t.double().view(H, S) for t in (rk, w, b))
    N = (S + 16) * U32
    mean = a.mean(2, keepdim=True)
    dev = a - mean
    em = N * a.abs().mean(2, keepdim=True)
    ed = em + U32 * dev.abs()
    rstd = 1 / torch.sqrt((dev ** 2).mean(2, keepdim=True) + eps)
    evar = (2 * dev.abs() * ed + ed ** 2).mean(2, keepdim=True) + N * (dev ** 2).mean(2, keepdim=True)
    er = 0.5 * evar * rstd ** 2 * 1.01 + 8 * U32                     # relative
    n = dev * rstd
    en = rstd * ed + n.abs() * (er + 4 * U32)
    terms = r * k * rk
    c, ec = terms.sum(2, keepdim=True), N * terms.abs().sum(2, keepdim=True)
    z = n * w + b + c * v
    ez = w.abs() * en + v.abs() * ec + 4 * U32 * ((n * w).abs() + b.abs() + (c * v).abs())
    if dout is None:
        out = z * g
        return out.view(rows, -1), (g.abs() * ez * 1.01 + 2 * U32 * out.abs()).view(rows, -1)
    d = dout.double().view(rows, H, S)
    dz = d * g
    dg, edg = d * z, d.abs() * ez + 2 * U32 * (d * z).abs()
    dv, edv = c * dz, dz.abs() * ec + 3 * U32 * (c * dz).abs()
    dc, edc = (dz * v).sum(2, keepdim=True), N * (dz * v).abs().sum(2, keepdim=True)
    dr, edr = dc * rk * k, edc * (rk * k).abs() + 4 * U32 * (dc * rk * k).abs()
    dk, edk = dc * rk * r, edc * (rk * r).abs() + 4 * U32 * (dc * rk * r).abs()
    e = dz * w
    m1, em1 = e.mean(2, keepdim=True), N * e.abs().mean(2, keepdim=True)
    m2 = (e * n).mean(2, keepdim=True)
    em2 = rstd * (e.abs() * ed).mean(2, keepdim=True) + (N + er + 4 * U32) * (e * n).abs().mean(2, keepdim=True)
    da = rstd * (e - m1 - n * m2)
    eda = rstd * (em1 + en * m2.abs() + n.abs() * em2) + (er + 8 * U32) * rstd * (e.abs() + m1.abs() + (n * m2).abs())
    R = (rows + 16) * U32
    drk, edrk = (dc * r * k).sum(0), R * (dc * r * k).abs().sum(0) + (edc * (r * k).abs()).sum(0)
    dw, edw = (dz * n).sum(0), R * (dz * n).abs().sum(0) + (dz.abs() * en).sum(0)
    db, edb = dz.sum(0), R * dz.abs().sum(0)
    rowwise = [(x.reshape(rows, -1), y.reshape(rows, -1) * 1.01) for x, y in
               ((da, eda), (dr, edr), (dk, edk), (dv, edv), (dg, edg))]
    return rowwise + [(drk, edrk * 1.01 + 1e-38), (dw.flatten(), edw.flatten() * 1.01 + 1e-38), (db.flatten(), edb.flatten() + 1e-38)]


def tail_inputs(rows, H, S, t, wd, seed):
    a = (rnd((rows, H, S), seed) * torch.exp(rnd((1, H, 1), seed + 1)) + rnd((rows, H, 1), seed + 2) * 0.3).view(rows, H * S).to(t)
    r, k, v, g, dout = (rnd((rows, H * S), seed + 3 + i, t) for i in range(5))
    rk, w, b = rnd((H, S), seed + 8, wd, 0.2), (rnd((H * S,), seed + 9) * 0.2 + 0.8).to(wd), rnd((H * S,), seed + 10, wd, 0.2)
    return (a, r, k, v, g, rk, w, b), dout


@pytest.mark.parametrize("dt", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("rows,H,S", TAIL_SIZES)
def test_tail(cuda, dt, rows, H, S):
    from swiftrwkv_b200 import block as B
    t = DTYPES[dt]
    for wd in PARAMS:
        ins, dout = tail_inputs(rows, H, S, t, wd, 400)
        out = B.tmixTailForward(*ins)
        want, tol = tail64(*ins, 64e-5)
        check(out, want, tol + u(t) * (want.abs() + tol), "out")
        got = B.tmixTailBackward(dout, *ins)
        names = ("dwkv", "dr", "dk", "dv", "dg", "drk", "dweight", "dbias")
        for name, x, (want, tol), like in zip(names, got, tail64(*ins, 64e-5, dout), ins):
            assert x.shape == like.shape and x.dtype == like.dtype
            check(x, want.view(x.shape), (tol + u(x.dtype) * (want.abs() + tol)).view(x.shape), name)
        again = B.tmixTailBackward(dout, *ins)
        assert all(torch.equal(a, c) for a, c in zip(again, got))
        bare = B.tmixTailBackward(dout, *ins, params=False)
        assert all(torch.equal(a, c) for a, c in zip(bare[:5], got)) and bare[5:] == (None,) * 3


@pytest.mark.parametrize("dt", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("rows,H,S", [(5, 1, 64), (1003, 2, 32), (1003, 40, 64), (37, 3, 128), (14, 2, 256)])
def test_tail_without_eps(cuda, dt, rows, H, S):
    """eps = 0 over heads that vary: finite, also where a thread's last step has no row left."""
    from swiftrwkv_b200 import block as B
    t = DTYPES[dt]
    ins, dout = tail_inputs(rows, H, S, t, torch.float32, 405)
    want, tol = tail64(*ins, 0.0)
    check(B.tmixTailForward(*ins, 0.0), want, tol + u(t) * (want.abs() + tol), "out")
    got = B.tmixTailBackward(dout, *ins, 0.0)
    for i, (x, (want, tol)) in enumerate(zip(got, tail64(*ins, 0.0, dout))):
        check(x, want.view(x.shape), (tol + u(x.dtype) * (want.abs() + tol)).view(x.shape), i)


@pytest.mark.parametrize("dt", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("rows,H,S", [(1003, 40, 64), (5003, 20, 32), (2501, 12, 128), (2999, 6, 256)])
def test_tail_of_several_rows_a_thread(cuda, dt, rows, H, S):
    """Past 113664 units of 8 channels, a number of rows that does not divide among the threads."""
    test_tail(cuda, dt, rows, H, S)


def test_tail_agrees_with_the_decode_form(cuda):
    """kernel.wkvTail computes the same in fp32: both within the bound."""
    from swiftrwkv_b200 import block as B, kernel as K
    ins, _ = tail_inputs(5, 12, 64, torch.float32, torch.float32, 420)
    a, r, k, v, g, rk, w, b = ins
    old = K.wkvTail(a, r, k, v, rk, w, b, g, 12, 64, rows=5)
    want, tol = tail64(*ins, 64e-5)
    check(old, want, tol, "wkvTail")
    check(B.tmixTailForward(*ins), want, tol, "tmixTail")


def test_tail_gradient_matches_differences(cuda):
    """The output is linear in every input but wkv (differences of a step of 1, up to
    the forward's roundings) and smooth in wkv (a step of 2^-6: 1e-2 of the largest
    gradient, as for the layer norm)."""
    from swiftrwkv_b200 import block as B
    ins, dout = tail_inputs(3, 2, 32, torch.float32, torch.float32, 430)
    f = lambda: (B.tmixTailForward(*ins).double() * dout.double()).sum()
    grads = B.tmixTailBackward(dout, *ins)
    off = lambda: (tail64(*ins, 64e-5)[1] * dout.double().abs()).sum()       # f's own error there
    own = [tol for _, tol in tail64(*ins, 64e-5, dout)]
    for i, (p, g) in enumerate(zip(ins, grads)):
        flat, gf = p.view(-1), g.reshape(-1)
        h = 2.0 ** -6 if i == 0 else 1.0
        for j in range(0, flat.numel(), 7):
            keep = float(flat[j])
            flat[j] = keep + h
            up, lim = f(), off()
            flat[j] = keep - h
            dn, lim = f(), lim + off()
            flat[j] = keep
            lim = 1e-2 * float(g.abs().max()) if i == 0 else float(lim) / 2 + float(own[i].flatten()[j])
            assert abs(float(up - dn) / (2 * h) - float(gf[j])) < lim + 2 ** -22 * abs(keep) * float(gf[j].abs()), i


def test_tail_forms_shapes_and_empty_batches(cuda):
    """[..., H, S] and [..., H S] alike; gradients in their inputs' forms; views; no rows."""
    from swiftrwkv_b200 import block as B
    ins, dout = tail_inputs(12, 3, 64, torch.bfloat16, torch.float32, 440)
    out, grads = B.tmixTailForward(*ins), B.tmixTailBackward(dout, *ins)
    heads = [t.view(3, 4, 3, 64) for t in ins[:5]]
    mixed = (heads[0], heads[1].flatten(2), heads[2], heads[3].flatten(2), ins[4].view(3, 4, 192), *ins[5:])
    o2 = B.tmixTailForward(*mixed)
    assert o2.shape == (3, 4, 192) and torch.equal(o2.view(12, 192), out)
    g2 = B.tmixTailBackward(dout.view(3, 4, 3, 64), *mixed)
    assert all(a.shape == m.shape and torch.equal(a.view(c.shape), c) for a, m, c in zip(g2, mixed, grads))
    strided = [t.view(4, 3, 192).transpose(0, 1) for t in ins[:5]]
    assert torch.equal(B.tmixTailForward(*strided, *ins[5:]), B.tmixTailForward(*[t.contiguous() for t in strided], *ins[5:]))
    off = [torch.cat((t.flatten()[:1], t.flatten()))[1:].view(t.shape) for t in ins]
    assert torch.equal(B.tmixTailForward(*off), out)
    assert all(torch.equal(a, c) for a, c in zip(B.tmixTailBackward(dout, *off), grads))
    empty = [t[:0] for t in ins[:5]]
    assert B.tmixTailForward(*empty, *ins[5:]).shape == (0, 192)
    g0 = B.tmixTailBackward(dout[:0], *empty, *ins[5:])
    assert g0[0].shape == (0, 192) and not any(t.any() for t in g0[5:])
    one = [t[0] for t in ins[:5]]
    assert torch.equal(B.tmixTailForward(*one, *ins[5:]), out[0])
    with pytest.raises(ValueError, match="S=48"):
        B.tmixTailForward(*[t[:, :96] for t in ins[:5]], ins[5].flatten()[:96].view(2, 48), ins[6][:96], ins[7][:96])
    with pytest.raises(ValueError, match="weight"):
        B.tmixTailForward(*ins[:6], ins[6][:64], ins[7])
    with pytest.raises(ValueError, match="k: dtype"):
        B.tmixTailForward(ins[0], ins[1], ins[2].float(), *ins[3:])


def test_tail_of_one_head_and_one_token(cuda):
    """[B, 1, S] is a token of [.., H S] and a head of [.., H, S]: the other form of either goes with it."""
    from swiftrwkv_b200 import block as B
    ins, dout = tail_inputs(3, 1, 64, torch.float32, torch.float32, 441)
    out, grads = B.tmixTailForward(*ins), B.tmixTailBackward(dout, *ins)
    flat, tokens, heads = [[t.view(shape) for t in ins[:5]] for shape in ((3, 64), (3, 1, 64), (3, 1, 1, 64))]
    for first, others in ((tokens, heads), (tokens, flat), (heads, tokens)):
        mixed = (*first[:1], *others[1:], *ins[5:])
        assert torch.equal(B.tmixTailForward(*mixed).view(3, 64), out)
        got = B.tmixTailBackward(dout.view(others[0].shape), *mixed)
        assert all(a.shape == m.shape and torch.equal(a.view(c.shape), c) for a, m, c in zip(got, mixed, grads))
    with pytest.raises(ValueError, match="r "):
        B.tmixTailForward(flat[0], *heads[1:], *ins[5:])


def test_tail_may_write_over_its_inputs(cuda):
    from swiftrwkv_b200 import _lib, block as B
    ins, dout = tail_inputs(1301, 4, 64, torch.bfloat16, torch.float32, 450)
    st = torch.cuda.current_stream().cuda_stream
    out, grads = B.tmixTailForward(*ins), B.tmixTailBackward(dout, *ins)
    for i in range(5):
        c = [t.clone() for t in ins]
        ps = [t.data_ptr() for t in c]
        _lib.call("rwkv_tmix_tail_forward", _lib.BF16, *ps[:5], _lib.F32, *ps[5:], 64e-5, ps[i], 1301, 4, 64, st)
        assert torch.equal(c[i], out)
    for turn in range(6):
        c = [t.clone() for t in ins]
        d = dout.clone()
        over = ([d] + c[:5])[turn:] + ([d] + c[:5])[:turn]
        ps = [t.data_ptr() for t in c]
        _lib.call("rwkv_tmix_tail_backward", _lib.BF16, d.data_ptr(), *ps[:5], _lib.F32, *ps[5:], 64e-5,
                  *[t.data_ptr() for t in over[:5]], None, None, None, 1301, 4, 64, None, 0, st)
        assert all(torch.equal(a, b) for a, b in zip(over, grads[:5]))


@pytest.mark.parametrize("dt", ["f32", "bf16"])
def test_tail_may_write_over_inputs_that_are_read_ahead(cuda, dt):
    """As above where a thread has several rows, whose later ones are on their way meanwhile."""
    from swiftrwkv_b200 import _lib, block as B
    rows, H, S, t = 1003, 40, 64, DTYPES[dt]
    ins, dout = tail_inputs(rows, H, S, t, torch.float32, 451)
    st, code = torch.cuda.current_stream().cuda_stream, B._DT[t]
    out, grads = B.tmixTailForward(*ins), B.tmixTailBackward(dout, *ins)
    for i in range(5):
        c = [v.clone() for v in ins]
        ps = [v.data_ptr() for v in c]
        _lib.call("rwkv_tmix_tail_forward", code, *ps[:5], _lib.F32, *ps[5:], 64e-5, ps[i], rows, H, S, st)
        assert torch.equal(c[i], out)
    for turn in range(6):
        c, d = [v.clone() for v in ins], dout.clone()
        over = ([d] + c[:5])[turn:] + ([d] + c[:5])[:turn]
        ps = [v.data_ptr() for v in c]
        _lib.call("rwkv_tmix_tail_backward", code, d.data_ptr(), *ps[:5], _lib.F32, *ps[5:], 64e-5,
                  *[v.data_ptr() for v in over[:5]], None, None, None, rows, H, S, None, 0, st)
        assert all(torch.equal(a, b) for a, b in zip(over, grads[:5]))


def test_tail_of_constant_heads_infinities_and_nan(cuda):
    """A head without variance gives its bias and finite gradients; a NaN or an
    infinity stays in its row and head."""
    from swiftrwkv_b200 import block as B
    ins, dout = tail_inputs(6, 3, 64, torch.float32, torch.float32, 460)
    a, r, k, v, g, rk, w, b = ins
    a.view(6, 3, 64)[1, 1] = 0.0
    a.view(6, 3, 64)[2, 2] = 1000.0
    out, want = B.tmixTailForward(*ins), tail64(*ins, 64e-5)
    check(out, want[0], want[1], "out")
    a.view(6, 3, 64)[4, 0, 5] = float("nan")
    k.view(6, 3, 64)[5, 1, 9] = float("inf")
    out = B.tmixTailForward(*ins).view(6, 3, 64)
    bad = ~torch.isfinite(out)
    assert bad[4, 0].all() and bad[5, 1].any() and int(bad.any(2).sum()) == 2
    grads = B.tmixTailBackward(dout, *ins)
    for x in grads[:5]:
        assert int((~torch.isfinite(x.view(6, 3, 64))).any(2).sum()) <= 2
    assert torch.isfinite(grads[0].view(6, 3, 64)[1, 1]).all() and torch.isfinite(grads[0].view(6, 3, 64)[2, 2]).all()
    for x in grads[5:]:
        assert torch.isfinite(x.view(3, 64)[2]).all()


def test_tail_differentiable(cuda):
    from swiftrwkv_b200 import block as B
    ins, dout = tail_inputs(10, 2, 64, torch.bfloat16, torch.bfloat16, 470)
    want = B.tmixTailBackward(dout, *ins)
    leaves = [t.clone().requires_grad_(True) for t in ins]
    out = B.tmixTail(*leaves)
    assert torch.equal(out.detach(), B.tmixTailForward(*ins))
    out.backward(dout)
    assert all(torch.equal(v.grad, g) for v, g in zip(leaves, want))
    frozen = [t.clone().requires_grad_(i < 5) for i, t in enumerate(ins)]
    B.tmixTail(*frozen).backward(dout)
    assert all(torch.equal(v.grad, g) for v, g in zip(frozen[:5], want)) and frozen[6].grad is None


def test_tail_past_32_bits(cuda):
    """Rows whose elements lie past 2^32."""
    from swiftrwkv_b200 import block as B
    rows, H, S = (1 << 16) + 7, 1024, 64
    p = rnd((H, S), 480), rnd((H * S,), 481), rnd((H * S,), 482)
    x = torch.zeros(rows, H * S, device="cuda", dtype=torch.float16)
    x[-9:] = rnd((9, H * S), 483, torch.float16)
    x[:2] = rnd((2, H * S), 484, torch.float16)
    out = B.tmixTailForward(x, x, x, x, x, *p)
    for part in (slice(0, 2), slice(rows - 9, rows)):
        y = x[part].contiguous()
        assert torch.equal(out[part], B.tmixTailForward(y, y, y, y, y, *p))
    del out
    grads = B.tmixTailBackward(x, x, x, x, x, x, *p, params=False)[:5]
    for part in (slice(0, 2), slice(rows - 9, rows)):
        y = x[part].contiguous()
        for a, c in zip(grads, B.tmixTailBackward(y, y, y, y, y, y, *p, params=False)):
            assert torch.equal(a[part], c)


# --------------------------------------------------------------- all together

def operators(x, seed):
    """One explicit pass through all four, forward and backward."""
    from swiftrwkv_b200 import block as B
    rows, T, D = x.shape
    dt = x.dtype
    w, b = rnd((D,), 500) * 0.1 + 1, rnd((D,), 501) * 0.1
    mix, rk = torch.rand(6, D, generator=torch.Generator(device="cuda").manual_seed(3), device="cuda"), rnd((D // 64, 64), 502) * 0.1

    def run(x, br, dy, seed, prev):
        d = B.dropoutForward(br, 0.2, seed, 1)
        s, y, mean, rstd, ck = B.residualNormForward(x, d, w, b, scale=0.5, p=0.1, seed=seed, offset=2, checkpoint=True)
        m, last = B.tokenMixForward(y, mix, prev)
        o = B.tmixTailForward(m[0], m[1], m[2], m[3], m[4], rk, w, b)
        gs = B.tmixTailBackward(dy, m[0], m[1], m[2], m[3], m[4], rk, w, b)
        dx, dmix, dprev = B.tokenMixBackward([*gs[:5], None], y, mix, prev, dlast=last)
        return [d, s, y, last, o, *gs, dmix, dprev, *B.residualNormBackward(dx, ck, w, mean, rstd, dy, 0.5, 0.1, seed, 2)]
    return run


def test_two_streams_at_once(cuda):
    cases = []
    for k in range(2):
        x = rnd((2, 200 + k, 512), 510 + k, torch.bfloat16)
        cases.append((operators(x, k), (x, rnd(x.shape, 512 + k, torch.bfloat16), rnd(x.shape, 514 + k, torch.bfloat16), k,
                                        rnd((2, 512), 516 + k, torch.bfloat16))))
    want = [f(*a) for f, a in cases]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    got = [[], []]
    for _ in range(5):
        for k, s in enumerate(streams):
            with torch.cuda.stream(s):
                got[k].append(cases[k][0](*cases[k][1]))
    torch.cuda.synchronize()
    for k in range(2):
        for g in got[k]:
            assert all(torch.equal(a, c) for a, c in zip(g, want[k]))


def test_captured_calls_replay_on_new_inputs_and_seeds(cuda):
    """Two graphs replayed in turn, with new inputs and a new seed in the captured buffers."""
    kept_, state = [], torch.tensor([1, 0], device="cuda")
    for T in (3, 70):
        x = rnd((2, T, 256), 520, torch.bfloat16)
        args = [x, rnd(x.shape, 521, torch.bfloat16), rnd(x.shape, 522, torch.bfloat16), state, rnd((2, 256), 523, torch.bfloat16)]
        f = operators(x, 0)
        s = torch.cuda.Stream()
        s.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(s):
            f(*args)
        torch.cuda.current_stream().wait_stream(s)
        gr = torch.cuda.CUDAGraph()
        with torch.cuda.graph(gr):
            out = f(*args)
        kept_.append((gr, f, args, out))
    for seed in (5, 9):
        state.copy_(torch.tensor([seed, seed * 3]))
        for k, (gr, _, args, _) in enumerate(kept_):
            for a in (0, 1, 2, 4):
                args[a].copy_(rnd(args[a].shape, 530 + 10 * seed + a + 5 * k, torch.bfloat16))
            gr.replay()
        for gr, f, args, out in kept_:
            assert all(torch.equal(a, c) for a, c in zip(out, f(*args)))
    first = [o.clone() for o in kept_[0][3]]
    state += 1
    kept_[0][0].replay()
    assert not torch.equal(first[0], kept_[0][3][0])


def test_differentiable_forms_refuse_capture(cuda):
    from swiftrwkv_b200 import block as B
    x = rnd((2, 4, 64), 540, torch.bfloat16)
    w, b, mix, rk = torch.ones(64, device="cuda"), torch.zeros(64, device="cuda"), torch.rand(2, 64, device="cuda"), torch.ones(1, 64, device="cuda")
    calls = [lambda x: B.dropout(x, 0.1, 1), lambda x: B.residualNorm(x, x, w, b, p=0.1)[0], lambda x: B.tokenMix(x, mix)[0][0],
             lambda x: B.tmixTail(x, x, x, x, x, rk, w, b)]
    xs = x.clone().requires_grad_(True)
    live = [f(xs) for f in calls]                        # eager graphs of the same leaf, alive meanwhile
    gr = torch.cuda.CUDAGraph()
    with torch.cuda.graph(gr):
        for f in calls:
            with pytest.raises(ValueError, match="capture"):
                f(xs)
        ys = [f(x) for f in calls]                       # nothing is recorded: taken
    gr.replay()
    assert all(torch.equal(y, f(x)) for y, f in zip(ys, calls))
    for y in live:
        y.backward(x)


@pytest.mark.parametrize("B_,T,p", [(1, 16, 0.0), (3, 48, 0.2)])
def test_block_run_and_its_gradients(cuda, B_, T, p):
    """A whole x070 block from these operators, the projections and the WKV path,
    against the same block in 64 bits: outputs and every gradient.  In the 2-norm: the
    longest path rounds about 20 times to bf16 forth and as often back, each at most 2^-8
    and of either sign, sqrt(40) 2^-8 = 2.5 %; the normed keys and the norms by head
    divide by lengths that vary by row, which weighs rows by up to about 3: bound 8 %."""
    from swiftrwkv_b200 import block as B, kernel as K
    D, F, H, t = 128, 512, 2, torch.bfloat16
    P = {k: rnd((D, D), 550 + i, t, D ** -0.5) for i, k in enumerate(("r", "k", "v", "w", "a", "g", "o"))}
    P |= {"key": rnd((F, D), 560, t, D ** -0.5), "value": rnd((D, F), 561, t, F ** -0.5)}
    for i, k in enumerate(("w1", "w2", "wx", "w3")):
        P[k] = rnd((D,), 562 + i, scale=0.1) + 1
    for i, k in enumerate(("b1", "b2", "bx", "b3")):
        P[k] = rnd((D,), 566 + i, scale=0.1)
    gen = torch.Generator(device="cuda").manual_seed(9)
    P |= {"mix": torch.rand(6, D, generator=gen, device="cuda"), "cmix": torch.rand(1, D, generator=gen, device="cuda"),
          "rk": rnd((H, 64), 571, scale=0.1)}
    x, dout = rnd((B_, T, D), 572, t), rnd((B_, T, D), 573, t)

    def wkv_inputs(rr, kk, ww, aa, vv):
        """What the WKV path takes, from the projections (elementwise, in their type's higher precision)."""
        n = kk.view(B_, T, H, 64)
        kn = n / (n.square().sum(-1, keepdim=True) + 1e-6).sqrt()
        al = torch.sigmoid(aa.view(B_, T, H, 64))
        return (rr.view(B_, T, H, 64), torch.exp(-0.606531 * torch.sigmoid(ww.view(B_, T, H, 64))), n, vv.view(B_, T, H, 64), -kn, kn * al)

    def ours(x, P):
        h = B.layerNorm(x, P["w1"], P["b1"])
        (mr, mw, mk, mv, ma, mg), _ = B.tokenMix(h, P["mix"])
        r, w, k, v, a = (B.projection(m, P[n]) for m, n in ((mr, "r"), (mw, "w"), (mk, "k"), (mv, "v"), (ma, "a")))
        g = B.projection(mg, P["g"], act="sigmoid")
        y, _ = K.wkv7TrainWithState(*[q.to(t).contiguous() for q in wkv_inputs(r.float(), k.float(), w.float(), a.float(), v.float())])
        o = B.projection(B.tmixTail(y, r, k, v, g, P["rk"], P["wx"], P["bx"]), P["o"])
        s, h = B.residualNorm(x, o, P["w2"], P["b2"], scale=0.5, p=p, seed=77, offset=1)
        (m,), _ = B.tokenMix(h, P["cmix"])
        c = B.dropout(B.channelMix(m, P["key"], P["value"], checkpoint=False), p, 77, 2)
        return B.residualNorm(s, c, P["w3"], P["b3"])[1]

    def norm(x, w, b):
        return torch.nn.functional.layer_norm(x, x.shape[-1:], w, b, 1e-5)

    def shift(x, mix):
        before = torch.nn.functional.pad(x, (0, 0, 1, 0))[:, :-1]
        return [x + (before - x) * m for m in mix]

    def plain(x, P):
        h = norm(x, P["w1"], P["b1"])
        mr, mw, mk, mv, ma, mg = shift(h, P["mix"])
        r, w, k, v, a = (m @ P[n].t() for m, n in ((mr, "r"), (mw, "w"), (mk, "k"), (mv, "v"), (ma, "a")))
        g = torch.sigmoid(mg @ P["g"].t())
        q = wkv_inputs(r, k, w, a, v)
        S, ys = torch.zeros(B_, H, 64, 64, device="cuda", dtype=torch.float64), []
        for i in range(T):
            ri, wi, ki, vi, ai, bi = (z[:, i] for z in q)
            S = S * wi[:, :, None] + vi[..., None] * ki[:, :, None] + (S @ ai[..., None]) * bi[:, :, None]
            ys.append((S @ ri[..., None])[..., 0])
        y = torch.stack(ys, 1)
        n = torch.nn.functional.layer_norm(y, (64,), None, None, 64e-5) * P["wx"].view(H, 64) + P["bx"].view(H, 64)
        heads = lambda z: z.view(B_, T, H, 64)
        z = n + (heads(r) * heads(k) * P["rk"]).sum(-1, keepdim=True) * heads(v)
        o = (z.flatten(2) * g) @ P["o"].t()
        drop = lambda z, offset: torch.where(mask(z.shape, p, 77, offset), z * factor(p), 0.0)
        s = x + 0.5 * drop(o, 1)
        (m,) = shift(norm(s, P["w2"], P["b2"]), P["cmix"])
        c = drop(torch.relu(m @ P["key"].t()) ** 2 @ P["value"].t(), 2)
        return norm(s + c, P["w3"], P["b3"])

    P = {k: v.requires_grad_(True) for k, v in P.items()}
    x.requires_grad_(True)
    y = ours(x, P)
    y.backward(dout)
    P64 = {k: v.detach().double().requires_grad_(True) for k, v in P.items()}
    x64 = x.detach().double().requires_grad_(True)
    y64 = plain(x64, P64)
    y64.backward(dout.double())
    rel = lambda a, b: float((a.double() - b).norm() / b.norm())
    assert rel(y.detach(), y64.detach()) < 0.08
    for name, a, b in [("x", x.grad, x64.grad)] + [(k, P[k].grad, P64[k].grad) for k in P]:
        assert rel(a, b) < 0.08, (name, rel(a, b))


@pytest.mark.parametrize("bad", ["1e-5", None, 10 ** 400, 1 + 0j], ids=["text", "none", "huge", "complex"])
def test_what_is_no_number_is_refused(cuda, bad):
    from swiftrwkv_b200 import block as B
    x, v = rnd((2, 64), 596), torch.ones(64, device="cuda")
    for f in (lambda: B.layerNormForward(x, v, v, bad), lambda: B.residualNormForward(x, x, v, v, bad),
              lambda: B.residualNormForward(x, x, v, v, scale=bad), lambda: B.residualNormForward(x, x, v, v, p=bad),
              lambda: B.residualNormBackward(x, x, v, x[:, 0], x[:, 1], scale=bad),
              lambda: B.tmixTailForward(x, x, x, x, x, v[None], v, v, bad),
              lambda: B.tmixTailBackward(x, x, x, x, x, x, v[None], v, v, bad), lambda: B.dropoutForward(x, bad, 1)):
        with pytest.raises(ValueError):
            f()


def test_host_tensors_beside_cuda_tensors_are_refused(cuda):
    """Tensors of two devices in one call are a ValueError."""
    from swiftrwkv_b200 import block as B
    x, v = rnd((2, 3, 64), 580), torch.ones(64, device="cuda")
    for f in (lambda: B.residualNormForward(x, x.cpu(), v, v), lambda: B.tokenMixForward(x, v[None], lengths=torch.ones(2, dtype=torch.int32)),
              lambda: B.tmixTailForward(x, x, x, x.cpu(), x, v[None], v, v), lambda: B.dropoutForward(x, 0.1, torch.zeros(2, dtype=torch.int64)),
              lambda: B.tokenMixBackward([x.cpu()], x, v[None])):
        with pytest.raises(ValueError, match="CUDA tensor"):
            f()


CAPTURE_FIRST = """
import sys
sys.path.insert(0, {root!r})
import torch
from swiftrwkv_b200 import block as B
g = torch.Generator(device="cuda").manual_seed(1)
def calls(dt, D):
    rnd = lambda *s: torch.randn(s, generator=g, device="cuda").to(dt)
    x, br, dy, prev, w = rnd(2, 37, D), rnd(2, 37, D), rnd(2, 37, D), rnd(2, D), rnd(D)
    mix, rk, seed = rnd(6, D), rnd(D // 64, 64), torch.tensor([3, 4], device="cuda")
    def run():
        d = B.dropoutForward(br, 0.2, seed, 1)
        s, y, mean, rstd, ck = B.residualNormForward(x, d, w, w, p=0.1, seed=seed, checkpoint=True)
        m, last = B.tokenMixForward(y, mix, prev)
        o = B.tmixTailForward(m[0], m[1], m[2], m[3], m[4], rk, w, w)
        gs = B.tmixTailBackward(dy, m[0], m[1], m[2], m[3], m[4], rk, w, w)
        dx, dmix, dprev = B.tokenMixBackward([*gs[:5], None], y, mix, prev, dlast=last)
        return [d, s, y, last, o, *gs, dmix, dprev, *B.residualNormBackward(dx, ck, w, mean, rstd, dy, 0.5, 0.1, seed, 2)]
    return run
for f in (calls(torch.bfloat16, 256), calls(torch.float32, 2560)):
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = f()
    graph.replay()
    assert all(torch.equal(a, c) for a, c in zip(got, f()))
print("ok")
"""


def test_first_calls_during_capture(cuda):
    """Nothing has to run before a capture: kernels of short and of long rows."""
    import os
    import subprocess
    import sys
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    r = subprocess.run([sys.executable, "-c", CAPTURE_FIRST.format(root=root)], capture_output=True, text=True, timeout=300)
    assert r.returncode == 0 and "ok" in r.stdout, r.stderr[-2000:]
