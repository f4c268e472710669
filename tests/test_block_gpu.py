"""GPU tests of the block operators against plain implementations in 64 bits.

Tolerances.  u(t) = finfo(t).eps / 2 bounds the relative error of one rounding
to type t.  A sum of n terms taken in fp32 in any order is off by at most
n 2^-24 sum|terms|; each term adds a few roundings of its own (counted as 16).
The tensor core adds its products in fp32 with rounding of its own, in far
fewer sequential steps than terms: 2^-20 sum|terms|, the bound that the
projection-backward tests of the frozen base use too.  A result is then off by
the error of its sums carried through the formula, plus its one rounding
u(t) |result|.
"""
from __future__ import annotations

import sys
import threading

import pytest
import torch

pytestmark = pytest.mark.gpu

DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
U32 = 2.0 ** -24
TC = 2.0 ** -20


def u(dt):
    return torch.finfo(dt).eps / 2


def rnd(shape, seed, dt=torch.float32, scale=1.0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return (torch.randn(shape, generator=g, device="cuda") * scale).to(dt)


def check(got, want, tol, what=""):
    """|got - want| <= tol elementwise; NaN at the same places.  u(t) |x| bounds
    a rounding only of normal numbers: below finfo.tiny a type's values are
    tiny eps apart, so that a rounding there is off by up to tiny eps / 2, which
    is added (fp16: 2^-14 2^-10 / 2 = 2^-25; the other types: below 1e-40)."""
    f = torch.finfo(got.dtype)
    tol = tol + f.tiny * f.eps / 2
    got, want = got.double(), want.double()
    assert got.shape == want.shape, (what, got.shape, want.shape)
    fin = torch.isfinite(want)
    assert torch.equal(torch.isnan(got), torch.isnan(want)), what
    off = (got - want).abs()[fin]
    lim = tol.expand_as(want)[fin] if torch.is_tensor(tol) else tol
    bad = ~(off <= lim)
    assert not bad.any(), f"{what}: {int(bad.sum())} of {off.numel()} beyond the bound, worst {float((off / lim).max()):.3g} of it"


# ------------------------------------------------------------------ formulas

def values64(x):
    """What the checkpoint of x stands for, from the definition, in 64 bits."""
    D = x.shape[-1]
    v = torch.nn.functional.pad(x.double(), (0, -D % 32))
    v = v.view(*x.shape[:-1], -1, 32)
    top = v.abs().amax(-1, keepdim=True)
    bad = ~torch.isfinite(top)
    top = torch.where(bad, torch.ones_like(top), top)
    e = torch.where(top > 0, torch.frexp(top).exponent - 7, -126).clamp(min=-126)
    s = torch.ldexp(torch.ones_like(top), e)
    q = torch.round(v / s).clamp(-127, 127) * s
    q = torch.where(bad.expand_as(q), torch.full_like(q, float("nan")), q)
    return q.flatten(-2)[..., :D]


def top_of_group(x):
    """max|x| of each element's group, as a tensor like x."""
    D = x.shape[-1]
    v = torch.nn.functional.pad(x.double(), (0, -D % 32)).view(*x.shape[:-1], -1, 32)
    return v.abs().amax(-1, keepdim=True).expand_as(v).flatten(-2)[..., :D]


def act64(z, act):
    if act == "relu2":
        return z.clamp(min=0) ** 2
    return torch.tanh(z) if act == "tanh" else torch.sigmoid(z) if act == "sigmoid" else z


def grad64(z, act):
    if act == "relu2":
        return 2 * z.clamp(min=0)
    if act == "tanh":
        return 1 / torch.cosh(z) ** 2
    if act == "sigmoid":
        return torch.sigmoid(z) * torch.sigmoid(-z)
    return torch.ones_like(z)


def slope(z, act, dz):
    """A bound of |act(z + d) - act(z)| for |d| <= dz."""
    if act == "relu2":
        return (2 * z.abs() + dz) * dz
    return dz


# --------------------------------------------------------------- checkpoints

@pytest.mark.parametrize("dt", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("rows,D", [(1, 1), (3, 31), (2, 32), (5, 40), (7, 33), (1, 2048), (257, 96), (64, 1000)])
def test_checkpoint_is_its_definition(cuda, dt, rows, D):
    from swiftrwkv_b200 import block as B
    x = rnd((rows, D), 1, DTYPES[dt])
    x[:, ::3] *= 1e-3
    ck = B.checkpoint8(x)
    assert ck.codes.shape == (rows, D) and ck.exps.shape == (rows, -(-D // 32))
    want = values64(x)
    got = B.checkpoint8Values(ck)
    assert got.dtype == x.dtype and torch.equal(got.double(), want)       # exact in every type
    assert torch.equal(B.checkpoint8Values(ck, dtype=torch.float32).double(), want)
    assert bool(((want - x.double()).abs() <= top_of_group(x) / 127.5).all())
    assert ck.nbytes == rows * (D + -(-D // 32))


def test_checkpoint_of_extremes(cuda):
    """Zeros, one huge value, the largest and smallest of the types, ties,
    infinities and NaN (their group stands for NaN, others are unharmed)."""
    from swiftrwkv_b200 import block as B
    for dt in DTYPES.values():
        f = torch.finfo(dt)
        x = torch.zeros(8, 96, device="cuda", dtype=dt)
        x[1, 5] = f.max
        x[2, 40] = f.tiny
        x[2, 41] = -f.smallest_normal
        x[3, :] = f.max
        x[4, :32] = torch.arange(32, device="cuda").to(dt) + 0.5      # top 31.5: ties at s = 1/4 do not occur
        x[4, 32:64] = torch.arange(32, device="cuda").to(dt) * 4 + 2  # top 126, s = 1: exact
        x[4, 64:] = torch.arange(32, device="cuda").to(dt) * 4 + 1.5  # ties to even at s = 1
        x[5, 33] = float("inf")
        x[6, 64] = float("nan")
        x[7, 1] = -float("inf")
        ck = B.checkpoint8(x)
        got, want = B.checkpoint8Values(ck, dtype=torch.float32), values64(x)
        assert torch.equal(torch.isnan(got), torch.isnan(want))
        assert torch.equal(torch.nan_to_num(got.double(), nan=7.0), torch.nan_to_num(want, nan=7.0))
        assert torch.isnan(got[5, 32:64]).all() and torch.isfinite(got[5, :32]).all() and torch.isfinite(got[5, 64:]).all()
    sub = torch.full((1, 32), 1e-42, device="cuda")                   # far below the smallest scale
    assert torch.equal(B.checkpoint8Values(B.checkpoint8(sub)), torch.zeros_like(sub))


@pytest.mark.parametrize("act", ["none", "relu2", "tanh", "sigmoid"])
@pytest.mark.parametrize("dt", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("rows,D", [(3, 31), (33, 96), (5, 200)])
def test_checkpoint_uses(cuda, act, dt, rows, D):
    """act(value) and dy * act'(value): elementary functions to 16 ulp of
    fp32 (twice over in a product), one rounding."""
    from swiftrwkv_b200 import block as B
    t = DTYPES[dt]
    x, dy = rnd((rows, D), 2, t, 3.0), rnd((rows, D), 3, t)
    ck = B.checkpoint8(x)
    v = values64(x)
    tiny = torch.finfo(t).tiny * u(t) * 2      # half a subnormal step
    y = act64(v, act)
    check(B.checkpoint8Values(ck, act), y, y.abs() * (u(t) + 16 * U32) + tiny, "value")
    for pre, z in ((ck, v), (x, x.double())):
        w = dy.double() * grad64(z, act)
        check(B.activationBackward(dy, pre, act), w, w.abs() * (u(t) + 32 * U32) + tiny, "gradient")


def test_activation_gradient_matches_differences(cuda):
    """act' against central differences of act, both the library's, fp32."""
    from swiftrwkv_b200 import block as B
    z = torch.linspace(-4, 4, 1024, device="cuda").view(32, 32)
    h = 2.0 ** -6
    for act in ("relu2", "tanh", "sigmoid"):
        # the library's act on exact inputs: projections with the identity would round; use the checkpoint of a grid
        zq = B.checkpoint8Values(B.checkpoint8(z))
        up, dn = (act64(zq.double() + s * h, act) for s in (1, -1))
        g = B.activationBackward(torch.ones_like(zq), zq, act)
        # central difference: exact for a square away from 0; h^2/6 max|act'''| (<= 2) elsewhere, h at relu's kink
        lim = 2 * h * h / 6 + 1e-5
        off = (g.double() - (up - dn) / (2 * h)).abs()
        near = zq.abs() <= h
        assert bool((off[~near] <= lim).all()) and bool((off[near] <= h + lim).all())


def test_activation_backward_may_write_over_dy(cuda):
    from swiftrwkv_b200 import _lib, block as B
    dy, z = rnd((65, 72), 5, torch.bfloat16), rnd((65, 72), 6, torch.bfloat16)
    want = B.activationBackward(dy, z, "tanh")
    buf = dy.clone()
    _lib.call("rwkv_act_backward", _lib.BF16, buf.data_ptr(), z.data_ptr(), None, None, 2, buf.data_ptr(), 65, 72,
              torch.cuda.current_stream().cuda_stream)
    assert torch.equal(buf, want)


# ----------------------------------------------------------------- layer norm

NORM_SIZES = [(1, 1), (1, 2048), (3, 7), (5, 64), (17, 96), (2, 768), (33, 1003), (4, 2560), (3, 4096), (2, 8200), (1, 10240),
              (2, 33000), (1003, 128)]


def norm64(x, w, b, eps):
    x = x.double()
    mean = x.mean(-1, keepdim=True)
    var = ((x - mean) ** 2).mean(-1, keepdim=True)
    rstd = 1 / torch.sqrt(var + eps)
    return (x - mean) * rstd * w.double() + b.double(), mean, rstd


@pytest.mark.parametrize("dt", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("rows,D", NORM_SIZES)
def test_layer_norm_forward(cuda, dt, rows, D):
    from swiftrwkv_b200 import block as B
    t = DTYPES[dt]
    x = (rnd((rows, D), 7) * 2 + 0.5).to(t)
    w, b = rnd((D,), 8) * 0.2 + 1, rnd((D,), 9) * 0.2
    eps = 1e-5
    y, mean, rstd, ck = B.layerNormForward(x, w, b, eps, checkpoint=True)
    y64, m64, r64 = norm64(x, w, b, eps)
    n = D + 16
    dm = n * U32 * x.double().abs().mean(-1, keepdim=True)           # error of the mean
    check(mean, m64[:, 0], dm[:, 0] + 2 * U32 * m64.abs()[:, 0], "mean")
    dev = (x.double() - m64).abs()
    # variance: terms off by 2 |d| dm + dm^2, the sum by n 2^-24; rstd by half its relative error
    dvar = (2 * dev * dm + dm * dm).mean(-1, keepdim=True) + n * U32 * (dev ** 2).mean(-1, keepdim=True)
    drel = 0.5 * dvar * r64 ** 2 * 1.01 + 8 * U32
    check(rstd, r64[:, 0], (r64 * drel)[:, 0], "rstd")
    tol = (w.double().abs() * r64 * (dm + dev * (drel + 4 * U32))) + 2 * U32 * (y64.abs() + b.double().abs())
    check(y, y64, tol * 1.01 + u(t) * (y64.abs() + tol), "y")
    assert torch.equal(B.checkpoint8Values(ck).double(), values64(x))
    y2, _, _, none = B.layerNormForward(x, w, b, eps)
    assert none is None and torch.equal(y2, y)


@pytest.mark.parametrize("kept", [False, True])
@pytest.mark.parametrize("dt", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("rows,D", NORM_SIZES)
def test_layer_norm_backward(cuda, dt, kept, rows, D):
    from swiftrwkv_b200 import block as B
    t = DTYPES[dt]
    x = (rnd((rows, D), 10) * 2 + 0.5).to(t)
    w, b = rnd((D,), 11) * 0.2 + 1, rnd((D,), 12)
    dy, dres = rnd((rows, D), 13, t), rnd((rows, D), 14, t)
    _, mean, rstd, ck = B.layerNormForward(x, w, b, checkpoint=True)
    dx, dw, db = B.layerNormBackward(dy, ck if kept else x, w, mean, rstd, dres=dres)
    xv = values64(x) if kept else x.double()
    m, r = mean.double()[:, None], rstd.double()[:, None]
    h = (xv - m) * r
    g = dy.double() * w.double()
    along, mg = (g * h).mean(1, keepdim=True), g.mean(1, keepdim=True)
    want = r * (g - mg - h * along) + dres.double()
    n = (D + 16) * U32
    hd = 3 * U32 * r * (xv.abs() + m.abs())                           # error of h
    tol = r * (g.abs() * 4 * U32 + n * g.abs().mean(1, keepdim=True) +
               h.abs() * (n * (g * h).abs().mean(1, keepdim=True) + (g.abs() * hd).mean(1, keepdim=True)) +
               hd * along.abs()) + 8 * U32 * (r * (g.abs() + mg.abs() + (h * along).abs()) + dres.double().abs())
    check(dx, want, tol * 1.01 + u(t) * (want.abs() + tol), "dx")
    k = (rows + 16) * U32
    check(dw, (dy.double() * h).sum(0), k * (dy.double() * h).abs().sum(0) + (dy.double().abs() * hd).sum(0) + 1e-38, "dw")
    check(db, dy.double().sum(0), k * dy.double().abs().sum(0) + 1e-38, "db")
    dx2, none, _ = B.layerNormBackward(dy, ck if kept else x, w, mean, rstd, dres=dres, params=False)
    assert none is None and torch.equal(dx2, dx)
    dx3, dw3, db3 = B.layerNormBackward(dy, ck if kept else x, w, mean, rstd, dres=dres)
    assert torch.equal(dx3, dx) and torch.equal(dw3, dw) and torch.equal(db3, db)   # deterministic


# on both sides of each length at which the kernels change their threads or
# their elements per thread: whole 16-byte vectors, and odd lengths
NORM_EDGES = [248, 256, 264, 512, 520, 768, 776, 1024, 1032, 1280, 1288, 1536, 1544, 2048, 2056, 2568, 4096, 4104, 5128,
              8192, 10248, 12288, 12296, 16392, 32768, 32776,
              255, 257, 511, 513, 1023, 1025, 1537, 2047, 2049, 4095, 4097, 6143, 6145, 10239, 10241]


@pytest.mark.parametrize("dt", ["f32", "bf16"])
@pytest.mark.parametrize("D", NORM_EDGES)
def test_layer_norm_around_the_length_classes(cuda, dt, D):
    test_layer_norm_forward(cuda, dt, 3, D)
    for kept in (False, True):
        test_layer_norm_backward(cuda, dt, kept, 3, D)


@pytest.mark.parametrize("dt", ["f32", "bf16"])
@pytest.mark.parametrize("D", [96, 250, 1003, 2056, 2560, 6001, 10241, 33000])
def test_layer_norm_may_write_over_its_inputs(cuda, dt, D):
    """y over x; dx over dy or dres (rwkv_cuda.h); more rows than resident blocks."""
    from swiftrwkv_b200 import _lib, block as B
    t, rows = DTYPES[dt], 1301
    code, st = B._DT[t], torch.cuda.current_stream().cuda_stream
    x, dy, dres = rnd((rows, D), 51, t), rnd((rows, D), 52, t), rnd((rows, D), 53, t)
    w, b = rnd((D,), 54) * 0.2 + 1, rnd((D,), 55)
    y, mean, rstd, ck = B.layerNormForward(x, w, b, checkpoint=True)
    buf, codes, exps = x.clone(), torch.empty_like(ck.codes), torch.empty_like(ck.exps)
    _lib.call("rwkv_layer_norm_forward", code, buf.data_ptr(), _lib.F32, w.data_ptr(), b.data_ptr(), 1e-5, buf.data_ptr(),
              None, None, codes.data_ptr(), exps.data_ptr(), rows, D, st)
    assert torch.equal(buf, y) and torch.equal(codes, ck.codes) and torch.equal(exps, ck.exps)
    n = _lib.lib().rwkv_layer_norm_backward_workspace_size(rows, D)
    ws = torch.empty(n, device="cuda", dtype=torch.uint8)
    for kept in (False, True):
        dx, dw, db = B.layerNormBackward(dy, ck if kept else x, w, mean, rstd, dres=dres)
        for over in ("dy", "dres"):
            a, r = dy.clone(), dres.clone()
            out, gw, gb = a if over == "dy" else r, torch.empty_like(w), torch.empty_like(w)
            _lib.call("rwkv_layer_norm_backward", code, a.data_ptr(), None if kept else x.data_ptr(),
                      ck.codes.data_ptr() if kept else None, ck.exps.data_ptr() if kept else None, _lib.F32, w.data_ptr(),
                      mean.data_ptr(), rstd.data_ptr(), r.data_ptr(), out.data_ptr(), gw.data_ptr(), gb.data_ptr(), rows, D,
                      ws.data_ptr(), n, st)
            assert torch.equal(out, dx) and torch.equal(gw, dw) and torch.equal(gb, db)


@pytest.mark.parametrize("dt", ["f32", "bf16"])
@pytest.mark.parametrize("rows,D", [(1301, 1003), (1301, 250), (1300, 1002), (999, 2412), (2500, 33), (700, 3001), (640, 8003)])
def test_layer_norm_of_odd_lengths_and_many_rows(cuda, dt, rows, D):
    """Rows that share a 16-byte vector with their neighbours, several per block."""
    test_layer_norm_forward(cuda, dt, rows, D)
    for kept in (False, True):
        test_layer_norm_backward(cuda, dt, kept, rows, D)


@pytest.mark.parametrize("dt", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("D", [9, 63, 1003, 2412, 5003])
def test_layer_norm_rows_do_not_touch_their_neighbours(cuda, dt, D):
    """Every third row NaN or infinite: the rows between give what they give alone;
    and what lies behind the last row stays as it was."""
    from swiftrwkv_b200 import _lib, block as B
    t, rows = DTYPES[dt], 700
    code, st = B._DT[t], torch.cuda.current_stream().cuda_stream
    x, dy, dres = rnd((rows, D), 61, t), rnd((rows, D), 62, t), rnd((rows, D), 63, t)
    w, b = rnd((D,), 64) * 0.2 + 1, rnd((D,), 65)
    y, mean, rstd, ck = B.layerNormForward(x, w, b, checkpoint=True)
    good = torch.arange(rows, device="cuda") % 3 != 1
    bad_x, bad_dy, bad_dres = x.clone(), dy.clone(), dres.clone()
    bad_x[1::6], bad_x[4::6] = float("nan"), float("inf")
    bad_dy[1::3], bad_dres[1::3] = float("inf"), float("nan")
    y2, mean2, rstd2, ck2 = B.layerNormForward(bad_x, w, b, checkpoint=True)
    assert torch.equal(y2[good], y[good]) and torch.equal(mean2[good], mean[good]) and torch.equal(rstd2[good], rstd[good])
    assert torch.equal(ck2.codes[good], ck.codes[good]) and torch.equal(ck2.exps[good], ck.exps[good])
    assert bool((ck2.exps[~good] == 255).all()) and bool(torch.isnan(y2[~good]).all())
    for kept in (False, True):
        want = B.layerNormBackward(dy, ck if kept else x, w, mean, rstd, dres=dres, params=False)[0]
        got = B.layerNormBackward(bad_dy, ck2 if kept else bad_x, w, mean2, rstd2, dres=bad_dres, params=False)[0]
        assert torch.equal(got[good], want[good]) and bool(torch.isnan(got[~good]).all())
    # outputs in the middle of larger buffers
    n, pad = rows * D, 64
    yb, xb = torch.full((n + pad,), 7.0, device="cuda", dtype=t), torch.full((n + pad,), 7.0, device="cuda", dtype=t)
    cb = torch.full((n + pad,), 77, device="cuda", dtype=torch.int8)
    eb = torch.full((ck.exps.numel() + pad,), 77, device="cuda", dtype=torch.uint8)
    _lib.call("rwkv_layer_norm_forward", code, x.data_ptr(), _lib.F32, w.data_ptr(), b.data_ptr(), 1e-5, yb.data_ptr(),
              None, None, cb.data_ptr(), eb.data_ptr(), rows, D, st)
    _lib.call("rwkv_layer_norm_backward", code, dy.data_ptr(), x.data_ptr(), None, None, _lib.F32, w.data_ptr(),
              mean.data_ptr(), rstd.data_ptr(), dres.data_ptr(), xb.data_ptr(), None, None, rows, D, None, 0, st)
    assert torch.equal(yb[:n].view(rows, D), y) and bool((yb[n:] == 7).all())
    assert torch.equal(cb[:n].view(rows, D), ck.codes) and bool((cb[n:] == 77).all())
    assert torch.equal(eb[:ck.exps.numel()].view_as(ck.exps), ck.exps) and bool((eb[ck.exps.numel():] == 77).all())
    assert torch.equal(xb[:n].view(rows, D), B.layerNormBackward(dy, x, w, mean, rstd, dres=dres, params=False)[0])
    assert bool((xb[n:] == 7).all())


@pytest.mark.parametrize("dt", ["f32", "bf16"])
def test_layer_norm_of_misaligned_rows(cuda, dt):
    """Tensors that start off a 16-byte boundary give what aligned copies give, as
    far as the order of sums allows."""
    from swiftrwkv_b200 import block as B
    t = DTYPES[dt]
    for rows, D in ((9, 64), (700, 1003), (40, 2560), (5, 5003)):
        buf = rnd((3, rows * D + 1), 66, t)
        x, dy, dres = (buf[i, 1:].view(rows, D) for i in range(3))
        assert x.data_ptr() % 16
        w, b = rnd((D,), 67) * 0.2 + 1, rnd((D,), 68)
        y, mean, rstd, ck = B.layerNormForward(x, w, b, checkpoint=True)
        yc, mc, rc, cc = B.layerNormForward(x.clone(), w, b, checkpoint=True)
        # the sums' orders differ by n 2^-24 of the sum of absolute terms each, carried
        # through as in test_layer_norm_forward; twice, and a rounding to t on both sides
        n = (D + 16) * U32
        m64, r64 = norm64(x, w, b, 1e-5)[1:]
        dm = n * x.double().abs().mean(-1, keepdim=True)
        dev = (x.double() - m64).abs()
        drel = 0.5 * ((2 * dev * dm + dm * dm).mean(-1, keepdim=True) + n * (dev ** 2).mean(-1, keepdim=True)) * r64 ** 2 * 1.01 + 8 * U32
        tol = w.double().abs() * r64 * (dm + dev * (drel + 4 * U32)) + 2 * U32 * (yc.double().abs() + 2 * b.double().abs())
        check(y, yc.double(), 2 * (tol * 1.01 + u(t) * (yc.double().abs() + tol)), "y")
        assert torch.equal(ck.codes, cc.codes) and torch.equal(ck.exps, cc.exps)
        dx, dw, db = B.layerNormBackward(dy, x, w, mc, rc, dres=dres)
        m, r = mc.double()[:, None], rc.double()[:, None]
        h, g = (x.double() - m) * r, dy.double() * w.double()
        along, mg = (g * h).mean(1, keepdim=True), g.mean(1, keepdim=True)
        want = r * (g - mg - h * along) + dres.double()
        hd = 3 * U32 * r * (x.double().abs() + m.abs())
        tol = r * (g.abs() * 4 * U32 + n * g.abs().mean(1, keepdim=True) +
                   h.abs() * (n * (g * h).abs().mean(1, keepdim=True) + (g.abs() * hd).mean(1, keepdim=True)) +
                   hd * along.abs()) + 8 * U32 * (r * (g.abs() + mg.abs() + (h * along).abs()) + dres.double().abs())
        check(dx, want, tol * 1.01 + u(t) * (want.abs() + tol), "dx")


def test_layer_norm_gradient_matches_differences(cuda):
    """The gradients against central differences of the forward in fp32: 1e-2
    of the largest gradient at a step of 2^-6 (the forward's own error,
    about 1e-6, divided by the step, and the third derivative)."""
    from swiftrwkv_b200 import block as B
    x, w, b, dy = rnd((4, 24), 15), rnd((24,), 16) * 0.2 + 1, rnd((24,), 17), rnd((4, 24), 18)
    f = lambda: (B.layerNormForward(x, w, b)[0].double() * dy.double()).sum()
    _, mean, rstd, _ = B.layerNormForward(x, w, b)
    grads = B.layerNormBackward(dy, x, w, mean, rstd)
    for p, g in zip((x, w, b), grads):
        flat, gf = p.view(-1), g.reshape(-1)
        for i in range(0, flat.numel(), 7):
            keep = float(flat[i])
            flat[i] = keep + 2.0 ** -6
            up = f()
            flat[i] = keep - 2.0 ** -6
            dn = f()
            flat[i] = keep
            assert abs(float(up - dn) * 2 ** 5 - float(gf[i])) < 1e-2 * float(g.abs().max())


def test_layer_norm_constant_rows_and_nan(cuda):
    """A constant row (variance 0) gives bias and finite gradients; a NaN or an
    infinity stays in its row."""
    from swiftrwkv_b200 import block as B
    x = rnd((6, 96), 19, torch.bfloat16)
    x[1] = 3.0
    x[3, 7] = float("nan")
    x[4, 50] = float("inf")
    w, b, dy = rnd((96,), 20), rnd((96,), 21), rnd((6, 96), 22, torch.bfloat16)
    y, mean, rstd, ck = B.layerNormForward(x, w, b, checkpoint=True)
    assert torch.equal(y[1], b.to(torch.bfloat16))
    assert torch.isnan(y[3]).all() and torch.isfinite(y[[0, 1, 2, 5]]).all() and torch.isnan(y[4]).any()
    dx, dw, _ = B.layerNormBackward(dy, x, w, mean, rstd)
    assert torch.isfinite(dx[[0, 1, 2, 5]]).all() and torch.isnan(dx[3]).all()
    assert torch.isnan(dw).any()


def test_layer_norm_far_from_zero(cuda):
    """Rows whose mean is large against their spread: a constant row gives the
    bias exactly, also at 1000 (its mean is exact, x - mean is 0), and its
    gradient has no part along h; a row at 1000 with spread 1 keeps the accuracy
    of the fp32 mean, 1000 2^-24 per rounding, 8 of them."""
    from swiftrwkv_b200 import block as B
    for D in (256, 2048, 2560, 100):
        x = torch.full((4, D), 1000.0, device="cuda")
        x[2:] += rnd((2, D), 130)
        w, b, dy = rnd((D,), 131), rnd((D,), 132), rnd((4, D), 133)
        y, mean, rstd, _ = B.layerNormForward(x, w, b)
        assert torch.equal(mean[:2], x[:2, 0]) and torch.equal(y[:2], b.expand(2, D))
        y64, m64, r64 = norm64(x, w, b, 1e-5)
        tol = 8 * 1000 * U32 * (w.double().abs() * r64 + 1)
        check(y[2:], y64[2:], (tol * (1 + (y64 - b.double()).abs()))[2:], "y")
        dx, _, _ = B.layerNormBackward(dy, x, w, mean, rstd, params=False)
        g = (dy * w).double()
        want = rstd.double()[:2, None] * (g - g.mean(1, keepdim=True))[:2]
        n = (D + 16) * U32
        check(dx[:2], want, rstd.double()[:2, None] * n * (g.abs() + g.abs().mean(1, keepdim=True))[:2], "dx")


def test_layer_norm_types_and_views(cuda):
    """Parameters in 16 bits, non-contiguous and misaligned inputs, leading
    dimensions, no rows."""
    from swiftrwkv_b200 import block as B
    x, w, b = rnd((2, 3, 64), 23, torch.bfloat16), rnd((64,), 24, torch.bfloat16), rnd((64,), 25, torch.bfloat16)
    y, mean, rstd, _ = B.layerNormForward(x, w, b)
    ref, _, _, _ = B.layerNormForward(x, w.float(), b.float())
    assert mean.shape == (2, 3) and torch.equal(y, ref)
    dy = rnd((2, 3, 64), 26, torch.bfloat16)
    _, dw, db = B.layerNormBackward(dy, x, w, mean, rstd)
    _, dw32, db32 = B.layerNormBackward(dy, x, w.float(), mean, rstd)
    assert dw.dtype == torch.bfloat16 and torch.equal(dw, dw32.to(dw.dtype)) and torch.equal(db, db32.to(db.dtype))
    big = rnd((2, 65, 3), 27, torch.bfloat16)
    v = big[:, :64].transpose(1, 2)                       # strided
    assert torch.equal(B.layerNormForward(v, w, b)[0], B.layerNormForward(v.contiguous(), w, b)[0])
    flat = rnd((6 * 64 + 1,), 28, torch.bfloat16)
    odd = flat[1:].view(6, 64)                            # 2-byte aligned rows take the scalar kernel
    n = 64 + 16
    a, m = B.layerNormForward(odd, w, b)[0], B.layerNormForward(odd.clone(), w, b)[0]
    assert bool(((a.double() - m.double()).abs() <= (2 * u(torch.bfloat16) + n * 16 * U32) * (m.double().abs() + 1)).all())
    y0, mean0, _, ck0 = B.layerNormForward(x[:, :0], w, b, checkpoint=True)
    assert y0.shape == (2, 0, 64) and mean0.shape == (2, 0) and ck0.codes.shape == (2, 0, 64)
    dx0, dw0, db0 = B.layerNormBackward(dy[:, :0], x[:, :0], w, mean0, mean0)
    assert dx0.shape == (2, 0, 64) and not dw0.any() and not db0.any()


# ---------------------------------------------------------------- projections

PROJ_SIZES = [(1, 8, 8), (1, 2048, 2048), (2, 24, 72), (3, 8192, 264), (7, 104, 2048), (16, 256, 1000), (17, 64, 64), (33, 520, 136),
              (64, 2048, 4096), (128, 128, 64), (129, 264, 72), (300, 96, 2048), (1000, 2048, 96), (257, 1032, 520),
              (2051, 768, 768)]


def proj_sums(a, b):
    """sum over the last dim of a b^T, and of |a| |b|^T, in 64 bits."""
    a, b = a.double(), b.double()
    return a @ b.t(), a.abs() @ b.abs().t()


@pytest.mark.parametrize("dt", ["bf16", "f16"])
@pytest.mark.parametrize("rows,OUT,IN", PROJ_SIZES)
def test_projection_forward(cuda, dt, rows, OUT, IN):
    from swiftrwkv_b200 import block as B
    t = DTYPES[dt]
    x, w = rnd((rows, IN), 30, t), rnd((OUT, IN), 31, t, IN ** -0.5)
    z0, s0 = proj_sums(x, w)
    y, none = B.projectionForward(x, w)
    assert none is None and y.dtype == t
    check(y, z0, TC * s0 + u(t) * (z0.abs() + TC * s0), "plain")
    f, _ = B.projectionForward(x, w, out_dtype=torch.float32)
    check(f, z0, TC * s0 + U32 * z0.abs(), "fp32 out")
    bias, res = rnd((OUT,), 32), rnd((rows, OUT), 33, t)
    z, dz = z0 + bias.double(), TC * (s0 + bias.double().abs())
    for act in ("none", "relu2", "tanh", "sigmoid"):
        want = act64(z, act) + res.double()
        tol = slope(z, act, dz) + 32 * U32 * (act64(z, act).abs() + want.abs())
        y, ck = B.projectionForward(x, w, bias, act, res, checkpoint=True)
        check(y, want, tol + u(t) * (want.abs() + tol), act)
        y2, pre = B.projectionForward(x, w, bias, act, res, preactivation=True)
        assert torch.equal(y2, y)
        check(pre, z, dz + u(t) * (z.abs() + dz), "z")
        # a code stands for z up to a 127.5th of its group's largest, both as the kernel saw them
        v = B.checkpoint8Values(ck, dtype=torch.float32)
        check(v, z, (top_of_group(z) + top_of_group(dz)) / 127.5 + top_of_group(dz), "checkpoint")
    h, _ = B.projectionForward(x, w, bias.to(t), "none", res)
    zb = z0 + bias.to(t).double() + res.double()
    tb = TC * s0 + 4 * U32 * (z0.abs() + 1 + res.double().abs() + bias.double().abs())
    check(h, zb, tb + u(t) * (zb.abs() + tb), "16-bit bias")
    f, _ = B.projectionForward(x, w, bias, "sigmoid", res.float(), out_dtype=torch.float32)
    want = act64(z, "sigmoid") + res.double()
    check(f, want, dz + 32 * U32 * (1 + want.abs()), "fp32 out with epilogue")


@pytest.mark.parametrize("dt", ["bf16", "f16"])
@pytest.mark.parametrize("rows,OUT,IN", PROJ_SIZES)
def test_projection_backward_input(cuda, dt, rows, OUT, IN):
    from swiftrwkv_b200 import block as B
    t = DTYPES[dt]
    dy, w = rnd((rows, OUT), 34, t), rnd((OUT, IN), 35, t, OUT ** -0.5)
    g, s = proj_sums(dy, w.t())
    dx = B.projectionBackwardInput(dy, w)
    check(dx, g, TC * s + u(t) * (g.abs() + TC * s), "plain")
    z, add = rnd((rows, IN), 36, t), rnd((rows, IN), 37, t)
    ck = B.checkpoint8(z)
    for act in ("none", "relu2", "tanh", "sigmoid"):
        for pre, zv in ((z, z.double()), (ck, values64(z))):
            d = grad64(zv, act)
            want = g * d + add.double()
            tol = TC * s * d.abs() + 64 * U32 * ((g * d).abs() + want.abs())
            got = B.projectionBackwardInput(dy, w, pre=pre, act=act, addend=add)
            check(got, want, tol + u(t) * (want.abs() + tol), act)
    f = B.projectionBackwardInput(dy, w, pre=ck, act="relu2", addend=add.float(), out_dtype=torch.float32)
    d = grad64(values64(z), "relu2")
    want = g * d + add.double()
    check(f, want, TC * s * d + 64 * U32 * ((g * d).abs() + want.abs() + add.double().abs()), "fp32 out")


@pytest.mark.parametrize("dt", ["bf16", "f16"])
@pytest.mark.parametrize("rows,OUT,IN", PROJ_SIZES)
def test_projection_backward_weight(cuda, dt, rows, OUT, IN):
    from swiftrwkv_b200 import block as B
    t = DTYPES[dt]
    dy, x = rnd((rows, OUT), 38, t), rnd((rows, IN), 39, t)
    want, s = proj_sums(dy.t(), x.t())
    dw, db = B.projectionBackwardWeight(dy, x, bias=True)
    check(dw, want, TC * s + u(t) * (want.abs() + TC * s), "dense")
    dbs = dy.double().abs().sum(0)
    check(db, dy.double().sum(0), (rows + 16) * U32 * dbs + 1e-38, "db")
    none, db2 = B.projectionBackwardWeight(dy, None, bias=True)
    assert none is None and torch.equal(db2, db)
    ck = B.checkpoint8(x)
    v = values64(x)
    want, s = proj_sums(dy.t(), v.t())
    f, none = B.projectionBackwardWeight(dy, ck, out_dtype=torch.float32)
    assert none is None
    check(f, want, TC * s + U32 * want.abs(), "checkpoint, fp32 out")     # the operand is exact
    for act in ("relu2", "tanh", "sigmoid"):
        for op, zv in ((ck, v), (x, x.double())):
            want, s = proj_sums(dy.t(), act64(zv, act).t())
            # each operand value rounded once: by u(t) of it, or by half of the
            # subnormal spacing tiny eps where it is below tiny (fp16 squares are)
            sub = torch.finfo(t).tiny * torch.finfo(t).eps / 2 * dy.double().abs().sum(0)[:, None]
            tol = (u(t) + 16 * U32 + TC) * s + sub
            got, _ = B.projectionBackwardWeight(dy, op, act=act)
            check(got, want, tol + u(t) * (want.abs() + tol), act)


@pytest.mark.parametrize("dt", ["bf16", "f16"])
@pytest.mark.parametrize("rows,OUT,IN", [(1018, 3000, 6544), (5, 24, 20000), (40, 64, 20000), (200, 20000, 136), (20000, 104, 264)])
def test_projection_of_long_sums(cuda, dt, rows, OUT, IN):
    """fp32 results of sums of up to 20000 terms.  The tensor core adds 16 products
    to its fp32 accumulator at a time and cuts off what does not fit, at most 2^-23
    of the running sum per step: K / 16 steps are off by at most (K / 16 + 1) 2^-23
    sum|terms| (one step more where splits are joined), and the result is fp32."""
    from swiftrwkv_b200 import block as B
    t = DTYPES[dt]
    x, w, dy = rnd((rows, IN), 71, t), rnd((OUT, IN), 72, t, IN ** -0.5), rnd((rows, OUT), 73, t)

    def compare(got, a, b, what):
        z, s0 = proj_sums(a, b)
        check(got, z, (a.shape[1] / 16 + 1) * 2.0 ** -23 * s0 + U32 * z.abs(), what)

    compare(B.projectionForward(x, w, out_dtype=torch.float32)[0], x, w, "y")
    compare(B.projectionBackwardInput(dy, w, out_dtype=torch.float32), dy, w.t(), "dx")
    dw, db = B.projectionBackwardWeight(dy, x, bias=True, out_dtype=torch.float32)
    compare(dw, dy.t(), x.t(), "dw")
    check(db, dy.double().sum(0), (rows + 16) * U32 * dy.double().abs().sum(0), "db")


def test_projection_results_repeat(cuda):
    """Split products and column sums are joined in a fixed order."""
    from swiftrwkv_b200 import block as B
    x, w, dy = rnd((700, 2048), 40, torch.bfloat16), rnd((96, 2048), 41, torch.bfloat16), rnd((700, 96), 42, torch.bfloat16)
    first = (B.projectionForward(x, w)[0], B.projectionBackwardInput(dy, w), *B.projectionBackwardWeight(dy, x, bias=True))
    for _ in range(3):
        again = (B.projectionForward(x, w)[0], B.projectionBackwardInput(dy, w),
                 *B.projectionBackwardWeight(dy, x, bias=True))
        assert all(torch.equal(a, b) for a, b in zip(first, again))


@pytest.mark.parametrize("rows,OUT,IN", [(5, 72, 64), (200, 264, 1032)])
def test_projection_leaves_what_lies_behind_its_outputs(cuda, rows, OUT, IN):
    """Outputs inside larger buffers: nothing past their end is written."""
    from swiftrwkv_b200 import _lib
    t = torch.bfloat16
    x, w = rnd((rows, IN), 43, t), rnd((OUT, IN), 44, t)
    n, groups = rows * OUT, rows * -(-OUT // 32)
    y = torch.full((n + 4096,), 7.0, device="cuda", dtype=t)
    z = torch.full((n + 4096,), 7.0, device="cuda", dtype=t)
    codes = torch.full((n + 4096,), 7, device="cuda", dtype=torch.int8)
    exps = torch.full((groups + 4096,), 7, device="cuda", dtype=torch.uint8)
    nb = _lib.lib().rwkv_projection_forward_workspace_size(rows, OUT, IN)
    ws = torch.full((nb + 4096,), 7, device="cuda", dtype=torch.uint8)
    _lib.call("rwkv_projection_forward", _lib.BF16, x.data_ptr(), w.data_ptr(), 0, None, 1, _lib.BF16, None, y.data_ptr(),
              z.data_ptr(), codes.data_ptr(), exps.data_ptr(), rows, OUT, IN, ws.data_ptr(), nb,
              torch.cuda.current_stream().cuda_stream)
    for buf, k in ((y, n), (z, n), (codes, n), (exps, groups), (ws, nb)):
        assert bool((buf[k:] == 7).all())


def test_projection_residual_may_be_the_output(cuda):
    from swiftrwkv_b200 import _lib, block as B
    for rows, OUT, IN in ((64, 256, 4096), (1000, 512, 128), (1, 512, 512)):
        x, w, res = rnd((rows, IN), 45, torch.float16), rnd((OUT, IN), 46, torch.float16, 0.02), rnd((rows, OUT), 47, torch.float16)
        want, _ = B.projectionForward(x, w, residual=res)
        nb = _lib.lib().rwkv_projection_forward_workspace_size(rows, OUT, IN)
        ws = torch.empty(max(nb, 16), device="cuda", dtype=torch.uint8)
        buf = res.clone()
        _lib.call("rwkv_projection_forward", _lib.F16, x.data_ptr(), w.data_ptr(), 0, None, 0, _lib.F16, buf.data_ptr(),
                  buf.data_ptr(), None, None, None, rows, OUT, IN, ws.data_ptr(), nb, torch.cuda.current_stream().cuda_stream)
        assert torch.equal(buf, want)


def test_projection_views_and_empty_batches(cuda):
    from swiftrwkv_b200 import block as B
    t = torch.bfloat16
    big, wb = rnd((3, 5, 2 * 64 + 3), 48, t), rnd((72, 65), 49, t)
    x, w = big[..., 1:65], wb[:, 1:]                       # strided, misaligned
    y, _ = B.projectionForward(x, w)
    assert y.shape == (3, 5, 72) and torch.equal(y, B.projectionForward(x.contiguous(), w.contiguous())[0])
    flat = rnd((64 * 64 + 3,), 50, t)[3:].view(64, 64)     # contiguous at an odd address
    assert torch.equal(B.projectionForward(flat, w)[0], B.projectionForward(flat.clone(), w)[0])
    v = rnd((64,), 51, t)                                  # no leading dimension
    assert torch.equal(B.projectionForward(v, w)[0], B.projectionForward(v[None], w)[0][0])
    y0, ck0 = B.projectionForward(x[:0], w, checkpoint=True)
    assert y0.shape == (0, 5, 72) and ck0.exps.shape == (0, 5, 3)
    assert B.projectionBackwardInput(y0, w).shape == (0, 5, 64)
    dw0, db0 = B.projectionBackwardWeight(y0, x[:0], bias=True)
    assert dw0.shape == (72, 64) and not dw0.any() and not db0.any()


def test_projection_of_infinities_and_nan(cuda):
    """A NaN or an infinity of x stays in its row, one of w in its column."""
    from swiftrwkv_b200 import block as B
    t = torch.bfloat16
    x, w = rnd((200, 136), 52, t), rnd((72, 136), 53, t)
    x[5, 100] = float("nan")
    x[150, 3] = float("inf")
    w[60, 7] = float("nan")
    for act in ("none", "relu2", "tanh", "sigmoid"):
        y, ck = B.projectionForward(x, w, act=act, checkpoint=True)
        rows = torch.ones(200, dtype=torch.bool, device="cuda")
        rows[[5, 150]] = False
        cols = torch.ones(72, dtype=torch.bool, device="cuda")
        cols[60] = False
        assert torch.isnan(y[5]).all() and torch.isnan(y[:, 60]).all()
        assert torch.isfinite(y[rows][:, cols]).all()
        v = B.checkpoint8Values(ck)
        assert torch.isnan(v[5]).all() and torch.isnan(v[:, 32:64]).all() and torch.isfinite(v[rows][:, :32]).all()
    dy = rnd((200, 72), 54, t)
    dx = B.projectionBackwardInput(dy, w[:, :], pre=x, act="relu2")
    assert torch.isnan(dx[:, 7]).all()
    dw, _ = B.projectionBackwardWeight(dy, x)
    assert torch.isnan(dw[:, 100]).all() and torch.isfinite(dw[:, 4:100]).all()


def test_python_refusals_on_cuda_tensors(cuda):
    from swiftrwkv_b200 import block as B
    x, w = rnd((4, 64), 55, torch.bfloat16), rnd((72, 64), 56, torch.bfloat16)
    bad = [lambda: B.projectionForward(x.float(), w), lambda: B.projectionForward(x, w.half()),
           lambda: B.projectionForward(x, w[:, :56]), lambda: B.projectionForward(x[:, :60], w[:, :60]),
           lambda: B.projectionForward(x, w, residual=x), lambda: B.projectionForward(x, w, out_dtype=torch.float16),
           lambda: B.projectionForward(x, w, bias=torch.zeros(71, device="cuda")),
           lambda: B.projectionForward(x, w, checkpoint=True, preactivation=True),
           lambda: B.projectionForward(x, w, bias=torch.zeros(72)),
           lambda: B.projectionBackwardInput(rnd((4, 72), 1, torch.bfloat16), w, act="tanh"),
           lambda: B.projectionBackwardInput(x, w), lambda: B.projectionBackwardWeight(x, w),
           lambda: B.layerNormForward(x, torch.ones(63, device="cuda"), torch.zeros(64, device="cuda")),
           lambda: B.layerNormForward(x, torch.ones(64, device="cuda"), torch.zeros(64, device="cuda").half()),
           lambda: B.layerNormForward(x.double(), torch.ones(64, device="cuda"), torch.zeros(64, device="cuda")),
           lambda: B.layerNormBackward(x, x.half(), torch.ones(64, device="cuda"), *torch.zeros(2, 4, device="cuda")),
           lambda: B.layerNormBackward(x, x, torch.ones(64, device="cuda"), *torch.zeros(2, 5, device="cuda")),
           lambda: B.activationBackward(x, x[:2], "tanh"), lambda: B.checkpoint8(x.to(torch.int8)),
           lambda: B.activationBackward(x, B.Checkpoint8(x.to(torch.int8), torch.zeros(4, 3, dtype=torch.uint8, device="cuda"),
                                                         x.dtype), "tanh")]
    for i, f in enumerate(bad):
        with pytest.raises(ValueError):
            f()
            pytest.fail(f"call {i} was taken")


# ------------------------------------------------- streams, graphs, together

def test_two_streams_at_once(cuda):
    """Calls on two streams, each with its own workspace, agree with calls made
    one after the other."""
    from swiftrwkv_b200 import block as B
    t = torch.bfloat16
    cases = [(rnd((700, 1024), s, t), rnd((256, 1024), s + 9, t), rnd((700, 256), s + 17, t)) for s in (60, 61)]
    def work(x, w, dy):
        y, ck = B.projectionForward(x, w, act="tanh", checkpoint=True)
        return y, B.activationBackward(dy, ck, "tanh"), B.projectionBackwardInput(dy, w), *B.projectionBackwardWeight(dy, x, bias=True)
    want = [work(*c) for c in cases]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    got = [[], []]
    for _ in range(5):
        for k, s in enumerate(streams):
            with torch.cuda.stream(s):
                got[k].append(work(*cases[k]))
    torch.cuda.synchronize()
    for k in range(2):
        for g in got[k]:
            assert all(torch.equal(a, b) for a, b in zip(g, want[k]))


def test_captured_calls_replay_on_new_inputs(cuda):
    """The explicit calls captured into two graphs, replayed in turn with new
    inputs in the captured buffers."""
    from swiftrwkv_b200 import block as B
    t = torch.bfloat16
    w1, w2 = rnd((512, 256), 70, t, 0.06), rnd((256, 512), 71, t, 0.06)
    g, b = rnd((256,), 72) * 0.1 + 1, rnd((256,), 73)
    def step(x, dy):
        h, mean, rstd, ckx = B.layerNormForward(x, g, b, checkpoint=True)
        k, ck = B.projectionForward(h, w1, act="relu2", checkpoint=True)
        y, _ = B.projectionForward(k, w2, residual=x)
        dz = B.projectionBackwardInput(dy, w2, pre=ck, act="relu2")
        dw2, _ = B.projectionBackwardWeight(dy, ck, act="relu2")
        dw1, db1 = B.projectionBackwardWeight(dz, h, bias=True)
        dh = B.projectionBackwardInput(dz, w1)
        return [y, dw1, db1, dw2, *B.layerNormBackward(dh, ckx, g, mean, rstd, dres=dy)]
    bufs, graphs = [], []
    for rows in (40, 300):
        x, dy = rnd((rows, 256), 74, t), rnd((rows, 256), 75, t)
        s = torch.cuda.Stream()
        s.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(s):
            step(x, dy)
        torch.cuda.current_stream().wait_stream(s)
        gr = torch.cuda.CUDAGraph()
        with torch.cuda.graph(gr):
            out = step(x, dy)
        bufs.append((x, dy, out))
        graphs.append(gr)
    for seed in (80, 81):
        for k, rows in enumerate((40, 300)):
            bufs[k][0].copy_(rnd((rows, 256), seed, t))
            bufs[k][1].copy_(rnd((rows, 256), seed + 10, t))
            graphs[k].replay()
        for k in range(2):
            x, dy, out = bufs[k]
            assert all(torch.equal(a, c) for a, c in zip(out, step(x, dy)))


def test_differentiable_forms_refuse_capture(cuda):
    from swiftrwkv_b200 import block as B
    x = rnd((4, 64), 76, torch.bfloat16).requires_grad_(True)
    w, b = torch.ones(64, device="cuda"), torch.zeros(64, device="cuda")
    B.layerNorm(x.detach(), w, b)
    gr = torch.cuda.CUDAGraph()
    with torch.cuda.graph(gr):
        with pytest.raises(ValueError, match="capture"):
            B.layerNorm(x, w, b)
        y = B.layerNorm(x.detach(), w, b)       # nothing is recorded: taken
    gr.replay()
    assert torch.equal(y, B.layerNorm(x.detach(), w, b))


def block_run(B, x, p, checkpoint):
    """ln -> low-rank branch (tanh, sigmoid with bias) -> cmix projections with
    the residual, as a block runs them."""
    h = B.layerNorm(x, p["g"], p["b"], checkpoint=checkpoint)
    d = B.projection(h, p["down"], act="tanh", checkpoint=checkpoint)
    s = B.projection(d, p["up"], bias=p["up_b"], act="sigmoid", residual=h, checkpoint=checkpoint)
    return B.channelMix(s, p["key"], p["value"], residual=x, checkpoint=checkpoint)


class Block64:
    """The same operators in 64 bits under torch's autograd."""
    @staticmethod
    def layerNorm(x, g, b, checkpoint):
        return torch.nn.functional.layer_norm(x, x.shape[-1:], g, b, 1e-5)

    @staticmethod
    def projection(x, w, bias=None, act="none", residual=None, checkpoint=False):
        z = x @ w.t()
        z = act64(z if bias is None else z + bias, act)
        return z if residual is None else z + residual

    @staticmethod
    def channelMix(x, key, value, residual=None, checkpoint=True):
        return torch.relu(x @ key.t()) ** 2 @ value.t() + residual


@pytest.mark.parametrize("checkpoint", [False, True])
@pytest.mark.parametrize("rows", [1, 37, 600])
def test_block_run_and_its_gradients(cuda, checkpoint, rows):
    """Outputs and every gradient of a run of the operators against the same
    run in 64 bits.  In the 2-norm: about ten roundings to bf16 along the
    longest path, each at most 2^-8 and of either sign, sqrt(10) 2^-8 = 1.3 %,
    bound 4 %; with checkpoints four activations are read back with an error
    of up to a 128th of their group's largest, about 1 % each in the 2-norm:
    bound 8 %."""
    from swiftrwkv_b200 import block as B
    D, R, F, t = 256, 64, 1024, torch.bfloat16
    p = {"g": rnd((D,), 90) * 0.1 + 1, "b": rnd((D,), 91) * 0.1, "down": rnd((R, D), 92, t, D ** -0.5),
         "up": rnd((D, R), 93, t, R ** -0.5), "up_b": rnd((D,), 94), "key": rnd((F, D), 95, t, D ** -0.5),
         "value": rnd((D, F), 96, t, F ** -0.5)}
    x = rnd((rows, D), 97, t)
    dy = rnd((rows, D), 98, t)
    p = {k: v.requires_grad_(True) for k, v in p.items()}
    x.requires_grad_(True)
    y = block_run(B, x, p, checkpoint)
    y.backward(dy)
    p64 = {k: v.detach().double().requires_grad_(True) for k, v in p.items()}
    x64 = x.detach().double().requires_grad_(True)
    y64 = block_run(Block64, x64, p64, checkpoint)
    y64.backward(dy.double())
    lim = 0.08 if checkpoint else 0.04
    rel = lambda a, b: float((a.double() - b).norm() / b.norm())
    assert rel(y.detach(), y64.detach()) < 0.04
    for name, a, b in [("x", x.grad, x64.grad)] + [(k, p[k].grad, p64[k].grad) for k in p]:
        assert a.dtype == (x.dtype if name == "x" else p[name].dtype)
        assert rel(a, b) < lim, (name, rel(a, b))


def test_differentiable_forms_compute_what_is_needed(cuda):
    """Frozen weights, frozen inputs and a bias alone; no gradient, no graph."""
    from swiftrwkv_b200 import block as B
    t = torch.bfloat16
    x, w, b = rnd((20, 64), 100, t), rnd((72, 64), 101, t, 0.1), rnd((72,), 102, t)
    dy = rnd((20, 72), 103, t)
    assert not B.projection(x, w, b, "tanh").requires_grad
    grads = []
    for need in ((1, 0, 0), (0, 1, 0), (0, 0, 1), (1, 1, 1)):
        ts = [v.clone().requires_grad_(bool(n)) for v, n in zip((x, w, b), need)]
        B.projection(*ts, "tanh").backward(dy)
        assert [v.grad is not None for v in ts] == [bool(n) for n in need]
        grads.append([v.grad for v in ts])
    for k in range(3):
        assert torch.equal(grads[k][k], grads[3][k])
    xs = x.clone().requires_grad_(True)
    with torch.no_grad():
        assert not B.channelMix(xs, rnd((128, 64), 104, t), rnd((64, 128), 105, t)).requires_grad


def test_checkpoint_saves_memory_for_the_backward_pass(cuda):
    """What a checkpointed channelMix keeps between forward and backward: codes
    and exponents of x and z, no 16-bit activation."""
    from swiftrwkv_b200 import block as B
    t, rows, D, F = torch.bfloat16, 512, 256, 1024
    key, value = rnd((F, D), 106, t).requires_grad_(True), rnd((D, F), 107, t).requires_grad_(True)
    x = rnd((rows, D), 108, t)
    kept = []
    with torch.autograd.graph.saved_tensors_hooks(lambda s: kept.append(s) or s, lambda s: s):
        B.channelMix(x, key, value)
    acts = [s for s in kept if s.data_ptr() not in (key.data_ptr(), value.data_ptr())]
    assert sum(s.numel() * s.element_size() for s in acts) == rows * (D + F) * 33 // 32


def test_wait_errors_are_reported_by_the_projections(cuda):
    """The projections share the tensor-core GEMMs' wait-error record: a set
    host record is reported once, and the next call is right."""
    from swiftrwkv_b200 import _lib, block as B
    t = torch.bfloat16
    x, w = rnd((300, 256), 110, t), rnd((256, 256), 111, t)
    want, _ = B.projectionForward(x, w)
    _lib.call("rwkv_q_gemm_inject_wait_error", 1, torch.cuda.current_stream().cuda_stream)
    with pytest.raises(_lib.RWKVError) as err:
        B.projectionForward(x, w)
    assert err.value.status == _lib.E_TIMEOUT
    assert torch.equal(B.projectionForward(x, w)[0], want)
    _lib.call("rwkv_q_gemm_inject_wait_error", 0, torch.cuda.current_stream().cuda_stream)
    B.projectionBackwardInput(x, w)                       # skips its work: the device flag is set
    assert _lib.status("rwkv_q_gemm_status", torch.cuda.current_stream().cuda_stream) == _lib.E_TIMEOUT
    assert torch.equal(B.projectionForward(x, w)[0], want)


@pytest.mark.parametrize("rows,OUT,IN", [(2304, 2304, 576), (2049, 2312, 1032), (4608, 1288, 520), (2500, 2048, 2048)])
def test_products_large_enough_for_pairs_of_sms(cuda, rows, OUT, IN):
    """Products that run on pairs of SMs (256 x 256 tiles, more than 512 terms),
    whole and ragged, with every epilogue; dW sums over the rows."""
    from swiftrwkv_b200 import block as B
    t = torch.bfloat16
    x, w, dy = rnd((rows, IN), 120, t), rnd((OUT, IN), 121, t, IN ** -0.5), rnd((rows, OUT), 122, t)
    bias, res = rnd((OUT,), 123), rnd((rows, OUT), 124, t)
    z0, s0 = proj_sums(x, w)
    y, _ = B.projectionForward(x, w)
    check(y, z0, TC * s0 + u(t) * (z0.abs() + TC * s0), "plain")
    z, dz = z0 + bias.double(), TC * (s0 + bias.double().abs())
    y, ck = B.projectionForward(x, w, bias, "relu2", res, checkpoint=True)
    want = act64(z, "relu2") + res.double()
    tol = slope(z, "relu2", dz) + 32 * U32 * (act64(z, "relu2").abs() + want.abs())
    check(y, want, tol + u(t) * (want.abs() + tol), "relu2")
    v = B.checkpoint8Values(ck, dtype=torch.float32)
    check(v, z, (top_of_group(z) + top_of_group(dz)) / 127.5 + top_of_group(dz), "checkpoint")
    f, _ = B.projectionForward(x, w, residual=res.float(), out_dtype=torch.float32)
    check(f, z0 + res.double(), TC * s0 + 4 * U32 * (z0.abs() + res.double().abs()), "fp32 out")
    ckx = B.checkpoint8(x)
    g, s = proj_sums(dy, w.t())
    d = grad64(values64(x), "relu2")
    got = B.projectionBackwardInput(dy, w, pre=ckx, act="relu2", addend=x)
    want = g * d + x.double()
    tol = TC * s * d.abs() + 64 * U32 * ((g * d).abs() + want.abs())
    check(got, want, tol + u(t) * (want.abs() + tol), "dx")
    want, s = proj_sums(dy.t(), values64(x).t())
    f, db = B.projectionBackwardWeight(dy, ckx, bias=True, out_dtype=torch.float32)
    check(f, want, TC * s + U32 * want.abs(), "dw")
    check(db, dy.double().sum(0), (rows + 16) * U32 * dy.double().abs().sum(0) + 1e-38, "db")
    again, _ = B.projectionBackwardWeight(dy, ckx, out_dtype=torch.float32)
    assert torch.equal(again, f)


def test_offsets_past_32_bits(cuda):
    """Tensors of more than 2^31 elements: the last rows come out as they do
    from a call on them alone (elementwise results and per-row statistics do not
    depend on the other rows), and the projection's against 64 bits."""
    from swiftrwkv_b200 import block as B
    t, D = torch.bfloat16, 2048
    rows = (1 << 31) // D + 1000
    x = torch.empty(rows, D, device="cuda", dtype=t)
    for i in range(0, rows, 1 << 18):
        x[i:i + (1 << 18)].normal_()
    tail = x[-300:].clone()
    w, b = rnd((D,), 140), rnd((D,), 141)
    y, mean, rstd, ck = B.layerNormForward(x, w, b, checkpoint=True)
    y1, mean1, rstd1, ck1 = B.layerNormForward(tail, w, b, checkpoint=True)
    assert torch.equal(y[-300:], y1) and torch.equal(mean[-300:], mean1) and torch.equal(rstd[-300:], rstd1)
    assert torch.equal(ck.codes[-300:], ck1.codes) and torch.equal(ck.exps[-300:], ck1.exps)
    v = B.checkpoint8Values(ck, "relu2")
    assert torch.equal(v[-300:], B.checkpoint8Values(ck1, "relu2"))
    del v
    dz = B.activationBackward(x, ck, "tanh")
    assert torch.equal(dz[-300:], B.activationBackward(tail, ck1, "tanh"))
    del dz
    dx, _, _ = B.layerNormBackward(x, ck, w, mean, rstd, dres=y)
    assert torch.equal(dx[-300:], B.layerNormBackward(tail, ck1, w, mean1, rstd1, dres=y1)[0])
    del dx, y
    h, pw = rnd((rows, 64), 142, t), rnd((D, 64), 143, t, 0.125)
    res = x
    p, ckp = B.projectionForward(h, pw, act="relu2", residual=res, checkpoint=True)
    z, s = proj_sums(h[-300:], pw)
    want = act64(z, "relu2") + res[-300:].double()
    tol = slope(z, "relu2", TC * s) + 32 * U32 * want.abs()
    check(p[-300:], want, tol + u(t) * (want.abs() + tol), "projection")
    last = B.Checkpoint8(ckp.codes[-300:], ckp.exps[-300:], t)
    check(B.checkpoint8Values(last, dtype=torch.float32), z, (top_of_group(z) + top_of_group(TC * s)) / 127.5 +
          top_of_group(TC * s), "checkpoint")
    g = B.projectionBackwardInput(p, pw)
    want, s = proj_sums(p[-300:], pw.t())
    check(g[-300:], want, TC * s + u(t) * (want.abs() + TC * s), "dx")


CAPTURE_FIRST = """
import sys; sys.path.insert(0, {root!r})
import torch
from swiftrwkv_b200 import _lib, block as B
x, w = torch.ones(32, 64, device="cuda", dtype=torch.bfloat16), torch.ones(64, 64, device="cuda", dtype=torch.bfloat16)
g = torch.cuda.CUDAGraph()
s = torch.cuda.Stream()
seen = []
with torch.cuda.stream(s):
    g.capture_begin()
    try:
        B.projectionForward(x, w)
    except _lib.RWKVError as e:
        seen.append(str(e))
    y = B.layerNormForward(x, w[0].float(), w[1].float())[0]   # needs nothing set up
    g.capture_end()
assert len(seen) == 1 and "before capturing" in seen[0], seen
g.replay()
torch.cuda.synchronize()
assert bool((y == 1).all())
assert float(B.projectionForward(x, w)[0][0, 0]) == 64.0
print("ok")
"""


def test_a_first_projection_during_capture_is_refused(cuda):
    """The wait-error record is not allocated while a stream is captured: the
    call is refused, the capture itself goes on, and later calls work."""
    import os
    import subprocess
    import sys
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    r = subprocess.run([sys.executable, "-c", CAPTURE_FIRST.format(root=root)], capture_output=True, text=True, timeout=300)
    assert r.returncode == 0 and "ok" in r.stdout, r.stdout + r.stderr


@pytest.mark.parametrize("bwd", [False, True])
@pytest.mark.parametrize("lengths", [(2560, 768), (8000, 4200), (2411, 259), (9001, 8301)])
def test_layer_norms_of_two_lengths_on_two_threads(cuda, bwd, lengths):
    """Rows of two lengths of one kernel, each in a loop on a host thread and a
    stream of its own: no call fails, and the results are those of single calls.
    The lengths differ in the shared memory that they need."""
    from swiftrwkv_b200 import _lib
    from swiftrwkv_b200 import block as B
    L, t, rows = _lib.lib(), torch.bfloat16, 8

    def job(D):
        x, dy, w, b = rnd((rows, D), 90, t), rnd((rows, D), 91, t), rnd((D,), 92), rnd((D,), 93)
        y, mean, rstd, _ = B.layerNormForward(x, w, b)
        want, out = (B.layerNormBackward(dy, x, w, mean, rstd, params=False)[0] if bwd else y), torch.empty_like(x)
        s = torch.cuda.Stream()
        if bwd:
            f = L.rwkv_layer_norm_backward
            args = (_lib.BF16, dy.data_ptr(), x.data_ptr(), None, None, _lib.F32, w.data_ptr(), mean.data_ptr(),
                    rstd.data_ptr(), None, out.data_ptr(), None, None, rows, D, None, 0, s.cuda_stream)
        else:
            f = L.rwkv_layer_norm_forward
            args = (_lib.BF16, x.data_ptr(), _lib.F32, w.data_ptr(), b.data_ptr(), 1e-5, out.data_ptr(), mean.data_ptr(),
                    rstd.data_ptr(), None, None, rows, D, s.cuda_stream)
        return f, args, want, out, (x, dy, w, b, mean, rstd, s)

    jobs, failed, go = [job(D) for D in lengths], [0, 0], threading.Barrier(2)
    torch.cuda.synchronize()

    def run(k):
        f, args = jobs[k][:2]
        go.wait()
        failed[k] = sum(f(*args) != _lib.OK for _ in range(20000))

    threads, interval = [threading.Thread(target=run, args=(k,)) for k in range(2)], sys.getswitchinterval()
    sys.setswitchinterval(1e-5)
    try:
        for th in threads:
            th.start()
        for th in threads:
            th.join()
    finally:
        sys.setswitchinterval(interval)
    torch.cuda.synchronize()
    assert failed == [0, 0]
    for _, _, want, out, _ in jobs:
        assert torch.equal(out, want)


@pytest.mark.parametrize("what,rows", [("y", 5), ("y", 2304), ("dx", 2304), ("dw", 2304)])
def test_projection_sums_too_long_for_one_accumulator(cuda, what, rows):
    """One product of 1 and 2^18 (in the few-row kernel 2^20) of just below 2^-25.
    The tensor core cuts each of the 16 products of a step off at 2^-25 of the
    largest addend's binade and the step's sum at 2^-23: less than 16 2^-25 + 2^-23 =
    5 2^-23 of the sum is lost per step, so that an accumulator of 32768 terms is off
    by at most 2048 steps 5 2^-23 sum|terms|; the splits' sums are joined by
    roundings of 2^-24 each, one per split.  An accumulator of all the terms
    loses nearly all of the small ones, 7.8e-3 (the few-row kernel's sixteen warps 1.9e-3)."""
    from swiftrwkv_b200 import block as B
    t, n = torch.bfloat16, 2304 if rows > 16 else 24
    K = 1 << (18 if rows > 16 else 20)
    small = 2.0 ** -13 * 1.984375

    def operand(m, first):
        a = torch.full((m, K) if first else (K, m), 2.0 ** -13, device="cuda", dtype=t)
        (a if first else a.t())[:, 0] = 1.0
        return a

    if what == "y":
        a, b = operand(rows, True), operand(n, True)
    elif what == "dx":
        a, b = operand(rows, True), operand(n, False)
    else:
        a, b = operand(rows, False), operand(n, False)
    (a if what != "dw" else a.t())[:, 1:] = small
    got = {"y": lambda: B.projectionForward(a, b, out_dtype=torch.float32)[0],
           "dx": lambda: B.projectionBackwardInput(a, b, out_dtype=torch.float32),
           "dw": lambda: B.projectionBackwardWeight(a, b, out_dtype=torch.float32)[0]}[what]()
    want = torch.full((rows, n), 1.0 + (K - 1) * small * 2.0 ** -13, device="cuda", dtype=torch.float64)
    check(got, want, (2048 * 5 * 2.0 ** -23 + K / 32768 * U32 + U32) * want, what)


@pytest.mark.parametrize("rows,n,K", [(5, 1024, 8), (200, 1024, 8), (40, 264, 4096), (2304, 2304, 576)])
@pytest.mark.parametrize("act", ["tanh", "sigmoid"])
@pytest.mark.parametrize("dt", ["bf16", "f16"])
def test_projection_fp32_results_of_activations(cuda, dt, act, rows, n, K):
    """Sums of one product, exact in fp32, so that what is off is the function.  CUDA
    gives expf and tanhf to 2 ulp, 2^-22 relative.  sigmoid = 1 / (1 + e): 2^-22 from
    e, 2^-24 for the sum and for the quotient.  The derivatives k^2 e / (1 + e)^2:
    2^-22 from e above; below, e's share of 1 + e is half at most, twice with a
    rounding of 2^-24 each; 2^-24 each for the square, the quotient and the product
    with the sum: (1 + 1 + 5 / 4) 2^-22."""
    from swiftrwkv_b200 import block as B
    t, f32 = DTYPES[dt], torch.float32
    x, w = torch.zeros(rows, K, device="cuda", dtype=t), torch.zeros(n, K, device="cuda", dtype=t)
    x[:, K // 2] = torch.linspace(0.5, 1, rows, device="cuda").to(t)
    w[:, K // 2] = torch.cat([torch.linspace(-12, 12, n // 2), torch.linspace(-0.1, 0.1, n - n // 2)]).cuda().to(t)
    z = x.double() @ w.double().t()
    want = act64(z, act)
    check(B.projectionForward(x, w, act=act, out_dtype=f32)[0], want, (1.0 if act == "tanh" else 1.5) * 2.0 ** -22 * want.abs())
    pre = z.to(t)
    want = x.double()[:, K // 2:K // 2 + 1] * grad64(pre.double(), act)
    ones = torch.zeros(K, n, device="cuda", dtype=t)
    ones[K // 2] = 1
    check(B.projectionBackwardInput(x, ones, pre=pre, act=act, out_dtype=f32), want, 3.25 * 2.0 ** -22 * want.abs())


def test_sigmoid_of_far_negative_values_in_fp32(cuda):
    """e^z below the normal numbers is kept to half of their spacing 2^-149 and the
    2 ulp of expf, where 1 / (1 + e^-z) would overflow to 0."""
    from swiftrwkv_b200 import block as B
    z = torch.linspace(-103, -60, 87, device="cuda").to(torch.bfloat16)
    x, w = torch.ones(20, 8, device="cuda", dtype=torch.bfloat16) / 8, z[:80, None].expand(80, 8).contiguous()
    want = act64(z.double(), "sigmoid")
    y = B.projectionForward(x, w, act="sigmoid", out_dtype=torch.float32)[0]
    assert bool(((y.double() - want[:80]).abs() <= 1.5 * 2.0 ** -22 * want[:80] + 2 * 2.0 ** -149).all())
    ck = B.checkpoint8(z[:, None].contiguous())        # one channel: 7 bits hold every value
    want = act64(B.checkpoint8Values(ck, dtype=torch.float32).double(), "sigmoid")
    y = B.checkpoint8Values(ck, act="sigmoid", dtype=torch.float32)
    assert bool(((y.double() - want).abs() <= 1.5 * 2.0 ** -22 * want + 2 * 2.0 ** -149).all()) and bool((y > 0).all())


@pytest.mark.parametrize("dt", ["f32", "bf16"])
@pytest.mark.parametrize("rows,D", [(150, 12289), (131, 16384), (65, 33000)])
def test_layer_norm_of_long_rows_in_more_rows_than_blocks(cuda, dt, rows, D):
    test_layer_norm_backward(cuda, dt, False, rows, D)
    test_layer_norm_backward(cuda, dt, True, rows, D)


def test_streams_by_public_names_alone(cuda, monkeypatch):
    from swiftrwkv_b200 import block as B
    x = rnd((5, 96), 95, torch.bfloat16)
    want = B.checkpoint8(x).codes
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        assert B._public_raw_stream(0) == B._raw_stream(0) == s.cuda_stream
        monkeypatch.setattr(B, "_raw_stream", B._public_raw_stream)
        monkeypatch.setattr(B, "_current_device", torch.cuda.current_device)
        got = B.checkpoint8(x).codes
    s.synchronize()
    assert torch.equal(got, want)


def test_what_the_entry_points_refuse_is_a_value_error(cuda):
    """Arguments that only the C entry points check: eps, and sizes past the limits."""
    from swiftrwkv_b200 import block as B
    t = torch.bfloat16
    x, v = rnd((4, 64), 96, t), torch.ones(64, device="cuda")
    for eps in (-1.0, float("nan")):
        with pytest.raises(ValueError, match="eps"):
            B.layerNormForward(x, v, v, eps)
    w = torch.zeros(8, 8, device="cuda", dtype=t)
    many = torch.zeros((1 << 24) + 1, 8, device="cuda", dtype=t)
    for f in (lambda: B.projectionForward(many, w), lambda: B.projectionBackwardInput(many, w),
              lambda: B.projectionBackwardWeight(many, many)):
        with pytest.raises(ValueError, match="too large"):
            f()
    del many
    wide = torch.zeros((1 << 30) + 8, device="cuda", dtype=t)
    with pytest.raises(ValueError, match="1..2\\^30"):
        B.checkpoint8(wide)
    with pytest.raises(ValueError, match="1..2\\^30"):
        B.layerNormForward(wide, wide, wide)


@pytest.mark.parametrize("act", ["none", "relu2", "tanh"])
@pytest.mark.parametrize("rows,OUT,IN", [(40, 24, 96), (300, 136, 40)])
def test_weight_gradient_of_values_at_the_ends_of_fp16(cuda, act, rows, OUT, IN):
    """The operand is act(value) in fp16: the checkpoint's values far below 2^-14 on
    the grid of 2^-24, and infinite past 65504 (relu2: from 256 on).  Rounded fp16
    operands from the formula, multiplied in 64 bits, give dW to the sums' bound;
    tanh is off by 2^-18 before its rounding, which can move it to a neighbour."""
    from swiftrwkv_b200 import block as B
    x = rnd((rows, IN), 97)
    x[::3] *= 2.0 ** -19          # values around 2^-20, scales below 2^-24
    x[1, :8], x[1, 8:16] = 70000.0, 300.0
    dy = rnd((rows, OUT), 98, torch.float16)
    dy[1, 0] = 0
    packed = B.checkpoint8(x)     # as a projection keeps its fp32 sums
    ck = B.Checkpoint8(packed.codes, packed.exps, torch.float16)
    values = B.checkpoint8Values(ck, dtype=torch.float32).double()
    assert float(values.abs().max()) > 65504 and 0 < float(values[values != 0].abs().min()) < 2.0 ** -24
    operand = act64(values, act).float().to(torch.float16).double()
    want, sums = dy.double().t() @ operand, dy.double().abs().t() @ operand.abs()
    step = dy.double().abs().t() @ (2.0 ** -10 * operand.abs() + 2.0 ** -24) if act == "tanh" else 0
    dw, _ = B.projectionBackwardWeight(dy, ck, act=act, out_dtype=torch.float32)
    # columns of row 1 past the end of fp16; beside 70000 the scale is 1024, and 300 is 0
    n = 0 if act == "tanh" else 8
    assert torch.isnan(dw[0, :n]).all() and torch.isinf(dw[1:, :n]).all() and torch.isfinite(dw[:, n:]).all()
    check(dw[:, n:], want[:, n:], (5 * 2.0 ** -23 * (rows / 16 + 1) * sums + U32 * want.abs() + step)[:, n:])


def test_weight_gradient_of_fp16_squares(cuda):
    """relu2's operand in fp16: 255^2 = 65025 rounds to 65024, 256^2 is infinite."""
    from swiftrwkv_b200 import block as B
    z, dy = torch.zeros(4, 8, device="cuda", dtype=torch.float16), torch.ones(4, 8, device="cuda", dtype=torch.float16)
    z[0, 0], z[0, 1], z[0, 2] = 255, 256, -300
    for out in (torch.float32, torch.float16):
        dw, _ = B.projectionBackwardWeight(dy, z, act="relu2", out_dtype=out)
        assert bool((dw[:, 0] == 65024).all()) and torch.isinf(dw[:, 1]).all() and not dw[:, 2:].any()


@pytest.mark.parametrize("act", ["none", "relu2", "tanh", "sigmoid"])
def test_activation_gradient_matches_differences_of_the_activation(cuda, act):
    """act' against central differences of act, both as the library computes them from
    a checkpoint's codes q h, h = 2^-5: off by h^2 / 6 max|act'''| (tanh: 2, sigmoid:
    1/8, the others 0 away from the corner), by act's 2^-22 |act| over h, and by the
    gradient's own 2^-20 |act'|."""
    from swiftrwkv_b200 import block as B
    h, q = 2.0 ** -5, torch.arange(-112, 112, device="cuda", dtype=torch.int8)
    def f(shift, g):
        codes = (q + shift).view(7, 32).contiguous()
        return g(B.Checkpoint8(codes, torch.full((7, 1), 122, dtype=torch.uint8, device="cuda"), torch.float32)).double()
    value = lambda ck: B.checkpoint8Values(ck, act=act)
    up, down = f(1, value), f(-1, value)
    got = f(0, lambda ck: B.activationBackward(torch.ones(7, 32, device="cuda"), ck, act))
    third = {"tanh": 2.0, "sigmoid": 0.125}.get(act, 0.0)
    tol = h * h / 6 * third + 2.0 ** -22 * torch.maximum(up.abs(), down.abs()) / h + 2.0 ** -20 * got.abs()
    if act == "relu2":
        tol = tol + h * (q.view(7, 32) == 0)         # ((h)^2 - 0) / 2h = h / 2 beside the corner
    assert bool((((up - down) / (2 * h) - got).abs() <= tol).all())


@pytest.mark.parametrize("rows,n,K", [(2305, 2312, 65560), (300, 200, 131080), (1, 24, 262152), (16, 2056, 262144),
                                      (40, 136, 32776), (4100, 2048, 40000)])
def test_projection_of_whole_numbers_over_long_sums(cuda, rows, n, K):
    """Operands of -1, 0 and 1: every partial sum is a whole number below 2^24, exact in
    fp32 whatever the order and the splits, and so are the epilogue's squares,
    bias and residual: the results are equal, tile by tile, in every direction."""
    from swiftrwkv_b200 import block as B
    t, f32 = torch.bfloat16, torch.float32
    g = torch.Generator(device="cuda").manual_seed(99)

    def whole(*s, most=1):
        return torch.randint(-most, most + 1, s, generator=g, device="cuda").to(t)

    def product(a, b):
        return torch.cat([a[i:i + 512].double() @ b.double().t() for i in range(0, a.shape[0], 512)])

    x, w = whole(rows, K), whole(n, K)
    z = product(x, w)
    assert float(z.abs().max()) < 2 ** 11
    assert torch.equal(B.projectionForward(x, w, out_dtype=f32)[0].double(), z)
    bias, res = whole(n, most=9).float(), whole(rows, n, most=9).float()
    y, ck = B.projectionForward(x, w, bias=bias, act="relu2", residual=res, checkpoint=True, out_dtype=f32)
    zb = z + bias.double()
    assert torch.equal(y.double(), act64(zb, "relu2") + res.double())
    assert torch.equal(B.checkpoint8Values(ck, dtype=f32).double(), values64(zb))
    del w
    wt, pre = whole(K, n), whole(rows, n, most=9)
    dx = B.projectionBackwardInput(x, wt, pre=B.checkpoint8(pre), act="relu2", addend=res, out_dtype=f32)
    assert torch.equal(dx.double(), product(x, wt.t()) * grad64(pre.double(), "relu2") + res.double())
    del wt
    x = x[:rows // 8 * 8]
    if rows >= 8:
        xs = whole(K, n)
        dw, db = B.projectionBackwardWeight(x.t().contiguous(), xs, bias=True, out_dtype=f32)
        assert torch.equal(dw.double(), product(x, xs.t()))
        assert torch.equal(db.double(), x.double().sum(1))
