"""CPU tests of the operators between a block's projections and its WKV path
(dropout, residual norm, token mix, tail of the time mix): every refusal happens on
the host, before anything launches; and the tests' own generator."""
from __future__ import annotations

import ctypes

import numpy as np
import pytest
import torch

from philox_oracle import kept, philox
from swiftrwkv_b200 import _lib
from swiftrwkv_b200 import block as B

FAKE = ctypes.c_void_p(0x1000)   # aligned, never dereferenced: checks fail first
ODD = ctypes.c_void_p(0x1001)
HALF = ctypes.c_void_p(0x1008)   # 8-byte aligned only
F32, BF16, F16 = _lib.F32, _lib.BF16, _lib.F16


def st(name, *a):
    return _lib.status(name, *a)


def test_the_generator_gives_its_published_answers():
    """The known answers that the generator's authors publish with it (Random123)."""
    for counter, key, words in (
            ((0, 0, 0, 0), (0, 0), (0x6627E8D5, 0xE169C58D, 0xBC57AC4C, 0x9B00DBD8)),
            ((2**32 - 1,) * 4, (2**32 - 1,) * 2, (0x408F276D, 0x41C83B0E, 0xA20BC7C6, 0x6D5451FD)),
            ((0x243F6A88, 0x85A308D3, 0x13198A2E, 0x03707344), (0xA4093822, 0x299F31D0),
             (0xD16CFE09, 0x94FDCCEB, 0x5001E420, 0x24126EA1))):
        assert tuple(int(w) for w in philox(counter, key)) == words


def test_kept_elements_are_places_of_the_whole():
    whole = kept(1000, 0.3, 5, 7)
    assert np.array_equal(kept(100, 0.3, 5, 7, first=333), whole[333:433])
    assert kept(10, 0.0, 1).all() and not kept(10, 1.0, 1).any()


def drop(dt=BF16, x=FAKE, p=0.1, seed=0, offset=0, state=None, y=FAKE, n=64):
    return st("rwkv_dropout", dt, x, p, seed, offset, state, y, n, None)


def test_dropout_refusals():
    assert drop(dt=3) == _lib.E_DTYPE
    assert drop(x=None) == _lib.E_NULL
    assert drop(y=None) == _lib.E_NULL
    for n in (0, -1, (1 << 40) + 1):
        assert drop(n=n) == _lib.E_SHAPE
    for p in (-1e-9, 1.0001, float("nan"), float("inf")):
        assert drop(p=p) == _lib.E_SHAPE
    assert drop(x=HALF) == _lib.E_UNSUPPORTED
    assert drop(y=ODD) == _lib.E_UNSUPPORTED
    assert drop(state=ODD) == _lib.E_UNSUPPORTED


def rn_fwd(dt=BF16, x=FAKE, br=FAKE, scale=1.0, p=0.0, state=None, wdt=F32, w=FAKE, b=FAKE, eps=1e-5, s=FAKE, y=FAKE,
           mean=FAKE, rstd=FAKE, c=None, e=None, rows=4, D=64):
    return st("rwkv_residual_norm_forward", dt, x, br, scale, p, 0, 0, state, wdt, w, b, ctypes.c_float(eps), s, y, mean,
              rstd, c, e, rows, D, None)


def test_residual_norm_forward_refusals():
    assert rn_fwd(dt=7) == _lib.E_DTYPE
    assert rn_fwd(wdt=-1) == _lib.E_DTYPE
    for k in ("x", "br", "w", "b", "s", "y"):
        assert rn_fwd(**{k: None}) == _lib.E_NULL
    assert rn_fwd(mean=None) == _lib.E_NULL
    assert rn_fwd(c=FAKE) == _lib.E_NULL
    assert rn_fwd(rows=0) == _lib.E_SHAPE
    assert rn_fwd(D=0) == _lib.E_SHAPE
    for eps in (-1.0, float("nan")):
        assert rn_fwd(eps=eps) == _lib.E_SHAPE
    for p in (-0.5, 1.5, float("nan")):
        assert rn_fwd(p=p) == _lib.E_SHAPE
    for scale in (float("inf"), float("nan"), 1e39, -1e300):
        assert rn_fwd(scale=scale) == _lib.E_SHAPE
    assert rn_fwd(scale=3e38, p=0.9) == _lib.E_SHAPE   # finite only before the division by 1 - q
    assert rn_fwd(D=60) == _lib.E_UNSUPPORTED
    assert rn_fwd(D=12296) == _lib.E_UNSUPPORTED
    assert rn_fwd(dt=F32, D=6152) == _lib.E_UNSUPPORTED
    for k in ("x", "br", "w", "b", "s", "y"):
        assert rn_fwd(**{k: HALF}) == _lib.E_UNSUPPORTED
    assert rn_fwd(state=ODD) == _lib.E_UNSUPPORTED


def rn_bwd(dt=BF16, dy=FAKE, s=FAKE, c=None, e=None, wdt=F32, w=FAKE, mean=FAKE, rstd=FAKE, dres=None, scale=1.0, p=0.1,
           state=None, dx=FAKE, dbr=FAKE, dw=FAKE, db=FAKE, rows=4, D=64, ws=FAKE, n=1 << 30):
    return st("rwkv_residual_norm_backward", dt, dy, s, c, e, wdt, w, mean, rstd, dres, scale, p, 0, 0, state, dx, dbr, dw,
              db, rows, D, ws, n, None)


def test_residual_norm_backward_refusals():
    assert rn_bwd(dt=3) == _lib.E_DTYPE
    for k in ("dy", "s", "w", "mean", "rstd", "dx", "dbr", "db"):
        assert rn_bwd(**{k: None}) == _lib.E_NULL
    assert rn_bwd(c=FAKE, e=FAKE) == _lib.E_NULL             # the sum and its checkpoint
    assert rn_bwd(s=None, c=FAKE) == _lib.E_NULL
    assert rn_bwd(rows=-1) == _lib.E_SHAPE
    assert rn_bwd(p=2.0) == _lib.E_SHAPE
    assert rn_bwd(scale=float("nan")) == _lib.E_SHAPE
    assert rn_bwd(D=4) == _lib.E_UNSUPPORTED
    assert rn_bwd(dres=HALF) == _lib.E_UNSUPPORTED
    need = _lib.lib().rwkv_residual_norm_backward_workspace_size(4, 64)
    assert need > 0
    assert rn_bwd(n=need - 1) == _lib.E_WORKSPACE
    assert rn_bwd(ws=None) == _lib.E_WORKSPACE
    assert rn_bwd(ws=HALF) == _lib.E_UNSUPPORTED


def test_residual_norm_scale_is_finite_where_everything_is_dropped():
    for scale in (float("inf"), float("nan"), -1e300):
        assert rn_fwd(scale=scale, p=1.0) == _lib.E_SHAPE
        assert rn_bwd(scale=scale, p=1.0) == _lib.E_SHAPE


def pointers(*ps):
    return (ctypes.c_void_p * len(ps))(*[p.value if p else None for p in ps])


def mix_fwd(dt=BF16, x=FAKE, mdt=F32, mix=FAKE, prev=None, lengths=None, y=(FAKE, FAKE), last=FAKE, b=2, t=3, d=64, j=2):
    return st("rwkv_token_mix_forward", dt, x, mdt, mix, prev, lengths, pointers(*y) if y else None, last, b, t, d, j, None)


def test_token_mix_forward_refusals():
    assert mix_fwd(dt=5) == _lib.E_DTYPE
    assert mix_fwd(mdt=5) == _lib.E_DTYPE
    for k in ("x", "mix", "last"):
        assert mix_fwd(**{k: None}) == _lib.E_NULL
    assert mix_fwd(y=(FAKE, None)) == _lib.E_NULL
    assert mix_fwd(y=None) == _lib.E_NULL
    for k in ("b", "t", "d"):
        assert mix_fwd(**{k: 0}) == _lib.E_SHAPE
    assert mix_fwd(j=0) == _lib.E_SHAPE
    assert mix_fwd(j=7, y=(FAKE,) * 7) == _lib.E_SHAPE
    assert mix_fwd(d=(1 << 20) + 8) == _lib.E_SHAPE
    assert mix_fwd(d=60) == _lib.E_UNSUPPORTED
    assert mix_fwd(y=(FAKE, HALF)) == _lib.E_UNSUPPORTED
    for k in ("x", "mix", "last", "prev"):
        assert mix_fwd(**{k: HALF}) == _lib.E_UNSUPPORTED
    assert mix_fwd(lengths=ODD) == _lib.E_UNSUPPORTED


def mix_bwd(dt=BF16, dy=(FAKE, None), x=FAKE, mdt=F32, mix=FAKE, prev=None, lengths=None, dlast=None, dx=FAKE, dmix=FAKE,
            dprev=None, b=2, t=3, d=64, j=2, ws=FAKE, n=1 << 40):
    return st("rwkv_token_mix_backward", dt, pointers(*dy) if dy else None, x, mdt, mix, prev, lengths, dlast, dx, dmix,
              dprev, b, t, d, j, ws, n, None)


def test_token_mix_backward_refusals():
    assert mix_bwd(dt=-1) == _lib.E_DTYPE
    for k in ("dy", "x", "mix", "dx"):
        assert mix_bwd(**{k: None}) == _lib.E_NULL
    assert mix_bwd(t=-2) == _lib.E_SHAPE
    assert mix_bwd(d=12) == _lib.E_UNSUPPORTED
    assert mix_bwd(dy=(HALF, FAKE)) == _lib.E_UNSUPPORTED
    for k in ("dlast", "dx", "dmix", "dprev", "ws"):
        assert mix_bwd(**{k: HALF}) == _lib.E_UNSUPPORTED
    size = _lib.lib().rwkv_token_mix_backward_workspace_size
    need = size(BF16, 2, 3, 64, 2)
    assert need >= 2 * 64 * 4 and need % (2 * 64 * 4) == 0
    assert mix_bwd(n=need - 1) == _lib.E_WORKSPACE
    assert mix_bwd(ws=None) == _lib.E_WORKSPACE
    assert size(BF16, 0, 3, 64, 2) == size(BF16, 2, 3, 60, 2) == size(BF16, 2, 3, 64, 7) == size(9, 2, 3, 64, 2) == 0


def tail_fwd(dt=BF16, a=FAKE, r=FAKE, k=FAKE, v=FAKE, g=FAKE, wdt=F32, rk=FAKE, w=FAKE, b=FAKE, eps=64e-5, out=FAKE, rows=3,
             h=2, s=64):
    return st("rwkv_tmix_tail_forward", dt, a, r, k, v, g, wdt, rk, w, b, ctypes.c_float(eps), out, rows, h, s, None)


def test_tail_forward_refusals():
    assert tail_fwd(dt=4) == _lib.E_DTYPE
    assert tail_fwd(wdt=4) == _lib.E_DTYPE
    for k in ("a", "r", "k", "v", "g", "rk", "w", "b", "out"):
        assert tail_fwd(**{k: None}) == _lib.E_NULL
        assert tail_fwd(**{k: HALF}) == _lib.E_UNSUPPORTED
    assert tail_fwd(rows=0) == _lib.E_SHAPE
    assert tail_fwd(h=0) == _lib.E_SHAPE
    assert tail_fwd(h=(1 << 16) + 1) == _lib.E_SHAPE
    for eps in (-1e-9, float("nan")):
        assert tail_fwd(eps=eps) == _lib.E_SHAPE
    for s in (0, 16, 48, 96, 512):
        assert tail_fwd(s=s) == _lib.E_UNSUPPORTED


def tail_bwd(dt=BF16, d=FAKE, a=FAKE, r=FAKE, k=FAKE, v=FAKE, g=FAKE, wdt=F32, rk=FAKE, w=FAKE, b=FAKE, eps=64e-5, da=FAKE,
             dr=FAKE, dk=FAKE, dv=FAKE, dg=FAKE, drk=FAKE, dw=FAKE, db=FAKE, rows=3, h=2, s=64, ws=FAKE, n=1 << 40):
    return st("rwkv_tmix_tail_backward", dt, d, a, r, k, v, g, wdt, rk, w, b, ctypes.c_float(eps), da, dr, dk, dv, dg, drk,
              dw, db, rows, h, s, ws, n, None)


def test_tail_backward_refusals():
    assert tail_bwd(dt=4) == _lib.E_DTYPE
    for k in ("d", "a", "r", "k", "v", "g", "rk", "w", "b", "da", "dr", "dk", "dv", "dg", "drk", "dw", "db"):
        assert tail_bwd(**{k: None}) == _lib.E_NULL
        assert tail_bwd(**{k: HALF}) == _lib.E_UNSUPPORTED
    assert tail_bwd(rows=-1) == _lib.E_SHAPE
    assert tail_bwd(s=40) == _lib.E_UNSUPPORTED
    size = _lib.lib().rwkv_tmix_tail_backward_workspace_size
    need = size(3, 2, 64)
    assert need >= 3 * 128 * 4 and need % (3 * 128 * 4) == 0
    assert tail_bwd(n=need - 1) == _lib.E_WORKSPACE
    assert tail_bwd(ws=None) == _lib.E_WORKSPACE
    assert tail_bwd(ws=HALF) == _lib.E_UNSUPPORTED
    assert size(0, 2, 64) == size(3, 0, 64) == size(3, 2, 65) == 0


def test_python_refusals_come_before_any_launch():
    x, v = torch.zeros(2, 3, 64), torch.ones(64)
    for f in (lambda: B.dropoutForward(x, 0.1, 0), lambda: B.residualNormForward(x, x, v, v),
              lambda: B.residualNormBackward(x, x, v, v, v), lambda: B.tokenMixForward(x, x[0]),
              lambda: B.tokenMixBackward([x] * 3, x, x[0]),
              lambda: B.tmixTailForward(x, x, x, x, x, v[None], v, v),
              lambda: B.tmixTailBackward(x, x, x, x, x, x, v[None], v, v), lambda: B.dropoutForward(None, 0.1, 0),
              lambda: B.tokenMixForward([x], x[0])):
        with pytest.raises(ValueError, match="CUDA tensor"):
            f()


def test_what_is_drawn_is_checked_on_the_host(monkeypatch):
    monkeypatch.setattr(B, "_tensor", lambda name, t, *a, **k: t)  # CPU tensors as far as the check that raises
    x, v = torch.zeros(2, 64), torch.ones(64)
    for p in (-0.1, 1.5, float("nan"), "0.1", None, torch.tensor(0.1)):
        with pytest.raises(ValueError, match="^p="):
            B.dropoutForward(x, p, 0)
        with pytest.raises(ValueError, match="^p="):
            B.residualNormBackward(x, x, v, v, v, p=p)
    for seed in (-1, 1 << 64, 0.5, None, "7"):
        with pytest.raises(ValueError, match="^seed="):
            B.dropoutForward(x, 0.1, seed)
    for offset in (-1, 1 << 64, 0.5, None):
        with pytest.raises(ValueError, match="^offset="):
            B.residualNormForward(x, x, v, v, p=0.1, offset=offset)
    for scale in (None, "1", torch.ones(())):
        with pytest.raises(ValueError, match="^scale="):
            B.residualNormBackward(x, x, v, v, v, scale=scale)


def test_shapes_are_checked_on_the_host(monkeypatch):
    monkeypatch.setattr(B, "_tensor", lambda name, t, *a, **k: t)
    x, mix = torch.zeros(2, 3, 64), torch.zeros(6, 64)
    with pytest.raises(ValueError, match=r"\[B, T, D\]"):
        B.tokenMixForward(x[0], mix)
    for bad in (mix[0], torch.zeros(7, 64), torch.zeros(0, 64), torch.zeros(6, 56)):
        with pytest.raises(ValueError, match="mix"):
            B.tokenMixForward(x, bad)
    for dys in ([x] * 5, x, None, 3.0):
        if not isinstance(dys, torch.Tensor):
            with pytest.raises(ValueError, match="dys"):
                B.tokenMixBackward(dys, x, mix)
    v = torch.ones(128)
    with pytest.raises(ValueError, match=r"rk .* must be \[H, S\]"):
        B.tmixTailForward(x, x, x, x, x, v, v, v)
    with pytest.raises(ValueError, match="wkv"):
        B.tmixTailForward(x, x, x, x, x, v.view(2, 64), v, v)
    y = torch.zeros(5, 128)
    with pytest.raises(ValueError, match="g .* must be"):
        B.tmixTailForward(y, y, y, y, y[:4], v.view(2, 64), v, v)


def differentiable_calls():
    """Each differentiable form on host tensors, by the name of its arguments."""
    x, v, mix = torch.ones(2, 3, 64), torch.ones(64), torch.ones(6, 64)
    tail = {k: torch.ones(2, 3, 64) for k in ("wkv", "r", "k", "v", "g")}
    return [(lambda x: B.dropout(x, 0.1, 0), dict(x=x)),
            (B.residualNorm, dict(x=x, branch=x.clone(), weight=v, bias=v.clone())),
            (B.tokenMix, dict(x=x, mix=mix, prev=torch.ones(2, 64))),
            (B.tmixTail, dict(**tail, rk=torch.ones(1, 64), weight=v, bias=v.clone()))]


@pytest.mark.parametrize("recorded", [False, True])
def test_tangents_are_refused(recorded):
    from torch.autograd import forward_ad
    for f, args in differentiable_calls():
        for name in args:
            with forward_ad.dual_level():
                dual = forward_ad.make_dual(args[name].clone().requires_grad_(recorded), torch.ones_like(args[name]))
                with pytest.raises(ValueError, match=f"^{name} carries a tangent"):
                    f(**{**args, name: dual})


def test_differentiable_forms_on_the_host_are_refused():
    for f, args in differentiable_calls():
        for name, t in args.items():
            for bad in (t.clone().requires_grad_(True), [1.0]):
                with pytest.raises(ValueError, match="CUDA tensor"):
                    f(**{**args, name: bad})
