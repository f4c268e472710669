"""CPU tests of the block operators (layer norm, projections, 8-bit
checkpoints): every refusal happens on the host, before anything launches."""
from __future__ import annotations

import ctypes
import os
import subprocess
import sys

import pytest
import torch

from swiftrwkv_b200 import _lib
from swiftrwkv_b200 import block as B

FAKE = ctypes.c_void_p(0x1000)   # aligned, never dereferenced: checks fail first
ODD = ctypes.c_void_p(0x1001)
HALF = ctypes.c_void_p(0x1008)   # 8-byte aligned only
F32, BF16, F16 = _lib.F32, _lib.BF16, _lib.F16


def st(name, *a):
    return _lib.status(name, *a)


def norm_fwd(dt=BF16, x=FAKE, wdt=F32, w=FAKE, b=FAKE, eps=1e-5, y=FAKE, mean=FAKE, rstd=FAKE, c=None, e=None, rows=4,
             D=64):
    return st("rwkv_layer_norm_forward", dt, x, wdt, w, b, ctypes.c_float(eps), y, mean, rstd, c, e, rows, D, None)


def test_layer_norm_forward_refusals():
    assert norm_fwd(dt=7) == _lib.E_DTYPE
    assert norm_fwd(wdt=-1) == _lib.E_DTYPE
    for k in ("x", "w", "b", "y"):
        assert norm_fwd(**{k: None}) == _lib.E_NULL
    assert norm_fwd(mean=None) == _lib.E_NULL       # statistics come together
    assert norm_fwd(c=FAKE) == _lib.E_NULL          # so do codes and exps
    assert norm_fwd(rows=0) == _lib.E_SHAPE
    assert norm_fwd(D=0) == _lib.E_SHAPE
    assert norm_fwd(D=(1 << 30) + 8) == _lib.E_SHAPE
    assert norm_fwd(eps=-1.0) == _lib.E_SHAPE
    assert norm_fwd(x=ODD) == _lib.E_UNSUPPORTED
    assert b"aligned" in _lib.lib().rwkv_last_error()


def norm_bwd(dt=BF16, dy=FAKE, x=FAKE, c=None, e=None, wdt=F32, w=FAKE, mean=FAKE, rstd=FAKE, dres=None, dx=FAKE,
             dw=FAKE, db=FAKE, rows=4, D=64, ws=FAKE, n=1 << 30):
    return st("rwkv_layer_norm_backward", dt, dy, x, c, e, wdt, w, mean, rstd, dres, dx, dw, db, rows, D, ws, n, None)


def test_layer_norm_backward_refusals():
    assert norm_bwd(dt=3) == _lib.E_DTYPE
    for k in ("dy", "w", "mean", "rstd", "dx"):
        assert norm_bwd(**{k: None}) == _lib.E_NULL
    assert norm_bwd(x=None) == _lib.E_NULL                   # neither x nor its checkpoint
    assert norm_bwd(c=FAKE, e=FAKE) == _lib.E_NULL           # both
    assert norm_bwd(x=None, c=FAKE) == _lib.E_NULL
    assert norm_bwd(db=None) == _lib.E_NULL
    need = _lib.lib().rwkv_layer_norm_backward_workspace_size(4, 64)
    assert need > 0
    assert norm_bwd(n=need - 1) == _lib.E_WORKSPACE
    assert norm_bwd(ws=None) == _lib.E_WORKSPACE
    assert norm_bwd(ws=HALF) == _lib.E_UNSUPPORTED
    assert norm_bwd(dres=ODD) == _lib.E_UNSUPPORTED
    assert norm_bwd(rows=-1) == _lib.E_SHAPE


def test_checkpoint_refusals():
    pack = lambda dt=BF16, x=FAKE, c=FAKE, e=FAKE, rows=4, D=64: st("rwkv_ckpt8_pack", dt, x, c, e, rows, D, None)
    assert pack(dt=9) == _lib.E_DTYPE
    for k in ("x", "c", "e"):
        assert pack(**{k: None}) == _lib.E_NULL
    assert pack(rows=0) == _lib.E_SHAPE
    assert pack(D=-3) == _lib.E_SHAPE
    assert pack(x=ODD) == _lib.E_UNSUPPORTED
    vals = lambda act=0, dt=BF16, out=FAKE, rows=1: st("rwkv_ckpt8_values", FAKE, FAKE, act, dt, out, rows, 32, None)
    assert vals(act=4) == _lib.E_UNSUPPORTED
    assert vals(dt=5) == _lib.E_DTYPE
    assert vals(out=None) == _lib.E_NULL
    assert vals(rows=0) == _lib.E_SHAPE
    back = lambda z=FAKE, c=None, e=None, act=1, dt=F32: st("rwkv_act_backward", dt, FAKE, z, c, e, act, FAKE, 2, 32, None)
    assert back(z=None) == _lib.E_NULL
    assert back(c=FAKE, e=FAKE) == _lib.E_NULL
    assert back(act=-1) == _lib.E_UNSUPPORTED
    assert back(dt=4) == _lib.E_DTYPE
    assert back(z=ODD) == _lib.E_UNSUPPORTED


def proj_fwd(dt=BF16, x=FAKE, w=FAKE, bdt=F32, b=None, act=0, ydt=BF16, res=None, y=FAKE, z=None, c=None, e=None,
             rows=4096, OUT=2048, IN=2048, ws=None, n=0):
    return st("rwkv_projection_forward", dt, x, w, bdt, b, act, ydt, res, y, z, c, e, rows, OUT, IN, ws, n, None)


def test_projection_forward_refusals():
    assert proj_fwd(dt=F32) == _lib.E_DTYPE
    assert proj_fwd(ydt=F16) == _lib.E_DTYPE          # the operands' own type, or fp32
    assert proj_fwd(b=FAKE, bdt=8) == _lib.E_DTYPE
    for k in ("x", "w", "y"):
        assert proj_fwd(**{k: None}) == _lib.E_NULL
    assert proj_fwd(c=FAKE) == _lib.E_NULL
    assert proj_fwd(rows=0) == _lib.E_SHAPE
    assert proj_fwd(IN=0) == _lib.E_SHAPE
    assert proj_fwd(rows=(1 << 26) + 1) == _lib.E_SHAPE
    assert proj_fwd(IN=2044) == _lib.E_UNSUPPORTED
    assert proj_fwd(OUT=2052) == _lib.E_UNSUPPORTED
    assert proj_fwd(act=9) == _lib.E_UNSUPPORTED
    assert proj_fwd(x=HALF) == _lib.E_UNSUPPORTED
    need = _lib.lib().rwkv_projection_forward_workspace_size(64, 256, 8192)
    assert need > 0
    assert proj_fwd(rows=64, OUT=256, IN=8192, ws=FAKE, n=need - 1) == _lib.E_WORKSPACE
    assert proj_fwd(rows=64, OUT=256, IN=8192) == _lib.E_WORKSPACE
    assert _lib.lib().rwkv_projection_forward_workspace_size(0, 256, 8192) == 0


def proj_dx(dt=BF16, dy=FAKE, w=FAKE, act=0, z=None, c=None, e=None, xdt=BF16, add=None, dx=FAKE, rows=4096, OUT=2048,
            IN=2048, ws=None, n=0):
    return st("rwkv_projection_dx", dt, dy, w, act, z, c, e, xdt, add, dx, rows, OUT, IN, ws, n, None)


def test_projection_dx_refusals():
    assert proj_dx(dt=F32) == _lib.E_DTYPE
    assert proj_dx(xdt=F16) == _lib.E_DTYPE
    for k in ("dy", "w", "dx"):
        assert proj_dx(**{k: None}) == _lib.E_NULL
    assert proj_dx(act=1) == _lib.E_NULL              # an activation needs its pre-activation
    assert proj_dx(z=FAKE, c=FAKE, e=FAKE) == _lib.E_NULL
    assert proj_dx(c=FAKE) == _lib.E_NULL
    assert proj_dx(act=-2) == _lib.E_UNSUPPORTED
    assert proj_dx(OUT=12) == _lib.E_UNSUPPORTED
    assert proj_dx(add=HALF) == _lib.E_UNSUPPORTED
    assert proj_dx(rows=-5) == _lib.E_SHAPE


def proj_dw(dt=BF16, dy=FAKE, act=0, x=FAKE, c=None, e=None, wdt=BF16, dw=FAKE, db=None, rows=4096, OUT=2048, IN=2048,
            ws=FAKE, n=1 << 40):
    return st("rwkv_projection_dw", dt, dy, act, x, c, e, wdt, dw, db, rows, OUT, IN, ws, n, None)


def test_projection_dw_refusals():
    assert proj_dw(dt=F32) == _lib.E_DTYPE
    assert proj_dw(wdt=F16) == _lib.E_DTYPE
    assert proj_dw(dy=None) == _lib.E_NULL
    assert proj_dw(dw=None) == _lib.E_NULL            # neither output
    assert proj_dw(x=None) == _lib.E_NULL
    assert proj_dw(c=FAKE, e=FAKE) == _lib.E_NULL
    assert proj_dw(act=5) == _lib.E_UNSUPPORTED
    assert proj_dw(IN=100) == _lib.E_UNSUPPORTED
    assert proj_dw(rows=0) == _lib.E_SHAPE
    L = _lib.lib()
    dense = L.rwkv_projection_dw_workspace_size(4096, 2048, 2048, 0)
    kept = L.rwkv_projection_dw_workspace_size(4096, 2048, 2048, 1)
    assert kept >= dense + 4096 * 2048 * 2            # the restored operand
    assert proj_dw(act=1, n=kept - 1) == _lib.E_WORKSPACE
    assert proj_dw(db=ODD) == _lib.E_UNSUPPORTED


def test_python_refusals_come_before_any_launch():
    x = torch.zeros(4, 64)
    with pytest.raises(ValueError, match="CUDA tensor"):
        B.layerNormForward(x, torch.ones(64), torch.zeros(64))
    with pytest.raises(ValueError, match="CUDA tensor"):
        B.checkpoint8(x)
    with pytest.raises(ValueError, match="CUDA tensor"):
        B.projectionForward(x, torch.zeros(8, 64))
    host = B.Checkpoint8(torch.zeros(4, 64, dtype=torch.int8), torch.ones(4, 2, dtype=torch.uint8), torch.bfloat16)
    with pytest.raises(ValueError, match="CUDA tensor"):
        B.checkpoint8Values(host)
    with pytest.raises(ValueError, match="Checkpoint8"):
        B.checkpoint8Values(x)
    with pytest.raises(ValueError, match="CUDA tensor"):
        B.layerNormBackward(x, host, torch.ones(64), torch.zeros(4), torch.ones(4))
    with pytest.raises(ValueError, match="activation"):
        B.activationBackward(x, x, "gelu")
    with pytest.raises(ValueError, match="activation"):
        B.projectionForward(x, x, act="silu")


def test_weight_gradient_without_x_asks_for_db_only(monkeypatch):
    monkeypatch.setattr(B, "_tensor", lambda name, t, *a, **k: t)  # a CPU tensor as far as the check that raises
    with pytest.raises(ValueError, match="only db"):
        B.projectionBackwardWeight(torch.zeros(4, 64, dtype=torch.bfloat16), None)


@pytest.mark.parametrize("rows,OUT,IN", [(1, 8, 8), (64, 2048, 8192), (129, 2048, 2048), (16384, 8192, 2048),
                                         (4093, 96, 2048), (1000, 256, 10240)])
def test_workspace_sizes_hold_whole_tiles(rows, OUT, IN):
    """A split product's partial sums are whole fp32 tiles of 128 x 128 or 128 x
    256, at least two of them; few-row forwards need none."""
    L = _lib.lib()
    for n in (L.rwkv_projection_forward_workspace_size(rows, OUT, IN), L.rwkv_projection_dx_workspace_size(rows, OUT, IN)):
        assert n % (128 * 128 * 4) == 0 and n // (128 * 128 * 4) != 1
    assert rows > 16 or L.rwkv_projection_forward_workspace_size(rows, OUT, IN) == 0


def test_sizes_past_31_bits_are_refused():
    """The entry points' sizes are ints, to which ctypes would cut 2^31 + 5 rows
    silently.  The tensors here are one element seen many times."""
    one = torch.zeros(1, 1, dtype=torch.bfloat16)
    many, wide = one.expand((1 << 32) + 5, 1), one.expand(1, (1 << 32) + 8)
    vec = torch.ones(1)
    for x in (many, wide, many.view(2, -1, 1) if many.is_contiguous() else many[None]):
        with pytest.raises(ValueError, match="rows or channels"):
            B.checkpoint8(x)
        with pytest.raises(ValueError, match="rows or channels"):
            B.layerNormForward(x, vec, vec)
        with pytest.raises(ValueError, match="rows or channels"):
            B.layerNormBackward(x, x, vec, vec, vec)
        with pytest.raises(ValueError, match="rows or channels"):
            B.activationBackward(x, x, "tanh")
        with pytest.raises(ValueError, match="rows or channels"):
            B.projectionForward(x, one)
        with pytest.raises(ValueError, match="rows or channels"):
            B.projectionBackwardInput(x, one)
        with pytest.raises(ValueError, match="rows or channels"):
            B.projectionBackwardWeight(x, x)
    codes = torch.zeros(1, 1, dtype=torch.int8).expand((1 << 31), 1)
    with pytest.raises(ValueError, match="rows or channels"):
        B.checkpoint8Values(B.Checkpoint8(codes, codes, torch.bfloat16))


def test_projection_widths_past_the_limit_are_refused(monkeypatch):
    monkeypatch.setattr(B, "_tensor", lambda name, t, *a, **k: t)  # a CPU tensor as far as the check that raises
    one = torch.zeros(1, 1, dtype=torch.bfloat16)
    x = one.expand(2, 8)
    for w in (one.expand((1 << 20) + 8, 8), one.expand(8, (1 << 32) + 8)):
        with pytest.raises(ValueError, match="at most 2\\^20"):
            B._weight(w, w.device, torch.bfloat16)
    with pytest.raises(ValueError, match="at most 2\\^20"):
        B.projectionBackwardWeight(x, one.expand(2, (1 << 20) + 8))


def test_what_is_no_tensor_is_refused(monkeypatch):
    with pytest.raises(ValueError, match="Checkpoint8"):
        B.checkpoint8Values(None)
    for x in (None, [1.0], 3.0):
        with pytest.raises(ValueError, match="CUDA tensor"):
            B.checkpoint8(x)
    monkeypatch.setattr(B, "_tensor", lambda name, t, *a, **k: t)
    with pytest.raises(ValueError, match="Checkpoint8"):
        B.projectionBackwardWeight(torch.zeros(4, 64, dtype=torch.bfloat16), [1.0])


def differentiable_calls():
    """Each differentiable form on host tensors, by the name of its arguments."""
    v, x, w, key, value = torch.ones(8), torch.ones(2, 8), torch.ones(16, 8), torch.ones(16, 8), torch.ones(8, 16)
    return [(B.layerNorm, dict(x=x, weight=v, bias=v)),
            (B.projection, dict(x=x, w=w, bias=torch.ones(16), residual=torch.ones(2, 16))),
            (B.channelMix, dict(x=x, key=key, value=value, residual=x))]


@pytest.mark.parametrize("recorded", [False, True])
def test_tangents_are_refused(recorded):
    """Forward mode would lose the tangent without a word: a derivative of zero."""
    from torch.autograd import forward_ad
    for f, args in differentiable_calls():
        for name in args:
            with forward_ad.dual_level():
                dual = forward_ad.make_dual(args[name].clone().requires_grad_(recorded), torch.ones_like(args[name]))
                with pytest.raises(ValueError, match=f"^{name} carries a tangent"):
                    f(**{**args, name: dual})
            with pytest.raises(ValueError, match=f"^{name} carries a tangent"):
                torch.func.jvp(lambda t: f(**{**args, name: t}), (args[name],), (args[name],))


def test_differentiable_forms_refuse_what_is_no_tensor():
    for f, args in differentiable_calls():
        for name in args:
            with pytest.raises(ValueError, match="CUDA tensor"):
                f(**{**args, name: [1.0]})


def test_layer_norm_workspace_of_long_rows():
    """Rows longer than the vector kernels take sum their columns in 64 blocks at
    most, and ask for no more."""
    size = _lib.lib().rwkv_layer_norm_backward_workspace_size
    assert size(4096, 65536) == 64 * 2 * 65536 * 4
    assert size(4096, 12289) == 64 * 2 * 12289 * 4
    assert size(40, 65536) == 40 * 2 * 65536 * 4
    assert size(4096, 12288) == 592 * 2 * 12288 * 4    # 16-bit rows of 1536 vectors


def test_a_torch_without_cuda_imports_and_refuses():
    code = """
import torch
for name in ("_cuda_getDevice", "_cuda_getCurrentRawStream"):
    delattr(torch._C, name)
from swiftrwkv_b200 import block as B
try:
    B.checkpoint8(torch.zeros(4, 64))
except ValueError as e:
    print(e)
"""
    root = os.path.dirname(os.path.dirname(os.path.abspath(_lib.__file__)))
    got = subprocess.run([sys.executable, "-c", code], cwd=root, capture_output=True, text=True, timeout=300)
    assert got.returncode == 0 and "a CUDA tensor is needed" in got.stdout, got.stderr


def test_projections_of_more_than_2_24_rows_are_refused():
    """2^24 rows are taken (here as far as the missing workspace), one more is not."""
    L, rows = _lib.lib(), 1 << 24
    for n, status in ((rows, _lib.E_WORKSPACE), (rows + 1, _lib.E_SHAPE)):
        assert proj_dw(rows=n, OUT=64, IN=64, ws=None, n=0) == status
    assert proj_fwd(rows=rows + 1, OUT=64, IN=64) == _lib.E_SHAPE
    assert proj_dx(rows=rows + 1, OUT=64, IN=64) == _lib.E_SHAPE
    # an accumulator takes 32768 rows: 512 splits of a 128 x 128 tile and the column sums
    assert L.rwkv_projection_dw_workspace_size(rows, 64, 64, 0) >= 512 * 128 * 128 * 4
    assert L.rwkv_projection_dw_workspace_size(rows + 1, 64, 64, 0) == 0


def test_capture_is_looked_up_on_the_tensors_device(monkeypatch):
    """A capture on another device than the tensors' is none of a call's business, one
    on theirs is, whatever device is current."""
    current = [0]

    class Device:
        def __init__(self, device):
            self.index = device.index

        def __enter__(self):
            self.before, current[0] = current[0], self.index

        def __exit__(self, *_):
            current[0] = self.before

    monkeypatch.setattr(B, "_current_device", lambda: current[0])
    monkeypatch.setattr(torch.cuda, "device", Device)
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: current[0] == 1)
    assert not B._capturing(torch.device("cuda", 0)) and B._capturing(torch.device("cuda", 1))
    current[0] = 1
    assert not B._capturing(torch.device("cuda", 0)) and B._capturing(torch.device("cuda", 1))
    assert not B._capturing(torch.device("cpu")) and current == [1]


def test_differentiable_forms_on_the_host_are_refused():
    """Recorded or not, and without their first argument, with a ValueError."""
    for f, args in differentiable_calls():
        for name, t in args.items():
            with pytest.raises(ValueError, match="CUDA tensor"):
                f(**{**args, name: t.clone().requires_grad_(True)})
        with pytest.raises(ValueError, match="CUDA tensor"):
            f(**{name: None if name == "x" else t.clone().requires_grad_(True) for name, t in args.items()})
