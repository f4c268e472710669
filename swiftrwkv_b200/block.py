"""The operators of an x070 block around the WKV path, forward and backward.

* Layer norm (ln0 / ln1 / ln2 / ln_out): `layerNormForward`,
  `layerNormBackward`, and `layerNorm`, differentiable.
* Projections with trainable weights (r / k / v / o, cmix key / value, the
  low-rank branches): `projectionForward` with bias, activation and residual in
  its epilogue, `projectionBackwardInput`, `projectionBackwardWeight`, and
  `projection`, differentiable.
* 8-bit activation checkpoints: `checkpoint8`, `checkpoint8Values`,
  `activationBackward`; every backward above takes a `Checkpoint8` in place of
  the activation it stands for.
* `channelMix`, the two projections of cmix around the squared ReLU,
  differentiable, with the pre-activation kept in 8 bits.
* Between them and the WKV path (kernel.py), each with its differentiable form:
  `tokenMixForward` / `tokenMixBackward` (`tokenMix`), the token shift and the
  interpolations that feed the projections; `tmixTailForward` /
  `tmixTailBackward` (`tmixTail`), the norm by head, bonus and gate that end the
  time mix; `residualNormForward` / `residualNormBackward` (`residualNorm`), a
  branch added to the residual stream, through dropout and scaled, and the sum
  normed; `dropoutForward` (`dropout`), whose mask is drawn from a counter and
  never stored.

The reference runs these as MLX layerNorm / matmul / elementwise ops under
MLX's autograd (Sources/RWKVGen/RWKVBlock.swift:163-307, X070Backbone.swift:
43-74); the C entry points are declared in include/rwkv_cuda.h.

Arrays are torch CUDA tensors of [..., D]; leading dimensions are rows, of any
number (also none).  All arithmetic runs in librwkvcuda, on the current stream
of the tensors' device.  Arguments that do not fit raise ValueError; a failed
CUDA call raises RWKVError.  The differentiable forms are for reverse mode, once:
they refuse inputs with a forward-mode tangent, and to record a graph while a
CUDA stream is being captured (capture the explicit forward and backward calls).
The explicit calls take their inputs as values: no gradient or tangent follows.
"""
from __future__ import annotations

from ctypes import ArgumentError
from dataclasses import dataclass
from functools import lru_cache

import torch
from torch.autograd.forward_ad import unpack_dual

from . import _lib
from ._lib import ACTS, BF16, F16, F32

_DT = {torch.float32: F32, torch.bfloat16: BF16, torch.float16: F16}
_HALF = (torch.bfloat16, torch.float16)
CKPT_GROUP = 32  # channels per scale of a checkpoint
_MAX = 2**31 - 1
_MAX_WIDTH = 1 << 20  # of a projection
_MAX_DROPOUT = 1 << 40  # elements


@dataclass
class Checkpoint8:
    """An activation [..., D] in 8 bits: int8 codes [..., D] and one exponent
    byte per group of 32 channels, exps [..., ceil(D / 32)]; a code q stands
    for q * 2^(e - 127), within max|x| / 127.5 of the group (2^-127 where max|x| is
    smaller than 2^-120).  `dtype` is the activation's own type."""
    codes: torch.Tensor
    exps: torch.Tensor
    dtype: torch.dtype

    @property
    def shape(self):
        return self.codes.shape

    @property
    def device(self):
        return self.codes.device

    @property
    def nbytes(self):
        return self.codes.numel() + self.exps.numel()


# ---------------------------------------------------------------- plumbing
#
# A small call costs about as much on the host as on the device, so the functions
# below test what a correct call satisfies in one expression (_fits) and leave the
# finding of what is wrong, or the copying of what is strided, to _tensor.  Outputs
# come from empty_like or new_empty(*sizes): 1.3 to 1.5 us, where new_empty(tuple)
# takes 1.8 to 2.1 and torch.empty(tuple) 2.2.

def _public_raw_stream(device):
    return torch.cuda.current_stream(device).cuda_stream


# what torch.cuda.current_device() and current_stream(...).cuda_stream return,
# without building a Stream object (2 us of a small call's 10); a torch without
# CUDA has neither of these names
_current_device = getattr(torch._C, "_cuda_getDevice", torch.cuda.current_device)
_raw_stream = getattr(torch._C, "_cuda_getCurrentRawStream", _public_raw_stream)


# what the entry points find wrong with arguments that the checks here let pass (eps, sizes)
_BAD_ARGUMENT = (_lib.E_NULL, _lib.E_SHAPE, _lib.E_DTYPE, _lib.E_UNSUPPORTED)


def _call(dev, name, *args):
    """An entry point on `dev` and its current stream (appended)."""
    fn, k = getattr(_lib.lib(), name), dev.index
    try:
        if k == _current_device():
            st = fn(*args, _raw_stream(k))
        else:
            with torch.cuda.device(dev):
                st = fn(*args, _raw_stream(k))
    except ArgumentError as e:  # an eps or a scale that is no number or too large for one
        raise ValueError(f"{name}: {e}") from None
    if not st:
        return
    why = _lib.lib().rwkv_last_error().decode()
    if st in _BAD_ARGUMENT:
        raise ValueError(why)
    raise _lib.RWKVError(name, st, why)


def _fits(t, dev, dtype, shape):
    return (type(t) in _TENSORS and t.dtype is dtype and t.shape == shape and t.device == dev and t.is_contiguous())


_TENSORS = (torch.Tensor, torch.nn.Parameter)


def _p(t):
    return None if t is None else t.data_ptr()


def _tensor(name, t, dev=None, dtypes=None, shape=None):
    """t, contiguous, after its checks."""
    if not isinstance(t, torch.Tensor) or not t.is_cuda:
        raise ValueError(f"{name}: a CUDA tensor is needed")
    if dev is not None and t.device != dev:
        raise ValueError(f"{name} is on {t.device}, the call's other tensors on {dev}")
    if t.dtype not in (dtypes or _DT):
        raise ValueError(f"{name}: dtype {t.dtype} not taken")
    if shape is not None and t.shape != shape:
        raise ValueError(f"{name} {tuple(t.shape)} must be {list(shape)}")
    return t if t.is_contiguous() else t.contiguous()


def _some(name, t, dtypes=None):
    """A call's first tensor [..., D], D >= 1, after its checks."""
    if (type(t) in _TENSORS and t.is_cuda and t.dtype in (dtypes or _DT) and 0 < t.numel() <= _MAX and t.dim() and
            t.is_contiguous()):
        return t
    # the entry points take ints, to which ctypes cuts what is longer
    if isinstance(t, torch.Tensor) and t.numel() > _MAX and t.dim() and max(t.shape[-1], t.numel() // t.shape[-1]) > _MAX:
        raise ValueError(f"{name} {tuple(t.shape)}: more than 2^31 - 1 rows or channels")
    t = _tensor(name, t, None, dtypes)
    if t.dim() < 1 or t.shape[-1] < 1:
        raise ValueError(f"{name} {tuple(t.shape)} must be [..., D] with D >= 1")
    return t


def _aligned(t):
    """t at a 16-byte aligned address (a view may start anywhere)."""
    return t if t is None or t.data_ptr() % 16 == 0 else t.clone(memory_format=torch.contiguous_format)


def _act(act):
    if act not in ACTS:
        raise ValueError(f"activation {act!r}: one of {sorted(ACTS)}")
    return ACTS[act]


def _activation(name, x, dev, dtype, shape):
    """An activation given as a tensor or as its checkpoint: (x, codes, exps)."""
    if type(x) is Checkpoint8 or isinstance(x, Checkpoint8):
        groups = shape[:-1] + (-(-shape[-1] // CKPT_GROUP),)
        codes, exps = x.codes, x.exps
        if not _fits(codes, dev, torch.int8, shape):
            codes = _tensor(f"{name}.codes", codes, dev, (torch.int8,), shape)
        if not _fits(exps, dev, torch.uint8, groups):
            exps = _tensor(f"{name}.exps", exps, dev, (torch.uint8,), groups)
        return None, codes, exps
    if not _fits(x, dev, dtype, shape):
        x = _tensor(name, x, dev, (dtype,), shape)
    return x, None, None


def _new_checkpoint(y, dtype):
    """An empty checkpoint of a tensor like y."""
    *lead, D = y.shape
    return Checkpoint8(torch.empty_like(y, dtype=torch.int8),
                       y.new_empty(*lead, -(-D // CKPT_GROUP), dtype=torch.uint8), dtype)


@lru_cache(maxsize=4096)
def _workspace_bytes(name, *sizes):
    return int(getattr(_lib.lib(), name + "_workspace_size")(*sizes))


def _workspace(nbytes, like):
    return like.new_empty(nbytes, dtype=torch.uint8) if nbytes else None


# ------------------------------------------------------- 8-bit checkpoints

def checkpoint8(x) -> Checkpoint8:
    """The 8-bit checkpoint of x [..., D]."""
    x = _some("x", x)
    ck = _new_checkpoint(x, x.dtype)
    n, D = x.numel(), x.shape[-1]
    if n:
        _call(x.device, "rwkv_ckpt8_pack", _DT[x.dtype], x.data_ptr(), ck.codes.data_ptr(), ck.exps.data_ptr(), n // D, D)
    return ck


def checkpoint8Values(ck: Checkpoint8, act: str = "none", dtype=None):
    """What a checkpoint stands for, or the activation behind a checkpointed
    pre-activation: act(value) in `dtype` (default: the activation's own)."""
    if not isinstance(ck, Checkpoint8):
        raise ValueError("checkpoint8Values: a Checkpoint8 is needed")
    a, dtype = _act(act), dtype or ck.dtype
    if dtype not in _DT:
        raise ValueError(f"checkpoint8Values: dtype {dtype} not taken")
    codes = _some("ck.codes", ck.codes, (torch.int8,))
    dev, shape = codes.device, codes.shape
    _, codes, exps = _activation("ck", ck, dev, None, shape)
    out = torch.empty_like(codes, dtype=dtype)
    n, D = codes.numel(), shape[-1]
    if n:
        _call(dev, "rwkv_ckpt8_values", codes.data_ptr(), exps.data_ptr(), a, _DT[dtype], out.data_ptr(), n // D, D)
    return out


def activationBackward(dy, pre, act: str):
    """dy * act'(pre) in dy's dtype; `pre` is a tensor or a Checkpoint8."""
    a = _act(act)
    dy = _some("dy", dy)
    dev, shape = dy.device, dy.shape
    z, codes, exps = _activation("pre", pre, dev, dy.dtype, shape)
    dz = torch.empty_like(dy)
    n, D = dy.numel(), shape[-1]
    if n:
        _call(dev, "rwkv_act_backward", _DT[dy.dtype], dy.data_ptr(), _p(z), _p(codes), _p(exps), a, dz.data_ptr(),
              n // D, D)
    return dz


# --------------------------------------------------------------- layer norm

def layerNormForward(x, weight, bias, eps: float = 1e-5, checkpoint: bool = False):
    """Layer norm over the last dimension: (y, mean, rstd, ck).  mean / rstd
    [...] fp32 are what the backward pass needs; ck is the 8-bit checkpoint of x
    (None without `checkpoint`)."""
    x = _some("x", x)
    dev, shape = x.device, x.shape
    D = shape[-1]
    if not _fits(weight, dev, torch.float32, (D,)):
        weight = _tensor("weight", weight, dev, None, (D,))
    if not _fits(bias, dev, weight.dtype, (D,)):
        bias = _tensor("bias", bias, dev, (weight.dtype,), (D,))
    y = torch.empty_like(x)
    mean = x.new_empty(*shape[:-1], dtype=torch.float32) if len(shape) > 1 else x.new_empty((), dtype=torch.float32)
    rstd = torch.empty_like(mean)
    codes = exps = ck = None
    if checkpoint:
        ck = _new_checkpoint(x, x.dtype)
        codes, exps = ck.codes.data_ptr(), ck.exps.data_ptr()
    n = x.numel()
    if n:
        _call(dev, "rwkv_layer_norm_forward", _DT[x.dtype], x.data_ptr(), _DT[weight.dtype], weight.data_ptr(),
              bias.data_ptr(), eps, y.data_ptr(), mean.data_ptr(), rstd.data_ptr(), codes, exps, n // D, D)
    return y, mean, rstd, ck


def layerNormBackward(dy, x, weight, mean, rstd, dres=None, params: bool = True):
    """(dx, dweight, dbias) of layerNormForward.  x: its input, or the
    checkpoint of it; mean, rstd: its statistics; dres: the gradient that
    reaches x past the norm, added to dx.  Without `params` dweight and dbias
    are None."""
    dy = _some("dy", dy)
    dev, dt, shape = dy.device, dy.dtype, dy.shape
    D = shape[-1]
    xt, codes, exps = _activation("x", x, dev, dt, shape)
    if not _fits(weight, dev, torch.float32, (D,)):
        weight = _tensor("weight", weight, dev, None, (D,))
    lead = shape[:-1]
    if not _fits(mean, dev, torch.float32, lead):
        mean = _tensor("mean", mean, dev, (torch.float32,), lead)
    if not _fits(rstd, dev, torch.float32, lead):
        rstd = _tensor("rstd", rstd, dev, (torch.float32,), lead)
    if dres is not None and not _fits(dres, dev, dt, shape):
        dres = _tensor("dres", dres, dev, (dt,), shape)
    dx = torch.empty_like(dy)
    rows = dy.numel() // D
    dw = torch.empty_like(weight) if params else None
    db = torch.empty_like(weight) if params else None
    if not rows:
        return dx, dw.zero_() if params else None, db.zero_() if params else None
    n = _workspace_bytes("rwkv_layer_norm_backward", rows, D) if params else 0
    ws = _workspace(n, dy)
    _call(dev, "rwkv_layer_norm_backward", _DT[dt], dy.data_ptr(), _p(xt), _p(codes), _p(exps), _DT[weight.dtype],
          weight.data_ptr(), mean.data_ptr(), rstd.data_ptr(), _p(dres), dx.data_ptr(), _p(dw), _p(db), rows, D, _p(ws),
          n)
    return dx, dw, db


# -------------------------------------------------------------- projections

def _weight(w, dev, dtype):
    """(w, OUT, IN) after its checks."""
    if not (type(w) in _TENSORS and w.dtype is dtype and w.device == dev and w.is_contiguous()):
        w = _tensor("w", w, dev, (dtype,))
    if w.dim() != 2:
        raise ValueError(f"w {tuple(w.shape)} must be [OUT, IN]")
    OUT, IN = w.shape
    if OUT % 8 or IN % 8 or not 0 < OUT <= _MAX_WIDTH or not 0 < IN <= _MAX_WIDTH:
        raise ValueError(f"w {tuple(w.shape)}: OUT and IN must be multiples of 8, at most 2^20")
    return _aligned(w), OUT, IN


def _result_dtype(fn, dtype, own):
    if dtype is None or dtype is own:
        return own
    if dtype is not torch.float32:
        raise ValueError(f"{fn}: out_dtype {dtype} ({own} or fp32)")
    return dtype


def projectionForward(x, w, bias=None, act: str = "none", residual=None, checkpoint: bool = False,
                      preactivation: bool = False, out_dtype=None):
    """y = act(x w^T + bias) + residual: (y, kept).  x [..., IN] and w [OUT, IN]
    in one 16-bit type; y and residual in `out_dtype` (that type, or fp32).
    kept is the 8-bit checkpoint of z = x w^T + bias with `checkpoint`, z itself
    with `preactivation`, else None."""
    a = _act(act)
    x = _aligned(_some("x", x, _HALF))
    dev, dt = x.device, x.dtype
    w, OUT, IN = _weight(w, dev, dt)
    if checkpoint and preactivation:
        raise ValueError("projectionForward: keep either the checkpoint or the pre-activation")
    ydt = _result_dtype("projectionForward", out_dtype, dt)
    lead = tuple(x.shape)
    if lead[-1] != IN:
        raise ValueError(f"x {lead} must be [..., {IN}]")
    shape = lead[:-1] + (OUT,)
    bdt = F32
    if bias is not None:
        if not _fits(bias, dev, torch.float32, (OUT,)):
            bias = _tensor("bias", bias, dev, None, (OUT,))
        bias = _aligned(bias)
        bdt = _DT[bias.dtype]
    if residual is not None:
        if not _fits(residual, dev, ydt, shape):
            residual = _tensor("residual", residual, dev, (ydt,), shape)
        residual = _aligned(residual)
    y = x.new_empty(*shape, dtype=ydt)
    codes = exps = kept = z = None
    if checkpoint:
        kept = _new_checkpoint(y, dt)
        codes, exps = kept.codes.data_ptr(), kept.exps.data_ptr()
    elif preactivation:
        kept = x.new_empty(*shape)
        z = kept.data_ptr()
    rows = x.numel() // IN
    if rows:
        n = _workspace_bytes("rwkv_projection_forward", rows, OUT, IN)
        ws = _workspace(n, x)
        _call(dev, "rwkv_projection_forward", _DT[dt], x.data_ptr(), w.data_ptr(), bdt, _p(bias), a, _DT[ydt],
              _p(residual), y.data_ptr(), z, codes, exps, rows, OUT, IN, _p(ws), n)
    return y, kept


def projectionBackwardInput(dy, w, pre=None, act: str = "none", addend=None, out_dtype=None):
    """dx = (dy w) * act'(pre) + addend in dy's dtype (or `out_dtype` fp32).
    pre [..., IN]: the pre-activation of the layer below, a tensor or a
    Checkpoint8 (None: the plain product); addend in dx's type."""
    a = _act(act)
    dy = _aligned(_some("dy", dy, _HALF))
    dev, dt = dy.device, dy.dtype
    w, OUT, IN = _weight(w, dev, dt)
    lead = tuple(dy.shape)
    if lead[-1] != OUT:
        raise ValueError(f"dy {lead} must be [..., {OUT}]")
    xdt = _result_dtype("projectionBackwardInput", out_dtype, dt)
    shape = lead[:-1] + (IN,)
    z = codes = exps = None
    if pre is not None:
        z, codes, exps = _activation("pre", pre, dev, dt, shape)
        z, codes = _aligned(z), _aligned(codes)
    elif a:
        raise ValueError(f"projectionBackwardInput: act {act!r} needs pre")
    if addend is not None:
        if not _fits(addend, dev, xdt, shape):
            addend = _tensor("addend", addend, dev, (xdt,), shape)
        addend = _aligned(addend)
    dx = dy.new_empty(*shape, dtype=xdt)
    rows = dy.numel() // OUT
    if rows:
        n = _workspace_bytes("rwkv_projection_dx", rows, OUT, IN)
        ws = _workspace(n, dy)
        _call(dev, "rwkv_projection_dx", _DT[dt], dy.data_ptr(), w.data_ptr(), a, _p(z), _p(codes), _p(exps), _DT[xdt],
              _p(addend), dx.data_ptr(), rows, OUT, IN, _p(ws), n)
    return dx


def projectionBackwardWeight(dy, x, act: str = "none", bias: bool = False, out_dtype=None):
    """(dw, db): dw [OUT, IN] = sum over rows of dy act(x)^T in dy's dtype (or
    `out_dtype` fp32), db [OUT] fp32 = sum over rows of dy (None without
    `bias`).  x [..., IN]: the projection's input, or with `act` the
    pre-activation behind it; a tensor or a Checkpoint8; None: only db (dw is
    None).  act(x) is rounded to dy's dtype for the product: in fp16 it is
    infinite past 65504 (relu2: from x = 256 on), also with fp32 results."""
    a = _act(act)
    dy = _aligned(_some("dy", dy, _HALF))
    dev, dt = dy.device, dy.dtype
    if x is None:
        if not bias or a:
            raise ValueError("projectionBackwardWeight: without x only db can be asked for")
    elif not isinstance(x, (torch.Tensor, Checkpoint8)) or len(x.shape) < 1:
        raise ValueError("projectionBackwardWeight: x must be a tensor [..., IN] or the Checkpoint8 of one")
    lead = tuple(dy.shape)
    OUT, IN = lead[-1], 8 if x is None else x.shape[-1]
    if OUT % 8 or IN % 8 or not IN or OUT > _MAX_WIDTH or IN > _MAX_WIDTH:
        raise ValueError(f"projectionBackwardWeight: OUT={OUT} and IN={IN} must be multiples of 8, at most 2^20")
    wdt = _result_dtype("projectionBackwardWeight", out_dtype, dt)
    xt = codes = exps = dw = None
    if x is not None:
        xt, codes, exps = _activation("x", x, dev, dt, lead[:-1] + (IN,))
        xt, codes = _aligned(xt), _aligned(codes)
        dw = dy.new_empty(OUT, IN, dtype=wdt)
    db = dy.new_empty(OUT, dtype=torch.float32) if bias else None
    rows = dy.numel() // OUT
    if not rows:
        return dw if dw is None else dw.zero_(), db.zero_() if bias else None
    n = _workspace_bytes("rwkv_projection_dw", rows, OUT, IN, int(codes is not None or a != 0))
    ws = _workspace(n, dy)
    _call(dev, "rwkv_projection_dw", _DT[dt], dy.data_ptr(), a, _p(xt), _p(codes), _p(exps), _DT[wdt], _p(dw), _p(db),
          rows, OUT, IN, _p(ws), n)
    return dw, db


# ----------------------------------------------------------------- dropout

_WORD = 1 << 64


def _draw(p, seed, offset, dev):
    """(seed, offset, the state or None) of a call with dropout, after their checks.
    The caller holds the state, which may be a copy, until its call is made."""
    if not isinstance(p, (int, float)) or not 0.0 <= p <= 1.0:
        raise ValueError(f"p={p!r} must be a number in 0..1")
    if not isinstance(offset, int) or not 0 <= offset < _WORD:
        raise ValueError(f"offset={offset!r} must be an integer in 0..2^64 - 1")
    if type(seed) is int or isinstance(seed, int):
        if not 0 <= seed < _WORD:
            raise ValueError(f"seed={seed!r} must be in 0..2^64 - 1")
        return seed, offset, None
    if not isinstance(seed, torch.Tensor):
        raise ValueError(f"seed={seed!r} must be an integer or a CUDA tensor int64 [2]")
    return 0, offset, _tensor("seed", seed, dev, (torch.int64,), (2,))


def _number(name, v):
    if not isinstance(v, (int, float)):
        raise ValueError(f"{name}={v!r} must be a number")
    return v


def dropoutForward(x, p: float, seed, offset: int = 0):
    """x / (1 - q) where kept and 0 where dropped, q = round(65536 p) / 65536; the
    gradient is the same call on dy.  An element is dropped by its place in x,
    `seed` and `offset` alone (rwkv_cuda.h has the generator), so that every call of a
    program with masks of its own takes another (seed, offset), and the backward pass
    the forward's.  x [..., D]: 2^40 elements at most.  seed: an integer, or a CUDA
    tensor int64 [2] that is read when the kernel runs (the seed, and what is added to
    `offset`): a captured graph then draws anew where the program changes the tensor
    between replays."""
    if isinstance(x, torch.Tensor) and x.numel() > _MAX:  # places alone count, not rows or channels
        if x.numel() > _MAX_DROPOUT:
            raise ValueError(f"x {tuple(x.shape)}: more than 2^40 elements")
        x = _tensor("x", x)
    else:
        x = _some("x", x)
    x = _aligned(x)
    dev = x.device
    seed, offset, state = _draw(p, seed, offset, dev)
    y = torch.empty_like(x)
    n = x.numel()
    if n:
        _call(dev, "rwkv_dropout", _DT[x.dtype], x.data_ptr(), p, seed, offset, _p(state), y.data_ptr(), n)
    return y


# ----------------------------------------------------------- residual norm

def residualNormForward(x, branch, weight, bias, eps: float = 1e-5, scale: float = 1.0, p: float = 0.0, seed=0,
                        offset: int = 0, checkpoint: bool = False):
    """s = x + scale dropout(branch) and its layer norm y: (s, y, mean, rstd, ck).
    x, branch [..., D] in one type, D a multiple of 8, at most 12288 (6144 in fp32).
    y, the statistics and ck (the 8-bit checkpoint of s; None without `checkpoint`)
    are those of the sum in fp32, before it is rounded to x's type.  p, seed,
    offset: as in dropoutForward, by the places in branch."""
    x = _some("x", x)
    dev, dt, shape = x.device, x.dtype, x.shape
    D = shape[-1]
    if not _fits(branch, dev, dt, shape):
        branch = _tensor("branch", branch, dev, (dt,), shape)
    if not _fits(weight, dev, torch.float32, (D,)):
        weight = _tensor("weight", weight, dev, None, (D,))
    if not _fits(bias, dev, weight.dtype, (D,)):
        bias = _tensor("bias", bias, dev, (weight.dtype,), (D,))
    seed, offset, state = _draw(p, seed, offset, dev)
    xp, bp, wp, cp = x.data_ptr(), branch.data_ptr(), weight.data_ptr(), bias.data_ptr()
    if (xp | bp | wp | cp) & 15:
        x, branch, weight, bias = map(_aligned, (x, branch, weight, bias))
        xp, bp, wp, cp = x.data_ptr(), branch.data_ptr(), weight.data_ptr(), bias.data_ptr()
    s, y = torch.empty_like(x), torch.empty_like(x)
    mean = x.new_empty(*shape[:-1], dtype=torch.float32) if len(shape) > 1 else x.new_empty((), dtype=torch.float32)
    rstd = torch.empty_like(mean)
    codes = exps = ck = None
    if checkpoint:
        ck = _new_checkpoint(x, dt)
        codes, exps = ck.codes.data_ptr(), ck.exps.data_ptr()
    n = x.numel()
    if n:
        _call(dev, "rwkv_residual_norm_forward", _DT[dt], xp, bp, _number("scale", scale), p, seed, offset, _p(state),
              _DT[weight.dtype], wp, cp, eps, s.data_ptr(), y.data_ptr(), mean.data_ptr(), rstd.data_ptr(), codes, exps,
              n // D, D)
    return s, y, mean, rstd, ck


def residualNormBackward(dy, s, weight, mean, rstd, dres=None, scale: float = 1.0, p: float = 0.0, seed=0,
                         offset: int = 0, params: bool = True):
    """(dx, dbranch, dweight, dbias) of residualNormForward.  s: its sum, or the
    checkpoint of it; mean, rstd: its statistics; dres: the gradient that reaches s
    past the norm.  Where nothing is dropped or scaled dbranch is dx itself.  Without
    `params` dweight and dbias are None."""
    dy = _some("dy", dy)
    dev, dt, shape = dy.device, dy.dtype, dy.shape
    seed, offset, state = _draw(p, seed, offset, dev)
    if _number("scale", scale) == 1.0 and round(65536 * p) == 0:
        dx, dw, db = layerNormBackward(dy, s, weight, mean, rstd, dres, params)
        return dx, dx, dw, db
    dy, D = _aligned(dy), shape[-1]
    st, codes, exps = _activation("s", s, dev, dt, shape)
    st, codes = _aligned(st), _aligned(codes)
    if not _fits(weight, dev, torch.float32, (D,)):
        weight = _tensor("weight", weight, dev, None, (D,))
    weight = _aligned(weight)
    lead = shape[:-1]
    if not _fits(mean, dev, torch.float32, lead):
        mean = _tensor("mean", mean, dev, (torch.float32,), lead)
    if not _fits(rstd, dev, torch.float32, lead):
        rstd = _tensor("rstd", rstd, dev, (torch.float32,), lead)
    if dres is not None:
        if not _fits(dres, dev, dt, shape):
            dres = _tensor("dres", dres, dev, (dt,), shape)
        dres = _aligned(dres)
    dx, dbranch = torch.empty_like(dy), torch.empty_like(dy)
    rows = dy.numel() // D
    dw = torch.empty_like(weight) if params else None
    db = torch.empty_like(weight) if params else None
    if not rows:
        return dx, dbranch, dw.zero_() if params else None, db.zero_() if params else None
    n = _workspace_bytes("rwkv_residual_norm_backward", rows, D) if params else 0
    ws = _workspace(n, dy)
    _call(dev, "rwkv_residual_norm_backward", _DT[dt], dy.data_ptr(), _p(st), _p(codes), _p(exps), _DT[weight.dtype],
          weight.data_ptr(), mean.data_ptr(), rstd.data_ptr(), _p(dres), scale, p, seed, offset, _p(state),
          dx.data_ptr(), dbranch.data_ptr(), _p(dw), _p(db), rows, D, _p(ws), n)
    return dx, dbranch, dw, db


# --------------------------------------------------------------- token mix

def _mix_args(x, mix, prev, lengths):
    """tokenMix's inputs after their checks."""
    x = _some("x", x)
    shape = x.shape
    if len(shape) != 3:
        raise ValueError(f"x {tuple(shape)} must be [B, T, D]")
    dev, (B, _, D) = x.device, shape
    if not (type(mix) in _TENSORS and mix.dtype is torch.float32 and mix.device == dev and mix.is_contiguous()):
        mix = _tensor("mix", mix, dev)
    ways = mix.shape
    if len(ways) != 2 or ways[1] != D or not 1 <= ways[0] <= 6:
        raise ValueError(f"mix {tuple(ways)} must be [J, {D}], J in 1..6")
    if prev is not None:
        if not _fits(prev, dev, x.dtype, (B, D)):
            prev = _tensor("prev", prev, dev, (x.dtype,), (B, D))
    if lengths is not None and not _fits(lengths, dev, torch.int32, (B,)):
        lengths = _tensor("lengths", lengths, dev, (torch.int32,), (B,))
    if (x.data_ptr() | mix.data_ptr() | (prev.data_ptr() if prev is not None else 0)) & 15:
        x, mix, prev = map(_aligned, (x, mix, prev))
    return x, mix, prev, lengths


_ADDRESSES = [_lib.P * n for n in range(7)]


def _addresses(ts):
    """A host array of the addresses of tensors (None: NULL)."""
    return _ADDRESSES[len(ts)](*[_p(t) for t in ts])


def _steps(t, n):
    """A host array of the addresses of t[0] .. t[n - 1]."""
    at, step = t.data_ptr(), t.stride(0) * t.element_size()
    return _ADDRESSES[n](*range(at, at + n * step, step)) if step else _ADDRESSES[n](*[at] * n)


def _token_mix(x, mix, prev, lengths, ys):
    """tokenMixForward into the tensors or addresses ys: last."""
    B, T, D = x.shape
    last = x.new_empty(B, D)
    if x.numel():
        _call(x.device, "rwkv_token_mix_forward", _DT[x.dtype], x.data_ptr(), _DT[mix.dtype], mix.data_ptr(), _p(prev),
              _p(lengths), ys, last.data_ptr(), B, T, D, len(ys))
    elif B:
        last.copy_(prev) if prev is not None else last.zero_()
    return last


def tokenMixForward(x, mix, prev=None, lengths=None):
    """Each token interpolated with the one before it: (y, last).  x [B, T, D], D a
    multiple of 8; mix [J, D], J in 1..6, in fp32, bf16 or fp16; prev [B, D] in x's
    type: the token before the first (None: zeros).
        y[j, b, t] = x[b, t] + (x[b, t-1] - x[b, t]) mix[j]
    lengths: int32 [B] of right-padded sequences, taken as 0..T (None: all T); from a
    sequence's length on x is not read and y is 0.  last [B, D] is each sequence's last
    token (prev where it is empty), the next call's prev."""
    x, mix, prev, lengths = _mix_args(x, mix, prev, lengths)
    J = mix.shape[0]
    y = x.new_empty(J, *x.shape)
    return y, _token_mix(x, mix, prev, lengths, _steps(y, J))


def tokenMixBackward(dys, x, mix, prev=None, lengths=None, dlast=None, params: bool = True):
    """(dx, dmix, dprev) of tokenMixForward.  dys: [J, B, T, D], or J tensors [B, T, D]
    of which any may be None (zeros); dlast [B, D]: the gradient of last (None: zeros).
    dx is 0 from a sequence's length on, where dys are not read.  dmix [J, D] in mix's
    type, None without `params`; dprev is None without prev."""
    x, mix, prev, lengths = _mix_args(x, mix, prev, lengths)
    dev, dt, shape, J = x.device, x.dtype, x.shape, mix.shape[0]
    B, T, D = shape
    if isinstance(dys, torch.Tensor):
        dys = _aligned(dys if _fits(dys, dev, dt, (J, *shape)) else _tensor("dys", dys, dev, (dt,), (J, *shape)))
        addresses = _steps(dys, J)
    else:
        if not isinstance(dys, (list, tuple)) or len(dys) != J:
            raise ValueError(f"dys: a tensor [{J}, B, T, D] or {J} tensors [B, T, D] are needed")
        dys = [t if t is None or _fits(t, dev, dt, shape) else _tensor("dys", t, dev, (dt,), shape) for t in dys]
        at = [0 if t is None else t.data_ptr() for t in dys]
        if any([a & 15 for a in at]):
            dys = [_aligned(t) for t in dys]
            at = [0 if t is None else t.data_ptr() for t in dys]
        addresses = _ADDRESSES[J](*at)
    if dlast is not None:
        dlast = _aligned(dlast if _fits(dlast, dev, dt, (B, D)) else _tensor("dlast", dlast, dev, (dt,), (B, D)))
    dx = torch.empty_like(x)
    dmix = torch.empty_like(mix) if params else None
    dprev = torch.empty_like(prev) if prev is not None else None
    if not x.numel():
        if dprev is not None:
            dprev.copy_(dlast) if dlast is not None else dprev.zero_()
        return dx, dmix.zero_() if params else None, dprev
    n = _workspace_bytes("rwkv_token_mix_backward", _DT[dt], B, T, D, J) if params else 0
    ws = _workspace(n, x)
    _call(dev, "rwkv_token_mix_backward", _DT[dt], addresses, x.data_ptr(), _DT[mix.dtype], mix.data_ptr(), _p(prev),
          _p(lengths), _p(dlast), dx.data_ptr(), _p(dmix), _p(dprev), B, T, D, J, _p(ws), n)
    return dx, dmix, dprev


# -------------------------------------------------------- tail of the time mix

_TAIL = ("wkv", "r", "k", "v", "g", "dout")


def _tail_args(rk, weight, bias, *ts):
    """(inputs, parameters, addresses of both, H, S) of tmixTail after their checks; ts as in _TAIL."""
    wkv = _some("wkv", ts[0])
    dev, dt, shape = wkv.device, wkv.dtype, wkv.shape
    if not (type(rk) in _TENSORS and rk.dtype is torch.float32 and rk.device == dev and rk.is_contiguous()):
        rk = _tensor("rk", rk, dev)
    if rk.dim() != 2 or not rk.numel():
        raise ValueError(f"rk {tuple(rk.shape)} must be [H, S]")
    H, S = rk.shape
    D = H * S
    if shape[-2:] == (H, S):
        other = shape[:-2] + (D,)
        # of one head also as [..., 1 token, D]
        more = shape[:-1] + (H, S) if H == 1 else other
    elif shape[-1] == D:
        other = more = shape[:-1] + (H, S)
    else:
        raise ValueError(f"wkv {tuple(shape)} must be [..., {H}, {S}] or [..., {D}]")
    ins = [wkv]
    for i, t in enumerate(ts[1:], 1):
        if not _fits(t, dev, dt, shape) and not _fits(t, dev, dt, other):
            t = _tensor(_TAIL[i], t, dev, (dt,))
            if t.shape not in (shape, other, more):
                raise ValueError(f"{_TAIL[i]} {tuple(t.shape)} must be {list(shape)} or {list(other)}")
        ins.append(t)
    if not _fits(weight, dev, rk.dtype, (D,)):
        weight = _tensor("weight", weight, dev, (rk.dtype,), (D,))
    if not _fits(bias, dev, rk.dtype, (D,)):
        bias = _tensor("bias", bias, dev, (rk.dtype,), (D,))
    ps = (rk, weight, bias)
    at = [t.data_ptr() for t in ins], [t.data_ptr() for t in ps]
    if any([a & 15 for a in at[0] + at[1]]):
        ins, ps = [_aligned(t) for t in ins], [_aligned(t) for t in ps]
        at = [t.data_ptr() for t in ins], [t.data_ptr() for t in ps]
    return ins, ps, at, H, S


def tmixTailForward(wkv, r, k, v, g, rk, weight, bias, eps: float = 64e-5):
    """The end of the time mix, per head of S channels (32, 64, 128 or 256):
    ((wkv - mean) rstd weight + bias + (sum r k rk) v) g, in g's shape.  wkv, r, k, v,
    g: [..., H, S] or [..., H S], in one type; rk [H, S], weight and bias [H S], in
    fp32, bf16 or fp16.  The training form of kernel.wkvTail."""
    ins, ps, at, H, S = _tail_args(rk, weight, bias, wkv, r, k, v, g)
    wkv, out = ins[0], torch.empty_like(ins[4])
    n = wkv.numel()
    if n:
        _call(wkv.device, "rwkv_tmix_tail_forward", _DT[wkv.dtype], *at[0], _DT[ps[0].dtype], *at[1], eps, out.data_ptr(),
              n // (H * S), H, S)
    return out


def tmixTailBackward(dout, wkv, r, k, v, g, rk, weight, bias, eps: float = 64e-5, params: bool = True):
    """(dwkv, dr, dk, dv, dg, drk, dweight, dbias) of tmixTailForward, each in its
    input's shape and type.  Without `params` the last three are None."""
    ins, ps, at, H, S = _tail_args(rk, weight, bias, wkv, r, k, v, g, dout)
    wkv = ins[0]
    grads = [torch.empty_like(t) for t in ins[:5]]
    pgrads = [torch.empty_like(t) for t in ps] if params else [None] * 3
    rows = wkv.numel() // (H * S)
    if not rows:
        return (*grads, *(t if t is None else t.zero_() for t in pgrads))
    n = _workspace_bytes("rwkv_tmix_tail_backward", rows, H, S) if params else 0
    ws = _workspace(n, wkv)
    _call(wkv.device, "rwkv_tmix_tail_backward", _DT[wkv.dtype], at[0][5], *at[0][:5], _DT[ps[0].dtype], *at[1], eps,
          *[t.data_ptr() for t in grads], *[_p(t) for t in pgrads], rows, H, S, _p(ws), n)
    return (*grads, *pgrads)


# --------------------------------------------------- the differentiable forms

def _capturing(device):
    """Whether the current stream of `device` is being captured."""
    if device.type != "cuda":
        return False
    if device.index == _current_device():
        return torch.cuda.is_current_stream_capturing()
    with torch.cuda.device(device):
        return torch.cuda.is_current_stream_capturing()


def _recording(**ts):
    """Whether autograd records this call; refused while a stream is captured,
    and for inputs that carry a forward-mode tangent, which the kernels would
    drop (the result would read as having a derivative of zero)."""
    for name, t in ts.items():
        if t is not None and not isinstance(t, torch.Tensor):
            raise ValueError(f"{name}: a CUDA tensor is needed")
        if t is not None and unpack_dual(t).tangent is not None:
            raise ValueError(f"{name} carries a tangent: the block operators have no forward-mode derivatives")
    if not torch.is_grad_enabled() or not any(t is not None and t.requires_grad for t in ts.values()):
        return False
    if _capturing(next(t for t in ts.values() if t is not None).device):
        raise ValueError("the differentiable block operators do not record a graph during stream capture: "
                         "capture the explicit forward and backward calls")
    return True


def _save(ctx, kept, *ts):
    """Saves tensors and activations kept as tensors or as checkpoints."""
    flat, ctx.kept = list(ts), []
    for k in kept:
        if isinstance(k, Checkpoint8):
            ctx.kept.append(k.dtype)
            flat += [k.codes, k.exps]
        else:
            ctx.kept.append(None)
            flat.append(k)
    ctx.n_plain = len(ts)
    ctx.save_for_backward(*flat)


def _saved(ctx):
    if torch.cuda.is_current_stream_capturing():
        raise RuntimeError("the differentiable block operators' backward does not run during stream capture: "
                           "capture the explicit backward calls")
    ts = list(ctx.saved_tensors)
    plain, rest, kept = ts[:ctx.n_plain], ts[ctx.n_plain:], []
    for dt in ctx.kept:
        kept.append(rest.pop(0) if dt is None else Checkpoint8(rest.pop(0), rest.pop(0), dt))
    return plain, kept


def _kept(x, checkpoint, needed):
    """A projection's input as its weight gradient needs it, or None."""
    return (checkpoint8(x) if checkpoint else x) if needed else None


class _LayerNorm(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, bias, eps, checkpoint):
        y, mean, rstd, ck = layerNormForward(x, weight, bias, eps, checkpoint)
        _save(ctx, [ck if checkpoint else x], weight, mean, rstd)
        return y

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dy):
        (weight, mean, rstd), (x,) = _saved(ctx)
        params = ctx.needs_input_grad[1] or ctx.needs_input_grad[2]
        return (*layerNormBackward(dy, x, weight, mean, rstd, params=params), None, None)


def layerNorm(x, weight, bias, eps: float = 1e-5, checkpoint: bool = False):
    """Differentiable layer norm.  With `checkpoint` its input is kept for the
    backward pass as an 8-bit checkpoint instead of in its own type."""
    if not _recording(x=x, weight=weight, bias=bias):
        return layerNormForward(x, weight, bias, eps)[0]
    return _LayerNorm.apply(x, weight, bias, eps, checkpoint)


class _Projection(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, w, bias, act, residual, checkpoint):
        keep = act != "none"
        y, z = projectionForward(x, w, bias, act, residual, checkpoint=keep and checkpoint,
                                 preactivation=keep and not checkpoint)
        kept = [_kept(x, checkpoint, ctx.needs_input_grad[1])]
        ctx.act = act
        ctx.bias_dtype = None if bias is None else bias.dtype
        _save(ctx, kept + ([z] if keep else []), w)
        return y

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dy):
        (w,), kept = _saved(ctx)
        need = ctx.needs_input_grad
        dz = activationBackward(dy, kept[1], ctx.act) if ctx.act != "none" else dy
        dx = projectionBackwardInput(dz, w) if need[0] else None
        dw = db = None
        if need[1] or need[2]:
            dw, db = projectionBackwardWeight(dz, kept[0], bias=need[2])
        if db is not None:
            db = db.to(ctx.bias_dtype)
        return dx, dw, db, None, dy if need[4] else None, None


def projection(x, w, bias=None, act: str = "none", residual=None, checkpoint: bool = False):
    """Differentiable y = act(x w^T + bias) + residual.  With `checkpoint` the
    backward pass works from 8-bit checkpoints of x and of the pre-activation."""
    if not _recording(x=x, w=w, bias=bias, residual=residual):
        return projectionForward(x, w, bias, act, residual)[0]
    return _Projection.apply(x, w, bias, act, residual, checkpoint)


class _ChannelMix(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, key, value, residual, checkpoint):
        k, z = projectionForward(x, key, act="relu2", checkpoint=checkpoint, preactivation=not checkpoint)
        y, _ = projectionForward(k, value, residual=residual)
        _save(ctx, [_kept(x, checkpoint, ctx.needs_input_grad[1]), z], key, value)
        return y

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dy):
        (key, value), (x, z) = _saved(ctx)
        need = ctx.needs_input_grad
        dv = projectionBackwardWeight(dy, z, act="relu2")[0] if need[2] else None
        dx = dk = None
        if need[0] or need[1]:
            dz = projectionBackwardInput(dy, value, pre=z, act="relu2")
            dk = projectionBackwardWeight(dz, x)[0] if need[1] else None
            dx = projectionBackwardInput(dz, key) if need[0] else None
        return dx, dk, dv, dy if need[3] else None, None


def channelMix(x, key, value, residual=None, checkpoint: bool = True):
    """The projections of cmix, differentiable: relu(x key^T)^2 value^T +
    residual (RWKVBlock.swift:299-307, after the token shift).  The squared
    ReLU ends the first product and its gradient the backward's, which reads the
    pre-activation z; with `checkpoint` z and x are kept in 8 bits (1 + 1/32
    bytes per channel) and the squared ReLU itself is not kept at all."""
    if not _recording(x=x, key=key, value=value, residual=residual):
        k, _ = projectionForward(x, key, act="relu2")
        return projectionForward(k, value, residual=residual)[0]
    return _ChannelMix.apply(x, key, value, residual, checkpoint)


class _Dropout(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, p, seed, offset):
        _save(ctx, [], *([seed] if isinstance(seed, torch.Tensor) else []))
        ctx.drawn = p, seed if isinstance(seed, int) else None, offset
        return dropoutForward(x, p, seed, offset)

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dy):
        state, _ = _saved(ctx)
        p, seed, offset = ctx.drawn
        return dropoutForward(dy, p, state[0] if state else seed, offset), None, None, None


def dropout(x, p: float, seed, offset: int = 0):
    """Differentiable dropoutForward.  A `seed` tensor keeps its values until the
    backward pass has run (autograd refuses one that was changed in place)."""
    if not _recording(x=x):
        return dropoutForward(x, p, seed, offset)
    return _Dropout.apply(x, p, seed, offset)


class _ResidualNorm(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, branch, weight, bias, eps, scale, p, seed, offset, checkpoint):
        s, y, mean, rstd, ck = residualNormForward(x, branch, weight, bias, eps, scale, p, seed, offset, checkpoint)
        ctx.set_materialize_grads(False)
        _save(ctx, [ck if checkpoint else s], weight, mean, rstd, *([seed] if isinstance(seed, torch.Tensor) else []))
        ctx.drawn = scale, p, seed if isinstance(seed, int) else None, offset
        return s, y

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, ds, dy):
        (weight, mean, rstd, *state), (s,) = _saved(ctx)
        scale, p, seed, offset = ctx.drawn
        need = ctx.needs_input_grad
        if dy is None:
            if ds is None:
                return (None,) * 10
            # ds passes as it is: zeros all round, since 0 times what a row or the weights hold may be NaN
            dy = s = torch.zeros_like(ds, memory_format=torch.contiguous_format)
            weight, mean, rstd = torch.zeros_like(weight), torch.zeros_like(mean), torch.zeros_like(rstd)
        dx, dbranch, dw, db = residualNormBackward(dy, s, weight, mean, rstd, ds, scale, p, state[0] if state else seed,
                                                   offset, params=need[2] or need[3])
        return (dx, dbranch, dw, db) + (None,) * 6


def residualNorm(x, branch, weight, bias, eps: float = 1e-5, scale: float = 1.0, p: float = 0.0, seed=0,
                 offset: int = 0, checkpoint: bool = False):
    """Differentiable (s, y) of residualNormForward.  With `checkpoint` the backward
    pass works from the 8-bit checkpoint of s."""
    if not _recording(x=x, branch=branch, weight=weight, bias=bias):
        return residualNormForward(x, branch, weight, bias, eps, scale, p, seed, offset)[:2]
    return _ResidualNorm.apply(x, branch, weight, bias, eps, scale, p, seed, offset, checkpoint)


class _TokenMix(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, mix, prev, lengths):
        x, mix, prev, lengths = _mix_args(x, mix, prev, lengths)
        ys = [torch.empty_like(x) for _ in range(mix.shape[0])]
        last = _token_mix(x, mix, prev, lengths, _addresses(ys))
        ctx.set_materialize_grads(False)
        ctx.given = prev is not None, lengths is not None
        _save(ctx, [], x, mix, *(t for t in (prev, lengths) if t is not None))
        return (*ys, last)

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, *grads):
        (x, mix, *rest), _ = _saved(ctx)
        prev = rest.pop(0) if ctx.given[0] else None
        lengths = rest.pop(0) if ctx.given[1] else None
        *dys, dlast = grads
        dx, dmix, dprev = tokenMixBackward(dys, x, mix, prev, lengths, dlast, params=ctx.needs_input_grad[1])
        return dx, dmix, dprev, None


def tokenMix(x, mix, prev=None, lengths=None):
    """Differentiable tokenMixForward: (the J tensors y_j [B, T, D], last)."""
    if not _recording(x=x, mix=mix, prev=prev):
        y, last = tokenMixForward(x, mix, prev, lengths)
        return y.unbind(0), last
    *ys, last = _TokenMix.apply(x, mix, prev, lengths)
    return tuple(ys), last


class _TmixTail(torch.autograd.Function):
    @staticmethod
    def forward(ctx, wkv, r, k, v, g, rk, weight, bias, eps):
        _save(ctx, [], wkv, r, k, v, g, rk, weight, bias)
        ctx.eps = eps
        return tmixTailForward(wkv, r, k, v, g, rk, weight, bias, eps)

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dout):
        ts, _ = _saved(ctx)
        return (*tmixTailBackward(dout, *ts, ctx.eps, params=any(ctx.needs_input_grad[5:8])), None)


def tmixTail(wkv, r, k, v, g, rk, weight, bias, eps: float = 64e-5):
    """Differentiable tmixTailForward."""
    if not _recording(wkv=wkv, r=r, k=k, v=v, g=g, rk=rk, weight=weight, bias=bias):
        return tmixTailForward(wkv, r, k, v, g, rk, weight, bias, eps)
    return _TmixTail.apply(wkv, r, k, v, g, rk, weight, bias, eps)
