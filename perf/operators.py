"""Workloads of the block operators: layer norm, the projection with its epilogue, and 8-bit activation checkpoints.

An x070 block around the WKV path is made of layer norms and projections.  A
projection ends in what follows it (a bias, tanh / sigmoid / squared ReLU, the
residual), and training keeps what the backward pass reads, in the
activations' own type or as 8-bit checkpoints.  Each case below is one pass
through one of them, forward or backward, with the sizes of the x070 models
(0.1B: 768 channels; 1.5B: 2048, low rank 96, feed-forward 8192; 2.9B: 2560).

`run` computes the plain form with elementary torch operations in 32 bits, or,
with `own`, calls swiftrwkv_b200.block.  `exact` evaluates the definitions in
64 bits.

Definitions (rows n, channels i, outputs o):
  layer norm   y = (x - mean) rstd w + b, rstd = 1 / sqrt(var + eps) over the row
  its gradient dx = rstd (g - mean(g) - h mean(g h)) + dres, g = dy w, h = (x - mean) rstd;
               dw = sum_n dy h, db = sum_n dy
  projection   y = act(x W^T + bias) + residual; act: none, relu2 (max(z, 0)^2), tanh, sigmoid
  its gradient dz = (dy W) act'(z); dW = dy^T act(z), db = sum_n dy
  checkpoint   per row and group of 32 channels one power of two s = 2^E with
               max|x| / s in [64, 128) (E >= -126) and codes q = round(x / s)
               (ties to even) clipped to [-127, 127]; stands for s q
"""
import math

import torch

own = False

DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
EPS = 1e-5
GROUP = 32


# ------------------------------------------------------------------- the cases

def listed():
    return [
        # one token through one norm of the 1.5B model: the smallest call, latency only
        {"name": "norm_token", "op": "norm", "rows": 1, "dim": 2048, "dtype": "bf16", "ckpt": False},
        # a training batch of 4 x 4096 tokens of the 2.9B model, its input kept in 8 bits
        {"name": "norm_batch_ckpt", "op": "norm", "rows": 16384, "dim": 2560, "dtype": "bf16", "ckpt": True},
        # an fp32 residual stream of the 0.1B model, a ragged number of tokens
        {"name": "norm_back_f32", "op": "norm_back", "rows": 1003, "dim": 768, "dtype": "f32", "ckpt": False},
        # the batch's backward pass from the 8-bit checkpoint
        {"name": "norm_back_ckpt", "op": "norm_back", "rows": 16384, "dim": 2560, "dtype": "bf16", "ckpt": True},
        # one token through the 1.5B feed-forward key projection
        {"name": "proj_token", "op": "proj", "rows": 1, "out": 8192, "in": 2048, "dtype": "bf16", "act": "relu2",
         "bias": False, "residual": False, "ckpt": False},
        # a decode batch of 64 rows through the value projection, added to the residual stream
        {"name": "proj_decode64", "op": "proj", "rows": 64, "out": 2048, "in": 8192, "dtype": "f16", "act": "none",
         "bias": False, "residual": True, "ckpt": False},
        # the up projection of a low-rank branch on a ragged batch: short inner dimension, bias and sigmoid
        {"name": "proj_rank_up", "op": "proj", "rows": 4093, "out": 2048, "in": 96, "dtype": "bf16", "act": "sigmoid",
         "bias": True, "residual": False, "ckpt": False},
        # the key projection over a training batch, its pre-activation kept in 8 bits: the largest product
        {"name": "proj_key_ckpt", "op": "proj", "rows": 16384, "out": 8192, "in": 2048, "dtype": "bf16", "act": "relu2",
         "bias": False, "residual": False, "ckpt": True},
        # backward of a low-rank up projection behind tanh, ragged, from a checkpoint: few outputs, long sums
        {"name": "proj_back_rank", "op": "proj_back", "rows": 4093, "out": 2048, "in": 96, "dtype": "bf16",
         "act": "tanh", "ckpt": True},
        # backward of the value projection behind the squared ReLU, from the checkpoint
        {"name": "proj_back_value", "op": "proj_back", "rows": 8192, "out": 2048, "in": 8192, "dtype": "bf16",
         "act": "relu2", "ckpt": True},
        # a small fp16 branch packed, restored and differentiated
        {"name": "ckpt_rank_f16", "op": "ckpt", "rows": 257, "dim": 96, "dtype": "f16", "act": "tanh"},
        # the feed-forward activations of a training batch, packed and used again in the backward pass
        {"name": "ckpt_ffn", "op": "ckpt", "rows": 16384, "dim": 8192, "dtype": "bf16", "act": "relu2"},
    ]


def _log_uniform(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["norm", "norm_back", "proj", "proj", "proj_back", "ckpt"])
    rows = _log_uniform(rng, 1, 16384)
    if op in ("norm", "norm_back", "ckpt"):
        dim = _log_uniform(rng, 64, 10240)
        if rng.random() < 0.7:
            dim = max(64, dim // 32 * 32)
        rows = max(1, min(rows, 16384 * 8192 // dim))
        case = {"op": op, "rows": rows, "dim": dim, "dtype": rng.choice(["bf16", "f16", "f32"])}
        if op == "ckpt":
            case["act"] = rng.choice(["none", "relu2", "tanh", "sigmoid"])
        else:
            case["ckpt"] = rng.random() < 0.5
        return case
    out, inn = (max(8, _log_uniform(rng, 32, 10240) // 8 * 8) for _ in range(2))
    most = 16384 * 8192 * 2048 // (2 if op == "proj_back" else 1)
    rows = max(1, min(rows, most // (out * inn)))
    case = {"op": op, "rows": rows, "out": out, "in": inn, "dtype": rng.choice(["bf16", "bf16", "f16"]),
            "act": rng.choice(["none", "relu2", "tanh", "sigmoid"]), "ckpt": rng.random() < 0.5}
    if op == "proj":
        case["bias"] = rng.random() < 0.5
        case["residual"] = rng.random() < 0.5
    return case


# ------------------------------------------------------------------ the inputs

def _inputs(case, seed):
    """The tensors of a case, from the seed alone."""
    g = torch.Generator(device="cuda").manual_seed(seed)
    dt = DTYPES[case["dtype"]]

    def normal(*shape, scale=1.0):
        return torch.randn(shape, generator=g, device="cuda").mul_(scale)

    rows, s = case["rows"], {}
    if case["op"] in ("norm", "norm_back"):
        dim = case["dim"]
        # a residual stream: channels of different size, an offset per channel
        scale = torch.exp(normal(dim, scale=0.5))
        s["x"] = (normal(rows, dim) * scale + normal(dim, scale=0.2)).to(dt)
        s["weight"] = normal(dim, scale=0.1) + 1.0
        s["bias"] = normal(dim, scale=0.1)
        if case["op"] == "norm_back":
            s["dy"] = normal(rows, dim).to(dt)
            s["dres"] = normal(rows, dim).to(dt)
            x = s["x"].float()
            s["mean"] = x.mean(1)
            s["rstd"] = torch.rsqrt((x - s["mean"][:, None]).square().mean(1) + EPS)
    elif case["op"] == "proj":
        s["x"] = normal(rows, case["in"]).to(dt)
        s["w"] = normal(case["out"], case["in"], scale=case["in"] ** -0.5).to(dt)
        s["bias"] = normal(case["out"], scale=0.5) if case["bias"] else None
        s["residual"] = normal(rows, case["out"]).to(dt) if case["residual"] else None
    elif case["op"] == "proj_back":
        s["dy"] = normal(rows, case["out"]).to(dt)
        s["w"] = normal(case["out"], case["in"], scale=case["out"] ** -0.5).to(dt)
        s["x"] = normal(rows, case["in"]).to(dt)
    else:
        s["x"] = normal(rows, case["dim"]).to(dt)
        s["dy"] = normal(rows, case["dim"]).to(dt)
    return s


def prepare(case, seed):
    s = _inputs(case, seed)
    if case["op"] in ("norm_back", "proj_back") and case["ckpt"]:
        s["codes"], s["exps"] = _pack(s.pop("x"))  # kept by the forward pass instead of x
    s["case"] = dict(case)
    return s


# -------------------------------------------------------------- the plain form

def _pack(x):
    """Codes int8 [rows, dim] and biased exponents uint8 [rows, groups] of x."""
    rows, dim = x.shape
    pad = -dim % GROUP
    v = torch.nn.functional.pad(x.float(), (0, pad)).view(rows, -1, GROUP)
    top = v.abs().amax(2)
    e = torch.where(top > 0, torch.frexp(top).exponent - 7, -126).clamp(min=-126)
    q = torch.round(torch.ldexp(v, -e[..., None])).clamp(-127, 127).to(torch.int8)
    return q.view(rows, -1)[:, :dim].contiguous(), (e + 127).to(torch.uint8)


def _values(codes, exps):
    """What the checkpoint stands for, in 32 bits."""
    e = exps.to(torch.int32).repeat_interleave(GROUP, 1)[:, : codes.shape[1]] - 127
    return torch.ldexp(codes.float(), e)


def _act(z, act):
    if act == "relu2":
        return torch.relu(z).square()
    return torch.tanh(z) if act == "tanh" else torch.sigmoid(z) if act == "sigmoid" else z


def _act_grad(z, act):
    if act == "relu2":
        return 2 * torch.relu(z)
    if act == "tanh":
        return 1 - torch.tanh(z).square()
    if act == "sigmoid":
        t = torch.sigmoid(z)
        return t * (1 - t)
    return torch.ones_like(z)


def _plain(s):
    case = s["case"]
    dt = DTYPES[case["dtype"]]
    if case["op"] == "norm":
        x = s["x"].float()
        mean = x.mean(1)
        d = x - mean[:, None]
        rstd = torch.rsqrt(d.square().mean(1) + EPS)
        y = d * rstd[:, None] * s["weight"] + s["bias"]
        kept = [_values(*_pack(s["x"])).to(dt)] if case["ckpt"] else []
        return [y.to(dt), mean, rstd] + kept
    if case["op"] == "norm_back":
        x = _values(s["codes"], s["exps"]) if case["ckpt"] else s["x"].float()
        dy, rstd = s["dy"].float(), s["rstd"][:, None]
        h = (x - s["mean"][:, None]) * rstd
        g = dy * s["weight"]
        dx = rstd * (g - g.mean(1, keepdim=True) - h * (g * h).mean(1, keepdim=True)) + s["dres"].float()
        return [dx.to(dt), (dy * h).sum(0), dy.sum(0)]
    if case["op"] == "proj":
        z = s["x"].float() @ s["w"].float().t()
        if s["bias"] is not None:
            z = z + s["bias"]
        y = _act(z, case["act"])
        if s["residual"] is not None:
            y = y + s["residual"].float()
        kept = [_values(*_pack(z)).to(dt)] if case["ckpt"] else []
        return [y.to(dt)] + kept
    if case["op"] == "proj_back":
        dy = s["dy"].float()
        z = _values(s["codes"], s["exps"]) if case["ckpt"] else s["x"].float()
        dz = (dy @ s["w"].float()) * _act_grad(z, case["act"])
        dw = dy.t() @ _act(z, case["act"])
        return [dz.to(dt), dw.to(dt), dy.sum(0)]
    z = _values(*_pack(s["x"]))
    return [z.to(dt), _act(z, case["act"]).to(dt), (s["dy"].float() * _act_grad(z, case["act"])).to(dt)]


# ------------------------------------------------------- the framework's calls

def _own(s):
    from swiftrwkv_b200 import block as B

    case = s["case"]
    if case["op"] == "norm":
        y, mean, rstd, ck = B.layerNormForward(s["x"], s["weight"], s["bias"], EPS, checkpoint=case["ckpt"])
        return [y, mean, rstd] + ([B.checkpoint8Values(ck)] if case["ckpt"] else [])
    if case["op"] in ("norm_back", "proj_back"):
        x = B.Checkpoint8(s["codes"], s["exps"], s["dy"].dtype) if case["ckpt"] else s["x"]
        if case["op"] == "norm_back":
            return list(B.layerNormBackward(s["dy"], x, s["weight"], s["mean"], s["rstd"], dres=s["dres"]))
        dz = B.projectionBackwardInput(s["dy"], s["w"], pre=x, act=case["act"])
        dw, db = B.projectionBackwardWeight(s["dy"], x, act=case["act"], bias=True)
        return [dz, dw, db]
    if case["op"] == "proj":
        y, ck = B.projectionForward(s["x"], s["w"], bias=s["bias"], act=case["act"], residual=s["residual"],
                                    checkpoint=case["ckpt"])
        return [y] + ([B.checkpoint8Values(ck)] if case["ckpt"] else [])
    ck = B.checkpoint8(s["x"])
    return [B.checkpoint8Values(ck), B.checkpoint8Values(ck, act=case["act"]),
            B.activationBackward(s["dy"], ck, act=case["act"])]


def run(state):
    return _own(state) if own else _plain(state)


# ----------------------------------------------------------------- its measure

def work(case):
    size = 4 if case["dtype"] == "f32" else 2
    rows = case["rows"]
    if case["op"] in ("norm", "norm_back", "ckpt"):
        dim = case["dim"]
        n, kept = rows * dim, rows * (dim + -(-dim // GROUP))
        if case["op"] == "norm":
            # x, y, the row statistics, weight and bias; the checkpoint written, read, and its values
            moved = 2 * n * size + 8 * rows + 8 * dim + ((2 * kept + n * size) if case["ckpt"] else 0)
            return {"bytes": moved, "flops": 8 * n}
        if case["op"] == "norm_back":
            moved = (3 * n * size) + (kept if case["ckpt"] else n * size) + 8 * rows + 12 * dim
            return {"bytes": moved, "flops": 14 * n}
        # x and dy in; the checkpoint written and read; values, act and gradient out
        return {"bytes": 5 * n * size + 2 * kept, "flops": 12 * n}
    out, inn = case["out"], case["in"]
    if case["op"] == "proj":
        n = rows * out
        kept = rows * (out + -(-out // GROUP))
        moved = (rows * inn + out * inn + n) * size + (4 * out if case["bias"] else 0)
        moved += n * size if case["residual"] else 0
        moved += 2 * kept + n * size if case["ckpt"] else 0
        return {"bytes": moved, "flops": 2 * n * inn}
    kept = rows * (inn + -(-inn // GROUP)) if case["ckpt"] else rows * inn * size
    moved = (rows * out + out * inn + rows * inn + out * inn) * size + kept + 4 * out
    return {"bytes": moved, "flops": 4 * rows * out * inn}


# ------------------------------------------------------- the definition, exact

def _exact_checkpoint(v):
    """What the checkpoint of v (64 bits) stands for, from its definition."""
    rows, dim = v.shape
    full = dim - dim % GROUP
    parts = [_exact_checkpoint_groups(v[:, :full].reshape(rows, -1, GROUP)).reshape(rows, full)] if full else []
    if full < dim:
        parts.append(_exact_checkpoint_groups(v[:, None, full:])[:, 0])
    return torch.cat(parts, 1)


def _exact_checkpoint_groups(v):
    top = v.abs().max(dim=2, keepdim=True).values
    e = torch.floor(torch.log2(torch.where(top > 0, top, torch.ones_like(top)))) - 6
    e = torch.where(top / torch.exp2(e) >= 128, e + 1, e)  # log2 rounded down past a power of two
    e = torch.where(top / torch.exp2(e) < 64, e - 1, e)
    e = torch.where(top > 0, e, torch.full_like(e, -126)).clamp(min=-126)
    s = torch.exp2(e)
    return torch.minimum(torch.maximum(torch.round(v / s), torch.full_like(v, -127)), torch.full_like(v, 127)) * s


def exact(case, seed):
    s = _inputs(case, seed)
    d = {k: (v.double() if v is not None else None) for k, v in s.items()}
    act = {"none": (lambda z: z, lambda z: torch.ones_like(z)),
           "relu2": (lambda z: z.clamp(min=0) ** 2, lambda z: 2 * z.clamp(min=0)),
           "tanh": (torch.tanh, lambda z: 1 / torch.cosh(z) ** 2),
           "sigmoid": (lambda z: 1 / (1 + torch.exp(-z)), lambda z: 1 / (2 + torch.exp(z) + torch.exp(-z)))}
    if case["op"] == "norm":
        x = d["x"]
        var, mean = torch.var_mean(x, 1, correction=0)
        rstd = 1 / torch.sqrt(var + EPS)
        y = torch.addcmul(d["bias"], (x - mean[:, None]) * rstd[:, None], d["weight"])
        return [y, mean, rstd] + ([_exact_checkpoint(x)] if case["ckpt"] else [])
    if case["op"] == "norm_back":
        x = _exact_checkpoint(d["x"]) if case["ckpt"] else d["x"]
        h = (x - d["mean"][:, None]) * d["rstd"][:, None]
        g = d["dy"] * d["weight"]
        dim = x.shape[1]
        along = torch.einsum("nd,nd->n", g, h) / dim
        dx = d["rstd"][:, None] * (g - (g.sum(1) / dim)[:, None] - h * along[:, None]) + d["dres"]
        return [dx, torch.einsum("nd,nd->d", d["dy"], h), torch.einsum("nd->d", d["dy"])]
    f, df = act[case.get("act", "none")]
    if case["op"] == "proj":
        z = torch.einsum("ni,oi->no", d["x"], d["w"])
        if d["bias"] is not None:
            z = z + d["bias"]
        y = f(z) if d["residual"] is None else f(z) + d["residual"]
        return [y] + ([_exact_checkpoint(z)] if case["ckpt"] else [])
    if case["op"] == "proj_back":
        z = _exact_checkpoint(d["x"]) if case["ckpt"] else d["x"]
        dz = torch.einsum("no,oi->ni", d["dy"], d["w"]) * df(z)
        return [dz, torch.einsum("no,ni->oi", d["dy"], f(z)), torch.einsum("no->o", d["dy"])]
    z = _exact_checkpoint(d["x"])
    return [z, f(z), d["dy"] * df(z)]
