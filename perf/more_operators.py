"""Workloads of the operators between a block's projections and its WKV path, in training and for single tokens.

An x070 block adds each branch to the residual stream and normalises the sum for
the next branch (with dropout on the branch, in training); the norm's result is
interpolated with the token before it, six ways for the time mix and one way for
the channel mix; and the time mix ends in a norm by head, a bonus and a gate.
Each case below is one pass through one of these, forward or backward, with the
sizes of the x070 models (0.1B: 768 channels; 1.5B: 2048; 2.9B: 2560; heads of 64).

`run` computes the plain form with elementary torch operations in 32 bits, or,
with `own`, calls swiftrwkv_b200.block.  `exact` evaluates the definitions in
64 bits.

Definitions (rows n, channels i):
  dropout       y = x / (1 - q) where kept, 0 where dropped; q = t / 65536, t = round(65536 p).
                Element i of the tensor is dropped where its 16 bits are below t: half i % 2
                (low half first) of word (i % 8) // 2 of the block of four 32-bit words that
                Philox4x32-10 (Salmon, Moraes, Dror and Shaw, "Parallel random numbers: as easy
                as 1, 2, 3", 2011) gives for the counter i // 8 (64 bits), offset (64 bits) and
                the key seed (64 bits)
  residual norm s = x + scale dropout(branch), y = (s - mean) rstd w + b over each row of s
  its gradient  ds = rstd (g - mean(g) - h mean(g h)) + dres, g = dy w, h = (s - mean) rstd;
                dx = ds, dbranch = scale dropout(ds), dw = sum_n dy h, db = sum_n dy
  token mix     y_j[t] = x[t] + (x[t-1] - x[t]) m_j, x[-1] = prev; 0 from a sequence's length on;
                last = x[length - 1] (prev for an empty sequence)
  its gradient  dx[t] = sum_j (1 - m_j) dy_j[t] + m_j dy_j[t+1], and dlast at the last token;
                dm_j = sum over tokens of dy_j[t] (x[t-1] - x[t]), dprev = sum_j m_j dy_j[0]
  tail          per row and head: n = (a - mean) rstd of the WKV output a, c = sum r k rk,
                out = (n w + b + c v) g
  its gradient  by the chain rule, to a, r, k, v, g, rk, w and b
"""
import math

import numpy as np
import torch

own = False

DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
EPS = 1e-5
EPS_HEAD = 64e-5
GROUP = 32  # channels per scale of an 8-bit checkpoint


# ------------------------------------------------------------------- the cases

def listed():
    return [
        # a low-rank branch of a short fine-tuning batch, odd number of rows: latency only
        {"name": "drop_rank_f16", "op": "drop", "rows": 257, "dim": 96, "dtype": "f16", "p": 0.1},
        # the feed-forward activations of a training batch of 4 x 4096 tokens
        {"name": "drop_ffn", "op": "drop", "rows": 16384, "dim": 8192, "dtype": "bf16", "p": 0.1},
        # one decoded token of the 1.5B model: branch added and normed
        {"name": "rnorm_token", "op": "rnorm", "rows": 1, "dim": 2048, "dtype": "bf16", "p": 0.0, "scale": 1.0,
         "ckpt": False},
        # a training batch of the 2.9B model, the sum kept in 8 bits
        {"name": "rnorm_batch_ckpt", "op": "rnorm", "rows": 16384, "dim": 2560, "dtype": "bf16", "p": 0.1, "scale": 1.0,
         "ckpt": True},
        # an fp32 residual stream of the 0.1B model, a ragged number of tokens, a scaled branch
        {"name": "rnorm_back_f32", "op": "rnorm_back", "rows": 1003, "dim": 768, "dtype": "f32", "p": 0.1, "scale": 0.5,
         "ckpt": False},
        # the batch's backward pass from the 8-bit checkpoint
        {"name": "rnorm_back_ckpt", "op": "rnorm_back", "rows": 16384, "dim": 2560, "dtype": "bf16", "p": 0.1,
         "scale": 1.0, "ckpt": True},
        # a decode batch of 64 sequences, one token each after its state: the time mix's six interpolations
        {"name": "mix_decode64", "op": "mix", "batch": 64, "len": 1, "dim": 2048, "ways": 6, "dtype": "f16",
         "prev": True, "ragged": False},
        # the time mix's interpolations of a right-padded training batch of the 2.9B model
        {"name": "mix_batch", "op": "mix", "batch": 4, "len": 4096, "dim": 2560, "ways": 6, "dtype": "bf16",
         "prev": False, "ragged": True},
        # its backward pass over whole sequences that continue from a state
        {"name": "mix_back_batch", "op": "mix_back", "batch": 4, "len": 4096, "dim": 2560, "ways": 6, "dtype": "bf16",
         "prev": True, "ragged": False},
        # one decoded token through the end of the 1.5B model's time mix
        {"name": "tail_token", "op": "tail", "rows": 1, "heads": 32, "size": 64, "dtype": "bf16"},
        # a ragged batch of the 1.5B model
        {"name": "tail_batch", "op": "tail", "rows": 16381, "heads": 32, "size": 64, "dtype": "bf16"},
        # the backward pass of the 2.9B model's training batch
        {"name": "tail_back_batch", "op": "tail_back", "rows": 16384, "heads": 40, "size": 64, "dtype": "bf16"},
    ]


def _log_uniform(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["drop", "rnorm", "rnorm_back", "mix", "mix_back", "tail", "tail_back"])
    case = {"op": op, "dtype": rng.choice(["bf16", "bf16", "f16", "f32"])}
    rows = _log_uniform(rng, 1, 16384)
    if op == "drop":
        dim = _log_uniform(rng, 16, 8192)
        if rng.random() < 0.5:
            dim = max(16, dim // 16 * 16)
        case |= {"rows": rows, "dim": dim, "p": round(rng.uniform(0.0, 0.6), 3)}
    elif op in ("rnorm", "rnorm_back"):
        dim = max(64, _log_uniform(rng, 64, 6144) // 8 * 8)
        if rng.random() < 0.6:
            dim = max(64, dim // 64 * 64)
        case |= {"rows": max(1, min(rows, 16384 * 2560 // dim)), "dim": dim,
                 "p": round(rng.uniform(0.02, 0.5), 3) if rng.random() < 0.6 else 0.0,
                 "scale": rng.choice([1.0, 1.0, 0.5, 0.125]), "ckpt": rng.random() < 0.5}
        if op == "rnorm" and case["dtype"] == "f32":
            case["ckpt"] = False  # restored in 32 bits, a sum next to a border is a whole step from its neighbour's code
    elif op in ("mix", "mix_back"):
        dim = max(64, _log_uniform(rng, 64, 8192) // 8 * 8)
        ways = rng.choice([6, 6, 1, 4])
        batch = _log_uniform(rng, 1, 64)
        most = 16384 * 2560 * 6 // (dim * ways * batch)
        length = max(1, min(_log_uniform(rng, 1, 16384), most))
        case |= {"batch": batch, "len": length, "dim": dim, "ways": ways, "prev": rng.random() < 0.5,
                 "ragged": rng.random() < 0.5}
    else:
        size = rng.choice([64, 64, 64, 32, 128])
        heads = _log_uniform(rng, 1, 64)
        case |= {"rows": max(1, min(rows, 16384 * 2560 // (heads * size))), "heads": heads, "size": size}
    return case


# ------------------------------------------------------------------ the inputs

def _inputs(case, seed):
    """The tensors of a case, from the seed alone."""
    g = torch.Generator(device="cuda").manual_seed(seed)
    dt, op = DTYPES[case["dtype"]], case["op"]

    def normal(*shape, scale=1.0):
        return torch.randn(shape, generator=g, device="cuda").mul_(scale)

    s = {}
    if op == "drop":
        s["x"] = normal(case["rows"], case["dim"]).to(dt)
    elif op in ("rnorm", "rnorm_back"):
        rows, dim = case["rows"], case["dim"]
        # a residual stream: channels of different size, an offset per channel
        x = normal(rows, dim) * torch.exp(normal(dim, scale=0.5)) + normal(dim, scale=0.2)
        s["weight"] = normal(dim, scale=0.1) + 1.0
        s["bias"] = normal(dim, scale=0.1)
        if op == "rnorm":
            s["x"] = x.to(dt)
            s["branch"] = normal(rows, dim).to(dt)
        else:
            s["s"] = x.to(dt)
            s["dy"] = normal(rows, dim).to(dt)
            s["dres"] = normal(rows, dim).to(dt)
            x = s["s"].float()
            s["mean"] = x.mean(1)
            s["rstd"] = torch.rsqrt((x - s["mean"][:, None]).square().mean(1) + EPS)
    elif op in ("mix", "mix_back"):
        B, T, D, J = case["batch"], case["len"], case["dim"], case["ways"]
        s["x"] = normal(B, T, D).to(dt)
        s["mix"] = torch.rand(J, D, generator=g, device="cuda")
        s["prev"] = normal(B, D).to(dt) if case["prev"] else None
        s["lengths"] = None
        if case["ragged"]:
            # right-padded: the longest fills its row; of several, one is empty
            lengths = torch.randint(0, T + 1, (B,), generator=g, device="cuda", dtype=torch.int32)
            lengths[0] = T
            if B > 1:
                lengths[1] = 0
            s["lengths"] = lengths
        if op == "mix_back":
            for j in range(J):
                s["dy%d" % j] = normal(B, T, D).to(dt)
            s["dlast"] = normal(B, D).to(dt) if case["prev"] else None
    else:
        rows, H, S = case["rows"], case["heads"], case["size"]
        # the WKV output grows along a sequence and differs by head
        size = torch.exp(normal(1, H, 1, scale=0.7))
        s["wkv"] = (normal(rows, H, S) * size).view(rows, H * S).to(dt)
        for name in ("r", "k", "v", "g"):
            s[name] = normal(rows, H * S).to(dt)
        s["rk"] = normal(H, S, scale=0.1)
        s["weight"] = normal(H * S, scale=0.1) + 0.7
        s["bias"] = normal(H * S, scale=0.1)
        if op == "tail_back":
            s["dout"] = normal(rows, H * S).to(dt)
    return s


def prepare(case, seed):
    s = _inputs(case, seed)
    if case["op"] == "rnorm_back" and case["ckpt"]:
        s["codes"], s["exps"] = _pack(s.pop("s").float())  # kept by the forward pass instead of the sum
    if case["op"] == "mix_back":
        s["dys"] = [s.pop("dy%d" % j) for j in range(case["ways"])]
    s["case"] = dict(case)
    s["seed"] = seed
    return s


# -------------------------------------------------------------- the plain form

def _mul(m, c):
    """(high, low) 32 bits of m * c, both below 2^32, in 64-bit integers that hold no such product."""
    low = m * (c & 0xFFFF)
    high = m * (c >> 16) + (low >> 16)
    return high >> 16, (high & 0xFFFF) << 16 | low & 0xFFFF


def _kept(n, threshold, seed, offset, device):
    """Which of n elements are kept."""
    block = torch.arange(-(-n // 8), device=device)
    c = [block & 0xFFFFFFFF, block >> 32] + [torch.full_like(block, w) for w in (offset & 0xFFFFFFFF, offset >> 32)]
    k0, k1 = seed & 0xFFFFFFFF, seed >> 32
    for _ in range(10):
        h0, l0 = _mul(0xD2511F53, c[0])
        h1, l1 = _mul(0xCD9E8D57, c[2])
        c = [h1 ^ c[1] ^ k0, l1, h0 ^ c[3] ^ k1, l0]
        k0, k1 = (k0 + 0x9E3779B9) & 0xFFFFFFFF, (k1 + 0xBB67AE85) & 0xFFFFFFFF
    words = torch.stack(c, 1)
    halves = torch.stack((words & 0xFFFF, words >> 16), 2).flatten()
    return halves[:n] >= threshold


def _dropped(x, p, seed, offset=0):
    """Dropout of x in 32 bits."""
    t = round(65536 * p)
    if t == 0:
        return x
    keep = _kept(x.numel(), t, seed, offset, x.device).view(x.shape)
    return torch.where(keep, x * (65536 / (65536 - t) if t < 65536 else 0.0), 0.0)


def _pack(x):
    """Codes int8 [rows, dim] and biased exponents uint8 [rows, groups] of x, fp32."""
    rows, dim = x.shape
    v = torch.nn.functional.pad(x, (0, -dim % GROUP)).view(rows, -1, GROUP)
    top = v.abs().amax(2)
    e = torch.where(top > 0, torch.frexp(top).exponent - 7, -126).clamp(min=-126)
    q = torch.round(torch.ldexp(v, -e[..., None])).clamp(-127, 127).to(torch.int8)
    return q.view(rows, -1)[:, :dim].contiguous(), (e + 127).to(torch.uint8)


def _values(codes, exps):
    """What the checkpoint stands for, in 32 bits."""
    e = exps.to(torch.int32).repeat_interleave(GROUP, 1)[:, : codes.shape[1]] - 127
    return torch.ldexp(codes.float(), e)


def _lengths(s):
    """(lengths [B], which tokens are real [B, T, 1])."""
    B, T, _ = s["x"].shape
    lengths = s["lengths"]
    if lengths is None:
        lengths = torch.full((B,), T, device=s["x"].device)
    real = torch.arange(T, device=lengths.device)[None] < lengths[:, None]
    return lengths.long(), real[..., None]


def _before(s):
    """(x, the token before each, the token before the first), in 32 bits."""
    x = s["x"].float()
    first = torch.zeros_like(x[:, 0]) if s["prev"] is None else s["prev"].float()
    return x, torch.cat((first[:, None], x[:, :-1]), 1), first


def _plain(s):
    case = s["case"]
    dt, op = DTYPES[case["dtype"]], case["op"]
    if op == "drop":
        return [_dropped(s["x"].float(), case["p"], s["seed"]).to(dt)]
    if op == "rnorm":
        v = s["x"].float() + case["scale"] * _dropped(s["branch"].float(), case["p"], s["seed"])
        mean = v.mean(1)
        d = v - mean[:, None]
        rstd = torch.rsqrt(d.square().mean(1) + EPS)
        y = d * rstd[:, None] * s["weight"] + s["bias"]
        kept = [_values(*_pack(v)).to(dt)] if case["ckpt"] else []
        return [v.to(dt), y.to(dt), mean, rstd] + kept
    if op == "rnorm_back":
        v = _values(s["codes"], s["exps"]) if case["ckpt"] else s["s"].float()
        dy, rstd = s["dy"].float(), s["rstd"][:, None]
        h = (v - s["mean"][:, None]) * rstd
        g = dy * s["weight"]
        ds = rstd * (g - g.mean(1, keepdim=True) - h * (g * h).mean(1, keepdim=True)) + s["dres"].float()
        branch = case["scale"] * _dropped(ds, case["p"], s["seed"])
        return [ds.to(dt), branch.to(dt), (dy * h).sum(0), dy.sum(0)]
    if op == "mix":
        lengths, real = _lengths(s)
        x, before, first = _before(s)
        y = torch.where(real, x + (before - x) * s["mix"][:, None, None], 0.0)
        at = (lengths - 1).clamp(min=0)[:, None, None].expand(-1, 1, x.shape[2])
        last = torch.where(lengths[:, None] > 0, x.gather(1, at)[:, 0], first)
        return [y.to(dt), last.to(dt)]
    if op == "mix_back":
        lengths, real = _lengths(s)
        x, before, _ = _before(s)
        m = s["mix"][:, None, None]
        dy = torch.where(real, torch.stack(s["dys"]).float(), 0.0)
        back = (dy * m).sum(0)
        dx = (dy * (1 - m)).sum(0)
        dx[:, :-1] += back[:, 1:]
        dprev = back[:, 0]
        if s["dlast"] is not None:
            dlast = s["dlast"].float()
            at = torch.arange(x.shape[1], device=x.device)[None] == lengths[:, None] - 1
            dx = dx + at[..., None] * dlast[:, None]
            dprev = dprev + torch.where(lengths[:, None] == 0, dlast, 0.0)
        dmix = (dy * (before - x)).sum((1, 2))
        return [dx.to(dt), dmix] + ([dprev.to(dt)] if s["prev"] is not None else [])
    rows, H, S = case["rows"], case["heads"], case["size"]
    a, r, k, v, g = (s[name].float().view(rows, H, S) for name in ("wkv", "r", "k", "v", "g"))
    rk, w, b = (s[name].view(H, S) for name in ("rk", "weight", "bias"))
    d = a - a.mean(2, keepdim=True)
    rstd = torch.rsqrt(d.square().mean(2, keepdim=True) + EPS_HEAD)
    n = d * rstd
    c = (r * k * rk).sum(2, keepdim=True)
    z = n * w + b + c * v
    if op == "tail":
        return [(z * g).view(rows, H * S).to(dt)]
    dout = s["dout"].float().view(rows, H, S)
    dz = dout * g
    dc = (dz * v).sum(2, keepdim=True)
    dn = dz * w
    da = rstd * (dn - dn.mean(2, keepdim=True) - n * (dn * n).mean(2, keepdim=True))
    out = [t.reshape(rows, H * S).to(dt) for t in (da, dc * k * rk, dc * r * rk, dz * c, dout * z)]
    return out + [(dc * r * k).sum(0), (dz * n).sum(0).flatten(), dz.sum(0).flatten()]


# ------------------------------------------------------- the framework's calls

def _own(s):
    from swiftrwkv_b200 import block as B

    case = s["case"]
    op = case["op"]
    if op == "drop":
        return [B.dropoutForward(s["x"], case["p"], s["seed"])]
    if op == "rnorm":
        v, y, mean, rstd, ck = B.residualNormForward(s["x"], s["branch"], s["weight"], s["bias"], EPS,
                                                     scale=case["scale"], p=case["p"], seed=s["seed"],
                                                     checkpoint=case["ckpt"])
        return [v, y, mean, rstd] + ([B.checkpoint8Values(ck)] if case["ckpt"] else [])
    if op == "rnorm_back":
        v = B.Checkpoint8(s["codes"], s["exps"], s["dy"].dtype) if case["ckpt"] else s["s"]
        return list(B.residualNormBackward(s["dy"], v, s["weight"], s["mean"], s["rstd"], dres=s["dres"],
                                           scale=case["scale"], p=case["p"], seed=s["seed"]))
    if op == "mix":
        return list(B.tokenMixForward(s["x"], s["mix"], prev=s["prev"], lengths=s["lengths"]))
    if op == "mix_back":
        dx, dmix, dprev = B.tokenMixBackward(s["dys"], s["x"], s["mix"], prev=s["prev"], lengths=s["lengths"],
                                             dlast=s["dlast"])
        return [dx, dmix] + ([dprev] if s["prev"] is not None else [])
    if op == "tail":
        return [B.tmixTailForward(s["wkv"], s["r"], s["k"], s["v"], s["g"], s["rk"], s["weight"], s["bias"], EPS_HEAD)]
    return list(B.tmixTailBackward(s["dout"], s["wkv"], s["r"], s["k"], s["v"], s["g"], s["rk"], s["weight"], s["bias"],
                                   EPS_HEAD))


def run(state):
    return _own(state) if own else _plain(state)


# ----------------------------------------------------------------- its measure

def work(case):
    size, op = 4 if case["dtype"] == "f32" else 2, case["op"]
    if op == "drop":
        n = case["rows"] * case["dim"]
        return {"bytes": 2 * n * size, "flops": n}
    if op in ("rnorm", "rnorm_back"):
        rows, dim = case["rows"], case["dim"]
        n, kept = rows * dim, rows * (dim + -(-dim // GROUP))
        if op == "rnorm":
            # x and branch in, sum and norm out, statistics, weight and bias; the checkpoint written, read, and its values
            moved = 4 * n * size + 8 * rows + 8 * dim + ((2 * kept + n * size) if case["ckpt"] else 0)
            return {"bytes": moved, "flops": 10 * n}
        # dy, dres and the sum in, dx out, and dbranch where it differs from it; statistics, weight and its gradients
        outs = 2 if case["p"] or case["scale"] != 1.0 else 1
        moved = (2 + outs) * n * size + (kept if case["ckpt"] else n * size) + 8 * rows + 12 * dim
        return {"bytes": moved, "flops": 16 * n}
    if op in ("mix", "mix_back"):
        B, T, D, J = case["batch"], case["len"], case["dim"], case["ways"]
        n, edge = B * T * D, B * D * size * (1 + case["prev"])
        if op == "mix":
            return {"bytes": (1 + J) * n * size + edge + 4 * J * D, "flops": 3 * J * n}
        return {"bytes": (2 + J) * n * size + 3 * B * D * size * case["prev"] + 8 * J * D, "flops": 7 * J * n}
    n, D = case["rows"] * case["heads"] * case["size"], case["heads"] * case["size"]
    if op == "tail":
        return {"bytes": 6 * n * size + 12 * D, "flops": 16 * n}
    return {"bytes": 11 * n * size + 24 * D, "flops": 44 * n}


# ------------------------------------------------------- the definition, exact

def _exact_keep(n, threshold, seed):
    """Which of n elements are kept, from the generator's definition in unsigned 64-bit integers."""
    w32 = np.uint64(0xFFFFFFFF)
    i = np.arange((n + 7) // 8, dtype=np.uint64)
    x0, x1, x2, x3 = i & w32, i >> np.uint64(32), np.zeros_like(i), np.zeros_like(i)
    for rnd in range(10):
        key = [np.uint64(((seed >> 32 * h) + rnd * step) % 2**32) for h, step in enumerate((0x9E3779B9, 0xBB67AE85))]
        a, b = x0 * np.uint64(0xD2511F53), x2 * np.uint64(0xCD9E8D57)
        x0, x1, x2, x3 = (b >> np.uint64(32)) ^ x1 ^ key[0], b & w32, (a >> np.uint64(32)) ^ x3 ^ key[1], a & w32
    bits = np.stack([x0, x1, x2, x3], axis=1).astype("<u4").reshape(-1).view("<u2")
    return torch.from_numpy(bits[:n].astype(np.int32) >= threshold)


def _exact_drop(x, p, seed):
    t = int(np.rint(p * 65536))
    if t >= 65536:
        return torch.zeros_like(x)
    mask = _exact_keep(x.numel(), t, seed).to(x.device).view_as(x)
    return torch.where(mask, x / (1.0 - t / 65536.0), torch.zeros_like(x))


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


def _exact_mix(case, d):
    """Token by token over the real tokens, gathered."""
    B, T, D = d["x"].shape
    device = d["x"].device
    lengths = d["lengths"].long().tolist() if d["lengths"] is not None else [T] * B
    before = torch.zeros_like(d["x"])
    before[:, 1:] = d["x"][:, :-1]
    if d["prev"] is not None:
        before[:, 0] = d["prev"]
    pad = torch.ones(B, T, 1, dtype=torch.bool, device=device)
    for b, n in enumerate(lengths):
        pad[b, :n] = False
    if case["op"] == "mix":
        y = torch.stack([torch.lerp(d["x"], before, m.expand(B, T, D)).masked_fill(pad, 0) for m in d["mix"]])
        last = [d["x"][b, n - 1] if n else before[b, 0] if d["prev"] is not None else torch.zeros_like(before[b, 0])
                for b, n in enumerate(lengths)]
        return [y, torch.stack(last)]
    grid = torch.zeros(B, T + 1, D, dtype=torch.float64, device=device)  # gradient of [prev, x]
    dmix = []
    for j, m in enumerate(d["mix"]):
        dy = d["dy%d" % j].masked_fill(pad, 0)
        grid[:, 1:] += dy * (1 - m)
        grid[:, :-1] += dy * m
        dmix.append(torch.einsum("btd,btd->d", dy, before - d["x"]))
    if d["dlast"] is not None:
        for b, n in enumerate(lengths):
            grid[b, n] += d["dlast"][b]
    return [grid[:, 1:], torch.stack(dmix)] + ([grid[:, 0]] if d["prev"] is not None else [])


def exact(case, seed):
    s = _inputs(case, seed)
    d = {k: (v.double() if v is not None else None) for k, v in s.items()}
    op = case["op"]
    if op == "drop":
        return [_exact_drop(d["x"], case["p"], seed)]
    if op == "rnorm":
        v = torch.add(d["x"], _exact_drop(d["branch"], case["p"], seed), alpha=case["scale"])
        var, mean = torch.var_mean(v, 1, correction=0)
        rstd = 1 / torch.sqrt(var + EPS)
        y = torch.addcmul(d["bias"], (v - mean[:, None]) * rstd[:, None], d["weight"])
        return [v, y, mean, rstd] + ([_exact_checkpoint(v)] if case["ckpt"] else [])
    if op == "rnorm_back":
        v = _exact_checkpoint(d["s"]) if case["ckpt"] else d["s"]
        h = (v - d["mean"][:, None]) * d["rstd"][:, None]
        g = d["dy"] * d["weight"]
        dim = v.shape[1]
        along = torch.einsum("nd,nd->n", g, h) / dim
        ds = d["rstd"][:, None] * (g - (g.sum(1) / dim)[:, None] - h * along[:, None]) + d["dres"]
        return [ds, case["scale"] * _exact_drop(ds, case["p"], seed), torch.einsum("nd,nd->d", d["dy"], h),
                torch.einsum("nd->d", d["dy"])]
    if op in ("mix", "mix_back"):
        return _exact_mix(case, d)
    rows, H, S = case["rows"], case["heads"], case["size"]
    head = {k: v.view(-1, H, S) for k, v in d.items()}
    var, mean = torch.var_mean(head["wkv"], 2, correction=0, keepdim=True)
    sd = torch.sqrt(var + EPS_HEAD)
    n = (head["wkv"] - mean) / sd
    c = torch.einsum("nhs,nhs,hs->nh", head["r"], head["k"], head["rk"][0])[..., None]
    z = torch.addcmul(head["bias"], n, head["weight"]) + c * head["v"]
    if op == "tail":
        return [(head["g"] * z).view(rows, -1)]
    dz = head["g"] * head["dout"]
    dc = torch.einsum("nhs,nhs->nh", dz, head["v"])[..., None]
    dn = dz * head["weight"]
    along = torch.einsum("nhs,nhs->nh", dn, n)[..., None] / S
    da = (dn - dn.sum(2, keepdim=True) / S - along * n) / sd
    outs = (da, dc * head["k"] * head["rk"], dc * head["r"] * head["rk"], c * dz, z * head["dout"])
    return [t.reshape(rows, -1) for t in outs] + [torch.einsum("nhs,nhs->hs", dc * head["r"], head["k"]),
                                                  torch.einsum("nhs,nhs->hs", dz, n).flatten(),
                                                  torch.einsum("nhs->hs", dz).flatten()]
