"""The operators of the residual path of an mHC layer, as measured cases.

Around a sublayer F, a layer with n = 4 residual streams X (tokens x 4 x width) does

  u  = sum_i h_pre[i] X[i],   F's input = LayerNorm(u)                 stream_norm
  X' = T X + h_post (x) dropout(F(...))                                stream_mix

with T the projected residual-mixing matrices; layer_norm and dropout are the same
operators on plain rows.  Dropout's mask is a function of (seed, offset, element):
Philox4x32-10 (Salmon, Moraes, Dror, Shaw: Parallel Random Numbers: As Easy as
1, 2, 3, SC 2011) with the key seed and the counter (element / 8, offset); its 128
bits are the 16-bit draws of eight neighbouring elements, and an element is kept
when its draw is at least p * 65536 rounded to the nearest whole number, scaled by the
inverse of the share of draws that keep it.

`own` chooses between the plain forms below (elementary torch operations in 32 bits)
and the calls a user makes of the framework.
"""
import math
import os
import random
import sys

import torch

own = False

EPS = 1e-5

# name, operator, direction, tokens, width, storage type, type of the norm's weight and bias, dropout's p
_LISTED = (
    # eight sequences generating one token each: latency counts
    ("norm_tokens", "layer_norm", "forward", 8, 4096, "bfloat16", "bfloat16", 0.0),
    # training, 16 sequences of 4096 tokens, with the weight's and bias's gradients kept in 32 bits
    ("norm_training_backward", "layer_norm", "backward", 65536, 4096, "bfloat16", "float32", 0.0),
    # an odd batch of odd rows in 32 bits: the last batch of an evaluation, an experiment's width
    ("norm_odd_backward", "layer_norm", "backward", 4099, 1111, "float32", "float32", 0.0),
    # dropout on the rows of a short prompt
    ("dropout_prompt", "dropout", "forward", 16, 1024, "float16", "", 0.1),
    # dropout on a sublayer's output in training
    ("dropout_training", "dropout", "forward", 65536, 4096, "bfloat16", "", 0.1),
    # its gradient, on odd rows in 32 bits
    ("dropout_odd_backward", "dropout", "backward", 4099, 1111, "float32", "", 0.25),
    # the four streams of four generated tokens read and normalised
    ("stream_norm_tokens", "stream_norm", "forward", 4, 2048, "float16", "float16", 0.0),
    # four sequences of 4096 tokens
    ("stream_norm_training", "stream_norm", "forward", 16384, 4096, "bfloat16", "float32", 0.0),
    ("stream_norm_training_backward", "stream_norm", "backward", 65536, 2048, "bfloat16", "float32", 0.0),
    # the residual update of eight generated tokens
    ("mix_tokens", "stream_mix", "forward", 8, 4096, "bfloat16", "", 0.0),
    # training, 16 sequences of 4096 tokens
    ("mix_training_backward", "stream_mix", "backward", 65536, 2048, "bfloat16", "", 0.1),
    # odd rows and a ragged batch
    ("mix_odd", "stream_mix", "forward", 5003, 1025, "bfloat16", "", 0.1),
)
_FIELDS = ("name", "op", "direction", "tokens", "width", "dtype", "affine", "p")


def listed():
    return [dict(zip(_FIELDS, c)) for c in _LISTED]


def draw(rng):
    op = rng.choice(("layer_norm", "dropout", "stream_norm", "stream_mix"))
    most = 1 << (26 if op in ("layer_norm", "dropout") else 25)  # tokens x width
    width = int(2 ** rng.uniform(4, 14))
    if rng.random() < 0.5:
        width = max(64, width // 64 * 64)
    tokens = max(1, min(int(2 ** rng.uniform(0, 16)), most // width))
    dtype = rng.choice(("bfloat16", "bfloat16", "float16", "float32"))
    affine = rng.choice((dtype, "float32")) if op.endswith("norm") else ""
    p = rng.choice((0.05, 0.1, 0.25, 0.5)) if op == "dropout" else rng.choice((0.0, 0.1)) if op == "stream_mix" else 0.0
    return dict(zip(_FIELDS[1:], (op, rng.choice(("forward", "backward")), tokens, width, dtype, affine, p)))


def work(case):
    n, c, e = case["tokens"], case["width"], 4 if case["dtype"] == "float32" else 2
    a = 4 if case["affine"] == "float32" else 2
    back, op = case["direction"] == "backward", case["op"]
    if op == "layer_norm":  # x, w, b -> y, mean, rstd; or g, x, mean, rstd, w -> dx, dw, db
        return {"bytes": (3 if back else 2) * n * c * e + (3 if back else 2) * c * a + 8 * n, "flops": (12 if back else 7) * n * c}
    if op == "dropout":
        return {"bytes": 2 * n * c * e, "flops": n * c}
    if op == "stream_norm":  # X, h_pre, w, b -> y, mean, rstd; or g, X, h_pre, mean, rstd, w -> dX, dh, dw, db
        return {"bytes": (9 if back else 5) * n * c * e + (3 if back else 2) * c * a + (40 if back else 24) * n,
                "flops": (32 if back else 14) * n * c}
    # X, T, y, h_post -> X'; or g, X, T, y, h_post -> dX, dT, dy, dh
    return {"bytes": (14 if back else 9) * n * c * e + (160 if back else 80) * n, "flops": (82 if back else 41) * n * c}


def prepare(case, seed):
    dev = torch.device("cuda")
    g = torch.Generator(device=dev).manual_seed(seed)
    n, c, dt = case["tokens"], case["width"], getattr(torch, case["dtype"])
    op, back = case["op"], case["direction"] == "backward"

    def normal(*shape):
        return torch.randn(*shape, device=dev, generator=g, dtype=torch.float32)

    s = dict(case)
    ints = random.Random(seed)
    s["seed"], s["offset"] = ints.getrandbits(63), ints.getrandbits(40)
    if op == "layer_norm":
        # rows of their own size and centre
        x = normal(n, c).mul_(0.5 + torch.rand(n, 1, device=dev, generator=g)).add_(0.3 * normal(n, 1))
        s["x"] = x.to(dt)
    elif op == "dropout":
        s["x"] = normal(n, c).to(dt)
    else:
        # four streams that share a part, as residual streams do
        s["X"] = normal(n, 4, c).add_(normal(n, 1, c)).to(dt)
    if op == "stream_norm":
        s["h_pre"] = torch.sigmoid(normal(n, 4))
    if op == "stream_mix":
        m = torch.exp(normal(n, 4, 4) + 2 * torch.eye(4, device=dev))
        for _ in range(20):
            m = m / m.sum(2, keepdim=True)
            m = m / m.sum(1, keepdim=True)
        s["T"], s["h_post"], s["y"] = m, 2 * torch.sigmoid(normal(n, 4)), normal(n, c).to(dt)
    if op.endswith("norm"):
        at = getattr(torch, case["affine"])
        s["weight"], s["bias"] = (1 + 0.2 * normal(c)).to(at), (0.2 * normal(c)).to(at)
        if back:  # what the forward pass kept
            u = s["x"] if op == "layer_norm" else _read(s["X"], s["h_pre"])
            _, s["mean"], s["rstd"] = _norm(u, s["weight"], s["bias"])
    if back:
        s["G"] = normal(*((n, 4, c) if op == "stream_mix" else (n, c))).to(dt)
    return s


def run(s):
    return (_run_own if own else _run_plain)[s["op"], s["direction"]](s)


# ---- the framework's calls ---------------------------------------------------

def _functions():
    if "mhc_proj" not in sys.modules:
        sys.path.insert(0, os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "mhc-proj_b200"))
    import mhc_proj

    return mhc_proj.torch


_run_own = {
    ("layer_norm", "forward"): lambda s: _functions().layer_norm(s["x"], s["weight"], s["bias"], EPS),
    ("layer_norm", "backward"): lambda s: _functions().layer_norm_backward(
        s["G"], s["x"], s["mean"], s["rstd"], s["weight"], s["bias"]),
    ("dropout", "forward"): lambda s: _functions().dropout(s["x"], s["p"], s["seed"], s["offset"]),
    ("dropout", "backward"): lambda s: _functions().dropout_backward(s["G"], s["p"], s["seed"], s["offset"]),
    ("stream_norm", "forward"): lambda s: _functions().stream_norm_n4(s["X"], s["h_pre"], s["weight"], s["bias"], EPS),
    ("stream_norm", "backward"): lambda s: _functions().stream_norm_n4_backward(
        s["G"], s["X"], s["h_pre"], s["mean"], s["rstd"], s["weight"], s["bias"]),
    ("stream_mix", "forward"): lambda s: _functions().stream_mix_n4(
        s["X"], s["T"], s["y"], s["h_post"], s["p"], s["seed"], s["offset"]),
    ("stream_mix", "backward"): lambda s: _functions().stream_mix_n4_backward(
        s["G"], s["X"], s["T"], s["y"], s["h_post"], s["p"], s["seed"], s["offset"]),
}


# ---- the plain forms ---------------------------------------------------------

def _read(X, h):
    return (X.float() * h.float()[:, :, None]).sum(1)


def _norm(u, weight, bias):
    u = u.float()
    mean = u.mean(-1, keepdim=True)
    d = u - mean
    rstd = torch.rsqrt((d * d).mean(-1, keepdim=True) + EPS)
    return d * rstd * weight.float() + bias.float(), mean[:, 0], rstd[:, 0]


def _norm_back(s, u):
    """du, dweight and dbias of LayerNorm(u)"""
    g, w = s["G"].float(), s["weight"].float()
    xhat = (u - s["mean"][:, None]) * s["rstd"][:, None]
    gw = g * w
    du = s["rstd"][:, None] * (gw - gw.mean(-1, keepdim=True) - xhat * (gw * xhat).mean(-1, keepdim=True))
    at = s["weight"].dtype
    return du, (g * xhat).sum(0, dtype=torch.float64).to(at), g.sum(0, dtype=torch.float64).to(at)


def _round_hi_lo(m, b):
    """The high and low 32 bits of m * b, both below 2^32, through 16-bit halves of b."""
    low, high = m * (b & 0xFFFF), m * (b >> 16)
    high = high + (low >> 16)
    return high >> 16, ((high & 0xFFFF) << 16) | (low & 0xFFFF)


def _draws(count, seed, offset, device):
    """The 16-bit draws of elements 0 .. count - 1."""
    group = torch.arange(-(-count // 8), device=device, dtype=torch.int64)
    c0, c1 = group & 0xFFFFFFFF, group >> 32
    c2, c3 = torch.full_like(group, offset & 0xFFFFFFFF), torch.full_like(group, offset >> 32)
    k0, k1 = seed & 0xFFFFFFFF, seed >> 32
    for _ in range(10):  # the rounds of the definition
        h0, l0 = _round_hi_lo(0xD2511F53, c0)
        h1, l1 = _round_hi_lo(0xCD9E8D57, c2)
        c0, c1, c2, c3 = h1 ^ c1 ^ k0, l1, h0 ^ c3 ^ k1, l0
        k0, k1 = (k0 + 0x9E3779B9) & 0xFFFFFFFF, (k1 + 0xBB67AE85) & 0xFFFFFFFF
    words = torch.stack((c0 & 0xFFFF, c0 >> 16, c1 & 0xFFFF, c1 >> 16, c2 & 0xFFFF, c2 >> 16, c3 & 0xFFFF, c3 >> 16), 1)
    return words.reshape(-1)[:count]


def _drop(x, p, seed, offset):
    """x (in 32 bits) with its dropped elements at zero and the others scaled."""
    limit = math.floor(p * 65536 + 0.5)
    if limit == 0:
        return x.float()
    kept = _draws(x.numel(), seed, offset, x.device).reshape(x.shape) >= limit
    return torch.where(kept, x.float() * (65536 / (65536 - limit)), 0.0)


def _plain_norm(s):
    y, mean, rstd = _norm(s["x"], s["weight"], s["bias"])
    return {"y": y.to(s["x"].dtype), "mean": mean, "rstd": rstd}


def _plain_norm_back(s):
    dx, dw, db = _norm_back(s, s["x"].float())
    return {"d_x": dx.to(s["x"].dtype), "d_weight": dw, "d_bias": db}


def _plain_dropout(s):
    return {"y": _drop(s["x"], s["p"], s["seed"], s["offset"]).to(s["x"].dtype)}


def _plain_dropout_back(s):
    return {"d_x": _drop(s["G"], s["p"], s["seed"], s["offset"]).to(s["G"].dtype)}


def _plain_stream_norm(s):
    y, mean, rstd = _norm(_read(s["X"], s["h_pre"]), s["weight"], s["bias"])
    return {"y": y.to(s["X"].dtype), "mean": mean, "rstd": rstd}


def _plain_stream_norm_back(s):
    X, h = s["X"].float(), s["h_pre"].float()
    du, dw, db = _norm_back(s, _read(X, h))
    return {"d_X": (h[:, :, None] * du[:, None]).to(s["X"].dtype), "d_h_pre": (X * du[:, None]).sum(-1).to(s["h_pre"].dtype),
            "d_weight": dw, "d_bias": db}


def _plain_mix(s):
    y = _drop(s["y"], s["p"], s["seed"], s["offset"])
    return {"X": (torch.matmul(s["T"].float(), s["X"].float()) + s["h_post"].float()[:, :, None] * y[:, None]).to(s["X"].dtype)}


def _plain_mix_back(s):
    G, X, T, h = s["G"].float(), s["X"].float(), s["T"].float(), s["h_post"].float()
    y = _drop(s["y"], s["p"], s["seed"], s["offset"])
    dy = _drop(torch.matmul(h[:, None], G)[:, 0], s["p"], s["seed"], s["offset"])
    return {"d_X": torch.matmul(T.transpose(1, 2), G).to(s["X"].dtype), "d_T": torch.matmul(G, X.transpose(1, 2)).to(s["T"].dtype),
            "d_y": dy.to(s["y"].dtype), "d_h_post": (G * y[:, None]).sum(-1).to(s["h_post"].dtype)}


_run_plain = {
    ("layer_norm", "forward"): _plain_norm, ("layer_norm", "backward"): _plain_norm_back,
    ("dropout", "forward"): _plain_dropout, ("dropout", "backward"): _plain_dropout_back,
    ("stream_norm", "forward"): _plain_stream_norm, ("stream_norm", "backward"): _plain_stream_norm_back,
    ("stream_mix", "forward"): _plain_mix, ("stream_mix", "backward"): _plain_mix_back,
}


# ---- the definitions in 64 bits ----------------------------------------------

def _kept(shape, p, seed, offset, device):
    """1 / (share kept) where an element is kept, 0 where not.  A 64-bit product's
    bits are the same signed or not, so its high word is a shift away."""
    limit = int(p * 65536 + 0.5)
    count = math.prod(shape)
    at = torch.arange((count + 7) // 8, device=device)
    x = [at % 2**32, at // 2**32, torch.zeros_like(at) + offset % 2**32, torch.zeros_like(at) + offset // 2**32]
    for r in range(10):
        a, b = x[0] * 0xD2511F53, x[2] * 0xCD9E8D57
        x = [((b >> 32) % 2**32) ^ x[1] ^ ((seed + r * 0x9E3779B9) % 2**32), b % 2**32,
             ((a >> 32) % 2**32) ^ x[3] ^ (((seed >> 32) + r * 0xBB67AE85) % 2**32), a % 2**32]
    bits = torch.empty(at.numel(), 4, 2, device=device, dtype=torch.int32)
    for i in range(4):
        bits[:, i, 0], bits[:, i, 1] = x[i] % 65536, x[i] // 65536
    keep = bits.view(-1)[:count].reshape(shape) >= limit
    return keep.double() * (65536.0 / (65536 - limit) if limit < 65536 else 0.0)


def exact(case, seed):
    s = prepare(case, seed)
    op, back = s["op"], s["direction"] == "backward"
    wide = {k: v.double().requires_grad_(back and k not in ("G", "mean", "rstd")) for k, v in s.items()
            if torch.is_tensor(v) and v.is_floating_point()}
    if op == "dropout":
        x = wide["G" if back else "x"].detach()
        y = x * _kept(x.shape, s["p"], s["seed"], s["offset"], x.device)
        return {"d_x" if back else "y": y}
    if op == "stream_mix":
        y = wide["y"]
        if s["p"]:
            y = y * _kept(y.shape, s["p"], s["seed"], s["offset"], y.device)
        out = torch.einsum("tij,tjc->tic", wide["T"], wide["X"]) + torch.einsum("ti,tc->tic", wide["h_post"], y)
        of = {"X": "d_X", "T": "d_T", "y": "d_y", "h_post": "d_h_post"}
    else:
        u = wide["x"] if op == "layer_norm" else torch.einsum("ti,tic->tc", wide["h_pre"], wide["X"])
        var, mean = torch.var_mean(u, -1, correction=0)
        out = (u - mean[:, None]) / torch.sqrt(var + EPS)[:, None] * wide["weight"] + wide["bias"]
        of = {"x": "d_x", "X": "d_X", "h_pre": "d_h_pre", "weight": "d_weight", "bias": "d_bias"}
        if not back:
            return {"y": out, "mean": mean, "rstd": 1 / torch.sqrt(var + EPS)}
    if not back:
        return {"X": out}
    to = [k for k in of if k in wide]
    return dict(zip([of[k] for k in to], torch.autograd.grad(out, [wide[k] for k in to], wide["G"])))
