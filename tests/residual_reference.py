"""The residual path's operators in 64 bits, with the bounds their outputs are
held to (not collected: imported by test_residual_cpu.py and
test_residual_gpu.py).

Each function returns {output: (value, magnitude, depth)}: `magnitude` is the
sum of the absolute values of the terms that the output is added up from, and
`depth` the longest chain of fp32 operations from an input to it.  An fp32
evaluation is then off by at most depth * 2^-24 * magnitude (to first order),
and the one rounding to the storage type by half a step of the value:

  |got - value| <= eps_t / 2 * |value| + (1 + eps_t) * depth * 2^-24 * magnitude

plus half the type's smallest subnormal; a value whose nearest one of the type
is infinite (over 65520 in fp16: a kept element under the scale 65536 of p =
0.99999) has to be that infinity.  The depths assume sums split over at
least 32 lanes and folded in trees: C / 32 + 32 for a sum over a row.  Sums over
the batch (a weight's gradient) are split over at least 8 lines of at most N / 8
rows, folded over at most 2048 partial sums: N / 8 + 2048 would be the depth of
one chain, but the partial sums of many rows are the long chains of few, so
N / 8 + 128.
"""
import torch

UNIT = 2.0 ** -24


def row_depth(C):
    return C / 32 + 32


def rows_depth(N):
    return N / 8 + 128


# ---- Philox4x32-10 ------------------------------------------------------------

def philox(counter, key):
    """Ten rounds on Python integers: counter (4 words), key (2 words)."""
    c, k = list(counter), list(key)
    for _ in range(10):
        p0, p1 = 0xD2511F53 * c[0], 0xCD9E8D57 * c[2]
        c = [(p1 >> 32) ^ c[1] ^ k[0], p1 & 0xFFFFFFFF, (p0 >> 32) ^ c[3] ^ k[1], p0 & 0xFFFFFFFF]
        k = [(k[0] + 0x9E3779B9) & 0xFFFFFFFF, (k[1] + 0xBB67AE85) & 0xFFFFFFFF]
    return c


def draw(e, seed, offset):
    """The 16-bit draw of element e."""
    q = e // 8
    w = philox((q & 0xFFFFFFFF, q >> 32, offset & 0xFFFFFFFF, (offset >> 32) & 0xFFFFFFFF),
               (seed & 0xFFFFFFFF, (seed >> 32) & 0xFFFFFFFF))
    return (w[e % 8 // 2] >> (16 * (e % 2))) & 0xFFFF


def limit_of(p):
    return int(p * 65536 + 0.5)


def drop_scale(p):
    limit = limit_of(p)
    return 65536.0 / (65536 - limit) if limit < 65536 else 0.0


def keep_mask(count, p, seed, offset, first=0):
    return torch.tensor([draw(e, seed, offset) >= limit_of(p) for e in range(first, first + count)], dtype=torch.bool)


def keep_mask_fast(count, p, seed, offset, device, first=0):
    """keep_mask on int64 tensors (a 64-bit product's bits are the same signed)."""
    q0, q1 = first // 8, (first + count + 7) // 8
    at = torch.arange(q0, q1, device=device, dtype=torch.int64)
    M = 0xFFFFFFFF
    c = [at & M, at >> 32, torch.full_like(at, offset & M), torch.full_like(at, (offset >> 32) & M)]
    k0, k1 = seed & M, (seed >> 32) & M
    for _ in range(10):
        p0, p1 = c[0] * 0xD2511F53, c[2] * 0xCD9E8D57
        c = [((p1 >> 32) & M) ^ c[1] ^ k0, p1 & M, ((p0 >> 32) & M) ^ c[3] ^ k1, p0 & M]
        k0, k1 = (k0 + 0x9E3779B9) & M, (k1 + 0xBB67AE85) & M
    d = torch.stack([x for w in c for x in (w & 0xFFFF, w >> 16)], 1).reshape(-1)
    return d[first - 8 * q0: first - 8 * q0 + count] >= limit_of(p)


def keep_factor(shape, p, seed, offset, device):
    n = 1
    for s in shape:
        n *= s
    if limit_of(p) == 0:
        return torch.ones(shape, dtype=torch.float64, device=device)
    return keep_mask_fast(n, p, seed, offset, device).reshape(shape).double() * drop_scale(p)


def dropped(x, factor):
    """x * factor with an exact zero where the factor is (whatever x is there)."""
    return torch.where(factor != 0, x * factor, torch.zeros_like(x))


# ---- the operators ---------------------------------------------------------------

def norm(u, u_mag, weight, bias, eps):
    """Layer norm of u, itself off by at most a few units of u_mag."""
    C = u.shape[-1]
    w = torch.ones(C, dtype=torch.float64, device=u.device) if weight is None else weight.double()
    b = torch.zeros(C, dtype=torch.float64, device=u.device) if bias is None else bias.double()
    mean = u.mean(-1, keepdim=True)
    d = u - mean
    rstd = (d.square().mean(-1, keepdim=True) + eps).rsqrt()
    mean_mag = u_mag.mean(-1, keepdim=True)
    d_mag = u_mag + mean_mag                       # of one distance from the mean
    rstd_rel = 2 + (d.abs() * d_mag).mean(-1, keepdim=True) * rstd.square()
    xhat = d * rstd
    y_mag = w.abs() * (d_mag * rstd + xhat.abs() * rstd_rel) + b.abs()
    D = row_depth(C)
    return {"y": (xhat * w + b, y_mag, D), "mean": (mean[:, 0], mean_mag[:, 0], D),
            "rstd": (rstd[:, 0], (rstd * rstd_rel)[:, 0], D)}


def norm_backward(g, u, u_mag, mean, rstd, weight, bias):
    """du and the parameters' gradients, from the statistics as given."""
    N, C = u.shape
    g, mean, rstd = g.double(), mean.double()[:, None], rstd.double()[:, None]
    w = torch.ones(C, dtype=torch.float64, device=u.device) if weight is None else weight.double()
    xhat = (u - mean) * rstd
    xhat_mag = (u_mag + mean.abs()) * rstd
    gw = g * w
    m2 = (gw * xhat).mean(-1, keepdim=True)
    m2_mag = (gw.abs() * xhat_mag).mean(-1, keepdim=True)
    du = rstd * (gw - gw.mean(-1, keepdim=True) - xhat * m2)
    du_mag = rstd * (gw.abs() + gw.abs().mean(-1, keepdim=True) + xhat_mag * m2_mag)
    out = {"du": (du, du_mag, row_depth(C))}
    if weight is not None:
        out["d_weight"] = ((g * xhat).sum(0), (g.abs() * xhat_mag).sum(0), rows_depth(N))
    if bias is not None:
        out["d_bias"] = (g.sum(0), g.abs().sum(0), rows_depth(N))
    return out


def layer_norm(x, weight, bias, eps):
    return norm(x.double(), x.double().abs(), weight, bias, eps)


def layer_norm_backward(G, x, mean, rstd, weight, bias):
    out = norm_backward(G, x.double(), x.double().abs(), mean, rstd, weight, bias)
    out["d_x"] = out.pop("du")
    return out


def read(X, h):
    t = X.double() * h.double()[:, :, None]
    return t.sum(1), t.abs().sum(1)


def stream_norm(X, h, weight, bias, eps):
    return norm(*read(X, h), weight, bias, eps)


def stream_norm_backward(G, X, h, mean, rstd, weight, bias):
    X, h = X.double(), h.double()
    out = norm_backward(G, *read(X, h), mean, rstd, weight, bias)
    du, du_mag, D = out.pop("du")
    out["d_X"] = (h[:, :, None] * du[:, None], h.abs()[:, :, None] * du_mag[:, None], D)
    out["d_h_pre"] = ((X * du[:, None]).sum(-1), (X.abs() * du_mag[:, None]).sum(-1), 2 * D)
    return out


def stream_mix(X, T, y, h, factor):
    X, T, h = X.double(), T.double(), h.double()
    y = dropped(y.double(), factor)
    return {"X": (T @ X + h[:, :, None] * y[:, None], T.abs() @ X.abs() + h.abs()[:, :, None] * y.abs()[:, None], 8)}


def stream_mix_backward(G, X, T, y, h, factor):
    G, X, T, h = G.double(), X.double(), T.double(), h.double()
    y = dropped(y.double(), factor)
    D = row_depth(X.shape[-1])
    hg, hg_mag = (h[:, None] @ G)[:, 0], (h.abs()[:, None] @ G.abs())[:, 0]
    return {"d_X": (T.transpose(1, 2) @ G, T.abs().transpose(1, 2) @ G.abs(), 8),
            "d_T": (G @ X.transpose(1, 2), G.abs() @ X.abs().transpose(1, 2), D),
            "d_y": (dropped(hg, factor), dropped(hg_mag, factor), 8),
            "d_h_post": ((G * y[:, None]).sum(-1), (G.abs() * y.abs()[:, None]).sum(-1), D)}


def check(got, want, what=""):
    """Holds every output of `want` in `got` to its bound."""
    for name, (value, mag, depth) in want.items():
        x = got[name]
        info = torch.finfo(x.dtype)
        assert x.shape == value.shape, (what, name, x.shape, value.shape)
        bound = (info.eps / 2 * value.abs() + (1 + info.eps) * depth * UNIT * mag + info.smallest_normal * info.eps / 2)
        nearest = value.to(x.dtype)
        over = torch.isinf(nearest)
        assert bool((x[over] == nearest[over]).all()), (what, name, "overflow")
        off = torch.where(over, 0.0, (x.double() - value).abs())
        assert bool(torch.isfinite(off).all()), (what, name, "not finite")
        worst = (off / bound).max().item() if off.numel() else 0.0
        assert worst <= 1.0, (what, name, f"{worst:.3g} times the bound")
