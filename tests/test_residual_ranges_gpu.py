"""The residual path's kernels where the choice of a launch, a sum or an
address depends on the size: the first call of a process, rows far from zero,
rows too wide for the rings, strided batches of many rows, and tensors of
different types.  The operators in 64 bits and most bounds are
residual_reference.py's; a tighter one of the norms' backward is derived here."""
import os
import subprocess
import sys
from concurrent.futures import ThreadPoolExecutor

import numpy
import pytest
import torch

import mhc_proj
import residual_reference as ref
from mhc_proj import residual
from test_residual_gpu import DTYPES, EPS, affine_of, gen, leaf, mixing, normal, offset_copy, rows, same_bits, streams

pytestmark = pytest.mark.gpu
f = mhc_proj.torch
HERE = os.path.dirname(os.path.abspath(__file__))


# ---- the first call of a process -----------------------------------------------------

# (type, width, offset of X): rows of single elements whose stages need between 28
# and 32 KB of dynamic shared memory beside the four streams' 20 KB of static
FIRST = [("float32", C, 0) for C in (41, 42, 43)] + [("float32", 44, 1)] \
    + [("bfloat16", C, 0) for C in range(81, 88)] + [("bfloat16", 88, 1), ("float16", 81, 0), ("float16", 88, 1)]

FIRST_CALL = """
import sys
import torch, mhc_proj
import residual_reference as ref
from test_residual_gpu import gen, normal, offset_copy, streams
dtype, C, offset = getattr(torch, sys.argv[1]), int(sys.argv[2]), int(sys.argv[3])
g = gen(C)
X, G, h = streams(9, C, g, dtype), normal(g, 9, C).to(dtype), torch.sigmoid(normal(g, 9, 4))
w, b = 1 + 0.3 * normal(g, C), 0.3 * normal(g, C)
mean, rstd = normal(g, 9), 0.5 + torch.rand(9, device="cuda", generator=g)
X = offset_copy(X, offset, 0)
out = mhc_proj.torch.stream_norm_n4_backward(G, X, h, mean, rstd, w, b)
ref.check(out, ref.stream_norm_backward(G, X, h, mean, rstd, w, b))
print("ok")
"""


def first_call(case):
    path = [HERE, os.path.join(os.path.dirname(HERE), "mhc-proj_b200"), os.environ.get("PYTHONPATH", "")]
    env = dict(os.environ, PYTHONPATH=os.pathsep.join(filter(None, path)))
    run = subprocess.run([sys.executable, "-c", FIRST_CALL, *map(str, case)], env=env, cwd=HERE, capture_output=True,
                         text=True, timeout=300)
    return run.stdout.strip() if run.returncode == 0 else run.stderr[-600:]


def test_a_process_may_begin_with_any_width():
    """A kernel's limit of dynamic shared memory, once raised, stays for the
    process, so a call that forgets to raise it fails only where no wider one
    came before it: each case is a process's first call."""
    with ThreadPoolExecutor(4) as pool:
        got = dict(zip(FIRST, pool.map(first_call, FIRST)))
    assert {k: v for k, v in got.items() if v != "ok"} == {}


# ---- rows far from zero ----------------------------------------------------------------

def near_backward(g, u, u_off, mean, rstd, weight, bias, depth, rows_depth):
    """residual_reference.norm_backward with the bound of an evaluation that
    takes the distance u - mean before it multiplies.  The statistics are
    given, so the distance is rounded relative to itself and xhat = (u - mean)
    rstd is off by 2 * 2^-24 |xhat|, and by `u_off` * 2^-24 * rstd where u is
    itself a rounded sum (its roundings times the sum of its terms' sizes).
    Neither grows with |mean|.  The roundings per term (at most 8) are among
    `depth` (at least 33)."""
    g, mean, rstd = g.double(), mean.double()[:, None], rstd.double()[:, None]
    one = torch.ones(u.shape[-1], dtype=torch.float64, device=u.device)
    w = one if weight is None else weight.double()
    xhat = (u - mean) * rstd
    xhat_off = u_off * rstd / depth
    gw = g * w
    m2, m2_mag = (gw * xhat).mean(-1, keepdim=True), (gw.abs() * (xhat.abs() + xhat_off)).mean(-1, keepdim=True)
    du = rstd * (gw - gw.mean(-1, keepdim=True) - xhat * m2)
    du_mag = rstd * (gw.abs() + gw.abs().mean(-1, keepdim=True) + (xhat.abs() + xhat_off) * m2_mag)
    out = {"du": (du, du_mag, depth)}
    if weight is not None:
        xhat_off = u_off * rstd / rows_depth
        out["d_weight"] = ((g * xhat).sum(0), (g.abs() * (xhat.abs() + xhat_off)).sum(0), rows_depth)
    if bias is not None:
        out["d_bias"] = (g.sum(0), g.abs().sum(0), rows_depth)
    return out


def near_layer_norm(G, x, mean, rstd, w, b, depth=None):
    out = near_backward(G, x.double(), 0.0, mean, rstd, w, b, depth or ref.row_depth(x.shape[-1]),
                        ref.rows_depth(len(x)))
    out["d_x"] = out.pop("du")
    return out


def near_stream_norm(G, X, h, mean, rstd, w, b, depth=None):
    u, mag = ref.read(X, h)
    D = depth or ref.row_depth(X.shape[-1])
    out = near_backward(G, u, 4 * mag, mean, rstd, w, b, D, ref.rows_depth(len(X)))
    du, du_mag, _ = out.pop("du")
    X, h = X.double(), h.double()
    out["d_X"] = (h[:, :, None] * du[:, None], h.abs()[:, :, None] * du_mag[:, None], D)
    out["d_h_pre"] = ((X * du[:, None]).sum(-1), (X.abs() * du_mag[:, None]).sum(-1), 2 * D)
    return out


@pytest.mark.parametrize("C", [7, 128, 1001, 4096, 5000, 9000, 20001])
@pytest.mark.parametrize("dtype", DTYPES)
def test_norm_gradients_of_rows_far_from_zero(dtype, C):
    """Centres of 2^10 and -2^9 under a spread of 1 to 8: a product mean * rstd
    rounded before the difference is taken puts 2^-24 * 2^10 on all of a row's
    xhat, where the distance from the mean has 2^-24 * |xhat|."""
    g = gen(C + 70)
    for N in (9, 300):
        centre = torch.where(torch.arange(N, device="cuda") % 2 == 0, 1024.0, -512.0)
        x, G = (8 * normal(g, N, C) + centre[:, None]).to(dtype), normal(g, N, C).to(dtype)
        w, b = affine_of("float32", C, g, dtype)
        out = f.layer_norm(x, w, b, EPS)
        got = f.layer_norm_backward(G, x, out["mean"], out["rstd"], w, b)
        ref.check(got, near_layer_norm(G, x, out["mean"], out["rstd"], w, b), (dtype, N, C))
        X = (8 * normal(g, N, 4, C) + centre[:, None, None]).to(dtype)
        h = torch.sigmoid(normal(g, N, 4))
        out = f.stream_norm_n4(X, h, w, b, EPS)
        got = f.stream_norm_n4_backward(G, X, h, out["mean"], out["rstd"], w, b)
        ref.check(got, near_stream_norm(G, X, h, out["mean"], out["rstd"], w, b), (dtype, N, C, "streams"))


@pytest.mark.parametrize("C", [8, 100, 1001, 4096, 9000, 20001])
@pytest.mark.parametrize("dtype", DTYPES)
def test_rows_at_their_mean_give_the_weight_no_gradient(dtype, C):
    """u = mean in every column: xhat is zero, and so is d_weight, exactly."""
    g = gen(C + 71)
    N = 37
    G, w = normal(g, N, C).to(dtype), 1 + 0.3 * normal(g, C)
    mean, rstd = torch.full((N,), 100.0, device="cuda"), torch.full((N,), EPS ** -0.5, device="cuda")
    x = torch.full((N, C), 100.0, device="cuda", dtype=dtype)
    got = f.layer_norm_backward(G, x, mean, rstd, w, w)
    assert not bool(got["d_weight"].any())
    ref.check(got, near_layer_norm(G, x, mean, rstd, w, w), (dtype, C))
    X, h = x[:, None].expand(N, 4, C), torch.full((N, 4), 0.25, device="cuda")
    got = f.stream_norm_n4_backward(G, X, h, mean, rstd, w, w)
    assert not bool(got["d_weight"].any())


def test_norm_gradients_of_tiny_and_huge_spreads():
    """rstd of 2^66 and 2^-60 in fp32: its square is no fp32 number, or a subnormal one."""
    g = gen(72)
    for C in (96, 4096, 20001):
        for size in (2.0 ** -66, 2.0 ** 60):
            x, G = normal(g, 5, C) * size, normal(g, 5, C)
            w, b = affine_of("float32", C, g, torch.float32)
            mean, rstd = torch.zeros(5, device="cuda"), torch.full((5,), 1 / size, device="cuda")
            got = f.layer_norm_backward(G, x, mean, rstd, w, b)
            ref.check(got, near_layer_norm(G, x, mean, rstd, w, b), (C, size))
            X, h = normal(g, 5, 4, C) * size, torch.rand(5, 4, device="cuda", generator=g)
            got = f.stream_norm_n4_backward(G, X, h, mean, rstd, w, b)
            ref.check(got, near_stream_norm(G, X, h, mean, rstd, w, b), (C, size, "streams"))


# ---- rows wider than the rings hold --------------------------------------------------------

# Terms that the wide rows' kernels add up in 32 bits at a time (64), the tree
# over a block, and the roundings of a term.
WIDE_DEPTH = 96


@pytest.mark.parametrize("C", [(1 << 20) + 5, 1 << 22])
@pytest.mark.parametrize("value", [0.1, 1.7])
def test_sums_of_very_wide_rows(C, value):
    """Rows of one value, whose running sum is rounded the same way again and
    again: C / 256 additions in a row are off by hundreds of units in the last
    place, and the bound here does not grow with C."""
    g = gen(73)
    x = torch.full((2, C), value, device="cuda")
    x[1, ::2] = 0.5 * value
    w, b = torch.full((C,), 1.5, device="cuda"), torch.full((C,), 0.25, device="cuda")
    out = f.layer_norm(x, w, b, EPS)
    ref.check(out, {k: (v, m, WIDE_DEPTH) for k, (v, m, _) in ref.layer_norm(x, w, b, EPS).items()}, C)
    G = torch.full((2, C), 0.3, device="cuda")
    got = f.layer_norm_backward(G, x, out["mean"], out["rstd"], w, b)
    ref.check(got, near_layer_norm(G, x, out["mean"], out["rstd"], w, b, WIDE_DEPTH), C)
    del got, G
    X, h = x[:, None].expand(2, 4, C), torch.rand(2, 4, device="cuda", generator=g)
    out = f.stream_norm_n4(X, h, w, b, EPS)
    ref.check(out, {k: (v, m, WIDE_DEPTH) for k, (v, m, _) in ref.stream_norm(X, h, w, b, EPS).items()}, C)
    G = torch.full((2, C), 0.3, device="cuda")
    G[:, ::3] = 0.7
    got = f.stream_norm_n4_backward(G, X, h, out["mean"], out["rstd"], w, b)
    ref.check(got, near_stream_norm(G, X, h, out["mean"], out["rstd"], w, b, WIDE_DEPTH), C)


# Terms of a coefficient's gradient that a thread adds up in 32 bits at a time (64
# steps of at most four), the tree over a warp or block, and the roundings of a term.
MIX_DEPTH = 288


@pytest.mark.parametrize("N,C,dtype", [(3, 1 << 22, torch.float32), (3, (1 << 22) + 3, torch.float32),
                                       (600, 1 << 18, torch.bfloat16), (600, (1 << 18) + 1, torch.bfloat16),
                                       (600, 1 << 18, torch.float32)])
def test_coefficient_gradients_of_very_wide_tokens(N, C, dtype):
    """Equal products, whose running sum is rounded the same way again and
    again: a token's sums for T and h_post, by a block (few tokens) or a warp."""
    g = gen(74)
    X, y = (torch.full((1, *s, C), 0.9, device="cuda").to(dtype).expand(N, *s, C) for s in ((4,), ()))
    G = torch.full((1, 4, C), 1.1, device="cuda").to(dtype).expand(N, 4, C)
    T, h = mixing(N, g), torch.sigmoid(normal(g, N, 4))
    got = f.stream_mix_n4_backward(G, X, T, y, h)
    for part in (slice(0, 2), slice(N - 1, N)):
        t = [v[part] for v in (G, X, T, y, h)]
        want = ref.stream_mix_backward(*t, torch.ones(t[3].shape, dtype=torch.float64, device="cuda"))
        ref.check({k: v[part] for k, v in got.items()},
                  {k: (v, m, MIX_DEPTH if k in ("d_T", "d_h_post") else d) for k, (v, m, d) in want.items()}, (N, C))


@pytest.mark.parametrize("C", [16384, 16385, 16392, 40000, 40001])
def test_mix_where_tokens_take_several_runs(C):
    g = gen(C)
    N, dtype = 600, torch.bfloat16
    X, y, G = streams(N, C, g, dtype), normal(g, N, C).to(dtype), normal(g, N, 4, C).to(dtype)
    T, h = mixing(N, g), 2 * torch.sigmoid(normal(g, N, 4))
    factor = ref.keep_factor(y.shape, 0.2, 4, 5, "cuda")
    ref.check(f.stream_mix_n4(X, T, y, h, 0.2, 4, 5), ref.stream_mix(X, T, y, h, factor), C)
    for n in (600, 5):
        t = [v[:n] for v in (G, X, T, y, h)]
        ref.check(f.stream_mix_n4_backward(*t, 0.2, 4, 5), ref.stream_mix_backward(*t, factor[:n]), (n, C))


@pytest.mark.parametrize("C", [10232, 10236, 10237, 10240, 10243, 10244, 10248, 12288, 12292, 12797, 14000])
def test_stream_norm_where_fp32_rows_leave_the_rings(C):
    """A stage of the backward holds the four streams and G, of the forward the
    four streams: in fp32 they outgrow a block's shared memory below the
    widest row of the 16-bit types."""
    g = gen(C)
    X, h = streams(300, C, g, torch.float32), torch.sigmoid(normal(g, 300, 4))
    w, b = affine_of("float32", C, g, torch.float32)
    for N in (5, 300):
        out = f.stream_norm_n4(X[:N], h[:N], w, b, EPS)
        ref.check(out, ref.stream_norm(X[:N], h[:N], w, b, EPS), (N, C))
        G = normal(g, N, C)
        got = f.stream_norm_n4_backward(G, X[:N], h[:N], out["mean"], out["rstd"], w, b)
        ref.check(got, near_stream_norm(G, X[:N], h[:N], out["mean"], out["rstd"], w, b), (N, C))


# ---- strides and offsets of batches that take the rings ---------------------------------------

LAYOUTS = [(0, 8), (8, 0), (1, 0), (3, 5), (0, 1), (4, 4)]


@pytest.mark.parametrize("offset,pad", LAYOUTS)
@pytest.mark.parametrize("dtype", DTYPES)
def test_layer_norm_strides_of_many_rows(dtype, offset, pad):
    """G lies as x does, and one element further on."""
    g = gen(80)
    for N, C in ((300, 256), (1500, 33), (1500, 1001), (1500, 1024), (300, 4096), (300, 4099), (300, 9000)):
        x, G = rows(N, C, g, dtype), normal(g, N, C).to(dtype)
        w, b = affine_of("same", C, g, dtype)
        what = (dtype, offset, pad, N, C)
        xs = offset_copy(x, offset, pad)
        out = f.layer_norm(xs, w, b, EPS)
        ref.check(out, ref.layer_norm(x, w, b, EPS), what)
        want = near_layer_norm(G, x, out["mean"], out["rstd"], w, b)
        for Gs in (offset_copy(G, offset, pad), offset_copy(G, offset + 1, pad), G):
            ref.check(f.layer_norm_backward(Gs, xs, out["mean"], out["rstd"], w, b), want, what)


@pytest.mark.parametrize("offset,pad", LAYOUTS)
@pytest.mark.parametrize("dtype", DTYPES)
def test_stream_norm_strides_of_many_rows(dtype, offset, pad):
    g = gen(81)
    for N, C in ((300, 256), (1500, 85), (700, 1001), (1500, 1024), (300, 4096), (300, 4099)):
        X, G, h = streams(N, C, g, dtype), normal(g, N, C).to(dtype), torch.sigmoid(normal(g, N, 4))
        w, b = affine_of("float32", C, g, dtype)
        what = (dtype, offset, pad, N, C)
        Xs, Gs = offset_copy(X, offset, pad), offset_copy(G, offset, pad)
        Xt = offset_copy(X.transpose(0, 1), offset, pad).transpose(0, 1)  # stream-major
        forward = ref.stream_norm(X, h, w, b, EPS)
        out = f.stream_norm_n4(Xs, h, w, b, EPS)
        backward = near_stream_norm(G, X, h, out["mean"], out["rstd"], w, b)
        ref.check(out, forward, what)
        ref.check(f.stream_norm_n4(Xt, h, w, b, EPS), forward, (what, "stream-major"))
        for A, B in ((Xs, Gs), (Xt, G)):
            ref.check(f.stream_norm_n4_backward(B, A, h, out["mean"], out["rstd"], w, b), backward, what)


@pytest.mark.parametrize("offset,pad", LAYOUTS)
@pytest.mark.parametrize("dtype", DTYPES)
def test_stream_mix_strides_of_many_rows(dtype, offset, pad):
    g = gen(82)
    for N, C in ((1500, 25), (700, 49), (1500, 256), (700, 1001), (1500, 1024), (700, 4096), (700, 4099)):
        X, y, G = streams(N, C, g, dtype), normal(g, N, C).to(dtype), normal(g, N, 4, C).to(dtype)
        T, h = mixing(N, g), 2 * torch.sigmoid(normal(g, N, 4))
        what = (dtype, offset, pad, N, C)
        Xs, ys, Gs = offset_copy(X, offset, pad), offset_copy(y, offset, pad), offset_copy(G, offset, pad)
        Xt, Gt = (offset_copy(t.transpose(0, 1), offset, pad).transpose(0, 1) for t in (X, G))
        factor = ref.keep_factor(y.shape, 0.2, 4, 5, "cuda")
        forward, backward = ref.stream_mix(X, T, y, h, factor), ref.stream_mix_backward(G, X, T, y, h, factor)
        for A, B, z in ((Xs, Gs, ys), (Xt, Gt, y), (X, Gt, ys)):
            ref.check(f.stream_mix_n4(A, T, z, h, 0.2, 4, 5), forward, what)
            ref.check(f.stream_mix_n4_backward(B, A, T, z, h, 0.2, 4, 5), backward, what)


@pytest.mark.parametrize("step", [1, 5, 8, 32])
@pytest.mark.parametrize("dtype", DTYPES)
def test_rows_that_overlap(dtype, step):
    """Windows of one array, `step` elements apart: rows that share elements."""
    g = gen(83)
    for N, C in ((700, 55), (700, 264)):
        line, y, G = normal(g, (4 * N - 1) * step + C).to(dtype), normal(g, N, C).to(dtype), normal(g, N, C).to(dtype)
        x, X = line.as_strided((N, C), (step, 1)), line.as_strided((N, 4, C), (4 * step, step, 1))
        out = f.layer_norm(x, None, None, EPS)
        ref.check(out, ref.layer_norm(x, None, None, EPS), (dtype, step, C))
        ref.check(f.layer_norm_backward(G, x, out["mean"], out["rstd"]),
                  near_layer_norm(G, x, out["mean"], out["rstd"], None, None), (dtype, step, C))
        h, T = torch.sigmoid(normal(g, N, 4)), mixing(N, g)
        out = f.stream_norm_n4(X, h, None, None, EPS)
        ref.check(out, ref.stream_norm(X, h, None, None, EPS), (dtype, step, C))
        ref.check(f.stream_norm_n4_backward(G, X, h, out["mean"], out["rstd"]),
                  near_stream_norm(G, X, h, out["mean"], out["rstd"], None, None), (dtype, step, C))
        factor = ref.keep_factor(y.shape, 0.2, 4, 5, "cuda")
        ref.check(f.stream_mix_n4(X, T, x, h, 0.2, 4, 5), ref.stream_mix(X, T, x, h, factor), (dtype, step, C))
        ref.check(f.stream_mix_n4_backward(X, X, T, x, h, 0.2, 4, 5), ref.stream_mix_backward(X, X, T, x, h, factor),
                  (dtype, step, C))


@pytest.mark.parametrize("C", [33, 96, 1001, 1024])
@pytest.mark.parametrize("dtype", DTYPES)
def test_operands_that_are_broadcast(dtype, C):
    """One row for all tokens, one stream for a token's four: strides of zero."""
    g = gen(C + 84)
    N = 700
    x, G = rows(1, C, g, dtype).expand(N, C), normal(g, 1, C).to(dtype).expand(N, C)
    w, b = affine_of("same", C, g, dtype)
    out = f.layer_norm(x, w, b, EPS)
    ref.check(out, ref.layer_norm(x, w, b, EPS), (dtype, C))
    ref.check(f.layer_norm_backward(G, x, out["mean"], out["rstd"], w, b),
              near_layer_norm(G, x, out["mean"], out["rstd"], w, b), (dtype, C))
    h, T = torch.sigmoid(normal(g, 1, 4)).expand(N, 4), mixing(1, g).expand(N, 4, 4)
    factor = ref.keep_factor((N, C), 0.3, 8, 9, "cuda")
    for X in (streams(1, C, g, dtype).expand(N, 4, C), rows(N, C, g, dtype)[:, None].expand(N, 4, C)):
        out = f.stream_norm_n4(X, h, w, b, EPS)
        ref.check(out, ref.stream_norm(X, h, w, b, EPS), (dtype, C))
        ref.check(f.stream_norm_n4_backward(G, X, h, out["mean"], out["rstd"], w, b),
                  near_stream_norm(G, X, h, out["mean"], out["rstd"], w, b), (dtype, C))
        ref.check(f.stream_mix_n4(X, T, x, h, 0.3, 8, 9), ref.stream_mix(X, T, x, h, factor), (dtype, C))
        G4 = G[:, None].expand(N, 4, C)
        ref.check(f.stream_mix_n4_backward(G4, X, T, x, h, 0.3, 8, 9), ref.stream_mix_backward(G4, X, T, x, h, factor),
                  (dtype, C))


@pytest.mark.parametrize("cd", DTYPES)
def test_coefficients_at_any_alignment(cd):
    """T and h that start one element into a buffer, and columns of a wider array."""
    g = gen(85)
    for N, C in ((5, 96), (700, 96), (700, 1001)):
        X, y, G = streams(N, C, g, torch.bfloat16), normal(g, N, C).bfloat16(), normal(g, N, 4, C).bfloat16()
        T, h = mixing(N, g, cd), torch.sigmoid(normal(g, N, 4)).to(cd)
        T1, h1 = offset_copy(T.reshape(1, -1), 1, 0).view(N, 4, 4), offset_copy(h.reshape(1, -1), 1, 0).view(N, 4)
        for A, c in ((T1, h1), (T, h1), (T1, h), (offset_copy(T, 0, 3), offset_copy(h, 1, 20))):
            assert same_bits(f.stream_mix_n4(X, A, y, c, 0.1, 5)["X"], f.stream_mix_n4(X, T, y, h, 0.1, 5)["X"])
            got, want = (f.stream_mix_n4_backward(G, X, *t, 0.1, 5) for t in ((A, y, c), (T, y, h)))
            assert all(same_bits(got[k], want[k]) for k in want)
            out = f.stream_norm_n4(X, c)
            assert same_bits(out["y"], f.stream_norm_n4(X, h)["y"])
            got, want = (f.stream_norm_n4_backward(y, X, t, out["mean"], out["rstd"]) for t in (c, h))
            assert all(same_bits(got[k], want[k]) for k in want)


# ---- tensors of different types -------------------------------------------------------------

@pytest.mark.parametrize("xt,yt", [(torch.float32, torch.bfloat16), (torch.bfloat16, torch.float32),
                                   (torch.float32, torch.float16), (torch.float16, torch.bfloat16)])
def test_mix_of_streams_and_outputs_of_different_types(xt, yt):
    """Streams kept in 32 bits around a 16-bit sublayer, and the other way round."""
    g = gen(90)
    for N, C in ((5, 96), (700, 1001)):
        X, y = streams(N, C, g, xt), normal(g, N, C).to(yt)
        T, h = mixing(N, g), 2 * torch.sigmoid(normal(g, N, 4))
        factor = ref.keep_factor(y.shape, 0.1, 6, 7, "cuda")
        out = f.stream_mix_n4(X, T, y, h, 0.1, 6, 7)
        assert out["X"].dtype == xt
        ref.check(out, ref.stream_mix(X, T, y, h, factor), (xt, yt, N, C))
        for G in (normal(g, N, 4, C).to(xt), normal(g, N, 4, C).to(yt)):
            got = f.stream_mix_n4_backward(G, X, T, y, h, 0.1, 6, 7)
            assert got["d_X"].dtype == xt and got["d_y"].dtype == yt
            ref.check(got, ref.stream_mix_backward(G, X, T, y, h, factor), (xt, yt, N, C))


def test_a_layer_with_streams_in_32_bits_and_a_16_bit_sublayer():
    g = gen(91)
    X, h, W = leaf(normal(g, 6, 4, 96)), leaf(torch.sigmoid(normal(g, 6, 4))), leaf(normal(g, 96, 96).bfloat16() / 8)
    T, norm, mix = mixing(6, g), mhc_proj.MHCStreamNormN4(96, device="cuda"), mhc_proj.MHCStreamMixN4()
    out = mix(X, T, norm(X, h).bfloat16() @ W, h)
    out.backward(torch.ones_like(out))
    assert out.dtype == X.grad.dtype == h.grad.dtype == torch.float32 and W.grad.dtype == torch.bfloat16
    n = f.stream_norm_n4(X.detach(), h.detach(), norm.weight.detach(), norm.bias.detach())["y"].bfloat16()
    y = n @ W.detach()
    assert same_bits(out.detach(), f.stream_mix_n4(X.detach(), T, y, h.detach())["X"])


# ---- gradients of some of the inputs -----------------------------------------------------------

def test_gradients_of_some_of_the_inputs():
    """Frozen inputs get none, and the others the same bits."""
    g = gen(92)
    N, C = 37, 264
    mix, norm, read = mhc_proj.MHCStreamMixN4(p=0.2), residual.MHCLayerNormFunction.apply, residual.MHCStreamNormN4Function.apply
    x, X, G, G4 = normal(g, N, C), normal(g, N, 4, C), normal(g, N, C), normal(g, N, 4, C)
    w, b, h, T = 1 + normal(g, C), normal(g, C), torch.rand(N, 4, device="cuda", generator=g), mixing(N, g)
    for call, inputs, grad in ((norm, (x, w, b), G), (read, (X, h, w, b), G),
                               (lambda *t: mix(*t, seed=3), (X, T, x, h), G4)):
        leaves = [leaf(t) for t in inputs]
        call(*leaves).backward(grad)
        for some in range(1, 1 << len(inputs)):
            part = [leaf(t) if some >> i & 1 else t for i, t in enumerate(inputs)]
            call(*part).backward(grad)
            for i, (p, full) in enumerate(zip(part, leaves)):
                assert same_bits(p.grad, full.grad) if some >> i & 1 else p.grad is None


def test_modules_on_empty_batches():
    x, X, C = torch.empty(2, 0, 8, device="cuda"), torch.empty(0, 3, 4, 8, device="cuda"), 8
    norm, read = mhc_proj.MHCLayerNorm(C, device="cuda"), mhc_proj.MHCStreamNormN4(C, device="cuda")
    mix, x, X = mhc_proj.MHCStreamMixN4(p=0.5), leaf(x), leaf(X)
    norm(x).sum().backward()
    h, T, y = leaf(torch.empty(0, 3, 4, device="cuda")), torch.empty(0, 3, 4, 4, device="cuda"), leaf(X.detach()[:, :, 0])
    (read(X, h).sum() + mix(X, T, y, h).sum() + mhc_proj.MHCDropout(0.5)(y).sum()).backward()
    for t in (x, X, h, y):
        assert t.grad.shape == t.shape
    for m in (norm, read):
        assert not bool(m.weight.grad.any()) and not bool(m.bias.grad.any())


# ---- the backward's workspace ---------------------------------------------------------------

def test_a_wide_backward_allocates_what_it_uses():
    """256 rows of 2^20 elements: 32 rows of partial sums (0.25 GB) beside d_x
    (0.5 GB), not one for every row (2 GB)."""
    N, C = 256, 1 << 20
    x = torch.ones(N, C, device="cuda", dtype=torch.bfloat16)
    w = torch.ones(C, device="cuda")
    mean, rstd = torch.zeros(N, device="cuda"), torch.ones(N, device="cuda")
    torch.cuda.synchronize()
    torch.cuda.reset_peak_memory_stats()
    before = torch.cuda.memory_allocated()
    got = f.layer_norm_backward(x, x, mean, rstd, w, w)
    torch.cuda.synchronize()
    assert torch.cuda.max_memory_allocated() - before < x.numel() * 2 + 33 * 2 * C * 4 + 2 * C * 4 + (1 << 22)
    assert bool((got["d_weight"] == N).all()) and bool((got["d_bias"] == N).all())


# ---- seeds -------------------------------------------------------------------------------------

def test_seeds_of_64_bits():
    """What torch.initial_seed() may return: the key is the seed's 64 bits."""
    x = torch.ones(1000, device="cuda")
    for seed in (2 ** 63, 2 ** 64 - 5):
        assert torch.equal(f.dropout(x, 0.5, seed, 1)["y"], f.dropout(x, 0.5, seed - 2 ** 64, 1)["y"])
    assert torch.equal(f.dropout(x, 0.5, numpy.int64(-7), 1)["y"], f.dropout(x, 0.5, -7, 1)["y"])
    m = mhc_proj.MHCDropout(0.5)
    assert torch.equal(m(x, seed=2 ** 63 + 9), f.dropout(x, 0.5, 9 - 2 ** 63)["y"])
