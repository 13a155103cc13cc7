"""The residual path's kernels against the operators in 64 bits
(residual_reference.py, where the bounds are derived)."""
import gc
import threading

import pytest
import torch

import mhc_proj
import residual_reference as ref
from mhc_proj import capi

pytestmark = pytest.mark.gpu
f = mhc_proj.torch

DTYPES = [torch.float32, torch.bfloat16, torch.float16]
EPS = 1e-5
# one element, both sides of a warp, of 16-byte pieces, of the widths at which
# the kernels change, and odd ones in between
WIDTHS = [1, 2, 7, 8, 31, 32, 33, 64, 136, 255, 256, 257, 512, 520, 1000, 1024, 1025, 1032, 2047, 2048, 4096, 4099, 4104,
          8192, 8200, 16384, 16392, 20001, 33000]


def gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def normal(g, *shape):
    return torch.randn(*shape, device="cuda", generator=g)


def affine_of(kind, C, g, dtype):
    """(weight, bias) of the kinds a caller has."""
    if kind == "none":
        return None, None
    at = dtype if kind == "same" else torch.float32
    w, b = (1 + 0.3 * normal(g, C)).to(at), (0.3 * normal(g, C)).to(at)
    return (w, None) if kind == "weight" else (w, b)


def rows(N, C, g, dtype):
    """Rows with centres and sizes of their own."""
    return (normal(g, N, C) * (0.1 + 2 * torch.rand(N, 1, device="cuda", generator=g)) + normal(g, N, 1)).to(dtype)


def same_bits(a, b):
    kind = torch.int16 if a.element_size() == 2 else torch.int32
    return a.dtype == b.dtype and a.shape == b.shape and torch.equal(a.contiguous().view(kind), b.contiguous().view(kind))


def offset_copy(x, offset, pad):
    """x's values in a view whose rows are `pad` elements apart and start `offset` elements into a buffer."""
    buf = torch.full((x.numel() // x.shape[-1] * (x.shape[-1] + pad) + offset + 1,), float("nan"), device=x.device,
                     dtype=x.dtype)
    C = x.shape[-1]
    strides, s = [], C + pad
    for n in reversed(x.shape[:-1]):
        strides.append(s)
        s *= n
    v = torch.as_strided(buf, x.shape, (*reversed(strides), 1), offset)
    v.copy_(x)
    return v


# ---- layer norm -----------------------------------------------------------------

def run_norm(x, w, b, G, what):
    out = f.layer_norm(x, w, b, EPS)
    ref.check(out, ref.layer_norm(x, w, b, EPS), (what, "forward"))
    assert out["y"].dtype == x.dtype and out["y"].is_contiguous()
    g = f.layer_norm_backward(G, x, out["mean"], out["rstd"], w, b)
    ref.check(g, ref.layer_norm_backward(G, x, out["mean"], out["rstd"], w, b), (what, "backward"))
    assert g["d_x"].dtype == x.dtype and ("d_weight" in g) == (w is not None) and ("d_bias" in g) == (b is not None)
    return out, g


@pytest.mark.parametrize("C", WIDTHS)
@pytest.mark.parametrize("dtype", DTYPES)
def test_layer_norm_widths(dtype, C):
    g = gen(C)
    for N, kind in ((1, "same"), (3, "float32"), (41, "same"), (300, "float32")):
        x, G = rows(N, C, g, dtype), normal(g, N, C).to(dtype)
        w, b = affine_of(kind, C, g, dtype)
        run_norm(x, w, b, G, (dtype, N, C, kind))


@pytest.mark.parametrize("kind", ["none", "weight", "same", "float32"])
@pytest.mark.parametrize("dtype", DTYPES)
def test_layer_norm_affine_kinds(dtype, kind):
    g = gen(5)
    for N, C in ((17, 96), (9, 1536), (5, 777)):
        x, G = rows(N, C, g, dtype), normal(g, N, C).to(dtype)
        run_norm(x, *affine_of(kind, C, g, dtype), G, (dtype, N, C, kind))


@pytest.mark.parametrize("dtype", DTYPES)
def test_layer_norm_many_rows(dtype):
    """More rows than the GPU holds at once, so that every block takes several."""
    g = gen(6)
    for N, C in ((20011, 64), (9001, 520), (5003, 1025), (3001, 2048), (30001, 33)):
        x, G = rows(N, C, g, dtype), normal(g, N, C).to(dtype)
        run_norm(x, *affine_of("float32", C, g, dtype), G, (dtype, N, C))


@pytest.mark.parametrize("offset,pad", [(0, 8), (8, 0), (1, 0), (3, 5), (0, 1), (4, 4)])
@pytest.mark.parametrize("dtype", DTYPES)
def test_layer_norm_strides_and_offsets(dtype, offset, pad):
    g = gen(7)
    for N, C in ((37, 256), (21, 1024), (11, 4096), (13, 1001)):
        x, G = rows(N, C, g, dtype), normal(g, N, C).to(dtype)
        w, b = affine_of("same", C, g, dtype)
        out, grad = run_norm(x, w, b, G, (N, C))
        xs, Gs = offset_copy(x, offset, pad), offset_copy(G, offset, 0)
        ws = offset_copy(w[None], 1, 0)[0]
        o2 = f.layer_norm(xs, ws, b, EPS)
        ref.check(o2, ref.layer_norm(x, w, b, EPS), (dtype, offset, pad, N, C))
        ref.check(f.layer_norm_backward(Gs, xs, out["mean"], out["rstd"], ws, b),
                  ref.layer_norm_backward(G, x, out["mean"], out["rstd"], w, b), (dtype, offset, pad, N, C))


def test_layer_norm_layouts_and_types_that_are_converted():
    g = gen(8)
    x = rows(64, 48, g, torch.float32)
    w, b = affine_of("float32", 48, g, torch.float32)
    want = f.layer_norm(x, w, b)["y"]
    assert same_bits(f.layer_norm(x.t().contiguous().t(), w, b)["y"], want)          # column-major
    assert same_bits(f.layer_norm(x[:1].expand(64, 48), w, b)["y"], want[:1].expand(64, 48).contiguous())
    d = f.layer_norm(x.double(), w.double(), b)
    assert d["y"].dtype == torch.float64 and torch.equal(d["y"].float(), want)
    c = f.layer_norm(x.cpu(), w, b)
    assert c["y"].device.type == "cpu" and torch.equal(c["y"], want.cpu())
    # G of another type than x: both as fp32, d_x in x's type
    xb, G = x.bfloat16(), normal(g, 64, 48)
    o = f.layer_norm(xb, w, b)
    m = f.layer_norm_backward(G, xb, o["mean"], o["rstd"], w, b.bfloat16())
    assert m["d_x"].dtype == torch.bfloat16 and m["d_weight"].dtype == torch.float32
    assert m["d_bias"].dtype == torch.bfloat16
    ref.check(m, ref.layer_norm_backward(G, xb, o["mean"], o["rstd"], w, b))


@pytest.mark.parametrize("C", [1, 8, 100, 4096])
def test_layer_norm_constant_rows(C):
    """Variance zero: y is the bias, and the gradient stays finite."""
    x = torch.full((5, C), 3.25, device="cuda")
    w, b = affine_of("float32", C, gen(9), torch.float32)
    out, _ = run_norm(x, w, b, normal(gen(10), 5, C), C)
    assert torch.equal(out["y"], b.expand(5, C))


@pytest.mark.parametrize("bad", [float("nan"), float("inf"), -float("inf")])
@pytest.mark.parametrize("C", [64, 1000, 4096])
def test_layer_norm_non_finite_rows_stay_alone(C, bad):
    g = gen(11)
    x = rows(33, C, g, torch.float32)
    w, b = affine_of("float32", C, g, torch.float32)
    want = f.layer_norm(x, w, b)["y"]
    x[7, C // 2] = bad
    got = f.layer_norm(x, w, b)["y"]
    assert bool(torch.isnan(got[7]).all())
    keep = torch.arange(33, device="cuda") != 7
    assert same_bits(got[keep], want[keep])


def test_layer_norm_far_from_zero():
    """A centre 2^10 times the spread: a difference of squares would lose the variance."""
    g = gen(12)
    for C in (128, 4096):
        x = (normal(g, 9, C) + 1024.0)
        run_norm(x, None, None, normal(g, 9, C), C)


def test_layer_norm_empty_batch():
    w = torch.ones(8, device="cuda")
    out = f.layer_norm(torch.empty(0, 8, device="cuda"), w, w)
    assert out["y"].shape == (0, 8) and out["mean"].shape == (0,)
    g = f.layer_norm_backward(torch.empty(0, 8, device="cuda"), torch.empty(0, 8, device="cuda"), out["mean"],
                              out["rstd"], w, w)
    assert torch.equal(g["d_weight"], torch.zeros(8, device="cuda")) and torch.equal(g["d_bias"], g["d_weight"])


# ---- dropout ---------------------------------------------------------------------

@pytest.mark.parametrize("p", [0.0, 1e-6, 0.1, 0.5, 0.99999, 1.0])
@pytest.mark.parametrize("dtype", DTYPES)
def test_dropout_values(dtype, p):
    g = gen(20)
    for count, seed, offset in ((1, 0, 0), (7, 3, 1), (8, -5, 2), (1000, 2 ** 62 + 1, 2 ** 41 + 3), (70001, 77, 0)):
        x = normal(g, count).to(dtype)
        y = f.dropout(x, p, seed, offset)["y"]
        factor = ref.keep_factor((count,), p, seed, offset, "cuda")
        want = ref.dropped(x.double(), factor)
        ref.check({"y": y}, {"y": (want, want.abs(), 2)}, (dtype, p, count))
        assert bool((y[factor == 0] == 0).all())
        assert same_bits(y, f.dropout_backward(x, p, seed, offset)["d_x"])


def test_dropout_mask_against_the_scalar_generator():
    x = torch.ones(333, device="cuda")
    for seed, offset in ((0, 0), (-1, 2 ** 62), (123456789012345, 9)):
        y = f.dropout(x, 0.3, seed, offset)["y"]
        assert torch.equal((y != 0).cpu(), ref.keep_mask(333, 0.3, seed, offset))


def test_dropout_drops_non_finite_values_to_zero():
    x = torch.full((4096,), float("nan"), device="cuda")
    x[::2] = float("inf")
    y = f.dropout(x, 0.5, 1)["y"]
    kept = ref.keep_mask_fast(4096, 0.5, 1, 0, "cuda")
    assert bool((y[~kept] == 0).all()) and not bool(torch.isfinite(y[kept]).any())


@pytest.mark.parametrize("dtype", DTYPES)
def test_dropout_layouts(dtype):
    """The mask goes by the element's logical index, whatever the layout."""
    g = gen(21)
    x = normal(g, 37, 53).to(dtype)
    want = f.dropout(x, 0.25, 5, 6)["y"]
    assert same_bits(f.dropout(x.reshape(-1), 0.25, 5, 6)["y"].view(37, 53), want)
    assert same_bits(f.dropout(x.t().contiguous().t(), 0.25, 5, 6)["y"], want)
    for offset in range(1, 9):
        assert same_bits(f.dropout(offset_copy(x.reshape(1, -1), offset, 0), 0.25, 5, 6)["y"].view(37, 53), want)
    assert f.dropout(x[:0], 0.25, 5)["y"].shape == (0, 53)


def test_dropout_seed_forms():
    x = torch.ones(1000, device="cuda")
    want = f.dropout(x, 0.5, -987654321, 3)["y"]
    for seed in (torch.tensor(-987654321), torch.tensor([-987654321]), torch.tensor([-987654321], device="cuda")):
        assert torch.equal(f.dropout(x, 0.5, seed, 3)["y"], want)
    assert not torch.equal(f.dropout(x, 0.5, -987654321, 4)["y"], want)
    assert not torch.equal(f.dropout(x, 0.5, -987654320, 3)["y"], want)


def test_dropout_in_place_through_the_c_abi():
    x = normal(gen(22), 10007)
    want = f.dropout(x, 0.4, 8, 9)["y"]
    capi.dropout(x.data_ptr(), x.data_ptr(), capi.MHC_DTYPE_F32, x.numel(), 0.4, 8, 0, 9,
                 torch.cuda.current_stream().cuda_stream)
    assert same_bits(x, want)


# ---- the normalised read of the streams -------------------------------------------

def streams(N, C, g, dtype):
    return (normal(g, N, 4, C) + normal(g, N, 1, C) + 0.5 * normal(g, N, 4, 1)).to(dtype)


def run_stream_norm(X, h, w, b, G, what):
    out = f.stream_norm_n4(X, h, w, b, EPS)
    ref.check(out, ref.stream_norm(X, h, w, b, EPS), (what, "forward"))
    g = f.stream_norm_n4_backward(G, X, h, out["mean"], out["rstd"], w, b)
    ref.check(g, ref.stream_norm_backward(G, X, h, out["mean"], out["rstd"], w, b), (what, "backward"))
    assert g["d_X"].dtype == X.dtype and g["d_h_pre"].dtype == h.dtype
    return out, g


@pytest.mark.parametrize("C", WIDTHS)
@pytest.mark.parametrize("dtype", DTYPES)
def test_stream_norm_widths(dtype, C):
    g = gen(C + 1)
    for N, kind, hd in ((1, "same", torch.float32), (3, "float32", dtype), (41, "same", torch.float32),
                        (300, "float32", torch.float32)):
        X, G, h = streams(N, C, g, dtype), normal(g, N, C).to(dtype), torch.sigmoid(normal(g, N, 4)).to(hd)
        run_stream_norm(X, h, *affine_of(kind, C, g, dtype), G, (dtype, N, C, kind))


@pytest.mark.parametrize("dtype", DTYPES)
def test_stream_norm_many_rows(dtype):
    g = gen(30)
    for N, C, kind in ((20011, 64, "float32"), (5003, 520, "weight"), (3001, 1025, "none"), (2003, 2048, "same")):
        X, G, h = streams(N, C, g, dtype), normal(g, N, C).to(dtype), torch.sigmoid(normal(g, N, 4))
        run_stream_norm(X, h, *affine_of(kind, C, g, dtype), G, (dtype, N, C))


@pytest.mark.parametrize("offset,pad", [(0, 8), (8, 0), (1, 0), (3, 5), (4, 4)])
@pytest.mark.parametrize("dtype", DTYPES)
def test_stream_norm_strides_and_offsets(dtype, offset, pad):
    g = gen(31)
    for N, C in ((37, 256), (11, 1024), (5, 4096), (13, 1001)):
        X, G, h = streams(N, C, g, dtype), normal(g, N, C).to(dtype), torch.sigmoid(normal(g, N, 4))
        w, b = affine_of("float32", C, g, dtype)
        out, _ = run_stream_norm(X, h, w, b, G, (N, C))
        Xs, Gs = offset_copy(X, offset, pad), offset_copy(G, offset, pad)
        Xt = Xs.transpose(0, 1).contiguous().transpose(0, 1)  # stream-major
        for Y in (Xs, Xt):
            ref.check(f.stream_norm_n4(Y, h, w, b, EPS), ref.stream_norm(X, h, w, b, EPS), (dtype, offset, pad))
            ref.check(f.stream_norm_n4_backward(Gs, Y, h, out["mean"], out["rstd"], w, b),
                      ref.stream_norm_backward(G, X, h, out["mean"], out["rstd"], w, b), (dtype, offset, pad))


def test_stream_norm_is_layer_norm_of_the_sum():
    """With one stream's weight 1 and the others' 0 it is that stream's layer norm."""
    g = gen(32)
    X = streams(19, 1032, g, torch.bfloat16)
    w, b = affine_of("same", 1032, g, torch.bfloat16)
    h = torch.zeros(19, 4, device="cuda")
    h[:, 2] = 1
    ref.check(f.stream_norm_n4(X, h, w, b), ref.layer_norm(X[:, 2], w, b, EPS))


def test_stream_norm_equal_streams():
    """Four copies of one stream, as after the embedding: dh is four equal sums that nearly cancel."""
    g = gen(33)
    x = normal(g, 7, 1, 2048)
    X, h = x.expand(7, 4, 2048), torch.sigmoid(normal(g, 7, 4))
    _, grad = run_stream_norm(X, h, *affine_of("float32", 2048, g, torch.float32), normal(g, 7, 2048), "equal")
    assert same_bits(grad["d_h_pre"][:, 0], grad["d_h_pre"][:, 3])


def test_stream_norm_empty_batch():
    w = torch.ones(8, device="cuda")
    X, h = torch.empty(0, 4, 8, device="cuda"), torch.empty(0, 4, device="cuda")
    out = f.stream_norm_n4(X, h, w)
    g = f.stream_norm_n4_backward(torch.empty(0, 8, device="cuda"), X, h, out["mean"], out["rstd"], w)
    assert torch.equal(g["d_weight"], torch.zeros(8, device="cuda")) and g["d_X"].shape == (0, 4, 8)


# ---- the residual update -------------------------------------------------------------

def mixing(N, g, dtype=torch.float32):
    return f.birkhoff_proj_n4(normal(g, N, 4, 4) + 2 * torch.eye(4, device="cuda"))["T"].to(dtype)


def run_mix(X, T, y, h, G, p, seed, offset, what):
    factor = ref.keep_factor(y.shape, p, seed, offset, "cuda")
    out = f.stream_mix_n4(X, T, y, h, p, seed, offset)
    ref.check(out, ref.stream_mix(X, T, y, h, factor), (what, "forward"))
    g = f.stream_mix_n4_backward(G, X, T, y, h, p, seed, offset)
    ref.check(g, ref.stream_mix_backward(G, X, T, y, h, factor), (what, "backward"))
    assert out["X"].dtype == X.dtype and g["d_T"].dtype == T.dtype and g["d_h_post"].dtype == h.dtype
    assert bool((g["d_y"][factor == 0] == 0).all())
    return out, g


@pytest.mark.parametrize("C", WIDTHS)
@pytest.mark.parametrize("dtype", DTYPES)
def test_stream_mix_widths(dtype, C):
    g = gen(C + 2)
    for N, p, cd in ((1, 0.1, torch.float32), (3, 0.0, dtype), (41, 0.5, torch.float32), (300, 0.1, dtype)):
        X, y, G = streams(N, C, g, dtype), normal(g, N, C).to(dtype), normal(g, N, 4, C).to(dtype)
        T, h = mixing(N, g, cd), 2 * torch.sigmoid(normal(g, N, 4))
        run_mix(X, T, y, h, G, p, C * 1000003, N, (dtype, N, C, p))


@pytest.mark.parametrize("dtype", DTYPES)
def test_stream_mix_many_rows(dtype):
    g = gen(40)
    for N, C, p in ((20011, 64, 0.1), (5003, 520, 0.0), (3001, 1025, 0.1), (2003, 2048, 0.1)):
        X, y, G = streams(N, C, g, dtype), normal(g, N, C).to(dtype), normal(g, N, 4, C).to(dtype)
        run_mix(X, mixing(N, g), y, 2 * torch.sigmoid(normal(g, N, 4)), G, p, 12345, 1, (dtype, N, C))


@pytest.mark.parametrize("offset,pad", [(0, 8), (8, 0), (1, 0), (3, 5), (4, 4)])
@pytest.mark.parametrize("dtype", DTYPES)
def test_stream_mix_strides_and_offsets(dtype, offset, pad):
    g = gen(41)
    for N, C in ((37, 256), (11, 1024), (5, 4096), (13, 1001)):
        X, y, G = streams(N, C, g, dtype), normal(g, N, C).to(dtype), normal(g, N, 4, C).to(dtype)
        T, h = mixing(N, g), 2 * torch.sigmoid(normal(g, N, 4))
        out, grad = run_mix(X, T, y, h, G, 0.2, 4, 5, (N, C))
        Xs, ys, Gs = offset_copy(X, offset, pad), offset_copy(y, offset, pad), offset_copy(G, offset, pad)
        Xt = Xs.transpose(0, 1).contiguous().transpose(0, 1)
        Gt = Gs.transpose(0, 1).contiguous().transpose(0, 1)
        factor = ref.keep_factor(y.shape, 0.2, 4, 5, "cuda")
        for A, B in ((Xs, Gs), (Xt, Gt), (Xs, G)):
            ref.check(f.stream_mix_n4(A, T, ys, h, 0.2, 4, 5), ref.stream_mix(X, T, y, h, factor), (dtype, offset, pad))
            ref.check(f.stream_mix_n4_backward(B, A, T, ys, h, 0.2, 4, 5),
                      ref.stream_mix_backward(G, X, T, y, h, factor), (dtype, offset, pad))


def test_stream_mix_dropout_is_the_dropout_operator():
    """The fused mask is dropout's for the same (p, seed, offset): with T = 0, h = e_0 and p = 1/2 (scale 2, exact)."""
    g = gen(42)
    for C in (96, 1001):
        X, y = streams(23, C, g, torch.bfloat16), normal(g, 23, C).to(torch.bfloat16)
        h = torch.zeros(23, 4, device="cuda")
        h[:, 0] = 1
        out = f.stream_mix_n4(torch.zeros_like(X), torch.zeros(23, 4, 4, device="cuda"), y, h, 0.5, 3, 7)["X"]
        assert torch.equal(out[:, 0], f.dropout(y, 0.5, 3, 7)["y"]) and not bool(out[:, 1:].any())


def test_stream_mix_p_one_drops_all_and_non_finite_dropped_values_vanish():
    g = gen(43)
    X, T, h = streams(9, 64, g, torch.float32), mixing(9, g), torch.rand(9, 4, device="cuda", generator=g)
    y = torch.full((9, 64), float("nan"), device="cuda")
    factor = torch.zeros(9, 64, device="cuda", dtype=torch.float64)
    ref.check(f.stream_mix_n4(X, T, y, h, 1.0, 1), ref.stream_mix(X, T, torch.zeros_like(y), h, factor))
    G = normal(g, 9, 4, 64)
    ref.check(f.stream_mix_n4_backward(G, X, T, y, h, 1.0, 1),
              ref.stream_mix_backward(G, X, T, torch.zeros_like(y), h, factor))


def test_stream_mix_empty_batch():
    e = lambda *s: torch.empty(0, *s, device="cuda")  # noqa: E731
    assert f.stream_mix_n4(e(4, 8), e(4, 4), e(8), e(4))["X"].shape == (0, 4, 8)
    g = f.stream_mix_n4_backward(e(4, 8), e(4, 8), e(4, 4), e(8), e(4))
    assert g["d_T"].shape == (0, 4, 4) and g["d_y"].shape == (0, 8)


# ---- neighbours ---------------------------------------------------------------------------

@pytest.mark.parametrize("bad", [float("nan"), float("inf")])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("N,C", [(9, 1001), (700, 33), (700, 1001), (700, 1025), (700, 72), (5, 4097)])
def test_non_finite_rows_stay_alone(N, C, dtype, bad):
    """Rows of odd widths share 16-byte pieces with their neighbours: every
    second row of all inputs is non-finite, the others keep their results."""
    g = gen(45)
    X, y, G4, G = streams(N, C, g, dtype), normal(g, N, C).to(dtype), normal(g, N, 4, C).to(dtype), rows(N, C, g, dtype)
    h, T = torch.sigmoid(normal(g, N, 4)), mixing(N, g)

    def call():
        a, s = f.layer_norm(y), f.stream_norm_n4(X, h)
        m = f.stream_mix_n4(X, T, y, h, 0.1, 3)
        outs = [a, s, m, f.layer_norm_backward(G, y, a["mean"], a["rstd"]),
                f.stream_norm_n4_backward(G, X, h, s["mean"], s["rstd"]),
                f.stream_mix_n4_backward(G4, X, T, y, h, 0.1, 3)]
        return {f"{i}{k}": v for i, o in enumerate(outs) for k, v in o.items()}

    want = call()
    for t in (X, y, G4, G):
        t[1::2] = bad
    got = call()
    for k in want:
        assert same_bits(got[k][::2], want[k][::2]), k
        assert not bool(torch.isfinite(got[k][1::2]).all()), k


# ---- all of them ------------------------------------------------------------------------

def all_calls(dtype, N, C, seed, drop_seed=7):
    """A closure that calls every function, on inputs made once."""
    g = gen(seed)
    X, y, G4, G = streams(N, C, g, dtype), normal(g, N, C).to(dtype), normal(g, N, 4, C).to(dtype), rows(N, C, g, dtype)
    w, b = affine_of("float32", C, g, dtype)
    h, T = torch.sigmoid(normal(g, N, 4)), mixing(N, g)

    def call():
        a = f.layer_norm(y, w, b)
        s = f.stream_norm_n4(X, h, w, b)
        outs = [a, s, f.layer_norm_backward(G, y, a["mean"], a["rstd"], w, b),
                f.stream_norm_n4_backward(G, X, h, s["mean"], s["rstd"], w, b), f.dropout(y, 0.1, drop_seed, 3),
                f.dropout_backward(G, 0.1, drop_seed, 3), f.stream_mix_n4(X, T, y, h, 0.1, drop_seed, 3),
                f.stream_mix_n4_backward(G4, X, T, y, h, 0.1, drop_seed, 3)]
        return [o[k] for o in outs for k in sorted(o)]

    return call


def test_results_do_not_depend_on_the_run():
    for dtype, N, C in ((torch.bfloat16, 3001, 1024), (torch.float32, 777, 333)):
        call = all_calls(dtype, N, C, 50)
        first = call()
        for _ in range(3):
            assert all(same_bits(a, b) for a, b in zip(first, call()))


def test_other_streams_and_two_at_once():
    calls = [all_calls(torch.bfloat16, 2001, 1024, s) for s in (51, 52)]
    want = [c() for c in calls]
    torch.cuda.synchronize()
    side = [torch.cuda.Stream() for _ in calls]
    for _ in range(5):
        got = []
        for c, s in zip(calls, side):
            with torch.cuda.stream(s):
                got.append(c())
        torch.cuda.synchronize()
        for a, b in zip(got, want):
            assert all(same_bits(x, y) for x, y in zip(a, b))


def test_host_threads_at_once():
    """Two host threads in one kernel with rows of two widths, which need
    different amounts of shared memory: neither call fails or changes the
    other's results."""
    g = gen(58)
    xs = [normal(g, 1200, C).bfloat16() for C in (1000, 2000)]
    Xs = [normal(g, 700, 4, C).bfloat16() for C in (520, 1000)]
    hs = [torch.rand(700, 4, device="cuda", generator=g) for _ in Xs]

    def work(i):
        o = f.layer_norm(xs[i])
        u = capi_layer_norm(xs[i])
        d = f.stream_norm_n4(Xs[i], hs[i])
        return o["y"], u, d["y"]

    def capi_layer_norm(x):
        y = torch.empty_like(x)
        capi.layer_norm(x.data_ptr(), x.stride(0), capi.MHC_DTYPE_BF16, 0, 0, capi.MHC_DTYPE_F32, y.data_ptr(), 0, 0,
                        1e-5, *x.shape, torch.cuda.current_stream().cuda_stream)
        return y

    want = [work(i) for i in range(2)]
    bad = []

    def loop(i):
        try:
            with torch.cuda.stream(torch.cuda.Stream()):
                for k in range(400):
                    got = work(i)
                    if k % 100 == 99 and not all(same_bits(a, b) for a, b in zip(got, want[i])):
                        bad.append((i, k))
        except Exception as e:
            bad.append((i, e))

    torch.cuda.synchronize()
    threads = [threading.Thread(target=loop, args=(i,)) for i in range(2)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    torch.cuda.synchronize()
    assert not bad


def test_captured_and_replayed_with_another_seed():
    seed = torch.tensor([5], device="cuda")
    call = all_calls(torch.bfloat16, 517, 1032, 53, seed)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        call()
    torch.cuda.current_stream().wait_stream(side)
    graphs = []
    for _ in range(2):  # two graphs, each with workspaces of its own
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            out = call()
        graphs.append((g, out))
    for value in (5, -77, 2 ** 62):
        seed.fill_(value)
        want = call()
        for g, out in graphs:
            for o in out:
                o.fill_(float("nan"))
        for g, out in graphs:
            g.replay()
        torch.cuda.synchronize()
        for g, out in graphs:
            assert all(same_bits(a, b) for a, b in zip(out, want))


@pytest.mark.parametrize("dtype,C", [(torch.bfloat16, 1001), (torch.float32, 48), (torch.float16, 4096)])
def test_nothing_is_written_past_the_outputs(dtype, C):
    """Through the C ABI, into buffers with guard bands on both sides."""
    N, band, code = 13, 64, {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}[dtype]
    g = gen(54)
    X, y, G4, G = streams(N, C, g, dtype), normal(g, N, C).to(dtype), normal(g, N, 4, C).to(dtype), rows(N, C, g, dtype)
    w, b = affine_of("float32", C, g, dtype)
    h, T, s = torch.sigmoid(normal(g, N, 4)), mixing(N, g), torch.cuda.current_stream().cuda_stream
    mean, rstd = normal(g, N), torch.rand(N, device="cuda", generator=g)
    bands = []

    def out(n, dt=dtype):
        t = torch.full((n + 2 * band,), 77.0, device="cuda", dtype=dt)
        bands.append(t)
        return t.data_ptr() + band * t.element_size()

    f32 = torch.float32
    ws_bytes = capi.layer_norm_backward_workspace(N, C)
    ws = out((ws_bytes + 3) // 4, f32)
    P = lambda t: t.data_ptr()  # noqa: E731
    capi.layer_norm(P(y), C, code, P(w), P(b), 0, out(N * C), out(N, f32), out(N, f32), 1e-5, N, C, s)
    capi.layer_norm_backward(P(G), C, P(y), C, code, P(mean), P(rstd), P(w), 0, out(N * C), out(C, f32), out(C, f32), N,
                             C, ws, ws_bytes, s)
    capi.dropout(P(y), out(N * C), code, N * C, 0.1, 5, 0, 0, s)
    capi.stream_norm_n4(P(X), 4 * C, C, code, P(h), 0, P(w), P(b), 0, out(N * C), out(N, f32), out(N, f32), 1e-5, N, C,
                        s)
    ws2_bytes = capi.stream_norm_n4_backward_workspace(N, C)
    ws2 = out((ws2_bytes + 3) // 4, f32)
    capi.stream_norm_n4_backward(P(G), C, P(X), 4 * C, C, code, P(h), 0, P(mean), P(rstd), P(w), 0, out(4 * N * C),
                                 out(4 * N, f32), out(C, f32), out(C, f32), N, C, ws2, ws2_bytes, s)
    capi.stream_mix_n4(P(X), 4 * C, C, P(y), C, code, P(T), 0, P(h), 0, out(4 * N * C), 0.1, 5, 0, 0, N, C, s)
    capi.stream_mix_n4_backward(P(G4), 4 * C, C, P(X), 4 * C, C, P(y), C, code, P(T), 0, P(h), 0, out(4 * N * C),
                                out(16 * N, f32), out(N * C), out(4 * N, f32), 0.1, 5, 0, 0, N, C, s)
    torch.cuda.synchronize()
    for t in bands:
        assert bool((t[:band] == 77).all()) and bool((t[-band:] == 77).all())


def test_forward_without_statistics_and_backward_without_parameters():
    """The C ABI's optional pointers."""
    N, C, s = 9, 264, torch.cuda.current_stream().cuda_stream
    g = gen(55)
    x, G = rows(N, C, g, torch.float32), normal(g, N, C)
    out = f.layer_norm(x)
    y, dx = torch.empty_like(x), torch.empty_like(x)
    capi.layer_norm(x.data_ptr(), C, 0, 0, 0, 0, y.data_ptr(), 0, 0, 1e-5, N, C, s)
    assert same_bits(y, out["y"])
    capi.layer_norm_backward(G.data_ptr(), C, x.data_ptr(), C, 0, out["mean"].data_ptr(), out["rstd"].data_ptr(), 0, 0,
                             dx.data_ptr(), 0, 0, N, C, 0, 0, s)
    assert same_bits(dx, f.layer_norm_backward(G, x, out["mean"], out["rstd"])["d_x"])


def test_more_than_2_31_elements():
    """Offsets past 32 bits: the last rows of tensors of over 2^31 elements against the same rows alone."""
    C, last = 4096, 5
    g = gen(56)
    n = (1 << 17) + 8 + last
    N = 4 * n
    x = torch.empty(N, C, device="cuda", dtype=torch.bfloat16).normal_(generator=g)
    w, b = affine_of("float32", C, g, torch.bfloat16)
    out = f.layer_norm(x, w, b)
    ref.check({k: v[-last:] for k, v in out.items()}, ref.layer_norm(x[-last:], w, b, EPS))
    y = out["y"]
    grad = f.layer_norm_backward(y, x, out["mean"], out["rstd"])
    ref.check({"d_x": grad["d_x"][-last:]},
              ref.layer_norm_backward(y[-last:], x[-last:], out["mean"][-last:], out["rstd"][-last:], None, None))
    del grad, out, y
    d = f.dropout(x, 0.1, 3, 4)["y"]
    kept = ref.keep_mask_fast(last * C, 0.1, 3, 4, "cuda", (N - last) * C).view(last, C)
    assert torch.equal(d[-last:] != 0, kept & (x[-last:] != 0))
    del d
    gc.collect()
    X = x.view(n, 4, C)
    h, T = torch.sigmoid(normal(g, n, 4)), mixing(n, g)
    y = x[-n:]
    s = f.stream_norm_n4(X, h, w, b)
    ref.check({k: v[-last:] for k, v in s.items()}, ref.stream_norm(X[-last:], h[-last:], w, b, EPS))
    grad = f.stream_norm_n4_backward(y, X, h, s["mean"], s["rstd"])
    ref.check({k: v[-last:] for k, v in grad.items()},
              ref.stream_norm_backward(y[-last:], X[-last:], h[-last:], s["mean"][-last:], s["rstd"][-last:], None, None))
    factor = torch.where(ref.keep_mask_fast(last * C, 0.1, 3, 4, "cuda", (n - last) * C).view(last, C),
                         ref.drop_scale(0.1), 0.0).double()
    m = f.stream_mix_n4(X, T, y, h, 0.1, 3, 4)["X"]
    ref.check({"X": m[-last:]}, ref.stream_mix(X[-last:], T[-last:], y[-last:], h[-last:], factor))
    grad = f.stream_mix_n4_backward(m, X, T, y, h, 0.1, 3, 4)
    ref.check({k: v[-last:] for k, v in grad.items()},
              ref.stream_mix_backward(m[-last:], X[-last:], T[-last:], y[-last:], h[-last:], factor))


@pytest.mark.skipif(torch.cuda.device_count() < 2, reason="needs two GPUs")
def test_tensors_on_another_device_than_the_current_one():
    g = gen(57)
    X, y = streams(33, 520, g, torch.bfloat16), rows(33, 520, g, torch.bfloat16)
    T, h, seed = mixing(33, g), torch.sigmoid(normal(g, 33, 4)), torch.tensor([5], device="cuda")

    def call(*t):
        X, y, T, h, seed = t
        return [f.layer_norm(y)["y"], f.dropout(y, 0.1, seed)["y"], f.stream_norm_n4(X, h)["y"],
                f.stream_mix_n4(X, T, y, h, 0.1, seed)["X"]]

    here, there = call(X, y, T, h, seed), call(*(t.to("cuda:1") for t in (X, y, T, h, seed)))
    for a, b in zip(here, there):
        assert b.device.index == 1 and same_bits(a, b.to("cuda:0"))


# ---- modules, and a run of them together ---------------------------------------------

def leaf(t):
    return t.detach().clone().requires_grad_(True)


def test_modules_against_the_functions():
    g = gen(60)
    C = 264
    norm = mhc_proj.MHCLayerNorm(C, device="cuda")
    read = mhc_proj.MHCStreamNormN4(C, device="cuda")
    for m in (norm, read):
        with torch.no_grad():
            m.weight.copy_(1 + 0.3 * normal(g, C))
            m.bias.copy_(0.3 * normal(g, C))
    x, X = leaf(normal(g, 3, 5, C).bfloat16()), leaf(normal(g, 3, 5, 4, C).bfloat16())
    h, T, h2 = leaf(torch.sigmoid(normal(g, 3, 5, 4))), leaf(mixing(15, g).view(3, 5, 4, 4)), leaf(torch.rand(3, 5, 4, device="cuda"))
    G, G4 = normal(g, 3, 5, C).bfloat16(), normal(g, 3, 5, 4, C).bfloat16()

    y = norm(x)
    y.backward(G)
    o = f.layer_norm(x.detach().view(-1, C), norm.weight.detach(), norm.bias.detach())
    d = f.layer_norm_backward(G.view(-1, C), x.detach().view(-1, C), o["mean"], o["rstd"], norm.weight.detach(),
                              norm.bias.detach())
    assert y.shape == x.shape and same_bits(y.detach().view(-1, C), o["y"])
    assert same_bits(x.grad.view(-1, C), d["d_x"]) and same_bits(norm.weight.grad, d["d_weight"])
    assert same_bits(norm.bias.grad, d["d_bias"])

    u = read(X, h)
    u.backward(G)
    X3, hh = X.detach().view(-1, 4, C), h.detach().view(-1, 4)
    o = f.stream_norm_n4(X3, hh, read.weight.detach(), read.bias.detach())
    d = f.stream_norm_n4_backward(G.view(-1, C), X3, hh, o["mean"], o["rstd"], read.weight.detach(), read.bias.detach())
    assert u.shape == x.shape and same_bits(u.detach().view(-1, C), o["y"])
    assert same_bits(X.grad.view(-1, 4, C), d["d_X"]) and same_bits(h.grad.view(-1, 4), d["d_h_pre"])

    X.grad = x.grad = None
    mix = mhc_proj.MHCStreamMixN4(p=0.25)
    out = mix(X, T, x, h2, seed=5, offset=2)
    out.backward(G4)
    args = (X3, T.detach().view(-1, 4, 4), x.detach().view(-1, C), h2.detach().view(-1, 4), 0.25, 5, 2)
    d = f.stream_mix_n4_backward(G4.view(-1, 4, C), *args)
    assert same_bits(out.detach().view(-1, 4, C), f.stream_mix_n4(*args)["X"])
    for t, k in ((X, "d_X"), (T, "d_T"), (x, "d_y"), (h2, "d_h_post")):
        assert same_bits(t.grad.reshape(d[k].shape), d[k])

    x.grad = None
    z = mhc_proj.MHCDropout(0.25)(x, seed=torch.tensor([5], device="cuda"), offset=2)
    z.backward(G)
    assert same_bits(z.detach(), f.dropout(x.detach(), 0.25, 5, 2)["y"])
    assert same_bits(x.grad, f.dropout(G, 0.25, 5, 2)["y"])


def test_dropout_seeds_come_from_torch_s_generator():
    x = torch.ones(5000, device="cuda")
    m = mhc_proj.MHCDropout(0.5)
    torch.manual_seed(3)
    a, b = m(x), m(x)
    torch.manual_seed(3)
    assert torch.equal(m(x), a) and torch.equal(m(x), b) and not torch.equal(a, b)
    mix = mhc_proj.MHCStreamMixN4(p=0.5)
    X, T, h = torch.zeros(50, 4, 100, device="cuda"), torch.zeros(50, 4, 4, device="cuda"), torch.ones(50, 4, device="cuda")
    torch.manual_seed(3)
    assert torch.equal(mix(X, T, x.view(50, 100), h)[:, 2].reshape(-1), a)


def test_no_second_derivative():
    """The backward is not differentiable: a second one raises, whether the
    incoming gradient depends on the leaf (square) or not (sum)."""
    x, norm = leaf(normal(gen(61), 4, 8)), mhc_proj.MHCLayerNorm(8, device="cuda")
    for loss, msg in ((lambda y: y.sum(), "does not require grad"), (lambda y: y.square().sum(), "once_differentiable")):
        (g,) = torch.autograd.grad(loss(norm(x)), x, create_graph=True)
        with pytest.raises(RuntimeError, match=msg):
            g.sum().backward()


def layer_forward(X, H, rms, alpha, b, W, modules, seed):
    """One mHC layer: the projection of its residual matrix, the sublayer (a
    product with W) on the normalised read, and the residual update."""
    proj, read, mix = modules
    T = proj(H[..., 8:24], rms, alpha, b)
    h_pre, h_post = torch.sigmoid(H[..., 0:4]), 2 * torch.sigmoid(H[..., 4:8])
    return mix(X, T, read(X, h_pre) @ W, h_post, seed=seed)


def test_one_layer_from_projection_to_update_and_back():
    """The operators as a layer uses them, fp32: the output and every leaf's
    gradient against the same layer in 64 bits with the projection's T taken
    as given (T's own gradient is the projection's, tested on its own) and its
    gradient carried on by the projection's backward.  The layer's sums are
    32-bit sums of up to 4 x 96 terms, each chain below 200 roundings:
    200 * 2^-24 = 1.2e-5 of the terms' sizes, which are below 8 here (streams
    below 5, weights below 2); with the layer's three stages 3e-4 covers it."""
    g = gen(62)
    N, C = 40, 96
    X, H, rms = leaf(normal(g, N, 4, C)), leaf(normal(g, N, 24)), 0.5 + torch.rand(N, device="cuda", generator=g)
    alpha, b = leaf(torch.tensor(0.9, device="cuda")), leaf(normal(g, 16))
    W = leaf(normal(g, C, C) / C ** 0.5)
    modules = (mhc_proj.MHCProjectionN4HRes(), mhc_proj.MHCStreamNormN4(C, device="cuda"), mhc_proj.MHCStreamMixN4(p=0.2))
    tf32 = torch.backends.cuda.matmul.allow_tf32
    torch.backends.cuda.matmul.allow_tf32 = False
    try:
        out = layer_forward(X, H, rms, alpha, b, W, modules, 9)
        G = normal(g, N, 4, C)
        grads = torch.autograd.grad(out, (X, H, W, modules[1].weight, modules[1].bias), G)
    finally:
        torch.backends.cuda.matmul.allow_tf32 = tf32
    T = f.birkhoff_proj_n4_hres(H.detach()[:, 8:24], rms, 0.9, b.detach())["T"]
    X64, H64, W64, T64 = (leaf(t.double()) for t in (X, H, W, T))
    w64, b64 = leaf(modules[1].weight.double()), leaf(modules[1].bias.double())
    u = (torch.sigmoid(H64[:, 0:4])[:, :, None] * X64).sum(1)
    n = torch.nn.functional.layer_norm(u, (C,), w64, b64, 1e-5)
    y = n @ W64 * ref.keep_factor((N, C), 0.2, 9, 0, "cuda")
    out64 = T64 @ X64 + 2 * torch.sigmoid(H64[:, 4:8])[:, :, None] * y[:, None]
    want = list(torch.autograd.grad(out64, (X64, H64, W64, w64, b64, T64), G.double()))
    dT = want.pop()
    want[1][:, 8:24] += f.birkhoff_proj_n4_hres_backward(dT.float(), T, H.detach()[:, 8:24], rms, 0.9)["d_h_res"].double()
    assert (out.double() - out64).abs().max().item() < 3e-4
    for a, w, name in zip(grads, want, ("X", "H", "W", "weight", "bias")):
        assert (a.double() - w).abs().max().item() <= 3e-4 * max(1.0, w.abs().max().item()), name


def test_a_training_step_captured_and_replayed():
    """Forward and backward of two layers in one graph, with the masks drawn
    from torch's generator inside it: replays with the generator at the same
    state give the same gradients."""
    g = gen(63)
    N, C = 64, 136
    X, H, rms = leaf(normal(g, N, 4, C)), leaf(normal(g, N, 24)), 0.5 + torch.rand(N, device="cuda", generator=g)
    alpha, b, W = torch.tensor(0.9, device="cuda"), normal(g, 16), leaf(normal(g, C, C) / C ** 0.5)
    modules = (mhc_proj.MHCProjectionN4HRes(), mhc_proj.MHCStreamNormN4(C, device="cuda"), mhc_proj.MHCStreamMixN4(p=0.2))
    leaves = (X, H, W, modules[1].weight)

    def step():
        out = layer_forward(layer_forward(X, H, rms, alpha, b, W, modules, None), H, rms, alpha, b, W, modules, None)
        return torch.autograd.grad(out.square().mean(), leaves)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for _ in range(2):
            step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured = step()
    seen = []
    for _ in range(2):
        torch.manual_seed(17)
        graph.replay()
        seen.append([t.clone() for t in captured])
    graph.replay()  # the generator has moved on: other masks
    torch.cuda.synchronize()
    assert all(same_bits(a, c) for a, c in zip(*seen))
    assert not same_bits(captured[0], seen[0][0])
    torch.manual_seed(17)
    eager = step()
    assert all(same_bits(a, c) for a, c in zip(eager, seen[0]))
