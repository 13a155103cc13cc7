"""The residual path without a GPU: the draws against the generator's published
vectors, the 64-bit reference's gradients against differences, and what the
functions, modules and C ABI refuse."""
import inspect

import pytest
import torch

import mhc_proj
import residual_reference as ref
from mhc_proj import capi

f = mhc_proj.torch
FAKE = 256  # a non-null address that is never dereferenced by these calls


# ---- the generator ---------------------------------------------------------------

@pytest.mark.parametrize("counter,key,words", [
    # the known answers published with the generator (Random123, philox4x32 10)
    ((0, 0, 0, 0), (0, 0), (0x6627e8d5, 0xe169c58d, 0xbc57ac4c, 0x9b00dbd8)),
    ((0xffffffff,) * 4, (0xffffffff,) * 2, (0x408f276d, 0x41c83b0e, 0xa20bc7c6, 0x6d5451fd)),
    ((0x243f6a88, 0x85a308d3, 0x13198a2e, 0x03707344), (0xa4093822, 0x299f31d0),
     (0xd16cfe09, 0x94fdcceb, 0x5001e420, 0x24126ea1)),
])
def test_philox_known_answers(counter, key, words):
    assert tuple(ref.philox(counter, key)) == words


def test_vectorised_draws_are_the_generator_s():
    for seed, offset, first in ((0, 0, 0), (-1, 5, 3), (2 ** 62 + 12345, 2 ** 40 + 7, 2 ** 35 - 9)):
        a = ref.keep_mask(101, 0.3, seed, offset, first)
        b = ref.keep_mask_fast(101, 0.3, seed, offset, "cpu", first)
        assert torch.equal(a, b)


def test_share_of_kept_elements():
    n = 1 << 18
    for p in (0.1, 0.5, 0.9):
        kept = ref.keep_mask_fast(n, p, 42, 1, "cpu").double().mean().item()
        assert abs(kept - (1 - p)) < 5 * (p * (1 - p) / n) ** 0.5 + 2 ** -16


# ---- the reference's gradients against differences ----------------------------------

def _directional(fn, grads, inputs, seed):
    """sum(grad . v) against the central difference of fn along v, in 64 bits.
    Step 1e-5: truncation and rounding are both below 1e-9 of the values here."""
    g = torch.Generator().manual_seed(seed)
    for name, x in inputs.items():
        v = torch.randn(x.shape, generator=g, dtype=torch.float64)
        h = 1e-5
        hi, lo = fn(**{**inputs, name: x + h * v}), fn(**{**inputs, name: x - h * v})
        want = ((hi - lo) / (2 * h)).item()
        got = (grads[name] * v).sum().item()
        assert abs(got - want) <= 1e-7 * max(1.0, abs(want)), (name, got, want)


def _rand(*shape, seed=0):
    return torch.randn(*shape, generator=torch.Generator().manual_seed(seed), dtype=torch.float64)


@pytest.mark.parametrize("N,C", [(1, 2), (5, 17)])
def test_norm_gradients_against_differences(N, C):
    x, w, b, G = _rand(N, C, seed=1), _rand(C, seed=2), _rand(C, seed=3), _rand(N, C, seed=4)

    def loss(x, w, b):
        return (ref.layer_norm(x, w, b, 1e-5)["y"][0] * G).sum()

    fwd = ref.layer_norm(x, w, b, 1e-5)
    bwd = ref.layer_norm_backward(G, x, fwd["mean"][0], fwd["rstd"][0], w, b)
    _directional(loss, {"x": bwd["d_x"][0], "w": bwd["d_weight"][0], "b": bwd["d_bias"][0]}, dict(x=x, w=w, b=b), 5)


def test_stream_norm_gradients_against_differences():
    N, C = 4, 13
    X, h, w, b, G = _rand(N, 4, C, seed=1), _rand(N, 4, seed=2), _rand(C, seed=3), _rand(C, seed=4), _rand(N, C, seed=5)

    def loss(X, h, w, b):
        return (ref.stream_norm(X, h, w, b, 1e-5)["y"][0] * G).sum()

    fwd = ref.stream_norm(X, h, w, b, 1e-5)
    bwd = ref.stream_norm_backward(G, X, h, fwd["mean"][0], fwd["rstd"][0], w, b)
    _directional(loss, {"X": bwd["d_X"][0], "h": bwd["d_h_pre"][0], "w": bwd["d_weight"][0], "b": bwd["d_bias"][0]},
                 dict(X=X, h=h, w=w, b=b), 6)


@pytest.mark.parametrize("p", [0.0, 0.25])
def test_mix_gradients_against_differences(p):
    N, C = 4, 13
    X, T, y, h, G = (_rand(N, 4, C, seed=1), _rand(N, 4, 4, seed=2), _rand(N, C, seed=3), _rand(N, 4, seed=4),
                     _rand(N, 4, C, seed=5))
    factor = ref.keep_factor((N, C), p, 11, 2, "cpu")

    def loss(X, T, y, h):
        return (ref.stream_mix(X, T, y, h, factor)["X"][0] * G).sum()

    bwd = ref.stream_mix_backward(G, X, T, y, h, factor)
    _directional(loss, {"X": bwd["d_X"][0], "T": bwd["d_T"][0], "y": bwd["d_y"][0], "h": bwd["d_h_post"][0]},
                 dict(X=X, T=T, y=y, h=h), 7)


# ---- refusals: functions ------------------------------------------------------------

z = torch.zeros


def test_signatures():
    assert "eps: typing.SupportsFloat = 1e-05" in f.layer_norm.__doc__
    for name, args in (("dropout", ("x", "p", "seed", "offset")), ("stream_mix_n4", ("X", "T", "y", "h_post", "p")),
                       ("stream_norm_n4_backward", ("G", "X", "h_pre", "mean", "rstd"))):
        doc = getattr(f, name).__doc__
        assert all(a + ":" in doc for a in args), doc


@pytest.mark.parametrize("call,msg", [
    (lambda: f.layer_norm(z(3)), "x must be"),
    (lambda: f.layer_norm(z(2, 0)), "x must be"),
    (lambda: f.layer_norm(z(2, 3, 4)), "x must be"),
    (lambda: f.layer_norm(z(2, 3), z(4)), "weight must be"),
    (lambda: f.layer_norm(z(2, 3), z(3), z(1, 3)), "bias must be"),
    (lambda: f.layer_norm(z(2, 3, dtype=torch.int32)), "floating-point"),
    (lambda: f.layer_norm_backward(z(2, 4), z(2, 3), z(2), z(2)), "G must be"),
    (lambda: f.layer_norm_backward(z(2, 3), z(2, 3), z(3), z(2)), "mean must be"),
    (lambda: f.layer_norm_backward(z(2, 3), z(2, 3), z(2), z(2, 1)), "rstd must be"),
    (lambda: f.dropout(z(2, 3, dtype=torch.int64), 0.1, 0), "floating-point"),
    (lambda: f.dropout(z(2, 3), 0.1, 0.5), "seed must be"),
    (lambda: f.dropout(z(2, 3), 0.1, torch.zeros(1)), "seed must be"),
    (lambda: f.dropout(z(2, 3), 0.1, torch.zeros(2, dtype=torch.int64)), "seed must be"),
    (lambda: f.stream_norm_n4(z(2, 3, 8), z(2, 4)), "X must be"),
    (lambda: f.stream_norm_n4(z(2, 4, 0), z(2, 4)), "X must be"),
    (lambda: f.stream_norm_n4(z(2, 4, 8), z(2, 3)), "h_pre must be"),
    (lambda: f.stream_norm_n4(z(2, 4, 8), z(2, 4), z(7)), "weight must be"),
    (lambda: f.stream_norm_n4_backward(z(2, 7), z(2, 4, 8), z(2, 4), z(2), z(2)), "G must be"),
    (lambda: f.stream_mix_n4(z(2, 4), z(2, 4, 4), z(2, 8), z(2, 4)), "X must be"),
    (lambda: f.stream_mix_n4(z(2, 4, 8), z(2, 16), z(2, 8), z(2, 4)), "T must be"),
    (lambda: f.stream_mix_n4(z(2, 4, 8), z(2, 4, 4), z(2, 9), z(2, 4)), "y must be"),
    (lambda: f.stream_mix_n4(z(2, 4, 8), z(2, 4, 4), z(2, 8), z(3, 4)), "h_post must be"),
    (lambda: f.stream_mix_n4_backward(z(2, 4, 9), z(2, 4, 8), z(2, 4, 4), z(2, 8), z(2, 4)), "G must be"),
])
def test_functions_refuse_shapes_and_types(call, msg):
    with pytest.raises(RuntimeError, match=msg):
        call()


@pytest.mark.parametrize("call", [
    lambda: f.layer_norm(z(2, 3), eps=-1.0),
    lambda: f.layer_norm(z(2, 3), eps=float("nan")),
    lambda: f.stream_norm_n4(z(2, 4, 8), z(2, 4), eps=-1.0),
    lambda: f.dropout(z(2, 3), -0.1, 0),
    lambda: f.dropout(z(2, 3), 1.1, 0),
    lambda: f.dropout_backward(z(2, 3), float("nan"), 0),
    lambda: f.stream_mix_n4(z(2, 4, 8), z(2, 4, 4), z(2, 8), z(2, 4), p=2.0),
    lambda: f.stream_mix_n4_backward(z(2, 4, 8), z(2, 4, 8), z(2, 4, 4), z(2, 8), z(2, 4), p=-1.0),
])
def test_functions_refuse_numbers(call):
    with pytest.raises(ValueError):
        call()


# ---- refusals: modules -----------------------------------------------------------

def test_module_defaults():
    assert inspect.signature(mhc_proj.MHCLayerNorm).parameters["eps"].default == 1e-5
    assert mhc_proj.MHCDropout().p == 0.5 and mhc_proj.MHCStreamMixN4().p == 0.0
    m = mhc_proj.MHCStreamNormN4(8, bias=False)
    assert m.weight.shape == (8,) and m.bias is None
    assert [p for p in mhc_proj.MHCLayerNorm(8, affine=False).parameters()] == []


def test_dropout_module_is_the_identity_in_eval_mode():
    x = torch.randn(3, 5)
    assert mhc_proj.MHCDropout(0.3).eval()(x) is x
    assert mhc_proj.MHCDropout(0.0)(x) is x


@pytest.mark.parametrize("call", [
    lambda: mhc_proj.MHCLayerNorm(8)(z(2, 7)),
    lambda: mhc_proj.MHCLayerNorm(0),
    lambda: mhc_proj.MHCStreamNormN4(8)(z(2, 4, 7), z(2, 4)),
    lambda: mhc_proj.MHCStreamNormN4(8)(z(2, 3, 8), z(2, 3)),
    lambda: mhc_proj.MHCStreamNormN4(8)(z(2, 4, 8), z(4, 2)),
    lambda: mhc_proj.MHCStreamMixN4()(z(2, 4, 8), z(2, 4), z(2, 8), z(2, 4)),
    lambda: mhc_proj.MHCStreamMixN4()(z(2, 4, 8), z(2, 4, 4), z(8), z(2, 4)),
    lambda: mhc_proj.MHCStreamMixN4()(z(2, 4, 8), z(2, 4, 4), z(2, 8), z(4)),
    lambda: mhc_proj.MHCDropout(1.5),
    lambda: mhc_proj.MHCStreamMixN4(p=-0.5),
])
def test_modules_refuse(call):
    with pytest.raises(ValueError):
        call()


# ---- refusals: C ABI ---------------------------------------------------------------

F = FAKE


@pytest.mark.parametrize("fn,args", [
    (capi.layer_norm, (F, 8, 0, F, F, 0, F, F, F, 1e-5, -1, 8)),
    (capi.layer_norm, (F, 8, 0, F, F, 0, F, F, F, 1e-5, 2, 0)),
    (capi.layer_norm, (F, -8, 0, F, F, 0, F, F, F, 1e-5, 2, 8)),
    (capi.layer_norm, (F, 8, 3, F, F, 0, F, F, F, 1e-5, 2, 8)),
    (capi.layer_norm, (F, 8, 0, F, F, -1, F, F, F, 1e-5, 2, 8)),
    (capi.layer_norm, (0, 8, 0, F, F, 0, F, F, F, 1e-5, 2, 8)),
    (capi.layer_norm, (F, 8, 0, F, F, 0, 0, F, F, 1e-5, 2, 8)),
    (capi.layer_norm, (F, 8, 0, F, F, 0, F, F, F, -1e-5, 2, 8)),
    (capi.layer_norm, (F, 8, 0, F, F, 0, F, F, F, float("nan"), 2, 8)),
    (capi.layer_norm_backward_workspace, (-1, 8)),
    (capi.layer_norm_backward_workspace, (2, 0)),
    (capi.layer_norm_backward, (F, 8, F, 8, 0, F, F, F, 0, F, F, F, 2, 8, 0, 1 << 20)),
    (capi.layer_norm_backward, (F, 8, F, 8, 0, F, F, F, 0, F, F, F, 2, 8, F, 4)),
    (capi.layer_norm_backward, (F, 8, F, 8, 0, 0, F, F, 0, F, F, F, 2, 8, F, 1 << 20)),
    (capi.layer_norm_backward, (F, -8, F, 8, 0, F, F, F, 0, F, F, F, 2, 8, F, 1 << 20)),
    (capi.dropout, (F, F, 0, -1, 0.1, 0)),
    (capi.dropout, (F, F, 0, 4, 1.1, 0)),
    (capi.dropout, (F, F, 0, 4, float("nan"), 0)),
    (capi.dropout, (F, F, 5, 4, 0.1, 0)),
    (capi.dropout, (F, 0, 0, 4, 0.1, 0)),
    (capi.stream_norm_n4, (F, 32, 8, 0, 0, 0, F, F, 0, F, F, F, 1e-5, 2, 8)),
    (capi.stream_norm_n4, (F, 32, -8, 0, F, 0, F, F, 0, F, F, F, 1e-5, 2, 8)),
    (capi.stream_norm_n4, (F, 32, 8, 0, F, 4, F, F, 0, F, F, F, 1e-5, 2, 8)),
    (capi.stream_norm_n4_backward, (F, 8, F, 32, 8, 0, F, 0, F, F, F, 0, F, 0, F, F, 2, 8, F, 1 << 20)),
    (capi.stream_norm_n4_backward_workspace, (2, -4)),
    (capi.stream_mix_n4, (F, 32, 8, F, 8, 0, F, 0, F, 0, F, -0.1, 0, 0, 0, 2, 8)),
    (capi.stream_mix_n4, (F, 32, 8, F, -8, 0, F, 0, F, 0, F, 0.1, 0, 0, 0, 2, 8)),
    (capi.stream_mix_n4, (F, 32, 8, F, 8, 0, F, 7, F, 0, F, 0.1, 0, 0, 0, 2, 8)),
    (capi.stream_mix_n4, (F, 32, 8, F, 8, 0, F, 0, 0, 0, F, 0.1, 0, 0, 0, 2, 8)),
    (capi.stream_mix_n4, (F, 32, 8, F, 8, 0, F, 0, F, 0, F, 0.1, 0, 0, 0, 2, 0)),
    (capi.stream_mix_n4_backward, (F, -32, 8, F, 32, 8, F, 8, 0, F, 0, F, 0, F, F, F, F, 0.1, 0, 0, 0, 2, 8)),
    (capi.stream_mix_n4_backward, (F, 32, 8, F, 32, 8, F, 8, 0, F, 0, F, 0, F, F, 0, F, 0.1, 0, 0, 0, 2, 8)),
])
def test_c_abi_refuses(fn, args):
    with pytest.raises(capi.MhcError) as e:
        fn(*args)
    assert e.value.code == capi.MHC_ERR_INVALID_VALUE


def test_empty_batches_launch_nothing():
    capi.layer_norm(0, 8, 0, 0, 0, 0, 0, 0, 0, 1e-5, 0, 8)
    capi.layer_norm_backward(0, 8, 0, 8, 0, 0, 0, 0, 0, 0, 0, 0, 0, 8, 0, 0)
    capi.dropout(0, 0, 1, 0, 0.1, 0)
    capi.stream_norm_n4(0, 32, 8, 0, 0, 0, 0, 0, 0, 0, 0, 0, 1e-5, 0, 8)
    capi.stream_norm_n4_backward(0, 8, 0, 32, 8, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 8, 0, 0)
    capi.stream_mix_n4(0, 32, 8, 0, 8, 0, 0, 0, 0, 0, 0, 0.1, 0, 0, 0, 0, 8)
    capi.stream_mix_n4_backward(0, 32, 8, 0, 32, 8, 0, 8, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0.1, 0, 0, 0, 0, 8)
