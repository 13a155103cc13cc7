"""Arrays that start between two of their elements are refused by the residual
path's C entries: a load from there would be a fault.  (The addresses are
never dereferenced; each call differs from one with aligned arrays in one of them.)"""
import pytest

from mhc_proj import capi

A = 256  # an aligned address
BF, F32 = capi.MHC_DTYPE_BF16, capi.MHC_DTYPE_F32
WS = 1 << 20

# arguments by position, {position: elements' bytes} of the arrays among them
CALLS = [
    (capi.layer_norm, [A, 8, BF, A, A, F32, A, A, A, 1e-5, 2, 8], {0: 2, 3: 4, 4: 4, 6: 2, 7: 4, 8: 4}),
    (capi.layer_norm_backward, [A, 8, A, 8, F32, A, A, A, BF, A, A, A, 2, 8, A, WS],
     {0: 4, 2: 4, 5: 4, 6: 4, 7: 2, 9: 4, 10: 2, 11: 2, 14: 4}),
    (capi.dropout, [A, A, BF, 4, 0.1, 0, A], {0: 2, 1: 2, 6: 8}),
    (capi.stream_norm_n4, [A, 32, 8, BF, A, F32, A, A, BF, A, A, A, 1e-5, 2, 8],
     {0: 2, 4: 4, 6: 2, 7: 2, 9: 2, 10: 4, 11: 4}),
    (capi.stream_norm_n4_backward, [A, 8, A, 32, 8, BF, A, F32, A, A, A, F32, A, A, A, A, 2, 8, A, WS],
     {0: 2, 2: 2, 6: 4, 8: 4, 9: 4, 10: 4, 12: 2, 13: 4, 14: 4, 15: 4, 18: 4}),
    (capi.stream_mix_n4, [A, 32, 8, A, 8, BF, A, F32, A, BF, A, 0.1, 0, A, 0, 2, 8],
     {0: 2, 3: 2, 6: 4, 8: 2, 10: 2, 13: 8}),
    (capi.stream_mix_n4_backward, [A, 32, 8, A, 32, 8, A, 8, F32, A, BF, A, F32, A, A, A, A, 0.1, 0, A, 0, 2, 8],
     {0: 4, 3: 4, 6: 4, 9: 2, 11: 4, 13: 4, 14: 2, 15: 4, 16: 4, 19: 8}),
]


@pytest.mark.parametrize("fn,args,at,size", [(fn, args, i, n) for fn, args, where in CALLS for i, n in where.items()])
def test_arrays_between_elements_are_refused(fn, args, at, size):
    for off in {1, size // 2}:
        bad = list(args)
        bad[at] += off
        with pytest.raises(capi.MhcError) as e:
            fn(*bad)
        assert e.value.code == capi.MHC_ERR_INVALID_VALUE


def test_a_count_near_2_63_is_refused():
    for count in (1 << 62, (1 << 63) - 1):
        for dtype in (F32, BF):
            with pytest.raises(capi.MhcError) as e:
                capi.dropout(A, A, dtype, count, 0.1, 0)
            assert e.value.code == capi.MHC_ERR_INVALID_VALUE
