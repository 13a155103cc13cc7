"""What dropout refuses as a seed before it looks for a GPU."""
import numpy
import pytest
import torch

import mhc_proj

f = mhc_proj.torch
x = torch.zeros(2, 4)


@pytest.mark.parametrize("seed", [2 ** 64, -2 ** 63 - 1, 10 ** 30])
@pytest.mark.parametrize("call", [
    lambda s: f.dropout(x, 0.1, s),
    lambda s: f.dropout_backward(x, 0.1, s),
    lambda s: f.stream_mix_n4(torch.zeros(2, 4, 4), torch.zeros(2, 4, 4), x, x, 0.1, s),
    lambda s: mhc_proj.MHCDropout(0.1)(x, seed=s),
])
def test_seeds_of_more_than_64_bits_are_refused(call, seed):
    with pytest.raises(ValueError, match="seed must be between"):
        call(seed)


@pytest.mark.parametrize("seed", [0.5, "7", numpy.float64(1), numpy.zeros(2, dtype=numpy.int64), torch.zeros(1),
                                  torch.zeros(2, dtype=torch.int64)])
def test_seeds_that_are_no_whole_number_are_refused(seed):
    with pytest.raises(RuntimeError, match="seed must be a whole number"):
        f.dropout(x, 0.1, seed)
