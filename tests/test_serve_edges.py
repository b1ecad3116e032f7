"""The serving operators where values, flags or sizes are unusual.

Bounds are those of test_serve_ops.py, derived there from the kernels' roundings.
"""
import math

import pytest
import torch

from tests.test_serve_ops import check_logprobs, randn

gpu = pytest.mark.gpu


@pytest.fixture(scope="module")
def f(cuda_device):
    import fp8gq
    fp8gq.device_error(clear=True)
    yield fp8gq
    torch.cuda.synchronize()
    assert fp8gq.device_error(clear=True) == 0


# --------------------------------------------------------------- logprobs --
@gpu
@pytest.mark.parametrize("t, v", [(6, 777), (6, 50257), (1, 151936)])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_logprobs_lowest_values_beside_ordinary_ones(f, dtype, t, v):
    """A mask of the type's lowest value is a finite logit: its log probability is
    the logit less the row's sum, not -inf."""
    low = torch.finfo(dtype).min
    x = randn(v, t, v, scale=3.0)
    masked = torch.rand(t, v, generator=torch.Generator("cuda").manual_seed(v), device="cuda") < 0.7
    x = x.masked_fill(masked, low).to(dtype)
    x[0, 5:] = low                                        # five left: the alternatives reach the masked
    x[0, :5] = torch.arange(5, device="cuda").to(dtype)
    tokens = masked.int().argmax(1)                       # of each row a masked one
    tokens[0] = v - 1
    if t > 3:
        x[2, 9], tokens[2] = -2.4e38, 9                   # x log2(e) leaves fp32, x does not
        x[3, 11] = -math.inf
    r = check_logprobs(f, x, tokens, 20)
    assert r.logprobs.isfinite().all() and r.top_logprobs[0].isfinite().all()
