"""GPU: the row operators where their arithmetic ends, against oracle/rows.py in float64.  The tolerances are those of test_gpu_rows.py."""
import math

import numpy as np
import pytest
import torch

from oracle import rows as orow
from test_gpu_rows import U, check_drawn, cuda, host, rows_of

pytestmark = pytest.mark.gpu
TYPES = [torch.float32, torch.bfloat16, torch.float16]


# ------------------------------------------------------------------------------------------------ drawing
@pytest.mark.parametrize("dtype,V", [(torch.float32, 48), (torch.float32, 1000), (torch.float32, 9000), (torch.bfloat16, 9000), (torch.bfloat16, 70000), (torch.float16, 70000)])
@pytest.mark.parametrize("k", [0, 600])
def test_a_row_s_top_p_of_nothing_keeps_the_first_token(dtype, V, k):
    """Flat rows: more tokens of one value than a bin's list (fp32) or a counter (16 bits, 70,000 tokens) holds."""
    from mucon_amd import ops

    x = rows_of("flat", 4, V, dtype, 1)
    x[1] = rows_of("normal", 1, V, dtype, 2)[0]
    x[2, V // 2] = 1.5
    x[3, :7] = -math.inf
    p = torch.tensor([0.0, -1.0, -math.inf, 0.0])
    u = torch.tensor([0.0, 0.5, 0.999, 0.7])
    for T in (1.0, 50.0):
        for m in (0.0, 0.5):
            token, logp = ops.sample_logits(*cuda(x, u), T, k, p.cuda(), m)
            assert token.tolist() == [int(orow.order(r)[0]) for r in host(x)]
            assert logp.tolist() == [0.0] * 4


@pytest.mark.parametrize("dtype,V", [(torch.float32, 9000), (torch.float32, 4097), (torch.bfloat16, 9000), (torch.bfloat16, 200000)])
@pytest.mark.parametrize("T", [1e30, 1.1e37, 3e37, 3.4e38, math.inf])
@pytest.mark.parametrize("k", [600, 5000, 0])
def test_draws_at_temperatures_near_the_end_of_fp32(dtype, V, T, k):
    """Few tokens above -inf, fewer than top_k; all of them are alike at these temperatures: weights within 2^-90 of 1.  (70,000 and more tokens of one 16-bit value
    run over its counter: -inf is counted apart, so the last size has that many finite ones.)"""
    from mucon_amd import ops

    x = torch.full((5, V), -math.inf)
    g = torch.Generator().manual_seed(3)
    for r, n in enumerate((20, 1, 599, 600, 601)):
        x[r, torch.randperm(V, generator=g)[:n]] = torch.randn(n, generator=g)
    if V > 65536:
        x[4, 1000:80000] = 0.5
    x = x.to(dtype)
    u = torch.tensor([0.6, 0.9, 0.999, 0.37, 0.99])
    token, logp = ops.sample_logits(*cuda(x, u), torch.full((5,), T).cuda(), k)
    for r in range(5):
        finite = int((x[r] > -math.inf).sum())
        n = min(finite, k) if k else finite
        at = min(int(np.float64(u[r]) * n), n - 1)      # the sums are whole numbers: the first above u n
        assert int(token[r]) == int(orow.order(host(x)[r])[at]), (r, n)
        assert abs(float(logp[r]) + math.log(n)) <= U * math.log(n) + 1e-11


def test_draws_of_logits_at_the_end_of_fp32():
    """A bin's borders in the row's units overflow where the logits themselves are near the largest of fp32."""
    from mucon_amd import ops

    V = 9000
    x = torch.full((3, V), -3.0e38)
    x[0, 17], x[0, 5] = 3.0e38, 2.9e38
    x[1, ::2] = 3.0e38
    x[2, 8000:] = 1.0e38
    u = torch.tensor([0.6, 0.9, 0.5])
    for T in (1e36, 3e37, 3e38):
        for k, p in ((0, 1.0), (600, 1.0), (0, 0.9), (5000, 0.9)):
            token, logp = ops.sample_logits(*cuda(x, u), torch.full((3,), T).cuda(), k, p)
            check_drawn(token.cpu(), logp.cpu(), host(x), u, (np.float32(T).item(), k, np.float32(p).item(), 0.0))
