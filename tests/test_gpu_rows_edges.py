"""GPU: the row operators where their arithmetic ends, against oracle/rows.py in float64.  The tolerances are those of test_gpu_rows.py."""
import math

import pytest
import torch

from oracle import rows as orow
from test_gpu_rows import cuda, host, rows_of

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
