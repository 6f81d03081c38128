"""The state space operators and sampling at their edges: what is not finite, types that differ, buffers that autograd holds, sizes past a grid's
threads, and the kernels' many-row, many-token and many-sequence forms.  Oracle and tolerances as in test_gpu_ssm.py unless a test says otherwise."""
import math

import pytest
import torch

from oracle import ssm as O
from tests import test_gpu_ssm as S
from tests.util import assert_close

pytestmark = pytest.mark.gpu
RTOL = S.RTOL


@pytest.mark.parametrize("weights", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("times", [1, 8, 22, 74])
@pytest.mark.parametrize("thousandths", [3, 7, 13])
def test_rows_in_8_bits_round_once(weights, times, thousandths):
    """y / scale where it lies in the middle of two values of 8 bits: a row of ones, so that y is the weight, of every such middle times the scale.  The
    quotient in fp32 is exact, the one rounding goes to even."""
    from rwkv_wkv_hip import ssm as K
    steps = [(1 + m / 8) * 2.0 ** e for e in range(-6, 9) for m in range(8) if (1 + m / 8) * 2.0 ** e <= 448]
    middles = torch.tensor([(a + b) / 2 for a, b in zip(steps, steps[1:])] + [448.0], dtype=torch.float64).repeat(times)
    weight = (middles * (thousandths / 1024)).to(weights)
    assert weights == torch.bfloat16 or torch.equal(weight.double(), middles * (thousandths / 1024))
    q, scale, _ = K.rms_norm_fp8(torch.ones(3, len(weight), dtype=torch.bfloat16, device="cuda"), weight.cuda(), eps=0.0)
    want = weight.float().abs().max() / 448
    assert (scale.cpu() == want).all()
    assert torch.equal(q.cpu().view(torch.uint8), (weight.float() / want).to(torch.float8_e4m3fn).view(torch.uint8).expand(3, -1))
