"""GPU: the sequence operators where values or offsets are extreme, and where autograd has to be told: against plain statements in 64 bits."""
import math

import pytest
import torch

import _sequence_ref as R

pytestmark = pytest.mark.gpu

DT = [torch.float32, torch.bfloat16]


def _att():
    from trajectorydiffusion_amd import attention
    return attention


def _normal(*shape, dtype=torch.float32, seed=0):
    return torch.randn(*shape, generator=torch.Generator().manual_seed(seed)).to(dtype)


# ---- what autograd is told --------------------------------------------------------------------------------------------------------------
def test_a_key_that_attention_kept_may_not_be_rotated_before_the_backward_pass():
    A = _att()
    q, k, v = (_normal(1, 20, 2, 32, seed=n).cuda() for n in range(3))
    pos = torch.arange(20.0, device="cuda")[:, None]
    q.requires_grad_()
    out = A.window_attention(q, k, v, 5, 0, 1)
    A.rotary_axes(k, pos, (16,), out=k)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        out.sum().backward()
