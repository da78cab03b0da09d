"""The readout's CPU oracle at rows of any offset, where a logsumexp that is rounded to 64 bits would swallow log(sum)."""
import math

import pytest
import torch

from oracle import readout as OR


@pytest.mark.parametrize("offset", [0.0, -1e9, 1e20, -1e30, torch.finfo(torch.float32).min])
def test_rows_of_one_value(offset):
    """log p = -log V, entropy log V, and a logsumexp's gradient of 1 / V each."""
    x = torch.full((2, 48), offset)
    t = torch.tensor([[0, 47], [5, -1]])
    lp, lse, ent, top, ids = OR.token_logprobs(x, t, 3)
    assert torch.allclose(lp, torch.where(t < 0, 0.0, -math.log(48)).double(), atol=1e-12) and torch.allclose(top, torch.full_like(top, -math.log(48)), atol=1e-12)
    assert torch.allclose(ent, torch.full_like(ent, math.log(48)), atol=1e-12) and ids.tolist() == [[0, 1, 2]] * 2
    assert torch.allclose(lse, x[:, 0].double() + math.log(48), rtol=1e-15)  # (the offset as fp32 has it)
    grad = OR.gradient(x, t, g_lse=torch.ones(2))
    assert torch.allclose(grad, torch.full_like(grad, 1 / 48), atol=1e-15)


@pytest.mark.parametrize("offset", [1024.0, -(2.0 ** 30)])
def test_offsets_change_nothing(offset):
    g = torch.Generator().manual_seed(0)
    x = torch.randint(-64, 64, (3, 30), generator=g) / 8.0  # exact at either offset
    t = torch.randint(0, 30, (3, 2), generator=g)
    w = [torch.randn(s, generator=g) for s in ((3, 2), (3,), (3,))]
    a, b = (OR.token_logprobs(y, t, 4) for y in (x.double(), x.double() + offset))
    assert torch.equal(a[0], b[0]) and torch.equal(a[2], b[2]) and torch.equal(a[3], b[3]) and torch.equal(a[4], b[4])
    assert torch.equal(OR.gradient(x.double(), t, None, *w), OR.gradient(x.double() + offset, t, None, *w))
    assert torch.allclose(a[0], torch.log_softmax(x.double(), 1).gather(1, t), atol=1e-13)
