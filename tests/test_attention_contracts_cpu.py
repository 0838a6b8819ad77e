"""What attention refuses whatever else its call asks for."""

import pytest
import torch

from peco_b200.attention import attention, attention_backward

Q = torch.zeros(2, 4, 6, 64, dtype=torch.bfloat16)
K = torch.zeros(2, 2, 9, 64, dtype=torch.bfloat16)
LSE = torch.zeros(2, 4, 6)


@pytest.mark.parametrize("wants", ["", "q", "k", "v", "qkv"])
def test_a_gradient_of_slopes_is_refused(wants):
    """Also where the call is recorded for the other gradients: it would give none for slopes without a word."""
    slopes = torch.zeros(4, requires_grad=True)
    q, k, v = (t.clone().requires_grad_(name in wants) for name, t in zip("qkv", (Q, K, K)))
    with pytest.raises(RuntimeError, match="gradient of slopes"):
        attention(q, k, v, slopes=slopes)
    with pytest.raises(RuntimeError, match="gradient of slopes"):
        attention_backward(Q, q, k, v, Q, LSE, slopes=slopes)
    with torch.no_grad(), pytest.raises(RuntimeError, match="CUDA"):
        attention(q, k, v, slopes=slopes)
    with pytest.raises(RuntimeError, match="CUDA"):
        attention(q, k, v, slopes=slopes.detach())
