"""Refusals of the layer operators' wrappers that need no GPU."""
import pytest
import torch

import a11spec


@pytest.mark.parametrize("x", [None, [1.0], 3])
def test_check_status_refuses_as_the_plain_call(x):
    """The status word's workspace is made only for tensors: the refusal stays an A11Error."""
    t = torch.zeros(4, 64, dtype=torch.bfloat16)
    with pytest.raises(a11spec.A11Error, match="tensor"):
        a11spec.linear(x, t, check_status=True)
    with pytest.raises(a11spec.A11Error, match="tensor"):
        a11spec.chunk_attention(x, t, t, t, t, check_status=True)
