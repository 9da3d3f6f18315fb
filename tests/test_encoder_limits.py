"""The encoder operators' limits of size are refused by name, before any launch."""
import pytest
import torch

import d2p_b200 as d2p


@pytest.mark.parametrize("shape", [(65536, 1, 1, 8), (1, 1, 65536, 8)])
def test_attention_names_its_limits(shape):
    q = torch.zeros(shape, dtype=torch.bfloat16)
    with pytest.raises(ValueError, match="at most 65535 problems and heads"):
        d2p.attention(q, q, q)
