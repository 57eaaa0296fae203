"""Arguments that the row operators' Python functions refuse as a ValueError before
anything reaches a GPU."""
import pytest
import torch

import hierarchicalkv_b200 as hkv


def order(tokens=4, top_k=2, experts=3):
    return hkv.ExpertOrder(torch.zeros(experts + 1, dtype=torch.int32),
                           torch.zeros((tokens, top_k), dtype=torch.int32),
                           torch.zeros(tokens * top_k, dtype=torch.int32))


def test_the_gradient_of_combine_needs_weights(product_lib):
    with pytest.raises(ValueError, match="weights"):
        hkv.expert_combine_backward(torch.zeros((4, 8)), torch.zeros((8, 8)), None, order())
