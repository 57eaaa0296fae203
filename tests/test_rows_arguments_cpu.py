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


def test_views_whose_memory_holds_other_values_are_refused(product_lib):
    """A conjugate view, and the imaginary part of one, share the memory of what they were
    taken from, and the operators read memory."""
    z = torch.complex(torch.ones(4, 1), torch.ones(4, 1)).conj()
    with pytest.raises(ValueError, match="resolve_conj"):
        hkv.expert_dispatch(z, order())
    assert z.imag.is_neg()
    for call in (lambda x: hkv.expert_dispatch(x, order()), hkv.layer_norm,
                 lambda x: hkv.expert_dispatch_backward(x, order(2)),
                 lambda x: hkv.expert_combine(x, torch.ones((2, 2)), order(2))):
        with pytest.raises(ValueError, match="resolve_neg"):
            call(z.imag)
