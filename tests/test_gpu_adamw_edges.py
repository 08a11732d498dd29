"""ops.TensorSet and ops.adamw_step at the edges of what they take: state buffers that are not aligned."""
import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu

U = 2.0 ** -24


@pytest.fixture(scope="module")
def ops():
    from discrete_dppm_graphs_amd import ops
    return ops


def shifted(t, by):
    """the same values, `by` of them behind an aligned address"""
    return torch.empty(t.numel() + by, device=t.device, dtype=t.dtype)[by:].copy_(t)


@pytest.mark.parametrize("bits", [8, 32])
def test_state_buffers_that_are_not_aligned_are_refused(ops, bits):
    p, g = torch.ones(700, device="cuda"), torch.ones(700, device="cuda")
    state = {k: v.clone() for k, v in ops.TensorSet([p], [g], state_bits=bits).state.items()}
    for k, v in state.items():
        if v.element_size() == 4 and bits == 8:
            continue                                    # a scale is one word
        for by in (1, 2, 3):
            with pytest.raises(ValueError, match="aligned"):
                ops.TensorSet([p], [g], state_bits=bits, state={**state, k: shifted(v.view(torch.uint8) if bits == 8 else v, by).view(v.dtype)})
    four = {k: shifted(v.view(torch.uint8), 4).view(v.dtype) if v.element_size() == 1 else shifted(v, 1 if bits == 8 else 4) for k, v in state.items()}
    q = p.clone()
    for params, held in ((p, state), (q, four)):        # one of 4 codes, 4 floats, one scale is aligned enough
        ops.adamw_step(ops.TensorSet([params], [g], state_bits=bits, state=held), 1e-2, 0.9, 0.999, 1e-8, 1)
    assert torch.equal(p, q) and all(torch.equal(state[k].view(torch.uint8), four[k].view(torch.uint8)) for k in state)
