"""ops.TensorSet and ops.adamw_step at the edges of what they take: state buffers that are not aligned, gradients whose squares are
denormal, norms that float32 cannot hold."""
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


@pytest.mark.parametrize("bits", [8, 32])
@pytest.mark.parametrize("eps", [0.0, 1e-30])
def test_gradients_whose_squares_are_denormal(ops, bits, eps):
    """v' = (1 - beta2) g^2 from 1e-43 on, against float64.  (1 - beta2) g is rounded, then its product with g, off by half of 2^-149 there:
    |dv| <= 4 u v + 2^-150, so the root by half of that relative to v; the rest of the update by 32 u, and 8 u where 1 - beta is rounded."""
    g = np.geomspace(1e-20, 1e-14, 256).astype(np.float32)
    p = torch.zeros(256, device="cuda")
    ops.adamw_step(ops.TensorSet([p], [torch.as_tensor(g).cuda()], state_bits=bits), 1e-3, 0.9, 0.999, eps, 1)
    g = g.astype(np.float64)
    want = -1e-3 * g / (g + eps)
    v = 0.001 * g * g
    assert (np.abs(p.double().cpu().numpy() - want) <= np.abs(want) * ((4 * U * v + 2.0 ** -150) / v + 40 * U)).all()


@pytest.mark.parametrize("bits", [8, 32])
@pytest.mark.parametrize("n,most,fits", [(2, 2.0 ** 127, True), (8, 2.0 ** 127, False), (3_000_000, 2.0 ** 125, False)])
def test_a_norm_that_float32_cannot_hold_is_infinite(ops, bits, n, most, fits):
    """finite gradients: their norm sqrt(n) most is returned, and the step made, while it is under 2^128; else it is infinite and nothing changes"""
    p, g = torch.ones(n, device="cuda"), torch.full((n,), most, device="cuda")
    tset = ops.TensorSet([p], [g], state_bits=bits)
    norm = ops.adamw_step(tset, 1e-2, 0.9, 0.999, 1e-8, 1, max_norm=1.0)
    assert (p != 1).all() if fits else (p == 1).all()
    assert all((v.view(torch.uint8) != 0).any().item() == fits for v in tset.state.values())
    assert abs(norm.item() / (n ** 0.5 * most) - 1) <= U if fits else norm.item() == float("inf")


@pytest.mark.parametrize("chunks", [1, 512, 513, 2047, 2048, 2049, 5000])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_norms_by_either_number_of_launches(ops, chunks, dtype):
    """summed in float64 and rounded once to float32; the clipped step is the unclipped one of the scaled gradients, whose factor is rounded (4 u
    of m' and root each side, 40 u of an update of at most lr)"""
    n = chunks * 4096 - 3
    g = torch.Generator(device="cuda").manual_seed(chunks)
    grad = torch.randn(n, generator=g, device="cuda").to(dtype)
    norm = grad.double().square().sum().sqrt().item()
    p, q = torch.ones(n, device="cuda"), torch.ones(n, device="cuda")
    got = ops.adamw_step(ops.TensorSet([p], [grad]), 1e-2, 0.9, 0.999, 1e-3, 1, max_norm=0.5 * norm)
    ops.adamw_step(ops.TensorSet([q], [grad]), 1e-2, 0.9, 0.999, 1e-3, 1, grad_scale=0.5 * norm / (norm + 1e-6))
    assert abs(got.item() - norm) <= 2 * U * norm
    assert (p - q).abs().max().item() <= 40 * U * 1e-2 + 2 * U
