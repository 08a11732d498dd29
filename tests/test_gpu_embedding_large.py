"""Lookup and gradient at sizes whose grids would have 2^32 threads or more (a launch has fewer in a dimension): exact results, since the
values are whole numbers that bfloat16 and float32 hold."""
import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def ops():
    from discrete_dppm_graphs_amd import ops
    return ops


def test_lookup_of_2_to_the_26_rows_of_129_values(ops):
    T, V, D = 2 ** 26 + 5, 50, 129
    g = torch.Generator(device="cuda").manual_seed(0)
    w = torch.randint(-100, 100, (V, D), generator=g, device="cuda").bfloat16()
    ids = torch.randint(-1, V, (T,), generator=g, device="cuda")
    out = ops.embedding_fwd(w, ids)
    padded = torch.cat([w, torch.zeros_like(w[:1])])
    for at in range(0, T, 2 ** 23):
        assert torch.equal(out[at:at + 2 ** 23], padded.index_select(0, ids[at:at + 2 ** 23] % (V + 1))), at


@pytest.mark.parametrize("accumulate", [False, True])
def test_gradient_of_2_to_the_30_positions(ops, accumulate):
    T, V = 2 ** 30 + 70, 300
    ids = torch.arange(T, device="cuda").mul_(7919).remainder_(V + 1)           # every class, and V: none
    dout = torch.ones(T, 1, device="cuda", dtype=torch.bfloat16)
    out = torch.full((V, 1), 3.0, device="cuda")
    ops.embedding_wgrad(dout, ids, V, out=out, accumulate=accumulate)
    want = torch.bincount(ids, minlength=V + 1)[:V].double() + (3 if accumulate else 0)
    assert want.max() < 2 ** 24 and torch.equal(out[:, 0].double(), want)


def test_gradient_of_2_to_the_30_classes(ops):
    V, ids = 2 ** 30 + 100, torch.tensor([0, 5, 2 ** 30 + 99, 5, -1, 2 ** 29, 2 ** 30 + 98])
    out = torch.full((V, 1), 3.0, device="cuda", dtype=torch.bfloat16)
    ops.embedding_wgrad(torch.arange(1.0, 8.0, device="cuda").view(7, 1), ids.cuda(), V, out=out)
    assert torch.equal(out[ids[[0, 1, 2, 5, 6]].cuda(), 0].float().cpu(), torch.tensor([1.0, 6.0, 3.0, 6.0, 7.0]))
    assert (out != 0).sum().item() == 5
