"""When the differentiable front of the class loss asks for gradients: on the CPU with the operator replaced by a record of its call, on the GPU
by what it allocates."""
import pytest
import torch

from discrete_dppm_graphs_amd import categorical, ops


@pytest.fixture
def calls(monkeypatch):
    seen = []

    def loss_ce(x, weight, target, row_weight=None, denom=None, want_grad=True):
        seen.append(want_grad)
        return (x.new_zeros(()), x.new_zeros(x.shape[0]), *((torch.ones_like(x), torch.ones_like(weight)) if want_grad else (None, None)))

    monkeypatch.setattr(ops, "loss_ce", loss_ce)
    return seen


@pytest.mark.parametrize("off", [torch.no_grad, torch.inference_mode, lambda: torch.set_grad_enabled(False)])
def test_an_evaluated_loss_asks_for_no_gradients(calls, off):
    x, w, y = torch.zeros(4, 3, requires_grad=True), torch.nn.Parameter(torch.zeros(5, 3)), torch.zeros(4, dtype=torch.int64)
    with off():
        loss = categorical.loss_func_ce(x, w, y)
    assert calls == [False] and not loss.requires_grad
    with torch.no_grad(), torch.enable_grad():
        categorical.loss_func_ce(x, w, y).backward()
    assert calls == [False, True] and (x.grad == 1).all() and (w.grad == 1).all()
    categorical.loss_func_ce(x.detach(), w.detach(), y)
    assert calls == [False, True, False]


@pytest.mark.parametrize("which", [0, 1])
def test_one_input_that_requires_a_gradient(calls, which):
    x, w, y = torch.zeros(4, 3), torch.zeros(5, 3), torch.zeros(4, dtype=torch.int64)
    (x, w)[which].requires_grad_(True)
    categorical.loss_func_ce(x, w, y).backward()
    assert calls == [True] and [t.grad is not None for t in (x, w)] == [which == 0, which == 1]


def test_a_row_weight_that_requires_a_gradient_is_refused(calls):
    x, w, y = torch.zeros(4, 3, requires_grad=True), torch.zeros(5, 3), torch.zeros(4, dtype=torch.int64)
    rw = torch.ones(4, requires_grad=True)
    with pytest.raises(ValueError, match="row_weight"):
        categorical.loss_func_ce(x, w, y, rw)
    assert calls == []
    with torch.no_grad():
        categorical.loss_func_ce(x, w, y, rw)
    categorical.loss_func_ce(x, w, y, rw.detach()).backward()
    assert calls == [False, True]


@pytest.mark.gpu
@pytest.mark.parametrize("T,V,D", [(600, 2000, 96), (3000, 5, 64)])
def test_an_evaluated_loss_allocates_no_gradients(T, V, D):
    x, w = torch.randn(T, D, device="cuda", requires_grad=True), torch.nn.Parameter(torch.randn(V, D, device="cuda"))
    y = torch.randint(-1, V, (T,), device="cuda")
    trained = categorical.loss_func_ce(x, w, y)
    want = ops.loss_ce(x.detach(), w.detach(), y, want_grad=False)[0]
    torch.cuda.synchronize()
    torch.cuda.reset_peak_memory_stats()
    before = torch.cuda.memory_allocated()
    with torch.no_grad():
        loss = categorical.loss_func_ce(x, w, y)
    peak = torch.cuda.max_memory_allocated() - before
    from discrete_dppm_graphs_amd._lib import lib
    assert torch.equal(loss, want) and not loss.requires_grad and trained.requires_grad
    assert peak <= lib.dppm_loss_ce_workspace_bytes(T, V, D, 0, 0) + 4 * T + 8192      # rounded up by the allocator
