"""The differentiable fronts captured into a graph, forward and backward, and replayed with the program's own work in between."""
import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("V,D", [(6, 48), (700, 72)])
def test_lookup_and_loss_with_their_gradients_in_a_graph(V, D, dtype):
    from discrete_dppm_graphs_amd.categorical import embedding, loss_func_ce
    T = 900
    table = torch.randn(V, D, device="cuda").mul_(0.3).to(dtype).requires_grad_(True)
    ids, target = torch.randint(-1, V, (T,), device="cuda"), torch.randint(-1, V, (T,), device="cuda")
    rw = torch.rand(T, device="cuda")

    def step():
        return torch.autograd.grad(3.0 * loss_func_ce(torch.tanh(embedding(table, ids, 1.5)), table, target, rw, 100.0), (table,))[0]

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()                       # its graph is gone before the capture begins
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    for k in range(4):
        if k:
            ids.copy_(torch.randint(-1, V, (T,)))
            target.copy_(torch.randint(-1, V, (T,)))
            with torch.no_grad():
                table.mul_(0.9)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, step()), k
