"""The class loss against a table that holds infinity or NaN, by every path: rows without a class keep their zeros."""
import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("T,V,D", [(90, 5, 64), (90, 5, 63), (300, 20, 40), (300, 5, 600), (300, 100, 64), (100, 300, 64), (100, 300, 65), (300, 300, 128), (200, 140, 70),
                                   (700, 2000, 40), (2100, 4100, 72), (4099, 1201, 100)])
@pytest.mark.parametrize("value", [float("inf"), float("nan")])
def test_rows_without_a_class_against_a_table_that_is_not_finite(T, V, D, dtype, value):
    from discrete_dppm_graphs_amd import ops
    g = torch.Generator().manual_seed(T + V)
    x, w = torch.randn(T, D, generator=g).to(dtype).cuda(), torch.randn(V, D, generator=g).to(dtype).cuda()
    y = torch.randint(0, V, (T,), generator=g)
    none = torch.rand(T, generator=g) < 0.5
    none[0], none[T - 1] = True, False
    y[none] = torch.tensor([-1, V, 2 ** 40])[torch.randint(0, 3, (int(none.sum()),), generator=g)]
    w[V // 2, D - 1] = value
    _, row_loss, dx, _ = ops.loss_ce(x, w, y.cuda())
    none = none.cuda()
    assert (row_loss[none] == 0).all() and (dx[none] == 0).all()
    assert not torch.isfinite(row_loss[~none]).any() if value != value else not torch.isfinite(dx[~none].float()).all(1).any()
    loss, row_loss, dx, dw = ops.loss_ce(x, w, torch.full((T,), -1).cuda())
    assert loss.item() == 0 and all((t == 0).all() for t in (row_loss, dx, dw))
