"""The class loss in several blocks of rows: how much its workspace holds (on the CPU), and blocks of few rows against float64."""
import pytest
import torch

from discrete_dppm_graphs_amd._lib import lib

U = 2.0 ** -24


def pitch(n):
    return ((n + 63) // 64 | 1) * 64


@pytest.mark.parametrize("bf16", [0, 1])
@pytest.mark.parametrize("V", [50001, 300000, 1 << 20, (1 << 21) + 1, 1 << 23])
@pytest.mark.parametrize("T", [100, 256, 896, 5368, 70001])
def test_workspace_holds_no_more_exponentials_than_stated(T, V, bf16):
    """D = 64.  A block has rows = max(64, 2^30 or 2^27 / V) at most; a pair costs its exponential (2 or 4 bytes; bfloat16 turns it in place,
    up to 128 rows into two planes) and three planes of 2 for float32; a pair of a row and a strip of 32 classes costs 8; a value of x or W
    2 bytes a plane where it is laid out, x again transposed; a row and dimension up to 256 parts of 4, a class and dimension of several blocks 4."""
    rows = min(T, max(64, (1 << (30 if bf16 else 27)) // V))
    held = (rows + 63) // 64 * 64 * pitch(V)
    planes = 1 if bf16 else 3
    allowed = held * (10 if not bf16 else 6 if T <= 128 else 2) + (V // 32 + 1) * rows * 8 + 2 * planes * (T + V) * 64 + 2 * planes * 64 * pitch(rows)
    allowed += 256 * rows * 64 * 4 + (V * 64 * 4 if bf16 and rows < T else 0) + rows * 16 + T // 2 + T // 1024 + 16384
    assert lib.dppm_loss_ce_workspace_bytes(T, V, 64, bf16, 1) <= allowed


@pytest.mark.gpu
@pytest.mark.parametrize("T,V,dtype", [(200, 1_100_003, torch.float32), (700, 300_001, torch.float32), (65, 2_100_001, torch.float32),
                                       (300, 1 << 23, torch.bfloat16)])
def test_blocks_of_few_rows(T, V, dtype):
    """blocks of 64, 256 and 128 rows, the last one smaller.  Tolerances as in test_gpu_loss_ce.py (D = 16; one more u a block is within the
    T-term sum's allowance)."""
    from discrete_dppm_graphs_amd import ops
    D, h = 16, 2.0 ** -8 if dtype == torch.bfloat16 else 0.0
    g = torch.Generator(device="cuda").manual_seed(T)
    w = (torch.randn(V, D, generator=g, device="cuda") * D ** -0.5).to(dtype)
    y = torch.randint(0, V, (T,), generator=g, device="cuda")
    x = (torch.randn(T, D, generator=g, device="cuda") + 6 * torch.rand(T, 1, generator=g, device="cuda") * w[y].float()).to(dtype)
    y[torch.rand(T, generator=g, device="cuda") < 0.1] = -1
    y[T // 2] = V - 1
    loss, row_loss, dx, dw = ops.loss_ce(x, w, y)
    only = ops.loss_ce(x, w, y, want_grad=False)
    n, ok, xd, wd = (y >= 0).sum().double(), y >= 0, x.double(), w.double()
    want_dw, tol_dw, total, tol_total = torch.zeros_like(wd), torch.zeros_like(wd), 0.0, 0.0
    for rows in torch.arange(T, device="cuda").split(32):
        s = xd[rows] @ wd.t()
        mag = (xd[rows].abs() @ wd.abs().t()).amax(1, keepdim=True)
        lse, at = torch.logsumexp(s, 1, keepdim=True), y[rows].clamp(min=0).unsqueeze(1)
        e = 2 * (D + 16) * U * mag + 64 * U + 4 * mag * U
        want = torch.where(ok[rows], (lse - s.gather(1, at)).squeeze(1), torch.zeros((), device="cuda").double())
        tol = (2 * e + 8 * U * (mag + 17)).squeeze(1)
        assert ((row_loss[rows].double() - want).abs() <= tol).all() and ((only[1][rows].double() - want).abs() <= tol).all()
        total, tol_total = total + want.sum(), tol_total + tol.sum() + 8 * U * want.sum()
        p = (s - lse).exp() * ok[rows].unsqueeze(1)
        d = (p.scatter_add(1, at, -ok[rows].double().unsqueeze(1))) / n
        dd = ((2.0 ** -11 + h if h else 0) + 16 * U) * d.abs() * (1 + h) + e * p / n * (1 + 2 * h) + 1e-37
        if h:
            dd += 2.0 ** -25 * (1 + h) * p.amax(1, keepdim=True) / n
        del s, p
        last = h if h else 4 * U
        want = d @ wd
        assert ((dx[rows].double() - want).abs() <= (dd @ wd.abs() + (V + 64) * U * (d.abs() @ wd.abs())) * (1 + last) + last * want.abs() + 1e-37).all()
        want_dw += d.t().contiguous() @ xd[rows]
        tol_dw += dd.t().contiguous() @ xd[rows].abs() + (T + 64) * U * (d.abs().t().contiguous() @ xd[rows].abs())
        del d, dd
    assert ((dw.double() - want_dw).abs() <= tol_dw * (1 + last) + last * want_dw.abs() + 1e-37).all()
    assert abs(loss.double() - total / n) <= tol_total / n and abs(only[0].double() - total / n) <= tol_total / n
