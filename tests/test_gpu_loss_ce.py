"""GPU parity of dppm_loss_ce_fwd_bwd (ops.loss_ce) against the float64 form of oracle/classes.py.

Tolerances, with u = 2^-24 and h = 2^-8 for bfloat16 inputs (half a step), 0 for float32:
  a score is a sum of D products; each float32 product is three-piece split work, under 2^-21 of it: |ds| <= (D + 16) u sum_k |x_k w_k|;
  an exponential of it: relative error |ds| + (8 + |s|) u at both ends of the subtraction, so e_t = 2 max_v |ds| + 64 u + 4 max |s| u for a row;
  row_loss: 2 e_t + 4 u |lse| + 4 u |s|;
  a gradient of the scores: for bfloat16 the stored exponential is rounded to half precision (2^-11 of it, or 2^-25 of the strip's largest where
  it is subnormal) and d to bfloat16 (h): |dd| <= (2^-11 + h + 16 u) |d| (1 + h) + 2^-25 max p g + e_t p g; for float32 three pieces keep 2^-23: 16 u |d|;
  dx: sum_v |dd| |W| + V-term sum in float32 + splits (V + 64) u sum |d| |W|, then its rounding (h or u); dW likewise over the rows."""
import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu

U, H = 2.0 ** -24, 2.0 ** -8
F32, BF16 = torch.float32, torch.bfloat16


@pytest.fixture(scope="module")
def ops():
    from discrete_dppm_graphs_amd import ops
    return ops


def make(T, V, D, dtype, seed, sure=6.0, missing=0.1):
    g = torch.Generator().manual_seed(seed)
    w = (torch.randn(V, D, generator=g) * D ** -0.5).to(dtype)
    y = torch.randint(0, V, (T,), generator=g)
    x = (torch.randn(T, D, generator=g) + sure * torch.rand(T, 1, generator=g) * w[y].float()).to(dtype)
    y[torch.rand(T, generator=g) < missing] = -1
    return x, w, y, torch.rand(T, generator=g) + 0.5


def bounds(x, w, y, rw, denom, want):
    """tolerances of (loss, row_loss, dx, dweight)"""
    _, row_loss, dx, dw, p, d = want
    h = H if x.dtype == BF16 else 0.0
    xd, wd, T, V, D = x.double().abs(), w.double().abs(), x.shape[0], w.shape[0], x.shape[1]
    ok = (y >= 0) & (y < V)
    n = float(ok.sum().clamp(min=1)) if denom is None else denom
    g = torch.where(ok, rw.double() if rw is not None else torch.ones(T).double(), torch.zeros(T).double()).unsqueeze(1) / n
    mag = (xd @ wd.t()).amax(1, keepdim=True)
    s_err = (D + 16) * U * mag
    e = 2 * s_err + 64 * U + 4 * mag * U
    row_tol = torch.where(ok, (2 * e + 8 * U * (mag + np.log(V) + 1)).squeeze(1), torch.zeros(()).double())
    loss_tol = (row_tol * g.squeeze(1)).sum() + 8 * U * (row_loss * g.squeeze(1)).sum()
    dd = ((2.0 ** -11 + h if h else 0) + 16 * U) * d.abs() * (1 + h) + (2.0 ** -25 * (1 + h) * p.amax(1, keepdim=True) * g if h else 0) + e * p * g * (1 + 2 * h) + 1e-37
    dx_tol = dd @ wd + (V + 64) * U * (d.abs() @ wd)
    dw_tol = dd.t() @ xd + (T + 64) * U * (d.abs().t() @ xd)
    last = h if h else 4 * U
    return loss_tol, row_tol, dx_tol * (1 + last) + last * dx.abs() + 1e-37, dw_tol * (1 + last) + last * dw.abs() + 1e-37


def check(ops, x, w, y, rw=None, denom=None):
    from oracle import classes
    want = classes.cross_entropy(x, w, y, rw, denom)
    tol = bounds(x, w, y, rw, denom, want)
    args = (x.cuda(), w.cuda(), y.cuda(), rw.cuda() if rw is not None else None, denom)
    got = ops.loss_ce(*args)
    for name, a, b, t in zip(("loss", "row_loss", "dx", "dweight"), got, want, tol):
        off = (a.cpu().double() - b).abs()
        assert torch.isfinite(a).all(), name
        assert (off <= t).all(), (name, (off / t).max().item())
    assert got[2].dtype == x.dtype and got[3].dtype == w.dtype
    only = ops.loss_ce(*args, want_grad=False)
    assert only[2] is None and only[3] is None
    assert ((only[0].cpu().double() - want[0]).abs() <= tol[0]) and ((only[1].cpu().double() - want[1]).abs() <= tol[1]).all()
    return got


CASES = [(1, 1, 1), (1, 2, 3), (2, 64, 64), (3, 65, 16), (5, 127, 128), (31, 129, 40), (32, 300, 64), (33, 300, 64), (64, 1000, 192), (65, 257, 100), (100, 5000, 33),
         (129, 640, 256), (257, 513, 320), (300, 70, 1000), (777, 1009, 128), (1000, 3, 8)]


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("T,V,D", CASES)
def test_loss_and_gradients(ops, T, V, D, dtype):
    x, w, y, rw = make(T, V, D, dtype, T + V + D)
    check(ops, x, w, y, rw)
    check(ops, x, w, y, None, 3.5)


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("T,V,D", [(512, 33000, 256), (2100, 4100, 72), (260, 66000, 64)])
def test_tiles_of_256(ops, T, V, D, dtype):
    """sizes whose products are cut into 256 x 256 tiles, with ragged edges"""
    x, w, y, rw = make(T, V, D, dtype, 1)
    check(ops, x, w, y, rw)


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("T,V,D", [(1001, 5003, 200), (4099, 1201, 100), (901, 4600, 264)])
def test_tiles_of_128(ops, T, V, D, dtype):
    """sizes whose scores are cut into 128 x 128 tiles, with ragged edges"""
    x, w, y, rw = make(T, V, D, dtype, 16)
    check(ops, x, w, y, rw)


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("T,V,D", [(2060, 2300, 2056), (600, 2300, 2050)])
def test_gradients_by_whole_and_cut_tiles_of_256(ops, T, V, D, dtype):
    x, w, y, rw = make(T, V, D, dtype, 17)
    check(ops, x, w, y, rw)


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_very_many_rows_of_few_classes(ops, dtype):
    """more than 65535 workgroups of 16 rows"""
    x, w, y, rw = make(1_100_003, 3, 8, dtype, 9)
    check(ops, x, w, y, rw)


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("T,V,D", [(1, 1, 8), (15, 16, 64), (16, 17, 64), (17, 32, 40), (300, 5, 128), (129, 20, 72), (1000, 16, 256), (4097, 31, 248), (65, 17, 256), (513, 7, 512),
                                   (90, 1, 264), (9001, 2, 8), (70000, 5, 64), (50, 33, 64), (50, 5, 520), (50, 17, 264),
                                   (700, 64, 128), (3001, 50, 96), (300, 64, 136), (700, 128, 64), (5003, 100, 48), (300, 129, 64), (300, 65, 72),
                                   (777, 5, 77), (50, 16, 511), (300, 32, 255), (1000, 64, 101), (1000, 64, 33), (300, 90, 63), (300, 128, 50), (5000, 3, 1), (700, 9, 130)])
def test_few_classes(ops, T, V, D, dtype):
    """few classes go in one pass, every size of it (16 classes of 512 values to 128 of 64); and the first sizes that do not"""
    x, w, y, rw = make(T, V, D, dtype, T + V + D)
    got = check(ops, x, w, y, rw)
    check(ops, x, w, y, None, 2.5)
    assert all(torch.equal(a, b) for a, b in zip(got, ops.loss_ce(x.cuda(), w.cuda(), y.cuda(), rw.cuda())))
    odd = torch.zeros(T * D + 1, dtype=dtype).cuda()[1:].view(T, D).copy_(x)         # not on 16 bytes
    from oracle import classes
    want = classes.cross_entropy(x, w, y, rw)
    for a, b, t in zip(ops.loss_ce(odd, w.cuda(), y.cuda(), rw.cuda()), want, bounds(x, w, y, rw, None, want)):
        assert ((a.cpu().double() - b).abs() <= t).all()


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("T,V,D", [(700, 5, 1000), (300, 16, 2048), (300, 16, 2056), (100, 2, 4096), (1000, 30, 600), (2000, 60, 200), (500, 90, 130), (700, 120, 256), (700, 128, 300), (129, 3, 1027),
                                   (5000, 20, 777), (1, 1, 513), (15, 33, 129), (9001, 7, 520), (40000, 40, 192)])
def test_few_classes_of_wide_rows(ops, T, V, D, dtype):
    """few classes in two passes: every number of classes, slices of dims that are whole and not, the first sizes beyond"""
    test_few_classes(ops, T, V, D, dtype)


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("V,D", [(5, 64), (5, 600), (90, 63), (300, 72), (300, 128), (2000, 40)])
def test_non_finite_rows_with_and_without_a_class(ops, V, D, dtype):
    x, w, y, rw = make(200, V, D, dtype, 12, missing=0.0)
    clean = ops.loss_ce(x.cuda(), w.cuda(), y.cuda(), rw.cuda(), 200.0)
    bad = torch.zeros(200, dtype=torch.bool)
    bad[3] = bad[40] = bad[199] = True
    x[3], x[40, 5], x[199] = float("inf"), float("nan"), float("-inf")
    _, row_loss, dx, _ = ops.loss_ce(x.cuda(), w.cuda(), y.cuda(), rw.cuda(), 200.0)
    assert torch.equal(torch.isfinite(row_loss.cpu()), ~bad) and torch.equal(torch.isfinite(dx.cpu().float()).all(1), ~bad)
    assert torch.equal(dx.cpu()[~bad], clean[2].cpu()[~bad])
    y[bad] = torch.tensor([-1, V, 2 ** 40])              # nothing that such rows hold counts once they have no class
    rw[bad] = torch.tensor([float("inf"), float("nan"), 1.0])
    loss, row_loss, dx, dw = ops.loss_ce(x.cuda(), w.cuda(), y.cuda(), rw.cuda(), 200.0)
    z = x.clone()
    z[bad] = 0
    ones = torch.where(bad, torch.ones(()), rw)
    want = ops.loss_ce(z.cuda(), w.cuda(), y.cuda(), ones.cuda(), 200.0)
    assert (row_loss[bad.cuda()] == 0).all() and (dx[bad.cuda()] == 0).all()
    assert all(torch.equal(a, b) for a, b in zip((loss, row_loss, dx, dw), want))
    none = ops.loss_ce(x.cuda(), w.cuda(), torch.full((200,), -1).cuda())
    assert none[0].item() == 0 and all((t == 0).all() for t in none)


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_few_classes_in_a_graph(ops, dtype):
    x, w, y, rw = (t.cuda() for t in make(10000, 6, 48, dtype, 13))
    eager = ops.loss_ce(x, w, y, rw)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = ops.loss_ce(x, w, y, rw)
    other = make(10000, 6, 48, dtype, 14)
    for k in range(4):
        if k == 2:
            x.copy_(other[0]), y.copy_(other[2])
            eager = ops.loss_ce(x, w, y, rw)
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(out, eager)), k


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("T,V,D", [(9001, 140, 9), (20000, 70, 72), (1_100_003, 65, 72)])
def test_many_rows_in_tiles(ops, T, V, D, dtype):
    """rows counted and losses summed by several workgroups; more than 65535 workgroups of the turn"""
    x, w, y, rw = make(T, V, D, dtype, 15)
    check(ops, x, w, y, rw)


@pytest.mark.parametrize("dtype,T,V", [(F32, 2500, 60000), (BF16, 9000, 131100)])
def test_several_blocks_of_rows(ops, dtype, T, V):
    """T V over 2^27 (float32) or 2^30 (bfloat16): the rows go in blocks whose parts of dweight add up in float32 (one more u a block, within
    the T-term sum's allowance); compared on the device against float64 there, with the tolerances of `bounds` for its largest entries"""
    x, w, y, rw = (t.cuda() for t in make(T, V, 64, dtype, 10))
    loss, row_loss, dx, dw = ops.loss_ce(x, w, y, rw)
    h = H if dtype == BF16 else 0.0
    ok = y >= 0
    share = (torch.where(ok, rw, torch.zeros(()).cuda()).double() / ok.sum()).unsqueeze(1)
    xd, wd = x.double(), w.double()
    want_dw, mag_dw = torch.zeros_like(wd), torch.zeros_like(wd)
    for rows in torch.arange(T, device="cuda").split(1500):
        s = xd[rows] @ wd.t()
        mag = (xd[rows].abs() @ wd.abs().t()).amax(1, keepdim=True)
        lse = torch.logsumexp(s, 1, keepdim=True)
        at = y[rows].clamp(min=0).unsqueeze(1)
        e = 2 * (64 + 16) * U * mag + 64 * U + 4 * mag * U
        off = (row_loss[rows].double() - torch.where(ok[rows], (lse - s.gather(1, at)).squeeze(1), torch.zeros(()).cuda().double())).abs()
        assert (off <= (2 * e + 8 * U * (mag + np.log(V) + 1)).squeeze(1)).all()
        p = (s - lse).exp()
        d = p.clone().scatter_add_(1, at, torch.full_like(lse, -1.0)) * share[rows]
        dd = ((2.0 ** -11 + h if h else 0) + 16 * U) * d.abs() * (1 + h) + e * p * share[rows] * (1 + 2 * h) + 1e-37
        if h:
            dd = dd + 2.0 ** -25 * (1 + h) * p.amax(1, keepdim=True) * share[rows]
        tol = dd @ wd.abs() + (V + 64) * U * (d.abs() @ wd.abs())
        want = d @ wd
        last = h if h else 4 * U
        assert ((dx[rows].double() - want).abs() <= tol * (1 + last) + last * want.abs() + 1e-37).all()
        want_dw += d.t() @ xd[rows]
        mag_dw += dd.t() @ xd[rows].abs() + (T + 64) * U * (d.abs().t() @ xd[rows].abs())
    assert ((dw.double() - want_dw).abs() <= mag_dw * (1 + last) + last * want_dw.abs() + 1e-37).all()


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_certain_and_hopeless_rows(ops, dtype):
    x, w, y, rw = make(200, 300, 64, dtype, 2, missing=0.0)
    x = (x.float() * 30).to(dtype)                       # scores of +-100: most probabilities are 0 or 1
    check(ops, x, w, y, rw)
    best = (x.double() @ w.double().t()).argmax(1)
    check(ops, x, w, best, rw)


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_rows_without_a_class(ops, dtype):
    x, w, y, _ = make(50, 40, 24, dtype, 3)
    for bad in (-1, 40, 2 ** 40, -2 ** 40):
        loss, row_loss, dx, dw = ops.loss_ce(x.cuda(), w.cuda(), torch.full((50,), bad).cuda())
        assert loss.item() == 0 and (row_loss == 0).all() and (dx == 0).all() and (dw == 0).all()
    y[7] = -1
    x[7] = float("nan")                                  # what such a row holds does not matter to the others
    rw = torch.ones(50)
    rw[7] = float("inf")
    ok = x.clone()
    ok[7] = 0
    loss, row_loss, dx, dw = ops.loss_ce(x.cuda(), w.cuda(), y.cuda(), rw.cuda())
    assert torch.isfinite(loss) and (dx[7] == 0).all() and row_loss[7] == 0 and torch.isfinite(dw).all()
    from oracle import classes
    rw[7] = 1
    want = classes.cross_entropy(ok, w, y, rw)
    tol = bounds(ok, w, y, rw, None, want)
    assert (loss.cpu().double() - want[0]).abs() <= tol[0] and ((dx.cpu().double() - want[2]).abs() <= tol[2]).all()


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_non_finite_scores_stay_in_their_rows(ops, dtype):
    x, w, y, _ = make(70, 90, 32, dtype, 4, missing=0.0)
    x[3] = float("inf")
    x[40, 5] = float("nan")
    _, row_loss, dx, _ = ops.loss_ce(x.cuda(), w.cuda(), y.cuda())
    bad = torch.zeros(70, dtype=torch.bool)
    bad[3] = bad[40] = True
    assert torch.equal(torch.isfinite(row_loss.cpu()), ~bad) and torch.equal(torch.isfinite(dx.cpu().float()).all(1), ~bad)


def test_gradient_against_differences(ops):
    """float32: central differences of the loss along random directions; the loss is off by at most `tol`, the step's own error is third order"""
    x, w, y, rw = make(60, 50, 24, F32, 5)
    got = ops.loss_ce(x.cuda(), w.cuda(), y.cuda(), rw.cuda())
    from oracle import classes
    tol = bounds(x, w, y, rw, None, classes.cross_entropy(x, w, y, rw))[0].item()
    g = torch.Generator().manual_seed(6)
    vx, vw = torch.randn(x.shape, generator=g), torch.randn(w.shape, generator=g)
    eps = 2.0 ** -6
    for dx, dw in ((vx, torch.zeros_like(w)), (torch.zeros_like(x), vw)):
        a, b = (ops.loss_ce((x + s * eps * dx).cuda(), (w + s * eps * dw).cuda(), y.cuda(), rw.cuda(), want_grad=False)[0].item() for s in (1, -1))
        slope = (got[2].cpu() * dx).sum().item() + (got[3].cpu() * dw).sum().item()
        third = [classes.cross_entropy(x.double() + s * eps * dx, w.double() + s * eps * dw, y, rw)[0].item() for s in (1, -1)]
        exact_diff = (third[0] - third[1]) / (2 * eps)
        assert abs((a - b) / (2 * eps) - exact_diff) <= 4 * tol / eps
        assert abs(slope - exact_diff) <= 4 * tol / eps + 0.05 * abs(slope) + 1e-2 * eps


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_unaligned_inputs_and_repeats(ops, dtype):
    x, w, y, rw = make(90, 200, 64, dtype, 7)
    want = ops.loss_ce(x.cuda(), w.cuda(), y.cuda(), rw.cuda())
    again = ops.loss_ce(x.cuda(), w.cuda(), y.cuda(), rw.cuda())
    assert all(torch.equal(a, b) for a, b in zip(want, again))
    odd = torch.zeros(90 * 64 + 1, dtype=dtype).cuda()[1:].view(90, 64).copy_(x)
    got = ops.loss_ce(odd, w.cuda(), y.cuda(), rw.cuda())
    assert all(torch.equal(a, b) for a, b in zip(want, got))


def test_streams_and_graph_replays(ops):
    x, w, y, rw = (t.cuda() for t in make(300, 500, 128, BF16, 8))
    want = ops.loss_ce(x, w, y, rw)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        got = ops.loss_ce(x, w, y, rw)
    torch.cuda.current_stream().wait_stream(s)
    assert all(torch.equal(a, b) for a, b in zip(want, got))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = ops.loss_ce(x, w, y, rw)
    for k in range(3):
        nx, _, ny, _ = make(300, 500, 128, BF16, 20 + k)
        x.copy_(nx)
        y.copy_(ny)
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(out, ops.loss_ce(x, w, y, rw)))


def test_no_rows(ops):
    w = torch.randn(5, 8, device="cuda")
    loss, row_loss, dx, dw = ops.loss_ce(w[:0], w, torch.empty(0, dtype=torch.int64, device="cuda"))
    assert loss.item() == 0 and row_loss.shape == (0,) and dx.shape == (0, 8) and (dw == 0).all() and dw.shape == (5, 8)


def test_refusals(ops):
    x, w, y = torch.zeros(6, 4, device="cuda"), torch.zeros(5, 4, device="cuda"), torch.zeros(6, dtype=torch.int64, device="cuda")
    for f, e in ((lambda: ops.loss_ce(x.half(), w.half(), y), TypeError), (lambda: ops.loss_ce(x, w.bfloat16(), y), TypeError),
                 (lambda: ops.loss_ce(x, w[:, :3], y), ValueError), (lambda: ops.loss_ce(x, w, y[:5]), ValueError), (lambda: ops.loss_ce(x, w, y.int()), TypeError),
                 (lambda: ops.loss_ce(x[0], w, y), ValueError), (lambda: ops.loss_ce(x.t(), w, y), ValueError), (lambda: ops.loss_ce(x, w, y, denom=0.0), ValueError),
                 (lambda: ops.loss_ce(x, w, y, denom=float("nan")), ValueError), (lambda: ops.loss_ce(x, w, y, torch.ones(5, device="cuda")), ValueError),
                 (lambda: ops.loss_ce(x, w[:0], y), RuntimeError), (lambda: ops.loss_ce(x, w, y.cpu()), RuntimeError)):
        with pytest.raises(e):
            f()
    torch.cuda.synchronize()
