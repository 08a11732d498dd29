"""What ops.loss_ce keeps of d beyond one bfloat16 plane: in dx of the row's own class (more than 128 rows), in both gradients of every class (up
to 128 rows).  The tolerances leave out the bfloat16 rounding of those entries, so that a kernel without it fails; that it would is shown on the CPU,
with d rounded to one plane in float64.

Tolerances, with u = 2^-24, h = 2^-8 (half a step of bfloat16), g = the row's weight / n and e = a row's relative error of an exponential (a score
is a sum of D products, each within u and summed in float32: |ds| <= (D + 16) u sum |x w|; e = 2 max |ds| + 64 u + 4 max |s| u):
  stored exponentials are halves: 2^-11 of each, or 2^-25 of the largest; the own class's comes from its float32 score;
  one plane keeps h of an entry; what a second plane, or a residual rounded to bfloat16, leaves of it is h h = 2^-16;
  sums in float32: (terms + 64) u of the sum of magnitudes; the result is rounded once: h of it."""
import pytest
import torch

from oracle import classes

U, H = 2.0 ** -24, 2.0 ** -8
# more than 128 rows: tiles of 128 x 128 and of 256 x 256, gradients whole and split, ragged; up to 128 rows: two planes
MANY = [(257, 4000, 64), (1001, 5003, 200), (300, 20000, 96), (513, 9001, 136), (2100, 4100, 72), (600, 2300, 2050), (5000, 140, 40), (2050, 33000, 264)]
TELLING = MANY[:5]       # with many rows a class or very long rows of x, what the other entries may lose covers what the own one does
FEW = [(8, 2584, 64), (33, 300, 64), (100, 5000, 33), (128, 4100, 192)]


def make(T, V, D, seed, hot=0.2, top=None, missing=0.1):
    """unlearned rows and nearly certain ones; a share `hot` of the rows in the class `top`; a share `missing` without a class"""
    gen = torch.Generator().manual_seed(seed)
    w = (torch.randn(V, D, generator=gen) * D ** -0.5).bfloat16()
    y = torch.randint(0, V, (T,), generator=gen)
    y[torch.rand(T, generator=gen) < hot] = V // 3 if top is None else top
    x = (torch.randn(T, D, generator=gen) + 6.0 * torch.rand(T, 1, generator=gen) * w[y].float()).bfloat16()
    y[torch.rand(T, generator=gen) < missing] = -1
    return x, w, y, torch.rand(T, generator=gen) + 0.5


def bounds(x, w, y, rw, want):
    _, _, dx, dw, p, d = want
    T, V, D = x.shape[0], w.shape[0], x.shape[1]
    xd, wd = x.double().abs(), w.double().abs()
    ok = (y >= 0) & (y < V)
    g = torch.where(ok, rw.double(), torch.zeros(()).double()).unsqueeze(1) / float(ok.sum().clamp(min=1))
    mag = (xd @ wd.t()).amax(1, keepdim=True)
    e = 2 * (D + 16) * U * mag + 64 * U + 4 * mag * U
    at = y.clamp(0, V - 1).unsqueeze(1)

    def entries(all_keep, own_keeps):
        dd = (2.0 ** -11 + all_keep + 16 * U) * d.abs() * (1 + H) + 2.0 ** -25 * (1 + H) * p.amax(1, keepdim=True) * g
        return dd.scatter_(1, at, (own_keeps + 16 * U) * (1 + H) * d.abs().gather(1, at)) + e * p * g * (1 + 2 * H)

    few = T <= 128
    dx_tol = entries(H * H if few else H, H * H) @ wd + (V + 64) * U * (d.abs() @ wd)
    dw_tol = entries(H * H if few else H, H * H if few else H).t() @ xd + (T + 64) * U * (d.abs().t() @ xd)
    return dx_tol * (1 + H) + H * dx.abs() + 1e-37, dw_tol * (1 + H) + H * dw.abs() + 1e-37


def rounded(x, w, y, rw, want, sign):
    """dx and dweight with n d in one plane and, in dx, `sign` times what the own entries lost added; all else in float64"""
    d, at = want[5], y.clamp(min=0)
    n = float((y >= 0).sum())
    q = (d * n).float().bfloat16().double()
    i = torch.arange(x.shape[0])
    lost = torch.where(y >= 0, d[i, at] * n - q[i, at], torch.zeros(()).double()).unsqueeze(1)
    return ((q @ w.double() + sign * lost * w.double()[at]) / n).float().bfloat16(), (q.t() @ x.double() / n).float().bfloat16()


def worst(got, want, tol):
    return ((got.double() - want).abs() / tol).max().item()


@pytest.mark.parametrize("T,V,D", TELLING)
def test_the_tolerances_tell_one_plane_from_more(T, V, D):
    x, w, y, rw = make(T, V, D, T + V)
    want = classes.cross_entropy(x, w, y, rw)
    dx_tol, dw_tol = bounds(x, w, y, rw, want)
    for sign in (1.0, 0.0, -1.0):
        dx, dw = rounded(x, w, y, rw, want, sign)
        assert (worst(dx, want[2], dx_tol) <= 1) == (sign == 1.0) and worst(dw, want[3], dw_tol) <= 1, sign


@pytest.mark.parametrize("T,V,D", FEW)
def test_the_tolerances_tell_two_planes_from_one(T, V, D):
    x, w, y, rw = make(T, V, D, T + V)
    want = classes.cross_entropy(x, w, y, rw)
    dx_tol, dw_tol = bounds(x, w, y, rw, want)
    for sign in (0.0, 1.0):       # one plane; one plane and the own entries' residuals in dx
        dx, dw = rounded(x, w, y, rw, want, sign)
        assert max(worst(dx, want[2], dx_tol), worst(dw, want[3], dw_tol)) > 1, sign
    dx, dw = want[2].float().bfloat16(), want[3].float().bfloat16()
    assert worst(dx, want[2], dx_tol) <= 1 and worst(dw, want[3], dw_tol) <= 1


@pytest.mark.gpu
@pytest.mark.parametrize("T,V,D", MANY + FEW)
def test_gradients_keep_the_own_entry(T, V, D):
    from discrete_dppm_graphs_amd import ops
    x, w, y, rw = make(T, V, D, T + V)
    want = classes.cross_entropy(x, w, y, rw)
    dx_tol, dw_tol = bounds(x, w, y, rw, want)
    args = [t.cuda() for t in (x, w, y, rw)]
    _, _, dx, dw = ops.loss_ce(*args)
    assert worst(dx.cpu(), want[2], dx_tol) <= 1, ("dx", worst(dx.cpu(), want[2], dx_tol))
    assert worst(dw.cpu(), want[3], dw_tol) <= 1, ("dweight", worst(dw.cpu(), want[3], dw_tol))
    again = ops.loss_ce(*args)
    assert torch.equal(dx, again[2]) and torch.equal(dw, again[3])


@pytest.mark.gpu
@pytest.mark.parametrize("top", ["first", "last"])
@pytest.mark.parametrize("missing", [0.0, 0.5])
@pytest.mark.parametrize("T,V,D", [(129, 640, 72), (200, 300, 64), (700, 700, 64), (4096, 129, 40), (4099, 300, 72), (9001, 200, 16)])
def test_all_rows_of_one_class(T, V, D, missing, top):
    """every row's own entry in the same row of dweight, of the first strip of classes or of the last"""
    from discrete_dppm_graphs_amd import ops
    x, w, y, rw = make(T, V, D, 3, 1.1, 0 if top == "first" else V - 1, missing)
    want = classes.cross_entropy(x, w, y, rw)
    dx_tol, dw_tol = bounds(x, w, y, rw, want)
    _, _, dx, dw = ops.loss_ce(*(t.cuda() for t in (x, w, y, rw)))
    assert worst(dx.cpu(), want[2], dx_tol) <= 1 and worst(dw.cpu(), want[3], dw_tol) <= 1
