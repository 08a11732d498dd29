"""GPU parity of dppm_embedding_fwd / dppm_embedding_wgrad against the float64 forms of oracle/classes.py.

Tolerances.  The lookup is one float32 product, rounded once more to bfloat16 where that is the type: u32 (+ u16) of the value, with
u32 = 2^-24 and u16 = 2^-8.  A gradient row is a sum of n terms in float32, off by at most n u32 of the sum of magnitudes (n <= number
of positions), then the product with scale and the rounding to its type."""
import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu

U32, U16 = 2.0 ** -24, 2.0 ** -8
F32, BF16 = torch.float32, torch.bfloat16


@pytest.fixture(scope="module")
def ops():
    from discrete_dppm_graphs_amd import ops
    return ops


def classes_of(rng, T, V, kind):
    if kind == "uniform":
        ids = rng.integers(0, V, size=T)
    elif kind == "one":
        ids = np.full(T, V - 1)
    elif kind == "skewed":
        ids = np.minimum(np.floor(V ** rng.random(T)).astype(np.int64) - 1, V - 1)
    elif kind == "none":
        ids = np.full(T, -1)
    else:      # "padded": runs without a class, and ids far outside the table
        ids = rng.integers(0, V, size=T)
        ids[rng.random(T) < 0.3] = -1
        ids[rng.random(T) < 0.1] = V
        ids[rng.random(T) < 0.1] = 2 ** 40
        ids[rng.random(T) < 0.1] = -2 ** 40
    return torch.as_tensor(ids.astype(np.int64))


def sums(dout, ids, V):
    """float64: sums over positions, sums of magnitudes, counts"""
    ok = (ids >= 0) & (ids < V)
    at, rows = ids[ok], dout.reshape(ids.numel(), dout.shape[-1])[ok.reshape(-1)].double()
    z = torch.zeros(V, dout.shape[-1], dtype=torch.float64)
    return z.clone().index_add_(0, at, rows), z.clone().index_add_(0, at, rows.abs()), torch.bincount(at, minlength=V).double().unsqueeze(1)


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("T,V,D", [(1, 1, 1), (1, 7, 8), (3, 5, 4), (5, 3, 33), (16, 1000, 128), (17, 300, 1000), (1000, 20, 7), (333, 50, 2056), (2, 9, 5000)])
def test_lookup(ops, T, V, D, dtype):
    from oracle import classes
    rng = np.random.default_rng(T + V + D)
    w = torch.as_tensor(rng.normal(size=(V, D)).astype(np.float32)).to(dtype)
    ids = classes_of(rng, T, V, "padded")
    got = ops.embedding_fwd(w.cuda(), ids.cuda(), scale=1.7).cpu()
    assert got.dtype == dtype
    want = classes.embedding(w, ids, float(np.float32(1.7)))
    tol = (U32 + (U16 if dtype == BF16 else 0)) * (1 + U32) * want.abs() + 1e-38
    assert ((got.double() - want).abs() <= tol).all()
    assert torch.equal(ops.embedding_fwd(w.cuda(), ids.cuda()).cpu(), classes.embedding(w, ids).to(dtype))     # scale 1: the rows themselves
    bad = (ids < 0) | (ids >= V)
    assert (ops.embedding_fwd(w.cuda(), ids.cuda(), scale=float("inf")).cpu()[bad] == 0).all()


def test_lookup_shapes_and_out(ops):
    w = torch.randn(11, 12).cuda()
    ids = torch.randint(0, 11, (3, 4, 5)).cuda()
    out = torch.full((3, 4, 5, 12), 9.0).cuda()
    assert ops.embedding_fwd(w, ids, out=out) is out and torch.equal(out, w[ids])
    assert ops.embedding_fwd(w, ids[:0]).shape == (0, 4, 5, 12)
    assert ops.embedding_fwd(w, ids[0, 0, 0]).shape == (12,)
    odd = torch.randn(11 * 12 + 1).cuda()[1:].view(11, 12)        # rows not aligned to 16 bytes
    assert torch.equal(ops.embedding_fwd(odd, ids), odd[ids])


CASES = [(1, 1, 1), (1, 300, 8), (2, 2, 3), (63, 5, 32), (64, 70000, 16), (65, 5, 33), (777, 300, 130), (2048, 17, 128), (5003, 1000, 128), (8192, 255, 24),
         (8193, 256, 24), (9000, 65536, 40), (20001, 300, 512), (70000, 3, 8), (300000, 70001, 8)]


@pytest.mark.parametrize("kind", ["uniform", "skewed", "one", "padded", "none"])
@pytest.mark.parametrize("T,V,D", CASES)
def test_gradient(ops, T, V, D, kind):
    rng = np.random.default_rng(T + V + D + len(kind))
    ids = classes_of(rng, T, V, kind)
    d32 = torch.as_tensor(rng.normal(size=(T, D)).astype(np.float32))
    for din, dw in ((F32, F32), (BF16, BF16), (BF16, F32), (F32, BF16)):
        d = d32.to(din)
        s, mag, n = sums(d, ids, V)
        out = torch.full((V, D), 7.0, dtype=dw, device="cuda")
        got = ops.embedding_wgrad(d.cuda(), ids.cuda(), V, scale=0.37, out=out).cpu().double()
        sc = float(np.float32(0.37))
        tol = (n + 1) * U32 * mag * sc
        tol = tol + (U16 * (s * sc).abs() + U16 * tol if dw == BF16 else 0)
        assert ((got - s * sc).abs() <= tol).all(), (din, dw)
        again = ops.embedding_wgrad(d.cuda(), ids.cuda(), V, scale=0.37, out=torch.empty_like(out))
        assert torch.equal(again, out)


@pytest.mark.parametrize("dw", [F32, BF16])
@pytest.mark.parametrize("T,V,D,kind", [(1, 5, 8, "uniform"), (500, 40, 33, "padded"), (9001, 700, 64, "skewed"), (64, 9, 4, "none"), (0, 9, 4, "none")])
def test_gradient_accumulates(ops, T, V, D, kind, dw):
    rng = np.random.default_rng(T)
    ids = classes_of(rng, T, V, kind)
    d = torch.as_tensor(rng.normal(size=(T, D)).astype(np.float32))
    start = torch.as_tensor(rng.normal(size=(V, D)).astype(np.float32)).to(dw)
    out = start.cuda()
    ops.embedding_wgrad(d.cuda(), ids.cuda(), V, out=out, accumulate=True)
    s, mag, n = sums(d, ids, V)
    want = start.double() + s
    tol = (n + 2) * U32 * (mag + start.double().abs())
    tol = tol + (U16 * (want.abs() + tol) if dw == BF16 else 0)
    untouched = (n == 0).squeeze(1)
    assert torch.equal(out.cpu()[untouched], start[untouched])
    assert ((out.cpu().double() - want).abs() <= tol).all()


def test_gradient_without_positions_is_zero(ops):
    out = torch.full((70, 3), 5.0, device="cuda")
    ops.embedding_wgrad(torch.empty(0, 3, device="cuda"), torch.empty(0, dtype=torch.int64, device="cuda"), 70, out=out)
    assert (out == 0).all()


def test_infinite_and_nan_rows_stay_in_their_class(ops):
    d = torch.ones(300, 16, device="cuda")
    ids = torch.arange(300, device="cuda") % 7
    d[3] = float("nan")
    d[4] = float("inf")
    got = ops.embedding_wgrad(d, ids, 9)
    assert torch.isnan(got[3]).all() and torch.isinf(got[4]).all() and torch.isfinite(got[[0, 1, 2, 5, 6, 7, 8]]).all() and (got[7:] == 0).all()
    d[3], d[4] = 1.0, 1.0
    ids[10] = -1
    d[10] = float("nan")                                       # a padded position's gradient is not read into any class
    assert torch.isfinite(ops.embedding_wgrad(d, ids, 9)).all()


def test_streams_and_graph_replays(ops):
    rng = np.random.default_rng(1)
    T, V, D = 9001, 500, 64
    ids = classes_of(rng, T, V, "skewed").cuda()
    w, d = torch.randn(V, D, device="cuda"), torch.randn(T, D, device="cuda")
    want = ops.embedding_fwd(w, ids, 2.0), ops.embedding_wgrad(d, ids, V, 2.0)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        got = ops.embedding_fwd(w, ids, 2.0), ops.embedding_wgrad(d, ids, V, 2.0)
    torch.cuda.current_stream().wait_stream(s)
    assert all(torch.equal(a, b) for a, b in zip(want, got))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y, dw = ops.embedding_fwd(w, ids, 2.0), ops.embedding_wgrad(d, ids, V, 2.0)
    for k in range(4):
        ids.copy_(classes_of(np.random.default_rng(50 + k), T, V, "padded"))
        d.normal_()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(y, ops.embedding_fwd(w, ids, 2.0)) and torch.equal(dw, ops.embedding_wgrad(d, ids, V, 2.0))


def test_refusals(ops):
    w, ids, d = torch.zeros(5, 4, device="cuda"), torch.zeros(6, dtype=torch.int64, device="cuda"), torch.zeros(6, 4, device="cuda")
    for f, e in ((lambda: ops.embedding_fwd(w.half(), ids), TypeError), (lambda: ops.embedding_fwd(w, ids.int()), TypeError),
                 (lambda: ops.embedding_fwd(w.t(), ids), ValueError), (lambda: ops.embedding_fwd(w[0], ids), ValueError),
                 (lambda: ops.embedding_fwd(w, ids, out=torch.zeros(6, 5, device="cuda")), ValueError), (lambda: ops.embedding_fwd(w, ids.cpu()), RuntimeError),
                 (lambda: ops.embedding_fwd(w, ids, out=d.bfloat16()), TypeError), (lambda: ops.embedding_fwd(w[:0], ids), RuntimeError),
                 (lambda: ops.embedding_fwd(w, ids[:5], out=w), ValueError), (lambda: ops.embedding_wgrad(d, ids, 6, out=d), ValueError),
                 (lambda: ops.embedding_wgrad(d[:5], ids, 5), ValueError), (lambda: ops.embedding_wgrad(d, ids, 5, accumulate=True), ValueError),
                 (lambda: ops.embedding_wgrad(d, ids, 0), RuntimeError), (lambda: ops.embedding_wgrad(d, ids, 5, out=torch.zeros(4, 4, device="cuda")), ValueError),
                 (lambda: ops.embedding_wgrad(d.t(), ids, 5), ValueError), (lambda: ops.embedding_wgrad(d.double(), ids, 5), TypeError)):
        with pytest.raises(e):
            f()
    torch.cuda.synchronize()


@pytest.mark.parametrize("T,V,D", [(1, 1, 1), (7, 2, 1), (2049, 1, 3), (5000, 5, 7), (3001, 38, 64), (3001, 39, 64), (2500, 77, 16), (2500, 78, 16), (2000, 155, 10), (2000, 156, 10),
                                   (300, 64, 2048), (300, 64, 2052), (600000, 100, 60), (777, 5, 300), (60, 3, 2052),
                                   (5, 9, 1025), (70000, 5, 64), (33000, 2, 512), (9000, 30, 128)])
def test_small_tables(ops, T, V, D):
    """tables whose sums lie in LDS, their first and last sizes, aligned and not, with rows added to and left alone"""
    rng = np.random.default_rng(T + 3 * V + D)
    ids = classes_of(rng, T, V, "padded")
    if V > 2:
        ids[ids == 1] = 0                              # class 1 never occurs
    for dtype in (F32, BF16):
        dout = torch.as_tensor(rng.normal(size=(T, D)).astype(np.float32)).to(dtype)
        want, mag, n = sums(dout, ids, V)
        s = float(np.float32(0.7))
        odd = torch.zeros(T * D + 1, dtype=dtype).cuda()[1:].view(T, D).copy_(dout)
        for rows in (dout.cuda(), odd):
            for out_type in (F32, BF16):
                out = torch.full((V, D), 5.0).to(out_type).cuda()
                got = ops.embedding_wgrad(rows, ids.cuda(), V, scale=0.7, out=out)
                tol = (n + 1) * U32 * mag * s + (U32 + (U16 if out_type == BF16 else 0)) * (want * s).abs() * 1.01 + 1e-38
                assert ((got.cpu().double() - want * s).abs() <= tol).all()
                assert torch.equal(ops.embedding_wgrad(rows, ids.cuda(), V, scale=0.7, out=torch.empty_like(out)), got)
                old = torch.as_tensor(rng.normal(size=(V, D)).astype(np.float32)).to(out_type)
                if V > 2:
                    old[1] = -0.0
                    old[1, 0] = float("nan")
                more = ops.embedding_wgrad(rows, ids.cuda(), V, scale=0.7, out=old.clone().cuda(), accumulate=True).cpu()
                present = n.squeeze(1) > 0
                bits = torch.int32 if out_type == F32 else torch.int16
                assert torch.equal(more[~present].view(bits), old[~present].view(bits))          # left as they are, to the bit
                total = old.double() + want * s
                tol = tol + 2 * U32 * total.abs() + (U16 if out_type == BF16 else 0) * total.abs()
                assert ((more.double() - total).abs() <= tol)[present].all()


@pytest.mark.parametrize("kind", ["uniform", "skewed", "one", "padded", "none"])
@pytest.mark.parametrize("T,V,D", [(1, 200, 8), (255, 200, 4), (257, 300, 20), (3000, 156, 64), (4096, 1000, 65), (5003, 1000, 128), (1280, 4096, 64), (1281, 4096, 64), (1280, 4097, 64),
                                   (8191, 300, 33), (8192, 160, 60), (100000, 157, 5), (655360, 159, 1), (8193, 160, 60), (700, 40000, 1), (700, 40001, 1), (20, 60000, 16), (900, 161, 130)])
def test_few_positions(ops, T, V, D, kind):
    """rows that are listed and not sorted, by one workgroup for a class or several; and the first sizes beyond"""
    rng = np.random.default_rng(T + 5 * V + D + len(kind))
    ids = classes_of(rng, T, V, kind)
    d32 = torch.as_tensor(rng.normal(size=(T, D)).astype(np.float32))
    for din, dw in ((F32, F32), (BF16, BF16), (F32, BF16)):
        d = d32.to(din)
        want, mag, n = sums(d, ids, V)
        out = torch.full((V, D), 7.0, dtype=dw, device="cuda")
        got = ops.embedding_wgrad(d.cuda(), ids.cuda(), V, scale=0.37, out=out).cpu().double()
        sc = float(np.float32(0.37))
        tol = (n + 1) * U32 * mag * sc
        tol = tol + (U16 * (want * sc).abs() + U16 * tol if dw == BF16 else 0)
        assert ((got - want * sc).abs() <= tol).all(), (din, dw)
        assert torch.equal(ops.embedding_wgrad(d.cuda(), ids.cuda(), V, scale=0.37, out=torch.empty_like(out)), out)
        start = torch.as_tensor(rng.normal(size=(V, D)).astype(np.float32)).to(dw)
        start[::3] = -0.0
        more = ops.embedding_wgrad(d.cuda(), ids.cuda(), V, out=start.clone().cuda(), accumulate=True).cpu()
        absent = (n == 0).squeeze(1)
        bits = torch.int32 if dw == F32 else torch.int16
        assert torch.equal(more[absent].view(bits), start[absent].view(bits))
        total = start.double() + want
        tol = (n + 2) * U32 * (mag + start.double().abs())
        tol = tol + (U16 * (total.abs() + tol) if dw == BF16 else 0)
        assert ((more.double() - total).abs() <= tol).all()


@pytest.mark.parametrize("kind", ["uniform", "skewed", "one", "padded", "none"])
@pytest.mark.parametrize("T,V,D", [(8192, 1000, 512), (5003, 5000, 128), (8192, 60000, 33), (1025, 70001, 40), (8193, 5000, 100), (20001, 9000, 64), (70000, 300000, 4)])
def test_sorted_positions(ops, T, V, D, kind):
    """sorted by one workgroup and by tiles, in one pass to three; same checks"""
    test_few_positions(ops, T, V, D, kind)


@pytest.mark.parametrize("T,V,D", [(8000, 9000, 64), (20000, 9000, 64), (900, 9000, 64), (900, 600, 64)])
def test_gradient_in_a_graph(ops, T, V, D):
    rng = np.random.default_rng(T)
    ids, d = classes_of(rng, T, V, "skewed").cuda(), torch.randn(T, D, device="cuda")
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        dw = ops.embedding_wgrad(d, ids, V, 2.0)
    for k in range(4):
        ids.copy_(classes_of(np.random.default_rng(90 + k), T, V, "padded"))
        d.normal_()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(dw, ops.embedding_wgrad(d, ids, V, 2.0)), k


@pytest.mark.parametrize("T,V", [(3000, 400), (8000, 9000), (20000, 9000)])
def test_nan_stays_in_its_class(ops, T, V):
    d = torch.ones(T, 40).cuda()
    ids = (torch.arange(T) % V).cuda()
    d[5], d[T - 1] = float("nan"), float("inf")
    got = ops.embedding_wgrad(d, ids, V + 10)
    bad = torch.zeros(V + 10, dtype=torch.bool)
    bad[5] = bad[(T - 1) % V] = True
    assert torch.equal(torch.isfinite(got.cpu()).all(1), ~bad) and (got[V:] == 0).all()


def test_small_tables_of_zeros(ops):
    """sums that are -0, and an infinite scale, for rows that do not occur"""
    dout = torch.full((40, 8), -0.0).cuda()
    ids = torch.full((40,), 2).cuda()
    got = ops.embedding_wgrad(dout, ids, 4, scale=float("inf"))
    assert (got[[0, 1, 3]] == 0).all()
    old = torch.full((4, 8), -0.0).cuda()
    ops.embedding_wgrad(dout, ids, 4, out=old, accumulate=True)
    assert torch.equal(old.cpu().view(torch.int32), torch.full((4, 8), -0.0).view(torch.int32))


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_small_tables_in_a_graph(ops, dtype):
    ids = torch.randint(-1, 6, (30000,)).cuda()
    dout = torch.randn(30000, 48).to(dtype).cuda()
    eager = ops.embedding_wgrad(dout, ids, 6)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = ops.embedding_wgrad(dout, ids, 6)
    for k in range(4):
        if k == 2:
            dout.mul_(2)
            ids.copy_(ids.flip(0))
            eager = ops.embedding_wgrad(dout, ids, 6)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, eager), k
