"""GPU parity of dppm_adamw_step (ops.TensorSet, ops.adamw_step) against the float64 form of oracle/classes.py.

Tolerances.  A float32 operation is off by at most u = 2^-24 of its result.  m' is three operations on operands that are exact here:
4 u of |m| + |g|.  v' is four: 6 u of v'.  The update is lr * (m' / (root / c + eps)): its own roundings add under 12 u to the 10 u of m'
and root, so 32 u of its size, plus 2 u of |p| for the decay and the subtraction; |update| is bounded below by its float64 value and
m's error by its operands, hence the `size` terms."""
import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
HYPER = dict(lr=1e-3, beta1=0.9, beta2=0.999, eps=1e-8)


@pytest.fixture(scope="module")
def ops():
    from discrete_dppm_graphs_amd import ops
    return ops


@pytest.fixture(scope="module")
def ref():
    from oracle import classes
    return classes


def make(rng, shapes, grad_dtype=torch.float32, copies=False):
    ps = [torch.as_tensor(rng.normal(size=s).astype(np.float32) * 0.1).cuda() for s in shapes]
    gs = [torch.as_tensor((rng.normal(size=s) * 10.0 ** rng.uniform(-4, 0)).astype(np.float32)).to(grad_dtype).cuda() for s in shapes]
    cs = [torch.full(s, 7.0, dtype=torch.bfloat16, device="cuda") for s in shapes] if copies else None
    return ps, gs, cs


def np64(t):
    return t.detach().double().cpu().numpy().reshape(-1)


def cut(tset, name, i):
    o = tset.offsets[i]
    return np64(tset.state[name][o:o + tset.params[i].numel()].float())


def moments8(tset, i):
    """m and r as the set holds them"""
    o, n = tset.offsets[i], tset.params[i].numel()
    out = []
    for k in ("exp_avg", "exp_avg_root"):
        s = np.repeat(np64(tset.state[k + "_scale"]), 256)[o:o + n]
        out.append(cut(tset, k, i) * s)
    return out


def check_step(ref, tset, before, gs, step, factor=1.0, hyper=HYPER):
    """parameters (and 32-bit moments) of every tensor after a step from `before` = [(p, m, v)]"""
    h = hyper
    for i, (p0, m0, v0) in enumerate(before):
        g = np64(gs[i])
        p, m, v = ref.adamw(p0, g, m0, v0, h["lr"], h["beta1"], h["beta2"], h["eps"], step, tset.weight_decay[i], factor)
        denom = np.sqrt(v / (1 - h["beta2"] ** step)) + h["eps"]
        size = h["lr"] / (1 - h["beta1"] ** step) * (np.abs(m0) + np.abs(g * factor) * 0.2) / denom
        np.testing.assert_array_less(np.abs(np64(tset.params[i]) - p), 32 * U * size + 3 * U * np.abs(p0) + 1e-30, err_msg=f"param {i}")
        if tset.state_bits == 32:
            np.testing.assert_array_less(np.abs(cut(tset, "exp_avg", i) - m), 6 * U * (np.abs(m0) + np.abs(g * factor)) + 1e-37)
            np.testing.assert_array_less(np.abs(cut(tset, "exp_avg_sq", i) - v), 10 * U * v + 1e-37)
        if tset.copies[i] is not None:
            assert torch.equal(tset.copies[i], tset.params[i].bfloat16())


SHAPES = {
    "one": [(1,)],
    "odd": [(3,), (255,), (256,), (257,), (1021,), (4095,), (4096,), (4097,)],
    "net": [(32, 2), (32,), (32, 32), (32,), (32, 64), (32,), (32, 194), (1, 32), (1,)],
    "empty tensor": [(5,), (0,), (7, 3)],
    "wide": [(501, 501), (501,), (1002, 501)],
}


@pytest.mark.parametrize("grad_dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("name", list(SHAPES))
def test_steps_32(ops, ref, name, grad_dtype):
    rng = np.random.default_rng(len(name))
    ps, gs, cs = make(rng, SHAPES[name], grad_dtype, copies=True)
    decay = [0.1 * (i % 2) for i in range(len(ps))]
    ts = ops.TensorSet(ps, gs, copies=cs, weight_decay=decay)
    for step in (1, 2, 3):
        before = [(np64(p), cut(ts, "exp_avg", i), cut(ts, "exp_avg_sq", i)) for i, p in enumerate(ps)]
        assert ops.adamw_step(ts, step=step, **HYPER) is None
        check_step(ref, ts, before, gs, step)


@pytest.mark.parametrize("grad_dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("name", list(SHAPES))
def test_steps_8(ops, ref, name, grad_dtype):
    rng = np.random.default_rng(100 + len(name))
    ps, gs, cs = make(rng, SHAPES[name], grad_dtype, copies=True)
    ts = ops.TensorSet(ps, gs, copies=cs, weight_decay=0.05, state_bits=8)
    seed = 0x123456789ABCDEF
    for step in (1, 2, 5):
        held = [moments8(ts, i) for i in range(len(ps))]
        before = [(np64(p), m, r * r) for p, (m, r) in zip(ps, held)]
        ops.adamw_step(ts, step=step, seed=seed, **HYPER)
        check_step(ref, ts, before, gs, step)
        for i, (p0, m0, v0) in enumerate(before):
            if p0.size == 0:
                continue
            g = np64(gs[i])
            _, m, v = ref.adamw(p0, g, m0, v0, step=step, **HYPER)
            for x, got, k, r16 in ((m, moments8(ts, i)[0], "exp_avg", 0), (np.sqrt(v), moments8(ts, i)[1], "exp_avg_root", 1)):
                scale, low, high, part = ref.e4m3_neighbours(x)
                have = np64(ts.state[k + "_scale"][ts.offsets[i] // 256:][:scale.size])
                np.testing.assert_allclose(have, scale, rtol=64 * U)      # m' itself is off by up to 6 u of its operands
                r = ref.round_bits(x.size, i, step, seed)[r16]
                want = np.where(part + r / 65536.0 >= 1.0, high, low)
                # where part + r/65536 is within the float32 error of 1, or of a grid value, either neighbour is right
                near = (np.abs(part + r / 65536.0 - 1.0) < 1e-4) | (part < 1e-4) | (part > 1 - 1e-4)
                tol = 1e-5 * np.abs(want) + 1e-30
                wrong = (np.abs(got - want) > tol) & ~near
                assert not wrong.any(), (k, i, np.flatnonzero(wrong)[:5], got[wrong][:5], want[wrong][:5])
                ulp = np.abs(high - low)
                assert (np.abs(got - want)[near] <= 1.001 * ulp[near] * 2 + tol[near]).all()


def test_padding_of_8_bit_state_stays_zero(ops):
    rng = np.random.default_rng(5)
    ps, gs, _ = make(rng, [(5,), (300,)])
    ts = ops.TensorSet(ps, gs, state_bits=8)
    for step in (1, 2, 3):
        ops.adamw_step(ts, step=step, seed=step, **HYPER)
    for k in ("exp_avg", "exp_avg_root"):
        x = ts.state[k].float()
        assert (x[5:256] == 0).all() and (x[256 + 300:] == 0).all()


@pytest.mark.parametrize("bits", [8, 32])
@pytest.mark.parametrize("max_norm", [1e-3, 1e6])
def test_clipping(ops, ref, bits, max_norm):
    rng = np.random.default_rng(7)
    ps, gs, _ = make(rng, [(1000, 37), (9,), (5003,)], torch.bfloat16)
    ts = ops.TensorSet(ps, gs, state_bits=bits)
    before = [(np64(p), np.zeros(p.numel()), np.zeros(p.numel())) for p in ps]
    norm = ops.adamw_step(ts, step=1, max_norm=max_norm, grad_scale=0.5, **HYPER)
    want = 0.5 * np.sqrt(sum((np64(g) ** 2).sum() for g in gs))
    assert abs(norm.item() - want) <= 2 * U * want
    check_step(ref, ts, before, gs, 1, factor=0.5 * min(1.0, max_norm / (want + 1e-6)))


@pytest.mark.parametrize("bits", [8, 32])
@pytest.mark.parametrize("bad", [float("inf"), float("-inf"), float("nan")])
def test_step_with_a_bad_norm_changes_nothing(ops, bits, bad):
    rng = np.random.default_rng(8)
    ps, gs, cs = make(rng, [(70, 9), (5000,)], copies=True)
    ts = ops.TensorSet(ps, gs, copies=cs, state_bits=bits)
    ops.adamw_step(ts, step=1, max_norm=1.0, **HYPER)
    gs[1][4321] = bad
    before = [t.clone() for t in (*ps, *cs, *ts.state.values())]
    norm = ops.adamw_step(ts, step=2, max_norm=1.0, **HYPER)
    assert not np.isfinite(norm.item())
    for a, b in zip(before, (*ps, *cs, *ts.state.values())):
        assert torch.equal(a.view(torch.uint8), b.view(torch.uint8))


def test_nan_without_clipping_reaches_its_block_only(ops):
    p, g = torch.ones(1024, device="cuda"), torch.ones(1024, device="cuda")
    g[300] = float("nan")
    ts = ops.TensorSet([p], [g], state_bits=8)
    ops.adamw_step(ts, step=1, **HYPER)
    assert torch.isnan(p).nonzero().flatten().tolist() == [300]
    g.fill_(1.0)
    ops.adamw_step(ts, step=2, **HYPER)
    assert torch.isnan(p).nonzero().flatten().tolist() == list(range(256, 512))


def test_zero_gradients_and_tiny_blocks(ops):
    p, g = torch.ones(600, device="cuda"), torch.zeros(600, device="cuda")
    g[256:512] = 1e-36                                        # its block's moments are under what a scale can hold: kept as zero
    ts = ops.TensorSet([p], [g], state_bits=8)
    ops.adamw_step(ts, step=1, **HYPER)
    assert torch.isfinite(p).all()
    for t in ts.state.values():
        assert torch.isfinite(t.float()).all() and (t.float()[:1] == 0).all()


def test_8_bit_second_moment_falls_and_follows_in_the_mean(ops):
    """From r = 1 with gradients of 0.5: v falls by a factor 0.999 + 0.001 * 0.25 / v in a step, far under half a step of e4m3.
    The mean over 4096 values of r after 200 steps is within 1 % of the recursion (each value's rounding noise is at most
    sqrt(200 * 0.0005 * 0.0625) = 0.08, the mean's 0.0013)."""
    n = 4096
    p, g = torch.zeros(n, device="cuda"), torch.full((n,), 0.5, device="cuda")
    ts = ops.TensorSet([p], [g], state_bits=8)
    ts.state["exp_avg_root"].copy_(torch.full((n,), 448.0, device="cuda").to(torch.float8_e4m3fn))
    ts.state["exp_avg_root_scale"].fill_(1.0 / 448.0)
    v = 1.0
    for step in range(1, 201):
        ops.adamw_step(ts, step=step, seed=3, **HYPER)
        v = 0.999 * v + 0.001 * 0.25
    r = ts.state["exp_avg_root"].float() * ts.state["exp_avg_root_scale"].repeat_interleave(256)
    assert abs(r.mean().item() - np.sqrt(v)) < 0.01 * np.sqrt(v)


@pytest.mark.parametrize("bits", [8, 32])
def test_many_tensors_equal_one_at_a_time_and_calls_repeat(ops, bits):
    rng = np.random.default_rng(9)
    shapes = [(int(n),) for n in rng.integers(1, 9000, size=40)]
    outs = []
    for _ in range(2):
        rng = np.random.default_rng(10)
        ps, gs, _ = make(rng, shapes)
        ts = ops.TensorSet(ps, gs, state_bits=bits)
        for step in (1, 2):
            norm = ops.adamw_step(ts, step=step, max_norm=0.5, seed=11, **HYPER)
        outs.append([*ps, norm.view(1), *ts.state.values()])
    assert all(torch.equal(a.view(torch.uint8), b.view(torch.uint8)) for a, b in zip(*outs))
    ps, gs, _ = make(np.random.default_rng(10), shapes)
    ts = ops.TensorSet(ps, gs, state_bits=bits)
    ops.adamw_step(ts, step=1, **HYPER)
    alone, gs2, _ = make(np.random.default_rng(10), shapes)
    for p, g in zip(alone, gs2):
        ops.adamw_step(ops.TensorSet([p], [g], state_bits=bits), step=1, **HYPER)
    assert all(torch.equal(a, b) for a, b in zip(ps, alone))      # the first step's parameters do not depend on the rounding


def test_side_stream_graph_replay_and_new_gradients(ops):
    ps, gs, _ = make(np.random.default_rng(12), [(1000,), (77, 3)])
    ts = ops.TensorSet(ps, gs, state_bits=8)
    keep = [t.clone() for t in (*ps, *ts.state.values())]
    ops.adamw_step(ts, step=1, max_norm=1.0, **HYPER)
    want = [t.clone() for t in (*ps, *ts.state.values())]

    def reset():
        for t, k in zip((*ps, *ts.state.values()), keep):
            t.copy_(k)

    reset()
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        ops.adamw_step(ts, step=1, max_norm=1.0, **HYPER)
    torch.cuda.current_stream().wait_stream(s)
    assert all(torch.equal(a.view(torch.uint8), b.view(torch.uint8)) for a, b in zip(want, (*ps, *ts.state.values())))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        norm = ops.adamw_step(ts, step=1, max_norm=1.0, **HYPER)
    for _ in range(3):
        reset()
        graph.replay()
        torch.cuda.synchronize()
        assert norm.item() > 0
        assert all(torch.equal(a.view(torch.uint8), b.view(torch.uint8)) for a, b in zip(want, (*ps, *ts.state.values())))
    reset()
    ts.set_grads([g.bfloat16() for g in gs])
    before = [p.clone() for p in ps]
    ops.adamw_step(ts, step=1, **HYPER)
    assert not any(torch.equal(a, b) for a, b in zip(before, ps))


def test_refusals(ops):
    p, g = torch.zeros(64, device="cuda"), torch.zeros(64, device="cuda")
    for args, kw in ((([], []), {}), (([p], [g[:32]]), {}), (([p], [g, g]), {}), (([p, p], [g, g]), {}), (([p, p[4:]], [g, g[4:]]), {}),
                     (([p], [p]), {}), (([p[:32]], [p[16:48]]), {}), (([p[:32], g], [p[32:], g[:64].clone()[:64]]), {"copies": [None, g.bfloat16()[:8]]}),
                     (([p], [g]), {"state_bits": 16}), (([p], [g]), {"weight_decay": [0.1, 0.2]}), (([p[1:]], [g[1:]]), {}),
                     (([p], [g]), {"copies": [torch.zeros(3, device="cuda", dtype=torch.bfloat16)]}),
                     (([p], [g]), {"state": {"exp_avg": p}}), (([p.view(8, 8).t()], [g]), {})):
        with pytest.raises(ValueError):
            ops.TensorSet(*args, **kw)
    for args, kw in ((([p.double()], [g]), {}), (([p], [g.half()]), {}), (([p], [g]), {"copies": [p]}), (([p], [3.0]), {})):
        with pytest.raises(TypeError):
            ops.TensorSet(*args, **kw)
    ts = ops.TensorSet([p], [g])
    with pytest.raises(RuntimeError, match="step=0"):
        ops.adamw_step(ts, step=0, **HYPER)
    with pytest.raises(ValueError):
        ops.adamw_step(ts, step=1, max_norm=0.0, **HYPER)
    with pytest.raises(RuntimeError, match="beta1"):
        ops.adamw_step(ts, 1e-3, 1.0, 0.999, 1e-8, 1)
    with pytest.raises(TypeError):
        ops.adamw_step([p], step=1, **HYPER)
    torch.cuda.synchronize()
