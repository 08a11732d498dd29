"""The operators for categorical states used together: classes looked up, a layer, the class loss, gradients, the AdamW step; and the
training loop's own use of the step (engine.FlatState).  Small sizes, against float64 on the CPU."""
import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu

U = 2.0 ** -24


def plain(table, mix, ids, target, scale):
    """float64 autograd of: positions without a class are zeros; hidden = tanh(x mix); tied read-out; mean loss over rows with a class"""
    t, m = table.double().requires_grad_(True), mix.double().requires_grad_(True)
    ok = (ids >= 0) & (ids < t.shape[0])
    x = torch.where(ok.unsqueeze(-1), t[ids.clamp(0, t.shape[0] - 1)] * scale, torch.zeros(()).double())
    loss = torch.nn.functional.cross_entropy(torch.tanh(x @ m) @ t.t(), torch.where(target < 0, -100, target), ignore_index=-100)
    loss.backward()
    return loss.item(), t.grad, m.grad


def test_lookup_layer_loss_and_step_together():
    """float32, a tied table.  Every stage is float32-grade: relative error of a gradient under 1e-4 of the largest (sums of up to 300 terms,
    three products deep, each within (64 + 300) u of its magnitudes: 3 * 364 * 2^-24 = 6.5e-5)."""
    from discrete_dppm_graphs_amd import ops
    from discrete_dppm_graphs_amd.categorical import embedding, loss_func_ce
    from oracle import classes
    torch.manual_seed(0)
    V, D = 300, 64
    table, mix = torch.randn(V, D) * 0.2, torch.randn(D, D) * 0.1
    ids, target = torch.randint(-1, V, (6, 25)), torch.randint(-1, V, (6, 25))
    tw, mw = table.cuda().requires_grad_(True), mix.cuda().requires_grad_(True)
    tset = None
    m64, v64 = [np.zeros(V * D), np.zeros(D * D)], [np.zeros(V * D), np.zeros(D * D)]
    for step in (1, 2):
        want_loss, gt, gm = plain(tw.detach().cpu(), mw.detach().cpu(), ids.reshape(-1), target.reshape(-1), 2.0)
        tw.grad = mw.grad = None
        loss = loss_func_ce(torch.tanh(embedding(tw, ids.cuda(), 2.0) @ mw), tw, target.cuda())
        loss.backward()
        assert abs(loss.item() - want_loss) < 1e-5 * abs(want_loss)
        for got, want in ((tw.grad, gt), (mw.grad, gm)):
            assert (got.cpu().double() - want).abs().max() < 1e-4 * want.abs().max()
        if tset is None:
            tset = ops.TensorSet([tw.data, mw.data], [tw.grad, mw.grad], weight_decay=[0.0, 0.1])
        else:
            tset.set_grads([tw.grad, mw.grad])
        before = [tw.detach().cpu().double().numpy().ravel(), mw.detach().cpu().double().numpy().ravel()]
        norm = ops.adamw_step(tset, 1e-2, 0.9, 0.999, 1e-8, step, max_norm=0.05)
        g = [x.grad.cpu().double().numpy().ravel() for x in (tw, mw)]
        all_norm = np.sqrt(sum((x ** 2).sum() for x in g))
        assert abs(norm.item() - all_norm) <= 2 * U * all_norm
        for k, (w, decay) in enumerate(((tw, 0.0), (mw, 0.1))):
            p, m64[k], v64[k] = classes.adamw(before[k], g[k], m64[k], v64[k], 1e-2, 0.9, 0.999, 1e-8, step, decay, min(1.0, 0.05 / (all_norm + 1e-6)))
            # the update is lr times a ratio of at most 10 here, off by 64 u of it
            assert np.abs(w.detach().cpu().double().numpy().ravel() - p).max() <= 64 * U * 1e-2 * 10 + 4 * U * np.abs(p).max()


def test_bfloat16_gradients_take_the_incoming_one_unrounded():
    from discrete_dppm_graphs_amd import ops
    from discrete_dppm_graphs_amd.categorical import loss_func_ce
    x, w, y = torch.randn(70, 40).bfloat16().cuda(), torch.randn(90, 40).bfloat16().cuda(), torch.randint(0, 90, (70,)).cuda()
    _, _, dx, dw = ops.loss_ce(x, w, y)
    x.requires_grad_(True), w.requires_grad_(True)
    (loss_func_ce(x, w, y) * 0.3).backward()
    assert torch.equal(x.grad, (dx.double() * float(np.float32(0.3))).float().bfloat16())      # 8 + 24 bits are exact in float64; float32, then bfloat16
    assert torch.equal(w.grad, (dw.double() * float(np.float32(0.3))).float().bfloat16())


def test_gradients_scale_with_the_incoming_one_and_stop_where_not_wanted():
    from discrete_dppm_graphs_amd.categorical import embedding, loss_func_ce
    torch.manual_seed(1)
    x, w, y = torch.randn(40, 32).cuda().requires_grad_(True), torch.randn(50, 32).cuda().requires_grad_(True), torch.randint(0, 50, (40,)).cuda()
    gx, gw = torch.autograd.grad(loss_func_ce(x, w, y), (x, w))
    hx, hw = torch.autograd.grad(4.0 * loss_func_ce(x, w, y), (x, w))
    assert torch.equal(4.0 * gx, hx) and torch.equal(4.0 * gw, hw)
    (only,) = torch.autograd.grad(loss_func_ce(x, w.detach(), y), (x,))
    assert torch.equal(only, gx)
    assert not loss_func_ce(x.detach(), w.detach(), y).requires_grad
    ids = torch.randint(0, 50, (3, 7)).cuda()
    (ge,) = torch.autograd.grad(embedding(w, ids, 0.5)[:, ::2].sum(), (w,))            # a gradient that is not contiguous
    want = torch.zeros(50, 32).index_add_(0, ids[:, ::2].reshape(-1).cpu(), torch.full((12, 32), 0.5))
    assert torch.allclose(ge.cpu(), want)


def _model(seed=5):
    from discrete_dppm_graphs_amd.model.ppgn import Powerful
    torch.manual_seed(seed)
    return Powerful(num_layers=2, hidden=16, hidden_final=16, normalization="instance", adj_out=True, cat_output=True).cuda()


def _batch(B=5, N=14):
    rng = np.random.default_rng(2)
    up = np.triu((rng.random((B, N, N)) < 0.4).astype(np.float32), 1)
    up[:, np.arange(N - 1), np.arange(1, N)] = 1
    return torch.as_tensor(up + up.transpose(0, 2, 1)).cuda(), rng


@pytest.mark.parametrize("clip", [None, 1e-3])
def test_flat_state_trains_with_adamw(clip):
    """engine.train_step_simple with optimizer="adamw": every step's parameters are those of the float64 step from the gradients it had.
    The update is lr times a ratio of at most 1 / (1 - beta1) here, off by 64 u of it."""
    from discrete_dppm_graphs_amd import engine
    from oracle import classes
    A, rng = _batch()
    model = _model()
    state = engine.FlatState(model, lr=1e-2, weight_decay=0.05, optimizer="adamw", max_grad_norm=clip)
    m, v = np.zeros(state.numel()), np.zeros(state.numel())
    for step in (1, 2, 3):
        before = state.flat.double().cpu().numpy()
        engine.train_step_simple(model, state, A, rng.uniform(0, 0.5, size=5), 3, step)
        g = state.grad.double().cpu().numpy()
        factor = 1.0
        if clip is not None:
            norm = np.sqrt((g ** 2).sum())
            assert abs(state.grad_norm.item() - norm) <= 2 * U * norm
            factor = min(1.0, clip / (norm + 1e-6))
        p, m, v = classes.adamw(before, g, m, v, 1e-2, 0.9, 0.999, 1e-8, step, 0.05, factor)
        assert np.abs(state.flat.double().cpu().numpy() - p).max() <= 64 * U * 1e-2 * 10 + 4 * U * np.abs(p).max()


@pytest.mark.parametrize("kind", ["adamw", "adamw8"])
def test_flat_state_resumes(kind, tmp_path):
    from discrete_dppm_graphs_amd import engine
    A, _ = _batch()
    sig = np.linspace(0.1, 0.4, 5)
    one, two = _model(), _model()
    a = engine.FlatState(one, lr=1e-3, weight_decay=0.01, optimizer=kind, max_grad_norm=1.0, seed=9)
    for step in range(4):
        engine.train_step_simple(one, a, A, sig, 3, step)
        if step == 1:
            torch.save({"model": one.state_dict(), "opt": a.state_dict()}, tmp_path / "s.pth")
    saved = torch.load(tmp_path / "s.pth", map_location="cuda", weights_only=True)
    two.load_state_dict(saved["model"])
    b = engine.FlatState(two, lr=5.0, optimizer=kind, max_grad_norm=1.0)
    b.load_state_dict(saved["opt"])
    for step in (2, 3):
        engine.train_step_simple(two, b, A, sig, 3, step)
    assert torch.equal(a.flat, b.flat)
    for k in a.tensors.state:
        assert torch.equal(a.tensors.state[k].view(torch.uint8), b.tensors.state[k].view(torch.uint8))
    with pytest.raises(ValueError, match="optimizer"):
        engine.FlatState(_model(), optimizer="adam").load_state_dict(saved["opt"])


def test_flat_state_refuses():
    from discrete_dppm_graphs_amd import engine
    for kw in ({"optimizer": "sgd"}, {"max_grad_norm": 1.0}, {"optimizer": "adamw", "max_grad_norm": 0.0}):
        with pytest.raises(ValueError):
            engine.FlatState(_model(), **kw)
