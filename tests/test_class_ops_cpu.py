"""CPU checks of the operators for categorical states: what their C entry points and Python front ends refuse before anything reaches a
GPU, and the plain forms of oracle/classes.py against torch's autograd and optimizer in float64."""
import ctypes as C

import numpy as np
import pytest
import torch

from discrete_dppm_graphs_amd import ops
from discrete_dppm_graphs_amd._lib import lib
from oracle import classes


def test_adamw_oracle_is_torch_adamw():
    rng = np.random.default_rng(0)
    p = torch.as_tensor(rng.normal(size=50))
    t = p.clone().requires_grad_(True)
    opt = torch.optim.AdamW([t], lr=1e-2, betas=(0.9, 0.999), eps=1e-8, weight_decay=0.1)
    q, m, v = p.numpy(), np.zeros(50), np.zeros(50)
    for step in range(1, 5):
        g = rng.normal(size=50)
        t.grad = torch.as_tensor(g)
        opt.step()
        q, m, v = classes.adamw(q, g, m, v, 1e-2, 0.9, 0.999, 1e-8, step, 0.1)
    np.testing.assert_allclose(q, t.detach().numpy(), rtol=1e-12)


def test_e4m3_neighbours_hold_the_value():
    x = np.random.default_rng(1).normal(size=1000) * np.repeat([1e-20, 1e-3, 1.0, 1e20], 250)
    scale, low, high, part = classes.e4m3_neighbours(x)
    assert (np.abs(low) <= np.abs(x) * (1 + 1e-12)).all() and (np.abs(x) <= np.abs(high)).all() and (part >= 0).all() and (part < 1).all()
    s = torch.as_tensor(np.repeat(scale, 256)[:1000])
    for y in (low, high):
        q = (torch.as_tensor(np.abs(y)) / s).clamp(max=448.0)      # above a block's largest value there is no neighbour
        assert torch.equal(q.float().to(torch.float8_e4m3fn).float(), q.float())


def test_adamw_entry_refuses():
    one = C.c_void_p(16)      # refused before any pointer is read
    good = dict(table=one, chunks=one, n=1, bf=0, bits=32, lr=1e-3, b1=0.9, b2=0.999, eps=1e-8, step=1, gs=1.0, mn=0.0, seed=0, norm=None, ws=None, wb=0, st=None)
    for bad in ({"table": None}, {"chunks": None}, {"n": -1}, {"bits": 4}, {"b1": 1.0}, {"b2": -0.1}, {"eps": -1.0}, {"step": 0}, {"b1": float("nan")},
                {"mn": 1.0}, {"mn": 1.0, "norm": one, "ws": one, "wb": 64}):
        assert lib.dppm_adamw_step(*{**good, **bad}.values()) == -1, bad
    assert lib.dppm_adamw_chunk() % 256 == 0 and lib.dppm_adamw_workspace_bytes() > 0


def test_front_ends_refuse_cpu_tensors():
    with pytest.raises(RuntimeError, match="no CPU fallback"):
        ops.TensorSet([torch.zeros(4)], [torch.zeros(4)])


def test_embedding_oracle_is_torch_embedding():
    torch.manual_seed(2)
    w = torch.randn(7, 3, dtype=torch.float64, requires_grad=True)
    ids = torch.randint(0, 7, (4, 5))
    d = torch.randn(4, 5, 3, dtype=torch.float64)
    y = torch.nn.functional.embedding(ids, w) * 1.5
    y.backward(d)
    assert torch.allclose(classes.embedding(w.detach(), ids, 1.5), y.detach()) and torch.allclose(classes.embedding_wgrad(d, ids, 7, 1.5), w.grad)
    assert (classes.embedding(w.detach(), torch.tensor([-1, 7]), 1.5) == 0).all()


def test_embedding_entries_refuse():
    one = C.c_void_p(16)
    for bad in ((-1, 5, 4), (3, 0, 4), (3, 5, 0), (1 << 31, 5, 4), (3, 1 << 31, 4), (3, 5, 1 << 24)):
        assert lib.dppm_embedding_fwd(one, 0, one, 1.0, one, *bad, None) == -1
        assert lib.dppm_embedding_wgrad(one, 0, one, 1.0, one, 0, 0, *bad, one, 1 << 40, None) == -1
        assert lib.dppm_embedding_wgrad_workspace_bytes(*bad) == 0
    for k in range(3):
        ptrs = [one, one, one]
        ptrs[k] = None
        assert lib.dppm_embedding_fwd(ptrs[0], 0, ptrs[1], 1.0, ptrs[2], 3, 5, 4, None) == -1
        assert lib.dppm_embedding_wgrad(ptrs[0], 0, ptrs[1], 1.0, ptrs[2], 0, 0, 3, 5, 4, one, 1 << 40, None) == -1
    need = lib.dppm_embedding_wgrad_workspace_bytes(3, 5, 4)
    assert lib.dppm_embedding_wgrad(one, 0, one, 1.0, one, 0, 0, 3, 5, 4, one, need - 1, None) == -1
    assert lib.dppm_embedding_wgrad(one, 0, one, 1.0, one, 0, 0, 3, 5, 4, C.c_void_p(8), need, None) == -1


def test_cross_entropy_oracle_is_torch_cross_entropy():
    torch.manual_seed(3)
    x, w = torch.randn(9, 4, dtype=torch.float64, requires_grad=True), torch.randn(6, 4, dtype=torch.float64, requires_grad=True)
    target = torch.tensor([0, 5, 3, -100, 2, 2, -100, 1, 4])
    loss = torch.nn.functional.cross_entropy(x @ w.t(), target, ignore_index=-100)
    loss.backward()
    got = classes.cross_entropy(x.detach(), w.detach(), target)
    assert torch.allclose(got[0], loss.detach()) and torch.allclose(got[2], x.grad) and torch.allclose(got[3], w.grad)
    weighted = classes.cross_entropy(x.detach(), w.detach(), target, torch.arange(9.0), 5.0)
    per_row = torch.nn.functional.cross_entropy(x @ w.t(), target, ignore_index=-100, reduction="none")
    g = torch.autograd.grad((per_row * torch.arange(9.0)).sum() / 5.0, (x, w))
    assert torch.allclose(weighted[2], g[0]) and torch.allclose(weighted[3], g[1])


def test_loss_ce_entry_refuses():
    one = C.c_void_p(16)
    good = dict(x=one, w=one, bf=1, target=one, rw=None, denom=0.0, T=4, V=5, D=8, loss=one, row=one, dx=one, dw=one, ws=one, n=1 << 40, st=None)
    for bad in ({"x": None}, {"w": None}, {"target": None}, {"loss": None}, {"row": None}, {"ws": None}, {"dx": None}, {"dw": None}, {"T": 0}, {"T": -1},
                {"T": 1 << 30}, {"V": 0}, {"V": (1 << 23) + 1}, {"D": 0}, {"D": (1 << 16) + 1}, {"denom": -1.0}, {"denom": float("nan")}, {"denom": 1e-50}, {"denom": float("inf")}, {"ws": C.c_void_p(8)}):
        assert lib.dppm_loss_ce_fwd_bwd(*{**good, **bad}.values()) == -1, bad
    need = lib.dppm_loss_ce_workspace_bytes(4, 5, 8, 1, 1)
    assert need > lib.dppm_loss_ce_workspace_bytes(4, 5, 8, 1, 0) > 0
    assert lib.dppm_loss_ce_fwd_bwd(*{**good, "n": 64}.values()) == -1
    # beside a copy of x, 16 bytes of partial loss for 32 rows and 4 of a count for 4096, memory is that of one block of rows, whatever their number
    many, more = lib.dppm_loss_ce_workspace_bytes(1 << 16, 1 << 17, 1024, 1, 1), lib.dppm_loss_ce_workspace_bytes(1 << 17, 1 << 17, 1024, 1, 1)
    assert more - many <= (1 << 16) * 1088 * 2 + (1 << 16) // 32 * 16 + (1 << 16) // 4096 * 4 + 4096 and more < 8 << 30


def test_optimizer_options_come_from_the_configuration():
    from discrete_dppm_graphs_amd import engine
    from discrete_dppm_graphs_amd.utils.easydict import EasyDict
    assert engine.optimizer_options(EasyDict(train=dict(lr_init=0.1))) == {"optimizer": "adam", "max_grad_norm": None, "seed": 0}
    assert engine.optimizer_options(EasyDict(seed=7, train=dict(optimizer="adamw8", max_grad_norm=1.0))) == {"optimizer": "adamw8", "max_grad_norm": 1.0, "seed": 7}


def test_differentiable_fronts_refuse_cpu_tensors():
    from discrete_dppm_graphs_amd.categorical import embedding, loss_func_ce
    with pytest.raises(RuntimeError, match="no CPU fallback"):
        embedding(torch.zeros(4, 2), torch.zeros(3, dtype=torch.int64))
    with pytest.raises(RuntimeError, match="no CPU fallback"):
        loss_func_ce(torch.zeros(3, 2), torch.zeros(4, 2), torch.zeros(3, dtype=torch.int64))
