"""Plain float64 forms of the operators for categorical states (TEST INFRASTRUCTURE, see oracle/__init__.py): embedding and its
gradient, softmax cross entropy over classes and its gradients, the AdamW step with float32 or 8-bit moments.  No counterpart in the
reference; written from the formulas."""
import numpy as np
import torch

from .philox import philox4x32_10

BLOCK = 256


def embedding(weight, ids, scale=1.0):
    w = weight.double() * scale
    out = torch.zeros(ids.numel(), w.shape[1], dtype=torch.float64)
    for t, i in enumerate(ids.reshape(-1).tolist()):
        if 0 <= i < w.shape[0]:
            out[t] = w[i]
    return out.view(*ids.shape, w.shape[1])


def embedding_wgrad(dout, ids, rows, scale=1.0):
    out = torch.zeros(rows, dout.shape[-1], dtype=torch.float64)
    for t, i in enumerate(ids.reshape(-1).tolist()):
        if 0 <= i < rows:
            out[i] += dout.reshape(-1, dout.shape[-1])[t].double()
    return out * scale


def cross_entropy(x, weight, target, row_weight=None, denom=None):
    """-> (loss, row_loss, dx, dweight, and the rows' softmax and d, the gradient of the scores) in float64."""
    x, w = x.double(), weight.double()
    T, V = x.shape[0], w.shape[0]
    ok = (target >= 0) & (target < V)
    n = float(ok.sum().clamp(min=1)) if denom is None else float(denom)
    share = torch.where(ok, torch.ones(T, dtype=torch.float64) if row_weight is None else row_weight.double(), torch.zeros(T, dtype=torch.float64)) / n
    s = x @ w.t()
    s = torch.where(ok.unsqueeze(1), s, torch.zeros((), dtype=torch.float64))      # a row without a class does not count, whatever it holds
    x = torch.where(ok.unsqueeze(1), x, torch.zeros((), dtype=torch.float64))
    lse = torch.logsumexp(s, 1, keepdim=True)
    at = target.clamp(0, V - 1).unsqueeze(1)
    row_loss = torch.where(ok, (lse - s.gather(1, at)).squeeze(1), torch.zeros((), dtype=torch.float64))
    p = (s - lse).exp()
    d = p.clone()
    d.scatter_add_(1, at, torch.full((T, 1), -1.0, dtype=torch.float64))
    d = torch.where(ok.unsqueeze(1), d * share.unsqueeze(1), torch.zeros((), dtype=torch.float64))
    return (row_loss * share).sum(), row_loss, d @ w, d.t() @ x, p, d


def round_bits(n, tensor, step, seed):
    """The two 16-bit numbers of every value of tensor number `tensor`: (for m, for sqrt(v))."""
    g = np.arange((n + 3) // 4, dtype=np.uint64)
    key = (np.uint32(seed & 0xFFFFFFFF), np.uint32((seed >> 32) & 0xFFFFFFFF))
    w = np.stack(philox4x32_10(((g & np.uint64(0xFFFFFFFF)).astype(np.uint32), np.uint32(tensor), (g >> np.uint64(32)).astype(np.uint32), np.uint32(step)), key), 1)
    w = w.reshape(-1)[:n]
    return (w >> 16).astype(np.float64), (w & 0xFFFF).astype(np.float64)


def adamw(p, g, m, v, lr, beta1, beta2, eps, step, decay=0.0, factor=1.0):
    """float64 arrays -> (p, m, v) after the step; factor: what the gradient is multiplied by."""
    g = g * factor
    m = beta1 * m + (1 - beta1) * g
    v = beta2 * v + (1 - beta2) * g * g
    p = p * (1 - lr * decay) - lr * (m / (1 - beta1 ** step)) / (np.sqrt(v / (1 - beta2 ** step)) + eps)
    return p, m, v


def e4m3_neighbours(x):
    """x [n] float64 -> (scales per 256, lower, upper grid values, position between them): what x is rounded to at random."""
    n = x.size
    pad = np.zeros((n + BLOCK - 1) // BLOCK * BLOCK)
    pad[:n] = np.abs(x)
    top = pad.reshape(-1, BLOCK).max(1)
    scale = np.where(top > 1e-30, top / 448.0, 0.0)
    s = np.repeat(scale, BLOCK)[:n]
    y = np.abs(x) / np.where(s > 0, s, 1.0) * (s > 0)
    ulp = 2.0 ** (np.floor(np.log2(np.maximum(y, 2.0 ** -6))) - 3)
    low = np.floor(y / ulp) * ulp
    return scale, np.sign(x) * low * s, np.sign(x) * (low + ulp) * s, y / ulp - np.floor(y / ulp)
