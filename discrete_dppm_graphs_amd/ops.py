"""Torch-tensor front end of the C-ABI (include/dppm_hip.h).  torch is used only as the owner of device memory and
of the current HIP stream; every function validates its operands on the host (shape, dtype, device, contiguity)
before a raw pointer reaches a kernel, and raises RuntimeError on a non-zero status.  No CPU path exists."""
import bisect
import contextlib
import ctypes as C

import numpy as np
import torch

from ._lib import PRECISIONS, PpgnLayer, PpgnParams, check, lib


def _stream():
    return C.c_void_p(torch.cuda.current_stream().cuda_stream)


def _launch(index, fn, name, *args):
    """fn(*args, stream) with the current stream of GPU `index`, which is made the current device if it is not."""
    if torch._C._cuda_getDevice() == index:
        rc = fn(*args, torch._C._cuda_getCurrentRawStream(index))
    else:
        with torch.cuda.device(index):
            rc = fn(*args, torch._C._cuda_getCurrentRawStream(index))
    if rc != 0:
        check(rc, name)


def _chk(t, name, shape=None, dtype=torch.float32):
    if not isinstance(t, torch.Tensor):
        raise TypeError(f"{name}: expected a torch.Tensor, got {type(t)}")
    if not t.is_cuda:
        raise RuntimeError(f"{name}: tensor is on {t.device}; the DDPM hot path runs on the GPU only (no CPU fallback)")
    if t.dtype != dtype:
        raise TypeError(f"{name}: dtype {t.dtype}, expected {dtype}")
    if not t.is_contiguous():
        raise ValueError(f"{name}: tensor must be contiguous")
    if shape is not None and tuple(t.shape) != tuple(shape):
        raise ValueError(f"{name}: shape {tuple(t.shape)}, expected {tuple(shape)}")
    return t


def _ptr(t):
    return C.c_void_p(t.data_ptr()) if t is not None else C.c_void_p(0)


def _rng_args(U, seed, graph_id0, offset, shape):
    if U is not None:
        _chk(U, "U", shape)
    return _ptr(U), C.c_uint64(int(seed) & (2 ** 64 - 1)), C.c_uint32(int(graph_id0)), C.c_uint32(int(offset))


def _f32c(t):
    return t.to(torch.float32).contiguous()


def _prec(precision):
    """'f32' | 'bf16x3' | 'bf16' | 'f32x6' -> DPPM_PREC_* (include/dppm_hip.h)"""
    try:
        return PRECISIONS[precision]
    except KeyError:
        raise ValueError(f"precision {precision!r}: expected one of {sorted(PRECISIONS)}") from None


def generate_mask(flags):
    flags = _chk(_f32c(flags), "flags")
    B, N = flags.shape
    mask = torch.empty(B, N, N, device=flags.device, dtype=torch.float32)
    check(lib.dppm_generate_mask(_ptr(flags), B, N, _ptr(mask), _stream()), "dppm_generate_mask")
    return mask


def _sigma_args(sigma, B, device):
    """python float -> scalar path; sequence / array / tensor of B doubles -> device array."""
    if isinstance(sigma, (float, int, np.floating)):
        return None, float(sigma)
    s = torch.as_tensor(np.asarray(sigma, dtype=np.float64) if not isinstance(sigma, torch.Tensor) else sigma)
    s = s.to(device=device, dtype=torch.float64).contiguous().view(-1)
    if s.numel() != B:
        raise ValueError(f"sigma: {s.numel()} values for a batch of {B} graphs")
    return s, 0.0


def edgeflip(A0, flags, sigma, U=None, seed=0, graph_id0=0, offset=0, want_target=True, out=None):
    """q(A_t|A_0): returns (A_t, target).  sigma: python float (all graphs) or B values (one per graph)."""
    A0 = _chk(A0, "A0")
    B, N, _ = A0.shape
    flags = _chk(flags, "flags", (B, N))
    sig_dev, sig_scalar = _sigma_args(sigma, B, A0.device)
    A_t = out if out is not None else torch.empty_like(A0)
    _chk(A_t, "out", (B, N, N))
    target = torch.empty_like(A0) if want_target else None
    u, sd, g0, off = _rng_args(U, seed, graph_id0, offset, (B, N, N))
    check(lib.dppm_edgeflip_fwd(_ptr(A0), _ptr(flags), _ptr(sig_dev), C.c_double(sig_scalar), u, sd, g0, off, B, N,
                                _ptr(A_t), _ptr(target), _stream()), "dppm_edgeflip_fwd")
    return A_t, target


def init_xT(flags, U=None, seed=0, graph_id0=0, offset=0):
    flags = _chk(flags, "flags")
    B, N = flags.shape
    out = torch.empty(B, N, N, device=flags.device, dtype=torch.float32)
    u, sd, g0, off = _rng_args(U, seed, graph_id0, offset, (B, N, N))
    check(lib.dppm_init_xT(_ptr(flags), u, sd, g0, off, B, N, _ptr(out), _stream()), "dppm_init_xT")
    return out


def reverse_step_simple(A_t, logits, flags, U=None, seed=0, graph_id0=0, offset=0, is_probs=False, out=None):
    A_t = _chk(A_t, "A_t")
    B, N, _ = A_t.shape
    logits = _chk(logits, "logits", (B, N, N))
    flags = _chk(flags, "flags", (B, N))
    out = out if out is not None else torch.empty_like(A_t)
    _chk(out, "out", (B, N, N))
    u, sd, g0, off = _rng_args(U, seed, graph_id0, offset, (B, N, N))
    check(lib.dppm_reverse_step_simple(_ptr(A_t), _ptr(logits), int(bool(is_probs)), _ptr(flags), u, sd, g0, off, B, N,
                                       _ptr(out), _stream()), "dppm_reverse_step_simple")
    return out


def reverse_step_vlb(A_t, logits, flags, sigmatilde_t, beta_t, sigmatilde_t1, U=None, seed=0, graph_id0=0, offset=0,
                     is_probs=False, out=None):
    A_t = _chk(A_t, "A_t")
    B, N, _ = A_t.shape
    logits = _chk(logits, "logits", (B, N, N))
    flags = _chk(flags, "flags", (B, N))
    out = out if out is not None else torch.empty_like(A_t)
    _chk(out, "out", (B, N, N))
    u, sd, g0, off = _rng_args(U, seed, graph_id0, offset, (B, N, N))
    check(lib.dppm_reverse_step_vlb(_ptr(A_t), _ptr(logits), int(bool(is_probs)), _ptr(flags), C.c_double(sigmatilde_t),
                                    C.c_double(beta_t), C.c_double(sigmatilde_t1), u, sd, g0, off, B, N, _ptr(out),
                                    _stream()), "dppm_reverse_step_vlb")
    return out


def _loss_ws(B, N, device):
    n = lib.dppm_loss_workspace_bytes(B, N)
    return torch.empty(max(n, 8) // 8, device=device, dtype=torch.float64), n


def loss_bce(score, target, sigmas, mask, B_global=None, want_grad=True):
    """returns (loss [float64 0-d tensor on device], dscore or None)."""
    score = _chk(score, "score")
    B, N, _ = score.shape
    target = _chk(target, "target", (B, N, N))
    mask = _chk(mask, "mask", (B, N, N))
    sig_dev, _ = _sigma_args(list(sigmas) if not isinstance(sigmas, torch.Tensor) else sigmas, B, score.device)
    ws, nbytes = _loss_ws(B, N, score.device)
    loss = torch.empty((), device=score.device, dtype=torch.float64)
    dscore = torch.empty_like(score) if want_grad else None
    check(lib.dppm_loss_bce_fwd_bwd(_ptr(score), _ptr(target), _ptr(sig_dev), _ptr(mask), B, N, int(B_global or B), _ptr(loss),
                                    _ptr(dscore), _ptr(ws), C.c_size_t(nbytes), _stream()), "dppm_loss_bce_fwd_bwd")
    return loss, dscore


def loss_vlb(score, A_t, A_0, sched, mask, want_grad=True):
    """sched: [B,3] doubles (sigmatilde_t, beta_t, sigmatilde_{t-1}).  returns (loss float32 0-d, dscore or None)."""
    score = _chk(score, "score")
    B, N, _ = score.shape
    A_t = _chk(A_t, "A_t", (B, N, N))
    A_0 = _chk(A_0, "A_0", (B, N, N))
    mask = _chk(mask, "mask", (B, N, N))
    sched = torch.as_tensor(np.asarray(sched, dtype=np.float64) if not isinstance(sched, torch.Tensor) else sched)
    sched = _chk(sched.to(device=score.device, dtype=torch.float64).contiguous(), "sched", (B, 3), torch.float64)
    ws, nbytes = _loss_ws(B, N, score.device)
    loss = torch.empty((), device=score.device, dtype=torch.float32)
    dscore = torch.empty_like(score) if want_grad else None
    check(lib.dppm_loss_vlb_fwd_bwd(_ptr(score), _ptr(A_t), _ptr(A_0), _ptr(sched), _ptr(mask), B, N, _ptr(loss), _ptr(dscore),
                                    _ptr(ws), C.c_size_t(nbytes), _stream()), "dppm_loss_vlb_fwd_bwd")
    return loss, dscore


# ------------------------------------------------------------------------------------------------- PPGN
LAYER_FIELDS = (("m1_w0", "m1.0.weight"), ("m1_b0", "m1.0.bias"), ("m1_w1", "m1.2.weight"), ("m1_b1", "m1.2.bias"),
                ("m2_w0", "m2.0.weight"), ("m2_b0", "m2.0.bias"), ("m2_w1", "m2.2.weight"), ("m2_b1", "m2.2.bias"),
                ("m4_w", "m4.0.weight"), ("m4_b", "m4.0.bias"))
TOP_FIELDS = (("in_w", "in_lin.0.weight"), ("in_b", "in_lin.0.bias"), ("cat_w", "layer_cat_lin.0.weight"),
              ("cat_b", "layer_cat_lin.0.bias"), ("after_w", "after_conv.0.weight"), ("after_b", "after_conv.0.bias"),
              ("final_w", "final_lin.0.weight"), ("final_b", "final_lin.0.bias"))


def used_param_names(num_layers):
    names = [n for _, n in TOP_FIELDS[:2]]
    for l in range(num_layers):
        names += [f"convs.{l}.{n}" for _, n in LAYER_FIELDS]
    names += [n for _, n in TOP_FIELDS[2:]]
    return names


def expected_shapes(num_layers, H):
    sh = {"in_lin.0.weight": (H, 2), "in_lin.0.bias": (H,), "layer_cat_lin.0.weight": (H, num_layers * H + 2),
          "layer_cat_lin.0.bias": (H,), "after_conv.0.weight": (H, H), "after_conv.0.bias": (H,),
          "final_lin.0.weight": (1, H), "final_lin.0.bias": (1,)}
    for l in range(num_layers):
        for m in ("m1", "m2"):
            for k in ("0", "2"):
                sh[f"convs.{l}.{m}.{k}.weight"] = (H, H)
                sh[f"convs.{l}.{m}.{k}.bias"] = (H,)
        sh[f"convs.{l}.m4.0.weight"] = (H, 2 * H)
        sh[f"convs.{l}.m4.0.bias"] = (H,)
    return sh


class ParamPack:
    """Host-side dppm_ppgn_params built from a {state_dict name: cuda tensor} mapping.  Keeps the tensors alive."""

    def __init__(self, tensors, num_layers, hidden, layer_cond=None):
        shapes = expected_shapes(num_layers, hidden)
        self.tensors = {}
        for name, shape in shapes.items():
            if name not in tensors:
                raise KeyError(f"missing PPGN parameter {name}")
            self.tensors[name] = _chk(tensors[name], name, shape)
        self.layers = (PpgnLayer * num_layers)()
        for l in range(num_layers):
            for field, suffix in LAYER_FIELDS:
                setattr(self.layers[l], field, self.tensors[f"convs.{l}.{suffix}"].data_ptr())
        self.struct = PpgnParams()
        self.struct.num_layers = num_layers
        self.struct.hidden = hidden
        for field, name in TOP_FIELDS:
            setattr(self.struct, field, self.tensors[name].data_ptr())
        self.struct.layers_host = C.cast(self.layers, C.POINTER(PpgnLayer))
        self.layer_cond = None
        self.set_layer_cond(layer_cond)

    def set_layer_cond(self, layer_cond):
        """[L, B] float32 on the device (Powerful_Ind conditioning, include/dppm_hip.h) or None."""
        if layer_cond is not None:
            if layer_cond.dim() != 2 or layer_cond.shape[0] != self.struct.num_layers:
                raise ValueError(f"layer_cond: shape {tuple(layer_cond.shape)}, expected [{self.struct.num_layers}, B]")
            _chk(layer_cond, "layer_cond")
        self.layer_cond = layer_cond
        self.struct.layer_cond = layer_cond.data_ptr() if layer_cond is not None else None

    def ref(self):
        return C.byref(self.struct)


def ppgn_workspace(B, N, H, L, training, device):
    nbytes = lib.dppm_ppgn_workspace_bytes(B, N, H, L, int(bool(training)))
    if nbytes == 0:
        raise ValueError(f"invalid PPGN geometry B={B} N={N} H={H} L={L}")
    return torch.empty((nbytes + 3) // 4, device=device, dtype=torch.float32)


def ppgn_forward(pack, A, mask, sigma, workspace, training=False, out=None, precision="f32"):
    A = _chk(A, "A")
    B, N, _ = A.shape
    mask = _chk(mask, "mask", (B, N, N))
    sigma = _chk(sigma, "sigma", (B,))
    if pack.layer_cond is not None and pack.layer_cond.shape[1] != B:
        raise ValueError(f"layer_cond holds {pack.layer_cond.shape[1]} graphs, the batch has {B}")
    _chk(workspace, "workspace")
    logits = out if out is not None else torch.empty(B, N, N, device=A.device, dtype=torch.float32)
    _chk(logits, "out", (B, N, N))
    check(lib.dppm_ppgn_forward(pack.ref(), _ptr(A), _ptr(mask), _ptr(sigma), B, N, _ptr(logits), _ptr(workspace),
                                C.c_size_t(workspace.numel() * 4), int(bool(training)), _prec(precision), _stream()),
          "dppm_ppgn_forward")
    return logits


def chain_supported(pack, N):
    """Whether a whole sampling chain of this network at N nodes runs as one launch (hidden 32, N <= 20: include/dppm_hip.h)."""
    return bool(lib.dppm_ppgn_chain_supported(pack.ref(), int(N)))


def _chain(fn, name, width, pack, flags, mask, level_table, seed, graph_id0, out, precision):
    flags = _chk(flags, "flags")
    B, N = flags.shape
    mask = _chk(mask, "mask", (B, N, N))
    level_table = _chk(level_table, "level_table")
    if level_table.dim() != 2 or level_table.shape[1] != width:
        raise ValueError(f"level_table must be [T, {width}], got {tuple(level_table.shape)}")
    x = out if out is not None else torch.empty(B, N, N, device=flags.device, dtype=torch.float32)
    _chk(x, "out", (B, N, N))
    check(fn(pack.ref(), _ptr(flags), _ptr(mask), _ptr(level_table), int(level_table.shape[0]), C.c_uint64(int(seed) & (2 ** 64 - 1)),
             C.c_uint32(int(graph_id0)), B, N, _ptr(x), _prec(precision), _stream()), name)
    return x


def chain_simple(pack, flags, mask, level_table, seed, graph_id0=0, out=None, precision="f32"):
    """x_T, then T x (re-noise, denoise, reverse step) in one launch; level_table [T, 3] float32 on the device
    (engine.level_table_simple).  Bit-identical to init_xT / edgeflip / ppgn_forward / reverse_step_simple level by level."""
    return _chain(lib.dppm_ppgn_chain_simple, "dppm_ppgn_chain_simple", 3, pack, flags, mask, level_table, seed, graph_id0, out, precision)


def chain_vlb(pack, flags, mask, level_table, seed, graph_id0=0, out=None, precision="f32"):
    """x_T, then T x (denoise, posterior reverse step) in one launch; level_table [T, 7] float32 on the device
    (engine.level_table_vlb).  Bit-identical to init_xT / ppgn_forward / reverse_step_vlb level by level."""
    return _chain(lib.dppm_ppgn_chain_vlb, "dppm_ppgn_chain_vlb", 7, pack, flags, mask, level_table, seed, graph_id0, out, precision)


def ppgn_backward(pack, grad_pack, A, mask, sigma, dlogits, workspace, dsigma=None):
    """Parameter gradients through `grad_pack`; dsigma ([B], optional) receives d/d sigma; when `pack` carries layer_cond,
    `grad_pack.layer_cond` ([L, B]) receives its gradient."""
    A = _chk(A, "A")
    B, N, _ = A.shape
    dlogits = _chk(dlogits, "dlogits", (B, N, N))
    if dsigma is not None:
        _chk(dsigma, "dsigma", (B,))
    if pack.layer_cond is not None and (grad_pack.layer_cond is None or grad_pack.layer_cond.shape != pack.layer_cond.shape):
        raise ValueError("ppgn_backward: grad_pack needs a layer_cond buffer of the parameters' layer_cond shape")
    check(lib.dppm_ppgn_backward(pack.ref(), grad_pack.ref(), _ptr(A), _ptr(mask), _ptr(sigma), B, N, _ptr(dlogits),
                                 _ptr(dsigma), _ptr(workspace), C.c_size_t(workspace.numel() * 4), _stream()),
          "dppm_ppgn_backward")


def plane_matmul(A, Bm, n, trans_a=False, trans_b=False, scale=None, mask=None, scale_div=1, precision="f32"):
    """A, Bm: [batch, n, ld] planes (ld = n rounded up to 4)."""
    A = _chk(A, "A")
    batch, n_, ld = A.shape
    if n_ != n:
        raise ValueError("plane_matmul: A must be [batch, n, ld]")
    Bm = _chk(Bm, "Bm", (batch, n, ld))
    out = torch.empty_like(A)
    check(lib.dppm_plane_matmul(_ptr(A), _ptr(Bm), _ptr(out), batch, n, ld, int(trans_a), int(trans_b), _ptr(scale), _ptr(mask),
                                int(scale_div), _prec(precision), _stream()), "dppm_plane_matmul")
    return out


def linear_fwd(W, X, bias=None, act=False, maskp=None, trans_w=False, out=None, accumulate=False):
    """X: [B, K, P] planes; W: [M, K] (or [K, M] with trans_w) -> Y [B, M, P]."""
    X = _chk(X, "X")
    B, K, P = X.shape
    if W.dim() != 2 or not W.is_cuda or W.dtype != torch.float32 or W.stride(1) != 1:
        raise ValueError("W: expected a 2-d float32 cuda tensor with unit column stride")
    M = W.shape[1] if trans_w else W.shape[0]
    if (W.shape[0] if trans_w else W.shape[1]) != K:
        raise ValueError(f"W: shape {tuple(W.shape)} does not match K={K}")
    Y = out if out is not None else torch.empty(B, M, P, device=X.device, dtype=torch.float32)
    _chk(Y, "out", (B, M, P))
    check(lib.dppm_linear_fwd(_ptr(W), int(W.stride(0)), int(trans_w), _ptr(X), C.c_long(K * P), K, _ptr(bias), int(act),
                              _ptr(maskp), _ptr(Y), C.c_long(M * P), M, B, P, int(accumulate), _stream()), "dppm_linear_fwd")
    return Y


def mlp_pair_fwd(X, weights, maskp=None, save_hidden=False, precision="f32"):
    """X: [B, H, P]; weights: dict with the ten `m1.0.weight` ... `m4.0.bias`-style keys of one layer (m4 unused).
    -> (o1, o2, hid1 or None, hid2 or None)"""
    X = _chk(X, "X")
    B, H, P = X.shape
    layer = PpgnLayer()
    keep = []
    for field, suffix in LAYER_FIELDS:
        if field.startswith("m4"):
            continue
        t = _chk(weights[suffix], suffix, (H, H) if suffix.endswith("weight") else (H,))
        keep.append(t)
        setattr(layer, field, t.data_ptr())
    o1, o2 = torch.empty_like(X), torch.empty_like(X)
    need_hid = save_hidden or H != 128
    h1 = torch.empty_like(X) if need_hid else None
    h2 = torch.empty_like(X) if need_hid else None
    check(lib.dppm_mlp_pair_fwd(_ptr(X), C.c_long(H * P), C.byref(layer), H, _ptr(maskp), _ptr(o1), _ptr(o2), _ptr(h1), _ptr(h2), B, P,
                                _prec(precision), _stream()), "dppm_mlp_pair_fwd")
    return o1, o2, h1, h2


def linear_wgrad(dY, X, want_bias=True):
    """dY: [B, M, P], X: [B, Nw, P] -> (dW [M, Nw], db [M] or None)."""
    dY = _chk(dY, "dY")
    B, M, P = dY.shape
    X = _chk(X, "X")
    Nw = X.shape[1]
    if X.shape[0] != B or X.shape[2] != P:
        raise ValueError("X: batch / plane size mismatch")
    nbytes = lib.dppm_linear_wgrad_workspace_bytes(M, Nw, B, P)
    ws = torch.empty((nbytes + 3) // 4, device=dY.device, dtype=torch.float32)
    dW = torch.empty(M, Nw, device=dY.device, dtype=torch.float32)
    db = torch.empty(M, device=dY.device, dtype=torch.float32) if want_bias else None
    check(lib.dppm_linear_wgrad(_ptr(dY), C.c_long(M * P), _ptr(X), C.c_long(Nw * P), M, Nw, B, P, _ptr(dW), Nw, _ptr(db), _ptr(ws),
                                C.c_size_t(nbytes), _stream()), "dppm_linear_wgrad")
    return dW, db


def inorm_fwd(y, maskp):
    """y: [B, C, P], maskp: [B, P] -> (u, mean [B,C], rstd [B,C])."""
    y = _chk(y, "y")
    B, Cc, P = y.shape
    maskp = _chk(maskp, "maskp", (B, P))
    u = torch.empty_like(y)
    mean = torch.empty(B, Cc, device=y.device, dtype=torch.float32)
    rstd = torch.empty_like(mean)
    check(lib.dppm_inorm_fwd(_ptr(y), C.c_long(Cc * P), _ptr(maskp), _ptr(u), C.c_long(Cc * P), B, Cc, P, _ptr(mean), _ptr(rstd),
                             _stream()), "dppm_inorm_fwd")
    return u, mean, rstd


def adam_step(param, grad, exp_avg, exp_avg_sq, lr, beta1, beta2, eps, weight_decay, step, grad_scale=1.0):
    for t, n in ((param, "param"), (grad, "grad"), (exp_avg, "exp_avg"), (exp_avg_sq, "exp_avg_sq")):
        _chk(t, n, (param.numel(),))
    check(lib.dppm_adam_step(_ptr(param), _ptr(grad), _ptr(exp_avg), _ptr(exp_avg_sq), C.c_size_t(param.numel()), lr, beta1,
                             beta2, eps, weight_decay, int(step), grad_scale, _stream()), "dppm_adam_step")


# ------------------------------------------------------------------------------------------------- categorical states
_BF16 = torch.bfloat16


def _chk_float(t, name, shape=None):
    """A contiguous float32 or bfloat16 tensor on a GPU."""
    if isinstance(t, torch.Tensor) and t.dtype is not torch.float32 and t.dtype is not _BF16:
        raise TypeError(f"{name}: dtype {t.dtype}, expected float32 or bfloat16")
    return _chk(t, name, shape, t.dtype if isinstance(t, torch.Tensor) else None)


def _chk_at(t, name, shape, dtype, index):
    """... of this type, on GPU `index`."""
    _chk(t, name, shape, dtype)
    if t.get_device() != index:
        raise ValueError(f"{name}: on {t.device}, expected cuda:{index}")


def _refuse_overlap(out, t, name):
    """Workgroups read t while others write out."""
    a, b = out.data_ptr(), t.data_ptr()
    if a < b + t.numel() * t.element_size() and b < a + out.numel() * out.element_size():
        raise ValueError(f"out: shares memory with {name}")


def embedding_fwd(weight, ids, scale=1.0, out=None):
    """scale * weight[ids]: weight [V, D] float32 or bfloat16, ids int64 of any shape -> [*ids.shape, D] in weight's type.  An id
    outside [0, V) (a padded position) gives a row of zeros.  out: where it goes."""
    _chk_float(weight, "weight")
    if weight.dim() != 2:
        raise ValueError(f"weight: shape {tuple(weight.shape)}, expected [V, D]")
    index = weight.get_device()
    _chk_at(ids, "ids", None, torch.int64, index)
    V, D = weight.shape
    if out is None:
        out = weight.new_empty((*ids.shape, D))
    else:
        _chk_at(out, "out", (*ids.shape, D), weight.dtype, index)
        _refuse_overlap(out, weight, "weight")
        _refuse_overlap(out, ids, "ids")
    _launch(index, lib.dppm_embedding_fwd, "dppm_embedding_fwd", weight.data_ptr(), weight.dtype is _BF16, ids.data_ptr(), scale,
            out.data_ptr(), ids.numel(), V, D)
    return out


def embedding_wgrad(dout, ids, num_rows, scale=1.0, out=None, accumulate=False):
    """Gradient of embedding_fwd: dout [*ids.shape, D] -> [num_rows, D], scale times the sum of dout over the positions of each class,
    the same bits from call to call.  out: where it goes (float32 or bfloat16; default: dout's type); accumulate=True adds to it and
    leaves rows without a position as they are."""
    _chk_float(dout, "dout")
    index = dout.get_device()
    _chk_at(ids, "ids", None, torch.int64, index)
    if dout.dim() != ids.dim() + 1 or dout.shape[:-1] != ids.shape:
        raise ValueError(f"dout: shape {tuple(dout.shape)}, expected [*{tuple(ids.shape)}, D]")
    T, V, D = ids.numel(), int(num_rows), dout.shape[-1]
    if out is None:
        if accumulate:
            raise ValueError("embedding_wgrad: accumulate needs an out")
        out = dout.new_empty((max(V, 0), D))
    else:
        _chk_float(out, "out", (V, D))
        _chk_at(out, "out", None, out.dtype, index)
        _refuse_overlap(out, dout, "dout")
        _refuse_overlap(out, ids, "ids")
    nbytes = lib.dppm_embedding_wgrad_workspace_bytes(T, V, D)
    ws = torch.empty(nbytes, device=dout.device, dtype=torch.uint8)
    _launch(index, lib.dppm_embedding_wgrad, "dppm_embedding_wgrad", dout.data_ptr(), dout.dtype is _BF16, ids.data_ptr(), scale, out.data_ptr(),
            out.dtype is _BF16, accumulate, T, V, D, ws.data_ptr(), nbytes)
    return out


def loss_ce(x, weight, target, row_weight=None, denom=None, want_grad=True):
    """Softmax cross entropy over classes: x [T, D], weight [V, D] (both float32 or both bfloat16), target [T] int64 (a class outside
    [0, V) means none: the row counts for nothing), row_weight None or [T] float32, denom a positive number (default: the number of rows
    that have a class).  Returns (loss float32 0-d, row_loss [T] float32, dx or None, dweight or None), gradients in x's type, of
    loss = sum(row_weight * row_loss) / denom (include/dppm_hip.h, dppm_loss_ce_fwd_bwd)."""
    _chk_float(x, "x")
    if x.dim() != 2:
        raise ValueError(f"x: shape {tuple(x.shape)}, expected [T, D]")
    T, D = x.shape
    if isinstance(weight, torch.Tensor) and (weight.dim() != 2 or weight.shape[1] != D):
        raise ValueError(f"weight: shape {tuple(weight.shape)}, expected [V, {D}]")
    index = x.get_device()
    _chk_at(weight, "weight", None, x.dtype, index)
    _chk_at(target, "target", (T,), torch.int64, index)
    if row_weight is not None:
        _chk_at(row_weight, "row_weight", (T,), torch.float32, index)
    if denom is not None and not 0 < float(denom) < float("inf"):
        raise ValueError(f"denom {denom}: expected a positive number or None")
    V, bf16 = weight.shape[0], x.dtype is _BF16
    if T == 0:
        zero = torch.zeros((), device=x.device, dtype=torch.float32)
        return (zero, zero.new_zeros(0), torch.empty_like(x), torch.zeros_like(weight)) if want_grad else (zero, zero.new_zeros(0), None, None)
    nbytes = lib.dppm_loss_ce_workspace_bytes(T, V, D, bf16, want_grad)
    out = torch.empty(T + 1, device=x.device, dtype=torch.float32)
    loss, row_loss = out[T], out[:T]
    dx, dweight = (torch.empty_like(x), torch.empty_like(weight)) if want_grad else (None, None)
    ws = torch.empty(nbytes, device=x.device, dtype=torch.uint8)
    _launch(index, lib.dppm_loss_ce_fwd_bwd, "dppm_loss_ce_fwd_bwd", x.data_ptr(), weight.data_ptr(), bf16, target.data_ptr(),
            None if row_weight is None else row_weight.data_ptr(), 0.0 if denom is None else float(denom), T, V, D, loss.data_ptr(),
            row_loss.data_ptr(), None if dx is None else dx.data_ptr(), None if dx is None else dweight.data_ptr(), ws.data_ptr(), nbytes)
    return loss, row_loss, dx, dweight


STATE_BLOCK = 256      # values of a tensor that share one scale of its 8-bit moments (include/dppm_hip.h, dppm_tensor_entry)


class TensorSet:
    """The tensors of one AdamW step, laid out once: a device table of their addresses, and their moments in flat buffers.

    params: contiguous float32 tensors on one GPU, 16-byte aligned, none overlapping another; grads: one for each, all float32 or all
    bfloat16, same number of values; copies: None, or for each parameter a bfloat16 tensor (or None) that every step writes the new
    parameter to.  weight_decay: one number, or one for each tensor.  state_bits: 32 (float32 moments) or 8 (e4m3 of m and of sqrt(v)
    with a float32 scale per 256 values).  state: buffers as in self.state to go on from (16-byte aligned, 8-bit ones and their scales 4); zeros
    if None.
    The set keeps its tensors alive; set_grads() points it at other gradients.  Moments of tensor i lie at self.offsets[i] of the flat
    buffers (offsets are multiples of 256 values)."""

    def __init__(self, params, grads, copies=None, weight_decay=0.0, state_bits=32, state=None):
        if state_bits not in (8, 32):
            raise ValueError(f"state_bits {state_bits}: expected 8 or 32")
        self.params = list(params)
        if not self.params:
            raise ValueError("TensorSet: no tensors")
        n = len(self.params)
        for i, p in enumerate(self.params):
            _chk(p, f"params[{i}]")
            if p.device != self.params[0].device:
                raise ValueError(f"params[{i}]: on {p.device}, params[0] on {self.params[0].device}")
        self.copies = [None] * n if copies is None else list(copies)
        if len(self.copies) != n:
            raise ValueError(f"copies: {len(self.copies)} entries for {n} tensors")
        self.weight_decay = self._per_tensor(weight_decay)
        for i, c in enumerate(self.copies):
            if c is not None:
                _chk(c, f"copies[{i}]", None, torch.bfloat16)
        self.device = self.params[0].device
        self.state_bits = state_bits
        sizes = [p.numel() for p in self.params]
        self.offsets = np.concatenate([[0], np.cumsum([(s + STATE_BLOCK - 1) // STATE_BLOCK * STATE_BLOCK for s in sizes])]).tolist()
        self.state = self._state(state)
        per = lib.dppm_adamw_chunk()
        counts = np.asarray([(s + per - 1) // per for s in sizes], dtype=np.int64)
        if counts.sum() > 2 ** 31 - 1:
            raise ValueError("TensorSet: too many values")
        which = np.repeat(np.arange(n, dtype=np.int64), counts)
        chunk = np.arange(counts.sum(), dtype=np.int64) - np.repeat(np.cumsum(counts) - counts, counts)
        self.chunks = torch.as_tensor(np.stack([which, chunk], 1).astype(np.int32), device=self.device)
        self.n_chunks = self.chunks.shape[0]
        self.table = torch.empty(n, 9, device=self.device, dtype=torch.int64)
        self.workspace = torch.empty(lib.dppm_adamw_workspace_bytes() // 8, device=self.device, dtype=torch.float64)
        self.set_grads(grads)

    def _per_tensor(self, weight_decay):
        w = [float(weight_decay)] * len(self.params) if isinstance(weight_decay, (int, float)) else [float(w) for w in weight_decay]
        if len(w) != len(self.params):
            raise ValueError(f"weight_decay: {len(w)} entries for {len(self.params)} tensors")
        return w

    def set_weight_decay(self, weight_decay):
        """One number, or one for each tensor (and the table is laid out again)."""
        self.weight_decay = self._per_tensor(weight_decay)
        self.set_grads(self.grads)

    def _state(self, given):
        total = self.offsets[-1]
        if self.state_bits == 32:
            want = {"exp_avg": (total, torch.float32), "exp_avg_sq": (total, torch.float32)}
        else:
            want = {"exp_avg": (total, torch.float8_e4m3fn), "exp_avg_scale": (total // STATE_BLOCK, torch.float32),
                    "exp_avg_root": (total, torch.float8_e4m3fn), "exp_avg_root_scale": (total // STATE_BLOCK, torch.float32)}
        if given is None:
            return {k: torch.zeros(s, device=self.device, dtype=torch.float32).to(t) for k, (s, t) in want.items()}
        if set(given) != set(want):
            raise ValueError(f"state: buffers {sorted(given)}, expected {sorted(want)}")
        for k, (s, t) in want.items():
            if _chk(given[k], f"state[{k!r}]", (s,), t).device != self.device:
                raise ValueError(f"state[{k!r}]: on {given[k].device}, the parameters on {self.device}")
            if given[k].data_ptr() % (16 if self.state_bits == 32 else 4):      # four moments at a time; four codes, one scale
                raise ValueError(f"state[{k!r}]: not aligned to {16 if self.state_bits == 32 else 4} bytes")
        return dict(given)

    def _refuse_shared(self, grads):
        """No byte that a step writes belongs to two tensors, or to a gradient: reads and writes of different workgroups would race."""
        def span(t):
            return t.data_ptr(), t.data_ptr() + t.numel() * t.element_size()

        spans = sorted(span(t) for t in [*self.params, *(c for c in self.copies if c is not None), *self.state.values()] if t.numel())
        ends = [e for _, e in spans]
        if any(begin < end for end, (begin, _) in zip(ends, spans[1:])):
            raise ValueError("TensorSet: two of the tensors share memory")
        for i, g in enumerate(grads):
            begin, end = span(g)
            at = bisect.bisect_right(ends, begin)                 # the first written span that ends behind the gradient's begin
            if begin < end and at < len(spans) and spans[at][0] < end:
                raise ValueError(f"grads[{i}]: shares memory with a tensor that the step writes")

    def set_grads(self, grads):
        """Points the set at these gradients (and lays its table out again: one small upload)."""
        grads = list(grads)
        if len(grads) != len(self.params):
            raise ValueError(f"grads: {len(grads)} tensors for {len(self.params)} parameters")
        kind = grads[0].dtype if isinstance(grads[0], torch.Tensor) else None
        if kind not in (torch.float32, torch.bfloat16):
            raise TypeError(f"grads[0]: dtype {kind}, expected float32 or bfloat16")
        rows = []
        eight = self.state_bits == 8
        m, v = self.state["exp_avg"], self.state["exp_avg_root" if eight else "exp_avg_sq"]
        for i, (p, g, c, off) in enumerate(zip(self.params, grads, self.copies, self.offsets)):
            _chk(g, f"grads[{i}]", None, kind)
            for t, name, align in ((p, "params", 16), (g, "grads", 4 * g.element_size()), (c, "copies", 8)):
                if t is None:
                    continue
                if t.numel() != p.numel() or t.device != self.device:
                    raise ValueError(f"{name}[{i}]: {t.numel()} values on {t.device}, the parameter {p.numel()} on {self.device}")
                if t.data_ptr() % align:
                    raise ValueError(f"{name}[{i}]: not aligned to {align} bytes")
            scales = [self.state[k + "_scale"].data_ptr() + off // STATE_BLOCK * 4 for k in ("exp_avg", "exp_avg_root")] if eight else [0, 0]
            decay = int(np.float64(self.weight_decay[i]).view(np.int64))
            rows.append([p.data_ptr(), g.data_ptr(), 0 if c is None else c.data_ptr(), m.data_ptr() + off * m.element_size(),
                         v.data_ptr() + off * v.element_size(), *scales, p.numel(), decay])
        self._refuse_shared(grads)
        self.grads = grads
        self.grad_bf16 = kind == torch.bfloat16
        self.table.copy_(torch.as_tensor(np.asarray(rows, dtype=np.int64)))


def adamw_step(tensors, lr, beta1, beta2, eps, step, max_norm=None, grad_scale=1.0, seed=0):
    """One AdamW step over a TensorSet: parameters, moments and copies are updated in place (include/dppm_hip.h, dppm_adamw_step).
    max_norm: clip the norm of all gradients together to it; then the norm before clipping is returned (float32, 0-d, on the device),
    and a step whose norm is infinite or NaN changes nothing.  Without it returns None, and such gradients reach the parameters.
    seed: key of the random bits that round 8-bit moments.  A captured call replays the step number it was captured with."""
    if not isinstance(tensors, TensorSet):
        raise TypeError(f"tensors: expected a TensorSet, got {type(tensors)}")
    if max_norm is not None and not max_norm > 0:
        raise ValueError(f"max_norm {max_norm}: expected a positive number or None")
    s = tensors
    norm = torch.empty((), device=s.device, dtype=torch.float32) if max_norm is not None else None
    _launch(s.device.index, lib.dppm_adamw_step, "dppm_adamw_step", s.table.data_ptr(), s.chunks.data_ptr(), s.n_chunks, s.grad_bf16, s.state_bits,
            lr, beta1, beta2, eps, int(step), grad_scale, 0.0 if norm is None else float(max_norm), int(seed) & (2 ** 64 - 1),
            None if norm is None else norm.data_ptr(), s.workspace.data_ptr(), s.workspace.numel() * 8)
    return norm


# ------------------------------------------------------------------------------------------------- graph statistics
def graph_stats(adj, bins=100):
    """adj [B, N, N] on the GPU -> (deg_hist [B, N], clus_hist [B, bins]) float32 counts (include/dppm_hip.h)."""
    adj = _chk(_f32c(adj), "adj")
    B, N, N2 = adj.shape
    if N != N2:
        raise ValueError(f"adj must be [B, N, N], got {tuple(adj.shape)}")
    edges = torch.as_tensor(np.linspace(0.0, 1.0, bins + 1), device=adj.device)      # numpy.histogram's float64 edges
    deg = torch.empty(B, N, device=adj.device, dtype=torch.float32)
    clus = torch.empty(B, bins, device=adj.device, dtype=torch.float32)
    check(lib.dppm_graph_stats(_ptr(adj), B, N, int(bins), _ptr(edges), _ptr(deg), _ptr(clus), _stream()), "dppm_graph_stats")
    return deg, clus


def mmd_gaussian_emd(h1, h2, sigma=1.0, distance_scaling=1.0):
    """h1 [n1, bins], h2 [n2, bins] (counts) -> float64 tensor {mmd, k11, k22, k12} on the device."""
    h1 = _chk(_f32c(h1), "h1")
    h2 = _chk(_f32c(h2), "h2")
    if h1.dim() != 2 or h2.dim() != 2 or h1.shape[1] != h2.shape[1]:
        raise ValueError("mmd_gaussian_emd: histograms must be [n, bins] with equal bins")
    n1, bins = h1.shape
    n2 = h2.shape[0]
    nbytes = lib.dppm_mmd_workspace_bytes(n1, n2)
    ws = torch.empty(max(nbytes, 8) // 8, device=h1.device, dtype=torch.float64)
    out = torch.empty(4, device=h1.device, dtype=torch.float64)
    check(lib.dppm_mmd_gaussian_emd(_ptr(h1), n1, _ptr(h2), n2, bins, C.c_double(sigma), C.c_double(distance_scaling), _ptr(out),
                                    _ptr(ws), C.c_size_t(nbytes), _stream()), "dppm_mmd_gaussian_emd")
    return out


PROF_CLASSES = ("linear_gemm", "plane_matmul", "wgrad_gemm", "inorm", "wstat_mlp2", "wstat_sum2", "wstat_cols", "head")


def prof_begin(max_records=200000):
    check(lib.dppm_prof_begin(int(max_records)), "dppm_prof_begin")


PROF_ARITH = ("f32", "bf16x3", "bf16", "f32x6", "none")   # the arithmetic a timed launch ran in (include/dppm_hip_debug.h)


def prof_end():
    """-> {(class, arith): {"ms": device time, "work": FLOPs (bytes for inorm), "bytes": algorithmic HBM bytes, "launches": n}} for
    every (kernel class, arithmetic) pair that saw a launch, and the truncated flag."""
    nc, na = len(PROF_CLASSES), len(PROF_ARITH)
    n = nc * na
    ms, work, nbytes, cnt = (C.c_double * n)(), (C.c_double * n)(), (C.c_double * n)(), (C.c_long * n)()
    rc = lib.dppm_prof_end(ms, work, nbytes, cnt, nc, na)
    if rc < 0:
        check(rc, "dppm_prof_end")
    out = {}
    for i, k in enumerate(PROF_CLASSES):
        for j, a in enumerate(PROF_ARITH):
            if cnt[i * na + j]:
                out[(k, a)] = {"ms": ms[i * na + j], "work": work[i * na + j], "bytes": nbytes[i * na + j], "launches": cnt[i * na + j]}
    return out, rc == 1


def debug_set(name, value):
    """Experiment switch of the library (include/dppm_hip_debug.h); returns the previous value."""
    old = C.c_int(0)
    check(lib.dppm_debug_get(name.encode(), C.byref(old)), "dppm_debug_get")
    check(lib.dppm_debug_set(name.encode(), int(value)), "dppm_debug_set")
    return old.value


@contextlib.contextmanager
def debug_switch(**switches):
    """with ops.debug_switch(DISABLE_HEAD3=1): ...   -- tests and A/B measurements only."""
    old = {k: debug_set(k, v) for k, v in switches.items()}
    try:
        yield
    finally:
        for k, v in old.items():
            debug_set(k, v)
