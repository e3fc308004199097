"""Op entry points used by the model code.

One rule decides the implementation: the device of the tensors. CUDA tensors run the
hand-written sm_100a kernels (``gdnet_b200.ops.cuda``, which refuses to work without
the compiled extension rather than fall back); CPU tensors run the plain-PyTorch
statement in ``gdnet_b200.ops.reference``. There is no other backend.
"""

from __future__ import annotations

import functools
import math

import torch
import torch.nn.functional as F

from . import reference as ref


def _on_gpu(t: torch.Tensor) -> bool:
    return t.is_cuda


_cuda_ops = None


def _cuda():
    global _cuda_ops
    if _cuda_ops is None:
        from . import cuda  # deferred: needs the compiled extension

        _cuda_ops = cuda
    return _cuda_ops


# --------------------------------------------------------------------------------------
# single ops
# --------------------------------------------------------------------------------------

def causal_dwconv(x, w, halo=None):
    if _on_gpu(x):
        return _cuda().causal_dwconv(x, w, halo)
    return ref.causal_dwconv(x, w, halo)


def rmsnorm(x, w, eps):
    if _on_gpu(x):
        return _cuda().rmsnorm(x, w, eps)
    return ref.rmsnorm(x, w, eps)


def fused_mem_read(q, gamma, e, tags, vals, alpha):
    if _on_gpu(q):
        return _cuda().fused_mem_read(q, gamma, e, tags, vals, alpha)
    out, w = ref.fused_mem_read(q, gamma, e, tags, vals, alpha)
    return out, w.detach()


def cross_entropy(logits, targets, ignore_index: int = -100):
    if _on_gpu(logits):
        return _cuda().cross_entropy(logits, targets, ignore_index)
    return ref.cross_entropy(logits.reshape(-1, logits.shape[-1]), targets.reshape(-1), ignore_index)


def linear_cross_entropy(x, head, targets, vocab: int, ignore_index: int = -100):
    """Mean cross-entropy of ``head(x)[..., :vocab]`` against ``targets``. On CUDA, for a bias-free bf16 or
    block-scaled FP8 head, the projection, the loss and the head's gradients run chunk by chunk over the rows
    without ever holding all logits (``ops/cuda.py:_LinearCrossEntropyFn``)."""
    x2 = x.reshape(-1, x.shape[-1])
    if _on_gpu(x2) and ignore_index == -100 and getattr(head, "bias", None) is None:
        from .fp8_linear import FP8Linear

        cu = _cuda()
        fp8 = isinstance(head, FP8Linear) and head.recipe == "block"
        plain = type(head) is torch.nn.Linear or fp8
        if plain and cu.linear_cross_entropy_ok(x2, head.weight, fp8):
            return cu.linear_cross_entropy(x2, head.weight, targets, vocab, fp8)
    logits = head(x)[..., :vocab]
    return cross_entropy(logits.reshape(-1, logits.shape[-1]), targets.reshape(-1), ignore_index)


def sample_top_p(logits: torch.Tensor, top_p: float, generator=None) -> torch.Tensor:
    """Nucleus sampling of one id from ``logits (1, V)``."""
    probs = F.softmax(logits, dim=-1)
    sp, si = torch.sort(probs, descending=True)
    before = torch.cumsum(sp, dim=-1) - sp
    sp = torch.where(before < top_p, sp, torch.zeros_like(sp))
    sp = sp / sp.sum(dim=-1, keepdim=True)
    pick = torch.multinomial(sp[0], 1, generator=generator)
    return si[0, pick]


# --------------------------------------------------------------------------------------
# token table
# --------------------------------------------------------------------------------------
_TABLE_TYPES = (torch.bfloat16, torch.float16, torch.float32)


def _check_tokens(tokens, like, what: str) -> None:
    if tokens.dtype not in (torch.int64, torch.int32):
        raise TypeError(f"{what}: tokens must be int64 or int32, got {tokens.dtype}")
    if tokens.device != like.device:
        raise ValueError(f"{what}: tokens are on {tokens.device}, the rows on {like.device}")


def _share_memory(a, b) -> bool:
    """Whether the memory ranges of two tensors meet."""
    if a.numel() == 0 or b.numel() == 0:
        return False
    span = [(t.data_ptr(), t.data_ptr() + (1 + sum((n - 1) * s for n, s in zip(t.shape, t.stride()))) * t.element_size()) for t in (a, b)]
    return span[0][0] < span[1][1] and span[1][0] < span[0][1]


def embedding(tokens, weight, scale: float = 1.0):
    """``scale * weight[tokens]``: ``tokens`` (any shape, int64 or int32) to ``tokens.shape + (width,)`` in the type of
    ``weight (vocab, width)`` (bf16, fp16 or fp32), multiplied in fp32 and rounded once.

    Differentiable in ``weight``. On CUDA the gradient is :func:`embedding_grad`: with a ``main_grad`` installed by the
    training engine it is added there in fp32 and autograd gets none. An id outside the table gives a row of zeros, no
    gradient, and a bad-argument code in the kernel status word (on CPU an ``IndexError``). Like every backward pass of torch,
    one that a CUDA graph captures needs the table to be in no live graph that was made outside the capture."""
    if weight.is_cuda:      # checked in the binding
        return _cuda().embedding(tokens, weight, scale)
    if weight.dim() != 2 or weight.dtype not in _TABLE_TYPES:
        raise TypeError(f"embedding: the table must be a bf16, fp16 or fp32 matrix, got {weight.dtype} {tuple(weight.shape)}")
    _check_tokens(tokens, weight, "embedding")
    return ref.embedding(tokens, weight, float(scale))


@torch.no_grad()
def embedding_grad(tokens, grad, num_rows: int, scale: float = 1.0, out=None):
    """Gradient of :func:`embedding`: ``(num_rows, width)``, row ``v`` is ``scale`` times the sum of the rows
    ``grad[t]`` with ``tokens[t] == v``. ``grad`` is ``tokens.shape + (width,)``.

    Without ``out`` a dense gradient in the type of ``grad`` (summed in fp32, rounded once; rows of absent ids are zero).
    With ``out`` (fp32, contiguous) the sums are added to it, only the rows of ids that occur are touched, and ``out``
    is returned; it must not share memory with ``grad`` or ``tokens``. The rows of an id are summed in a fixed order: the same
    inputs give the same bits. Ids outside the table are left out."""
    if grad.dtype not in _TABLE_TYPES or grad.dim() < 1:
        raise TypeError(f"embedding_grad: grad must be bf16, fp16 or fp32, got {grad.dtype}")
    _check_tokens(tokens, grad, "embedding_grad")
    if grad.shape[:-1] != tokens.shape:
        raise ValueError(f"embedding_grad: grad {tuple(grad.shape)} does not fit tokens {tuple(tokens.shape)}")
    num_rows = int(num_rows)
    if num_rows < 0:
        raise ValueError("embedding_grad: num_rows is negative")
    if out is not None:
        if out.dtype != torch.float32 or not out.is_contiguous() or out.device != grad.device:
            raise ValueError("embedding_grad: out must be a contiguous fp32 tensor on the gradient's device")
        if tuple(out.shape) != (num_rows, grad.shape[-1]):
            raise ValueError(f"embedding_grad: out {tuple(out.shape)} is not ({num_rows}, {grad.shape[-1]})")
        if _share_memory(out, grad) or _share_memory(out, tokens):
            raise ValueError("embedding_grad: out shares memory with grad or tokens")
    if _on_gpu(grad):
        return _cuda().embedding_grad(tokens, grad, num_rows, float(scale), out)
    return ref.embedding_grad(tokens, grad, num_rows, float(scale), out)


# --------------------------------------------------------------------------------------
# orthogonalised update of matrices
# --------------------------------------------------------------------------------------
NS_COEFFICIENTS = (3.4445, -4.7750, 2.0315)     # steep at zero: singular values from 1e-2 up land in about [0.7, 1.2] after five steps
_NS_LIMIT = 3.9                                 # bound of the operand format (csrc/orthogonalize.cu)


@functools.lru_cache(maxsize=64)
def _ns_check(coefficients: tuple, steps: int) -> None:
    """Refuse coefficients under which a singular value that starts in [0, 1], or a factor of the products, leaves the
    range of the operand format."""
    a, b, c = coefficients
    top = 1.0
    for _ in range(steps):
        s = [top * i / 2048 for i in range(2049)]
        poly = max(abs(x * (a + b * x * x + c * x**4)) for x in s)
        factor = max(abs(b * x * x + c * x**4) for x in s)
        if not (max(poly, factor, top * top) <= _NS_LIMIT):
            raise ValueError(f"orthogonalize: coefficients {coefficients} let the iteration grow past {_NS_LIMIT}")
        top = max(poly, 1e-6)


def _ns_arguments(steps, coefficients, eps, what: str):
    if steps == 5 and coefficients is NS_COEFFICIENTS and eps == 1e-7:      # the defaults
        return steps, coefficients, eps
    steps, eps = int(steps), float(eps)
    coefficients = tuple(float(x) for x in coefficients)
    if not 0 <= steps <= 100:
        raise ValueError(f"{what}: steps must be in [0, 100], got {steps}")
    if len(coefficients) != 3 or not all(math.isfinite(x) for x in coefficients):
        raise ValueError(f"{what}: three finite coefficients, got {coefficients}")
    if not (eps >= 1e-37 and math.isfinite(eps)):      # a matrix of zeros is divided by it
        raise ValueError(f"{what}: eps must be at least 1e-37, got {eps}")
    _ns_check(coefficients, steps)
    return steps, coefficients, eps


def _ns_pairs(dtype) -> bool:
    """Whether the products run on pairs of fp16 values: not where the result is rounded to bf16 anyway."""
    return dtype != torch.bfloat16


def orthogonalize(x, steps: int = 5, coefficients=NS_COEFFICIENTS, eps: float = 1e-7, out_dtype=None):
    """Newton-Schulz orthogonalisation of the matrices ``x (..., r, c)`` (bf16, fp16 or fp32): each is divided by its
    Frobenius norm plus ``eps``, then its singular values go ``steps`` times through ``a s + b s^3 + c s^5`` while its singular
    vectors stay. A matrix of zeros stays zero. Returns a new tensor in ``out_dtype`` (default: that of ``x``); a
    bf16 result is computed from fp16 products, others as exactly as in fp32. Has no gradient."""
    out_dtype = x.dtype if out_dtype is None else out_dtype
    if x.dim() < 2 or x.dtype not in _TABLE_TYPES or out_dtype not in _TABLE_TYPES:
        raise TypeError(f"orthogonalize: bf16, fp16 or fp32 matrices, got {x.dtype} {tuple(x.shape)} to {out_dtype}")
    steps, coefficients, eps = _ns_arguments(steps, coefficients, eps, "orthogonalize")
    if torch.is_grad_enabled() and x.requires_grad:
        raise ValueError("orthogonalize has no gradient: detach its input")
    if _on_gpu(x):
        return _cuda().orthogonalize(x, steps, coefficients, eps, out_dtype, _ns_pairs(out_dtype))
    return ref.orthogonalize(x, steps, coefficients, eps, out_dtype)


def _overlap(written, read) -> bool:
    """Whether a written tensor shares memory with another written or a read one (all contiguous)."""
    spans = [(t.data_ptr(), t.data_ptr() + t.numel() * t.element_size(), 1) for t in written if t.numel()]
    spans += [(t.data_ptr(), t.data_ptr() + t.numel() * t.element_size(), 0) for t in read if t.numel()]
    end_any = end_written = 0
    for lo, hi, w in sorted(spans):
        if lo < (end_any if w else end_written):
            return True
        end_any = max(end_any, hi)
        if w:
            end_written = max(end_written, hi)
    return False


@torch.no_grad()
def muon_update_(params, grads, momenta, *, lr: float, momentum: float = 0.95, nesterov: bool = True,
                 weight_decay: float = 0.0, steps: int = 5, coefficients=NS_COEFFICIENTS, eps: float = 1e-7,
                 update_scale: float | None = None, info_grads=None, scalars=None, beta: float = 0.0) -> None:
    """One momentum update of matrices by orthogonalised directions, in place. For every matrix::

        g <- scalars[1] * ((1 - beta * scalars[0]) * grad + beta * info_grad)      (g = grad without scalars)
        m <- momentum * m + g;      u = g + momentum * m                           (u = m without nesterov)
        p <- p * (1 - lr * weight_decay) - lr * update_scale * orthogonalize(u)

    ``params`` (bf16, fp16 or fp32) and ``grads`` (and ``info_grads``) are lists of contiguous tensors ``(r, c)`` or banks of
    matrices ``(n, r, c)``, ``momenta`` the same in fp32; shapes may differ from entry to entry. ``scalars`` is a
    device tensor (projection coefficient, gradient scale) as the training engine keeps it. ``update_scale`` defaults to
    ``0.2 sqrt(max(r, c))``, which gives the update the size of an AdamW step of the same ``lr``. No two
    entries may share memory. Pass the parameters themselves rather than ``.data``: the copies of weights that the kernels
    keep (FP8, folded) are renewed by the parameter's version."""
    params, grads, momenta = list(params), list(grads), list(momenta)
    infos = list(info_grads) if info_grads is not None else []
    if not (len(params) == len(grads) == len(momenta)) or (infos and len(infos) != len(params)):
        raise ValueError("muon_update_: params, grads, momenta (and info_grads) must have the same length")
    steps, coefficients, eps = _ns_arguments(steps, coefficients, eps, "muon_update_")
    if infos and scalars is None:
        raise ValueError("muon_update_: info_grads need scalars (projection coefficient, gradient scale)")
    if not params:
        return
    dev = params[0].device
    if scalars is not None and (scalars.dtype != torch.float32 or scalars.numel() < 2 or scalars.device != dev):
        raise ValueError("muon_update_: scalars must be two fp32 values on the params' device")
    if update_scale is not None and not update_scale >= 0.0:
        raise ValueError(f"muon_update_: update_scale must not be negative, got {update_scale}")
    if dev.type == "cuda":      # the entries' own checks are made where they are gathered, in the binding
        _cuda().muon_update_(params, grads, momenta, infos, scalars, lr=float(lr), momentum=float(momentum), nesterov=bool(nesterov),
                             weight_decay=float(weight_decay), steps=steps, coefficients=coefficients, eps=eps,
                             update_scale=update_scale, beta=float(beta))
        return
    for i, p in enumerate(params):
        mine = [p, grads[i], momenta[i]] + ([infos[i]] if infos else [])
        if p.dim() not in (2, 3) or any(t.shape != p.shape for t in mine):
            raise ValueError(f"muon_update_: entry {i} needs matrices of one shape, got {[tuple(t.shape) for t in mine]}")
        if any(t.device != dev or not t.is_contiguous() for t in mine):
            raise ValueError(f"muon_update_: entry {i} must be contiguous and on {dev}")
        if p.dtype not in _TABLE_TYPES or grads[i].dtype not in _TABLE_TYPES or momenta[i].dtype != torch.float32:
            raise TypeError(f"muon_update_: entry {i} has types {[t.dtype for t in mine]}")
        if infos and infos[i].dtype != grads[i].dtype:
            raise TypeError(f"muon_update_: entry {i} has gradients of two types")
    if _overlap(params + momenta, grads + infos):
        raise ValueError("muon_update_: entries share memory")
    for i, p in enumerate(params):
        g = grads[i].float()
        if scalars is not None:
            g = (1 - beta * scalars[0]) * g + (beta * infos[i].float() if infos else 0.0)
            g = scalars[1] * g
        step = lr * (0.2 * math.sqrt(max(p.shape[-2:])) if update_scale is None else update_scale)
        ref.muon_update_(p, g, momenta[i], lr=lr, momentum=momentum, nesterov=nesterov, weight_decay=weight_decay, step=step,
                         steps=steps, coefficients=coefficients, eps=eps)


# --------------------------------------------------------------------------------------
# one GDLayer step
# --------------------------------------------------------------------------------------

def _module_linear(mod, x):
    """``mod(x)`` for a plain ``nn.Linear`` (weights cast to ``x.dtype``) or an FP8 linear."""
    from .fp8_linear import FP8Linear

    if isinstance(mod, FP8Linear):
        return mod(x)
    return ref.linear(x, mod.weight, mod.bias)


def layer_step(fwd, side, layer, conv_name: str, g: str, r: str, sp_group=None, sp_slot=None,
               return_gate: bool | str = False):
    """Run one step of ``layer`` with the parameter set ``(conv_name, g, r)``.

    Returns ``(fwd', side')`` or ``(fwd', side', gate)`` where ``gate`` is the forward
    gate tensor (``return_gate=True``) or its mean (``return_gate="mean"``). ``side=None`` stands for an
    all-zero side stream: the CUDA path then leaves out the recovery gate, which only ever multiplies it.
    """
    conv = getattr(layer, conv_name)
    k = conv.size
    if _on_gpu(fwd):
        return _cuda().layer_step(fwd, side, layer, conv_name, g, r, sp_group, sp_slot, return_gate)
    if side is None:          # ``None`` stands for an all-zero side stream (the first forward step of a layer)
        side = torch.zeros_like(fwd)

    halo = None
    if sp_group is not None and k > 1:
        from ..parallel.sp import halo_exchange

        halo = halo_exchange(ref.conv_tail(fwd, k).contiguous(), sp_group)

    c = ref.causal_dwconv(fwd, conv.taps, halo)
    s = side.to(c.dtype)
    u = torch.cat([s, c], dim=-1)
    w1r, w2r, nr = getattr(layer, f"{r}_W1"), getattr(layer, f"{r}_W2"), getattr(layer, f"{r}_norm")
    z = _module_linear(w2r, F.silu(_module_linear(w1r, u)))
    eps_r = nr.eps if nr.eps is not None else ref.default_rms_eps(z.dtype)
    R = torch.sigmoid(ref.rmsnorm(z, nr.weight, eps_r).float())
    w1g, w2g, ng = getattr(layer, f"{g}_W1"), getattr(layer, f"{g}_W2"), getattr(layer, f"{g}_norm")
    g_pre = ref.gate_pre(c, w1g.weight, w1g.bias, ng.weight, w2g.weight, w2g.bias)
    fwd_out, side_out, gate = ref.gate_stream_update(g_pre, c, s, R)
    if return_gate == "mean":
        return fwd_out, side_out, gate.mean()
    if return_gate:
        return fwd_out, side_out, gate.to(c.dtype)
    return fwd_out, side_out
