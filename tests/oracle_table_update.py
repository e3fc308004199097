"""Plain 64-bit statements of the token-table and Newton-Schulz operators, and what their arithmetic may lose."""

import torch

NS = (3.4445, -4.7750, 2.0315)
HALF_STEP = {torch.bfloat16: 2.0**-8, torch.float16: 2.0**-11, torch.float32: 2.0**-24}


def table_grad(tokens, grad, num_rows, scale):
    """(dense gradient, bound of an fp32 sum's error) in 64 bits. Summing n values in fp32 in any order is off by at most
    n 2^-24 times the sum of their magnitudes; the product with the scale rounds once more."""
    t = tokens.reshape(-1).long().cpu()
    g = grad.reshape(t.numel(), grad.shape[-1]).double().cpu()
    live = (t >= 0) & (t < num_rows)
    t, g = t[live], g[live]
    total = torch.zeros(num_rows, grad.shape[-1], dtype=torch.float64).index_add_(0, t, g) * scale
    size = torch.zeros(num_rows, grad.shape[-1], dtype=torch.float64).index_add_(0, t, g.abs()) * abs(scale)
    count = torch.zeros(num_rows, dtype=torch.float64).index_add_(0, t, torch.ones(t.numel(), dtype=torch.float64))
    return total, (count[:, None] + 2) * 2.0**-24 * size


def orthogonalize(x, steps=5, coefficients=NS, eps=1e-7, dtype=torch.float64, round_to=lambda v: v):
    """The iteration in ``dtype``. ``round_to`` rounds the operands of the products (X, A, B), not the linear term a X:
    the model of products with 16-bit operands."""
    a, b, c = coefficients
    x = x.double()
    x = (x / (x.pow(2).sum(dim=(-2, -1), keepdim=True).sqrt() + eps)).to(dtype)
    tall = x.shape[-2] > x.shape[-1]
    x = x.mT if tall else x
    for _ in range(steps):
        h = round_to(x)
        A = round_to(h @ h.mT)
        x = a * x + round_to(b * A + c * (A @ A)) @ h
    return x.mT if tall else x


def fp16_operand(v):
    """Scaled by 2^14 and rounded to fp16."""
    return (v * 16384.0).half().to(v.dtype) / 16384.0


def rel(got, want):
    return float((got.double().cpu() - want.double().cpu()).norm() / want.double().cpu().norm().clamp(min=1e-300))


def orthogonalize_bound(x, out_dtype, **kw):
    """How far (2-norm) a result in ``out_dtype`` may be from the 64-bit one, from models of the arithmetic alone.
    bf16: twice what fp16 operands cost (the kernel may round a border value the other way), plus the last rounding.
    Others: pairs of fp16 values hold 22 bits and leave out lo x lo (2^-22 of a product), against 24 bits and fp32 sums in
    the fp32 model; a tensor-core sum may cut where fp32 rounds and there are three of them: 8 times the fp32 model's
    error, plus 2^-20 for a model that happens to be near exact."""
    want = orthogonalize(x, **kw)
    if out_dtype == torch.bfloat16:
        model = rel(orthogonalize(x, round_to=fp16_operand, **kw), want)
        return want, 2 * model + HALF_STEP[out_dtype]
    model = rel(orthogonalize(x, dtype=torch.float32, **kw), want)
    return want, 8 * model + 2.0**-20 + HALF_STEP[out_dtype]


def gradient_like(g, n, rows, cols, device="cpu"):
    """A few strong directions over noise, as gradients of weight matrices have them."""
    k = max(1, min(rows, cols) // 16)
    x = torch.randn(n, rows, k, generator=g) @ torch.randn(n, k, cols, generator=g) * (0.5 / k**0.5)
    return ((x + torch.randn(n, rows, cols, generator=g)) * 1e-3).to(device)
