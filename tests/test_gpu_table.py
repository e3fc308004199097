"""Token table on the GPU: lookup with scaling and its gradient by sorted tokens, against 64-bit sums."""

import pytest
import torch

from gdnet_b200.ops import functional as ops
from oracle_table_update import HALF_STEP, table_grad

pytestmark = pytest.mark.gpu
DEV = "cuda"
BF, FP, F32 = torch.bfloat16, torch.float16, torch.float32

# (tokens shape, vocab, width): one token, none, odd widths (2-, 4- and 16-byte rows), several sort passes, wide rows
SIZES = [((1,), 16, 8), ((0,), 16, 8), ((3, 5), 7, 1), ((257,), 4096, 200), ((2, 129), 50257, 771), ((4, 1000), 300000, 34),
         ((8, 512), 32000, 1024), ((1000,), 1, 64), ((33,), 511, 4100), ((5000,), 512, 12)]


def _tokens(shape, vocab, g):
    u = torch.rand(shape, generator=g, dtype=torch.float64)
    return ((vocab + 1.0) ** u).floor().long().sub(1).clamp(0, vocab - 1).to(DEV)


@pytest.mark.parametrize("shape,vocab,width", SIZES)
@pytest.mark.parametrize("dtype,scale", [(BF, 1.0), (BF, 27.75), (FP, 0.3), (F32, 5.5)])
def test_lookup(shape, vocab, width, dtype, scale):
    g = torch.Generator().manual_seed(1)
    tok = _tokens(shape, vocab, g)
    w = torch.randn(vocab, width, generator=g).to(DEV, dtype)
    for t in (tok, tok.int()):
        got = ops.embedding(t, w, scale)
        want = (w[tok].float() * scale).to(dtype)          # the same single rounding
        assert got.shape == (*shape, width) and torch.equal(got, want)


def test_lookup_strides_and_alignment():
    g = torch.Generator().manual_seed(2)
    big = torch.randn(101, 80, generator=g).to(DEV, BF)
    tok = torch.randint(0, 100, (6, 7), generator=g).to(DEV)
    for w in (big[1:, 3:70], big[:, 8:72], big[:100, :64]):       # odd start, pitch larger than the width
        assert torch.equal(ops.embedding(tok, w), w[tok])
        assert torch.equal(ops.embedding(tok.t(), w, 2.0), w[tok.t()] * 2)


def test_ids_outside_the_table_are_reported():
    from gdnet_b200 import _ext

    w = torch.randn(10, 16, device=DEV)
    tok = torch.tensor([3, -1, 10, 9, 1 << 40], device=DEV)
    got = ops.embedding(tok, w)
    with pytest.raises(_ext.KernelArgumentError):
        _ext.check_status(w)
    assert torch.equal(got[[0, 3]], w[[3, 9]]) and not got[[1, 2, 4]].any()
    gy = torch.ones(5, 16, device=DEV)
    dense = ops.embedding_grad(tok, gy, 10)
    with pytest.raises(_ext.KernelArgumentError):
        _ext.check_status(w)
    want, _ = table_grad(tok, gy, 10, 1.0)
    assert torch.equal(dense.cpu().double(), want)
    ops.embedding_grad(torch.full((40,), -7, device=DEV), torch.ones(40, 16, device=DEV), 10, out=dense)
    with pytest.raises(_ext.KernelArgumentError):
        _ext.check_status(w)
    assert torch.equal(dense.cpu().double(), want)


@pytest.mark.parametrize("shape,vocab,width", SIZES)
@pytest.mark.parametrize("dtype,scale", [(BF, 1.0), (FP, 27.75), (F32, 0.3)])
def test_gradient(shape, vocab, width, dtype, scale):
    g = torch.Generator().manual_seed(3)
    tok = _tokens(shape, vocab, g)
    gy = torch.randn(*shape, width, generator=g).to(DEV, dtype)
    want, bound = table_grad(tok, gy, vocab, scale)
    got = ops.embedding_grad(tok, gy, vocab, scale)
    assert got.dtype == dtype and got.shape == (vocab, width)
    tol = bound + HALF_STEP[dtype] * (want.abs() + bound) + (2.0**-25 if dtype == FP else 0.0)    # half of fp16's smallest step
    assert ((got.double().cpu() - want).abs() <= tol).all()
    base = torch.randn(vocab, width, generator=g).to(DEV)
    out = base.clone()
    assert ops.embedding_grad(tok, gy, vocab, scale, out=out) is out
    tol = bound + HALF_STEP[F32] * (base.double().cpu().abs() + want.abs() + bound)
    assert ((out.double().cpu() - (base.double().cpu() + want)).abs() <= tol).all()
    untouched = torch.ones(vocab, dtype=torch.bool, device=DEV)
    untouched[tok.reshape(-1)] = False
    assert torch.equal(out[untouched], base[untouched])
    again = ops.embedding_grad(tok, gy, vocab, scale)
    assert torch.equal(got, again)                          # fixed order of the sums


@pytest.mark.parametrize("runs", [[5000], [1, 16, 15, 17, 1, 64, 3000, 32, 31, 33], [128] * 40, [127, 129] * 20])
def test_gradient_runs_that_cross_chunks(runs):
    """Ids whose rows fill, touch and cross the pieces that the sorted list is cut into."""
    g = torch.Generator().manual_seed(4)
    tok = torch.repeat_interleave(torch.arange(len(runs)) * 3, torch.tensor(runs))
    tok = tok[torch.randperm(tok.numel(), generator=g)].to(DEV)
    gy = torch.randn(tok.numel(), 72, generator=g).to(DEV)
    want, bound = table_grad(tok, gy, 3 * len(runs), 1.0)
    got = ops.embedding_grad(tok, gy, 3 * len(runs))
    assert ((got.double().cpu() - want).abs() <= bound + HALF_STEP[F32] * want.abs()).all()


def test_gradient_of_strided_and_misaligned_rows():
    g = torch.Generator().manual_seed(5)
    tok = torch.randint(0, 50, (40,), generator=g).to(DEV)
    big = torch.randn(40, 100, generator=g).to(DEV, BF)
    for gy in (big[:, 3:60], big[:, 8:72], torch.randn(64, 40, generator=g).to(DEV, BF).t(), big[:1, :64].expand(40, 64)):
        want, bound = table_grad(tok, gy, 50, 1.0)
        got = ops.embedding_grad(tok, gy, 50)
        assert ((got.double().cpu() - want).abs() <= bound + HALF_STEP[BF] * (want.abs() + bound)).all()
        out = torch.zeros(51 * gy.shape[1], device=DEV)[1 : 1 + 50 * gy.shape[1]].view(50, -1)       # a destination off 16 bytes
        ops.embedding_grad(tok, gy, 50, out=out)
        assert ((out.double().cpu() - want).abs() <= bound + HALF_STEP[F32] * want.abs()).all()


@pytest.mark.parametrize("dtype", [BF, F32])
def test_autograd_and_main_grad(dtype):
    g = torch.Generator().manual_seed(6)
    tok = _tokens((2, 300), 1000, g)
    w = torch.randn(1000, 96, generator=g).to(DEV, dtype).requires_grad_()
    gy = torch.randn(2, 300, 96, generator=g).to(DEV, dtype)
    y = ops.embedding(tok, w, 1.5)
    (dw,) = torch.autograd.grad(y, w, gy, retain_graph=True)
    assert torch.equal(dw, ops.embedding_grad(tok, gy, 1000, 1.5))
    w.main_grad = torch.full((1000, 96), 2.0, device=DEV)
    y.backward(gy)
    assert w.grad is None
    assert torch.equal(w.main_grad, ops.embedding_grad(tok, gy, 1000, 1.5, out=torch.full((1000, 96), 2.0, device=DEV)))


def test_gradient_against_differences():
    g = torch.Generator().manual_seed(7)
    tok = torch.randint(0, 9, (30,), generator=g).to(DEV)
    w = torch.randn(9, 5, generator=g).to(DEV).requires_grad_()
    coef = torch.randn(30, 5, generator=g).to(DEV)
    (dw,) = torch.autograd.grad((ops.embedding(tok, w, 2.0) * coef).sum(), w)
    h = 0.5       # the function is linear: differences are exact up to rounding (values below 2^8, 30 terms of 2^-24 each)
    with torch.no_grad():
        for i, j in ((0, 0), (3, 4), (8, 2)):
            e = torch.zeros_like(w)
            e[i, j] = h
            d = ((ops.embedding(tok, w + e, 2.0) - ops.embedding(tok, w - e, 2.0)).double() * coef.double()).sum() / (2 * h)
            assert abs(float(d) - float(dw[i, j])) <= 2.0**8 * 32 * 2.0**-24


def test_graph_capture_and_other_stream():
    g = torch.Generator().manual_seed(8)
    tok = torch.randint(0, 700, (900,), generator=g).to(DEV)
    w = torch.randn(700, 64, generator=g).to(DEV, BF)
    gy = torch.randn(900, 64, generator=g).to(DEV, BF)
    ops.embedding(tok, w), ops.embedding_grad(tok, gy, 700)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        y = ops.embedding(tok, w, 2.0)
        dw = ops.embedding_grad(tok, gy, 700, 2.0)
    tok.copy_(torch.randint(0, 700, (900,), generator=g))
    gy.copy_(torch.randn(900, 64, generator=g))
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(y, ops.embedding(tok, w, 2.0)) and torch.equal(dw, ops.embedding_grad(tok, gy, 700, 2.0))
    with torch.cuda.stream(side):
        there = ops.embedding_grad(tok, gy, 700, 2.0)
    side.synchronize()
    assert torch.equal(there, dw)


def test_large_list_and_offsets_past_32_bits():
    """More than 2^31 elements of gradient rows, most of them one id."""
    n, width = (1 << 21) + 5, 1032
    tok = torch.zeros(n, dtype=torch.int64, device=DEV)
    tok[::1000] = 3
    tok[-1] = 4
    gy = torch.ones(n, width, dtype=BF, device=DEV)
    got = ops.embedding_grad(tok, gy, 5, out=torch.zeros(5, width, device=DEV))
    want = torch.bincount(tok, minlength=5).float()          # sums of ones: exact in fp32 below 2^24
    assert torch.equal(got, want[:, None].expand(5, width))
    y = ops.embedding(tok, torch.arange(5, dtype=BF, device=DEV)[:, None].expand(5, width).contiguous())
    assert torch.equal(y[:, 0].long(), tok) and torch.equal(y[:, -1].long(), tok)


def test_refusals():
    """Arguments that the binding refuses before anything is launched."""
    w, tok = torch.ones(5, 3, device=DEV), torch.zeros(4, dtype=torch.int64, device=DEV)
    for bad in (w.double(), w[0], w.int()):
        with pytest.raises(TypeError):
            ops.embedding(tok, bad)
    for t in (tok.float(), tok.bool()):
        with pytest.raises(TypeError):
            ops.embedding(t, w)
        with pytest.raises(TypeError):
            ops.embedding_grad(t, torch.ones(4, 3, device=DEV), 5)
    with pytest.raises(ValueError):
        ops.embedding(tok.cpu(), w)
    with pytest.raises(RuntimeError):
        ops.embedding(tok, torch.ones(3, 5, device=DEV).t())
    gy = torch.ones(4, 3, device=DEV)
    for out in (torch.zeros(5, 4, device=DEV), torch.zeros(4, 3, device=DEV), torch.zeros(5, 3), torch.zeros(3, 5, device=DEV).t()):
        with pytest.raises(ValueError):
            ops.embedding_grad(tok, gy, 5, out=out)


def test_model_looks_up_through_the_table_op():
    """GDNet's token path: the same rows as the module's, its gradient in autograd, and the module itself where it has hooks or
    options."""
    from gdnet_b200.model import GDNet
    from gdnet_b200.ops import cuda as cu

    torch.manual_seed(0)
    m = GDNet(vocab_size=100, d_embed=32, d=32, n_layers=1, n_cycles=1, kernel_size=3, chunk_size=16, embed_scale=2.0).to(DEV)
    tok = torch.randint(0, 100, (2, 16), device=DEV)
    n0 = cu.launch_count()
    y = m._embed(tok)
    assert cu.launch_count() == n0 + 1
    assert torch.equal(y, m.proj_in(m.embed(tok) * 2.0))
    (g,) = torch.autograd.grad(y.sum(), m.embed.weight)
    rows = torch.ones_like(y) @ m.proj_in.weight.detach()
    assert torch.equal(g, ops.embedding_grad(tok, rows, m.embed.weight.shape[0], 2.0))
    m.embed.padding_idx = 0
    n0 = cu.launch_count()
    assert torch.equal(m._embed(tok), y) and cu.launch_count() == n0
    with torch.inference_mode():
        m.embed.padding_idx = None
        assert torch.equal(m._embed(tok), y)
        out = torch.zeros(100, 32, device=DEV)
        ops.embedding_grad(tok, torch.ones(2, 16, 32, device=DEV), 100, out=out)
        assert float(out.sum()) == 2 * 16 * 32
