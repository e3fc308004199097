"""Newton-Schulz products and the momentum update on the GPU, against 64-bit arithmetic."""

import math

import pytest
import torch

from gdnet_b200.ops import functional as ops
from oracle_table_update import HALF_STEP, gradient_like, orthogonalize, orthogonalize_bound, rel

pytestmark = pytest.mark.gpu
DEV = "cuda"
BF, FP, F32 = torch.bfloat16, torch.float16, torch.float32


# one element, one row or column, sides under a tile, tile borders, tall and wide, both tile forms, many matrices
@pytest.mark.parametrize("n,r,c", [(1, 1, 1), (3, 1, 70), (2, 90, 1), (1, 16, 16), (5, 33, 47), (2, 128, 128), (3, 129, 64),
                                   (1, 64, 1000), (2, 256, 256), (1, 256, 700), (2, 257, 257), (1, 300, 520), (1, 520, 301),
                                   (2, 1, 2500), (1, 5000, 3), (2, 384, 1024), (1, 1030, 515), (1, 512, 512), (70, 40, 24)])
@pytest.mark.parametrize("dtype", [BF, FP, F32])
def test_orthogonalize(n, r, c, dtype):
    g = torch.Generator().manual_seed(r * 1000 + c)
    x = gradient_like(g, n, r, c, DEV).to(dtype)
    got = ops.orthogonalize(x)
    assert got.dtype == dtype and got.shape == x.shape and got.is_contiguous()
    want, tol = orthogonalize_bound(x.cpu(), dtype)
    for i in range(n):          # every matrix by itself
        assert rel(got[i], want[i]) <= 2 * tol, (i, rel(got[i], want[i]), tol)
    assert torch.equal(got, ops.orthogonalize(x))


@pytest.mark.parametrize("kind", ["powers", "rank one", "two sizes", "tiny", "huge"])
@pytest.mark.parametrize("out_dtype", [BF, F32])
def test_spectra(kind, out_dtype):
    g = torch.Generator().manual_seed(9)
    u = torch.linalg.qr(torch.randn(160, 160, generator=g)).Q
    v = torch.linalg.qr(torch.randn(300, 300, generator=g)).Q[:, :160]
    i = torch.arange(160) + 1.0
    s = {"powers": i**-2, "rank one": (i == 1).float(), "two sizes": torch.where(i <= 8, 1.0, 1e-3)}.get(kind, torch.ones(160))
    x = (u * s) @ v.T * {"tiny": 1e-24, "huge": 1e24}.get(kind, 1.0)
    eps = 1e-30 if kind == "tiny" else 1e-7
    got = ops.orthogonalize(x.to(DEV), eps=eps, out_dtype=out_dtype)
    want, tol = orthogonalize_bound(x, out_dtype, eps=eps)
    assert rel(got, want) <= tol


@pytest.mark.parametrize("steps,coefficients", [(0, ops.NS_COEFFICIENTS), (1, ops.NS_COEFFICIENTS), (12, ops.NS_COEFFICIENTS),
                                               (7, (1.5, -0.5, 0.0)), (4, (2.0, -1.5, 0.5))])
def test_steps_and_coefficients(steps, coefficients):
    g = torch.Generator().manual_seed(10)
    x = gradient_like(g, 2, 100, 150)
    for out_dtype in (BF, F32):
        got = ops.orthogonalize(x.to(DEV), steps=steps, coefficients=coefficients, out_dtype=out_dtype)
        want, tol = orthogonalize_bound(x, out_dtype, steps=steps, coefficients=coefficients)
        assert rel(got, want) <= tol


def test_zeros_infinities_and_strides():
    g = torch.Generator().manual_seed(11)
    x = gradient_like(g, 4, 200, 300, DEV)
    clean = ops.orthogonalize(x)
    x[1] = 0
    x[2, 5, 7] = float("nan")
    x[3, 150, 2] = float("inf")
    got = ops.orthogonalize(x)
    assert torch.equal(got[0], clean[0]) and not got[1].any()       # a bad matrix does not reach its neighbours
    assert got[2].isnan().all() and got[3].isnan().any()
    big = gradient_like(g, 2, 64, 97, DEV)
    for v in (big[:, 1:60, 3:90], big.mT, big[:1].expand(3, 64, 97), big[0]):
        assert torch.equal(ops.orthogonalize(v), ops.orthogonalize(v.contiguous()))
    assert ops.orthogonalize(big[:0]).shape == (0, 64, 97) and ops.orthogonalize(big[:, :0]).shape == (2, 0, 97)
    four = gradient_like(g, 6, 20, 30, DEV).view(2, 3, 20, 30)
    assert torch.equal(ops.orthogonalize(four).view(6, 20, 30), ops.orthogonalize(four.view(6, 20, 30)))


def test_result_is_near_orthogonal():
    g = torch.Generator().manual_seed(12)
    o = ops.orthogonalize(gradient_like(g, 1, 300, 600, DEV)[0])
    s = torch.linalg.svdvals(o.double())
    # five steps take [0.01, 1] into the attracting range of the polynomial, about [0.68, 1.21]
    assert float(s.min()) > 0.6 and float(s.max()) < 1.25


def _muon_case(g, shapes, dtype, gdtype):
    ps = [torch.randn(*s, generator=g).div(8).to(DEV, dtype) for s in shapes]
    gs = [gradient_like(g, s[0] if len(s) == 3 else 1, *s[-2:]).view(s).to(DEV, gdtype) for s in shapes]
    gi = [gradient_like(g, s[0] if len(s) == 3 else 1, *s[-2:]).view(s).to(DEV, gdtype) for s in shapes]
    ms = [gradient_like(g, s[0] if len(s) == 3 else 1, *s[-2:]).view(s).to(DEV) * 8 for s in shapes]
    return ps, gs, gi, ms


SHAPES = [(64, 64), (64, 128), (64, 64), (130, 33), (3, 40, 40), (1, 1), (64, 64)]


@pytest.mark.parametrize("dtype,gdtype", [(BF, F32), (BF, BF), (F32, F32), (FP, FP)])
@pytest.mark.parametrize("nesterov,projected", [(True, False), (False, True), (True, True)])
def test_muon_update(dtype, gdtype, nesterov, projected):
    g = torch.Generator().manual_seed(13)
    ps, gs, gi, ms = _muon_case(g, SHAPES, dtype, gdtype)
    p0, m0 = [p.double().cpu() for p in ps], [m.double().cpu() for m in ms]
    sc = torch.tensor([0.3, 0.7], device=DEV) if projected else None
    kw = dict(info_grads=gi, scalars=sc, beta=0.1) if projected else {}
    ops.muon_update_(ps, gs, ms, lr=0.02, momentum=0.9, nesterov=nesterov, weight_decay=0.1, **kw)
    for i, s in enumerate(SHAPES):
        grad = gs[i].double().cpu()
        size = grad.abs()
        if projected:
            c, k = (float(v) for v in sc)
            size = k * ((1 - 0.1 * c) * grad.abs() + 0.1 * gi[i].double().cpu().abs())
            grad = k * ((1 - 0.1 * c) * grad + 0.1 * gi[i].double().cpu())
        m = 0.9 * m0[i] + grad
        # a handful of fp32 roundings (coefficients, two products, two sums)
        m_tol = 8 * 2.0**-24 * (0.9 * m0[i].abs() + size)
        assert ((ms[i].double().cpu() - m).abs() <= m_tol).all()
        u = grad + 0.9 * m if nesterov else m
        want, tol = orthogonalize_bound(u, dtype)
        step = 0.02 * 0.2 * math.sqrt(max(s[-2:]))
        p = p0[i] * (1 - 0.02 * 0.1) - step * want
        off = float((ps[i].double().cpu() - p).norm())
        # the direction's own error (without its rounding to 16 bits: it is not rounded here), then p's one rounding
        assert off <= step * tol * float(want.norm()) * 2 + (HALF_STEP[dtype] + 4 * 2.0**-24) * float(p.norm()), (i, off)


def test_muon_groups_and_many_matrices():
    """More matrices of a shape than one launch takes, all updated, none twice."""
    g = torch.Generator().manual_seed(14)
    ps, gs, _, ms = _muon_case(g, [(32, 32)] * 150, BF, F32)
    one = [[t[-1].clone()] for t in (ps, gs, ms)]
    ops.muon_update_(ps, gs, ms, lr=0.1)
    ops.muon_update_(*one, lr=0.1)
    assert torch.equal(ps[-1], one[0][0]) and torch.equal(ms[-1], one[2][0])
    for p, gr in zip(ps, gs):
        assert p.isfinite().all()


def test_capture_and_replay():
    g = torch.Generator().manual_seed(15)
    x = gradient_like(g, 3, 300, 280, DEV)
    ps, gs, _, ms = _muon_case(g, [(64, 96), (64, 96)], BF, F32)
    ops.orthogonalize(x)
    start = [t.clone() for t in ps + ms]
    graph, second = torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        o = ops.orthogonalize(x)
    with torch.cuda.graph(second, pool=graph.pool()):
        ops.muon_update_(ps, gs, ms, lr=0.1)
    x.copy_(gradient_like(g, 3, 300, 280))
    graph.replay()
    second.replay()
    torch.cuda.synchronize()
    assert torch.equal(o, ops.orthogonalize(x))
    for t, s in zip(ps + ms, start):
        captured = t.clone()
        t.copy_(s)
        s.copy_(captured)
    ops.muon_update_(ps, gs, ms, lr=0.1)
    for t, s in zip(ps + ms, start):
        assert torch.equal(t, s)


def test_two_streams_at_once():
    g = torch.Generator().manual_seed(16)
    xs = [gradient_like(g, 4, 520, 512, DEV) for _ in range(2)]
    want = [ops.orthogonalize(x) for x in xs]
    streams = [torch.cuda.Stream() for _ in xs]
    torch.cuda.synchronize()
    got = [None, None]
    for rep in range(3):
        for k, (x, st) in enumerate(zip(xs, streams)):
            with torch.cuda.stream(st):
                got[k] = ops.orthogonalize(x)
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(got, want))


def test_engine_step_with_muon():
    """A training step as a user runs it: token lookup and its gradient added into the flat fp32 buffers, AdamW for the
    table and the vectors, the orthogonalised update for the layer matrices, both from the projected gradient."""
    from gdnet_b200 import _ext
    from gdnet_b200.model import GDNet
    from gdnet_b200.ops import reference as ref
    from gdnet_b200.train.engine import TrainEngine
    from gdnet_b200.utils.fp8 import cast_for_precision

    torch.manual_seed(0)
    model = GDNet(vocab_size=1000, d_embed=128, d=128, n_layers=2, n_cycles=2, kernel_size=4, chunk_size=256, embed_scale=2.0).to(DEV)
    cast_for_precision(model, "fp8")
    lr, wd = 1e-2, 0.1
    eng = TrainEngine(model, lr=lr, weight_decay=wd, precision="fp8", matrix_optimizer="muon", muon_momentum=0.9)
    seen = {}
    update = eng._update

    def watched(beta, clip):
        seen["before"] = [(g.flat.clone(), g.g_task.clone(), g.g_info.clone(), g.m.clone(), g.v.clone()) for g in eng.groups]
        update(beta, clip)

    eng._update = watched
    gen = torch.Generator().manual_seed(3)
    for step in range(1, 4):
        tok = torch.randint(0, 1000, (2, 257), generator=gen).to(DEV)
        loss = eng.projected_step(tok[:, :-1], tok[:, 1:], grad_clip=1.0)
        assert loss.isfinite()
        coef, scale = (float(v) for v in eng.scalars)
        for g, (p0, gt, gi, m0, v0) in zip(eng.groups, seen["before"]):
            if g.optimizer == "adamw":
                ref.projected_adamw_(p0, gt, gi, m0, v0, coef=coef, beta_proj=0.1, grad_scale=scale, lr=lr, beta1=0.9, beta2=0.999,
                                     eps=1e-8, weight_decay=wd, step=step)
                assert rel(g.flat, p0) <= 2 * HALF_STEP[g.dtype] + 1e-5
                continue
            for p, before, a, b, m, m_old in zip(g.params, g.views(p0), g.views(gt), g.views(gi), g.views(g.m), g.views(m0)):
                grad = scale * ((1 - 0.1 * coef) * a.double().cpu() + 0.1 * b.double().cpu())
                want_m = 0.9 * m_old.double().cpu() + grad
                assert rel(m, want_m) <= 8 * 2.0**-24 * 10       # roundings of terms at most a few times the sum
                want, tol = orthogonalize_bound(grad + 0.9 * want_m, BF)
                size = lr * 0.2 * math.sqrt(max(p.shape))
                after = before.double().cpu() * (1 - lr * wd) - size * want
                off = float((p.double().cpu() - after).norm())
                assert off <= 2 * size * tol * float(want.norm()) + 1.1 * HALF_STEP[BF] * float(after.norm())
    _ext.check_status(tok)


def test_engine_gradient_of_the_table_is_the_sum_by_token():
    """The buffer of a tied table holds the head's gradient plus the lookup's, each added in fp32: the same two additions
    made one by one give the same bits."""
    from gdnet_b200.ops import cuda as cu

    w = torch.randn(512, 64, device=DEV, dtype=BF).requires_grad_()
    tok = torch.randint(0, 512, (4, 64), device=DEV)
    w.main_grad = torch.zeros(512, 64, device=DEV)
    x = cu.embedding(tok, w, 2.0)
    cu.linear_cross_entropy(x.reshape(-1, 64), w, tok.reshape(-1), 512, False).backward()
    assert w.grad is None
    both, w.main_grad = w.main_grad, torch.zeros(512, 64, device=DEV)
    leaf = x.detach().requires_grad_()
    cu.linear_cross_entropy(leaf.reshape(-1, 64), w, tok.reshape(-1), 512, False).backward()
    assert w.main_grad.any() and leaf.grad.any()
    assert torch.equal(both, ops.embedding_grad(tok, leaf.grad, 512, 2.0, out=w.main_grad))


# sides around 128 and 256: one cluster keeps the matrix, with 1 to 16 CTAs; long sides at and around the slices they hold
@pytest.mark.parametrize("n,r,c", [(2, 128, 256), (1, 127, 257), (3, 100, 64), (2, 128, 512), (2, 513, 90), (1, 20, 1000), (1, 128, 1025),
                                   (2, 1024, 128), (1, 33, 2048), (1, 2049, 128), (1, 128, 2048), (40, 17, 300), (2, 256, 256), (1, 129, 130),
                                   (2, 200, 700), (1, 1024, 256), (1, 256, 1025), (3, 250, 999), (20, 256, 512)])
@pytest.mark.parametrize("dtype", [BF, F32])
def test_small_side(n, r, c, dtype):
    g = torch.Generator().manual_seed(r * 1000 + c)
    x = gradient_like(g, n, r, c, DEV).to(dtype)
    got = ops.orthogonalize(x)
    want, tol = orthogonalize_bound(x.cpu(), dtype)
    for i in range(n):
        assert rel(got[i], want[i]) <= 2 * tol, (i, rel(got[i], want[i]), tol)
    assert torch.equal(got, ops.orthogonalize(x))
    if n > 1 and min(r, c) <= 128:       # the others' number does not change a matrix
        assert torch.equal(got[-1], ops.orthogonalize(x[-1]))


def test_muon_refusals():
    """Arguments that the binding refuses before anything is launched."""
    def call(ps=None, gs=None, ms=None, **kw):
        one = lambda: torch.ones(4, 4, device=DEV)
        ops.muon_update_([one()] if ps is None else ps, [one()] if gs is None else gs, [one()] if ms is None else ms, lr=0.1, **kw)

    call()
    t, flat = torch.ones(4, 4, device=DEV), torch.ones(40, device=DEV)
    u, v = torch.ones(4, 4, device=DEV), torch.ones(4, 4, device=DEV)
    for kw in (dict(gs=[]), dict(ps=[t[0]], gs=[t[0]], ms=[t[0]]), dict(gs=[torch.ones(4, 5, device=DEV)]), dict(gs=[torch.ones(4, 4)]),
               dict(ps=[torch.ones(4, 8, device=DEV)[:, ::2]]), dict(ps=[t], gs=[t]), dict(ps=[t], ms=[t]), dict(steps=200),
               dict(ps=[t, t], gs=[u, u], ms=[u.clone(), v]), dict(info_grads=[u]), dict(scalars=torch.ones(2)),
               dict(ps=[flat[:16].view(4, 4), flat[8:24].view(4, 4)], gs=[t, t], ms=[u, v])):
        with pytest.raises(ValueError):
            call(**kw)
    for kw in (dict(ps=[t.double()]), dict(ms=[t.to(BF)]), dict(info_grads=[t.to(BF)], scalars=torch.ones(2, device=DEV))):
        with pytest.raises(TypeError):
            call(**kw)
    version = t._version
    ops.muon_update_([t], [u], [v], lr=0.1)
    assert t._version > version


def test_muon_shapes_side_by_side():
    """Several shapes in one call (their groups run on two streams) give what one call for each gives, also captured, with banks
    and empty entries among them."""
    g = torch.Generator().manual_seed(17)
    shapes = [(300, 300), (64, 64), (2, 64, 128), (0, 5, 5), (300, 520), (64, 64)]
    ps, gs, _, ms = _muon_case(g, [s for s in shapes if s[0]], BF, F32)
    ps.insert(3, torch.empty(0, 5, 5, device=DEV, dtype=BF)), gs.insert(3, torch.empty(0, 5, 5, device=DEV)), ms.insert(3, torch.empty(0, 5, 5, device=DEV))
    start = [t.clone() for t in ps + ms]
    one = [[t.clone() for t in ts] for ts in (ps, ms)]
    for p, gr, m in zip(one[0], gs, one[1]):
        ops.muon_update_([p], [gr], [m], lr=0.1)
    side = torch.cuda.Stream()
    torch.cuda.synchronize()
    with torch.cuda.stream(side):
        ops.muon_update_(ps, gs, ms, lr=0.1)
    torch.cuda.current_stream().wait_stream(side)
    for a, b in zip(ps + ms, one[0] + one[1]):
        assert torch.equal(a, b)
    for t, s in zip(ps + ms, start):
        t.copy_(s)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        ops.muon_update_(ps, gs, ms, lr=0.1)
    graph.replay()
    torch.cuda.synchronize()
    for a, b in zip(ps + ms, one[0] + one[1]):
        assert torch.equal(a, b)


# pairs of CTAs: long sums of one matrix, and many small matrices, with sides off the tiles; a bank just past those that stay in clusters
@pytest.mark.parametrize("n,r,c", [(1, 1281, 1300), (1, 1500, 1283), (1, 1290, 2049), (24, 257, 300), (22, 600, 261), (33, 256, 200),
                                   (32, 200, 256), (60, 130, 258)])
@pytest.mark.parametrize("dtype", [BF, F32])
def test_pairs_of_blocks(n, r, c, dtype):
    g = torch.Generator().manual_seed(r * 1000 + c)
    x = gradient_like(g, n, r, c, DEV).to(dtype)
    got = ops.orthogonalize(x)
    want, tol = orthogonalize_bound(x.cpu(), dtype)
    for i in range(n):
        assert rel(got[i], want[i]) <= 2 * tol, (i, rel(got[i], want[i]), tol)
    assert torch.equal(got, ops.orthogonalize(x))
