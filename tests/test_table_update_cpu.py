"""Token table and orthogonalised update on the CPU: the plain statements against 64-bit arithmetic, the arguments that the
entry points refuse, and the engine, checkpoint and configuration around them."""

import pytest
import torch

from gdnet_b200.model import GDNet
from gdnet_b200.ops import functional as ops
from gdnet_b200.runtime.ckpt import CheckpointError, load_sharded, save_sharded
from gdnet_b200.train.engine import TrainEngine
from oracle_table_update import HALF_STEP, gradient_like, orthogonalize, rel, table_grad

BF = torch.bfloat16


def _model(seed=0, **kw):
    torch.manual_seed(seed)
    return GDNet(vocab_size=64, d_embed=32, d=32, n_layers=2, n_cycles=1, kernel_size=3, chunk_size=16, n_slots=4, **kw)


@pytest.mark.parametrize("dtype", [BF, torch.float16, torch.float32])
@pytest.mark.parametrize("scale", [1.0, 5.5])
def test_table_reference(dtype, scale):
    g = torch.Generator().manual_seed(1)
    tok = torch.randint(0, 20, (3, 11), generator=g)
    w = torch.randn(23, 9, generator=g).to(dtype).requires_grad_()
    y = ops.embedding(tok, w, scale)
    assert torch.equal(y, (w[tok].float() * scale).to(dtype))
    gy = torch.randn(3, 11, 9, generator=g).to(dtype)
    want, bound = table_grad(tok, gy, 23, scale)
    dense = ops.embedding_grad(tok, gy, 23, scale)
    smallest = 2.0**-25 if dtype == torch.float16 else 0.0
    assert dense.dtype == dtype
    assert ((dense.double() - want).abs() <= bound + HALF_STEP[dtype] * (want.abs() + bound) + smallest).all()
    out = torch.ones(23, 9)
    assert ops.embedding_grad(tok.int(), gy, 23, scale, out=out) is out
    assert ((out.double() - 1 - want).abs() <= bound + HALF_STEP[torch.float32] * (1 + want.abs() + bound)).all()
    if dtype == torch.float32:
        (dw,) = torch.autograd.grad(y, w, gy)
        assert ((dw.double() - want).abs() <= bound + HALF_STEP[dtype] * want.abs()).all()


def test_table_leaves_out_ids_outside():
    tok = torch.tensor([-1, 2, 5, 2])
    got = ops.embedding_grad(tok, torch.ones(4, 3), 5)
    assert torch.equal(got[:, 0], torch.tensor([0.0, 0, 2, 0, 0]))
    assert ops.embedding_grad(tok[:0], torch.ones(0, 3), 5).eq(0).all()
    with pytest.raises(IndexError):
        ops.embedding(tok, torch.ones(5, 3))


def test_table_refusals():
    w, tok = torch.ones(5, 3), torch.zeros(4, dtype=torch.int64)
    for bad in (torch.ones(5, 3, dtype=torch.float64), torch.ones(5), torch.ones(5, 3, dtype=torch.int32)):
        with pytest.raises(TypeError):
            ops.embedding(tok, bad)
    with pytest.raises(TypeError):
        ops.embedding(tok.float(), w)
    gy = torch.ones(4, 3)
    with pytest.raises(TypeError):
        ops.embedding_grad(tok, gy.double(), 5)
    with pytest.raises(TypeError):
        ops.embedding_grad(tok.bool(), gy, 5)
    with pytest.raises(ValueError):
        ops.embedding_grad(tok[:3], gy, 5)
    with pytest.raises(ValueError):
        ops.embedding_grad(tok, gy, -1)
    for out in (torch.zeros(5, 4), torch.zeros(4, 3), torch.zeros(5, 3, dtype=BF), torch.zeros(3, 5).t()):
        with pytest.raises(ValueError):
            ops.embedding_grad(tok, gy, 5, out=out)
    with pytest.raises(ValueError):
        ops.embedding(tok, w.to("meta"))


def test_gradient_refuses_its_own_memory():
    tok = torch.tensor([2, 0, 1, 2])
    flat = torch.zeros(40)
    for gy, out in ((flat[:12].view(4, 3), flat[11:26].view(5, 3)), (flat[:24].view(4, 6)[:, ::2], flat[20:35].view(5, 3))):
        with pytest.raises(ValueError):
            ops.embedding_grad(tok, gy, 5, out=out)
    with pytest.raises(ValueError):
        ops.embedding_grad(flat[:8].view(torch.int64), flat[20:32].view(4, 3), 5, out=flat[7:22].view(5, 3))
    ops.embedding_grad(tok, flat[:12].view(4, 3), 5, out=flat[12:27].view(5, 3))


@pytest.mark.parametrize("n,r,c", [(2, 16, 16), (1, 5, 33), (3, 40, 12), (1, 1, 1)])
def test_orthogonalize_reference(n, r, c):
    g = torch.Generator().manual_seed(2)
    x = gradient_like(g, n, r, c)
    want = orthogonalize(x)
    # fp32 arithmetic: a few dozen roundings of 2^-24 relative to operands of norm up to 2.8, amplified below 100 times
    assert rel(ops.orthogonalize(x), want) <= 2.0**-24 * 50 * 100
    assert rel(ops.orthogonalize(x, out_dtype=BF), want) <= HALF_STEP[BF] * 1.01
    assert rel(ops.orthogonalize(x.mT), want.mT) <= 2.0**-24 * 50 * 100
    assert not ops.orthogonalize(torch.zeros(n, r, c)).any()


def test_orthogonalize_refusals():
    x = torch.randn(4, 6)
    for bad in (x.double(), x[0], x.int()):
        with pytest.raises(TypeError):
            ops.orthogonalize(bad)
    with pytest.raises(TypeError):
        ops.orthogonalize(x, out_dtype=torch.float64)
    for kw in (dict(steps=-1), dict(steps=101), dict(eps=0.0), dict(eps=1e-50), dict(eps=float("nan")), dict(coefficients=(1.0, 2.0)),
               dict(coefficients=(1.0, float("inf"), 0.0)), dict(coefficients=(4.0, 0.0, 0.0)), dict(coefficients=(3.4445, -4.775, 9.0))):
        with pytest.raises(ValueError):
            ops.orthogonalize(x, **kw)
    with pytest.raises(ValueError):
        ops.orthogonalize(x.clone().requires_grad_())
    with torch.no_grad():
        ops.orthogonalize(x.clone().requires_grad_())


def test_default_coefficients_stay_in_the_operand_format():
    """The bound that the operand format relies on, on a finer grid than the check's own."""
    a, b, c = ops.NS_COEFFICIENTS
    s = torch.linspace(0, 1.2025, 200001, dtype=torch.float64)      # the map's largest value from [0, 1] is 1.2024
    p = s * (a + b * s**2 + c * s**4)
    assert float(p.max()) < 1.2025 and float(p.min()) > -1e-9
    assert float((b * s**2 + c * s**4).abs().max()) < 2.82 < 3.9


def test_muon_reference_and_refusals():
    g = torch.Generator().manual_seed(3)
    p, gr, m = torch.randn(8, 12, generator=g), gradient_like(g, 1, 8, 12)[0], gradient_like(g, 1, 8, 12)[0]
    gi = gradient_like(g, 1, 8, 12)[0]
    p0, m0 = p.double(), m.double()
    sc = torch.tensor([0.3, 0.7])
    ops.muon_update_([p], [gr], [m], lr=0.02, momentum=0.9, weight_decay=0.1, info_grads=[gi], scalars=sc, beta=0.1)
    grad = 0.7 * ((1 - 0.1 * 0.3) * gr.double() + 0.1 * gi.double())
    want_m = 0.9 * m0 + grad
    assert rel(m, want_m) < 1e-6
    want = p0 * (1 - 0.002) - 0.02 * 0.2 * 12**0.5 * orthogonalize(grad + 0.9 * want_m)
    assert rel(p, want) < 1e-6

    def call(ps=None, gs=None, ms=None, **kw):
        a, b, c = torch.ones(4, 4), torch.ones(4, 4), torch.ones(4, 4)
        ops.muon_update_([a] if ps is None else ps, [b] if gs is None else gs, [c] if ms is None else ms, lr=0.1, **kw)

    call()
    call(ps=[], gs=[], ms=[])
    t = torch.ones(4, 4)
    for kw in (dict(gs=[]), dict(ps=[torch.ones(4)], gs=[torch.ones(4)], ms=[torch.ones(4)]), dict(gs=[torch.ones(4, 5)]),
               dict(ps=[torch.ones(4, 8)[:, ::2]]), dict(ps=[t], gs=[t]), dict(ps=[t], ms=[t]), dict(steps=200),
               dict(ps=[t, t], gs=[torch.ones(4, 4)] * 2, ms=[torch.ones(4, 4), torch.ones(4, 4)]),
               dict(info_grads=[torch.ones(4, 4)]), dict(update_scale=-1.0), dict(scalars=torch.ones(1)), dict(scalars=torch.ones(2, dtype=torch.float64))):
        with pytest.raises(ValueError):
            call(**kw)
    flat = torch.ones(40)
    with pytest.raises(ValueError, match="share memory"):
        call(ps=[flat[:16].view(4, 4), flat[8:24].view(4, 4)], gs=[t, t], ms=[torch.ones(4, 4), torch.ones(4, 4)])
    for kw in (dict(ps=[torch.ones(4, 4, dtype=torch.float64)]), dict(ms=[torch.ones(4, 4, dtype=BF)]),
               dict(info_grads=[torch.ones(4, 4, dtype=BF)], scalars=torch.ones(2))):
        with pytest.raises(TypeError):
            call(**kw)


def test_model_scales_its_tokens():
    plain, scaled = _model(), _model(embed_scale=3.0)
    tok = torch.arange(12).view(2, 6)
    assert plain.state_dict().keys() == scaled.state_dict().keys()
    assert torch.equal(plain._embed(tok), plain.proj_in(plain.embed(tok)))
    assert torch.equal(scaled._embed(tok), scaled.proj_in(scaled.embed(tok) * 3.0))
    seen = []
    scaled.embed.register_forward_hook(lambda m, i, o: seen.append(o))
    scaled._embed(tok)
    assert len(seen) == 1
    plain.double()._embed(tok)                              # other types go through the module, as before


def test_engine_groups_and_state():
    eng = TrainEngine(_model(), precision="bf16", matrix_optimizer="muon")
    by_kind = {k: [p for g in eng.groups if g.optimizer == k for p in g.params] for k in ("adamw", "muon")}
    assert len(by_kind["muon"]) == 2 * 8 and all(p.dim() == 2 for p in by_kind["muon"])
    assert len(by_kind["adamw"]) + len(by_kind["muon"]) == len(eng.params)
    assert all(g.v.numel() == (g.m.numel() if g.optimizer == "adamw" else 0) for g in eng.groups)
    state = eng.state_dict_optim()
    eng.load_state_dict_optim(state)
    plain = TrainEngine(_model(), precision="bf16")
    with pytest.raises(ValueError):
        plain.load_state_dict_optim(state)
    old = {k: v for k, v in plain.state_dict_optim().items() if k != "optimizers"}      # written before there was a choice
    plain.load_state_dict_optim(old)
    with pytest.raises(ValueError):
        eng.load_state_dict_optim(dict(old, m=state["m"], v=state["v"]))
    with pytest.raises(ValueError, match="matrix optimizer"):
        TrainEngine(_model(), precision="bf16", matrix_optimizer="sgd")


def test_sharded_checkpoint_knows_the_optimizer(tmp_path):
    eng = TrainEngine(_model(), precision="bf16", matrix_optimizer="muon")
    for g in eng.groups:
        g.m.normal_()
    save_sharded(tmp_path, 3, eng)
    again = TrainEngine(_model(1), precision="bf16", matrix_optimizer="muon")
    assert load_sharded(tmp_path, again)[0] == 3
    for a, b in zip(eng.groups, again.groups):
        for x, y in zip(a.views(a.m), b.views(b.m)):
            assert torch.equal(x, y)
        assert all(torch.equal(x, y) for x, y in zip(a.params, b.params))
    with pytest.raises(CheckpointError, match="moments do not carry over"):
        load_sharded(tmp_path, TrainEngine(_model(1), precision="bf16"))


def test_trainer_refuses_muon_without_the_engine():
    from gdnet_b200.config import Config
    from gdnet_b200.train.trainer import train

    cfg = Config(vocab_size=64, d_embed=32, d=32, n_layers=1, n_cycles=1, sp_size=1, precision="fp32", matrix_optimizer="muon",
                 phases=[{"dataset": "synthetic", "seq_len": 16, "steps": 1}])
    with pytest.raises(ValueError, match="needs the training engine"):
        train(cfg)
