"""What is measured of the operators at the two ends of a training step: the token table (lookup with scaling, and its
gradient by sorted tokens) and the orthogonalised update of the layer matrices (Newton-Schulz products, and the whole
momentum update around them).

``run`` computes a case in plain torch operations (``own = False``) or through the framework's entry points
(``own = True``); ``exact`` states the same in 64 bits.
"""

import math

import torch

own = False

DEV = "cuda"
TYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
NS = (3.4445, -4.7750, 2.0315)      # coefficients of the quintic Newton-Schulz step
EPS = 1e-7
LR, MOMENTUM, DECAY, BETA = 0.02, 0.95, 0.1, 0.1


def _lookup(name, rows, cols, vocab, width, dtype, scale=1.0):
    return dict(name=name, op="lookup", rows=rows, cols=cols, vocab=vocab, width=width, dtype=dtype, scale=scale)


def _grad(name, rows, cols, vocab, width, dtype, add, scale=1.0):
    return dict(name=name, op="grad", rows=rows, cols=cols, vocab=vocab, width=width, dtype=dtype, add=add, scale=scale)


def _orth(name, n, rows, cols, dtype):
    return dict(name=name, op="orth", n=n, rows=rows, cols=cols, dtype=dtype)


def _muon(name, layers, d, dtype, projected):
    return dict(name=name, op="muon", layers=layers, d=d, dtype=dtype, projected=projected)


def listed():
    return [
        # generation looks up one new id per step: nothing but latency
        _lookup("lookup of one token", 1, 1, 32000, 1024, "bf16"),
        # the flagship training batch: 8 sequences of 4096 tokens, vocabulary 32000, width 1024
        _lookup("lookup of a training batch", 8, 4096, 32000, 1024, "bf16"),
        # a table of odd width in full precision, scaled by the root of its width
        _lookup("lookup, odd width, scaled", 3, 1365, 50257, 771, "fp32", 27.75),
        # the gradient of the flagship batch, added into the engine's flat fp32 gradient buffer
        _grad("gradient added in fp32", 8, 4096, 32000, 1024, "bf16", True),
        # a dense bf16 gradient as autograd hands it on: 65536 tokens of the large-vocabulary configuration
        _grad("dense gradient, large vocabulary", 8, 8192, 100288, 512, "bf16", False),
        # a short ragged batch of a small fp32 model
        _grad("dense gradient, short batch", 1, 257, 4096, 200, "fp32", False, 14.25),
        # one small matrix: a chain of tiny dependent products
        _orth("orthogonalise one matrix", 1, 256, 256, "bf16"),
        # the six square matrices of one layer of the flagship model
        _orth("orthogonalise a layer", 6, 1024, 1024, "bf16"),
        # tall matrices of odd sizes, fp32 in and out
        _orth("orthogonalise, tall and odd", 2, 1030, 515, "fp32"),
        # every layer matrix of the small test model, one update
        _muon("update of a small model", 2, 256, "bf16", False),
        # two layers of width 2048 (the largest matrices in use: 2048 x 4096)
        _muon("update of two wide layers", 2, 2048, "bf16", False),
        # all 24 layers of the flagship model, with the projected information gradient
        _muon("update of the flagship model", 24, 1024, "bf16", True),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["lookup", "grad", "orth", "muon"])
    if op in ("lookup", "grad"):
        cols, width = _log(rng, 1, 8192), _log(rng, 8, 2048)
        rows = max(1, min(_log(rng, 1, 64), (1 << 25) // (cols * width)))
        c = dict(op=op, rows=rows, cols=cols, vocab=max(16, min(_log(rng, 256, 131072), (1 << 26) // width)), width=width,
                 dtype=rng.choice(["bf16", "bf16", "fp16", "fp32"]), scale=rng.choice([1.0, round(math.sqrt(width), 3)]))
        if op == "grad":
            c["add"] = rng.random() < 0.5
        return c
    if op == "orth":
        rows, cols = _log(rng, 16, 2048), _log(rng, 16, 2048)
        n = max(1, min(_log(rng, 1, 48), (1 << 23) // (rows * cols)))
        return dict(op="orth", n=n, rows=rows, cols=cols, dtype=rng.choice(["bf16", "bf16", "fp16", "fp32"]))
    d = _log(rng, 64, 2048)
    return dict(op="muon", layers=max(1, min(_log(rng, 1, 24), (1 << 23) // (d * d))), d=d,
                dtype=rng.choice(["bf16", "bf16", "fp32"]), projected=rng.random() < 0.5)


# -- inputs ---------------------------------------------------------------------------------------

def _tokens(g, rows, cols, vocab):
    """Ids as text has them: the frequency of an id falls as one over its rank."""
    u = torch.rand(rows, cols, generator=g, device=DEV, dtype=torch.float64)
    return (torch.exp(u * math.log(vocab + 1.0)).floor().long() - 1).clamp_(0, vocab - 1)


def _gradients(g, n, rows, cols):
    """Gradients of weight matrices: a few strong directions over a floor of noise, small in size."""
    k = max(1, min(rows, cols) // 16)
    left = torch.randn(n, rows, k, generator=g, device=DEV)
    right = torch.randn(n, k, cols, generator=g, device=DEV)
    noise = torch.randn(n, rows, cols, generator=g, device=DEV)
    return (left @ right * (0.5 / math.sqrt(k)) + noise) * 1e-3


def prepare(case, seed):
    g = torch.Generator(device=DEV).manual_seed(int(seed))
    op, dtype = case["op"], TYPES[case["dtype"]]
    s = dict(case)
    if op in ("lookup", "grad"):
        rows, cols, vocab, width = case["rows"], case["cols"], case["vocab"], case["width"]
        s["tokens"] = _tokens(g, rows, cols, vocab)
        if op == "lookup":
            s["table"] = torch.randn(vocab, width, generator=g, device=DEV).to(dtype)
        else:
            s["grad"] = (torch.randn(rows, cols, width, generator=g, device=DEV) * 1e-2).to(dtype)
            if case["add"]:
                s["into"] = torch.randn(vocab, width, generator=g, device=DEV) * 1e-2
    elif op == "orth":
        s["x"] = _gradients(g, case["n"], case["rows"], case["cols"]).to(dtype)
    else:
        d, layers = case["d"], case["layers"]
        banks = []
        for n, cols in ((6 * layers, d), (2 * layers, 2 * d)):      # per layer six (d, d) matrices and two (d, 2 d)
            p = (torch.randn(n, d, cols, generator=g, device=DEV) / math.sqrt(cols)).to(dtype)
            gt = _gradients(g, n, d, cols)
            gi = _gradients(g, n, d, cols) if case["projected"] else None
            banks.append((p, gt, gi, _gradients(g, n, d, cols) * 8.0))
        s["banks"] = banks
        if case["projected"]:
            s["scalars"] = torch.tensor([0.3, 0.7], device=DEV)      # projection coefficient, clip factor
        # the program holds every matrix as a tensor of its own
        s["lists"] = [[m for b in banks if b[i] is not None for m in b[i].unbind(0)] for i in range(4)]
    return s


# -- one pass -------------------------------------------------------------------------------------

def _plain_orth(x):
    a, b, c = NS
    x = x / (torch.sqrt((x * x).sum(dim=(-2, -1), keepdim=True)) + EPS)
    tall = x.shape[-2] > x.shape[-1]
    if tall:
        x = x.transpose(-2, -1)
    for _ in range(5):
        q = x @ x.transpose(-2, -1)
        x = a * x + (b * q + c * (q @ q)) @ x
    return x.transpose(-2, -1) if tall else x


def _plain_muon(p, gt, gi, m, scalars):
    g = gt
    if gi is not None:
        g = scalars[1] * ((1.0 - BETA * scalars[0]) * gt + BETA * gi)
    m.mul_(MOMENTUM).add_(g)
    o = _plain_orth(g + MOMENTUM * m)
    step = LR * 0.2 * math.sqrt(max(p.shape[-2:]))
    p.copy_(p.float() * (1.0 - LR * DECAY) - step * o)


def run(s):
    op = s["op"]
    if own:
        from gdnet_b200.ops import functional as ops

        if op == "lookup":
            return ops.embedding(s["tokens"], s["table"], scale=s["scale"])
        if op == "grad":
            return ops.embedding_grad(s["tokens"], s["grad"], s["vocab"], scale=s["scale"], out=s.get("into"))
        if op == "orth":
            return ops.orthogonalize(s["x"])
        params, grads, infos, moments = s["lists"]
        ops.muon_update_(params, grads, moments, lr=LR, momentum=MOMENTUM, weight_decay=DECAY,
                         info_grads=infos or None, scalars=s.get("scalars"), beta=BETA if infos else 0.0)
        return [b[0] for b in s["banks"]] + [b[3] for b in s["banks"]]

    if op == "lookup":
        return (s["table"][s["tokens"]].float() * s["scale"]).to(s["table"].dtype)
    if op == "grad":
        rows = s["grad"].reshape(-1, s["width"]).float() * s["scale"]
        into = s.get("into")
        if into is not None:
            return into.index_add_(0, s["tokens"].reshape(-1), rows)
        out = torch.zeros(s["vocab"], s["width"], device=DEV)
        return out.index_add_(0, s["tokens"].reshape(-1), rows).to(s["grad"].dtype)
    if op == "orth":
        return _plain_orth(s["x"].float()).to(s["x"].dtype)
    for bank in s["banks"]:
        _plain_muon(*bank, s.get("scalars"))
    return [b[0] for b in s["banks"]] + [b[3] for b in s["banks"]]


# -- what a pass cannot do without ------------------------------------------------------------------

def _ns_flops(n, rows, cols):
    """Five steps on the smaller side k of a matrix: the two symmetric products need one triangle each."""
    k, w = min(rows, cols), max(rows, cols)
    return 5.0 * n * (k * (k + 1) * w + k * (k + 1) * k + 2.0 * k * k * w)


def work(case):
    size = 4 if case["dtype"] == "fp32" else 2
    if case["op"] in ("lookup", "grad"):
        tokens, vocab, width = case["rows"] * case["cols"], case["vocab"], case["width"]
        # ids whose frequency falls as one over the rank: expected number of different ones
        p = torch.log1p(1.0 / torch.arange(1, vocab + 1, dtype=torch.float64)) / math.log(vocab + 1.0)
        distinct = float((1.0 - (1.0 - p) ** tokens).sum())
        if case["op"] == "lookup":
            return {"bytes": 8.0 * tokens + (distinct + tokens) * width * size, "flops": float(tokens * width)}
        out = 8.0 * distinct * width if case["add"] else float(vocab * width * size)
        return {"bytes": 8.0 * tokens + tokens * width * size + out, "flops": 2.0 * tokens * width}
    if case["op"] == "orth":
        n, rows, cols = case["n"], case["rows"], case["cols"]
        return {"bytes": 2.0 * n * rows * cols * size, "flops": _ns_flops(n, rows, cols)}
    d, layers = case["d"], case["layers"]
    elements = 10.0 * layers * d * d
    per = 2 * size + 8 + (8 if case["projected"] else 4)       # p and momentum read and written, gradients read
    return {"bytes": elements * per, "flops": _ns_flops(6 * layers, d, d) + _ns_flops(2 * layers, d, 2 * d)}


# -- 64 bits ----------------------------------------------------------------------------------------

def _exact_orth(x):
    """The same polynomial of the singular values, each step applied from the other side: x (a + b h + c h^2) with
    h = x^T x, the wide matrices transposed so that h is the small one."""
    if x.shape[-2] < x.shape[-1]:
        return _exact_orth(x.transpose(-2, -1)).transpose(-2, -1)
    x = x / (x.pow(2).sum(dim=(-2, -1), keepdim=True).sqrt() + EPS)
    for _ in range(5):
        h = torch.matmul(x.transpose(-2, -1), x)
        y = torch.matmul(x, h)
        x = NS[0] * x + NS[1] * y + NS[2] * torch.matmul(y, h)
    return x


def exact(case, seed):
    s = prepare(case, seed)
    op = case["op"]
    if op == "lookup":
        return torch.index_select(s["table"], 0, s["tokens"].reshape(-1)).double().mul(s["scale"]).reshape(*s["tokens"].shape, -1)
    if op == "grad":
        out = s["into"].double() if case["add"] else torch.zeros(case["vocab"], case["width"], device=DEV, dtype=torch.float64)
        return out.index_put_((s["tokens"].reshape(-1),), s["grad"].double().reshape(-1, case["width"]) * s["scale"], accumulate=True)
    if op == "orth":
        return _exact_orth(s["x"].double())
    new_p, new_m = [], []
    for p, gt, gi, m in s["banks"]:
        g = gt.double()
        if gi is not None:
            coef, clip = (float(v) for v in s["scalars"])
            g = clip * (1.0 - BETA * coef) * g + clip * BETA * gi.double()
        m = MOMENTUM * m.double() + g
        o = torch.cat([_exact_orth(part) for part in (g + MOMENTUM * m).split(16)])
        new_p.append((1.0 - LR * DECAY) * p.double() - (LR * 0.2 * math.sqrt(max(p.shape[-2:]))) * o)
        new_m.append(m)
    return new_p + new_m
