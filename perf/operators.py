"""The score head's operators, as cases that can be timed and compared: layer norm, the matrix product with its epilogue and
its two gradients, and the softmax loss over the class scores.

`run` computes a case with elementary torch operations in 32 bits (`own` false) or with the calls that a user makes of
opal_amd.Engine (`own` true); `exact` computes it in 64 bits, apart from both.  Class counts (355, 356, 1563, 1564) and batch sizes
are those of bench.py and the tests; hidden widths are generic powers of two and odd numbers around them."""
import torch

own = False

_engines = {}
TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}


def _engine():
    """The Engine a user's program keeps for as long as it runs."""
    if 0 not in _engines:
        import opal_amd
        _engines[0] = opal_amd.Engine(0)
    return _engines[0]


def listed():
    return [
        # one read of a serving loop: its 356 scores, normalised for the hidden layer
        dict(name="norm_one_356", op="norm", n=1, cols=356, x="f32", y="bf16", stats=False),
        # the scores of a training batch at 1564 classes, with the statistics that the backward pass needs
        dict(name="norm_1564", op="norm", n=250_000, cols=1564, x="f32", y="bf16", stats=True),
        # the backward pass at an odd class count, a batch of half a million reads
        dict(name="norm_back_355", op="norm_back", n=500_009, cols=355, x="f32", y="bf16"),
        # one read through the hidden layer: the weights are what is read
        dict(name="linear_one_1564x512", op="linear", n=1, k=1564, m=512, t="bf16", act="gelu", bias=True, res="", y="bf16", pre=False),
        # the hidden layer in training: its pre-activation is kept
        dict(name="linear_hidden_1564x512", op="linear", n=250_000, k=1564, m=512, t="bf16", act="gelu", bias=True, res="", y="bf16", pre=True),
        # the output layer at an odd class count: scores added as the residual, logits in 32 bits
        dict(name="linear_logits_512x1563", op="linear", n=60_001, k=512, m=1563, t="bf16", act="none", bias=True, res="bf16", y="f32", pre=False),
        # the gradient that goes from the logits through the activation of the hidden layer
        dict(name="grad_input_1564x512", op="grad_input", n=100_000, k=512, m=1564, t="f16", act="gelu", res="", y="f16"),
        # a small batch of a head in 32 bits, back to the normalised scores, with the skip connection's share
        dict(name="grad_input_f32_100x356", op="grad_input", n=2_048, k=356, m=100, t="f32", act="none", res="f32", y="f32"),
        # the output layer's weights: a long sum over the reads
        dict(name="grad_weight_1564x512", op="grad_weight", n=100_000, k=512, m=1564, t="bf16"),
        # a ragged batch at few classes
        dict(name="grad_weight_63x355", op="grad_weight", n=1_999, k=355, m=63, t="bf16"),
        # the loss over 1564 classes and its gradient, in the type the products take
        dict(name="loss_1564", op="loss", n=250_000, cols=1564, x="f32", y="bf16"),
        # the answer for a few hundred reads: class and probability
        dict(name="class_356", op="class", n=333, cols=356, x="f32"),
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(lo * (hi / lo) ** rng.random()))))


def draw(rng):
    """Batches from one read to a quarter of a million, 2 to 1600 classes, hidden layers of 16 to 1024; all types and directions."""
    op = rng.choice(["norm", "norm_back", "linear", "linear", "grad_input", "grad_weight", "loss", "class"])
    n, cols, hidden = _log(rng, 1, 250_000), _log(rng, 2, 1600), _log(rng, 16, 1024)
    if op in ("norm", "norm_back"):
        c = dict(op=op, n=n, cols=cols, x=rng.choice(["f32", "f32", "bf16", "f16"]), y=rng.choice(["f32", "bf16", "f16"]))
        return dict(c, stats=rng.random() < 0.5) if op == "norm" else c
    if op in ("loss", "class"):
        c = dict(op=op, n=n, cols=cols, x=rng.choice(["f32", "f32", "bf16"]))
        return dict(c, y=rng.choice(["f32", "bf16"])) if op == "loss" else c
    k, m = (cols, hidden) if rng.random() < 0.5 else (hidden, cols)
    t = rng.choice(["bf16", "bf16", "f16", "f32"])
    most = 1.5e10 if t == "f32" else 1.2e11               # multiply-adds: no case is dearer than the largest listed one
    n = max(1, min(n, int(most / (k * m))))
    if op == "grad_weight":
        return dict(op=op, n=n, k=k, m=m, t=t)
    act, res, y = rng.choice(["none", "relu", "silu", "gelu"]), rng.choice(["", "", t, "f32"]), rng.choice([t, "f32"])
    if op == "grad_input":
        return dict(op=op, n=n, k=k, m=m, t=t, act=act, res=res, y=y)
    return dict(op=op, n=n, k=k, m=m, t=t, act=act, bias=rng.random() < 0.8, res=res, y=y, pre=rng.random() < 0.5)


def _rows(x, t):
    """A [n, cols] matrix whose rows begin on 16 bytes, as the framework's own results do."""
    n, cols = x.shape
    step = 16 // torch.empty(0, dtype=t).element_size()
    full = torch.zeros(n, -(-cols // step) * step, dtype=t, device=x.device)
    full[:, :cols] = x.to(t)
    return full[:, :cols]


def _scores(n, cols, g, t):
    """What the linear model answers with: most classes near -1, the read's own and its sister classes above."""
    s = torch.randn(n, cols, device="cuda", generator=g) * 0.25 - 0.6
    near = torch.randint(cols, (n, 1), device="cuda", generator=g)
    for step, rise in ((0, 1.4), (1, 0.8), (2, 0.3)):
        s.scatter_add_(1, (near + step) % cols, torch.full((n, 1), rise, device="cuda"))
    return _rows(s, t), near[:, 0]


def prepare(case, seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    op, n = case["op"], case["n"]

    def randn(*shape):
        return torch.randn(*shape, device="cuda", generator=g)

    if op in ("norm", "norm_back"):
        cols, t = case["cols"], TYPES[case["x"]]
        s = dict(case=case, x=_scores(n, cols, g, t)[0], gamma=1 + 0.2 * randn(cols), beta=0.1 * randn(cols), eps=1e-5)
        if op == "norm_back":
            s["dy"] = _rows(randn(n, cols) * 0.01, TYPES[case["y"]])
            x = s["x"].double()                                       # the forward pass's statistics
            s["mean"] = x.mean(1).float()
            s["rstd"] = (x.var(1, unbiased=False) + s["eps"]).rsqrt().float()
        return s
    if op in ("loss", "class"):
        scores, near = _scores(n, case["cols"], g, torch.float32)
        scores = _rows(scores * 6, TYPES[case["x"]])                  # logits of a trained head
        labels = torch.where(torch.rand(n, device="cuda", generator=g) < 0.9, near + 1, torch.randint(0, case["cols"] + 1, (n,), device="cuda", generator=g))
        return dict(case=case, scores=scores, labels=labels.int(), scale=1.0 / n)     # label 0: a read without a known class
    k, m, t = case["k"], case["m"], TYPES[case["t"]]
    s = dict(case=case)
    if op == "grad_weight":
        return dict(s, x=_rows(randn(n, k), t), dy=_rows(randn(n, m) * 0.1, t))
    s["w"] = _rows(randn(m, k) * (k if op == "linear" else m) ** -0.5, t)
    if op == "linear":
        s["x"] = _rows(randn(n, k), t)
        s["bias"] = 0.1 * randn(m) if case["bias"] else None
        s["res"] = _rows(randn(n, m), TYPES[case["res"]]) if case["res"] else None
    else:
        s["dy"] = _rows(randn(n, m) * 0.1, t)
        s["pre"] = _rows(randn(n, k), t) if case["act"] != "none" else None
        s["res"] = _rows(randn(n, k) * 0.1, TYPES[case["res"]]) if case["res"] else None
    return s


GELU_A, GELU_B = 1.5957691216057308, 0.044715               # gelu(v) = v sigmoid(A (v + B v^3))


def _act(v, act):
    if act == "relu":
        return torch.where(v > 0, v, torch.zeros_like(v))
    if act == "silu":
        return v / (1 + torch.exp(-v))
    if act == "gelu":
        return v / (1 + torch.exp(-GELU_A * (v + GELU_B * v * v * v)))
    return v


def _act_slope(v, act):
    if act == "relu":
        return (v > 0).to(v.dtype)
    if act == "silu":
        p = 1 / (1 + torch.exp(-v))
        return p + v * p * (1 - p)
    if act == "gelu":
        p = 1 / (1 + torch.exp(-GELU_A * (v + GELU_B * v * v * v)))
        return p + v * p * (1 - p) * GELU_A * (1 + 3 * GELU_B * v * v)
    return torch.ones_like(v)


def _plain(s):
    c = s["case"]
    op = c["op"]
    if op == "norm":
        x = s["x"].float()
        mean = x.mean(1, keepdim=True)
        d = x - mean
        rstd = 1 / torch.sqrt((d * d).mean(1, keepdim=True) + s["eps"])
        y = (d * rstd * s["gamma"] + s["beta"]).to(TYPES[c["y"]])
        return (y, mean[:, 0], rstd[:, 0]) if c["stats"] else y
    if op == "norm_back":
        dy, rstd = s["dy"].float(), s["rstd"][:, None]
        xh = (s["x"].float() - s["mean"][:, None]) * rstd
        h = dy * s["gamma"]
        dx = rstd * (h - h.mean(1, keepdim=True) - xh * (h * xh).mean(1, keepdim=True))
        return dx, (dy * xh).sum(0), dy.sum(0)
    if op == "linear":
        pre = s["x"].float() @ s["w"].float().t()
        if s["bias"] is not None:
            pre = pre + s["bias"]
        y = _act(pre, c["act"])
        if s["res"] is not None:
            y = y + s["res"].float()
        y = y.to(TYPES[c["y"]])
        return (y, pre.to(TYPES[c["t"]])) if c["pre"] else y
    if op == "grad_input":
        dx = s["dy"].float() @ s["w"].float()
        if s["pre"] is not None:
            dx = dx * _act_slope(s["pre"].float(), c["act"])
        if s["res"] is not None:
            dx = dx + s["res"].float()
        return dx.to(TYPES[c["y"]])
    if op == "grad_weight":
        dy = s["dy"].float()
        return dy.t() @ s["x"].float(), dy.sum(0)
    scores = s["scores"].float()
    top, at = scores.max(1)
    e = torch.exp(scores - top[:, None])
    total = e.sum(1)
    if op == "class":
        first = (scores == top[:, None]).int().argmax(1)               # ties go to the lowest class
        return (first + 1).int(), 1 / total
    known = s["labels"] > 0
    at = (s["labels"].long() - 1).clamp(min=0)[:, None]
    loss = torch.where(known, torch.log(total) + top - scores.gather(1, at)[:, 0], torch.zeros_like(top))
    grad = e / total[:, None]
    grad.scatter_add_(1, at, torch.full_like(top, -1)[:, None])
    grad = torch.where(known[:, None], grad * s["scale"], torch.zeros_like(grad))
    return loss, grad.to(TYPES[c["y"]])


def _own(s):
    c, eng = s["case"], _engine()
    op = c["op"]
    if op == "norm":
        y, mean, rstd = eng.layer_norm(s["x"], s["gamma"], s["beta"], eps=s["eps"], out_dtype=TYPES[c["y"]], want_stats=c["stats"])
        return (y, mean, rstd) if c["stats"] else y
    if op == "norm_back":
        return eng.layer_norm_backward(s["dy"], s["x"], s["gamma"], s["mean"], s["rstd"], out_dtype=torch.float32)
    if op == "linear":
        y, pre = eng.linear(s["x"], s["w"], s["bias"], activation=c["act"], residual=s["res"], out_dtype=TYPES[c["y"]], want_pre=c["pre"])
        return (y, pre) if c["pre"] else y
    if op == "grad_input":
        return eng.linear_grad_input(s["dy"], s["w"], pre=s["pre"], activation=c["act"], residual=s["res"], out_dtype=TYPES[c["y"]])
    if op == "grad_weight":
        return eng.linear_grad_weight(s["dy"], s["x"])
    if op == "class":
        return eng.softmax_class(s["scores"])
    return eng.softmax_loss(s["scores"], s["labels"], scale=s["scale"], out_dtype=TYPES[c["y"]])


def run(state):
    return _own(state) if own else _plain(state)


def work(case):
    """Each input read once, each output written once; a multiply-add counts two."""
    size = {"f32": 4, "f16": 2, "bf16": 2, "": 0}
    op, n = case["op"], case["n"]
    if op == "norm":
        e = n * case["cols"]
        return {"bytes": e * (size[case["x"]] + size[case["y"]]) + 8 * case["cols"] + (8 * n if case["stats"] else 0), "flops": 8 * e}
    if op == "norm_back":
        e = n * case["cols"]
        return {"bytes": e * (size[case["x"]] + size[case["y"]] + 4) + 12 * case["cols"] + 8 * n, "flops": 14 * e}
    if op == "loss":
        e = n * case["cols"]
        return {"bytes": e * (size[case["x"]] + size[case["y"]]) + 8 * n, "flops": 6 * e}
    if op == "class":
        e = n * case["cols"]
        return {"bytes": e * size[case["x"]] + 8 * n, "flops": 4 * e}
    k, m, z = case["k"], case["m"], size[case["t"]]
    if op == "linear":
        out = size[case["y"]] + size[case["res"]] + (z if case["pre"] else 0)
        return {"bytes": z * (n * k + m * k) + out * n * m + (4 * m if case["bias"] else 0), "flops": 2 * n * k * m}
    if op == "grad_input":
        out = size[case["y"]] + size[case["res"]] + (z if case["act"] != "none" else 0)
        return {"bytes": z * (n * m + m * k) + out * n * k, "flops": 2 * n * k * m}
    return {"bytes": z * n * (k + m) + 4 * (k * m + m), "flops": 2 * n * k * m}


def exact(case, seed):
    """The definitions, in 64 bits."""
    s = prepare(case, seed)
    op = case["op"]
    d = {name: v.to(torch.float64) for name, v in s.items() if isinstance(v, torch.Tensor) and v.is_floating_point()}
    cols = case.get("cols")
    if op == "norm":
        mean = d["x"].sum(dim=1) / cols
        var = (d["x"] ** 2).sum(dim=1) / cols - mean ** 2              # 64 bits leave room for the difference
        rstd = (var + s["eps"]) ** -0.5
        y = torch.addcmul(d["beta"], (d["x"] - mean[:, None]) * rstd[:, None], d["gamma"])
        return (y, mean, rstd) if case["stats"] else y
    if op == "norm_back":
        # the Jacobian of the normalised row, applied to gamma * dy
        xh = d["rstd"][:, None] * (d["x"] - d["mean"][:, None])
        v = d["gamma"][None, :] * d["dy"]
        a, b = v.sum(dim=1) / cols, torch.mul(v, xh).sum(dim=1) / cols
        return (v - a[:, None] - b[:, None] * xh) * d["rstd"][:, None], torch.mul(d["dy"], xh).sum(dim=0), d["dy"].sum(dim=0)
    if op == "linear":
        pre = torch.matmul(d["x"], d["w"].transpose(0, 1)) + (d["bias"] if case["bias"] else 0.0)
        f = case["act"]
        if f == "relu":
            y = pre.clamp(min=0)
        elif f == "silu":
            y = pre * torch.sigmoid(pre)
        elif f == "gelu":
            y = 0.5 * pre * (1 + torch.tanh(GELU_A / 2 * (pre + GELU_B * pre ** 3)))
        else:
            y = pre
        if case["res"]:
            y = y + d["res"]
        return (y, pre) if case["pre"] else y
    if op == "grad_input":
        dx = torch.matmul(d["dy"], d["w"])
        f = case["act"]
        if f == "relu":
            dx = dx.masked_fill(d["pre"] <= 0, 0.0)
        elif f == "silu":
            dx = dx * torch.sigmoid(d["pre"]) * (1 + d["pre"] * torch.sigmoid(-d["pre"]))
        elif f == "gelu":
            v = d["pre"]
            th = torch.tanh(GELU_A / 2 * (v + GELU_B * v ** 3))
            dx = dx * (0.5 * (1 + th) + 0.25 * GELU_A * v * (1 - th ** 2) * (1 + 3 * GELU_B * v ** 2))
        return dx + d["res"] if case["res"] else dx
    if op == "grad_weight":
        return torch.matmul(d["dy"].transpose(0, 1), d["x"]), d["dy"].sum(dim=0)
    lse = torch.logsumexp(d["scores"], dim=1)
    if op == "class":
        best = d["scores"].amax(dim=1)
        rank = torch.arange(cols, 0, -1, device=best.device)           # the first of equal scores has the highest rank
        return (cols + 1 - ((d["scores"] == best[:, None]) * rank).amax(dim=1)).int(), torch.exp(best - lse)
    labels = s["labels"].long()
    known = labels > 0
    one = torch.nn.functional.one_hot(labels, cols + 1)[:, 1:]
    loss = (lse - torch.where(one > 0, d["scores"], 0.0).sum(dim=1)) * known
    return loss, (torch.exp(d["scores"] - lse[:, None]) - one) * (known[:, None] * s["scale"])
