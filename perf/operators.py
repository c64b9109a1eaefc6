"""Performance cases of the operators around a language model's products.

* ``quantize``  -- values to microscaled 4-bit floats (E2M1 elements, one power-of-two scale per 32
  of them along K) and back: what a weight goes through once and an activation before every product.
* ``product``   -- ``C = A . B^T`` of two such operands, with the product's epilogue.
* ``xent``      -- softmax cross entropy of a head's product ``x . w^T`` with its gradients.
* ``distill``   -- the same head trained on a teacher's top logits, with its gradients.

Plain forms are elementary torch operations in 32 bits (64 for the power-of-two scales);
``exact`` computes the same definitions in 64 bits on another route.
"""

import math

import torch

own = False

_TYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}


# ----------------------------------------------------------------------------------------------
# cases
# ----------------------------------------------------------------------------------------------
def listed():
    return [
        # One decode step's activations: a handful of rows, where the launches are the cost.
        dict(name="quantize_step", op="quantize", rows=16, k=8192, dtype="bf16"),
        # A prompt's activations, or one weight matrix being laid out.
        dict(name="quantize_prompt", op="quantize", rows=8192, k=8192, dtype="bf16"),
        # fp32 master weights of odd height; K leaves half a 64-element group at the end.
        dict(name="quantize_master", op="quantize", rows=5003, k=4128, dtype="f32"),
        # Decode: 16 tokens against one square layer; the product streams its weights.
        dict(name="product_step", op="product", m=16, n=8192, k=8192, out="bf16", bias=False, relu=False),
        # A square layer over a prompt.
        dict(name="product_4096", op="product", m=4096, n=4096, k=4096, out="bf16", bias=False, relu=False),
        # A wide layer over a long prompt.
        dict(name="product_8192", op="product", m=8192, n=8192, k=8192, out="bf16", bias=False, relu=False),
        # A ragged batch through a layer with bias and ReLU, fp32 out.
        dict(name="product_ragged", op="product", m=1037, n=2000, k=4128, out="f32", bias=True, relu=True),
        # Scoring a few tokens: log-likelihoods only, no gradients; the head's weights are read once.
        dict(name="xent_score", op="xent", tokens=8, d=4096, vocab=32768, dtype="bf16", smoothing=0.0, ignored=0.0, reduction="none", grad=False),
        # One training micro-batch.
        dict(name="xent_train", op="xent", tokens=8192, d=4096, vocab=32768, dtype="bf16", smoothing=0.0, ignored=0.1, reduction="mean", grad=True),
        # A ragged batch, an odd vocabulary, half precision and label smoothing.
        dict(name="xent_ragged", op="xent", tokens=1021, d=1032, vocab=50021, dtype="f16", smoothing=0.1, ignored=0.3, reduction="sum", grad=True),
        # Distillation of one micro-batch from the teacher's 64 best logits.
        dict(name="distill_train", op="distill", tokens=4096, d=2048, vocab=32768, dtype="bf16", top=64, temperature=2.0, missing=0.05, grad=True),
        # A short ragged batch with few teacher logits, some rows without any.
        dict(name="distill_ragged", op="distill", tokens=333, d=520, vocab=16001, dtype="f16", top=7, temperature=1.0, missing=0.3, grad=True),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["quantize", "product", "xent", "distill"])
    if op == "quantize":
        while True:
            rows, k = _log(rng, 1, 16384), 32 * _log(rng, 8, 512)
            if 2 ** 16 <= rows * k <= 8192 * 8192:
                return dict(op=op, rows=rows, k=k, dtype=rng.choice(["bf16", "f16", "f32"]))
    if op == "product":
        while True:
            m = _log(rng, 1, 8192)
            n, k = _log(rng, 512, 16384), 32 * _log(rng, 16, 512)
            if m * n * k <= 8192 ** 3:
                bias = rng.random() < 0.5
                return dict(op=op, m=m, n=n, k=k, out=rng.choice(["bf16", "f32"]), bias=bias, relu=bias and rng.random() < 0.5)
    grad = rng.random() < 0.75
    while True:
        tokens = _log(rng, 1, 8192)
        d, vocab = 8 * _log(rng, 32, 1024), _log(rng, 4000, 131072)
        if tokens * d * vocab <= (8192 * 4096 * 32768) // 2:
            break
    dtype = rng.choice(["bf16", "bf16", "f16"])
    if op == "xent":
        return dict(op=op, tokens=tokens, d=d, vocab=vocab, dtype=dtype, smoothing=rng.choice([0.0, 0.0, 0.1]),
                    ignored=rng.choice([0.0, 0.1, 0.5]), reduction=rng.choice(["mean", "sum"]) if grad else "none", grad=grad)
    return dict(op=op, tokens=tokens, d=d, vocab=vocab, dtype=dtype, top=rng.choice([1, 8, 17, 64, 128]),
                temperature=rng.choice([1.0, 2.0, 0.7]), missing=rng.choice([0.0, 0.1]), grad=grad)


# ----------------------------------------------------------------------------------------------
# inputs
# ----------------------------------------------------------------------------------------------
def _inputs(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed * 7919 + 17)

    def normal(*shape):
        return torch.randn(*shape, device="cuda", generator=g)

    op = case["op"]
    if op == "quantize":
        # Activations differ in size from channel to channel: a few channels are large.
        x = normal(case["rows"], case["k"])
        x *= torch.exp(normal(case["k"]))
        return dict(x=x.to(_TYPES[case["dtype"]]))
    if op == "product":
        out = {}
        for name, rows in (("a", case["m"]), ("b", case["n"])):
            x = normal(rows, case["k"])
            x *= torch.exp(0.5 * normal(rows, 1)) * (1.0 if name == "a" else case["k"] ** -0.5)
            out[name + "_codes"], out[name + "_scales"] = _codes(x)
        out["bias"] = 0.1 * normal(case["n"]) if case["bias"] else None
        return out
    dtype, tokens, d, vocab = _TYPES[case["dtype"]], case["tokens"], case["d"], case["vocab"]
    x = normal(tokens, d).to(dtype)
    w = (2.0 * d ** -0.5 * normal(vocab, d)).to(dtype)  # logits of standard deviation 2
    out = dict(x=x, w=w)
    if op == "xent":
        # Words are far from equally frequent.
        target = (vocab * torch.rand(tokens, device="cuda", generator=g) ** 3).long().clamp_(0, vocab - 1)
        ignored = torch.rand(tokens, device="cuda", generator=g) < case["ignored"]
        ignored[0] = False
        out["target"] = torch.where(ignored, -100, target)
    else:
        # The teacher's best entries of every row, in falling order, with distinct words.
        top = case["top"]
        start = (vocab * torch.rand(tokens, 1, device="cuda", generator=g) ** 2).long()
        step = torch.randint(1, max(2, vocab // top), (tokens, 1), device="cuda", generator=g)
        ids = (start + step * torch.arange(top, device="cuda")) % vocab  # step * top <= vocab: distinct
        logits = (8.0 + 2.0 * normal(tokens, top)).sort(dim=1, descending=True).values
        gone = torch.rand(tokens, top, device="cuda", generator=g) < case["missing"]
        gone |= torch.rand(tokens, 1, device="cuda", generator=g) < 0.5 * case["missing"]
        gone[0, 0] = False
        out["teacher_ids"] = torch.where(gone, -1, ids)
        out["teacher_logits"] = logits.to(dtype)
    return out


def prepare(case, seed):
    state = dict(case=case, **_inputs(case, seed))
    if case["op"] == "product" and own:
        # The operands as the framework holds them: packed codes and scales in the product's order.
        from aster_b200 import torch_op

        for name in ("a", "b"):
            values = _values(state[name + "_codes"], state[name + "_scales"])
            state[name], state["s" + name] = torch_op.quantize_mx_direct(values)
    if case["op"] in ("xent", "distill"):
        state["x"].requires_grad_(case["grad"])
        state["w"].requires_grad_(case["grad"])
    return state


# ----------------------------------------------------------------------------------------------
# one pass
# ----------------------------------------------------------------------------------------------
def run(state):
    case = state["case"]
    return globals()[("_own_" if own else "_plain_") + case["op"]](state, case)


def _own_quantize(state, case):
    from aster_b200 import torch_op

    codes, scales = torch_op.quantize_mx_direct(state["x"])
    return torch_op.dequantize_mx_direct(codes, scales, _TYPES[case["dtype"]])


def _own_product(state, case):
    from aster_b200 import torch_op

    return torch_op.gemm_mx_nt_direct(state["a"], state["sa"], state["b"], state["sb"], state["bias"], case["relu"], _TYPES[case["out"]])


def _own_xent(state, case):
    from aster_b200 import head_loss

    x, w = state["x"], state["w"]
    loss = head_loss.linear_cross_entropy(x, w, state["target"], label_smoothing=case["smoothing"], reduction=case["reduction"])
    return (loss, *torch.autograd.grad(loss, (x, w))) if case["grad"] else loss


def _own_distill(state, case):
    from aster_b200 import head_loss

    x, w = state["x"], state["w"]
    loss = head_loss.linear_distillation(x, w, state["teacher_logits"], state["teacher_ids"], temperature=case["temperature"])
    return (loss, *torch.autograd.grad(loss, (x, w))) if case["grad"] else loss


# ---- plain forms ----
def _codes(x):
    """4-bit codes [rows, K] (sign in bit 3) and shared exponents [rows, K/32] of fp32 values: the
    largest magnitude of 32 sets the exponent floor(log2) - 2; elements round to nearest even."""
    blocks = x.float().reshape(x.shape[0], -1, 32)
    amax = blocks.abs().amax(dim=2)
    e = torch.where(amax > 0, torch.frexp(amax).exponent - 3, torch.zeros_like(amax, dtype=torch.int32)).clamp(-127, 127)
    mag = (blocks.abs().double() * torch.exp2(-e.double())[..., None]).clamp_(max=6.0).float()
    # steps of 1/2 below 2, of 1 below 4, of 2 up to 6
    step = torch.where(mag < 2, 0.5, torch.where(mag < 4, 1.0, 2.0))
    mag = torch.round(mag / step) * step
    code = torch.where(mag < 2, 2 * mag, torch.where(mag < 4, mag + 2, mag / 2 + 4)).to(torch.uint8)
    code |= torch.signbit(blocks).to(torch.uint8) << 3
    return code.reshape(x.shape), e


def _values(codes, e):
    """fp32 values of 4-bit codes and their shared exponents."""
    m = (codes & 7).float()
    mag = torch.where(m < 4, m / 2, torch.where(m < 6, m - 2, 2 * m - 8))
    mag = torch.where(codes >= 8, -mag, mag).reshape(codes.shape[0], -1, 32)
    return (mag.double() * torch.exp2(e.double())[..., None]).float().reshape(codes.shape)


def _plain_quantize(state, case):
    return _values(*_codes(state["x"])).to(_TYPES[case["dtype"]])


def _plain_product(state, case):
    c = _values(state["a_codes"], state["a_scales"]) @ _values(state["b_codes"], state["b_scales"]).T
    if state["bias"] is not None:
        c = c + state["bias"]
    if case["relu"]:
        c = torch.clamp(c, min=0.0)
    return c.to(_TYPES[case["out"]])


def _head(x, w, temperature):
    """Logits over the temperature, their maximum and the logarithm of the sum of exponentials."""
    z = (x.detach().float() @ w.detach().float().T) / temperature
    top = z.amax(dim=1, keepdim=True)
    return z, top + torch.log(torch.exp(z - top).sum(dim=1, keepdim=True))


def _plain_xent(state, case):
    x, w, target = state["x"], state["w"], state["target"]
    eps, vocab = case["smoothing"], case["vocab"]
    z, lse = _head(x, w, 1.0)
    kept = target != -100
    at = torch.where(kept, target, 0)[:, None]
    rows = lse[:, 0] - (1 - eps) * torch.gather(z, 1, at)[:, 0]
    if eps:
        rows = rows - eps * z.sum(dim=1) / vocab
    rows = torch.where(kept, rows, 0.0)
    if case["reduction"] == "none":
        return rows
    share = 1.0 / kept.sum() if case["reduction"] == "mean" else torch.ones((), device=x.device)
    loss = rows.sum() * share
    if not case["grad"]:
        return loss
    g = torch.exp(z - lse) - eps / vocab
    g.scatter_add_(1, at, torch.full_like(at, -(1 - eps), dtype=torch.float32))
    g *= torch.where(kept, share, 0.0)[:, None]
    return loss, (g @ w.detach().float()).to(x.dtype), (g.T @ x.detach().float()).to(w.dtype)


def _plain_distill(state, case):
    x, w, ids, tau = state["x"], state["w"], state["teacher_ids"], case["temperature"]
    listed_ = ids >= 0
    kept = listed_.any(dim=1)
    t = torch.where(listed_, state["teacher_logits"].float() / tau, -torch.inf)
    t = torch.where(kept[:, None], t, 0.0)
    t = t - t.amax(dim=1, keepdim=True)
    p = torch.exp(t)
    total = p.sum(dim=1, keepdim=True)
    logp = torch.where(listed_, t - torch.log(total), 0.0)
    p = torch.where(listed_, p / total, 0.0)
    z, lse = _head(x, w, tau)
    at = torch.where(listed_, ids, 0)
    rows = torch.where(kept, (p * (logp - (torch.gather(z, 1, at) - lse))).sum(dim=1), 0.0)
    share = tau * tau / kept.sum()
    loss = rows.sum() * share
    if not case["grad"]:
        return loss
    g = torch.exp(z - lse)
    g.scatter_add_(1, at, -p)
    g *= torch.where(kept, share / tau, 0.0)[:, None]
    return loss, (g @ w.detach().float()).to(x.dtype), (g.T @ x.detach().float()).to(w.dtype)


# ----------------------------------------------------------------------------------------------
# what a pass cannot do without
# ----------------------------------------------------------------------------------------------
def work(case):
    op = case["op"]
    if op == "quantize":
        n = case["rows"] * case["k"]
        size = 4 if case["dtype"] == "f32" else 2
        # values in, codes and scales out, codes and scales in, values out; a few operations a value
        return {"bytes": 2 * n * size + 2 * (n // 2 + n // 32), "flops": 4 * n}
    if op == "product":
        m, n, k = case["m"], case["n"], case["k"]
        size = 4 if case["out"] == "f32" else 2
        return {"bytes": (m + n) * (k // 2 + k // 32) + m * n * size + (4 * n if case["bias"] else 0), "flops": 2 * m * n * k}
    t, d, v = case["tokens"], case["d"], case["vocab"]
    operands = 2 * (t + v) * d
    labels = 8 * t if op == "xent" else 10 * t * case["top"]
    loss = 4 * t if case.get("reduction") == "none" else 4
    # one product forward, two backward; the gradients are as large as the operands
    return {"bytes": operands * (2 if case["grad"] else 1) + labels + loss, "flops": 2 * t * d * v * (3 if case["grad"] else 1)}


# ----------------------------------------------------------------------------------------------
# the definitions in 64 bits
# ----------------------------------------------------------------------------------------------
_GRID = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)


def _exact_values(codes, e):
    grid = torch.tensor(_GRID + tuple(-v for v in _GRID), dtype=torch.float64, device=codes.device)
    return grid[codes.long()] * torch.pow(torch.tensor(2.0, dtype=torch.float64, device=codes.device), e.double()).repeat_interleave(32, dim=1)


def _exact_quantize(data, case):
    x = data["x"].double()
    grid = torch.tensor(_GRID, dtype=torch.float64, device=x.device)
    # the middle between two neighbours goes to the one with the even code
    middles = (grid[1:] + grid[:-1]) / 2
    out = torch.empty_like(x)
    for lo in range(0, x.shape[0], 1024):
        b = x[lo:lo + 1024].reshape(-1, 32)
        amax = b.abs().amax(dim=1, keepdim=True)
        e = torch.floor(torch.log2(amax))
        e = torch.where(torch.pow(2.0, e + 1) <= amax, e + 1, e)  # a logarithm just below a whole number
        scale = torch.where(amax > 0, torch.pow(2.0, e.clamp(-125, 129) - 2), 1.0)
        m = b.abs() / scale
        below, at_or_below = torch.bucketize(m, middles), torch.bucketize(m, middles, right=True)
        code = torch.where(below % 2 == 0, below, at_or_below)
        out[lo:lo + 1024] = (torch.where(b < 0, -1.0, 1.0) * grid[code] * scale).reshape(-1, x.shape[1])
    return out


def _exact_product(data, case):
    c = _exact_values(data["a_codes"], data["a_scales"]) @ _exact_values(data["b_codes"], data["b_scales"]).T
    if data["bias"] is not None:
        c += data["bias"].double()
    return torch.relu_(c) if case["relu"] else c


def _exact_rows(data, case, row_weights, tau, count_scale):
    """Loss rows and gradients of sum_t s_t * (lse(z_t) - sum_v a_tv z_tv + c_t), z = x.w^T / tau, with
    the weights of a row block given by ``row_weights(lo, hi) -> (a, c, kept)``."""
    x, w = data["x"].double(), data["w"].double()
    tokens = x.shape[0]
    rows = torch.zeros(tokens, dtype=torch.float64, device=x.device)
    dx, dw = torch.zeros_like(x), torch.zeros_like(w)
    block = max(1, min(tokens, (1 << 28) // w.shape[0]))
    for lo in range(0, tokens, block):
        hi = min(tokens, lo + block)
        a, c, kept = row_weights(lo, hi)
        z = torch.addmm(torch.zeros(1, dtype=torch.float64, device=x.device), x[lo:hi], w.T, alpha=1.0 / tau)
        lse = torch.logsumexp(z, dim=1)
        rows[lo:hi] = torch.where(kept, lse - (a * z).sum(dim=1) + c, 0.0)
        if case["grad"]:
            z.sub_(lse[:, None]).exp_().sub_(a)
            z[~kept] = 0.0
            z *= count_scale / tau
            dx[lo:hi] = z @ w
            dw.addmm_(z.T, x[lo:hi])
    return rows, dx, dw


def _exact_xent(data, case):
    target, vocab, eps = data["target"], case["vocab"], case["smoothing"]
    scale = 1.0 / float((target != -100).sum()) if case["reduction"] == "mean" else 1.0

    def weights(lo, hi):
        t = target[lo:hi]
        kept = t != -100
        a = torch.full((hi - lo, vocab), eps / vocab, dtype=torch.float64, device=t.device)
        i = torch.nonzero(kept)[:, 0]
        a[i, t[i]] += 1.0 - eps
        return a, torch.zeros(hi - lo, dtype=torch.float64, device=t.device), kept

    rows, dx, dw = _exact_rows(data, case, weights, 1.0, scale)
    loss = rows if case["reduction"] == "none" else rows.sum() * scale
    return (loss, dx, dw) if case["grad"] else loss


def _exact_distill(data, case):
    ids, tau, vocab = data["teacher_ids"], case["temperature"], case["vocab"]
    kept_all = (ids >= 0).any(dim=1)
    scale = tau * tau / float(kept_all.sum())

    def weights(lo, hi):
        i, kept = ids[lo:hi], kept_all[lo:hi]
        t = data["teacher_logits"][lo:hi].double() / tau
        t[i < 0] = -torch.inf
        t[~kept] = 0.0
        p = torch.softmax(t, dim=1)
        entropy = torch.special.entr(p).sum(dim=1)
        a = torch.zeros((hi - lo, vocab + 1), dtype=torch.float64, device=i.device)
        a.scatter_add_(1, torch.where(i < 0, vocab, i), p)
        return a[:, :vocab], -entropy, kept

    rows, dx, dw = _exact_rows(data, case, weights, tau, scale)
    loss = rows.sum() * scale
    return (loss, dx, dw) if case["grad"] else loss


def exact(case, seed):
    return globals()["_exact_" + case["op"]](_inputs(case, seed), case)
