"""Cross entropy and distillation of a head's product against their formulas in 64 bits.

Bounds (u = half a step of the 16-bit type, torch.finfo(t).eps / 2; s = |x| . |w|^T):
* a logit is a sum of exact products, 16 to an MMA, so at most hidden/16 + 1 roundings of at most
  2^-23 (the accumulator may truncate) of partial sums of at most s: dz = (hidden/16 + 1) 2^-23 s;
* exponentials: the argument's rounding, |z - max| * 2^-24, and the approximation's 2 ulp; the sums of
  a tile and of the tiles each add a few fp32 roundings: 2^-16 covers them for arguments up to 64;
* loss: twice dz, that, and the rounding of lse: 2^-22 |lse|;
* G = c (softmax - labels) is rounded once to 16 bits: u |G|, and softmax is off by r = 2 dz + 2^-16
  relative; dX = G w then by (u + K/16 2^-23) |G| |w| + r c softmax |w|, plus u |dX| of its own rounding.
The worst case of a long sum is loose, so the norm is tested, too: the roundings of G's entries are
independent, hence |error|^2 <= sum u^2 G^2 w^2 in the mean (half a step is an upper bound of their
deviation, which is a step / sqrt(12)) plus the systematic parts."""

import math

import numpy as np
import pytest
import torch

import aster_b200.torch_op as top
from aster_b200 import _native as nat
from aster_b200 import head_loss as hl

BF16, F16 = torch.bfloat16, torch.float16


def make(T, D, V, dtype, seed, spread=2.0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    x = torch.randn(T, D, device="cuda", generator=g).to(dtype)
    w = (spread / math.sqrt(D) * torch.randn(V, D, device="cuda", generator=g)).to(dtype)
    return x, w, g


class Reference:
    """Loss rows, G and gradients in 64 bits for row weights `labels` [T, V] (probabilities), `const` [T] and `kept` [T]."""

    def __init__(self, x, w, labels, const, kept, tau=1.0, reduction="mean", grad=None):
        self.x, self.w, self.tau, self.dtype = x.double(), w.double(), tau, x.dtype
        z = self.x @ self.w.T / tau
        self.lse = torch.logsumexp(z, 1)
        q = torch.exp(z - self.lse[:, None])
        self.rows = torch.where(kept, tau * tau * (self.lse - (labels * z).nan_to_num(0.0).sum(1) + const), 0.0)
        n = kept.sum().double()
        share = 1.0 / n if reduction == "mean" else 1.0
        self.loss = self.rows if reduction == "none" else self.rows.sum() * share
        grad = torch.ones((), dtype=torch.float64, device=x.device) if grad is None else grad.double()
        self.c = torch.where(kept, tau * share * grad * torch.ones_like(self.rows), 0.0)
        self.g = self.c[:, None] * (q - labels)
        self.q = self.c.abs()[:, None] * q
        self.dx, self.dw = self.g @ self.w, self.g.T @ self.x
        D = x.shape[1]
        s = (self.x.abs() @ self.w.abs().T) / tau
        self.dz = (D / 16 + 1) * 2.0 ** -23 * s.amax(1)
        self.row_tol = tau * tau * (2 * self.dz + 2.0 ** -16 + 2.0 ** -22 * self.lse.abs())

    def check_loss(self, loss):
        if self.loss.dim():
            assert bool(((loss.double() - self.loss).abs() <= self.row_tol).all())
        else:
            n = self.rows.numel()
            scale = float(self.loss / self.rows.sum()) if float(self.rows.sum()) else 1.0
            tol = float(self.row_tol.sum()) * abs(scale) + n * 2.0 ** -24 * abs(float(self.loss))
            assert abs(loss.item() - float(self.loss)) <= tol

    def check_grad(self, got, want, a, q, other, k):
        """`got` against a @ other, a being G or its transpose."""
        u = torch.finfo(self.dtype).eps / 2
        r = float(2 * self.dz.max()) + 2.0 ** -16
        # the smallest fp16 numbers are 2^-24 apart
        tiny = 2.0 ** -24 if self.dtype == F16 else 0.0
        sys = r * (q @ other.abs()) + k / 16 * 2.0 ** -23 * (a.abs() @ other.abs()) + u * want.abs() + tiny
        worst = u * (a.abs() @ other.abs()) * 1.01 + sys
        err = (got.double() - want).abs()
        assert bool((err <= worst).all()), float((err / worst).max())
        mean_square = u * u * ((a * a) @ (other * other)).sum()
        assert float(err.norm()) <= float(mean_square.sqrt()) + float(sys.norm())

    def check_grads(self, dx, dw):
        self.check_grad(dx, self.dx, self.g, self.q, self.w, self.w.shape[0])
        self.check_grad(dw, self.dw, self.g.T, self.q.T, self.x, self.x.shape[0])


def xent_reference(x, w, target, eps=0.0, ignore=-100, **kw):
    T, V = x.shape[0], w.shape[0]
    kept = target != ignore
    labels = torch.full((T, V), eps / V, dtype=torch.float64, device=x.device)
    i = torch.nonzero(kept)[:, 0]
    labels[i, target[i].long()] += 1 - eps
    return Reference(x, w, labels, torch.zeros(T, dtype=torch.float64, device=x.device), kept, **kw)


def distill_reference(x, w, logits, ids, tau, **kw):
    T, V = x.shape[0], w.shape[0]
    t = logits.double() / tau
    listed = (ids >= 0) & (t != -math.inf)
    kept = listed.any(1)
    t = torch.where(kept[:, None], torch.where(listed, t, -math.inf), 0.0)
    p = torch.where(listed, torch.softmax(t, 1), 0.0)
    labels = torch.zeros((T, V), dtype=torch.float64, device=x.device)
    labels.scatter_add_(1, torch.where(listed, ids, 0).long(), p)
    return Reference(x, w, labels, -torch.special.entr(p).sum(1), kept, tau=tau, **kw)


def targets(T, V, g, ignored=0.2):
    t = torch.randint(0, V, (T,), device="cuda", generator=g)
    t = torch.where(torch.rand(T, device="cuda", generator=g) < ignored, -100, t)
    t[0] = V - 1
    return t


def teacher(T, V, top, g, dtype=torch.float32, duplicates=False):
    if duplicates:
        ids = torch.randint(0, V, (T, top), device="cuda", generator=g)
    else:
        ids = torch.argsort(torch.rand(T, V, device="cuda", generator=g), 1)[:, :top]
    logits = (3 * torch.randn(T, top, device="cuda", generator=g)).to(dtype)
    gone = torch.rand(T, top, device="cuda", generator=g)
    ids = torch.where(gone < 0.1, -1, ids)
    logits = torch.where(gone > 0.95, -math.inf, logits)
    if T > 2:
        ids[1], logits[2] = -7, -math.inf  # rows with nothing left
    ids[0, 0], logits[0, 0] = V - 1, 1.0
    return ids, logits


SHAPES = [(1, 8, 1), (1, 64, 50), (7, 64, 257), (33, 128, 1000), (65, 200, 130), (128, 256, 512), (130, 72, 4097), (257, 264, 3001), (300, 520, 2048), (600, 1032, 5003),
          (3, 1040, 261), (20, 2056, 700), (50, 1200, 90)]


class TestOnHost:
    def test_cpu_tensors_are_refused(self):
        x, w = torch.zeros(4, 16, dtype=BF16), torch.zeros(32, 16, dtype=BF16)
        with pytest.raises(RuntimeError, match="no CPU path"):
            hl.linear_cross_entropy(x, w, torch.zeros(4, dtype=torch.long))
        with pytest.raises(RuntimeError, match="no CPU path"):
            hl.linear_distillation(x, w, torch.zeros(4, 2), torch.zeros(4, 2, dtype=torch.long))

    def test_fake_shapes(self):
        x, w = torch.empty(2, 5, 64, dtype=BF16, device="meta"), torch.empty(100, 64, dtype=BF16, device="meta")
        t = torch.empty(2, 5, dtype=torch.long, device="meta")
        loss, lse, saved = torch.ops.aster_b200.linear_cross_entropy(x, w, t, -100, 0.0, "none")
        assert loss.shape == (2, 5) and lse.shape == (10,) and loss.dtype == lse.dtype == torch.float32 and saved.dtype == torch.uint8
        loss, _, saved = torch.ops.aster_b200.linear_distillation(x, w, torch.empty(2, 5, 7, device="meta"), torch.empty(2, 5, 7, dtype=torch.long, device="meta"))
        assert loss.shape == () and saved.numel() == 256 + 256 + 2 * 512

    @staticmethod
    def desc(**change):
        d = nat.HeadDesc()
        d.tokens, d.hidden, d.vocab, d.x_stride, d.w_stride = 64, 128, 1000, 128, 128
        d.kind, d.dtype, d.reduction, d.index_bits, d.top, d.dtype_teacher, d.temperature = nat.HEAD_CROSS_ENTROPY, nat.BF16, nat.REDUCE_MEAN, 64, 4, nat.F32, 1.0
        for k, v in change.items():
            setattr(d, k, v)
        return d

    def test_refused_descriptions(self, native_lib):
        distill = dict(kind=nat.HEAD_DISTILL)
        for change, text in ((dict(tokens=0), "tokens"), (dict(vocab=0), "vocab"), (dict(hidden=4), "hidden"), (dict(hidden=12, x_stride=16, w_stride=16), "multiple of 8"),
                             (dict(x_stride=120), "x_stride"), (dict(w_stride=132), "w_stride"), (dict(dtype=nat.F32), "dtype"), (dict(reduction=3), "reduction"),
                             (dict(index_bits=16), "index_bits"), (dict(kind=2), "kind"), (dict(label_smoothing=1.0), "label_smoothing"), (dict(label_smoothing=-0.1), "label_smoothing"),
                             (dict(label_smoothing=math.nan), "label_smoothing"), (dict(grad_bytes=-1), "grad_bytes"), (dict(tokens=1 << 31), "below 2"),
                             (dict(top=0, **distill), "top"), (dict(top=1025, **distill), "top"), (dict(temperature=0.0, **distill), "temperature"),
                             (dict(temperature=math.inf, **distill), "temperature"), (dict(temperature=math.nan, **distill), "temperature"), (dict(dtype_teacher=nat.I8, **distill), "dtype_teacher")):
            with pytest.raises(nat.B200Error, match=text):
                hl._sizes(self.desc(**change))

    def test_sizes(self, native_lib):
        """Ranges of the vocabulary respect the limit, cover it, and are whole 64-column groups."""
        for T, D, V in SHAPES + [(8192, 4096, 32768), (100000, 512, 131072), (8, 4096, 131072)]:
            for limit in (0, 1 << 20, 1 << 30):
                s = hl._sizes(self.desc(tokens=T, hidden=D, vocab=V, x_stride=D, w_stride=D, grad_bytes=limit))
                assert s.grad_columns % 64 == 0 and s.grad_columns < V + 256
                assert s.grad_columns * T * 2 <= max(limit or 256 << 20, 256 * T * 2)
                assert s.cta_group in (1, 2) and s.tile_n % 32 == 0 and 64 <= s.tile_n <= 256
                assert s.backward_workspace >= s.grad_columns * T * 2

    def test_refused_calls(self, native_lib):
        """Refused before anything touches a device: the addresses are never read."""
        import ctypes as C

        d, ok = self.desc(), 1 << 20
        f = lambda **k: nat.call("b200_head_loss_forward", C.byref(k.get("d", d)), *(k.get(n, ok) for n in ("x", "w", "labels")), k.get("teacher"),
                                 *(k.get(n, ok) for n in ("loss", "lse", "saved", "ws")), k.get("bytes", 1 << 30), None)
        for k, text in ((dict(x=None), "NULL"), (dict(w=ok + 8), "16-byte"), (dict(labels=ok + 4), "aligned"), (dict(ws=None), "workspace"), (dict(bytes=100), "workspace"),
                        (dict(teacher=ok), "teacher_logits"), (dict(d=self.desc(kind=nat.HEAD_DISTILL)), "teacher_logits"), (dict(loss=None), "NULL")):
            with pytest.raises(nat.B200Error, match=text):
                f(**k)
        b = lambda **k: nat.call("b200_head_loss_backward", C.byref(d), *(k.get(n, ok) for n in ("x", "w", "labels", "lse", "saved", "grad", "dx", "dw", "ws")), k.get("bytes", 1 << 30), None)
        for k, text in ((dict(lse=None), "NULL"), (dict(grad=None), "NULL"), (dict(saved=None), "NULL"), (dict(bytes=100), "workspace")):
            with pytest.raises(nat.B200Error, match=text):
                b(**k)


@pytest.mark.gpu
class TestCrossEntropy:
    @pytest.mark.parametrize("dtype", [BF16, F16])
    @pytest.mark.parametrize("shape", SHAPES)
    @pytest.mark.parametrize("eps", [0.0, 0.1])
    def test_mean_with_gradients(self, gpu, shape, dtype, eps):
        T, D, V = shape
        x, w, g = make(T, D, V, dtype, T + V)
        t = targets(T, V, g)
        ref = xent_reference(x, w, t, eps)
        x.requires_grad_(), w.requires_grad_()
        loss = hl.linear_cross_entropy(x, w, t, label_smoothing=eps)
        ref.check_loss(loss)
        ref.check_grads(*torch.autograd.grad(loss, (x, w)))
        assert hl.head_loss_status() == [0, 0, 0, 0]

    @pytest.mark.parametrize("shape", [(7, 64, 257), (130, 72, 4097), (300, 520, 2048)])
    @pytest.mark.parametrize("dtype", [BF16, F16])
    def test_rows_and_sum(self, gpu, shape, dtype):
        T, D, V = shape
        x, w, g = make(T, D, V, dtype, T)
        x.requires_grad_(), w.requires_grad_()
        t = targets(T, V, g).int()
        # factors over many orders of magnitude, one of them zero
        grad = torch.randn(T, device="cuda", generator=g) * torch.exp(3 * torch.randn(T, device="cuda", generator=g)) * 1e-3
        grad[T // 2] = 0
        ref = xent_reference(x.detach(), w.detach(), t, reduction="none", grad=grad)
        loss = hl.linear_cross_entropy(x, w, t, reduction="none")
        assert loss.shape == t.shape
        ref.check_loss(loss)
        ref.check_grads(*torch.autograd.grad(loss, (x, w), grad))
        ref = xent_reference(x.detach(), w.detach(), t, reduction="sum", grad=torch.tensor(-0.37))
        loss = hl.linear_cross_entropy(x, w, t, reduction="sum")
        ref.check_loss(loss)
        ref.check_grads(*torch.autograd.grad(loss, (x, w), torch.tensor(-0.37, device="cuda")))

    @pytest.mark.parametrize("limit", [1, 300 * 2 * 512, 300 * 2 * 1024])
    def test_ranges_of_the_vocabulary(self, gpu, limit):
        x, w, g = make(300, 136, 2500, BF16, 5)
        t = targets(300, 2500, g)
        ref = xent_reference(x, w, t)
        x.requires_grad_(), w.requires_grad_()
        ref.check_grads(*torch.autograd.grad(hl.linear_cross_entropy(x, w, t, grad_bytes=limit), (x, w)))

    @pytest.mark.parametrize("shape", [(5000, 64, 300), (3000, 264, 700), (6001, 136, 1500)])
    @pytest.mark.parametrize("dtype", [BF16, F16])
    def test_many_tokens_and_few_tiles(self, gpu, shape, dtype):
        """dW's few tiles are cut along the tokens; in one range and in several."""
        T, D, V = shape
        x, w, g = make(T, D, V, dtype, 50 + V)
        t = targets(T, V, g)
        ref = xent_reference(x, w, t, 0.1)
        x.requires_grad_(), w.requires_grad_()
        for limit in (0, 2 * T * 256, 2 * T * 512):
            loss = hl.linear_cross_entropy(x, w, t, label_smoothing=0.1, grad_bytes=limit)
            ref.check_loss(loss)
            ref.check_grads(*torch.autograd.grad(loss, (x, w)))

    def test_larger_than_the_grid(self, gpu):
        """Several rounds of pair tiles, several ranges, cut and uncut vocabulary axes."""
        x, w, g = make(1500, 512, 20011, BF16, 6)
        t = targets(1500, 20011, g)
        ref = xent_reference(x, w, t)
        x.requires_grad_(), w.requires_grad_()
        for limit in (0, 1500 * 2 * 8192):
            loss = hl.linear_cross_entropy(x, w, t, grad_bytes=limit)
            ref.check_loss(loss)
            ref.check_grads(*torch.autograd.grad(loss, (x, w)))

    def test_offsets_beyond_32_bits(self, gpu):
        """A stored range of dL/dz of more than 2^31 elements (4.4 GB) gives what short ranges give."""
        T, D, V = 66000, 64, 33001
        x, w, g = make(T, D, V, BF16, 19)
        t = targets(T, V, g)
        x.requires_grad_(), w.requires_grad_()
        assert hl._sizes(hl._xent_head(x, w, t, -100, 0.0, "mean", 1 << 34).desc).grad_columns * T > 1 << 31
        long = torch.autograd.grad(hl.linear_cross_entropy(x, w, t, grad_bytes=1 << 34), (x, w))
        short = torch.autograd.grad(hl.linear_cross_entropy(x, w, t), (x, w))
        # another order of the same sums (fp32 roundings), rounded to bf16
        for a, b in zip(long, short):
            assert bool(((a.double() - b.double()).abs() <= 2.0 ** -7 * b.double().abs() + 2.0 ** -15 * b.double().abs().max()).all())
        rows = torch.tensor([0, T - 1, T // 2, 65535], device="cuda")
        q = torch.softmax(x.detach()[rows].double() @ w.detach().double().T, 1)
        kept = t[rows] >= 0
        q[torch.nonzero(kept)[:, 0], t[rows][kept]] -= 1
        want = torch.where(kept[:, None], q @ w.detach().double() / (t >= 0).sum(), 0.0)
        assert bool(((long[0][rows].double() - want).abs() <= 2.0 ** -6 * want.abs().max()).all())

    def test_against_differences(self, gpu):
        x, w, g = make(40, 64, 300, F16, 7)
        t = targets(40, 300, g)
        h = 2.0 ** -4
        step = torch.randn(40, 64, device="cuda", generator=g)
        a, b = (x.float() - h * step).half(), (x.float() + h * step).half()
        la, lb = (xent_reference(v, w, t, reduction="sum") for v in (a, b))
        mid = ((a.double() + b.double()) / 2).half()
        ref = xent_reference(mid, w, t, reduction="sum")
        mid.requires_grad_()
        dx, = torch.autograd.grad(hl.linear_cross_entropy(mid, w, t, reduction="sum"), mid)
        delta = b.double() - a.double()
        difference = float(lb.loss - la.loss)
        # what the difference quotient itself misses (and the rounding of the midpoint), from the 64-bit gradient
        quotient = abs(difference - float((ref.dx * delta).sum()))
        tol = quotient + 2.0 ** -10 * float(((ref.g.abs() @ w.double().abs()) * delta.abs()).sum())
        assert abs(float((dx.double() * delta).sum()) - difference) <= tol
        assert quotient < 0.1 * abs(difference)

    def test_masked_rows(self, gpu):
        x, w, g = make(40, 64, 300, BF16, 8)
        t = torch.full((40,), -100, device="cuda")
        x.requires_grad_(), w.requires_grad_()
        for reduction in ("mean", "sum", "none"):
            loss = hl.linear_cross_entropy(x, w, t, reduction=reduction)
            assert bool(torch.isnan(loss)) if reduction == "mean" else bool((loss == 0).all())
            dx, dw = torch.autograd.grad(loss.sum(), (x, w))
            assert bool((dx == 0).all()) and bool((dw == 0).all())
        # another ignored class, which is a valid index, too
        t = torch.randint(0, 4, (40,), device="cuda", generator=g)
        loss = hl.linear_cross_entropy(x, w, t, ignore_index=2)
        xent_reference(x.detach(), w.detach(), t, ignore=2).check_loss(loss)

    def test_ignored_rows_hide_what_they_hold(self, gpu):
        x, w, g = make(70, 64, 300, BF16, 9)
        t = targets(70, 300, g, 0.0)
        t[[5, 40]] = -100
        clean = hl.linear_cross_entropy(x, w, t)
        x[5], x[40, 3] = math.nan, math.inf
        x.requires_grad_()
        loss = hl.linear_cross_entropy(x, w, t)
        dx, = torch.autograd.grad(loss, x)
        assert torch.equal(loss, clean) and bool((dx[[5, 40]] == 0).all()) and bool(torch.isfinite(dx).all())

    def test_bad_targets_and_logits_show(self, gpu):
        x, w, g = make(70, 64, 300, BF16, 10)
        t = targets(70, 300, g, 0.0)
        t[3], t[50], t[60] = 300, -1, 1 << 40
        x.data[20, 0] = math.nan
        x.requires_grad_()
        loss = hl.linear_cross_entropy(x, w, t, reduction="none")
        bad = torch.zeros(70, dtype=torch.bool, device="cuda")
        bad[[3, 20, 50, 60]] = True
        assert torch.equal(torch.isnan(loss), bad)
        dx, = torch.autograd.grad(loss.sum(), x)
        assert torch.equal(torch.isnan(dx).all(1), bad) and torch.equal(torch.isnan(dx).any(1), bad)

    def test_extreme_logits(self, gpu):
        """Logits of some hundreds, minus infinity for part of the vocabulary, and for all of a row."""
        x, w, g = make(40, 64, 700, BF16, 11, spread=100.0)
        w[100:200, 0] = -math.inf
        x[:, 0] = 1.0
        t = targets(40, 700, g, 0.0)
        t[(t >= 100) & (t < 200)] = 7
        ref = xent_reference(x, w[torch.isfinite(w[:, 0])], torch.where(t >= 200, t - 100, t))
        loss = hl.linear_cross_entropy(x, w, t, reduction="none")
        assert bool(((loss.double() - ref.rows).abs() <= ref.row_tol + 2.0 ** -24 * 700).all())
        w[:, 0] = -math.inf
        assert bool(torch.isnan(hl.linear_cross_entropy(x, w, t, reduction="none")).all())  # no distribution left

    def test_views_streams_and_partial_gradients(self, gpu):
        g = torch.Generator(device="cuda").manual_seed(12)
        base_x = torch.randn(6, 9, 200, device="cuda", generator=g).to(BF16)
        base_w = (0.2 * torch.randn(500, 144, device="cuda", generator=g)).to(BF16)
        for x, w in ((base_x[..., :136], base_w[:, 8:144]), (base_x[:, ::2, 3:139], base_w[:, 4:140]), (base_x[..., :136].transpose(0, 1), base_w[::2, :136])):
            t = torch.randint(0, w.shape[0], x.shape[:-1], device="cuda", generator=g)
            xc, wc = x.clone(memory_format=torch.contiguous_format).requires_grad_(), w.clone(memory_format=torch.contiguous_format).requires_grad_()
            want = hl.linear_cross_entropy(xc, wc, t, reduction="none")
            gx, gw = torch.autograd.grad(want.sum(), (xc, wc))
            x, w = x.detach().requires_grad_(), w.detach().requires_grad_()
            side = torch.cuda.Stream()
            side.wait_stream(torch.cuda.current_stream())
            with torch.cuda.stream(side):
                loss = hl.linear_cross_entropy(x, w, t, reduction="none")
                total = loss.sum()
                dx, = torch.autograd.grad(total, x, retain_graph=True)
                dw, = torch.autograd.grad(total, w)
            torch.cuda.current_stream().wait_stream(side)
            assert loss.shape == t.shape and torch.equal(loss, want) and torch.equal(dx, gx) and torch.equal(dw, gw)

    def test_no_tokens(self, gpu):
        x, w = torch.zeros(0, 64, device="cuda", dtype=BF16, requires_grad=True), torch.zeros(30, 64, device="cuda", dtype=BF16, requires_grad=True)
        t = torch.zeros(0, dtype=torch.long, device="cuda")
        assert math.isnan(hl.linear_cross_entropy(x, w, t).item()) and hl.linear_cross_entropy(x, w, t, reduction="none").shape == (0,)
        dx, dw = torch.autograd.grad(hl.linear_cross_entropy(x, w, t, reduction="sum"), (x, w))
        assert dx.shape == (0, 64) and bool((dw == 0).all())

    def test_refusals(self, gpu):
        x, w, _ = make(8, 64, 100, BF16, 13)
        t = torch.zeros(8, dtype=torch.long, device="cuda")
        for args, kw in (((x.float(), w.float(), t), {}), ((x.half(), w, t), {}), ((x[:, :60], w[:, :60], t), {}), ((x, w[:, :56], t), {}), ((x, w, t[:7]), {}), ((x, w, t.float()), {}),
                         ((x, w, t.cpu()), {}), ((x, w, t), {"reduction": "avg"}), ((x, w, t), {"label_smoothing": 1.0}), ((x[0], w, t[0]), {}), ((x, w[:0], t), {})):
            with pytest.raises(RuntimeError):
                hl.linear_cross_entropy(*args, **kw)

    def test_same_bits_every_time(self, gpu):
        x, w, g = make(700, 256, 9001, BF16, 14)
        t = targets(700, 9001, g)
        x.requires_grad_(), w.requires_grad_()
        first = None
        for _ in range(5):
            loss = hl.linear_cross_entropy(x, w, t, label_smoothing=0.05)
            got = (loss.detach(), *torch.autograd.grad(loss, (x, w)))
            first = first or got
            assert all(torch.equal(a, b) for a, b in zip(first, got))

    def test_captured_step(self, gpu):
        x, w, g = make(200, 128, 3000, BF16, 15)
        t = targets(200, 3000, g)
        x.requires_grad_(), w.requires_grad_()
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            torch.autograd.grad(hl.linear_cross_entropy(x, w, t), (x, w))
        torch.cuda.current_stream().wait_stream(side)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            loss = hl.linear_cross_entropy(x, w, t)
            dx, dw = torch.autograd.grad(loss, (x, w))
        for seed in range(3):
            with torch.no_grad():
                x.copy_(torch.randn(200, 128, generator=torch.Generator().manual_seed(seed)))
                t.copy_(torch.randint(0, 3000, (200,), generator=torch.Generator().manual_seed(seed)))
            graph.replay()
            xe, we = x.detach().requires_grad_(), w.detach().requires_grad_()
            want = hl.linear_cross_entropy(xe, we, t)
            wx, ww = torch.autograd.grad(want, (xe, we))
            assert torch.equal(loss, want) and torch.equal(dx, wx) and torch.equal(dw, ww)

    @pytest.mark.parametrize("distill", [False, True])
    def test_capture_beside_an_eager_graph_of_the_same_leaves_is_refused(self, gpu, distill):
        x, w, g = make(64, 64, 500, BF16, 18)
        t = targets(64, 500, g)
        ids, logits = teacher(64, 500, 4, g)
        x.requires_grad_(), w.requires_grad_()
        call = (lambda: hl.linear_distillation(x, w, logits, ids)) if distill else (lambda: hl.linear_cross_entropy(x, w, t))
        alive = call()
        with pytest.raises(RuntimeError, match="still alive"):
            with torch.cuda.graph(torch.cuda.CUDAGraph()):
                call()
        alive.backward()  # the eager graph is none the worse for it
        assert bool(torch.isfinite(x.grad).all())
        x.grad = w.grad = None
        del alive
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            dx, dw = torch.autograd.grad(call(), (x, w))
        graph.replay()
        want = torch.autograd.grad(call(), (x, w))
        assert torch.equal(dx, want[0]) and torch.equal(dw, want[1])

    def test_from_other_threads(self, gpu):
        """Threads whose first CUDA call is the loss, or its backward pass, all at once."""
        import threading

        problems = [make(60 + i, 64, 900, BF16, 40 + i) for i in range(4)]
        labels = [targets(60 + i, 900, p[2]) for i, p in enumerate(problems)]
        leaves = [(p[0].requires_grad_(), p[1].requires_grad_()) for p in problems]
        want = [torch.autograd.grad(hl.linear_cross_entropy(*l, t), l) for l, t in zip(leaves, labels)]
        torch.cuda.synchronize()
        got, errors = {}, []

        def work(i):
            try:
                for _ in range(10):
                    got[i] = torch.autograd.grad(hl.linear_cross_entropy(*leaves[i], labels[i]), leaves[i])
                torch.cuda.synchronize()
            except Exception as e:
                errors.append(e)

        threads = [threading.Thread(target=work, args=(i,)) for i in range(4)]
        for t in threads:
            t.start()
        for t in threads:
            t.join()
        assert not errors
        assert all(torch.equal(a, b) for i in range(4) for a, b in zip(got[i], want[i]))

    def test_operator_of_the_dispatcher(self, gpu):
        x, w, g = make(50, 64, 400, BF16, 16)
        t = targets(50, 400, g)
        x.requires_grad_(), w.requires_grad_()
        want = hl.linear_cross_entropy(x, w, t, label_smoothing=0.1)
        gx, gw = torch.autograd.grad(want, (x, w))
        loss, lse, _ = torch.ops.aster_b200.linear_cross_entropy(x, w, t, -100, 0.1, "mean")
        dx, dw = torch.autograd.grad(loss, (x, w))
        assert torch.equal(loss, want) and torch.equal(dx, gx) and torch.equal(dw, gw)
        ref = xent_reference(x.detach(), w.detach(), t)
        assert bool(((lse.double() - ref.lse).abs() <= ref.row_tol).all())

    def test_changed_inputs_are_noticed(self, gpu):
        x, w, g = make(8, 64, 100, BF16, 17)
        x.requires_grad_(), w.requires_grad_()
        t = targets(8, 100, g)
        loss = hl.linear_cross_entropy(x, w, t)
        with torch.no_grad():
            w.mul_(2)
        with pytest.raises(RuntimeError, match="modified by an inplace operation"):
            loss.backward()


@pytest.mark.gpu
class TestDistillation:
    @pytest.mark.parametrize("dtype", [BF16, F16])
    @pytest.mark.parametrize("case", [(1, 8, 1, 1, 1.0), (1, 64, 50, 3, 2.0), (7, 64, 257, 7, 1.0), (33, 128, 1000, 64, 0.7), (65, 200, 130, 130, 1.5), (130, 72, 4097, 17, 2.0),
                                      (257, 264, 3001, 128, 1.0), (600, 1032, 5003, 64, 3.0), (40, 64, 2000, 1000, 1.0)])
    def test_mean_with_gradients(self, gpu, case, dtype):
        T, D, V, k, tau = case
        x, w, g = make(T, D, V, dtype, T + V + k)
        ids, logits = teacher(T, V, k, g)
        ref = distill_reference(x, w, logits, ids, tau)
        x.requires_grad_(), w.requires_grad_()
        loss = hl.linear_distillation(x, w, logits, ids, temperature=tau)
        ref.check_loss(loss)
        ref.check_grads(*torch.autograd.grad(loss, (x, w)))
        assert hl.head_loss_status() == [0, 0, 0, 0]

    @pytest.mark.parametrize("teacher_dtype", [torch.float32, BF16, F16])
    @pytest.mark.parametrize("index", [torch.int32, torch.int64])
    def test_rows_duplicates_and_types(self, gpu, teacher_dtype, index):
        x, w, g = make(90, 72, 600, BF16, 21)
        ids, logits = teacher(90, 600, 24, g, teacher_dtype, duplicates=True)
        ids[3] = 17  # one id 24 times
        ids[4, ::2] = ids[4, 1::2]
        ids = ids.to(index)
        grad = torch.randn(90, device="cuda", generator=g)
        ref = distill_reference(x, w, logits, ids, 1.3, reduction="none", grad=grad)
        x.requires_grad_(), w.requires_grad_()
        loss = hl.linear_distillation(x, w, logits, ids, temperature=1.3, reduction="none")
        ref.check_loss(loss)
        assert bool((loss[[1, 2]] == 0).all())  # rows with nothing left
        dx, dw = torch.autograd.grad(loss, (x, w), grad)
        ref.check_grads(dx, dw)
        assert bool((dx[[1, 2]] == 0).all())

    def test_ranges_of_the_vocabulary(self, gpu):
        x, w, g = make(300, 136, 2500, BF16, 22)
        ids, logits = teacher(300, 2500, 40, g)
        ids[5:50, :20] = torch.arange(500, 520, device="cuda")  # around a range's edge
        ref = distill_reference(x, w, logits, ids, 2.0)
        x.requires_grad_(), w.requires_grad_()
        ref.check_grads(*torch.autograd.grad(hl.linear_distillation(x, w, logits, ids, temperature=2.0, grad_bytes=300 * 2 * 512), (x, w)))

    @pytest.mark.parametrize("operand", ["x", "w"])
    def test_against_differences(self, gpu, operand):
        x, w, g = make(40, 64, 300, F16, 28)
        ids, logits = teacher(40, 300, 12, g)
        loss64 = lambda x, w: distill_reference(x, w, logits, ids, 1.5, reduction="sum")
        base = x if operand == "x" else w
        step = 2.0 ** -4 * torch.randn(base.shape, device="cuda", generator=g) * base.float().std()
        a, b = (base.float() - step).half(), (base.float() + step).half()
        mid = ((a.double() + b.double()) / 2).half()
        at = lambda v: (v, w) if operand == "x" else (x, v)
        difference = float(loss64(*at(b)).loss - loss64(*at(a)).loss)
        ref = loss64(*at(mid))
        mid.requires_grad_()
        got, = torch.autograd.grad(hl.linear_distillation(*at(mid), logits, ids, temperature=1.5, reduction="sum"), mid)
        delta = b.double() - a.double()
        want, spread = (ref.dx, ref.g.abs() @ ref.w.abs()) if operand == "x" else (ref.dw, ref.g.T.abs() @ ref.x.abs())
        # what the difference quotient itself misses (and the rounding of the midpoint), from the 64-bit gradient
        quotient = abs(difference - float((want * delta).sum()))
        tol = quotient + 2.0 ** -10 * float((spread * delta.abs()).sum())
        assert abs(float((got.double() * delta).sum()) - difference) <= tol
        assert quotient < 0.1 * abs(difference)

    def test_one_certain_entry_is_cross_entropy(self, gpu):
        x, w, g = make(60, 64, 500, BF16, 23)
        t = targets(60, 500, g)
        ids = torch.where(t < 0, -1, t)[:, None]
        a = hl.linear_cross_entropy(x, w, t, reduction="none")
        b = hl.linear_distillation(x, w, torch.zeros(60, 1, device="cuda"), ids, reduction="none")
        ref = xent_reference(x, w, t)
        assert bool(((a - b).double().abs() <= 2 * ref.row_tol).all())

    def test_bad_entries_show(self, gpu):
        x, w, g = make(50, 64, 300, BF16, 24)
        ids, logits = teacher(50, 300, 5, g)
        ids[10:14], logits[10:14] = torch.arange(5, device="cuda"), 0.5
        ids[10, 2], ids[11, 0], logits[12, 1], logits[13, 4] = 300, 1 << 33, math.nan, math.inf
        bad = torch.zeros(50, dtype=torch.bool, device="cuda")
        bad[10:14] = True
        x.requires_grad_()
        loss = hl.linear_distillation(x, w, logits, ids, reduction="none")
        assert torch.equal(torch.isnan(loss), bad)
        dx, = torch.autograd.grad(loss.sum(), x)
        assert torch.equal(torch.isnan(dx).any(1), bad)

    def test_nothing_left_at_all(self, gpu):
        x, w, g = make(20, 64, 300, BF16, 25)
        x.requires_grad_(), w.requires_grad_()
        loss = hl.linear_distillation(x, w, torch.zeros(20, 3, device="cuda"), torch.full((20, 3), -1, device="cuda"))
        assert math.isnan(loss.item())
        dx, dw = torch.autograd.grad(loss, (x, w))
        assert bool((dx == 0).all()) and bool((dw == 0).all())

    def test_refusals(self, gpu):
        x, w, _ = make(8, 64, 100, BF16, 26)
        ids, logits = torch.zeros(8, 3, dtype=torch.long, device="cuda"), torch.zeros(8, 3, device="cuda")
        for args, kw in (((x, w, logits, ids[:, :2]), {}), ((x, w, logits, ids[:7]), {}), ((x, w, logits.double(), ids), {}), ((x, w, logits.cpu(), ids), {}), ((x, w, logits, ids.float()), {}),
                         ((x, w, logits, ids), {"temperature": 0.0}), ((x, w, logits, ids), {"temperature": math.nan}), ((x, w, logits[:, :0], ids[:, :0]), {}),
                         ((x, w, logits, ids), {"reduction": "batchmean"}), ((x, w, torch.zeros(8, 1025, device="cuda"), torch.zeros(8, 1025, dtype=torch.long, device="cuda")), {})):
            with pytest.raises(RuntimeError):
                hl.linear_distillation(*args, **kw)

    def test_operator_of_the_dispatcher(self, gpu):
        x, w, g = make(2 * 25, 64, 400, F16, 27)
        ids, logits = teacher(50, 400, 6, g)
        x = x.view(2, 25, 64).requires_grad_()
        w.requires_grad_()
        ids, logits = ids.view(2, 25, 6), logits.view(2, 25, 6)
        want = hl.linear_distillation(x, w, logits, ids, temperature=2.0)
        gx, gw = torch.autograd.grad(want, (x, w))
        loss, _, _ = torch.ops.aster_b200.linear_distillation(x, w, logits, ids, 2.0, "mean")
        dx, dw = torch.autograd.grad(loss, (x, w))
        assert dx.shape == x.shape and torch.equal(loss, want) and torch.equal(dx, gx) and torch.equal(dw, gw)


@pytest.mark.gpu
def test_a_step_through_all_of_them(gpu):
    """A 4-bit layer feeds the head; its losses train the head and give the layer's output its gradient."""
    T, D, V, k = 150, 256, 3001, 16
    g = torch.Generator(device="cuda").manual_seed(31)
    h = torch.randn(T, 512, device="cuda", generator=g).to(BF16)
    layer = (0.05 * torch.randn(D, 512, device="cuda", generator=g)).to(BF16)
    w = (0.1 * torch.randn(V, D, device="cuda", generator=g)).to(BF16).requires_grad_()
    wq, ws = top.quantize_mx_direct(layer)
    q, s = top.quantize_mx_direct(h)
    x = top.gemm_mx_nt_direct(q, s, wq, ws, out_dtype=BF16)
    exact = top.dequantize_mx_direct(q, s).double() @ top.dequantize_mx_direct(wq, ws).double().T
    bound = 512 * 2.0 ** -23 * (top.dequantize_mx_direct(q, s).double().abs() @ top.dequantize_mx_direct(wq, ws).double().abs().T) + 2.0 ** -8 * exact.abs()
    assert bool(((x.double() - exact).abs() <= bound).all())
    x.requires_grad_()
    t = targets(T, V, g)
    ids, logits = teacher(T, V, k, g)
    refs = (xent_reference(x.detach(), w.detach(), t), distill_reference(x.detach(), w.detach(), logits, ids, 2.0))
    losses = (hl.linear_cross_entropy(x, w, t), hl.linear_distillation(x, w, logits, ids, temperature=2.0))
    for ref, loss in zip(refs, losses):
        ref.check_loss(loss)
        ref.check_grads(*torch.autograd.grad(loss, (x, w), retain_graph=True))
    dx, dw = torch.autograd.grad(losses[0] + 0.5 * losses[1], (x, w))
    assert bool(torch.isfinite(dx).all()) and bool(torch.isfinite(dw).all())
