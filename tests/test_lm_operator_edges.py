"""Calls of the language-model operators from their edges."""

import numpy as np
import pytest
import torch

import aster_b200.torch_op as top
from aster_b200 import _native as nat
from aster_b200 import dtypes
from aster_b200 import head_loss as hl
from aster_b200.gemm import GemmPlan, gemm
import test_head_loss as basics
from test_head_loss import distill_reference, make, teacher

BF16 = torch.bfloat16


def strided_problem(device, T=70, D=136, V=300, seed=3):
    """Rows of x and w wider apart than they are long."""
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(T, 2 * D, generator=g).to(device, BF16)[:, :D]
    w = (0.2 * torch.randn(V, D + 64, generator=g)).to(device, BF16)[:, 8:8 + D]
    t = torch.randint(0, V, (T,), generator=g).to(device)
    return x, w, t


class TestSavedTensors:
    def test_strides_follow_the_tensors_on_the_host(self):
        x, w, t = strided_problem("cpu")
        forward = hl._Head(x, w, t, "mean", kind=0)
        assert (forward.desc.x_stride, forward.desc.w_stride) == (272, 200)
        kept = forward.without_tensors()
        for x2, w2 in ((x.clone(memory_format=torch.contiguous_format), w), (x, w.clone(memory_format=torch.contiguous_format)), (x, w)):
            back = kept.with_tensors(x2, w2, t)
            assert (back.desc.x_stride, back.desc.w_stride) == (back.x.stride(0), back.w.stride(0)) == (x2.stride(0), w2.stride(0))
            assert (back.desc.tokens, back.desc.hidden, back.desc.vocab) == (70, 136, 300)
        assert (kept.desc.x_stride, kept.desc.w_stride) == (272, 200)  # another thread may be reading it

    def test_other_shapes_and_types_are_refused_on_the_host(self):
        x, w, t = strided_problem("cpu")
        kept = hl._Head(x, w, t, "mean", kind=0).without_tensors()
        for x2, w2, t2 in ((x[:60], w, t), (x, w[:299], t), (x, w, t[:69]), (x.float(), w, t), (x.half(), w.half(), t), (x, w, t.int()), (x.to("meta"), w, t)):
            with pytest.raises(RuntimeError, match="came back"):
                kept.with_tensors(x2, w2, t2)

    @pytest.mark.gpu
    @pytest.mark.parametrize("hook", ["clone", "cpu", "strided"])
    @pytest.mark.parametrize("distill", [False, True])
    def test_hooks_that_lay_tensors_out_anew(self, gpu, hook, distill):
        x, w, t = strided_problem("cuda")
        ids = torch.stack([t, (t + 7) % 300], 1)
        logits = torch.tensor([[1.0, 0.5]], device="cuda").expand(70, 2)

        def wide(v):  # rows further apart than they were
            if v.dim() != 2:
                return v
            out = v.new_zeros(v.shape[0], 2 * v.shape[1] + 8)
            out[:, :v.shape[1]] = v
            return out[:, :v.shape[1]]

        hooks = {"clone": torch.autograd.graph.saved_tensors_hooks(lambda v: v, lambda v: v.clone(memory_format=torch.contiguous_format)),
                 "cpu": torch.autograd.graph.save_on_cpu(), "strided": torch.autograd.graph.saved_tensors_hooks(lambda v: v, wide)}[hook]
        x.requires_grad_(), w.requires_grad_()
        call = (lambda: hl.linear_distillation(x, w, logits, ids)) if distill else (lambda: hl.linear_cross_entropy(x, w, t))
        want = torch.autograd.grad(call(), (x, w))
        with hooks:
            loss = call()
        got = torch.autograd.grad(loss, (x, w))
        assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])

    @pytest.mark.gpu
    def test_backward_operator_checks_what_it_is_given(self, gpu):
        x, w, t = strided_problem("cuda")
        loss, lse, saved = torch.ops.aster_b200.linear_cross_entropy(x, w, t)
        back = torch.ops.aster_b200.linear_cross_entropy_backward
        one = torch.ones((), device="cuda")
        for grad, l, s in ((one, lse[:69], saved), (one, lse.double(), saved), (one, lse, saved[:16]), (one, lse, saved.cpu()), (one.expand(70), lse, saved)):
            with pytest.raises(RuntimeError, match="must be"):
                back(grad, x, w, t, l, s, -100, 0.0, "mean")
        with pytest.raises(RuntimeError, match="must be"):
            back(one, x, w, t, lse, saved, -100, 0.0, "none")


class TestForwardMode:
    """A tangent is refused, never dropped."""

    @staticmethod
    def check(x, w, t, ids, logits, dual_x, requires_grad, no_grad, dispatcher=True):
        from torch.autograd import forward_ad

        x, w = x.clone().requires_grad_(requires_grad), w.clone().requires_grad_(requires_grad)
        ops = torch.ops.aster_b200
        with forward_ad.dual_level(), torch.set_grad_enabled(not no_grad):
            if dual_x:
                x = forward_ad.make_dual(x, torch.ones_like(x))
            else:
                w = forward_ad.make_dual(w, torch.ones_like(w))
            calls = [lambda: hl.linear_cross_entropy(x, w, t), lambda: hl.linear_distillation(x, w, logits, ids)]
            if dispatcher:
                calls += [lambda: ops.linear_cross_entropy(x, w, t), lambda: ops.linear_distillation(x, w, logits, ids)]
            for call in calls:
                with pytest.raises((RuntimeError, NotImplementedError), match="forward.mode"):
                    call()

    @pytest.mark.parametrize("dual_x", [True, False])
    @pytest.mark.parametrize("requires_grad", [True, False])
    @pytest.mark.parametrize("no_grad", [True, False])
    def test_on_the_host(self, dual_x, requires_grad, no_grad):
        x, w, t = strided_problem("cpu")
        # with a graph to record, torch refuses the operators itself, but only after their forward pass
        self.check(x, w, t, t[:, None], torch.zeros(70, 1), dual_x, requires_grad, no_grad, dispatcher=no_grad or not requires_grad)

    @pytest.mark.gpu
    @pytest.mark.parametrize("dual_x", [True, False])
    @pytest.mark.parametrize("requires_grad", [True, False])
    @pytest.mark.parametrize("no_grad", [True, False])
    def test_on_the_gpu(self, gpu, dual_x, requires_grad, no_grad):
        x, w, t = strided_problem("cuda")
        self.check(x, w, t, t[:, None], torch.zeros(70, 1, device="cuda"), dual_x, requires_grad, no_grad)
        hl.linear_cross_entropy(x, w, t)  # without a tangent as before


def exact_operand(rows, K, rng):
    """4-bit codes under scales of 1: products are multiples of 1/4 of at most 36, sums of a few thousand exact in fp32."""
    q = dtypes.pack_e2m1(rng.integers(0, 16, (rows, K)).astype(np.uint8))
    scales = np.full((rows, K // 32), 127, np.uint8)
    return q, scales, dtypes.dequantize_mx(q, scales, "e2m1").astype(np.float64)


class TestFewRowsShortK:
    """One K block (K <= 256) is planned like several: narrow tiles for up to 128 rows."""

    @pytest.mark.parametrize("K", [32, 96, 256])
    @pytest.mark.parametrize("M", [1, 16, 60, 128])
    @pytest.mark.parametrize("N", [64, 2048, 65536])
    def test_plan(self, native_lib, M, N, K):
        r = GemmPlan(M, N, K, "mxe2m1", "bf16").resources()
        assert r.cta_group == 1 and r.tail_parts <= 1
        if M > 64 and N > 3 * 148 * 128:  # full tiles in many rounds, whose outputs decide
            assert r.tile_n == 256
        else:
            assert r.tile_n == GemmPlan(M, N, 288, "mxe2m1", "bf16").resources().tile_n and r.tile_n in (64, 128)

    @pytest.mark.gpu
    @pytest.mark.parametrize("K", [32, 160, 256])
    @pytest.mark.parametrize("M", [1, 40, 100, 128])
    @pytest.mark.parametrize("N", [64, 263, 2048, 40000, 60000])
    def test_exact_sums(self, gpu, M, N, K):
        rng = np.random.default_rng(M + N + K)
        (qa, sa, a), (qb, sb, b) = exact_operand(M, K, rng), exact_operand(N, K, rng)
        got = gemm(qa, qb, dtype_ab="mxe2m1", dtype_c="f32", block_scales_a=sa, block_scales_b=sb)
        assert np.array_equal(got, (a @ b.T).astype(np.float32))


@pytest.mark.gpu
class TestNanUnderRelu:
    @pytest.mark.parametrize("dtype_c", ["f32", "bf16"])
    @pytest.mark.parametrize("shape", [(300, 260, 416), (300, 263, 160), (20, 264, 288), (60, 261, 416), (100, 320, 4128)])
    @pytest.mark.parametrize("plan", [{}, {"cta_group": 1, "tile_n": 128}, {"tile_n": 64}, {"max_ctas": 2, "tail_split": True}])
    def test_every_ending_of_the_product_keeps_it(self, gpu, dtype_c, shape, plan):
        """Whole tiles, ragged columns, short A stages, K cut between CTAs: NaN stays, negative sums become 0."""
        M, N, K = shape
        rng = np.random.default_rng(M + N + K)
        (qa, sa, a), (qb, sb, b) = exact_operand(M, K, rng), exact_operand(N, K, rng)
        row, column = M - 2, N - 3
        sa[row, 0] = sb[column, 1] = 255
        bias = rng.integers(-8, 8, N).astype(np.float32)
        got = gemm(qa, qb, dtype_ab="mxe2m1", dtype_c=dtype_c, block_scales_a=sa, block_scales_b=sb, bias=bias, relu=True, **plan)
        got = got if dtype_c == "f32" else dtypes.bf16_bits_to_f32(got)
        bad = np.zeros((M, N), bool)
        bad[row], bad[:, column] = True, True
        assert np.isnan(got[bad]).all()
        want = np.maximum(a @ b.T + bias, 0).astype(np.float32)
        want = want if dtype_c == "f32" else dtypes.bf16_round(want)
        assert (want[~bad] == 0).any() and np.array_equal(got[~bad], want[~bad])

    def test_from_values_to_the_layer_behind(self, gpu):
        x = torch.randn(64, 256, device="cuda")
        x[3, 40], x[9, 200] = float("nan"), float("inf")
        w = top.quantize_mx_direct(torch.randn(128, 256, device="cuda"))
        c = top.gemm_mx_nt_direct(*top.quantize_mx_direct(x), *w, relu=True)
        bad = torch.zeros(64, dtype=torch.bool, device="cuda")
        bad[[3, 9]] = True
        assert torch.equal(torch.isnan(c).all(1), bad) and torch.equal(torch.isnan(c).any(1), bad) and bool((c[~bad] >= 0).all())


@pytest.mark.gpu
class TestCaptureBesideAGraph:
    @pytest.mark.parametrize("distill", [False, True])
    @pytest.mark.parametrize("eager", ["function", "operator"])
    @pytest.mark.parametrize("captured", ["function", "operator"])
    def test_every_form_is_seen_and_refused(self, gpu, distill, eager, captured):
        x, w, t = strided_problem("cuda")
        x, w = x.contiguous().requires_grad_(), w.contiguous().requires_grad_()
        ids, logits = t[:, None], torch.zeros(70, 1, device="cuda")
        ops = torch.ops.aster_b200
        forms = {"function": (lambda: hl.linear_distillation(x, w, logits, ids)) if distill else (lambda: hl.linear_cross_entropy(x, w, t)),
                 "operator": (lambda: ops.linear_distillation(x, w, logits, ids)[0]) if distill else (lambda: ops.linear_cross_entropy(x, w, t)[0])}
        forms[captured]()  # the first call on a device comes before a capture
        alive = forms[eager]()
        with pytest.raises(RuntimeError, match="still alive"):
            with torch.cuda.graph(torch.cuda.CUDAGraph()):
                forms[captured]()
        want = torch.autograd.grad(alive, (x, w))
        del alive
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            got = torch.autograd.grad(forms[captured](), (x, w))
        graph.replay()
        assert all(torch.equal(a, b) for a, b in zip(got, want))


class TestTemperatures:
    """1 / T and T^2 leave fp32 long before T does."""

    def test_extremes_are_refused(self, native_lib):
        for tau in (1e-45, 1e-40, 1e-30, 2.0 ** -61, 2.0 ** 61, 1e25, 3e38):
            with pytest.raises(nat.B200Error, match="temperature"):
                hl._sizes(basics.TestOnHost.desc(kind=nat.HEAD_DISTILL, temperature=tau))
        for tau in (2.0 ** -60, 1e-3, 2.0 ** 60):
            hl._sizes(basics.TestOnHost.desc(kind=nat.HEAD_DISTILL, temperature=tau))

    @pytest.mark.gpu
    def test_extremes_are_refused_on_tensors(self, gpu):
        x, w, t = strided_problem("cuda")
        for tau in (1e-30, 1e-50, 1e25, 1e50):
            with pytest.raises(RuntimeError, match="temperature"):
                hl.linear_distillation(x, w, torch.zeros(70, 1, device="cuda"), t[:, None], temperature=tau)

    @pytest.mark.gpu
    @pytest.mark.parametrize("tau", [2.0 ** -20, 2.0 ** 20])
    def test_far_from_one(self, gpu, tau):
        """Finite, and the limit's value: one certain entry's distance to the largest logit, or the entropies' difference."""
        x, w, g = make(40, 64, 300, BF16, 62)
        ids = torch.randint(0, 300, (40, 1), device="cuda", generator=g)
        loss = hl.linear_distillation(x, w, torch.zeros(40, 1, device="cuda"), ids, temperature=tau, reduction="none")
        z = x.double() @ w.double().T / tau
        want = tau * tau * (torch.logsumexp(z, 1) - z.gather(1, ids)[:, 0])
        # a logit is off by 5 roundings of at most 2^-23 of |x| . |w|, twice; lse and z each by half a step of 2^-24
        dz = 5 * 2.0 ** -23 * (x.double().abs() @ w.double().abs().T).amax(1) / tau
        bound = tau * tau * (2 * dz + 2.0 ** -16 + 2.0 ** -22 * z.abs().amax(1))
        assert bool(((loss.double() - want).abs() <= bound).all())


@pytest.mark.gpu
class TestEndsOfTheRange:
    @pytest.mark.parametrize("teacher_dtype", [torch.float32, BF16, torch.float16])
    @pytest.mark.parametrize("tau", [0.5, 1.0, 3.0])
    def test_teacher_logits_as_large_as_their_type(self, gpu, teacher_dtype, tau):
        """Only minus infinity leaves an entry out: the type's lowest value is an entry without weight, or with
        the same weight as its neighbours where a row holds nothing else."""
        x, w, g = make(40, 64, 300, BF16, 61)
        ids, logits = teacher(40, 300, 6, g, teacher_dtype)
        lowest, largest = torch.finfo(teacher_dtype).min, torch.finfo(teacher_dtype).max
        ids[4:12] = torch.arange(6, device="cuda") * 7
        logits[4:7, :4], logits[7:9], logits[9:11, 2], logits[11, :] = lowest, lowest, largest, largest
        logits[4:7, 4:], logits[9:11, :2], logits[9:11, 3:] = 0.25, 1.0, lowest
        ref = distill_reference(x, w, logits, ids, tau, reduction="none")
        x.requires_grad_(), w.requires_grad_()
        loss = hl.linear_distillation(x, w, logits, ids, temperature=tau, reduction="none")
        ref.check_loss(loss)
        ref.check_grads(*torch.autograd.grad(loss.sum(), (x, w)))
        ref = distill_reference(x.detach(), w.detach(), logits, ids, tau)
        ref.check_loss(hl.linear_distillation(x, w, logits, ids, temperature=tau))


@pytest.mark.gpu
class TestWaitsThatRunOut:
    @pytest.mark.parametrize("dtype", ["bf16", "mxe2m1"])
    @pytest.mark.parametrize("cta_group", [1, 2])
    def test_an_abort_waits_for_its_own_copies(self, gpu, dtype, cta_group):
        """No stage is handed over (the plan's own switch for this test): after the wait limit the producer waits
        for each of its four slots, 20 ms at most, instead of leaving at once because the CTA is aborting."""
        import time

        plan = GemmPlan(512, 256, 8192, dtype, "f32", cta_group=cta_group, tile_n=128, stages=4, debug_mode=8, wait_limit_ms=20)
        a, b, c = (torch.zeros(512 * 8192, dtype=torch.bfloat16, device="cuda") for _ in range(3))
        scales = torch.full((1 << 20,), 127, dtype=torch.uint8, device="cuda")
        if dtype == "mxe2m1":
            plan.set_mx_scales(scales.data_ptr(), scales.data_ptr())
        torch.cuda.synchronize()
        t0 = time.perf_counter()
        plan.run(a.data_ptr(), b.data_ptr(), c.data_ptr())
        with pytest.raises(nat.B200Error, match="code 0x"):
            plan.status()
        elapsed = time.perf_counter() - t0
        assert 0.02 + 4 * 0.02 <= elapsed < 1.0
        assert plan.status() == [0, 0, 0, 0]

    @pytest.mark.parametrize("T", [100, 256])  # one CTA, a pair
    def test_a_loss_whose_product_gave_up_is_nan(self, gpu, T):
        """A product of two tiles with 65536 K blocks each (several milliseconds) under a limit of 1 ms: the status
        names the wait, losses and gradients are NaN until it is read, and the next call is right again."""
        x, w, g = make(T, 64, 128, BF16, 71)
        t = torch.randint(0, 128, (T,), device="cuda", generator=g)
        x.requires_grad_(), w.requires_grad_()
        before = hl.linear_cross_entropy(x, w, t)
        want = torch.autograd.grad(before, (x, w))
        before = hl.linear_cross_entropy(x, w, t)  # a graph from before the lost wait
        rows = hl.linear_cross_entropy(x, w, t, reduction="none")
        long_x, long_w = (torch.zeros(n, 1 << 22, dtype=BF16, device="cuda") for n in (T, 128))
        for reduction in ("mean", "none"):
            assert hl.head_loss_status() == [0, 0, 0, 0]
            slow = hl._xent_head(long_x, long_w, t, -100, 0.0, reduction)
            slow.desc.wait_limit_ms = 1
            loss, _, _ = slow.forward()
            assert bool(torch.isnan(loss).all())
            assert bool(torch.isnan(hl.linear_cross_entropy(x, w, t)))
            for kept in (before, rows.sum()):
                assert all(bool(torch.isnan(v).all()) for v in torch.autograd.grad(kept, (x, w), retain_graph=True))
            with pytest.raises(nat.B200Error, match="code 0x"):
                hl.head_loss_status()
        del long_x, long_w, slow
        after = hl.linear_cross_entropy(x, w, t)
        got = torch.autograd.grad(after, (x, w))
        assert torch.equal(after, before) and all(torch.equal(a, b) for a, b in zip(got, want))
        assert hl.head_loss_status() == [0, 0, 0, 0]


class TestOperatorsMakeWhatIsWanted:
    """A frozen head or a frozen body costs the dispatcher's backward pass no gradient that nobody asked for."""

    @staticmethod
    def operators(x, w, t, logits):
        ops = torch.ops.aster_b200
        return lambda: ops.linear_cross_entropy(x, w, t)[0], lambda: ops.linear_distillation(x, w, logits, t[:, None])[0]

    @pytest.mark.parametrize("which", [0, 1])
    @pytest.mark.parametrize("want", ["x", "w", "both"])
    def test_on_the_host(self, which, want):
        from torch.utils._python_dispatch import TorchDispatchMode

        class Record(TorchDispatchMode):
            made = []

            def __torch_dispatch__(self, func, types, args=(), kwargs=None):
                out = func(*args, **(kwargs or {}))
                if "_backward" in str(func):
                    self.made += [tuple(o.shape) for o in out]
                return out

        x, w, t = (v.to("meta") for v in strided_problem("cpu"))
        x.requires_grad_(want != "w"), w.requires_grad_(want != "x")
        loss = self.operators(x, w, t, torch.zeros(70, 1, device="meta"))[which]()
        with Record() as record:
            loss.backward()
        assert record.made == [(0,) if want == "w" else (70, 136), (0,) if want == "x" else (300, 136)]
        assert (x.grad is None) == (want == "w") and (w.grad is None) == (want == "x")

    @pytest.mark.gpu
    @pytest.mark.parametrize("which", [0, 1])
    def test_on_the_gpu(self, gpu, which):
        x, w, t = strided_problem("cuda")
        call = self.operators(x, w, t, torch.zeros(70, 1, device="cuda"))[which]
        x.requires_grad_(), w.requires_grad_()
        want = torch.autograd.grad(call(), (x, w))
        for i, (leaf, other) in enumerate(((x, w), (w, x))):
            other.requires_grad_(False)
            got, = torch.autograd.grad(call(), leaf)
            other.requires_grad_()
            assert torch.equal(got, want[i])


class TestProductHasNoBackward:
    """A bias that wants a gradient is not left without one silently."""

    def test_a_result_that_refuses_on_the_host(self):
        out, bias = torch.zeros(3, 8), torch.zeros(8, requires_grad=True)
        c = top._without_gradient(out, bias)
        assert c.requires_grad and torch.equal(c.detach(), out)
        with pytest.raises(RuntimeError, match="no backward pass"):
            c.sum().backward()
        top._without_gradient(out, bias).add_(1.0)  # in place, like any fresh result
        assert bool((out == 1).all())

    @pytest.mark.gpu
    @pytest.mark.parametrize("form", ["direct", "operator"])
    def test_on_the_gpu(self, gpu, form):
        q = top.quantize_mx_direct(torch.randn(40, 64, device="cuda"))
        w = top.quantize_mx_direct(torch.randn(72, 64, device="cuda"))
        bias = torch.randn(72, device="cuda")
        call = top.gemm_mx_nt_direct if form == "direct" else torch.ops.aster_b200.gemm_mx_nt
        want = call(*q, *w, bias)
        assert not want.requires_grad
        bias.requires_grad_()
        got = call(*q, *w, bias)
        with pytest.raises(RuntimeError, match="backward"):
            got.sum().backward()
        with torch.no_grad():
            assert torch.equal(call(*q, *w, bias), want) and torch.equal(got, want)

        from torch.autograd import forward_ad

        bias.requires_grad_(False)
        with forward_ad.dual_level(), pytest.raises(RuntimeError, match="forward-mode"):
            call(*q, *w, forward_ad.make_dual(bias, bias))


@pytest.mark.gpu
class TestOperatorsAsTorchKnowsThem:
    def test_every_byte_of_the_outputs_is_defined(self, gpu):
        """`saved` is an output, too: two calls give the same bytes, whatever was in the memory before."""
        x, w, t = strided_problem("cuda")
        ids, logits = torch.stack([t, (t + 7) % 300, torch.full_like(t, -1)], 1), torch.zeros(70, 3, device="cuda")
        for call in (lambda: torch.ops.aster_b200.linear_cross_entropy(x, w, t), lambda: torch.ops.aster_b200.linear_distillation(x, w, logits, ids)):
            outs = []
            for fill in (0, 255, 7):
                torch.cuda.synchronize()
                torch.cuda.empty_cache()
                torch.full((64 << 20,), fill, dtype=torch.uint8, device="cuda")  # what the allocator hands out next
                outs.append(call())
            assert all(torch.equal(a, b) for out in outs[1:] for a, b in zip(outs[0], out))

    def test_opcheck(self, gpu):
        from torch.library import opcheck

        x, w, t = strided_problem("cuda")
        ids, logits = t[:, None].contiguous(), torch.zeros(70, 1, device="cuda")
        ops = torch.ops.aster_b200
        for frozen in (None, x, w):
            x.requires_grad_(frozen is not x), w.requires_grad_(frozen is not w)
            opcheck(ops.linear_cross_entropy.default, (x, w, t, -100, 0.1, "none" if frozen is None else "mean"))
            opcheck(ops.linear_distillation.default, (x, w, logits, ids, 2.0))

    @pytest.mark.parametrize("backend", ["eager", "aot_eager"])
    def test_functions_inside_a_compiled_program(self, gpu, backend):
        x, w, t = strided_problem("cuda")
        x.requires_grad_(), w.requires_grad_()
        ids, logits = t[:, None].contiguous(), torch.zeros(70, 1, device="cuda")
        for call in (lambda x, w: hl.linear_cross_entropy(x, w, t, label_smoothing=0.1, grad_bytes=1), lambda x, w: hl.linear_distillation(x, w, logits, ids, reduction="none").sum()):
            want = call(x, w)
            loss = torch.compile(call, backend=backend, fullgraph=True)(x, w)
            assert torch.equal(loss, want)
            for a, b in zip(torch.autograd.grad(loss, (x, w)), torch.autograd.grad(want, (x, w))):
                assert torch.equal(a, b)

        def layer(h, v):
            q, s = top.quantize_mx_direct(h)
            u, r = top.quantize_mx_direct(v)
            return top.gemm_mx_nt_direct(q, s, u, r, None, True, torch.bfloat16), top.dequantize_mx_direct(q, s, torch.bfloat16)

        h, v = torch.randn(48, 128, device="cuda").bfloat16(), torch.randn(72, 128, device="cuda").bfloat16()
        for a, b in zip(torch.compile(layer, backend=backend, fullgraph=True)(h, v), layer(h, v)):
            assert torch.equal(a, b)


class TestOperatorsTakeWhatTheFunctionsTake:
    def test_limit_of_the_stored_range_on_the_host(self):
        x, w, t = (v.to("meta") for v in strided_problem("cpu"))
        x.requires_grad_()
        ops = torch.ops.aster_b200
        ops.linear_cross_entropy(x, w, t, -100, 0.0, "mean", 1 << 20)[0].backward()
        ops.linear_distillation(x, w, torch.zeros(70, 1, device="meta"), t[:, None], 1.0, "mean", 1 << 20)[0].backward()

    @pytest.mark.gpu
    def test_limit_of_the_stored_range(self, gpu):
        x, w, t = strided_problem("cuda")
        x.requires_grad_(), w.requires_grad_()
        want = torch.autograd.grad(hl.linear_cross_entropy(x, w, t, grad_bytes=1), (x, w))
        got = torch.autograd.grad(torch.ops.aster_b200.linear_cross_entropy(x, w, t, grad_bytes=1)[0], (x, w))
        assert all(torch.equal(a, b) for a, b in zip(got, want))


@pytest.mark.gpu
class TestTwoAtOnce:
    """Two captured graphs of the same shapes, replayed on two streams at the same time, and eager calls beside them."""

    @staticmethod
    def replay(graphs, outs, wants, beside):
        streams = [torch.cuda.Stream() for _ in graphs]
        for _ in range(20):
            torch.cuda.synchronize()
            for stream, graph in zip(streams, graphs):
                with torch.cuda.stream(stream):
                    for _ in range(5):
                        graph.replay()
            eager = beside()
            torch.cuda.synchronize()
            for out, want in zip(outs + [eager], wants + [wants[0]]):
                assert all(torch.equal(a, b) for a, b in zip(out, want))

    @pytest.mark.parametrize("shape", [(16, 1024, 8192), (300, 520, 1056)])  # K cut between CTAs, pair tiles
    def test_products_of_one_plan(self, gpu, shape):
        M, N, K = shape
        operands = [top.quantize_mx_direct(torch.randn(M, K, device="cuda")) + top.quantize_mx_direct(torch.randn(N, K, device="cuda")) for _ in range(2)]
        wants = [[top.gemm_mx_nt_direct(*o)] for o in operands]
        graphs, outs = [torch.cuda.CUDAGraph() for _ in operands], []
        for graph, o in zip(graphs, operands):
            with torch.cuda.graph(graph):
                outs.append([top.gemm_mx_nt_direct(*o)])
        self.replay(graphs, outs, wants, lambda: [top.gemm_mx_nt_direct(*operands[0])])

    @pytest.mark.parametrize("distill", [False, True])
    def test_training_steps(self, gpu, distill):
        def step(x, w, t):
            loss = hl.linear_distillation(x, w, torch.zeros(70, 1, device="cuda"), t[:, None]) if distill else hl.linear_cross_entropy(x, w, t, label_smoothing=0.1)
            return [loss.detach(), *torch.autograd.grad(loss, (x, w))]

        problems = []
        for seed in (3, 4):
            x, w, t = strided_problem("cuda", V=3001, seed=seed)
            problems.append((x.requires_grad_(), w.requires_grad_(), t))
        wants = [step(*p) for p in problems]
        graphs, outs = [torch.cuda.CUDAGraph() for _ in problems], []
        for graph, p in zip(graphs, problems):
            with torch.cuda.graph(graph):
                outs.append(step(*p))
        self.replay(graphs, outs, wants, lambda: step(*problems[0]))
        assert hl.head_loss_status() == [0, 0, 0, 0]
