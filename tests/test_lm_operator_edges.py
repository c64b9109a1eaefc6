"""Calls of the language-model operators from their edges."""

import pytest
import torch

from aster_b200 import head_loss as hl

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
