"""Block-scaled fp4 (E2M1 elements, one E8M0 scale per 32): quantisation, its inverse and the product.

Codes, scales and dequantised values are exact by definition and compared bit for bit.  The products
are compared for equality, too: the operands are drawn so that every partial sum is a multiple of one
unit u and stays below 2^24 u, which fp32 holds exactly in any order of summation."""

import numpy as np
import pytest
import torch

import aster_b200.torch_op as top
from aster_b200 import _native as nat
from aster_b200 import dtypes
from aster_b200.gemm import GemmPlan, HostGemmPipeline, gemm

GRID = [0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0]


def nearest_even_codes(x):
    """Brute force: the grid value with the smallest distance in 64 bits, ties to the even code."""
    x = np.asarray(x, np.float64)
    d = np.abs(np.abs(x)[..., None] - np.array(GRID))
    best = d.min(axis=-1, keepdims=True)
    even = np.where(d == best, np.arange(8) % 2 * 8 + np.arange(8), 99)
    code = even.min(axis=-1) % 8
    return (code + 8 * np.signbit(x)).astype(np.uint8)


def unpack_scales(packed, rows, K):
    """[rows][K/32] bytes out of the streaming order."""
    groups = (K + 127) // 128
    blocks = packed.reshape((rows + 127) // 128, groups, 32, 4, 4)  # [row block][K group][r % 32][r / 32][K block]
    return blocks.transpose(0, 3, 2, 1, 4).reshape(-1, groups * 4)[:rows, :K // 32]


def values(rows, K, seed, dtype=np.float32):
    rng = np.random.default_rng(seed)
    x = rng.standard_normal((rows, K)) * np.exp(2 * rng.standard_normal((rows, K // 32))).repeat(32, axis=1)
    return x.astype(dtype)


class TestOnHost:
    def test_codes_match_brute_force(self):
        x = np.concatenate([np.linspace(-7, 7, 2801), np.array([0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0, -0.0, -0.25, 1e-30, 1e30])]).astype(np.float32)
        assert np.array_equal(dtypes.f32_to_e2m1_codes(x), nearest_even_codes(np.clip(x, -6, 6)))
        codes = np.arange(16, dtype=np.uint8)
        assert np.array_equal(dtypes.f32_to_e2m1_codes(dtypes.e2m1_codes_to_f32(codes)), codes)

    def test_packing(self):
        codes = np.random.default_rng(0).integers(0, 16, (5, 64)).astype(np.uint8)
        packed = dtypes.pack_e2m1(codes)
        assert packed.shape == (5, 32) and packed[0, 0] == codes[0, 0] | codes[0, 1] << 4
        assert np.array_equal(dtypes.unpack_e2m1(packed), codes)

    @pytest.mark.parametrize("scale", [2.0 ** -140, 2.0 ** -126, 2.0 ** -60, 1.0, 2.0 ** 100, 2.0 ** 126])
    def test_quantize_matches_the_rule(self, scale):
        x = (np.clip(values(7, 96, 3), -3, 3) * scale).astype(np.float32)
        bits, scales = dtypes.quantize_mx(x, "e2m1")
        amax = np.abs(x.astype(np.float64)).reshape(7, 3, 32).max(-1)
        e = np.clip(np.floor(np.log2(amax)) - 2, -127, 127)
        assert np.array_equal(scales, (e + 127).astype(np.uint8))
        want = nearest_even_codes(np.clip(x.astype(np.float64).reshape(7, 3, 32) / 2.0 ** e[..., None], -6, 6))
        assert np.array_equal(dtypes.unpack_e2m1(bits), want.reshape(7, 96))

    def test_zero_nan_and_infinite_blocks(self):
        x = np.ones((1, 128), np.float32)
        x[0, :32] = 0
        x[0, 40] = np.nan
        x[0, 70] = -np.inf
        bits, scales = dtypes.quantize_mx(x, "e2m1")
        assert scales.tolist() == [[127, 255, 255, 125]]
        y = dtypes.dequantize_mx(bits, scales, "e2m1")
        assert (y[0, :32] == 0).all() and np.isnan(y[0, 32:96]).all() and (y[0, 96:] == 1).all()

    def test_fake_shapes(self):
        x = torch.empty(130, 160, dtype=torch.bfloat16, device="meta")
        q, s = torch.ops.aster_b200.quantize_mx(x)
        assert q.shape == (130, 80) and s.shape == (2 * 2 * 512,) and q.dtype == s.dtype == torch.uint8
        assert torch.ops.aster_b200.dequantize_mx(q, s, torch.float16).shape == (130, 160)
        assert torch.ops.aster_b200.gemm_mx_nt(q, s, q, s, None, False, torch.bfloat16).shape == (130, 130)

    def test_cpu_tensors_are_refused(self):
        q, s = torch.zeros(8, 16, dtype=torch.uint8), torch.zeros(512, dtype=torch.uint8)
        for call in (lambda: top.quantize_mx_direct(torch.zeros(8, 32)), lambda: top.dequantize_mx_direct(q, s), lambda: top.gemm_mx_nt_direct(q, s, q, s)):
            with pytest.raises(RuntimeError, match="no CPU path"):
                call()

    def test_abi_refusals(self, native_lib):
        """Refused before anything touches a device: the addresses are never read."""
        good = dict(x=4096, dtype_x=nat.BF16, rows=4, K=64, stride=64, dtype_q=nat.MXE2M1, q=8192, s=12288, stream=None)
        for change, text in ((dict(x=None), "NULL"), (dict(K=48), "multiple of 32"), (dict(K=0), "multiple of 32"), (dict(rows=0), "rows must be"),
                             (dict(stride=32), "row_stride"), (dict(dtype_q=nat.MXE4M3), "dtype_q"), (dict(dtype_x=nat.I8), "dtype_x"),
                             (dict(q=8200), "16-byte aligned"), (dict(x=4097), "aligned to its elements")):
            with pytest.raises(nat.B200Error, match=text):
                nat.call("b200_quantize_mx", *{**good, **change}.values())
        good = dict(q=8192, s=12288, dtype_q=nat.MXE2M1, rows=4, K=64, dtype_out=nat.F32, out=4096, stream=None)
        for change, text in ((dict(out=None), "NULL"), (dict(K=33), "multiple of 32"), (dict(out=4104), "16-byte aligned"), (dict(dtype_out=nat.E4M3), "dtype_out")):
            with pytest.raises(nat.B200Error, match=text):
                nat.call("b200_dequantize_mx", *{**good, **change}.values())

    def test_plan_refusals(self, native_lib):
        with pytest.raises(nat.B200Error, match="K % 32 == 0"):
            GemmPlan(128, 128, 144, "mxe2m1", "f32")
        with pytest.raises(nat.B200Error, match="split_k"):
            GemmPlan(128, 128, 2048, "mxe2m1", "f32", split_k=2)
        with pytest.raises(nat.B200Error, match="row-major B"):
            GemmPlan(128, 128, 2048, "mxe2m1", "f32", b_layout="packed")
        for bad in (dict(tile_n=64, cta_group=2), dict(tile_n=192, cta_group=1), dict(tile_n=32)):
            with pytest.raises(nat.B200Error, match="tile_n"):
                GemmPlan(512, 512, 2048, "mxe2m1", "f32", **bad)
        with pytest.raises(nat.B200Error, match="tile_k"):
            GemmPlan(128, 128, 2048, "mxe2m1", "f32", tile_k=128)
        assert GemmPlan(512, 512, 2048, "mxe2m1", "bf16").resources().tile_k == 256


@pytest.mark.gpu
class TestQuantizeOnGpu:
    @pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
    @pytest.mark.parametrize("shape", [(1, 32), (3, 64), (16, 8192), (129, 160), (257, 1056), (1000, 4128)])
    def test_matches_the_host(self, gpu, dtype, shape):
        rows, K = shape
        x = torch.from_numpy(values(rows, K, rows + K)).to(dtype)
        bits, scales = dtypes.quantize_mx(x.float().numpy(), "e2m1")
        q, s = top.quantize_mx_direct(x.cuda())
        assert np.array_equal(q.cpu().numpy(), bits)
        packed = s.cpu().numpy()
        assert np.array_equal(unpack_scales(packed, rows, K), scales)
        pad = np.ones((packed.size // 512 * 128, 4), bool)  # every padding byte is 127
        whole = unpack_scales(packed, (rows + 127) // 128 * 128, (K + 127) // 128 * 128)
        assert (whole[rows:] == 127).all() and (whole[:, K // 32:] == 127).all() and pad.size == whole.size
        for out_dtype in (torch.float32, torch.bfloat16, torch.float16):
            y = top.dequantize_mx_direct(q, s, out_dtype)
            want = torch.from_numpy(dtypes.dequantize_mx(bits, scales, "e2m1")).to(out_dtype)
            assert torch.equal(y.cpu(), want)

    def test_extremes(self, gpu):
        rng = np.random.default_rng(5)
        x = rng.standard_normal((12, 256)).astype(np.float32)
        for i, scale in enumerate([2.0 ** -148, 2.0 ** -127, 2.0 ** -126, 2.0 ** -125, 2.0 ** -100, 1e-20, 1e20, 2.0 ** 100, 2.0 ** 125]):
            x[i] = np.clip(x[i], -3, 3) * np.float32(scale)
        x[9, :32] = 0
        x[9, 40] = np.nan
        x[9, 100] = np.inf
        x[9, 101:128] = np.nan
        x[10] = np.tile(np.array([0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0, 6.0, -0.0, -0.25, -5.0, 7.9, -7.9, 4.0, 0.5, 1e-38], np.float32), 16)
        x[11, ::2] = -0.0
        bits, scales = dtypes.quantize_mx(x, "e2m1")
        q, s = top.quantize_mx_direct(torch.from_numpy(x).cuda())
        assert np.array_equal(q.cpu().numpy(), bits) and np.array_equal(unpack_scales(s.cpu().numpy(), 12, 256), scales)
        y = top.dequantize_mx_direct(q, s).cpu().numpy()
        assert np.array_equal(y, dtypes.dequantize_mx(bits, scales, "e2m1"), equal_nan=True)

    @pytest.mark.parametrize("offset,stride", [(0, 128), (8, 104), (1, 97), (3, 200)])
    def test_strided_and_unaligned_rows(self, gpu, offset, stride):
        base = torch.randn(40 * stride + 64, device="cuda").bfloat16()
        x = base.as_strided((33, 96), (stride, 1), offset)
        q, s = top.quantize_mx_direct(x)
        want = top.quantize_mx_direct(x.contiguous())
        assert torch.equal(q, want[0]) and torch.equal(s, want[1])
        columns = torch.randn(64, 40, device="cuda")  # K not the fastest dimension
        for view in (columns.T, torch.randn(1, 64, device="cuda").expand(5, 64)):
            q, s = top.quantize_mx_direct(view)
            want = top.quantize_mx_direct(view.contiguous().clone())
            assert torch.equal(q, want[0]) and torch.equal(s, want[1])

    def test_offsets_beyond_32_bits(self, gpu):
        rows, K = 265000, 8192  # 2.17e9 values
        x = torch.randn(rows, K, device="cuda", dtype=torch.bfloat16)
        q, s = top.quantize_mx_direct(x)
        tail = 128 * 3
        first = rows // 128 * 128 - tail
        q2, s2 = top.quantize_mx_direct(x[first:])
        assert torch.equal(q[first:], q2) and torch.equal(s[-s2.numel():], s2)
        y = top.dequantize_mx_direct(q, s, torch.bfloat16)
        assert torch.equal(y[first:], top.dequantize_mx_direct(q2, s2, torch.bfloat16))

    def test_refusals(self, gpu):
        x = torch.zeros(4, 64, device="cuda")
        for bad in (x[:, :48], x[:0], x.double(), x[0], x[:, :0]):
            with pytest.raises(RuntimeError):
                top.quantize_mx_direct(bad)
        with pytest.raises(RuntimeError, match="e2m1"):
            top.quantize_mx_direct(x, "e4m3")
        q, s = top.quantize_mx_direct(x)
        for args in ((q, s[:-1]), (q[:, :8], s), (q.int(), s), (q, s.cpu()), (q, s, torch.float64), (q[:0], s)):
            with pytest.raises(RuntimeError):
                top.dequantize_mx_direct(*args)


def exact_operand(rows, K, rng, lo=126, hi=128):
    """Random codes with scales of 1/2, 1 and 2: products are multiples of 1/16 of at most 144."""
    codes = rng.integers(0, 16, (rows, K)).astype(np.uint8)
    scales = rng.integers(lo, hi + 1, (rows, K // 32)).astype(np.uint8)
    return dtypes.pack_e2m1(codes), scales, dtypes.dequantize_mx(dtypes.pack_e2m1(codes), scales, "e2m1").astype(np.float64)


def product(a, b):
    want = a @ b.T
    # every partial sum of any order is a multiple of 1/16 below 2^24 / 16, so that fp32 holds it
    assert (np.abs(a) @ np.abs(b).T).max() * 16 < 2 ** 24
    return want


SHAPES = [(1, 32, 32), (16, 256, 96), (128, 128, 256), (130, 200, 288), (33, 520, 4128), (300, 264, 1056), (512, 512, 4096), (1000, 1100, 544)]


@pytest.mark.gpu
class TestProductOnGpu:
    def test_known_answers(self, gpu):
        M = N = 16
        a = dtypes.pack_e2m1(dtypes.f32_to_e2m1_codes(np.full((M, 256), 1.5, np.float32)))
        b = dtypes.pack_e2m1(dtypes.f32_to_e2m1_codes(np.full((N, 256), -3.0, np.float32)))
        sa, sb = np.full((M, 8), 129, np.uint8), np.full((N, 8), 128, np.uint8)
        got = gemm(a, b, dtype_ab="mxe2m1", dtype_c="f32", block_scales_a=sa, block_scales_b=sb)
        assert np.array_equal(got, np.full((M, N), -1.5 * 3 * 256 * 8, np.float32))
        # each block of 32 with its own scale: sum over blocks of 32 * 1 * 2^e
        ones = dtypes.pack_e2m1(dtypes.f32_to_e2m1_codes(np.ones((N, 256), np.float32)))
        sa = np.repeat(np.uint8([[120, 121, 122, 123, 124, 125, 126, 127]]), M, axis=0)
        got = gemm(ones, ones, dtype_ab="mxe2m1", dtype_c="f32", block_scales_a=sa, block_scales_b=np.full((N, 8), 127, np.uint8))
        assert np.array_equal(got, np.full((M, N), 32 * (2.0 - 2.0 ** -7), np.float32))

    def test_each_row_and_block_uses_its_own_scale(self, gpu):
        M, N, K = 384, 512, 512
        rng = np.random.default_rng(1)
        sa = rng.integers(124, 131, (M, K // 32)).astype(np.uint8)
        sb = rng.integers(124, 131, (N, K // 32)).astype(np.uint8)
        ones = dtypes.pack_e2m1(dtypes.f32_to_e2m1_codes(np.ones((max(M, N), K), np.float32)))
        want = 32.0 * (np.exp2(sa.astype(np.float64) - 127) @ np.exp2(sb.astype(np.float64) - 127).T)
        for kw in ({}, {"tile_n": 128}, {"cta_group": 1}, {"cta_group": 1, "tile_n": 256}, {"tile_n": 192}, {"tile_n": 192, "max_ctas": 2}):
            got = gemm(ones[:M], ones[:N], dtype_ab="mxe2m1", dtype_c="f32", block_scales_a=sa, block_scales_b=sb, **kw)
            assert np.array_equal(got, want.astype(np.float32)), kw

    @pytest.mark.parametrize("plan", [{}, {"cta_group": 1, "tile_n": 128}, {"cta_group": 1, "tile_n": 256}, {"cta_group": 2, "tile_n": 128},
                                      {"cta_group": 2, "tile_n": 256}, {"tile_n": 192}, {"tile_n": 64}, {"tile_n": 64, "tile_m": 128}, {"stages": 2}, {"max_ctas": 4}])
    @pytest.mark.parametrize("shape", SHAPES)
    def test_exact_sums(self, gpu, shape, plan):
        M, N, K = shape
        rng = np.random.default_rng(M + N + K)
        (qa, sa, a), (qb, sb, b) = exact_operand(M, K, rng), exact_operand(N, K, rng)
        want = product(a, b)
        kw = dict(dtype_ab="mxe2m1", block_scales_a=sa, block_scales_b=sb, **plan)
        assert np.array_equal(gemm(qa, qb, dtype_c="f32", **kw), want.astype(np.float32))
        got = dtypes.bf16_bits_to_f32(gemm(qa, qb, dtype_c="bf16", **kw))
        assert np.array_equal(got, dtypes.bf16_round(want.astype(np.float32)))

    @pytest.mark.parametrize("extra", [{}, {"max_ctas": 4, "tail_split": True}, {"cta_group": 1, "tile_n": 128, "max_ctas": 3, "tail_split": True},
                                       {"cta_group": 2, "tile_n": 256, "max_ctas": 2, "tail_split": True}, {"tile_n": 192, "max_ctas": 6, "tail_split": True}, {"tile_n": 192, "max_ctas": 2}, {"static_b": True},
                                       {"static_b": True, "cta_group": 1, "stages": 2}, {"split_k": -1}, {"tile_n": 64, "max_ctas": 3}])
    def test_epilogue_and_schedules(self, gpu, extra):
        M, N, K = 384, 256, 6144 + 32
        rng = np.random.default_rng(9)
        (qa, sa, a), (qb, sb, b) = exact_operand(M, K, rng, 127, 127), exact_operand(N, K, rng, 127, 127)
        bias = rng.integers(-8, 8, N).astype(np.float32)
        want = np.maximum(product(a, b) + bias, 0).astype(np.float32)
        got = gemm(qa, qb, dtype_ab="mxe2m1", dtype_c="f32", block_scales_a=sa, block_scales_b=sb, bias=bias, relu=True, **extra)
        assert np.array_equal(got, want)

    @pytest.mark.parametrize("M", [1, 17, 40, 100])
    @pytest.mark.parametrize("N", [64, 200, 4096, 9500])
    def test_few_rows(self, gpu, M, N):
        """The forms that stream B: 64- and 128-column tiles, short A stages, and K cut between the CTAs of a cluster."""
        for K, extra in ((2080, {}), (16384, {}), (16384, {"tile_n": 128}), (16384, {"tile_n": 64})):
            rng = np.random.default_rng(M + N + K)
            (qa, sa, a), (qb, sb, b) = exact_operand(M, K, rng, 127, 127), exact_operand(N, K, rng, 127, 127)
            want = a @ b.T  # multiples of 1/4 below 36 * 16384 < 2^24 / 4
            got = gemm(qa, qb, dtype_ab="mxe2m1", dtype_c="f32", block_scales_a=sa, block_scales_b=sb, **extra)
            assert np.array_equal(got, want.astype(np.float32)), (K, extra)

    def test_nan_scales_stay_in_their_rows(self, gpu):
        """A NaN block in one row of A or B reaches that row or column of C only, wherever the data ends
        inside a stage (the scales behind a row group's last block belong to the next row group)."""
        for K in (96, 160, 256, 288, 416):
            rng = np.random.default_rng(K)
            (qa, sa, a), (qb, sb, b) = exact_operand(300, K, rng), exact_operand(260, K, rng)
            sa[200, 0] = sb[133, 1] = 255
            got = gemm(qa, qb, dtype_ab="mxe2m1", dtype_c="f32", block_scales_a=sa, block_scales_b=sb)
            bad = np.zeros((300, 260), bool)
            bad[200], bad[:, 133] = True, True
            assert np.isnan(got[bad]).all()
            assert np.array_equal(got[~bad], product(a, b).astype(np.float32)[~bad])

    def test_torch_operator_chain(self, gpu):
        """Quantise both operands, multiply with the epilogue, on a side stream, against the
        dequantised values; the fp32 bound is K roundings of partial sums of at most |a|.|b|."""
        M, N, K = 77, 344, 1056
        g = torch.Generator(device="cuda").manual_seed(3)
        x, w = torch.randn(M, K, device="cuda", generator=g).bfloat16(), torch.randn(N, K, device="cuda", generator=g).bfloat16()
        bias = torch.randn(N, device="cuda", generator=g)
        stream = torch.cuda.Stream()
        stream.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(stream):
            (q, s), (wq, ws) = torch.ops.aster_b200.quantize_mx(x), torch.ops.aster_b200.quantize_mx(w)
            c = torch.ops.aster_b200.gemm_mx_nt(q, s, wq, ws, bias, True, torch.bfloat16)
            a, b = (torch.ops.aster_b200.dequantize_mx(*t).double() for t in ((q, s), (wq, ws)))
        stream.synchronize()
        want = torch.relu(a @ b.T + bias.double())
        bound = K * 2.0 ** -23 * (a.abs() @ b.abs().T + bias.abs().double()) + 2.0 ** -8 * want
        assert bool(((c.double() - want).abs() <= bound).all())
        again = top.gemm_mx_nt_direct(q, s, wq, ws, bias, True, torch.bfloat16)
        assert torch.equal(c, again)

    def test_views_and_refusals(self, gpu):
        x = torch.randn(64, 256, device="cuda")
        q, s = top.quantize_mx_direct(x)
        want = top.gemm_mx_nt_direct(q, s, q, s)
        wide = torch.zeros(64, 300, dtype=torch.uint8, device="cuda")
        wide[:, 5:133] = q  # rows neither contiguous nor aligned
        shifted = torch.zeros(s.numel() + 3, dtype=torch.uint8, device="cuda")
        shifted[3:] = s
        assert torch.equal(top.gemm_mx_nt_direct(wide[:, 5:133], shifted[3:], q, s), want)
        q2, s2 = top.quantize_mx_direct(x[:, :128].contiguous())
        for args in ((q, s, q2, s2), (q, s2, q, s), (q, s, q, s, torch.zeros(63, device="cuda")), (q, s, q, s, torch.zeros(64, device="cuda").half()),
                     (q, s, q, s, None, False, torch.float16)):
            with pytest.raises(RuntimeError):
                top.gemm_mx_nt_direct(*args)

    def test_first_call_inside_a_capture_is_refused(self, gpu):
        q, s = top.quantize_mx_direct(torch.randn(23, 96, device="cuda"))
        with pytest.raises(RuntimeError, match="before the stream capture"):
            with torch.cuda.graph(torch.cuda.CUDAGraph()):
                top.gemm_mx_nt_direct(q, s, q, s)
        want = top.gemm_mx_nt_direct(q, s, q, s)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            c = top.gemm_mx_nt_direct(q, s, q, s)
        graph.replay()
        assert torch.equal(c, want)

    def test_first_use_of_the_library_inside_a_capture_is_refused(self, gpu):
        """In a process of its own: refused, and everything works afterwards."""
        import subprocess
        import sys

        code = """
import torch
import aster_b200.torch_op as top, aster_b200.head_loss as hl
x = torch.randn(16, 64, device="cuda").bfloat16()
t = torch.zeros(16, dtype=torch.long, device="cuda")
for call in (lambda: top.quantize_mx_direct(x), lambda: hl.linear_cross_entropy(x, x, t)):
    try:
        with torch.cuda.graph(torch.cuda.CUDAGraph()):
            call()
        raise SystemExit("not refused")
    except RuntimeError as e:
        assert "before the stream capture" in str(e), e
hl.linear_cross_entropy(x, x, t)
graph = torch.cuda.CUDAGraph()
with torch.cuda.graph(graph):
    loss, (q, s) = hl.linear_cross_entropy(x, x, t), top.quantize_mx_direct(x)
graph.replay()
assert torch.equal(loss, hl.linear_cross_entropy(x, x, t)) and torch.equal(q, top.quantize_mx_direct(x)[0])
print("ok")
"""
        import os

        root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
        out = subprocess.run([sys.executable, "-c", code], capture_output=True, text=True, cwd=root, timeout=300)
        assert out.returncode == 0 and out.stdout.strip().endswith("ok"), out.stderr[-2000:]

    def test_from_other_threads(self, gpu):
        """A thread whose first CUDA call is the product, and several that share one plan."""
        import threading

        pairs = [top.quantize_mx_direct(torch.randn(40, 256, device="cuda")) + top.quantize_mx_direct(torch.randn(72, 256, device="cuda")) for _ in range(4)]
        want = [top.gemm_mx_nt_direct(*p) for p in pairs]
        torch.cuda.synchronize()
        got, errors = {}, []

        def work(i):
            try:
                got[i] = [top.gemm_mx_nt_direct(*pairs[i]) for _ in range(50)]
                torch.cuda.synchronize()
            except Exception as e:
                errors.append(e)

        threads = [threading.Thread(target=work, args=(i,)) for i in range(4)]
        for t in threads:
            t.start()
        for t in threads:
            t.join()
        assert not errors
        assert all(torch.equal(c, want[i]) for i in range(4) for c in got[i])

    def test_graph_replay(self, gpu):
        """A captured quantise + product reads its inputs anew on each replay."""
        x, w = torch.randn(48, 512, device="cuda").bfloat16(), torch.randn(96, 512, device="cuda").bfloat16()
        wq, ws = top.quantize_mx_direct(w)
        top.gemm_mx_nt_direct(*top.quantize_mx_direct(x), wq, ws)  # the plan allocates once
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            c = top.gemm_mx_nt_direct(*top.quantize_mx_direct(x), wq, ws)
        for seed in range(3):
            x.copy_(torch.randn(48, 512, generator=torch.Generator().manual_seed(seed)))
            graph.replay()
            assert torch.equal(c, top.gemm_mx_nt_direct(*top.quantize_mx_direct(x), wq, ws))

    def test_host_pipeline(self, gpu):
        """The host pipeline moves K/2 bytes per row of a 4-bit operand."""
        M, N, K = 96, 128, 512
        rng = np.random.default_rng(2)
        (qa, sa, a), (qb, sb, b) = exact_operand(M, K, rng), exact_operand(N, K, rng)
        plan = GemmPlan(M, N, K, "mxe2m1", "f32")
        packed = []
        for q, sc in ((a, sa), (b, sb)):
            packed.append(top.quantize_mx_direct(torch.from_numpy(q.astype(np.float32)).cuda()))
        # requantising exact values keeps them, but may pick another power of two: take its codes and scales
        plan.set_mx_scales(packed[0][1].data_ptr(), packed[1][1].data_ptr())
        pipe = HostGemmPipeline(plan)
        hA, hB = pipe.pinned_operands()
        hA.array[:], hB.array[:] = packed[0][0].cpu().numpy(), packed[1][0].cpu().numpy()
        assert pipe.h2d_bytes_per_problem == (M + N) * K // 2
        got = [pipe.result(pipe.submit(hA, hB)).copy() for _ in range(3)]
        pipe.close()
        hA.free(), hB.free()
        assert all(np.array_equal(g, product(a, b).astype(np.float32)) for g in got)
