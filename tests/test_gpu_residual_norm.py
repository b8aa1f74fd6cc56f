"""GPU tests of the residual addition with its RMSNorm (BF16 and MXFP8 outputs) against the
formula in 64 bits.

n = s * (mean(s^2) + eps)^-1/2 * w is computed to over 40 bits, rounded to FP32 and then to
BF16, as a conversion from 64 bits does. It equals the formula rounded that way except where
the 64-bit value lies within 2^-40 (relative) of a border: no element in the sizes tested
here is expected there, and the comparison is for equality."""

from __future__ import annotations

import pytest
import torch

pytestmark = pytest.mark.gpu

EPS = 1e-6


def _inputs(rows: int, width: int, seed: int):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(rows, width, generator=g).bfloat16()
    residual = (3 * torch.randn(rows, width, generator=g) * torch.exp2(torch.randint(-8, 8, (rows, 1), generator=g).float())).bfloat16()
    weight = (1 + 0.2 * torch.randn(width, generator=g)).bfloat16()
    return x.cuda(), residual.cuda(), weight.cuda()


def _formula(s: torch.Tensor, weight: torch.Tensor, eps: float = EPS) -> torch.Tensor:
    eps = float(torch.tensor(eps, dtype=torch.float32))  # eps crosses the ABI in 32 bits
    v = s.double()
    n = v / torch.sqrt(v.square().mean(1, keepdim=True) + eps) * weight.double()
    return n.float().bfloat16()


SIZES = [(1, 1), (1, 8), (1, 512), (3, 31), (2, 33), (5, 128), (7, 769), (64, 512), (130, 1000),
         (9, 2048), (4, 4104), (3, 8192), (2, 8200), (2, 20000), (1, 65536), (1, 70001), (700, 128), (3000, 264),
         # Rows enough for the blocks to take several in turn, at each of their widths.
         (70000, 33), (30000, 100), (40001, 128), (14000, 250), (9601, 512), (9600, 509), (4000, 1000), (4000, 1001),
         (2001, 2048), (2000, 2045), (1000, 4096), (1000, 4001), (500, 8192), (500, 8191), (300, 16384), (300, 16001),
         (100, 32768), (100, 32001)]


@pytest.mark.parametrize("rows,width", SIZES)
def test_add_rmsnorm_forward_is_the_rounded_formula(rows: int, width: int) -> None:
    from ce4b200 import kernels

    x, residual, weight = _inputs(rows, width, rows + width)
    total, n = kernels.add_rmsnorm_forward(x, residual, weight)
    expected = (x.float() + residual.float()).bfloat16()
    assert torch.equal(total, expected)
    assert torch.equal(n, _formula(expected, weight))


@pytest.mark.parametrize("rows,width", [(1, 512), (5, 129), (33, 2048)])
def test_without_a_residual_it_is_the_norm_of_x(rows: int, width: int) -> None:
    from ce4b200 import kernels

    x, _, weight = _inputs(rows, width, 3)
    total, n = kernels.add_rmsnorm_forward(x, None, weight)
    assert total is x
    assert torch.equal(n, _formula(x, weight))
    # The FP32 operator rounds a value whose error is about 2^-22 of it (sum, root, two
    # products): it may fall on the other BF16 neighbour, one step of at most 2^-7 away.
    torch.testing.assert_close(kernels.rmsnorm_forward(x, weight).float(), n.float(), rtol=2.0**-7, atol=0)


@pytest.mark.parametrize("rows,width", [(1, 128), (3, 512), (64, 512), (127, 384), (129, 2048), (256, 1024),
                                        (2, 8192), (1, 16384), (300, 4224), (9700, 512), (5000, 896), (1300, 2048),
                                        (700, 4096), (330, 8192), (160, 16384), (90, 32768)])
def test_mxfp8_output_equals_quantising_the_bf16_one(rows: int, width: int) -> None:
    from ce4b200 import kernels
    from oracle import mxfp8

    x, residual, weight = _inputs(rows, width, rows * width)
    residual[0, :32] = -x[0, :32]  # an all-zero scale block
    total, q = kernels.add_rmsnorm_mxfp8(x, residual, weight)
    plain_total, n = kernels.add_rmsnorm_forward(x, residual, weight)
    assert torch.equal(total, plain_total)
    padded = torch.zeros(-(-rows // 128) * 128, width, dtype=torch.bfloat16)
    padded[:rows] = n.cpu()
    codes, scales = mxfp8.quantize(padded)
    assert torch.equal(q.values.view(torch.uint8).cpu(), codes[:rows])
    got, want = mxfp8.unswizzle_scales(q.scales.cpu()), mxfp8.unswizzle_scales(scales)
    assert torch.equal(got[:rows], want[:rows])
    assert not got[rows:].any()


def test_a_row_does_not_depend_on_the_batch_or_the_alignment() -> None:
    from ce4b200 import kernels

    x, residual, weight = _inputs(600, 512, 11)
    total, n = kernels.add_rmsnorm_forward(x, residual, weight)
    for r in (0, 17, 599):
        one_total, one = kernels.add_rmsnorm_forward(x[r:r + 1], residual[r:r + 1], weight)
        assert torch.equal(one_total[0], total[r]) and torch.equal(one[0], n[r])
    # The same values at addresses that no wide load may touch.
    shift = [torch.empty(t.numel() + 1, dtype=t.dtype, device="cuda")[1:].view(t.shape).copy_(t)
             for t in (x, residual, weight)]
    assert shift[0].data_ptr() % 4 == 2
    odd_total, odd = kernels.add_rmsnorm_forward(*shift)
    assert torch.equal(odd_total, total) and torch.equal(odd, n)
    _, q = kernels.add_rmsnorm_mxfp8(x, residual, weight)
    _, odd_q = kernels.add_rmsnorm_mxfp8(*shift)
    assert torch.equal(q.values.view(torch.uint8), odd_q.values.view(torch.uint8))
    assert torch.equal(q.scales, odd_q.scales)


def test_special_values_stay_in_their_row() -> None:
    from ce4b200 import kernels

    x, residual, weight = _inputs(6, 256, 5)
    x[1], residual[1] = 0, 0
    x[2, 7] = float("nan")
    x[3, 9] = float("inf")
    x[4] = 2.0**100  # squares beyond FP32
    residual[4] = 2.0**100
    total, n = kernels.add_rmsnorm_forward(x, residual, weight)
    clean = [0, 5]
    assert torch.equal(n[clean], _formula(total[clean], weight))
    assert not n[1].any()
    assert n[2].isnan().all()
    assert n[3, 9].isnan() and not n[3, :9].any() and not n[3, 10:].any()
    assert torch.equal(n[4], _formula(total[4:5], weight)[0])


def test_the_c_entry_writes_the_sum_in_place() -> None:
    from ce4b200 import _lib, kernels

    x, residual, weight = _inputs(37, 640, 8)
    total, n = kernels.add_rmsnorm_forward(x, residual, weight)
    stream = torch.cuda.current_stream().cuda_stream
    for target in ("x", "residual"):
        a, b = x.clone(), residual.clone()
        out = torch.empty_like(x)
        s = a if target == "x" else b
        _lib.check(_lib.library().ce4b_add_rmsnorm(
            a.data_ptr(), b.data_ptr(), weight.data_ptr(), s.data_ptr(), out.data_ptr(), 37, 640, EPS, stream))
        assert torch.equal(s, total) and torch.equal(out, n)


def test_graph_replay_reads_new_inputs() -> None:
    from ce4b200 import kernels

    x, residual, weight = _inputs(48, 512, 21)
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        kernels.add_rmsnorm_mxfp8(x, residual, weight)
    torch.cuda.current_stream().wait_stream(stream)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        total, n = kernels.add_rmsnorm_forward(x, residual, weight)
        total8, q = kernels.add_rmsnorm_mxfp8(total, n, weight)
    x2, residual2, _ = _inputs(48, 512, 22)
    x.copy_(x2)
    residual.copy_(residual2)
    graph.replay()
    want_total, want_n = kernels.add_rmsnorm_forward(x2, residual2, weight)
    want_total8, want_q = kernels.add_rmsnorm_mxfp8(want_total, want_n, weight)
    assert torch.equal(total, want_total) and torch.equal(n, want_n) and torch.equal(total8, want_total8)
    assert torch.equal(q.values.view(torch.uint8), want_q.values.view(torch.uint8))
    assert torch.equal(q.scales, want_q.scales)


@pytest.mark.parametrize("rows,d,h", [(1, 256, 512), (77, 512, 1536), (128, 256, 768), (300, 512, 1024)])
def test_mxfp8_blocks_of_a_ragged_batch(rows: int, d: int, h: int) -> None:
    """Two MXFP8 products as a tower chains them: the norm's codes feed the block-scaled GEMM
    with any number of rows, and the next norm adds the product to the stream. Each product
    is compared with the 64-bit product of the dequantised operands: one BF16 rounding (2^-8)
    and FP32 sums of K / 32 steps, each off by at most 2^-22 of the sum of magnitudes."""

    from ce4b200 import kernels
    from oracle import mxfp8

    g = torch.Generator().manual_seed(rows + d)
    x, residual, weight = _inputs(rows, d, 4)
    up = kernels.quantize_mxfp8((torch.randn(h, d, generator=g) / d**0.5).bfloat16().cuda())
    down = kernels.quantize_mxfp8((torch.randn(d, h, generator=g) / h**0.5).bfloat16().cuda())
    ones = torch.ones(h, dtype=torch.bfloat16, device="cuda")

    def product(left, right):
        got = kernels.mxfp8_gemm(left, right)
        pad = -(-rows // 128) * 128
        codes = torch.zeros(pad, left.values.shape[1], dtype=torch.uint8)
        codes[:rows] = left.values.view(torch.uint8).cpu()
        a = mxfp8.dequantize(codes, left.scales.cpu())[:rows].double()
        b = mxfp8.dequantize(right.values.view(torch.uint8).cpu(), right.scales.cpu()).double()
        ref, mags = a @ b.T, a.abs() @ b.abs().T
        err = (got.double().cpu() - ref).abs()
        assert bool((err <= ref.abs() * 2.0**-8 + mags * (b.shape[1] / 32 * 2.0**-22)).all())
        return got

    total, n = kernels.add_rmsnorm_mxfp8(x, residual, weight)
    hidden = product(n, up)
    _, hidden8 = kernels.add_rmsnorm_mxfp8(hidden, None, ones)
    y = product(hidden8, down)
    final, q = kernels.add_rmsnorm_mxfp8(y, total, weight)
    assert torch.equal(final, (y.float() + total.float()).bfloat16())
    assert q.values.shape == (rows, d)
    with pytest.raises(ValueError, match="padded"):
        kernels.mxfp8_gemm(kernels.Mxfp8Tensor(n.values[:1], n.scales[:0]), up)


def test_a_row_of_the_largest_width() -> None:
    """Column counters past 2^31 do not come back negative. The row repeats 2^16 values, so that
    its statistics and its results are those of one period."""

    from ce4b200 import kernels

    width, period = 2**31 - 256, 2**16
    whole = width // period * period
    values, _, gains = _inputs(1, period, 11)

    def repeated(v: torch.Tensor) -> torch.Tensor:
        row = torch.empty(width, dtype=torch.bfloat16, device="cuda")
        row[:whole].view(-1, period).copy_(v.view(1, -1).expand(whole // period, -1))
        row[whole:] = v.flatten()[: width - whole]
        return row

    squares = values.double().square().flatten()
    mean = (squares.sum() * (whole // period) + squares[: width - whole].sum()) / width
    eps = float(torch.tensor(EPS, dtype=torch.float32))
    expected = (values.double() / torch.sqrt(mean + eps) * gains.double()).float().bfloat16().flatten()
    _, n = kernels.add_rmsnorm_forward(repeated(values)[None], None, repeated(gains))
    n = n.flatten()
    for start in range(0, whole, 2**28):
        assert bool((n[start : min(start + 2**28, whole)].view(-1, period) == expected).all())
    assert torch.equal(n[whole:], expected[: width - whole])
