"""GPU tests at the edges of the residual norm and the MXFP4 operators: weights and rows that are
not finite, scales next to the end of BF16, sums written in place off 16 bytes, batches of many
blocks, and the dense block as the chain of its operators. Tolerances of the products are those of
test_gpu_mxfp4."""

from __future__ import annotations

import pytest
import torch

from test_gpu_mxfp4 import _assert_product, _product, _values, _weight

pytestmark = pytest.mark.gpu

EPS = 1e-6


@pytest.mark.parametrize("rows", [2, 12, 20, 40])
@pytest.mark.parametrize("bad", [0, 7, 130, 299])
def test_a_weight_row_of_nan_spoils_its_output_column_alone(rows: int, bad: int) -> None:
    from ce4b200 import kernels

    g = torch.Generator().manual_seed(rows)
    w = _weight(300, 512, 12)
    x = torch.randn(rows, 512, generator=g).bfloat16().cuda()
    clean = kernels.mxfp4_linear(x, kernels.quantize_mxfp4(w.cuda()))
    w[bad, 40] = float("nan")
    got = kernels.mxfp4_linear(x, kernels.quantize_mxfp4(w.cuda()))
    others = [c for c in range(300) if c != bad]
    assert got[:, bad].isnan().all()
    assert clean.isfinite().all() and torch.equal(got[:, others], clean[:, others])


@pytest.mark.parametrize("rows", [2, 12, 20, 40])
def test_scales_next_to_the_end_of_bf16(rows: int) -> None:
    """Scale codes to 254: a code whose value leaves BF16 (2^128 and more) counts as infinite, in
    the matrix that the weight stands for and in the products. The first weight rows hold 0 and 1
    alone, times at most 2^127."""

    from ce4b200 import kernels

    g = torch.Generator().manual_seed(rows)
    n, k, finite = 140, 256, 70
    codes = torch.randint(0, 256, (n, k // 2), generator=g, dtype=torch.uint8)
    codes[:finite] &= 0xAA  # of each code the sign and the bit that stands for 1
    scales = torch.randint(249, 255, (2, k // 128, 32, 16), generator=g, dtype=torch.uint8)
    q = kernels.Mxfp4Tensor(codes.cuda(), scales.cuda())
    values = _values(q)
    expected = torch.where(values.abs() >= 2.0**128, values.sign() * float("inf"), values)
    assert torch.equal(kernels.dequantize_mxfp4(q).cpu().double(), expected)
    x = torch.randn(rows, k, generator=g)
    x = ((x.abs() + 0.25) * x.sign() * 2.0**-100).bfloat16().cuda()
    got = kernels.mxfp4_linear(x, q)
    ref, mags = _product(x, values[:finite])
    _assert_product(got[:, :finite], ref, mags, k)
    infinite = expected.isinf().any(1)
    assert infinite[finite:].any() and not infinite[:finite].any()
    assert not got.cpu()[:, infinite].isfinite().any()


@pytest.mark.parametrize("rows", [2, 12, 20, 40])
@pytest.mark.parametrize("low", [0, 1, 5, 40, 200, 245])
def test_swiglu_with_scale_codes_of_other_quantisers(rows: int, low: int) -> None:
    """Bound as in test_gpu_mxfp4.test_swiglu. A result below BF16's smallest normal number, 2^-126,
    is rounded to a multiple of 2^-133."""

    from ce4b200 import kernels

    g = torch.Generator().manual_seed(low + rows)
    hidden, k = 70, 256
    codes = torch.randint(0, 256, (2 * hidden, k // 2), generator=g, dtype=torch.uint8)
    scales = torch.randint(low, low + 4, (2, k // 128, 32, 16), generator=g, dtype=torch.uint8)
    q = kernels.Mxfp4Tensor(codes.cuda(), scales.cuda())
    x = (torch.randn(rows, k, generator=g) * 2.0 ** max(-100, min(110, 127 - low))).bfloat16().cuda()
    got = kernels.mxfp4_swiglu(x, q)
    y, mags = _product(x, _values(q))
    gate, up = y[:, :hidden], y[:, hidden:]
    off = mags * (k / 128) * 2.0**-19
    silu = gate * torch.sigmoid(gate)
    ref = silu * up
    bound = ref.abs() * (2.0**-8 + 2.0**-20) + 1.1 * (up.abs() + off[:, hidden:]) * off[:, :hidden] + silu.abs() * off[:, hidden:]
    err = (got.double().cpu() - ref).abs()
    assert bool((err <= bound * (1 + 2.0**-7) + 2.0**-134).all()), float((err / bound.clamp(min=1e-300)).max())


@pytest.mark.parametrize("rows", [200, 640, 4097])
def test_products_of_many_blocks_of_rows(rows: int) -> None:
    from ce4b200 import kernels

    g = torch.Generator().manual_seed(rows)
    n, k = 300, 256
    q = kernels.quantize_mxfp4(_weight(n, k, 9).cuda())
    x = torch.randn(rows, k, generator=g).bfloat16().cuda()
    residual = torch.randn(rows, n, generator=g).bfloat16().cuda()
    ref, mags = _product(x, _values(q))
    _assert_product(kernels.mxfp4_linear(x, q, residual=residual), ref + residual.cpu().double(), mags, k)
    hidden = kernels.mxfp4_swiglu(x, q)
    # Blocks of 64 rows are computed alike, whatever their number.
    for r in range(0, rows - 63, 64):
        assert torch.equal(hidden[r:r + 64], kernels.mxfp4_swiglu(x[r:r + 64], q))


@pytest.mark.parametrize("rows,d,h", [(1, 128, 384), (5, 512, 1536), (17, 256, 768), (64, 512, 1536), (70, 256, 1024)])
def test_the_dense_block_is_the_chain_of_its_operators(rows: int, d: int, h: int) -> None:
    from ce4b200 import kernels

    g = torch.Generator().manual_seed(d + rows)
    x = torch.randn(rows, d, generator=g).bfloat16().cuda()
    norm_weight = (1 + 0.1 * torch.randn(d, generator=g)).bfloat16().cuda()
    gate_up = kernels.quantize_mxfp4(_weight(2 * h, d, 1, spread=1).cuda())
    down = kernels.quantize_mxfp4(_weight(d, h, 2, spread=1).cuda())
    for eps in (EPS, 0.5):
        out = kernels.dense_block_forward(x, norm_weight, gate_up, down, precision="mxfp4", eps=eps)
        _, n = kernels.add_rmsnorm_forward(x, None, norm_weight, eps)
        assert torch.equal(out, kernels.mxfp4_linear(kernels.mxfp4_swiglu(n, gate_up), down, residual=x))


def _offset(t: torch.Tensor, elements: int) -> torch.Tensor:
    """The values of t in a buffer that starts `elements` off a wide boundary."""

    return torch.empty(t.numel() + elements, dtype=t.dtype, device=t.device)[elements:].view(t.shape).copy_(t)


def _norm_inputs(rows: int, width: int, seed: int) -> list[torch.Tensor]:
    g = torch.Generator().manual_seed(seed)
    x, residual = (torch.randn(rows, width, generator=g).bfloat16() for _ in range(2))
    return [x.cuda(), (3 * residual).cuda(), (1 + 0.2 * torch.randn(width, generator=g)).bfloat16().cuda()]


@pytest.mark.parametrize("offset", [0, 1, 4])
@pytest.mark.parametrize("rows,width", [(37, 641), (4000, 33), (2001, 1001), (64, 640), (300, 8201), (3, 40000)])
def test_the_sum_in_place_at_any_width_and_offset(rows: int, width: int, offset: int) -> None:
    """Rows off 16 bytes share chunks with their neighbours, which other blocks write meanwhile."""

    from ce4b200 import _lib, kernels

    x, residual, weight = _norm_inputs(rows, width, rows)
    total, n = kernels.add_rmsnorm_forward(x, residual, weight)
    s = total.double()
    want = s / torch.sqrt(s.square().mean(1, keepdim=True) + float(torch.tensor(EPS))) * weight.double()
    assert torch.equal(total, (x.float() + residual.float()).bfloat16()) and torch.equal(n, want.float().bfloat16())
    stream = torch.cuda.current_stream().cuda_stream
    for target in (0, 1):
        for _ in range(5):
            pair = [_offset(x, offset), _offset(residual, offset)]
            out = torch.empty_like(x)
            _lib.check(_lib.library().ce4b_add_rmsnorm(
                pair[0].data_ptr(), pair[1].data_ptr(), weight.data_ptr(), pair[target].data_ptr(), out.data_ptr(),
                rows, width, EPS, stream))
            assert torch.equal(pair[target], total) and torch.equal(out, n)
            assert torch.equal(pair[1 - target], (residual, x)[target])


@pytest.mark.parametrize("offset", [0, 1])
@pytest.mark.parametrize("rows,width", [(6, 256), (200, 512), (9700, 512), (6, 40960)])
def test_mxfp8_norm_of_rows_that_are_not_finite(rows: int, width: int, offset: int) -> None:
    """Bit for bit the codes and scales of the BF16 norm, which holds NaN and zeros there."""

    from ce4b200 import kernels

    x, residual, weight = _norm_inputs(rows, width, width)
    x[1], residual[1] = 0, 0
    x[2, 7] = float("nan")
    x[3, 9], x[3, width - 1] = float("inf"), float("-inf")
    x[4] = residual[4] = 2.0**100
    x, residual, weight = (_offset(t, offset) for t in (x, residual, weight))
    total, q = kernels.add_rmsnorm_mxfp8(x, residual, weight)
    plain_total, n = kernels.add_rmsnorm_forward(x, residual, weight)
    assert torch.equal(total.view(torch.int16), plain_total.view(torch.int16))
    assert n[2].isnan().all() and not n[1].any() and n[[0, 4, 5]].isfinite().all()
    padded = torch.zeros(-(-rows // 128) * 128, width, dtype=torch.bfloat16, device="cuda")
    padded[:rows] = n
    want = kernels.quantize_mxfp8(padded)
    assert torch.equal(q.values.view(torch.uint8), want.values.view(torch.uint8)[:rows])

    def by_row(scales: torch.Tensor) -> torch.Tensor:
        rt, ct = scales.shape[:2]
        return scales.reshape(rt, ct, 32, 4, 4).permute(0, 3, 2, 1, 4).reshape(rt * 128, ct * 4)

    assert torch.equal(by_row(q.scales)[:rows], by_row(want.scales)[:rows])
    assert not by_row(q.scales)[rows:].any()


def test_mxfp8_gemm_takes_scales_of_the_scale_type() -> None:
    from ce4b200 import kernels

    g = torch.Generator().manual_seed(1)
    a, b = (kernels.quantize_mxfp8(torch.randn(m, 256, generator=g).bfloat16().cuda()) for m in (128, 256))
    a8 = kernels.Mxfp8Tensor(a.values, a.scales.view(torch.float8_e8m0fnu))
    assert torch.equal(kernels.mxfp8_gemm(a8, b), kernels.mxfp8_gemm(a, b))
