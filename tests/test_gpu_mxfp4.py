"""GPU tests of MXFP4 weights: the quantiser against a plain restatement, the products with
few BF16 rows against the dequantised product in 64 bits.

Tolerances of the products. Weights (code times scale) and activations are BF16 values and
their products exact in FP32. What is off is the FP32 sum: K / 16 steps of a tensor core, each
off by at most two FP32 steps (2^-22) of a partial sum, which is at most the sum of magnitudes,
so K / 16 * 2^-22 = K / 128 * 2^-19 of that sum; and one BF16 rounding, at most half a step,
2^-8 of the value."""

from __future__ import annotations

import pytest
import torch

pytestmark = pytest.mark.gpu

GRID = torch.tensor([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0])


def _unswizzle(scales: torch.Tensor, rows: int) -> torch.Tensor:
    rt, ct = scales.shape[:2]
    s = scales.reshape(rt, ct, 32, 4, 4).permute(0, 3, 2, 1, 4)
    return s.reshape(rt * 128, ct * 4)[:rows]


def _values(q) -> torch.Tensor:
    """FP64 [rows, cols] on the CPU of an Mxfp4Tensor, from the format's definition."""

    codes = q.values.cpu().long()
    nibbles = torch.stack((codes & 15, codes >> 4), 2).flatten(1)
    table = torch.cat((GRID, -GRID)).double()
    power = _unswizzle(q.scales.cpu(), codes.shape[0])
    scale = torch.where(power == 255, float("nan"), torch.exp2(power.double() - 127))
    return table[nibbles] * scale.repeat_interleave(32, 1)


def _reference_quantize(w: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor]:
    """(values FP64, scale codes) of a finite BF16 matrix, group by group."""

    g = w.cpu().double().reshape(w.shape[0], -1, 32)
    top = g.abs().amax(2)
    power = torch.full_like(top, -39)
    for e in range(-39, 127):  # the smallest power that holds the group
        power = torch.where((top > 6 * 2.0**e), e + 1.0, power)
    mag = (g.abs() * torch.exp2(-power)[:, :, None])
    distance = (mag[..., None] - GRID.double()).abs()
    # nearest, and of two nearest the one with the even code
    best = (distance + torch.tensor([0, 1, 0, 1, 0, 1, 0, 1]) * 1e-9).argmin(3)
    values = GRID.double()[best] * torch.sign(g) * torch.exp2(power)[:, :, None]
    return values.reshape(w.shape), (power + 127).to(torch.uint8)


def _weight(rows: int, cols: int, seed: int, spread: int = 4) -> torch.Tensor:
    g = torch.Generator().manual_seed(seed)
    scale = torch.exp2(torch.randint(-spread, spread + 1, (rows, cols // 32, 1), generator=g).float())
    w = (0.02 * torch.randn(rows, cols // 32, 32, generator=g) * scale).reshape(rows, cols)
    return w.bfloat16()


@pytest.mark.parametrize("rows,cols", [(1, 128), (3, 256), (127, 128), (130, 640), (512, 1536), (129, 2048)])
def test_quantizer_is_the_nearest_code_under_the_smallest_scale(rows: int, cols: int) -> None:
    from ce4b200 import kernels

    w = _weight(rows, cols, rows + cols, spread=20)
    w[0, :32] = 0
    w[-1, 32:64] = torch.linspace(-6, 6, 32).bfloat16()            # ties between codes
    w[0, 64:96] = torch.tensor([0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0, 6.0] * 4).bfloat16() / 16
    w[0, 96:128] = 1e-30                                           # below the smallest scale
    q = kernels.quantize_mxfp4(w.cuda())
    values, scales = _reference_quantize(w)
    assert q.shape == (rows, cols)
    assert torch.equal(_unswizzle(q.scales.cpu(), rows), scales)
    padding = _unswizzle(q.scales.cpu(), q.scales.shape[0] * 128)[rows:]
    assert not padding.any()
    assert torch.equal(_values(q), values)
    assert torch.equal(kernels.dequantize_mxfp4(q).cpu().double(), values)


def test_quantizer_marks_groups_that_are_not_finite() -> None:
    from ce4b200 import kernels

    w = _weight(4, 256, 9)
    w[1, 40] = float("nan")
    w[2, 200] = float("-inf")
    w[3, 0] = torch.finfo(torch.bfloat16).max
    q = kernels.quantize_mxfp4(w.cuda())
    got = kernels.dequantize_mxfp4(q).cpu()
    bad = torch.zeros(4, 256, dtype=torch.bool)
    bad[1, 32:64] = True
    bad[2, 192:224] = True
    assert torch.equal(got.isnan(), bad)
    assert torch.equal(_unswizzle(q.scales.cpu(), 4)[[1, 2, 3], [1, 6, 0]], torch.tensor([255, 255, 253], dtype=torch.uint8))


def _assert_product(got: torch.Tensor, ref: torch.Tensor, mags: torch.Tensor, k: int) -> None:
    bound = ref.abs() * 2.0**-8 + mags * (k / 128) * 2.0**-19 * (1 + 2.0**-8)
    err = (got.double().cpu() - ref).abs()
    assert bool((err <= bound).all()), float((err / bound.clamp(min=1e-300)).max())


def _product(x: torch.Tensor, w: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor]:
    return x.cpu().double() @ w.T, x.cpu().double().abs() @ w.abs().T


ROWS = [1, 2, 7, 8, 9, 16, 17, 31, 33, 63, 64, 65, 130]
SHAPES = [(1, 128), (16, 128), (127, 256), (128, 384), (130, 512), (512, 1536), (1000, 1024), (2048, 128), (257, 4096)]


@pytest.mark.parametrize("rows", ROWS)
def test_linear_over_row_counts(rows: int) -> None:
    from ce4b200 import kernels

    n, k = 200, 640
    g = torch.Generator().manual_seed(rows)
    q = kernels.quantize_mxfp4(_weight(n, k, 77).cuda())
    x = torch.randn(rows, k, generator=g).bfloat16().cuda()
    residual = torch.randn(rows, n, generator=g).bfloat16().cuda()
    ref, mags = _product(x, _values(q))
    _assert_product(kernels.mxfp4_linear(x, q), ref, mags, k)
    _assert_product(kernels.mxfp4_linear(x, q, residual=residual), ref + residual.cpu().double(), mags, k)


@pytest.mark.parametrize("rows", [1, 12, 20, 48, 64])
@pytest.mark.parametrize("n,k", SHAPES)
def test_linear_over_shapes(rows: int, n: int, k: int) -> None:
    from ce4b200 import kernels

    g = torch.Generator().manual_seed(n + k + rows)
    q = kernels.quantize_mxfp4(_weight(n, k, n * k).cuda())
    # Activations over many binades inside a group, exact zeros, one large channel.
    x = torch.randn(rows, k, generator=g) * torch.exp2(torch.randint(-12, 4, (rows, k), generator=g).float())
    x[torch.rand(rows, k, generator=g) < 0.1] = 0
    x[:, 5] *= 300
    x = x.bfloat16().cuda()
    ref, mags = _product(x, _values(q))
    _assert_product(kernels.mxfp4_linear(x, q), ref, mags, k)


@pytest.mark.parametrize("n,k", [(2400, 256), (9500, 384), (20001, 128), (1030, 8192), (4100, 1152)])
@pytest.mark.parametrize("rows", [3, 9, 30, 41])
def test_linear_over_large_weights(rows: int, n: int, k: int) -> None:
    """Weights of many row tiles, or of K blocks that the warps share unevenly."""

    from ce4b200 import kernels

    g = torch.Generator().manual_seed(n)
    q = kernels.quantize_mxfp4(_weight(n, k, 5, spread=2).cuda())
    x = torch.randn(rows, k, generator=g).bfloat16().cuda()
    residual = torch.randn(rows, n, generator=g).bfloat16().cuda()
    ref, mags = _product(x, _values(q))
    _assert_product(kernels.mxfp4_linear(x, q, residual=residual), ref + residual.cpu().double(), mags, k)


@pytest.mark.parametrize("rows", [1, 5, 12, 17, 33, 64, 100])
@pytest.mark.parametrize("hidden,k", [(1, 128), (64, 256), (100, 128), (192, 512), (1536, 512), (300, 2048), (4777, 256)])
def test_swiglu(rows: int, hidden: int, k: int) -> None:
    """silu(g) u is off by |d(silu u)| <= 1.1 |u| dg + |silu(g)| du for sums off by dg, du
    (|silu'| < 1.1), by a few FP32 roundings of the formula, and by one BF16 rounding."""

    from ce4b200 import kernels

    g = torch.Generator().manual_seed(rows + hidden + k)
    q = kernels.quantize_mxfp4((4 * _weight(2 * hidden, k, hidden + k, spread=1).float()).bfloat16().cuda())
    x = torch.randn(rows, k, generator=g).bfloat16().cuda()
    got = kernels.mxfp4_swiglu(x, q)
    y, mags = _product(x, _values(q))
    gate, up = y[:, :hidden], y[:, hidden:]
    off = mags * (k / 128) * 2.0**-19
    silu = gate * torch.sigmoid(gate)
    ref = silu * up
    bound = ref.abs() * (2.0**-8 + 2.0**-20) + 1.1 * (up.abs() + off[:, hidden:]) * off[:, :hidden] + silu.abs() * off[:, hidden:]
    err = (got.double().cpu() - ref).abs()
    assert bool((err <= bound * (1 + 2.0**-7)).all()), float((err / bound.clamp(min=1e-300)).max())


def test_gate_far_from_zero_saturates() -> None:
    """silu of a large negative gate is -0 or tiny, of a large positive one the gate itself."""

    from ce4b200 import kernels

    w = torch.zeros(4, 128, dtype=torch.bfloat16)
    w[0, 0], w[1, 0], w[2:, 1] = 4.0, -4.0, 1.0
    x = torch.zeros(1, 128, dtype=torch.bfloat16)
    x[0, 0], x[0, 1] = 1000.0, 2.0
    got = kernels.mxfp4_swiglu(x.cuda(), kernels.quantize_mxfp4(w.cuda())).cpu()
    assert got[0, 0] == 8000 and got[0, 1] == 0


@pytest.mark.parametrize("power", [-37, -20, 2, 10, 60])
def test_scales_over_the_whole_range(power: int) -> None:
    from ce4b200 import kernels

    g = torch.Generator().manual_seed(5)
    w = (_weight(130, 256, 4, spread=0).float() * 50 * 2.0**power).bfloat16()
    q = kernels.quantize_mxfp4(w.cuda())
    x = (torch.randn(3, 256, generator=g) * 2.0**-power).bfloat16().cuda()
    ref, mags = _product(x, _values(q))
    _assert_product(kernels.mxfp4_linear(x, q), ref, mags, 256)


@pytest.mark.parametrize("rows", [2, 40])
@pytest.mark.parametrize("low", [0, 1, 5, 40, 200, 245])
def test_scale_codes_of_other_quantisers(rows: int, low: int) -> None:
    """Scales that quantize_mxfp4 does not choose: from 2^-127 (weights that are subnormal in
    BF16) to 2^121."""

    from ce4b200 import kernels

    g = torch.Generator().manual_seed(low)
    codes = torch.randint(0, 256, (140, 128), generator=g, dtype=torch.uint8)
    scales = torch.randint(low, low + 4, (2, 2, 32, 16), generator=g, dtype=torch.uint8)
    q = kernels.Mxfp4Tensor(codes.cuda(), scales.cuda())
    assert torch.equal(kernels.dequantize_mxfp4(q).cpu().double(), _values(q))
    x = (torch.randn(rows, 256, generator=g) * 2.0 ** max(-100, min(110, 127 - low))).bfloat16().cuda()
    ref, mags = _product(x, _values(q))
    _assert_product(kernels.mxfp4_linear(x, q), ref, mags, 256)


def test_tiny_and_huge_activations() -> None:
    from ce4b200 import kernels

    g = torch.Generator().manual_seed(6)
    q = kernels.quantize_mxfp4(_weight(64, 256, 8).cuda())
    base = torch.randn(4, 256, generator=g)
    for power in (-100, 100):
        x = (base * 2.0**power).bfloat16().cuda()
        ref, mags = _product(x, _values(q))
        _assert_product(kernels.mxfp4_linear(x, q), ref, mags, 256)


@pytest.mark.parametrize("rows", [12, 20, 40])
def test_values_that_are_not_finite_stay_in_their_row(rows: int) -> None:
    from ce4b200 import kernels

    g = torch.Generator().manual_seed(3)
    w = _weight(300, 512, 12)
    q = kernels.quantize_mxfp4(w.cuda())
    x = torch.randn(rows, 512, generator=g).bfloat16()
    clean = kernels.mxfp4_linear(x.cuda(), q)
    x[3, 100] = float("nan")
    x[11, 511] = float("inf")
    got = kernels.mxfp4_linear(x.cuda(), q)
    others = [r for r in range(rows) if r not in (3, 11)]
    assert torch.equal(got[others], clean[others])
    assert not got[[3, 11]].isfinite().any()
    # A weight row that is not finite spoils its output column alone.
    w[7, 40] = float("nan")
    got, clean = (kernels.mxfp4_linear(x[:2].cuda(), p) for p in (kernels.quantize_mxfp4(w.cuda()), q))
    assert got[:, 7].isnan().all() and torch.equal(got[:, 8:], clean[:, 8:])


def test_a_row_does_not_depend_on_its_neighbours() -> None:
    from ce4b200 import kernels

    g = torch.Generator().manual_seed(31)
    q = kernels.quantize_mxfp4(_weight(256, 1024, 2).cuda())
    x = torch.randn(8, 1024, generator=g).bfloat16().cuda()
    full = kernels.mxfp4_linear(x, q)
    x2 = x.clone()
    x2[1:] = 0
    assert torch.equal(kernels.mxfp4_linear(x2, q)[0], full[0])
    assert torch.equal(kernels.mxfp4_linear(x, q), full)  # and calls repeat bit for bit


@pytest.mark.parametrize("rows,d,h", [(1, 128, 384), (17, 256, 768), (64, 512, 1536), (70, 256, 1024)])
def test_dense_block_mxfp4_runs_norm_products_and_residual(rows: int, d: int, h: int) -> None:
    """The block against its formula in 64 bits on the dequantised weights, with the two BF16
    roundings between its operators restated: a product off by its tolerance may move such a
    rounding by one step (2^-7 of the value), so steps of n and of the hidden row are allowed."""

    from ce4b200 import kernels

    g = torch.Generator().manual_seed(d)
    x = torch.randn(rows, d, generator=g).bfloat16().cuda()
    norm_weight = (1 + 0.1 * torch.randn(d, generator=g)).bfloat16().cuda()
    wgu, wd = _weight(2 * h, d, 1, spread=1).cuda(), _weight(d, h, 2, spread=1).cuda()
    gate_up, down = kernels.quantize_mxfp4(wgu), kernels.quantize_mxfp4(wd)
    out = kernels.dense_block_forward(x, norm_weight, gate_up, down, precision="mxfp4")
    assert torch.equal(out, kernels.dense_block_forward(x, norm_weight, wgu, wd, precision="mxfp4"))
    v = x.double().cpu()
    n = (v / torch.sqrt(v.square().mean(1, keepdim=True) + 1e-6) * norm_weight.double().cpu()).bfloat16().double()
    y = n @ _values(gate_up).T
    gate, up = y[:, :h], y[:, h:]
    hidden = (gate * torch.sigmoid(gate) * up).bfloat16().double()
    ref = v + hidden @ _values(down).T
    mags = hidden.abs() @ _values(down).abs().T
    err = (out.double().cpu() - ref).abs()
    assert bool((err <= ref.abs() * 2.0**-8 + mags * 2.0**-7).all())
    assert float(err.norm() / ref.norm()) <= 2.0**-8


def test_blocks_chained_by_the_residual_norm() -> None:
    """Two 4-bit blocks as a tower runs them: the norm between them adds the residual."""

    from ce4b200 import kernels

    d, h, rows = 256, 768, 24
    g = torch.Generator().manual_seed(8)
    x = torch.randn(rows, d, generator=g).bfloat16().cuda()
    w = [(1 + 0.1 * torch.randn(d, generator=g)).bfloat16().cuda() for _ in range(2)]
    gate_up = [kernels.quantize_mxfp4(_weight(2 * h, d, 10 + i, spread=1).cuda()) for i in range(2)]
    down = [kernels.quantize_mxfp4(_weight(d, h, 20 + i, spread=1).cuda()) for i in range(2)]
    _, n = kernels.add_rmsnorm_forward(x, None, w[0])
    y = kernels.mxfp4_linear(kernels.mxfp4_swiglu(n, gate_up[0]), down[0])
    total, n = kernels.add_rmsnorm_forward(y, x, w[1])
    out = kernels.mxfp4_linear(kernels.mxfp4_swiglu(n, gate_up[1]), down[1], residual=total)
    stepped = kernels.dense_block_forward(x, w[0], gate_up[0], down[0], precision="mxfp4")
    stepped = kernels.dense_block_forward(stepped, w[1], gate_up[1], down[1], precision="mxfp4")
    # The chained form rounds the down product before the sum, the block form after it: the
    # stream differs by half a BF16 step of the product (2^-8), carried through one block.
    assert float((out.float() - stepped.float()).norm() / stepped.float().norm()) <= 2.0**-7


def test_the_c_entry_adds_into_the_residual() -> None:
    from ce4b200 import _lib, kernels

    g = torch.Generator().manual_seed(2)
    q = kernels.quantize_mxfp4(_weight(300, 256, 6).cuda())
    stream = torch.cuda.current_stream().cuda_stream
    for rows in (5, 40):
        x = torch.randn(rows, 256, generator=g).bfloat16().cuda()
        residual = torch.randn(rows, 300, generator=g).bfloat16().cuda()
        want = kernels.mxfp4_linear(x, q, residual=residual)
        _lib.check(_lib.library().ce4b_mxfp4_linear(
            x.data_ptr(), q.values.data_ptr(), q.scales.data_ptr(), residual.data_ptr(), residual.data_ptr(),
            rows, 300, 256, stream))
        assert torch.equal(residual, want)


@pytest.mark.parametrize("rows", [9, 50])
def test_graph_replay_and_two_streams(rows: int) -> None:
    from ce4b200 import kernels

    g = torch.Generator().manual_seed(13)
    q = kernels.quantize_mxfp4(_weight(384, 512, 3).cuda())
    x = torch.randn(rows, 512, generator=g).bfloat16().cuda()
    kernels.mxfp4_linear(x, q)
    torch.cuda.synchronize()
    graphs, outs = [], []
    for _ in range(2):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs.append(kernels.mxfp4_linear(kernels.mxfp4_linear(x, q).repeat(1, 2)[:, :512].contiguous(), q))
        graphs.append(graph)
    x.copy_(torch.randn(rows, 512, generator=g).bfloat16())
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    for _ in range(20):
        for graph, stream in zip(graphs, streams):
            with torch.cuda.stream(stream):
                graph.replay()
    torch.cuda.synchronize()
    want = kernels.mxfp4_linear(kernels.mxfp4_linear(x, q).repeat(1, 2)[:, :512].contiguous(), q)
    assert torch.equal(outs[0], want) and torch.equal(outs[1], want)


def test_every_operand_may_come_from_the_kernel_before() -> None:
    """Kernels start under their predecessor's tail; what it writes last, a norm weight or a
    quantised matrix included, is read after it."""

    from ce4b200 import kernels

    g = torch.Generator().manual_seed(5)
    base = torch.randn(2048, 1024, generator=g).bfloat16().cuda()

    def chain(x: torch.Tensor, wait: bool) -> list[torch.Tensor]:
        pause = torch.cuda.synchronize if wait else lambda: None
        _, n = kernels.add_rmsnorm_forward(x, None, x[0])
        pause()
        _, n2 = kernels.add_rmsnorm_forward(n, x, n[-1])  # the weight: the rows written last
        pause()
        packed = kernels.quantize_mxfp4(n2)
        pause()
        back = kernels.dequantize_mxfp4(packed)
        pause()
        total, _ = kernels.add_rmsnorm_mxfp8(back, n2, back[-1])
        pause()
        y = kernels.mxfp4_linear(total[-3:].contiguous(), packed)
        pause()
        return [n, n2, packed.values, packed.scales, back, total, y]

    for i in range(8):
        x = base.roll(i, 0) * (i + 1)
        for a, b in zip(chain(x, False), chain(x, True), strict=True):
            assert torch.equal(a, b)
