"""CPU tests: what the residual norm and the MXFP4 operators refuse, in Python and at the C ABI,
before any GPU work."""

from __future__ import annotations

import pytest
import torch

from ce4b200 import _lib, kernels


class _Fake(torch.Tensor):
    """A CPU tensor that says it is on a GPU, to reach the checks behind the device's."""

    @property
    def device(self):  # type: ignore[override]
        return torch.device("cuda", getattr(self, "_index", 0))


def _gpu(*shape: int, dtype: torch.dtype = torch.bfloat16, index: int = 0) -> torch.Tensor:
    t = torch.zeros(*shape, dtype=dtype).as_subclass(_Fake)
    t._index = index
    return t


def _weight(rows: int, cols: int, **kw) -> kernels.Mxfp4Tensor:
    return kernels.Mxfp4Tensor(
        values=_gpu(rows, cols // 2, dtype=torch.uint8, **kw),
        scales=_gpu(-(-rows // 128), cols // 128, 32, 16, dtype=torch.uint8, **kw),
    )


def test_cpu_tensors_are_refused() -> None:
    x, w = torch.zeros(2, 128, dtype=torch.bfloat16), torch.ones(128, dtype=torch.bfloat16)
    for call in (kernels.add_rmsnorm_forward, kernels.add_rmsnorm_mxfp8):
        with pytest.raises(ValueError, match="CUDA"):
            call(x, None, w)
    with pytest.raises(ValueError, match="CUDA"):
        kernels.quantize_mxfp4(x)
    weight = kernels.Mxfp4Tensor(torch.zeros(4, 64, dtype=torch.uint8), torch.zeros(1, 1, 32, 16, dtype=torch.uint8))
    with pytest.raises(ValueError, match="CUDA"):
        kernels.dequantize_mxfp4(weight)
    with pytest.raises(ValueError, match="CUDA"):
        kernels.mxfp4_linear(x, weight)
    with pytest.raises(ValueError, match="CUDA"):
        kernels.dense_block_forward(x, w, weight, weight, precision="mxfp4")


@pytest.mark.parametrize("call", [kernels.add_rmsnorm_forward, kernels.add_rmsnorm_mxfp8])
def test_norm_refusals(call) -> None:
    x, w = _gpu(4, 256), _gpu(256)
    for bad in (_gpu(4, 128), _gpu(8, 256)):
        with pytest.raises(ValueError, match="residual must match x"):
            call(x, bad, w)
    with pytest.raises(ValueError, match="bfloat16"):
        call(_gpu(4, 256, dtype=torch.float16), None, w)
    with pytest.raises(ValueError, match="contiguous"):
        call(_gpu(4, 512)[:, ::2], None, w)
    with pytest.raises(ValueError, match="contiguous"):
        call(_gpu(256), None, w)
    with pytest.raises(ValueError, match=r"\[256\]"):
        call(x, None, _gpu(255))
    with pytest.raises(ValueError, match="x's device"):
        call(x, _gpu(4, 256, index=1), w)
    with pytest.raises(ValueError, match="x's device"):
        call(x, None, _gpu(256, index=1))
    with pytest.raises(ValueError, match="positive"):
        call(_gpu(0, 256), None, w)
    with pytest.raises(ValueError, match="positive"):
        call(_gpu(4, 0), None, _gpu(0))


def test_mxfp8_norm_needs_whole_scale_tiles() -> None:
    with pytest.raises(ValueError, match="multiple of 128"):
        kernels.add_rmsnorm_mxfp8(_gpu(4, 192), None, _gpu(192))


def test_mxfp4_weight_refusals() -> None:
    x = _gpu(3, 256)
    good = _weight(200, 256)
    bad = [
        (kernels.Mxfp4Tensor(_gpu(200, 128, dtype=torch.int8), good.scales), "uint8 CUDA"),
        (kernels.Mxfp4Tensor(_gpu(200, 256, dtype=torch.uint8)[:, ::2], good.scales), "contiguous"),
        (kernels.Mxfp4Tensor(_gpu(200, 96, dtype=torch.uint8), good.scales), "multiple of 128"),
        (kernels.Mxfp4Tensor(_gpu(0, 128, dtype=torch.uint8), good.scales), "positive"),
        (kernels.Mxfp4Tensor(good.values, _gpu(1, 2, 32, 16, dtype=torch.uint8)), r"\[2, 2, 32, 16\]"),
        (kernels.Mxfp4Tensor(good.values, _gpu(2, 2, 32, 16, dtype=torch.int32)), "uint8"),
        (kernels.Mxfp4Tensor(good.values, _gpu(2, 2, 32, 16, dtype=torch.uint8, index=1)), "device"),
        (_weight(200, 256, index=1), "x's device"),
        (good.values, "Mxfp4Tensor"),
    ]
    for weight, match in bad:
        for call in (kernels.mxfp4_linear, kernels.mxfp4_swiglu):
            with pytest.raises(ValueError, match=match):
                call(x, weight)
    with pytest.raises(ValueError, match="reduction"):
        kernels.mxfp4_linear(_gpu(3, 128), good)
    with pytest.raises(ValueError, match="reduction"):
        kernels.mxfp4_swiglu(_gpu(3, 384), good)
    with pytest.raises(ValueError, match="even"):
        kernels.mxfp4_swiglu(x, _weight(201, 256))
    for residual in (_gpu(3, 256), _gpu(2, 200), _gpu(3, 200, index=1)):
        with pytest.raises(ValueError, match=r"\[3, 200\]"):
            kernels.mxfp4_linear(x, good, residual=residual)
    with pytest.raises(ValueError, match="positive"):
        kernels.mxfp4_linear(_gpu(0, 256), good)
    with pytest.raises(ValueError, match="multiple of 128"):
        kernels.quantize_mxfp4(_gpu(4, 64))
    with pytest.raises(ValueError, match="positive"):
        kernels.quantize_mxfp4(_gpu(0, 128))


def test_dense_block_checks_mxfp4_shapes() -> None:
    x, w = _gpu(3, 256), _gpu(256)
    with pytest.raises(ValueError, match=r"\[1024, 256\]"):
        kernels.dense_block_forward(x, w, _weight(512, 256), _weight(256, 512), precision="mxfp4")
    with pytest.raises(ValueError, match=r"\[256, 512\]"):
        kernels.dense_block_forward(x, w, _weight(1024, 256), _weight(128, 512), precision="mxfp4")
    for precision in ("bf16", "mxfp8"):
        with pytest.raises(ValueError, match="BF16 weights"):
            kernels.dense_block_forward(x, w, _weight(1024, 256), _weight(256, 512), precision=precision)


def test_c_entries_check_on_the_host() -> None:
    lib, bad, p = _lib.library(), _lib.CE4B_ERR_INVALID_ARGUMENT, 4096

    def refused(status: int, text: str) -> None:
        assert status == bad and text in _lib.last_error()

    refused(lib.ce4b_add_rmsnorm(None, None, p, None, p, 1, 8, 1e-6, None), "null")
    refused(lib.ce4b_add_rmsnorm(p, p, p, None, p, 1, 8, 1e-6, None), "sum")
    refused(lib.ce4b_add_rmsnorm(p, None, p, None, p, 0, 8, 1e-6, None), "positive")
    refused(lib.ce4b_add_rmsnorm_mxfp8(p, None, p, None, p, p, 1, 64, 1e-6, None), "multiple of 128")
    refused(lib.ce4b_add_rmsnorm_mxfp8(p, None, p, None, p + 8, p, 1, 128, 1e-6, None), "aligned")
    refused(lib.ce4b_quantize_mxfp4(p, p, None, 1, 128, None), "null")
    refused(lib.ce4b_quantize_mxfp4(p, p, p, 1, 96, None), "multiple of 128")
    refused(lib.ce4b_quantize_mxfp4(p + 2, p, p, 1, 128, None), "aligned")
    refused(lib.ce4b_quantize_mxfp4(p, p, p + 4, 1, 128, None), "aligned")
    refused(lib.ce4b_dequantize_mxfp4(p, p + 4, p, 1, 128, None), "aligned")
    refused(lib.ce4b_dequantize_mxfp4(p, p, p, -1, 128, None), "positive")
    refused(lib.ce4b_dequantize_mxfp4(p, p, p + 2, 1, 128, None), "aligned")
    refused(lib.ce4b_mxfp4_linear(p, p, p, None, None, 1, 8, 128, None), "null")
    refused(lib.ce4b_mxfp4_linear(p, p, p, None, p, 1, 0, 128, None), "positive")
    refused(lib.ce4b_mxfp4_linear(p, p, p, None, p, 1, 8, 100, None), "multiple of 128")
    refused(lib.ce4b_mxfp4_linear(p + 2, p, p, None, p, 1, 8, 128, None), "aligned")
    refused(lib.ce4b_mxfp4_swiglu(p, p + 4, p, p, 1, 8, 128, None), "aligned")
    refused(lib.ce4b_mxfp4_swiglu(p, p, p, p, 1, 2**30, 128, None), "too large")


def test_c_entries_refuse_extents_that_would_wrap() -> None:
    lib, bad, p, top = _lib.library(), _lib.CE4B_ERR_INVALID_ARGUMENT, 4096, 2**31 - 1

    def refused(status: int) -> None:
        assert status == bad and ("too large" in _lib.last_error() or "at most" in _lib.last_error())

    refused(lib.ce4b_add_rmsnorm(p, None, p, None, p, 1, top, 1e-6, None))
    refused(lib.ce4b_add_rmsnorm(p, None, p, None, p, top, 1, 1e-6, None))
    refused(lib.ce4b_add_rmsnorm_mxfp8(p, None, p, None, p, p, top, 128, 1e-6, None))
    refused(lib.ce4b_quantize_mxfp4(p, p, p, top, 128, None))
    refused(lib.ce4b_dequantize_mxfp4(p, p, p, top, 128, None))
    refused(lib.ce4b_mxfp4_linear(p, p, p, None, p, 1, top, 128, None))
    refused(lib.ce4b_mxfp4_linear(p, p, p, None, p, top, 8, 128, None))
    refused(lib.ce4b_mxfp4_swiglu(p, p, p, p, 1, top // 2, 128, None))
    refused(lib.ce4b_mxfp8_gemm(p, p, p, p, p, top, 128, 128, None))


def test_c_entries_refuse_addresses_between_elements() -> None:
    """Any alignment of the elements: an address off two bytes holds no BF16 element."""

    lib, bad, p = _lib.library(), _lib.CE4B_ERR_INVALID_ARGUMENT, 4096

    def refused(status: int) -> None:
        assert status == bad and "2-byte aligned" in _lib.last_error()

    for i in range(5):
        x, residual, w, total, out = (p + (j == i) for j in range(5))
        refused(lib.ce4b_add_rmsnorm(x, residual, w, total, out, 1, 8, 1e-6, None))
        if i < 4:
            refused(lib.ce4b_add_rmsnorm_mxfp8(x, residual, w, total, p, p, 1, 128, 1e-6, None))
    refused(lib.ce4b_mxfp4_linear(p, p, p, p + 1, p, 1, 8, 128, None))
    refused(lib.ce4b_mxfp4_linear(p, p, p, None, p + 1, 1, 8, 128, None))
    refused(lib.ce4b_mxfp4_swiglu(p, p, p, p + 1, 1, 8, 128, None))
