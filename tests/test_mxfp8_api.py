"""CPU tests: what the MXFP8 product refuses before any GPU work. Its kernel copies whole scale
tiles, so a scale tensor of another size, type, order or device would be read out of range."""

from __future__ import annotations

import pytest
import torch

from ce4b200 import _lib, kernels


class _Fake(torch.Tensor):
    """A CPU tensor that says it is on a GPU, to reach the checks behind the device's."""

    @property
    def device(self):  # type: ignore[override]
        return torch.device(*getattr(self, "_where", ("cuda", 0)))


def _gpu(*shape: int, dtype: torch.dtype = torch.uint8, where: tuple = ("cuda", 0)) -> torch.Tensor:
    t = torch.zeros(*shape, dtype=torch.uint8 if dtype.itemsize == 1 else dtype)
    t = t.view(dtype).as_subclass(_Fake)
    t._where = where
    return t


def _operand(rows: int, cols: int, scales: torch.Tensor | None = None, **kw) -> kernels.Mxfp8Tensor:
    values = _gpu(rows, cols, dtype=torch.float8_e4m3fn, **kw)
    if scales is None:
        scales = _gpu(-(-rows // 128), cols // 128, 32, 16, **kw)
    return kernels.Mxfp8Tensor(values=values, scales=scales)


BAD_SCALES = [
    (lambda: _gpu(1, 2, 32, 16), "padded"),                                # of half the rows
    (lambda: _gpu(3, 2, 32, 16), "padded"),                                # of a larger batch
    (lambda: _gpu(2, 1, 32, 16), "padded"),                                # of half the columns
    (lambda: _gpu(0, 2, 32, 16), "padded"),
    (lambda: _gpu(2048), "padded"),
    (lambda: _gpu(2, 2, 32, 16, dtype=torch.int32), "dtype"),
    (lambda: _gpu(2, 2, 32, 32)[..., ::2], "contiguous"),
    (lambda: _gpu(2, 2, 32, 16, where=("cuda", 1)), "values' device"),
    (lambda: _gpu(2, 2, 32, 16, where=("cpu",)), "values' device"),
]


@pytest.mark.parametrize("rows", [200, 256])
@pytest.mark.parametrize("scales,match", BAD_SCALES)
def test_scales_that_do_not_belong_to_the_left_values(rows: int, scales, match: str) -> None:
    with pytest.raises(ValueError, match=match):
        kernels.mxfp8_gemm(_operand(rows, 256, scales()), _operand(128, 256))


@pytest.mark.parametrize("scales,match", BAD_SCALES)
def test_scales_that_do_not_belong_to_the_right_values(scales, match: str) -> None:
    with pytest.raises(ValueError, match=match):
        kernels.mxfp8_gemm(_operand(100, 256), _operand(256, 256, scales()))


def test_operands_on_two_devices() -> None:
    with pytest.raises(ValueError, match="one device"):
        kernels.mxfp8_gemm(_operand(128, 256), _operand(128, 256, where=("cuda", 1)))


def test_the_c_entry_refuses_addresses_that_its_copies_cannot_take() -> None:
    """Scale tiles travel in bulk copies, which fault off 16 bytes."""

    lib, p = _lib.library(), 4096
    for i in range(5):
        for off in (1, 2, 4, 8):
            args = [p + off * (j == i) for j in range(5)]
            assert lib.ce4b_mxfp8_gemm(*args, 128, 128, 128, None) == _lib.CE4B_ERR_INVALID_ARGUMENT
            assert "aligned" in _lib.last_error()
