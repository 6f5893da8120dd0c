"""CPU: operands are handed to the library as TMA can read them - base, pitch and matrix stride multiples of 16 bytes -
by a copy in wide words where they do not lie that way.  The layout logic needs no device."""
import pytest
import torch

from open64_b200.engine import _ld, _tma


def values(shape, dtype):
    n = 1
    for s in shape:
        n *= s
    return (torch.arange(n) % 120).to(torch.uint8).view(shape).float().to(dtype)


def check(t):
    e = t.element_size()
    got = _tma(t)
    assert got.shape == t.shape and got.dtype == t.dtype
    assert torch.equal(got.float(), t.float())
    assert got.data_ptr() % 16 == 0 and (got.shape[-1] <= 1 or got.stride(-1) == 1) and _ld(got) * e % 16 == 0 and _ld(got) >= got.shape[-1]
    if got.dim() == 3 and got.shape[0] > 1:
        assert got.stride(0) * e % 16 == 0 and got.stride(0) >= (got.shape[1] - 1) * _ld(got) + got.shape[2]
    return got


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float8_e4m3fn], ids=["bf16", "e4m3"])
@pytest.mark.parametrize("pitch", [5003, 40, 41, 42, 44, 48])
@pytest.mark.parametrize("cols", [1, 2, 7, 16, 24, 33, 40])
def test_rows_of_a_wider_matrix(dtype, pitch, cols):
    big = values((10, pitch), dtype)
    for first in (0, 1, 3, 4, 8):
        if first + cols <= pitch:
            check(big[:, first:first + cols])
            for row in range(10):  # one token of it: its pitch is no layout of its own
                check(big[row:row + 1, first:first + cols])


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float8_e4m3fn], ids=["bf16", "e4m3"])
@pytest.mark.parametrize("rows,pitch", [(5, 24), (3, 41), (7, 20), (1, 13)])
def test_matrices_of_a_stack(dtype, rows, pitch):
    flat = values((6 * (rows * pitch + 3) + 8,), dtype)
    for base in (0, 1, 2, 8):
        stack = flat[base:].as_strided((6, rows, pitch), (rows * pitch + 3, pitch, 1))
        for cols in (8, 12, 13):
            check(stack[:, :, :cols])
            for one in range(6):  # one expert of it, and one row of each
                check(stack[one:one + 1, :, :cols])
            check(stack[:, :1, :cols])
            check(stack[2:3, rows - 1:, :cols])


def test_what_lies_well_is_not_copied():
    a = values((10, 48), torch.bfloat16)
    assert check(a).data_ptr() == a.data_ptr() and check(a[:, 8:40]).data_ptr() == a[:, 8:40].data_ptr()
    one = values((10, 5003), torch.bfloat16)[8:9, :5000]  # 16 bytes divide the base of this row
    assert one.data_ptr() % 16 == 0 and check(one).data_ptr() == one.data_ptr()


def test_columns_apart_broadcast_and_empty():
    a = values((40, 24), torch.bfloat16)
    check(a.t()), check(a.t()[:1]), check(a[:1].expand(5, 24)), check(a[None].expand(3, 40, 24)), check(a[:, ::2]), check(a[1:2, 1::2])
    assert _tma(a[:0]).shape == (0, 24) and _tma(a[:, :0]).shape == (40, 0)


def test_operands_that_are_being_trained():
    w = values((10, 43), torch.float32).to(torch.bfloat16).requires_grad_()
    assert not check(w).requires_grad and not check(w[3:4, :40]).requires_grad


def test_a_buffer_whose_own_base_is_odd():
    raw = bytearray(400)
    for shift in (0, 2, 4, 8):  # element 0 lies `shift` bytes behind a boundary, views of it on one
        t = torch.frombuffer(raw, dtype=torch.bfloat16, offset=shift, count=150)
        t.copy_(values((150,), torch.bfloat16))
        for first in range(9):
            check(t[first:first + 120].view(5, 24))
            check(t[first:first + 8].view(1, 8))
