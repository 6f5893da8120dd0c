"""GPU: one token or one expert cut out of tensors whose pitches are no multiple of 16 bytes gives what a contiguous
operand gives."""
import pytest
import torch

import open64_b200 as o

pytestmark = pytest.mark.gpu


def gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def bf16(shape, g):
    return torch.randn(shape, generator=g, device="cuda").to(torch.bfloat16)


def e4m3(shape, g):
    return (torch.randn(shape, generator=g, device="cuda") * 60).clamp(-448, 448).to(torch.float8_e4m3fn)


def plain(t):
    return t.detach().clone(memory_format=torch.contiguous_format)


@pytest.mark.parametrize("row", range(8))
def test_one_token(eng, row):
    g = gen(row)
    K, N = 1000, 72
    tokens, b = bf16((8, K + 3), g), bf16((2, N, K), g)
    off = torch.tensor([0, 1, 1], device="cuda", dtype=torch.int32)
    a = tokens[row:row + 1, :K]
    assert torch.equal(eng.gemm_grouped_bf16(a, off, b), eng.gemm_grouped_bf16(plain(a), off, b))
    dc = bf16((8, N + 5), g)[row:row + 1, :N]
    assert torch.equal(eng.gemm_grouped_bf16_wgrad(dc, a, off), eng.gemm_grouped_bf16_wgrad(plain(dc), plain(a), off))
    wide, w, sw = e4m3((8, K + 13), g), e4m3((N, K), g), torch.rand((1, 8), generator=g, device="cuda")
    a8, sa = wide[row:row + 1, 4:4 + K], torch.rand((1, 8), generator=g, device="cuda")
    assert torch.equal(eng.gemm_fp8_block(a8, sa, w, sw), eng.gemm_fp8_block(plain(a8), sa, w, sw))


@pytest.mark.parametrize("transB", [True, False], ids=["nk", "kn"])
@pytest.mark.parametrize("expert", range(4))
def test_one_expert(eng, expert, transB):
    g = gen(expert)
    rows, cols = 41, 44
    flat = bf16((4 * (rows * 51 + 1) + 64,), g)
    stack = flat[2:].as_strided((4, rows, 51), (rows * 51 + 1, 51, 1))
    b = stack[expert:expert + 1, :, :cols]
    a = bf16((9, cols if transB else rows), g)
    off = torch.tensor([0, 9], device="cuda", dtype=torch.int32)
    assert torch.equal(eng.gemm_grouped_bf16(a, off, b, transB=transB), eng.gemm_grouped_bf16(a, off, plain(b), transB=transB))


def test_weights_that_are_being_trained(eng):
    g = gen(1)
    a, b = bf16((20, 43), g), bf16((2, 30, 43), g).requires_grad_()
    off = torch.tensor([0, 7, 20], device="cuda", dtype=torch.int32)
    c = eng.gemm_grouped_bf16(a, off, b)
    assert not c.requires_grad and torch.equal(c, eng.gemm_grouped_bf16(a, off, b.detach()))
