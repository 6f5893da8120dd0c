"""GPU: the tail of the e4m3 SwiGLU products, silu(gate) * up and its way to e4m3, on products whose sums are exact.

Operands hold one or two non-zero terms a result, so gate and up are known numbers; with 64 for a gate exp(-gate)
vanishes beside 1 and silu(gate) is gate."""
import pytest
import torch

import open64_b200 as o

pytestmark = pytest.mark.gpu
FP8 = torch.float8_e4m3fn
ROWS = [5, 40, 300, 1200]  # few rows (with and without a cluster over K), CTA pairs


def call(eng, a, sa, w, sw, groups):
    if not groups:
        return eng.gemm_fp8_block_swiglu(a, sa, w, sw)
    T = a.shape[0]
    off = torch.tensor([T * i // groups for i in range(groups + 1)], device="cuda", dtype=torch.int32)
    return eng.gemm_grouped_fp8_block_swiglu(a, sa, off, w.expand(groups, *w.shape).contiguous(), sw.expand(groups, *sw.shape).contiguous())


@pytest.mark.parametrize("M", ROWS)
@pytest.mark.parametrize("groups", [0, 3])
@pytest.mark.parametrize("N,K", [(128, 128), (2048, 1024)])
def test_values_on_the_border_of_two_e4m3_numbers(eng, M, N, K, groups):
    """h / scale lies exactly between two e4m3 numbers, for odd factors whose reciprocal is none: q = e4m3(h / scale)
    is the even one."""
    up = torch.tensor([(8 + j) * 2.0 ** e + 2.0 ** (e - 1) for e in range(-2, 5) for j in range(8)] + [(8 + j) * 32.0 + 16 for j in range(6)], device="cuda")
    up = up.repeat(3)[:127]
    low = torch.where(up.log2().floor() > 7, up - 16, up - 2.0 ** (up.log2().floor() - 4))  # the e4m3 number below, and the rest
    assert torch.equal(low.to(FP8).float(), low) and torch.equal((up - low).to(FP8).float(), up - low)
    w = torch.zeros((2 * N, K), device="cuda")
    w[:N, 0] = 64.0
    for b in range(N // 128):
        w[N + 128 * b:N + 128 * b + 127, 0], w[N + 128 * b:N + 128 * b + 127, 1] = low, up - low
        w[N + 128 * b + 127, 0] = 448.0
    a = torch.zeros((M, K), device="cuda")
    a[:, :2] = 1.0
    t = 1.0 + 2.0 * (torch.arange(M, device="cuda") % 1500)  # t * t has at most 23 bits
    sa = t[:, None].expand(M, K // 128).contiguous()
    h, scales = call(eng, a.to(FP8), sa, w.to(FP8), torch.ones((2 * N // 128, K // 128), device="cuda"), groups)
    # h = 64 t t up is a number of fp32 where 31 t t < 2^24 (up has five bits, 448 = 7 * 64 three): only there is it known
    # to the last bit.  t <= 735 is the case in all rows up to 368, and in those that follow 1500 apart.
    known = 31 * t * t < 2 ** 24
    want = torch.cat([up, torch.tensor([448.0], device="cuda")]).double().to(FP8)
    assert torch.equal(scales[known], (64 * t * t)[known, None].expand(-1, N // 128))
    assert torch.equal(h[known].float(), want.float().repeat(N // 128).expand(int(known.sum()), N))


@pytest.mark.parametrize("M", ROWS + [20000])
@pytest.mark.parametrize("low,high", [(-20, 20), (-1, 1), (-60, -20)])
def test_silu(eng, M, low, high):
    """The scale of a block of equal values shows silu(gate) to all its bits: within 2^-20 of the value, and the
    roundings of the product with up and of the division by 448."""
    g = torch.Generator(device="cuda").manual_seed(M)
    x = low + (high - low) * torch.rand(M, generator=g, device="cuda")
    a = torch.zeros((M, 128), device="cuda")
    a[:, 0] = torch.sign(x)
    w = torch.zeros((256, 128), device="cuda")
    w[:, 0] = 1.0
    sa = x.abs()[:, None].contiguous()
    _, scales = call(eng, a.to(FP8), sa, w.to(FP8), torch.ones((2, 1), device="cuda"), 0)
    v = x.double()
    want = v * torch.sigmoid(v) * v / 448  # the second factor: up is the same number
    off = (scales[:, 0].double() / want.abs() - 1).abs()
    assert (off <= 2.0 ** -20 + 2 * 2.0 ** -24)[want.abs() >= 2.0 ** -126].all(), off.max().log2().item()


@pytest.mark.parametrize("M", [4, 300, 1200])
def test_silu_far_out(eng, M):
    """Gates of any size: as they are above, zero below, infinite and NaN where the formula is."""
    inf, nan = float("inf"), float("nan")
    gates = torch.tensor([1e30, -1e30, 3e38, -3e38, 200.0, -200.0, -89.0, 1e-30, -1e-30, inf, -inf, nan], device="cuda")
    gates = gates.repeat(-(-M // 12))[:M]
    a = torch.zeros((M, 128), device="cuda")
    a[:, 0] = torch.where(gates < 0, -1.0, 1.0)
    w = torch.zeros((256, 128), device="cuda")
    w[:, 0] = 1.0
    _, scales = call(eng, a.to(FP8), gates.abs()[:, None].contiguous(), w.to(FP8), torch.tensor([[1.0], [2.0 ** -40]], device="cuda"), 0)
    v = gates.double()
    h = v * torch.sigmoid(v) * (v * 2.0 ** -40)
    got = scales[:, 0].double()
    assert torch.equal(torch.isnan(got), torch.isnan(h))
    big = h.abs() > 3.5e38
    assert torch.isinf(got[big]).all()
    small = h.abs() / 448 < 2.0 ** -126  # a block of nothing: its scale is 1
    assert (got[small] == 1).all()
    rest = ~(big | small | torch.isnan(h))
    assert ((got / (h.abs() / 448) - 1).abs()[rest] <= 2.0 ** -20 + 2 * 2.0 ** -24).all()
