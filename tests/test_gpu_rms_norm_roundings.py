"""GPU: what RMS norm rounds, on inputs where everything else is exact.

e4m3, bf16 w, no residual: s * w has 16 bits, a block's quotients are 448 u / m with u and m such numbers, so one is
either on the border of two e4m3 numbers or at least 2^-21 of itself away from it: every value is the one of the
definition, ties included.  1 / rms: sums of squares of small whole numbers are exact in fp32, so it is the
correctly rounded number."""
import pytest
import torch

import open64_b200 as o

pytestmark = pytest.mark.gpu
SHAPES = [(3, 256), (1, 4096), (200, 1000), (7, 32768), (4800, 2048), (2400, 4096), (601, 16384), (4800, 2051), (1300, 5003)]


def data(T, N):
    g = torch.Generator(device="cuda").manual_seed(T + N)
    return torch.randn((T, N), generator=g, device="cuda").to(torch.bfloat16), (1 + 0.2 * torch.randn(N, generator=g, device="cuda")).to(torch.bfloat16)


@pytest.mark.parametrize("T,N", SHAPES)
@pytest.mark.parametrize("block", [128, 0])
def test_every_quotient_is_the_nearest(eng, T, N, block):
    x, w = data(T, N)
    x[0, :min(N, 128)] = torch.arange(min(N, 128), device="cuda") + 1  # whole numbers: many ties
    w[:min(N, 128)] = 1
    y, scales, _, rstd = eng.rms_norm(x, w, out_kind=o.OUT_E4M3, scale_block=block)
    u = x.double() * w.double()
    wide = torch.nn.functional.pad(u, (0, -N % (block or N))).view(T, -1, block or N)
    m = wide.abs().amax(2, keepdim=True)
    want = (448 * wide / m).view(T, -1)[:, :N].to(torch.float8_e4m3fn)
    assert torch.equal(y.view(torch.uint8), want.view(torch.uint8))
    # a scale: 1 / rms to its own accuracy, and one rounding
    goal = m[:, :, 0] * rstd.double()[:, None] / 448
    assert ((scales.double().view(T, -1) / goal - 1).abs() <= 2.0 ** -24 * (1 + 2.0 ** -10)).all()


@pytest.mark.parametrize("T,N", SHAPES)
@pytest.mark.parametrize("out_kind", [o.OUT_BF16, o.OUT_E4M3], ids=["bf16", "e4m3"])
def test_rstd_is_rounded_once(eng, T, N, out_kind):
    g = torch.Generator(device="cuda").manual_seed(N)
    x = torch.randint(-7, 8, (T, N), generator=g, device="cuda").to(torch.bfloat16)
    eps = 2.0 ** -20
    rstd = eng.rms_norm(x, torch.ones(N, device="cuda"), eps=eps, out_kind=out_kind)[3]
    want = 1 / torch.sqrt(x.double().square().sum(1) / N + eps)
    # half a step, and 2^-40 for the 64-bit arithmetic of both sides
    assert ((rstd.double() / want - 1).abs() <= 2.0 ** -24 * (1 + 2.0 ** -16)).all()
