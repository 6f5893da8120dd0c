"""GPU: few-row products that follow one another in the same buffers.  Each call's scales, offsets and operands were
written by the call just before, over values that a call just before that has read; nothing waits in between."""
import pytest
import torch

import open64_b200 as o

pytestmark = pytest.mark.gpu


def gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def e4m3(shape, g):
    return (torch.randn(shape, generator=g, device="cuda") * 60).clamp(-448, 448).to(torch.float8_e4m3fn)


@pytest.mark.parametrize("rows", [2, 24, 60])
def test_the_same_buffers_again_and_again(eng, rows):
    G, D, F, times = 3, 512, 384, 40
    g = gen(rows)
    T = rows * G
    w13, s13 = e4m3((G, 2 * F, D), g), torch.rand((G, 2 * F // 128, D // 128), generator=g, device="cuda") * 1e-4
    w2, s2 = e4m3((G, D, F), g), torch.rand((G, D // 128, F // 128), generator=g, device="cuda") * 1e-2
    xs = [torch.randn((T, D), generator=g, device="cuda").to(torch.bfloat16) for _ in range(times)]
    cuts = [torch.tensor([0, (i * 7) % T, T - (i * 3) % (T - (i * 7) % T), T], device="cuda", dtype=torch.int32) for i in range(times)]
    weight = torch.ones((D,), device="cuda")
    a, sa = torch.empty((T, D), device="cuda", dtype=torch.float8_e4m3fn), torch.empty((T, D // 128), device="cuda")
    h, sh = torch.empty((T, F), device="cuda", dtype=torch.float8_e4m3fn), torch.empty((T, F // 128), device="cuda")
    off = torch.empty(4, device="cuda", dtype=torch.int32)

    def step(i, out, wait):
        off.copy_(cuts[i])
        wait()
        eng.rms_norm(xs[i], weight, out_kind=o.OUT_E4M3, out=a, scales=sa)
        wait()
        eng.gemm_grouped_fp8_block_swiglu(a, sa, off, w13, s13, out=h, scales=sh)
        wait()
        eng.gemm_grouped_fp8_block(h, sh, off, w2, s2, out=out)
        wait()

    def run(wait):
        outs = [torch.zeros((T, D), device="cuda", dtype=torch.bfloat16) for _ in range(times)]
        torch.cuda.synchronize()
        for i in range(times):
            step(i, outs[i], wait)
        torch.cuda.synchronize()
        return outs

    want = run(torch.cuda.synchronize)
    assert all(torch.isfinite(c.float()).all() for c in want)
    for _ in range(5):
        assert all(torch.equal(c, w) for c, w in zip(run(lambda: None), want))
    assert eng.last_status() == (o.OK, 0)
