"""GPU: offsets that overlap would make more tiles than the grid is sized for (few rows and a long K: clusters divide the K
blocks of a tile, and each has one).  The call takes no longer than another, reports the offsets, writes nothing outside
the rows of the operands, and the next call is right."""
import time

import pytest
import torch

import open64_b200 as o

pytestmark = pytest.mark.gpu
BAD = [[0, 100, 0, 100], [0, 90, 5, 100], [0, 100, 0, 50], [0, 17, 1, 100]]


def gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def bf16(shape, g):
    return torch.randn(shape, generator=g, device="cuda").to(torch.bfloat16)


def e4m3(shape, g):
    return (torch.randn(shape, generator=g, device="cuda") * 60).clamp(-448, 448).to(torch.float8_e4m3fn)


@pytest.mark.parametrize("kind", ["bf16", "bf16_kn", "e4m3", "e4m3_kn", "swiglu"])
@pytest.mark.parametrize("K", [512, 4096])
def test_overlapping_offsets(eng, kind, K):
    T, G, N = 100, 3, 256
    g = gen(K)
    guard = torch.full((T + 20, N), 3.0, device="cuda", dtype=torch.bfloat16)
    out = guard[10:10 + T]
    cols = 2 * N if kind == "swiglu" else N
    shape = (K, cols) if kind.endswith("kn") else (cols, K)
    if kind.startswith("bf16"):
        a, b = bf16((T, K), g), bf16((G, *shape), g)
        call = lambda off: eng.gemm_grouped_bf16(a, off, b, transB=shape[1] == K, out=out)
    else:
        a, sa = e4m3((T, K), g), torch.rand((T, K // 128), generator=g, device="cuda") * 1e-3
        b, sb = e4m3((G, *shape), g), torch.rand((G, shape[0] // 128, shape[1] // 128), generator=g, device="cuda") * 1e-3
        if kind == "swiglu":
            call = lambda off: eng.gemm_grouped_fp8_block_swiglu(a, sa, off, b, sb, o.OUT_BF16, out=out)[0]
        else:
            call = lambda off: eng.gemm_grouped_fp8_block(a, sa, off, b, sb, transB=shape[1] == K, out=out)
    good = torch.tensor([0, 33, 33, 100], device="cuda", dtype=torch.int32)
    want = call(good).clone()
    assert eng.last_status() == (o.OK, 0) and torch.isfinite(want.float()).all()
    for bad in BAD:
        off = torch.tensor(bad, device="cuda", dtype=torch.int32)
        torch.cuda.synchronize()
        at = time.perf_counter()
        call(off)
        assert eng.last_status()[0] == o.ERR_CONFORM
        assert time.perf_counter() - at < 0.5  # no wait ran out: the budget of one is two seconds
        assert (guard[:10] == 3).all() and (guard[10 + T:] == 3).all()
        assert torch.equal(call(good), want) and eng.last_status() == (o.OK, 0)


def test_thousands_of_groups_that_all_overlap(eng):
    """Every second group claims all rows: the work stays that of one of them."""
    T, G, N, K = 4096, 2000, 256, 512
    g = gen(1)
    a, b, dc = bf16((T, K), g), bf16((1, N, K), g).expand(G, N, K).contiguous(), bf16((T, N), g)
    off = torch.tensor([0, T] * (G // 2) + [0], device="cuda", dtype=torch.int32)
    for call in (lambda: eng.gemm_grouped_bf16(a, off, b), lambda: eng.gemm_grouped_bf16_wgrad(dc, a, off)):
        start, end = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
        call()
        start.record()
        call()
        end.record()
        assert eng.last_status()[0] == o.ERR_CONFORM
        assert start.elapsed_time(end) < 20  # milliseconds; a thousand times all rows would be 1000 x 1 GFLOP and more
