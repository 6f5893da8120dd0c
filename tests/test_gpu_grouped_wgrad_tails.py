"""GPU: weight gradients of many short groups.  Every group ends inside a K step, so that each tile's last block is
loaded, cleared behind the group's end in both CTAs of a pair and only then multiplied, several times within one turn
of the ring.  Values against 64-bit products, every repetition the same bits, and no wait may have run out.

Tolerances: each addition to an fp32 sum within 2^-23 of the sum of the terms' magnitudes (16 terms at a time), bf16
results half a step more."""
import pytest
import torch

import open64_b200 as o

pytestmark = pytest.mark.gpu


def bf16(shape, seed):
    return torch.randn(shape, generator=torch.Generator(device="cuda").manual_seed(seed), device="cuda").to(torch.bfloat16)


def offsets_of(sizes):
    return torch.tensor([0] + sizes, device="cuda").cumsum(0).to(torch.int32)


def check(eng, sizes, N, K, out_kind, times):
    T, off = sum(sizes), offsets_of(sizes)
    dc, a = bf16((T, N), N), bf16((T, K), K + 1)
    first = None
    for _ in range(times):
        db = eng.gemm_grouped_bf16_wgrad(dc, a, off, out_kind)
        assert eng.last_status() == (o.OK, 0)
        if first is None:
            first = db
        assert torch.equal(db, first)
    most = max(sizes)
    rows = torch.arange(most, device="cuda")
    ends = off.long()
    for at in range(0, len(sizes), 64):  # groups side by side, rows behind a group's end zero
        b, e = ends[at:at + 65][:-1, None], ends[at:at + 65][1:, None]
        there = b + rows < e
        pick = (b + rows).clamp(max=T - 1)
        d, x = dc.double()[pick] * there[..., None], a.double()[pick] * there[..., None]
        want, size = d.mT @ x, d.abs().mT @ x.abs()
        bound = (most / 16 + 8) * 2.0 ** -23 * size + (2.0 ** -8 * want.abs() if out_kind == o.OUT_BF16 else 0)
        assert ((first[at:at + 64].double() - want).abs() <= 2 * bound).all()


@pytest.mark.parametrize("rows", [1, 5, 65, 127, 129, 150, 193, 200, 257, 300])  # one to five K blocks of 64
@pytest.mark.parametrize("N,K", [(128, 128), (40, 72), (136, 128), (128, 264)])
def test_equal_groups(eng, rows, N, K):
    """N, K <= 128: the second CTA's operands lie outside the matrices, its loads only fill."""
    check(eng, [rows] * 450, N, K, o.OUT_BF16, 4)


@pytest.mark.parametrize("out_kind", [o.OUT_BF16, o.OUT_F32], ids=["bf16", "f32"])
@pytest.mark.parametrize("N,K", [(64, 128), (300, 200)])
def test_mixed_groups(eng, N, K, out_kind):
    """Cut and whole last blocks, groups without rows, one long group between short ones."""
    sizes = [(37 * i) % 330 if i % 7 else 0 for i in range(600)]
    sizes[300] = 2001
    sizes[301:310] = [16, 64, 128, 320, 1, 15, 17, 63, 65]
    check(eng, sizes, N, K, out_kind, 4)


def test_many_tails_a_pair(eng):
    """Thousands of groups of one cut block each: dozens of them follow one another in a pair."""
    check(eng, [1 + (i % 15) for i in range(4000)], 32, 64, o.OUT_F32, 3)
