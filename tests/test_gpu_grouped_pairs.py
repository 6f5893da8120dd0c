"""GPU: the grouped and block-scaled products at the sizes where they run on CTA pairs (256 x 256 tiles) - several tiles a
pair, more K blocks than the ring has stages, groups that are empty, ragged or shorter than a tile, every operand
layout and result - and at those of the few-row kernel's largest tile.  The first test says that the sizes do what they
are here for.  Tolerances: test_gpu_grouped.py."""
import pytest
import torch

import open64_b200 as o
from test_gpu_grouped import bf16, check_swiglu, close_bf16, e4m3, gen, grouped, offsets_of, scales, swiglu_reference, up, value

pytestmark = pytest.mark.gpu
FP8 = torch.float8_e4m3fn
NAN = float("nan")

RAGGED = [700, 0, 257, 1, 1030, 0, 0, 513, 255, 2, 640]
GROUPS = {"ragged": RAGGED, "long_between_empty": [0, 900, 0, 0, 1500, 256], "one": [2000], "remainder_of_one": [1025, 0, 300]}
SIZES = [(2056, 1000), (4104, 904)]  # columns; K: 16 and 15 blocks of 64 in bf16, 8 of 128 in e4m3, the last ones cut
MIDDLE = [150, 97, 129]              # e4m3: tiles of 128 rows, few-row kernel


def weights8(G, N, K, transB, g):
    shape = (N, K) if transB else (K, N)
    return e4m3((G, *shape), g), scales((G, up(shape[0]), up(shape[1])), g)


def kernels(f):
    from torch.profiler import ProfilerActivity, profile
    f()
    torch.cuda.synchronize()
    with profile(activities=[ProfilerActivity.CUDA, ProfilerActivity.CPU]) as p:
        f()
        torch.cuda.synchronize()
    seen = [e.key for e in p.key_averages()]
    if not any("kernel" in k for k in seen):
        pytest.skip("the profiler shows no kernels on this machine")
    return [k for k in seen if "grouped_" in k]


def test_these_sizes_run_where_they_should(eng):
    g = gen(1)
    for name, sizes in GROUPS.items():
        T, G, off = sum(sizes), len(sizes), offsets_of(sizes)
        for N, K in SIZES:
            a, a8, sa = bf16((T, K), g), e4m3((T, K), g), scales((T, up(K)), g)
            for transB in (True, False):
                b, (b8, sb) = bf16((G, N, K) if transB else (G, K, N), g), weights8(G, N, K, transB, g)
                for f in (lambda: eng.gemm_grouped_bf16(a, off, b, transB=transB), lambda: eng.gemm_grouped_fp8_block(a8, sa, off, b8, sb, transB=transB)):
                    ran = kernels(f)
                    assert len(ran) == 1 and "grouped_pair_kernel" in ran[0], (name, N, K, transB, ran)
            F = N // 256 * 128
            w, sw = weights8(G, 2 * F, K, True, g)
            ran = kernels(lambda: eng.gemm_grouped_fp8_block_swiglu(a8, sa, off, w, sw))
            assert len(ran) == 1 and "grouped_pair_kernel" in ran[0], (name, F, K, ran)
    T, off = sum(MIDDLE), offsets_of(MIDDLE)
    a8, sa, (b8, sb) = e4m3((T, 1000), g), scales((T, 8), g), weights8(3, 2056, 1000, True, g)
    ran = kernels(lambda: eng.gemm_grouped_fp8_block(a8, sa, off, b8, sb))
    assert len(ran) == 1 and "grouped_rows_kernel" in ran[0] and "128" in ran[0], ran


@pytest.mark.parametrize("name", GROUPS)
@pytest.mark.parametrize("N,K", SIZES)
@pytest.mark.parametrize("transB", [True, False], ids=["nk", "kn"])
def test_bf16(eng, name, N, K, transB):
    """Rows before, between and behind: left alone where they are nobody's; one that is NaN stays alone."""
    sizes, first = GROUPS[name], 6
    g = gen(N + K)
    n, G = sum(sizes), len(sizes)
    T, end = first + n + 50, first + n
    a, b = bf16((T, K), g), bf16((G, N, K) if transB else (G, K, N), g)
    a[:first], a[end:] = NAN, float("inf")
    off = offsets_of(sizes, first)
    c = torch.full((T, N), 3.0, device="cuda", dtype=torch.bfloat16)
    assert eng.gemm_grouped_bf16(a, off, b, transB=transB, out=c) is c
    want, size = grouped(a[first:end].double(), sizes, b.double().mT if transB else b.double())
    close_bf16(c[first:end], want, size, K)
    assert (c[:first] == 3).all() and (c[end:] == 3).all()
    bad = [first, end - 1, first + n // 2]
    a[bad, 5] = NAN
    d = eng.gemm_grouped_bf16(a, off, b, transB=transB, out=torch.full_like(c, 3.0))
    assert torch.isnan(d[bad].float()).all()
    rest = [i for i in range(T) if i not in bad]
    assert torch.equal(d[rest], c[rest])


@pytest.mark.parametrize("name", list(GROUPS) + ["middle"])
@pytest.mark.parametrize("N,K", SIZES)
@pytest.mark.parametrize("transB", [True, False], ids=["nk", "kn"])
def test_e4m3(eng, name, N, K, transB):
    sizes, first = GROUPS.get(name, MIDDLE), 6
    g = gen(N + K)
    n, G = sum(sizes), len(sizes)
    T, end = first + n + 50, first + n
    a, sa, (b, sb) = e4m3((T, K), g), scales((T, up(K)), g), weights8(G, N, K, transB, g)
    sa[:first], sa[end:] = NAN, NAN
    a.view(torch.uint8)[end:] = 0x7f
    off = offsets_of(sizes, first)
    c = torch.full((T, N), 3.0, device="cuda", dtype=torch.bfloat16)
    eng.gemm_grouped_fp8_block(a, sa, off, b, sb, transB=transB, out=c)
    B = value(b, sb, 128)
    want, size = grouped(value(a, sa, 1)[first:end], sizes, B.mT if transB else B)
    close_bf16(c[first:end], want, size, K)
    assert (c[:first] == 3).all() and (c[end:] == 3).all()
    bad = [first, end - 1, first + n // 2]
    sa[bad, 2] = NAN
    d = eng.gemm_grouped_fp8_block(a, sa, off, b, sb, transB=transB, out=torch.full_like(c, 3.0))
    assert torch.isnan(d[bad].float()).all()
    rest = [i for i in range(T) if i not in bad]
    assert torch.equal(d[rest], c[rest])


@pytest.mark.parametrize("name", GROUPS)
@pytest.mark.parametrize("F,K", [(1024, 1000), (2048, 904)])
@pytest.mark.parametrize("out_kind", [o.OUT_BF16, o.OUT_E4M3], ids=["bf16", "e4m3"])
def test_swiglu(eng, name, F, K, out_kind):
    sizes, first = GROUPS[name], 6
    g = gen(F + K)
    n, G = sum(sizes), len(sizes)
    T, end = first + n + 50, first + n
    a, sa, (w, sw) = e4m3((T, K), g), scales((T, up(K)), g) * 0.1, weights8(G, 2 * F, K, True, g)
    sw *= 0.2
    sa[:first], sa[end:] = NAN, NAN
    off = offsets_of(sizes, first)
    out = torch.zeros((T, F), device="cuda", dtype=FP8 if out_kind == o.OUT_E4M3 else torch.bfloat16)
    sh = torch.full((T, F // 128), -1.0, device="cuda") if out_kind == o.OUT_E4M3 else None
    h, s = eng.gemm_grouped_fp8_block_swiglu(a, sa, off, w, sw, out_kind, out=out, scales=sh)
    A, W, at = value(a, sa, 1), value(w, sw, 128), first
    for e, rows in enumerate(sizes):
        if rows:
            part = slice(at, at + rows)
            check_swiglu(h[part], None if s is None else s[part], swiglu_reference(A[part], W[e], F), K)
        at += rows
    assert (h[:first].float() == 0).all() and (h[end:].float() == 0).all()
    if s is not None:
        assert (s[:first] == -1).all() and (s[end:] == -1).all()


@pytest.mark.parametrize("M", [3000, 2561, 300])
@pytest.mark.parametrize("transB", [True, False], ids=["nk", "kn"])
def test_dense(eng, M, transB):
    N, K = 2056, 1000
    g = gen(M)
    a, sa, (b, sb) = e4m3((M, K), g), scales((M, up(K)), g), weights8(1, N, K, transB, g)
    c = eng.gemm_fp8_block(a, sa, b[0], sb[0], transB=transB)
    A, B = value(a, sa, 1), value(b[0], sb[0], 128)
    B = B.mT if transB else B
    close_bf16(c, A @ B, A.abs() @ B.abs(), K)
    assert torch.equal(eng.gemm_grouped_fp8_block(a, sa, offsets_of([M]), b, sb, transB=transB), c)


@pytest.mark.parametrize("out_kind", [o.OUT_BF16, o.OUT_E4M3], ids=["bf16", "e4m3"])
def test_dense_swiglu(eng, out_kind):
    M, F, K = 3000, 1152, 1000
    g = gen(F)
    a, sa, (w, sw) = e4m3((M, K), g), scales((M, up(K)), g) * 0.05, weights8(1, 2 * F, K, True, g)
    sw *= 0.1
    h, sh = eng.gemm_fp8_block_swiglu(a, sa, w[0], sw[0], out_kind)
    check_swiglu(h, sh, swiglu_reference(value(a, sa, 1), value(w[0], sw[0], 128), F), K)


@pytest.mark.parametrize("pad", [8, 5])
def test_results_in_wider_tensors(eng, pad):
    """Rows of a pitch that bulk stores take, and of one they do not, and of columns that end inside a store's box."""
    N, K = 2056, 1000
    g = gen(pad)
    T, G, off = sum(RAGGED), len(RAGGED), offsets_of(RAGGED)
    a, b = bf16((T, K), g), bf16((G, N, K), g)
    want = eng.gemm_grouped_bf16(a, off, b)
    c = torch.full((T, N + pad), 3.0, device="cuda", dtype=torch.bfloat16)
    eng.gemm_grouped_bf16(a, off, b, out=c[:, :N])
    assert torch.equal(c[:, :N], want) and (c[:, N:] == 3).all()
    d = torch.full((T * (N + pad) + 1,), 3.0, device="cuda", dtype=torch.bfloat16)[1:].view(T, N + pad)  # a base off 16 bytes
    eng.gemm_grouped_bf16(a, off, b, out=d[:, :N])
    assert torch.equal(d[:, :N], want) and (d[:, N:] == 3).all()
    a8, sa, (w, sw) = e4m3((T, K), g), scales((T, up(K)), g), weights8(G, 2048, K, True, g)
    want, want_s = eng.gemm_grouped_fp8_block_swiglu(a8, sa, off, w, sw)
    h, s = torch.zeros((T, 1024 + pad), device="cuda", dtype=FP8), torch.full((T, 8 + pad), -1.0, device="cuda")
    eng.gemm_grouped_fp8_block_swiglu(a8, sa, off, w, sw, out=h[:, :1024], scales=s[:, :8])
    assert torch.equal(h[:, :1024].float(), want.float()) and torch.equal(s[:, :8], want_s)
    assert (h[:, 1024:].float() == 0).all() and (s[:, 8:] == -1).all()
    pads = torch.zeros((T, 8 + pad), device="cuda")  # scales of A whose rows are not 16 bytes apart
    pads[:, 1:9 if pad > 1 else 8] = sa
    h2, s2 = eng.gemm_grouped_fp8_block_swiglu(a8, pads[:, 1:9], off, w, sw)
    assert torch.equal(h2.float(), want.float()) and torch.equal(s2, want_s)


def test_offsets_past_32_bits(eng):
    if torch.cuda.mem_get_info()[0] < 30 << 30:
        pytest.skip("needs 30 GB of free memory")
    T, ld, N, K = 1500, 1 << 22, 1032, 1000  # row 1024 of A and of C starts 8 GiB into its tensor
    g = gen(12)
    vals, b = bf16((T, K), g), bf16((2, N, K), g)
    off = offsets_of([700, 800])
    want = eng.gemm_grouped_bf16(vals, off, b)
    a = torch.empty(((T - 1) * ld + K,), device="cuda", dtype=torch.bfloat16).as_strided((T, K), (ld, 1))
    a.copy_(vals)
    c = torch.empty(((T - 1) * ld + N,), device="cuda", dtype=torch.bfloat16).as_strided((T, N), (ld, 1))
    assert torch.equal(eng.gemm_grouped_bf16(a, off, b, out=c), want)


def test_bad_offsets(eng):
    N, K, T = 2056, 1000, 2600
    g = gen(6)
    a, b = bf16((T, K), g), bf16((3, N, K), g)
    good = offsets_of([700, 1200, 700])
    want = eng.gemm_grouped_bf16(a, good, b)
    guard = torch.full((T + 20, N), 3.0, device="cuda", dtype=torch.bfloat16)
    for bad in ([0, 1500, 20, 2600], [0, 10, 20, 2000000000], [-5, 10, 20, 30], [2500, 1800, 700, 60], [0, 2600, 0, 2600]):
        eng.gemm_grouped_bf16(a, torch.tensor(bad, device="cuda", dtype=torch.int32), b, out=guard[10:10 + T])
        assert eng.last_status()[0] == o.ERR_CONFORM
        assert (guard[:10] == 3).all() and (guard[10 + T:] == 3).all()
        assert torch.equal(eng.gemm_grouped_bf16(a, good, b), want) and eng.last_status() == (o.OK, 0)


def test_streams_graphs_and_calls_without_a_wait(eng):
    D, F, G = 1024, 1152, 3
    g = gen(2)
    sizes = [700, 3, 800]
    T, off = sum(sizes), offsets_of(sizes)
    x, w = bf16((T, D), g), torch.rand((D,), generator=g, device="cuda") + 0.5
    (w13, s13), (w2, s2) = weights8(G, 2 * F, D, True, g), weights8(G, D, F, True, g)
    s13 *= 0.05
    s2 *= 0.05

    def layer(wait=lambda: None):
        y = x
        for _ in range(3):
            y, _ = eng.mlp_swiglu_fp8(y, w, w13, s13, w2, s2, residual=y, offsets=off)
            wait()
        return y

    want = layer(torch.cuda.synchronize)
    assert torch.isfinite(want.float()).all()
    side, got = [torch.cuda.Stream(), torch.cuda.Stream()], []
    for s in side:
        s.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(s):
            got.append(layer())
    got += [layer() for _ in range(5)]
    torch.cuda.synchronize()
    assert all(torch.equal(y, want) for y in got)
    graphs = []
    for _ in range(2):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            y = layer()
        graphs.append((graph, y))
    x.copy_(bf16((T, D), gen(77)))
    off.copy_(offsets_of([1, 1402, 100]))  # the groups move between replays
    for graph, _ in graphs:
        graph.replay()
    torch.cuda.synchronize()
    want = layer()
    assert all(torch.equal(y, want) for _, y in graphs)
    assert eng.last_status() == (o.OK, 0)


@pytest.mark.parametrize("out_kind", [o.OUT_BF16, o.OUT_F32], ids=["bf16", "f32"])
@pytest.mark.parametrize("N,K", [(2056, 1000), (1024, 2048)])
def test_weight_gradient(eng, N, K, out_kind):
    """Several tiles a pair and groups of many blocks (groups of few: test_gpu_grouped_wgrad_tails.py)."""
    sizes = RAGGED
    g = gen(N)
    T = sum(sizes)
    dc, a = bf16((T, N), g), bf16((T, K), g)
    db = eng.gemm_grouped_bf16_wgrad(dc, a, offsets_of(sizes), out_kind)
    assert eng.last_status() == (o.OK, 0)
    at = 0
    for e, n in enumerate(sizes):
        d, x = dc[at:at + n].double(), a[at:at + n].double()
        at += n
        want, size = d.mT @ x, d.abs().mT @ x.abs()
        if out_kind == o.OUT_BF16:
            close_bf16(db[e], want, size, n)
        else:
            assert ((db[e].double() - want).abs() <= (n / 16 + 8) * 2.0 ** -23 * size).all()


@pytest.mark.parametrize("transB", [True, False], ids=["nk", "kn"])
@pytest.mark.parametrize("sizes", [MIDDLE, [128, 128, 120], [376, 0, 0], [1, 128, 247]], ids=str)
def test_tiles_of_128_rows(eng, sizes, transB):
    N, K = 2056, 1000
    g = gen(sum(sizes[:1]))
    T, off = sum(sizes), offsets_of(sizes)
    a, sa, (b, sb) = e4m3((T, K), g), scales((T, up(K)), g), weights8(3, N, K, transB, g)
    ran = kernels(lambda: eng.gemm_grouped_fp8_block(a, sa, off, b, sb, transB=transB))
    assert len(ran) == 1 and "grouped_rows_kernel" in ran[0] and "128" in ran[0], ran
    c = eng.gemm_grouped_fp8_block(a, sa, off, b, sb, transB=transB)
    B = value(b, sb, 128)
    want, size = grouped(value(a, sa, 1), sizes, B.mT if transB else B)
    close_bf16(c, want, size, K)
