"""GPU: the e4m3 product with a scale for each block of 128, and the products grouped by expert, against
64-bit products of the same operands.

Tolerances.  With S = |A| |B| (the sum of the magnitudes of a result's terms): the tensor cores add 32 bytes of
a row at a time (16 bf16 or 32 e4m3 terms, whose products are exact) to an fp32 accumulator, each addition
within 2^-23 of S (a truncation counts as a whole unit), and block scales add three roundings a block:
A(K) = (K / 16 + 8) * 2^-23 * S covers both.  A bf16 result adds 2^-8 of its value.  The SwiGLU tail: the
slope of silu(g) * u is at most 1.1 |u| in g and |g| in u, exp and the division stay within 2^-19 relative."""
import pytest
import torch

import open64_b200 as o

pytestmark = pytest.mark.gpu
BF16, E4M3 = 2.0 ** -8, 2.0 ** -4
FP8 = torch.float8_e4m3fn


def acc(K):
    return (K / 16 + 8) * 2.0 ** -23


def gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def bf16(shape, g, scale=1.0):
    return (torch.randn(shape, generator=g, device="cuda") * scale).to(torch.bfloat16)


def e4m3(shape, g):
    return (torch.randn(shape, generator=g, device="cuda") * 60).clamp(-448, 448).to(FP8)


def scales(shape, g):
    return torch.rand(shape, generator=g, device="cuda") * 0.03 + 1e-3


def up(n, m=128):
    return -(-n // m)


def value(q, s, rows):
    """The numbers an e4m3 matrix with scales of rows x 128 blocks stands for, in 64 bits."""
    return q.double() * s.double().repeat_interleave(rows, -2)[..., :q.shape[-2], :].repeat_interleave(128, -1)[..., :q.shape[-1]]


def offsets_of(sizes, first=0):
    return torch.tensor([first] + sizes, device="cuda").cumsum(0).to(torch.int32)


def close_bf16(got, want, size, K):
    assert got.dtype == torch.bfloat16
    off = (got.double() - want).abs()
    bound = BF16 * want.abs() + 2 * acc(K) * size
    assert (off <= bound).all(), (off / bound.clamp_min(1e-300)).max().item()


def refused(code, f):
    with pytest.raises(o.O64Error) as e:
        f()
    assert e.value.status == code


# ---- e4m3 with block scales ----------------------------------------------------------------------
FP8_SHAPES = [(1, 1, 1), (1, 128, 128), (1, 8192, 1024), (2, 16, 272), (7, 136, 100), (16, 1000, 4096), (33, 264, 129), (64, 4104, 512), (128, 256, 128),
              (129, 257, 255), (200, 2056, 640), (256, 512, 2048), (300, 72, 3000), (515, 640, 1040), (1000, 1000, 1000), (1024, 2048, 384)]


@pytest.mark.parametrize("M,N,K", FP8_SHAPES)
@pytest.mark.parametrize("transB", [True, False], ids=["nk", "kn"])
def test_fp8_block(eng, M, N, K, transB):
    g = gen(M + N + K)
    a, sa = e4m3((M, K), g), scales((M, up(K)), g)
    shape = (N, K) if transB else (K, N)
    b, sb = e4m3(shape, g), scales((up(shape[0]), up(shape[1])), g)
    c = eng.gemm_fp8_block(a, sa, b, sb, transB=transB)
    A, B = value(a, sa, 1), value(b, sb, 128)
    B = B.mT if transB else B
    close_bf16(c, A @ B, A.abs() @ B.abs(), K)


def test_fp8_block_scales_enter_at_their_block(eng):
    """One K block, one row or one 128-column block at a time has a scale of its own: products of ones are exact."""
    M, N, K = 150, 300, 400
    for transB in (True, False):
        a, b = torch.ones((M, K), device="cuda").to(FP8), torch.ones((N, K) if transB else (K, N), device="cuda").to(FP8)
        sa, sb = torch.zeros((M, 4), device="cuda"), torch.ones((3, 4) if transB else (4, 3), device="cuda")
        sa[140, 3] = 2.0  # 16 terms
        sa[3, 1] = 1.0    # 128 terms
        (sb if transB else sb.t())[2, 3] = 4.0
        want = torch.zeros((M, N), device="cuda")
        want[140] = 32.0
        want[140, 256:] = 128.0
        want[3] = 128.0
        assert torch.equal(eng.gemm_fp8_block(a, sa, b, sb, transB=transB).float(), want)


def swiglu_reference(A, W, N):
    gate, upv = A @ W[:N].mT, A @ W[N:].mT
    sg, su = A.abs() @ W[:N].abs().mT, A.abs() @ W[N:].abs().mT
    h = gate * torch.sigmoid(gate) * upv
    return h, sg, su, gate, upv


def check_swiglu(h, sh, ref, K):
    want, sg, su, gate, upv = ref
    err = acc(K) * (1.1 * upv.abs() * sg + gate.abs() * su + acc(K) * sg * su) + 2.0 ** -19 * want.abs()
    if sh is None:
        assert ((h.double() - want).abs() <= BF16 * (want.abs() + err) + err).all()
        return
    T, N = want.shape
    peak = want.abs().view(T, -1, 128).amax(2)
    worst = err.view(T, -1, 128).amax(2)
    goal = torch.where(peak / 448 < 2.0 ** -126, torch.ones_like(peak), peak / 448)
    assert ((sh.double() - goal).abs() <= worst / 448 + 2.0 ** -22 * goal).all()
    at = sh.double().repeat_interleave(128, 1)
    off = (h.double() * at - want).abs()
    assert (off <= E4M3 * (1 + 2.0 ** -16) * (want.abs() + err) + 2.0 ** -10 * at + err + 448 * at * 2.0 ** -22).all()


@pytest.mark.parametrize("M,N,K", [(1, 128, 128), (3, 256, 400), (16, 1024, 2048), (40, 384, 96), (130, 128, 1000), (300, 640, 512), (520, 2048, 640)])
@pytest.mark.parametrize("out_kind", [o.OUT_BF16, o.OUT_E4M3], ids=["bf16", "e4m3"])
def test_fp8_block_swiglu(eng, M, N, K, out_kind):
    g = gen(M * N + K)
    a, sa = e4m3((M, K), g), scales((M, up(K)), g) * 0.05
    w, sw = e4m3((2 * N, K), g), scales((2 * N // 128, up(K)), g) * 0.1
    h, sh = eng.gemm_fp8_block_swiglu(a, sa, w, sw, out_kind)
    check_swiglu(h, sh, swiglu_reference(value(a, sa, 1), value(w, sw, 128), N), K)


def test_nan_stays_in_its_row_and_block(eng):
    M, N, K = 40, 256, 300
    g = gen(8)
    a, sa, w, sw = e4m3((M, K), g), scales((M, 3), g), e4m3((2 * N, K), g), scales((4, 3), g)
    clean, clean_s = eng.gemm_fp8_block_swiglu(a, sa, w, sw)
    c = eng.gemm_fp8_block(a, sa, w, sw)
    sa2 = sa.clone()
    sa2[5, 2] = float("nan")
    h, s = eng.gemm_fp8_block_swiglu(a, sa2, w, sw)
    rows = [i for i in range(M) if i != 5]
    assert torch.isnan(s[5]).all() and torch.isnan(h[5].float()).all()
    assert torch.equal(h[rows].view(torch.uint8), clean[rows].view(torch.uint8)) and torch.equal(s[rows], clean_s[rows])
    d = eng.gemm_fp8_block(a, sa2, w, sw)
    assert torch.isnan(d[5].float()).all() and torch.equal(d[rows], c[rows])
    w8 = w.view(torch.uint8).clone()
    w8[2 * N - 1, 7] = 0x7f  # NaN in the last up row: only the last block of 128 columns sees it
    h, s = eng.gemm_fp8_block_swiglu(a, sa, w8.view(FP8), sw)
    assert torch.isnan(s[:, 1]).all() and torch.equal(s[:, 0], clean_s[:, 0])
    assert torch.equal(h[:, :128].view(torch.uint8), clean[:, :128].view(torch.uint8))


# ---- groups --------------------------------------------------------------------------------------
SIZES = {"one": [5], "even": [64, 64, 64, 64], "ragged": [1, 0, 300, 17, 0, 0, 256, 129, 2], "tail_empty": [40, 0, 0], "first_empty": [0, 0, 33],
         "single_rows": [1] * 20 + [0] * 5, "none": [0, 0, 0], "long": [700, 3, 257]}


def grouped(A, sizes, B):
    out, size, first = [], [], 0
    for n, b in zip(sizes, B):
        out.append(A[first:first + n] @ b)
        size.append(A[first:first + n].abs() @ b.abs())
        first += n
    return torch.cat(out), torch.cat(size)


@pytest.mark.parametrize("name", SIZES)
@pytest.mark.parametrize("N,K", [(256, 512), (136, 72), (1000, 264), (8, 1000)])
@pytest.mark.parametrize("transB", [True, False], ids=["nk", "kn"])
def test_grouped_bf16(eng, name, N, K, transB):
    sizes = SIZES[name]
    g = gen(N + K)
    T, G = sum(sizes), len(sizes)
    a, b = bf16((T, K), g), bf16((G, N, K) if transB else (G, K, N), g)
    c = eng.gemm_grouped_bf16(a, offsets_of(sizes), b, transB=transB)
    want, size = grouped(a.double(), sizes, b.double().mT if transB else b.double())
    close_bf16(c, want, size, K)


@pytest.mark.parametrize("name", SIZES)
@pytest.mark.parametrize("N,K", [(256, 512), (136, 72), (264, 1000)])
@pytest.mark.parametrize("out_kind", [o.OUT_BF16, o.OUT_F32], ids=["bf16", "f32"])
def test_grouped_wgrad(eng, name, N, K, out_kind):
    sizes = SIZES[name]
    g = gen(N * 3 + K)
    T = sum(sizes)
    dc, a = bf16((T, N), g), bf16((T, K), g)
    db = eng.gemm_grouped_bf16_wgrad(dc, a, offsets_of(sizes), out_kind)
    first = 0
    for e, n in enumerate(sizes):
        d, x = dc[first:first + n].double(), a[first:first + n].double()
        first += n
        want, size = d.mT @ x, d.abs().mT @ x.abs()
        if out_kind == o.OUT_BF16:
            close_bf16(db[e], want, size, n)
        else:
            assert db.dtype == torch.float32 and ((db[e].double() - want).abs() <= acc(n) * size).all()


@pytest.mark.parametrize("name", SIZES)
@pytest.mark.parametrize("N,K", [(256, 512), (136, 100), (1000, 272)])
@pytest.mark.parametrize("transB", [True, False], ids=["nk", "kn"])
def test_grouped_fp8_block(eng, name, N, K, transB):
    sizes = SIZES[name]
    g = gen(N * 5 + K)
    T, G = sum(sizes), len(sizes)
    shape = (N, K) if transB else (K, N)
    a, sa, b, sb = e4m3((T, K), g), scales((T, up(K)), g), e4m3((G, *shape), g), scales((G, up(shape[0]), up(shape[1])), g)
    c = eng.gemm_grouped_fp8_block(a, sa, offsets_of(sizes), b, sb, transB=transB)
    B = value(b, sb, 128)
    want, size = grouped(value(a, sa, 1), sizes, B.mT if transB else B)
    close_bf16(c, want, size, K)


@pytest.mark.parametrize("name", SIZES)
@pytest.mark.parametrize("out_kind", [o.OUT_BF16, o.OUT_E4M3], ids=["bf16", "e4m3"])
def test_grouped_fp8_block_swiglu(eng, name, out_kind):
    sizes, N, K = SIZES[name], 384, 528
    g = gen(len(name))
    T, G = sum(sizes), len(sizes)
    a, sa = e4m3((T, K), g), scales((T, up(K)), g) * 0.1
    w, sw = e4m3((G, 2 * N, K), g), scales((G, 2 * N // 128, up(K)), g) * 0.2
    h, sh = eng.gemm_grouped_fp8_block_swiglu(a, sa, offsets_of(sizes), w, sw, out_kind)
    A, W, first = value(a, sa, 1), value(w, sw, 128), 0
    for e, n in enumerate(sizes):
        rows = slice(first, first + n)
        first += n
        if n:
            check_swiglu(h[rows], None if sh is None else sh[rows], swiglu_reference(A[rows], W[e], N), K)


def test_many_groups(eng):
    G, N, K = 300, 64, 128
    g = gen(4)
    sizes = [(i * 7) % 5 for i in range(G)]
    T = sum(sizes)
    a, b = bf16((T, K), g), bf16((G, N, K), g)
    want, size = grouped(a.double(), sizes, b.double().mT)
    close_bf16(eng.gemm_grouped_bf16(a, offsets_of(sizes), b), want, size, K)
    dc = bf16((T, N), g)
    db = eng.gemm_grouped_bf16_wgrad(dc, a, offsets_of(sizes))
    first = 0
    for e, n in enumerate(sizes):
        d, x = dc[first:first + n].double(), a[first:first + n].double()
        first += n
        close_bf16(db[e], d.mT @ x, d.abs().mT @ x.abs(), n)


@pytest.mark.parametrize("rows", [3, 100])
def test_rows_outside_the_groups_are_left_alone_and_never_read_into_a_result(eng, rows):
    sizes, first, N, K = [rows, 0, 2 * rows + 1], 6, 256, 320
    g = gen(1)
    T = first + sum(sizes) + 50
    end = T - 50
    off = offsets_of(sizes, first)
    nan = float("nan")
    a, b = bf16((T, K), g), bf16((3, N, K), g)
    a[:first], a[end:] = nan, nan
    c = torch.full((T, N), 3.0, device="cuda", dtype=torch.bfloat16)
    assert eng.gemm_grouped_bf16(a, off, b, out=c) is c
    want, size = grouped(a[first:end].double(), sizes, b.double().mT)
    close_bf16(c[first:end], want, size, K)
    assert (c[:first] == 3).all() and (c[end:] == 3).all()
    # the weight gradient: rows behind a group are its neighbours' or NaN
    dc = bf16((T, N), g)
    dc[:first], dc[end:] = nan, float("inf")
    db = eng.gemm_grouped_bf16_wgrad(dc, a, off)
    at = first
    for e, n in enumerate(sizes):
        d, x = dc[at:at + n].double(), a[at:at + n].double()
        at += n
        close_bf16(db[e], d.mT @ x, d.abs().mT @ x.abs(), n)
    a8, sa = e4m3((T, K), g), scales((T, up(K)), g)
    w, sw = e4m3((3, 2 * N, K), g), scales((3, 4, up(K)), g)
    sa[:first], sa[end:] = nan, nan
    a8.view(torch.uint8)[end:] = 0x7f
    h = torch.zeros((T, N), device="cuda", dtype=FP8)
    sh = torch.full((T, 2), -1.0, device="cuda")
    eng.gemm_grouped_fp8_block_swiglu(a8, sa, off, w, sw, out=h, scales=sh)
    assert (sh[:first] == -1).all() and (sh[end:] == -1).all() and (h[:first].float() == 0).all() and (h[end:].float() == 0).all()
    assert torch.isfinite(sh[first:end]).all() and torch.isfinite(h[first:end].float()).all()
    c.fill_(3.0)
    eng.gemm_grouped_fp8_block(a8, sa, off, w[:, :N].contiguous(), sw[:, :2].contiguous(), out=c)
    assert (c[:first] == 3).all() and (c[end:] == 3).all() and torch.isfinite(c[first:end].float()).all()


def test_nothing_to_add(eng):
    off = offsets_of([2, 0, 3], 1)
    c = torch.full((8, 64), 3.0, device="cuda", dtype=torch.bfloat16)
    eng.gemm_grouped_bf16(torch.empty((8, 0), device="cuda", dtype=torch.bfloat16), off,
                          torch.empty((3, 64, 0), device="cuda", dtype=torch.bfloat16), out=c)
    assert (c[1:6] == 0).all() and (c[0] == 3).all() and (c[6:] == 3).all()
    h, s = eng.gemm_fp8_block_swiglu(torch.empty((4, 0), device="cuda", dtype=FP8), torch.empty((4, 0), device="cuda"),
                                     torch.empty((256, 0), device="cuda", dtype=FP8), torch.empty((2, 0), device="cuda"))
    assert (h.float() == 0).all() and (s == 1).all()
    none = torch.empty((0, 64), device="cuda", dtype=torch.bfloat16)
    db = eng.gemm_grouped_bf16_wgrad(none, none, torch.zeros(4, device="cuda", dtype=torch.int32), o.OUT_F32)
    assert db.shape == (3, 64, 64) and (db == 0).all()
    assert eng.gemm_grouped_bf16(none, torch.zeros(4, device="cuda", dtype=torch.int32), torch.empty((3, 8, 64), device="cuda", dtype=torch.bfloat16)).shape == (0, 8)


def test_strides_and_bases(eng):
    """Slices, transposed views, bases off 16 bytes and broadcast weights give what contiguous operands give."""
    sizes, N, K = [33, 100, 7], 200, 136
    g = gen(9)
    T, off = sum(sizes), offsets_of(sizes)
    a, b = bf16((T, K), g), bf16((3, N, K), g)
    want = eng.gemm_grouped_bf16(a, off, b)
    wide = torch.zeros((T, K + 24), device="cuda", dtype=torch.bfloat16)
    for at in (8, 3):
        wide[:, at:at + K] = a
        assert torch.equal(eng.gemm_grouped_bf16(wide[:, at:at + K], off, b), want)
    assert torch.equal(eng.gemm_grouped_bf16(a.t().contiguous().t(), off, b), want)
    big = torch.zeros((3, N + 5, K + 8), device="cuda", dtype=torch.bfloat16)
    big[:, 2:2 + N, 8:] = b
    assert torch.equal(eng.gemm_grouped_bf16(a, off, big[:, 2:2 + N, 8:]), want)
    assert torch.equal(eng.gemm_grouped_bf16(a, off, b.mT.contiguous(), transB=False), want)
    shared = b[:1].expand(3, N, K)
    assert torch.equal(eng.gemm_grouped_bf16(a, off, shared), eng.gemm_grouped_bf16(a, off, shared.contiguous()))
    for pad in (8, 5):
        c = torch.full((T, N + pad), 3.0, device="cuda", dtype=torch.bfloat16)
        eng.gemm_grouped_bf16(a, off, b, out=c[:, :N])
        assert torch.equal(c[:, :N], want) and (c[:, N:] == 3).all()
    db = eng.gemm_grouped_bf16_wgrad(bf16((T, N), gen(3)), a, off)
    for pad in (8, 5):
        d = torch.full((3, N + 1, K + pad), 3.0, device="cuda", dtype=torch.bfloat16)
        eng.gemm_grouped_bf16_wgrad(bf16((T, N), gen(3)), a, off, out=d[:, :N, :K])
        assert torch.equal(d[:, :N, :K], db) and (d[:, N:] == 3).all() and (d[:, :, K:] == 3).all()
    a8, sa, w, sw = e4m3((T, K), g), scales((T, 2), g), e4m3((3, N, K), g), scales((3, 2, 2), g)
    want = eng.gemm_grouped_fp8_block(a8, sa, off, w, sw)
    pads = torch.zeros((T, 9), device="cuda")
    pads[:, 3:5] = sa
    assert torch.equal(eng.gemm_grouped_fp8_block(a8, pads[:, 3:5], off, w, sw), want)
    assert torch.equal(eng.gemm_grouped_fp8_block(a8, sa.t().contiguous().t(), off, w, sw.mT.contiguous().mT), want)
    assert torch.equal(eng.gemm_fp8_block(a8[:1, :7], sa[:1, :1], w[0, :, :7], sw[0, :, :1]),
                       eng.gemm_fp8_block(a8[:1, :7].contiguous(), sa[:1, :1].contiguous(), w[0, :, :7].contiguous(), sw[0, :, :1].contiguous()))


def test_offsets_past_32_bits(eng):
    if torch.cuda.mem_get_info()[0] < 24 << 30:
        pytest.skip("needs 24 GB of free memory")
    ld, N, K = 1 << 30, 256, 256  # row 3 of A and of C starts 6 GiB into its tensor
    g = gen(12)
    vals, b = bf16((4, K), g), bf16((2, N, K), g)
    a = torch.empty((3 * ld + K,), device="cuda", dtype=torch.bfloat16).as_strided((4, K), (ld, 1))
    a.copy_(vals)
    c = torch.empty((3 * ld + N,), device="cuda", dtype=torch.bfloat16).as_strided((4, N), (ld, 1))
    off = offsets_of([1, 3])
    assert torch.equal(eng.gemm_grouped_bf16(a, off, b, out=c), eng.gemm_grouped_bf16(vals, off, b))


def test_bad_offsets_are_reported_and_followed_nowhere(eng):
    N, K, T = 64, 128, 100
    g = gen(6)
    a, b = bf16((T, K), g), bf16((3, N, K), g)
    c = torch.full((T, N), 3.0, device="cuda", dtype=torch.bfloat16)
    for bad in ([0, 50, 20, 100], [0, 10, 20, 2000000000], [-5, 10, 20, 30], [90, 80, 70, 60]):
        eng.gemm_grouped_bf16(a, torch.tensor(bad, device="cuda", dtype=torch.int32), b, out=c)
        assert eng.last_status()[0] == o.ERR_CONFORM
        assert eng.last_status() == (o.OK, 0)
        eng.gemm_grouped_bf16_wgrad(c, a, torch.tensor(bad, device="cuda", dtype=torch.int32))
        assert eng.last_status()[0] == o.ERR_CONFORM
    assert eng.last_status() == (o.OK, 0)


def test_streams_and_graphs(eng):
    sizes, N, K = [40, 3, 90], 256, 384
    g = gen(2)
    T, off = sum(sizes), offsets_of(sizes)
    a8, sa, w, sw = e4m3((T, K), g), scales((T, 3), g) * 0.1, e4m3((3, 2 * N, K), g), scales((3, 4, 3), g)
    w2, sw2 = e4m3((3, K, N), g), scales((3, 3, 2), g)

    def chain(x, s):
        h, sh = eng.gemm_grouped_fp8_block_swiglu(x, s, off, w, sw)
        return eng.gemm_grouped_fp8_block(h, sh, off, w2, sw2)

    want = chain(a8, sa)
    side = [torch.cuda.Stream(), torch.cuda.Stream()]
    got = []
    for s in side:  # two calls at once
        s.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(s):
            got.append(chain(a8, sa))
    torch.cuda.synchronize()
    assert all(torch.equal(c, want) for c in got)
    graphs = []
    for _ in range(2):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            c = chain(a8, sa)
        graphs.append((graph, c))
    a8.copy_(e4m3((T, K), gen(77)))
    off.copy_(offsets_of([1, 100, 32]))  # the groups move between replays
    for graph, _ in graphs:
        graph.replay()
    torch.cuda.synchronize()
    want = chain(a8, sa)
    assert all(torch.equal(c, want) for _, c in graphs)


@pytest.mark.parametrize("rows", [1, 5, 40, 90, 300])
def test_calls_that_follow_one_another_without_a_wait(eng, rows):
    """Each call reads what the one before has just written (few-row kernels set up while it still runs): the same
    bits as with a wait between, every time."""
    D, F, G = 384, 256, 3
    g = gen(rows)
    T = rows * G
    off = offsets_of([rows] * G)
    x, w = bf16((T, D), g), torch.rand((D,), generator=g, device="cuda") + 0.5
    w13, s13, w2, s2 = e4m3((G, 2 * F, D), g), scales((G, 4, 3), g) * 0.05, e4m3((G, D, F), g), scales((G, 3, 2), g) * 0.05
    b = bf16((G, D, D), g, 0.05)

    def layer(y, wait):
        for _ in range(3):
            y, _ = eng.mlp_swiglu_fp8(y, w, w13, s13, w2, s2, residual=y, offsets=off)
            wait()
            y = eng.gemm_grouped_bf16(y, off, b, transB=False)
            wait()
            y = eng.rms_norm(y, w)[0]
            wait()
        return y

    want = layer(x, torch.cuda.synchronize)
    got = [layer(x, lambda: None) for _ in range(20)]
    torch.cuda.synchronize()
    assert torch.isfinite(want.float()).all() and all(torch.equal(y, want) for y in got)


def test_the_first_call_of_a_process_may_be_captured(built):
    code = """
import sys, torch
sys.path.insert(0, {root!r})
import open64_b200 as o
e = o.Engine(0)
a, b = torch.randn(20, 256, device="cuda").to(torch.bfloat16), torch.randn(2, 128, 256, device="cuda").to(torch.bfloat16)
big = torch.randn(700, 256, device="cuda").to(torch.bfloat16)
off, off2 = (torch.tensor(v, device="cuda", dtype=torch.int32) for v in ([0, 7, 20], [0, 600, 700]))
w = torch.ones(256, device="cuda")
torch.cuda.synchronize()
graph = torch.cuda.CUDAGraph()
with torch.cuda.graph(graph):
    c, d = e.gemm_grouped_bf16(a, off, b), e.gemm_grouped_bf16(big, off2, b)
    y, _, s, rstd = e.rms_norm(big, w)
    dx, dw = e.rms_norm_backward(big, s, w, rstd)
    db = e.gemm_grouped_bf16_wgrad(d, big, off2)
graph.replay()
torch.cuda.synchronize()
assert torch.equal(c, e.gemm_grouped_bf16(a, off, b)) and torch.equal(d, e.gemm_grouped_bf16(big, off2, b))
assert torch.equal(db, e.gemm_grouped_bf16_wgrad(d, big, off2)) and torch.equal(dx, e.rms_norm_backward(big, s, w, rstd)[0])
assert e.last_status() == (o.OK, 0)
print("captured")
"""
    import os
    import subprocess
    import sys
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    r = subprocess.run([sys.executable, "-c", code.format(root=root)], capture_output=True, text=True, timeout=300)
    assert r.returncode == 0 and "captured" in r.stdout, r.stderr[-2000:]


def test_thousands_of_groups(eng):
    G, N, K = 3000, 16, 64
    g = gen(14)
    sizes = [1 if i % 31 == 0 else 0 for i in range(G)]
    sizes[-1] = 40
    T = sum(sizes)
    a, b = bf16((T, K), g), bf16((G, N, K), g)
    want, size = grouped(a.double(), sizes, b.double().mT)
    close_bf16(eng.gemm_grouped_bf16(a, offsets_of(sizes), b), want, size, K)


def test_gradients_of_a_grouped_layer_agree_with_differences(eng):
    """loss = sum(W . (A B^T)) by group: its gradients through the input_grad and weight_grad forms against
    central differences in 64 bits of the same loss."""
    sizes, N, K = [3, 0, 5], 16, 24
    g = gen(31)
    T, off = sum(sizes), offsets_of(sizes)
    a, b, dc = bf16((T, K), g), bf16((3, N, K), g), bf16((T, N), g)
    da = eng.gemm_grouped_bf16(dc, off, b, transB=False)
    db = eng.gemm_grouped_bf16_wgrad(dc, a, off, o.OUT_F32)
    loss = lambda aa, bb: float((grouped(aa, sizes, bb.mT)[0] * dc.double()).sum())
    for i, j in ((0, 0), (2, 23), (7, 5)):
        e = torch.zeros((T, K), device="cuda", dtype=torch.float64)
        e[i, j] = 0.5
        d = loss(a.double() + e, b.double()) - loss(a.double() - e, b.double())
        assert abs(float(da[i, j]) - d) <= BF16 * abs(d) + 1e-4
    for k, i, j in ((0, 0, 0), (1, 3, 3), (2, 15, 23)):
        e = torch.zeros((3, N, K), device="cuda", dtype=torch.float64)
        e[k, i, j] = 0.5
        d = loss(a.double(), b.double() + e) - loss(a.double(), b.double() - e)
        assert abs(float(db[k, i, j]) - d) <= 1e-4


def test_feed_forward_block_in_8_bits(eng):
    """norm -> gate/up with SiLU -> down, as mlp_swiglu_fp8 runs them: every stage against the 64-bit form of
    that stage on the operand it was given; with one group, the dense and the grouped calls give the same bits."""
    T, D, F = 70, 512, 384
    g = gen(40)
    x, r, w = bf16((T, D), g), bf16((T, D), g), torch.rand((D,), generator=g, device="cuda") + 0.5
    w13, s13, w2, s2 = e4m3((2, 2 * F, D), g), scales((2, 6, 4), g) * 0.05, e4m3((2, D, F), g), scales((2, 4, 3), g) * 0.05
    off = offsets_of([41, 29])
    out, stream = eng.mlp_swiglu_fp8(x, w, w13, s13, w2, s2, residual=r, offsets=off)
    a, sa, summed, _ = eng.rms_norm(x, w, r, out_kind=o.OUT_E4M3)
    assert torch.equal(stream, summed) and torch.equal(summed, (x.float() + r.float()).to(torch.bfloat16))
    h, sh = eng.gemm_grouped_fp8_block_swiglu(a, sa, off, w13, s13)
    A, W = value(a, sa, 1), value(w13, s13, 128)
    for e, rows in enumerate((slice(0, 41), slice(41, 70))):
        check_swiglu(h[rows], sh[rows], swiglu_reference(A[rows], W[e], F), D)
    want, size = grouped(value(h, sh, 1), [41, 29], value(w2, s2, 128).mT)
    close_bf16(out, want, size, F)
    dense, _ = eng.mlp_swiglu_fp8(x, w, w13[0], s13[0], w2[0], s2[0], residual=r)
    alone, _ = eng.mlp_swiglu_fp8(x, w, w13[:1], s13[:1], w2[:1], s2[:1], residual=r, offsets=offsets_of([T]))
    assert torch.equal(dense, alone)


def test_refusals(eng):
    g = gen(3)
    a, b, off = bf16((10, 64), g), bf16((2, 32, 64), g), offsets_of([4, 6])
    a8, sa, w, sw = e4m3((10, 256), g), scales((10, 2), g), e4m3((2, 256, 256), g), scales((2, 2, 2), g)
    refused(o.ERR_DTYPE, lambda: eng.gemm_grouped_bf16(a.float(), off, b))
    refused(o.ERR_DTYPE, lambda: eng.gemm_grouped_bf16(a, off.long(), b))
    refused(o.ERR_CONFORM, lambda: eng.gemm_grouped_bf16(a, off[:2], b))
    refused(o.ERR_CONFORM, lambda: eng.gemm_grouped_bf16(a[:, :32], off, b))
    refused(o.ERR_RANK, lambda: eng.gemm_grouped_bf16(a, off, b[0]))
    refused(o.ERR_RANK, lambda: eng.gemm_grouped_bf16(a, off.cpu(), b))
    refused(o.ERR_CONFORM, lambda: eng.gemm_grouped_bf16(a, off, b, out=torch.empty((10, 31), device="cuda", dtype=torch.bfloat16)))
    refused(o.ERR_CONFORM, lambda: eng.gemm_grouped_bf16(a, off, b, out=torch.empty((1, 32), device="cuda", dtype=torch.bfloat16).expand(10, 32)))
    refused(o.ERR_CONFORM, lambda: eng.gemm_grouped_bf16_wgrad(a, a[:9], off))
    refused(o.ERR_DTYPE, lambda: eng.gemm_grouped_bf16_wgrad(a, a, off, o.OUT_E4M3))
    refused(o.ERR_CONFORM, lambda: eng.gemm_grouped_bf16_wgrad(a, a, off[:0]))
    refused(o.ERR_CONFORM, lambda: eng.gemm_fp8_block(a8, sa[:, :1], w[0], sw[0]))
    refused(o.ERR_CONFORM, lambda: eng.gemm_fp8_block(a8, sa, w[0], sw[0, :1]))
    refused(o.ERR_DTYPE, lambda: eng.gemm_fp8_block(a, sa, w[0], sw[0]))
    refused(o.ERR_DTYPE, lambda: eng.gemm_fp8_block(a8, sa.half(), w[0], sw[0]))
    refused(o.ERR_CONFORM, lambda: eng.gemm_fp8_block_swiglu(a8, sa, w[0, :128], sw[0, :1]))
    refused(o.ERR_DTYPE, lambda: eng.gemm_fp8_block_swiglu(a8, sa, w[0], sw[0], o.OUT_S8))
    refused(o.ERR_RANK, lambda: eng.gemm_grouped_fp8_block(a8, sa, off, w[0], sw[0]))
    L, P = eng.lib, lambda t: t.data_ptr()
    c = torch.empty((10, 32), device="cuda", dtype=torch.bfloat16)
    s = torch.cuda.current_stream().cuda_stream
    call = lambda **k: L.o64_gemm_grouped_bf16(*{**dict(h=eng._h, G=2, T=10, N=32, K=64, A=P(a), lda=64, off=P(off), B=P(b), ldb=64, sb=32 * 64, t=1,
                                                        C=P(c), ldc=32, st=s), **k}.values())
    assert call() == o.OK
    assert call(A=P(a) + 2) == o.ERR_ALIGN and call(lda=65) == o.ERR_ALIGN and call(sb=32 * 64 + 4) == o.ERR_ALIGN
    assert call(off=None) == o.ERR_RANK and call(A=None) == o.ERR_RANK and call(C=None) == o.ERR_RANK and call(G=-1) == o.ERR_RANK
    assert call(lda=56) == o.ERR_CONFORM and call(ldc=24) == o.ERR_CONFORM and call(sb=31 * 64) == o.ERR_CONFORM
    host = torch.zeros(4096, dtype=torch.bfloat16)
    assert call(A=P(host)) == o.ERR_RANK and call(off=P(host)) == o.ERR_RANK
    torch.cuda.synchronize()
