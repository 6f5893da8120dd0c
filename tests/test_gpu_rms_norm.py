"""GPU: RMS norm with the residual's addition, its e4m3 result and its gradient, against 64-bit formulas.

Tolerances.  fp32 arithmetic on N terms: the mean of squares is within (N/threads + log2) additions, here
bounded by 64 * 2^-24 relative; rstd halves that; h = s * rstd * w adds three roundings.  H = 2^-17 covers all
of it relative to |h| (s itself is one fp32 rounding of x + r: relative to |x| + |r|, so where they cancel the
error is counted against that sum).  A bf16 result adds half a step, 2^-8 |h|; an e4m3 one 2^-4 |h|, or half of
the smallest step 2^-10 * scale.  dw: T terms added in fp32, at most (rows a group + groups / 16 + 20) additions
in sequence, each within 2^-24 of the partial sum of magnitudes."""
import numpy as np
import pytest
import torch

import open64_b200 as o

pytestmark = pytest.mark.gpu
H = 2.0 ** -17
BF16, E4M3 = 2.0 ** -8, 2.0 ** -4


def data(T, N, seed, residual=True, w_dtype=torch.float32):
    g = torch.Generator(device="cuda").manual_seed(seed)
    x = torch.randn((T, N), generator=g, device="cuda").to(torch.bfloat16)
    r = (torch.randn((T, N), generator=g, device="cuda") * 3).to(torch.bfloat16) if residual else None
    w = (1 + 0.2 * torch.randn((N,), generator=g, device="cuda")).to(w_dtype)
    return x, r, w


def formula(x, r, w, eps):
    s = x.double() + (r.double() if r is not None else 0)
    rstd = 1 / torch.sqrt((s * s).mean(1) + eps)
    size = x.double().abs() + (r.double().abs() if r is not None else 0)
    return s, rstd, s * rstd[:, None] * w.double(), size * rstd[:, None] * w.double().abs()


def blocks(h, block):
    T, N = h.shape
    if not block:
        return h.abs().amax(1, keepdim=True)
    return torch.nn.functional.pad(h.abs(), (0, -N % block)).view(T, -1, block).amax(2)


def check_e4m3(y, scales, h, size, block):
    """y * scale is h to half a step, and scale is its block's largest value / 448."""
    peak = blocks(h, block)
    want = torch.where(peak / 448 < 2.0 ** -126, torch.ones_like(peak), peak / 448)
    got = scales.double() if block else scales.double()[:, None]
    assert ((got - want).abs() <= 2 * H * blocks(size, block) / 448 + 2.0 ** -23 * want).all()
    at = got.repeat_interleave(block, 1)[:, :h.shape[1]] if block else got
    off = (y.double() * at - h).abs()
    assert (off <= E4M3 * (1 + 2.0 ** -16) * h.abs() + 2.0 ** -10 * at + 4 * H * size).all()


SHAPES = [(1, 1), (1, 4096), (3, 64), (2, 127), (5, 128), (4, 129), (33, 1000), (129, 1024), (7, 2141), (300, 4096), (9, 5003), (65, 8192),
          (2, 16392), (1, 32768), (700, 136), (3, 32761)]


@pytest.mark.parametrize("T,N", SHAPES)
@pytest.mark.parametrize("residual", [True, False], ids=["residual", "plain"])
def test_bf16(eng, T, N, residual):
    x, r, w = data(T, N, T + N, residual, torch.bfloat16 if N % 2 else torch.float32)
    s, rstd, h, size = formula(x, r, w, 1e-5)
    y, scales, summed, got_rstd = eng.rms_norm(x, w, r, eps=1e-5)
    assert scales is None and y.dtype == torch.bfloat16
    assert ((y.double() - h).abs() <= BF16 * h.abs() + 2 * H * size).all()
    assert ((got_rstd.double() - rstd).abs() <= H * rstd).all()
    if residual:
        assert torch.equal(summed, (x.float() + r.float()).to(torch.bfloat16))
    else:
        assert summed is x


@pytest.mark.parametrize("T,N", SHAPES)
@pytest.mark.parametrize("block", [128, 0])
def test_e4m3(eng, T, N, block):
    x, r, w = data(T, N, T + 2 * N, T % 2 == 1, torch.float32 if N % 2 else torch.bfloat16)
    _, _, h, size = formula(x, r, w, 1e-6)
    y, scales, _, _ = eng.rms_norm(x, w, r, out_kind=o.OUT_E4M3, scale_block=block)
    assert y.dtype == torch.float8_e4m3fn and scales.shape == ((T, -(-N // 128)) if block else (T,))
    check_e4m3(y, scales, h, size, block)


MANY = [(1500, 2048), (1000, 4096), (1200, 5000), (601, 8192), (300, 16384), (890, 2056), (4800, 257), (1300, 5003), (2500, 1001), (601, 8190), (300, 16383)]  # rows in a ring of bulk copies


@pytest.mark.parametrize("T,N", MANY)
@pytest.mark.parametrize("residual", [True, False], ids=["residual", "plain"])
def test_many_rows(eng, T, N, residual):
    x, r, w = data(T, N, T + N, residual, torch.bfloat16 if T % 3 else torch.float32)
    x[17], w[5] = 0, 0
    s, rstd, h, size = formula(x, r, w, 1e-6)
    y, _, summed, got_rstd = eng.rms_norm(x, w, r)
    assert ((y.double() - h).abs() <= BF16 * h.abs() + 2 * H * size).all()
    assert ((got_rstd.double() - rstd).abs() <= H * rstd).all()
    if residual:
        assert torch.equal(summed, (x.float() + r.float()).to(torch.bfloat16))
    y, scales, _, _ = eng.rms_norm(x, w, r, out_kind=o.OUT_E4M3)
    check_e4m3(y, scales, h, size, 128)
    if residual:  # in place, and rows apart
        wide = torch.full((T, N + 8), 7.0, device="cuda", dtype=torch.bfloat16)
        wide[:, :N] = r
        y2, scales2, s2, _ = eng.rms_norm(x, w, wide[:, :N], out_kind=o.OUT_E4M3, summed=wide[:, :N])
        assert torch.equal(y2.float(), y.float()) and torch.equal(scales2, scales) and torch.equal(s2, summed) and (wide[:, N:] == 7).all()


def test_zero_rows_tiny_values_and_block_of_zeros(eng):
    x = torch.zeros((4, 300), device="cuda", dtype=torch.bfloat16)
    x[1] = 2.0 ** -120
    x[2, :128] = 1.0  # the other blocks are zero
    w = torch.ones(300, device="cuda")
    y, scales, _, rstd = eng.rms_norm(x, w, out_kind=o.OUT_E4M3)
    assert (y[0].float() == 0).all() and (scales[0] == 1).all() and rstd[0].item() == pytest.approx(1e3, rel=1e-6)
    assert (scales[2, 1:] == 1).all() and (y[2, 128:].float() == 0).all() and (y[2, :128].float() == 448).all()
    _, _, h, size = formula(x, None, w, 1e-6)
    check_e4m3(y, scales, h, size, 128)


@pytest.mark.parametrize("T,N", [(3, 256), (4800, 2048), (4800, 2051)])
def test_e4m3_signs_of_zeros_and_a_block_past_the_largest_float(eng, T, N):
    """h of column 5 is past fp32's largest: its block's scale is infinite, its finite values are zeros, inf / inf is NaN."""
    x, _, w = data(T, N, 5, residual=False)
    x[:, 5], w[5] = 8, 3e38
    x[:, 130], x[:, 131] = 0.0, -0.0
    y, scales, _, _ = eng.rms_norm(x, w, out_kind=o.OUT_E4M3)
    torch.cuda.synchronize()
    assert torch.isinf(scales[:, 0]).all()
    assert torch.isnan(y[:, 5].float()).all()
    assert (y[:, :5].float() == 0).all() and (y[:, 6:128].float() == 0).all()
    assert (y[:, 130].view(torch.uint8) == 0).all() and (y[:, 131].view(torch.uint8) == 0x80).all()
    _, _, h, size = formula(x, None, w, 1e-6)
    check_e4m3(y[:, 128:], scales[:, 1:], h[:, 128:], size[:, 128:], 128)


def test_nan_and_infinity_stay_in_their_row_and_block(eng):
    x, r, w = data(6, 1000, 5)
    clean, clean_scales, _, _ = eng.rms_norm(x, w, r, out_kind=o.OUT_E4M3)
    w2 = w.clone()
    w2[200] = float("nan")
    y, scales, _, _ = eng.rms_norm(x, w2, r, out_kind=o.OUT_E4M3)
    assert torch.isnan(scales[:, 1]).all() and torch.isnan(y[:, 128:256].float()).all()
    keep = [0, 2, 3, 4, 5, 6, 7]
    assert torch.equal(scales[:, keep], clean_scales[:, keep])
    x[2, 7] = float("inf")
    x[4, 9] = float("nan")
    y, scales, _, rstd = eng.rms_norm(x, w, r, out_kind=o.OUT_E4M3)
    for row in (0, 1, 3, 5):
        assert torch.equal(y[row].view(torch.uint8), clean[row].view(torch.uint8)) and torch.equal(scales[row], clean_scales[row])
    assert rstd[2] == 0 and torch.isnan(rstd[4]) and torch.isnan(scales[4]).all()


def test_in_place_strides_and_what_lies_between(eng):
    T, N = 37, 1000
    x, r, w = data(T, N, 11)
    _, _, h, size = formula(x, r, w, 1e-6)
    for pad in (8, 3):  # vector path, and rows that start anywhere (another order of the sum: its own values to compare with)
        bx = torch.full((T, N + pad), 7.0, device="cuda", dtype=torch.bfloat16)
        br = bx.clone()
        bx[:, :N], br[:, :N] = x, r
        want = eng.rms_norm(bx[:, :N], w, br[:, :N], out_kind=o.OUT_E4M3)
        check_e4m3(want[0], want[1], h, size, 128)
        by = torch.zeros((T, N + pad), device="cuda", dtype=torch.float8_e4m3fn)
        bs = torch.full((T, 11), -1.0, device="cuda")
        y, scales, summed, _ = eng.rms_norm(bx[:, :N], w, br[:, :N], out_kind=o.OUT_E4M3, out=by[:, :N], scales=bs[:, :8], summed=br[:, :N])
        assert torch.equal(y.float(), want[0].float()) and torch.equal(scales, want[1]) and torch.equal(summed, want[2])
        assert (bx[:, N:] == 7).all() and (br[:, N:] == 7).all() and (by[:, N:].float() == 0).all() and (bs[:, 8:] == -1).all()


def test_offsets_past_32_bits(eng):
    T, N, ld = 3, 256, 1 << 30  # the third row starts 4 GiB into the tensor
    if torch.cuda.mem_get_info()[0] < 12 << 30:
        pytest.skip("needs 12 GB of free memory")
    big = torch.empty((2 * ld + N,), dtype=torch.bfloat16, device="cuda")
    x = big.as_strided((T, N), (ld, 1))
    vals, _, w = data(T, N, 3, False)
    x.copy_(vals)
    assert torch.equal(eng.rms_norm(x, w)[0], eng.rms_norm(vals, w)[0])


BACK = [(1, 1), (1, 4096), (3, 64), (5, 127), (130, 128), (64, 1000), (1000, 512), (445, 2141), (900, 4096), (50, 5000), (13, 8192), (3, 16392),
        (2, 32768), (4, 32761), (2000, 2048), (1300, 5000), (601, 8192), (305, 16384), (888, 4104), (4800, 257), (1300, 5003), (2500, 1001), (601, 8190), (305, 16383)]


@pytest.mark.parametrize("T,N", BACK)
@pytest.mark.parametrize("residual", [True, False], ids=["residual", "plain"])
def test_backward(eng, T, N, residual):
    x, r, w = data(T, N, T * 3 + N, True, torch.float32 if T % 2 else torch.bfloat16)
    g = torch.Generator(device="cuda").manual_seed(N)
    dy = torch.randn((T, N), generator=g, device="cuda").to(torch.bfloat16)
    dr = torch.randn((T, N), generator=g, device="cuda").to(torch.bfloat16) if residual else None
    _, _, s, rstd = eng.rms_norm(x, w, r)
    dx, dw = eng.rms_norm_backward(dy, s, w, rstd, dr)
    n = s.double() * rstd.double()[:, None]
    gw = dy.double() * w.double()
    want = rstd.double()[:, None] * (gw - n * (gw * n).mean(1, keepdim=True))
    size = rstd.double()[:, None] * (gw.abs() + n.abs() * (gw * n).abs().mean(1, keepdim=True))
    if residual:
        want = want + dr.double()
        size = size + dr.double().abs()
    assert ((dx.double() - want).abs() <= BF16 * want.abs() + 2 * H * size).all()
    terms = dy.double() * n
    groups = min(T, 444)
    steps = -(-T // groups) + groups / 16 + 20
    assert ((dw.double() - terms.sum(0)).abs() <= (steps + 2) * 2.0 ** -24 * terms.abs().sum(0)).all()
    again = eng.rms_norm_backward(dy, s, w, rstd, dr)
    assert torch.equal(again[0], dx) and torch.equal(again[1], dw)


def test_backward_agrees_with_differences(eng):
    """The gradient's formula against central differences of the 64-bit norm, at the kernel's own inputs."""
    T, N = 3, 40
    x, _, w = data(T, N, 77, False)
    dy = torch.randn((T, N), device="cuda", generator=torch.Generator(device="cuda").manual_seed(1)).to(torch.bfloat16)
    rstd = eng.rms_norm(x, w)[3]
    dx, dw = eng.rms_norm_backward(dy, x, w, rstd)
    loss = lambda xx, ww: float((formula(xx, None, ww, 1e-6)[2] * dy.double()).sum())
    step = 1e-5
    for i, j in ((0, 0), (1, 17), (2, 39)):
        e = torch.zeros((T, N), device="cuda", dtype=torch.float64)
        e[i, j] = step
        d = (loss(x.double() + e, w.double()) - loss(x.double() - e, w.double())) / (2 * step)
        assert abs(float(dx[i, j]) - d) <= BF16 * abs(d) + 1e-4
        d = (loss(x.double(), w.double() + e[i]) - loss(x.double(), w.double() - e[i])) / (2 * step)
        assert abs(float(dw[j]) - d) <= 1e-4


def test_backward_in_place_and_without_weight_gradient(eng):
    T, N = 100, 776
    x, r, w = data(T, N, 21)
    _, _, s, rstd = eng.rms_norm(x, w, r)
    dy, dr = x.clone(), r.clone()
    want, _ = eng.rms_norm_backward(dy, s, w, rstd, dr)
    got, _ = eng.rms_norm_backward(dy, s, w, rstd, dr, dx=dr)
    assert got is dr and torch.equal(got, want)
    out = torch.empty_like(want)
    P = lambda t: t.data_ptr()
    rc = eng.lib.o64_rmsnorm_bf16_backward(eng._h, T, N, P(dy), N, P(s), N, P(w), 1, P(rstd), P(r), N, P(out), N, None, None,
                                           torch.cuda.current_stream().cuda_stream)
    assert rc == o.OK and torch.equal(out, want)


@pytest.mark.parametrize("T,N", [(1300, 5003), (1500, 2048), (4800, 257)])
def test_many_rows_in_place(eng, T, N):
    """dx over dr, the sum over the residual, in rows that share 16-byte chunks with their neighbours."""
    x, r, w = data(T, N, 31)
    want = eng.rms_norm(x, w, r)
    r2 = r.clone()
    got = eng.rms_norm(x, w, r2, summed=r2)
    assert got[2] is r2 and all(torch.equal(a, b) for a, b in zip((got[0], got[2], got[3]), (want[0], want[2], want[3])))
    dx, dw = eng.rms_norm_backward(x, want[2], w, want[3], r)
    r3 = r.clone()
    got = eng.rms_norm_backward(x, want[2], w, want[3], r3, dx=r3)
    assert got[0] is r3 and torch.equal(r3, dx) and torch.equal(got[1], dw)
    x2 = x.clone()
    got = eng.rms_norm_backward(x2, want[2], w, want[3], r, dx=x2)
    assert torch.equal(x2, dx) and torch.equal(got[1], dw)
    view = torch.zeros((T * N + 1,), device="cuda", dtype=torch.bfloat16)[1:].view(T, N)  # a base off 16 bytes
    view.copy_(x)
    odd = eng.rms_norm(view, w, r, out_kind=o.OUT_E4M3)
    _, _, h, size = formula(x, r, w, 1e-6)
    check_e4m3(odd[0], odd[1], h, size, 128)


def test_no_rows(eng):
    w = torch.ones(64, device="cuda")
    x = torch.empty((0, 64), device="cuda", dtype=torch.bfloat16)
    y, _, _, rstd = eng.rms_norm(x, w)
    assert y.shape == (0, 64)
    dx, dw = eng.rms_norm_backward(x, x, w, rstd)
    assert dx.shape == (0, 64) and (dw == 0).all()


def test_other_stream_and_graph(eng):
    x, r, w = data(50, 1024, 2)
    want = eng.rms_norm(x, w, r, out_kind=o.OUT_E4M3)
    want_dx, want_dw = eng.rms_norm_backward(x, want[2], w, want[3], r)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = eng.rms_norm(x, w, r, out_kind=o.OUT_E4M3)
        got_dx, got_dw = eng.rms_norm_backward(x, got[2], w, got[3], r)
    side.synchronize()
    assert torch.equal(got[0].float(), want[0].float()) and torch.equal(got_dx, want_dx) and torch.equal(got_dw, want_dw)
    graphs = []
    for _ in range(2):  # two graphs at once: neither may use the other's memory
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            y = eng.rms_norm(x, w, r, out_kind=o.OUT_E4M3)
            d = eng.rms_norm_backward(x, y[2], w, y[3], r)
        graphs.append((graph, y, d))
    x2, r2, _ = data(50, 1024, 3)
    x.copy_(x2), r.copy_(r2)
    for graph, _, _ in graphs:
        graph.replay()
    torch.cuda.synchronize()
    want = eng.rms_norm(x, w, r, out_kind=o.OUT_E4M3)
    want_dx, want_dw = eng.rms_norm_backward(x, want[2], w, want[3], r)
    for _, y, d in graphs:
        assert torch.equal(y[0].float(), want[0].float()) and torch.equal(y[1], want[1])
        assert torch.equal(d[0], want_dx) and torch.equal(d[1], want_dw)


def test_refusals(eng):
    x, r, w = data(4, 256, 1)

    def refused(code, f):
        with pytest.raises(o.O64Error) as e:
            f()
        assert e.value.status == code

    refused(o.ERR_DTYPE, lambda: eng.rms_norm(x.float(), w))
    refused(o.ERR_DTYPE, lambda: eng.rms_norm(x, w.half()))
    refused(o.ERR_DTYPE, lambda: eng.rms_norm(x, w, out_kind=o.OUT_S8))
    refused(o.ERR_DTYPE, lambda: eng.rms_norm(x, w, out_kind=o.OUT_E4M3, scale_block=64))
    refused(o.ERR_CONFORM, lambda: eng.rms_norm(x, w[:255]))
    refused(o.ERR_CONFORM, lambda: eng.rms_norm(x, w, r[:3]))
    refused(o.ERR_CONFORM, lambda: eng.rms_norm(x, w, summed=x))
    refused(o.ERR_CONFORM, lambda: eng.rms_norm(x, w, out=torch.empty((256, 4), device="cuda", dtype=torch.bfloat16).t()))
    refused(o.ERR_RANK, lambda: eng.rms_norm(x.cpu(), w.cpu()))
    refused(o.ERR_RANK, lambda: eng.rms_norm(x, w.cpu()))
    wide = torch.zeros((1, 32769), device="cuda", dtype=torch.bfloat16)
    refused(o.ERR_RANK, lambda: eng.rms_norm(wide, wide[0].float()))
    refused(o.ERR_RANK, lambda: eng.rms_norm(x[:, :0], w[:0]))
    refused(o.ERR_DTYPE, lambda: eng.rms_norm(x[:1], w, rstd=torch.empty(1, device="cuda", dtype=torch.float64)))
    refused(o.ERR_CONFORM, lambda: eng.rms_norm(x, w, rstd=torch.empty(8, device="cuda")[::2]))
    refused(o.ERR_CONFORM, lambda: eng.rms_norm_backward(x, x, w, torch.empty(3, device="cuda")))
    L, P = eng.lib, lambda t: t.data_ptr()
    s = torch.cuda.current_stream().cuda_stream
    call = lambda **k: L.o64_rmsnorm_bf16(*{**dict(h=eng._h, T=4, N=256, X=P(x), ldx=256, R=None, ldr=0, S=None, lds=0, W=P(w), f=1, eps=1e-6,
                                                   kind=0, block=128, Y=P(r), ldy=256, sc=None, ldsc=0, rstd=None, st=s), **k}.values())
    host = np.zeros(4096, dtype=np.float32)
    assert call(X=host.ctypes.data) == o.ERR_RANK  # host memory is not staged here
    assert call(ldx=255) == o.ERR_CONFORM and call(T=-1) == o.ERR_RANK and call(W=None) == o.ERR_RANK
    assert call(kind=o.OUT_E4M3) == o.ERR_RANK  # no room for the scales
    assert call(kind=o.OUT_E4M3, sc=P(w), ldsc=1) == o.ERR_CONFORM
