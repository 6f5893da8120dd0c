"""Cases of the operators around a feed-forward layer's products - RMS norm with the residual's addition
and an e4m3 result, the e4m3 product with a scale for each block of 128, the products grouped by expert -
with their plain forms, the calls of the framework and the values in 64 bits.

A case is a dict of plain values.  ``op`` is one of

  norm        h = s * rsqrt(mean(s^2) + eps) * w with s = x + residual, bf16 or e4m3 with scales per 128;
              direction "backward": the gradients of x (and of the residual, the same) and of w
  fp8         C = sum over blocks of 128 of K: scaleA[m,kb] * scaleB[nb,kb] * (A8 B8^T)[m,n] in that block;
              ``trans_b`` false: B8 stored [K,N], which is how the gradient of A reads a weight [N,K]
  experts_fp8 the same product by expert (rows sorted, offsets on the device); ``swiglu``: gate and up
              columns side by side, silu(gate) * up as e4m3 with scales per 128
  experts     the bf16 product by expert: "forward", "input_grad" (weight read as it lies), "weight_grad"
"""
import torch

own = False
BLOCK = 128
E4M3_MAX = 448.0
MIN_NORMAL = 2.0 ** -126
EPS = 1e-6


# ---- cases -------------------------------------------------------------------------------------
def listed():
    return [
        # one new token enters a layer: launch latency is everything
        dict(name="norm_token", op="norm", direction="forward", T=1, N=4096, out="e4m3", residual=True, w="bf16"),
        # a long prompt (or a large training batch) in front of an 8-bit product: a pass over HBM
        dict(name="norm_prefill", op="norm", direction="forward", T=16384, N=8192, out="e4m3", residual=True, w="bf16"),
        # training step, odd row count, a width that is no multiple of the scale block
        dict(name="norm_backward", op="norm", direction="backward", T=8191, N=5000, out="bf16", residual=True, w="f32"),
        # one token through a large linear: the weight's 64 MiB stream from HBM
        dict(name="fp8_token", op="fp8", M=1, N=8192, K=8192, trans_b=True),
        # gradient of a linear's input at sizes that fill no tile, scale block or K block
        dict(name="fp8_ragged_grad", op="fp8", M=515, N=4104, K=4208, trans_b=False),
        # prompt through a large linear: the tensor pipe
        dict(name="fp8_prefill", op="fp8", M=4096, N=8192, K=8192, trans_b=True),
        # decoding with experts: three rows an expert, some have none; all their weights stream from HBM
        dict(name="experts_fp8_tokens", op="experts_fp8", T=96, G=32, N=2048, K=4096, trans_b=True, swiglu=True, load="gaps"),
        # prompt through the gate and up projections of eight experts, unevenly loaded
        dict(name="experts_fp8_prefill", op="experts_fp8", T=8192, G=8, N=14336, K=4096, trans_b=True, swiglu=True, load="skewed"),
        # a few rows through the experts' bf16 down projection
        dict(name="experts_tokens", op="experts", direction="forward", T=16, G=8, N=4096, K=14336, load="even"),
        # training step of the same layer: forward, gradient of the input, gradient of the weights
        dict(name="experts_forward", op="experts", direction="forward", T=8192, G=8, N=4096, K=14336, load="skewed"),
        dict(name="experts_input_grad", op="experts", direction="input_grad", T=4099, G=16, N=2056, K=4096, load="gaps"),
        dict(name="experts_weight_grad", op="experts", direction="weight_grad", T=8192, G=8, N=4096, K=14336, load="skewed"),
    ]


def _log(rng, lo, hi):
    return int(round(lo * (hi / lo) ** rng.random()))


def _multiple(v, of):
    return max(of, v // of * of)


def draw(rng):
    op = rng.choice(["norm", "norm", "fp8", "fp8", "experts_fp8", "experts", "experts"])
    if op == "norm":
        n = _log(rng, 64, 16384)
        if rng.random() < 0.7:
            n = _multiple(n, 8)
        t = _log(rng, 1, min(16384, (1 << 27) // n))
        direction = rng.choice(["forward", "forward", "backward"])
        return dict(op=op, direction=direction, T=t, N=n, out=rng.choice(["bf16", "e4m3"]) if direction == "forward" else "bf16",
                    residual=rng.random() < 0.7, w=rng.choice(["bf16", "f32"]))
    if op == "fp8":
        m, n, k = _log(rng, 1, 8192), _log(rng, 64, 8192), _multiple(_log(rng, 128, 8192), 16)
        if m * n * k > 4096 * 8192 * 8192:
            m //= 2
        return dict(op=op, M=m, N=_multiple(n, 8) if rng.random() < 0.7 else _multiple(n, 16), K=k, trans_b=rng.random() < 0.7)
    g = _log(rng, 1, 64)
    t = _log(rng, 1, 8192)
    k = _multiple(_log(rng, 256, 8192), 32)
    load = rng.choice(["even", "skewed", "gaps"])
    if op == "experts_fp8":
        swiglu = rng.random() < 0.5
        n = _multiple(_log(rng, 128, 8192), 128 if swiglu else 16)
        if n * k > 14336 * 4096:
            k //= 2
        while g * n * k > 4 * 14336 * 4096:
            g = max(1, g // 2)
        return dict(op=op, T=t, G=g, N=n, K=k, trans_b=swiglu or rng.random() < 0.7, swiglu=swiglu, load=load)
    n = _multiple(_log(rng, 64, 8192), 8)
    if n * k > 14336 * 4096:
        k //= 2
    while g * n * k > 4 * 14336 * 4096:
        g = max(1, g // 2)
    return dict(op=op, direction=rng.choice(["forward", "forward", "input_grad", "weight_grad"]), T=t, G=g, N=n, K=k, load=load)


def _sizes(case):
    """Rows of each expert: even; in proportion to 1, 1/2, 1/3, ... ; or even with every third expert left out."""
    T, G, load = case["T"], case["G"], case["load"]
    share = [1.0 / (1 + (5 * i) % G) if load == "skewed" and G % 5 else 1.0 / (1 + i) if load == "skewed" else
             0.0 if load == "gaps" and i % 3 == 1 else 1.0 for i in range(G)]
    total, ends, run_sum = sum(share), [0], 0.0
    for s in share:
        run_sum += s
        ends.append(int(round(T * run_sum / total)))
    return [b - a for a, b in zip(ends, ends[1:])]


# ---- inputs ------------------------------------------------------------------------------------
def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _randn(shape, g, scale=1.0):
    return torch.randn(shape, generator=g, device="cuda").mul_(scale)


def _activations(shape, g):
    """Unit variance with a few channels that are an order of magnitude larger, as hidden states have."""
    x = _randn(shape, g)
    channels = torch.rand(shape[-1], generator=g, device="cuda")
    return x * torch.where(channels < 0.01, 8.0, 1.0)


def _padded(x, rows, cols):
    return torch.nn.functional.pad(x, (0, -x.shape[-1] % cols, 0, -x.shape[-2] % rows))


def _scale_of(amax):
    scale = amax / E4M3_MAX
    return torch.where(scale < MIN_NORMAL, torch.ones_like(scale), scale)


def _quantized(x, rows):
    """Input data in e4m3: scales of blocks of `rows` x 128 (amax / 448)."""
    r, c = x.shape
    p = _padded(x, rows, BLOCK)
    blocks = p.view(p.shape[0] // rows, rows, p.shape[1] // BLOCK, BLOCK)
    scale = _scale_of(blocks.abs().amax(dim=(1, 3)))
    q = (blocks / scale[:, None, :, None]).clamp_(-E4M3_MAX, E4M3_MAX).view_as(p)[:r, :c]
    return q.to(torch.float8_e4m3fn).contiguous(), scale.contiguous()


def _weights(count, rows, cols, g, bf16):
    if bf16:
        return torch.stack([_randn((rows, cols), g, 0.02).to(torch.bfloat16) for _ in range(count)])
    made = [_quantized(_randn((rows, cols), g, 0.02), BLOCK) for _ in range(count)]
    return torch.stack([q for q, _ in made]), torch.stack([s for _, s in made])


def prepare(case, seed):
    g = _gen(seed)
    s = dict(case)
    op = case["op"]
    if op == "norm":
        T, N = case["T"], case["N"]
        s["x"] = _activations((T, N), g).to(torch.bfloat16)
        s["r"] = _activations((T, N), g).mul_(3.0).to(torch.bfloat16) if case["residual"] else None
        w = 1.0 + 0.2 * _randn((N,), g)
        s["weight"] = w.to(torch.bfloat16) if case["w"] == "bf16" else w
        if case["direction"] == "backward":
            # what the forward pass left behind: the stream after the addition and its 1 / rms
            total = s["x"].float() + (s["r"].float() if case["residual"] else 0.0)
            s["summed"] = total.to(torch.bfloat16)
            s["rstd"] = torch.rsqrt(total.square().mean(dim=1) + EPS)
            s["dy"] = _randn((T, N), g, 0.1).to(torch.bfloat16)
            s["dr"] = _randn((T, N), g, 0.1).to(torch.bfloat16) if case["residual"] else None
    elif op == "fp8":
        M, N, K = case["M"], case["N"], case["K"]
        s["a"], s["sa"] = _quantized(_activations((M, K), g), 1)
        b, sb = _weights(1, *((N, K) if case["trans_b"] else (K, N)), g, False)
        s["b"], s["sb"] = b[0], sb[0]
    else:
        T, G, N, K = case["T"], case["G"], case["N"], case["K"]
        s["sizes"] = _sizes(case)
        ends = torch.tensor([0] + s["sizes"], device="cuda").cumsum(0)
        s["offsets"] = ends.to(torch.int32)
        if op == "experts_fp8":
            s["a"], s["sa"] = _quantized(_activations((T, K), g), 1)
            rows = 2 * N if case["swiglu"] else N
            s["b"], s["sb"] = _weights(G, *((rows, K) if case["trans_b"] else (K, rows)), g, False)
        elif case["direction"] == "weight_grad":
            s["a"] = _activations((T, K), g).to(torch.bfloat16)
            s["dc"] = _randn((T, N), g, 0.1).to(torch.bfloat16)
        else:
            # the gradient of the input is the product with the weight [K,N] read as it lies: rows are the sum's index
            s["a"] = _activations((T, K), g).to(torch.bfloat16)
            s["b"] = _weights(G, *((N, K) if case["direction"] == "forward" else (K, N)), g, True)
    return s


# ---- one pass ----------------------------------------------------------------------------------
_engines = {}


def _engine():
    import open64_b200

    device = torch.cuda.current_device()
    if device not in _engines:
        _engines[device] = open64_b200.Engine(device)
    return open64_b200, _engines[device]


def _run_own(s):
    o, eng = _engine()
    op = s["op"]
    if op == "norm" and s["direction"] == "forward":
        y, scales, summed, rstd = eng.rms_norm(s["x"], s["weight"], s["r"], eps=EPS, out_kind=o.OUT_E4M3 if s["out"] == "e4m3" else o.OUT_BF16)
        return {"y": y, "scales": scales, "summed": summed, "rstd": rstd}
    if op == "norm":
        dx, dw = eng.rms_norm_backward(s["dy"], s["summed"], s["weight"], s["rstd"], s["dr"])
        return {"dx": dx, "dw": dw}
    if op == "fp8":
        return {"c": eng.gemm_fp8_block(s["a"], s["sa"], s["b"], s["sb"], transB=s["trans_b"])}
    if op == "experts_fp8":
        if s["swiglu"]:
            h, scales = eng.gemm_grouped_fp8_block_swiglu(s["a"], s["sa"], s["offsets"], s["b"], s["sb"])
            return {"h": h, "scales": scales}
        return {"c": eng.gemm_grouped_fp8_block(s["a"], s["sa"], s["offsets"], s["b"], s["sb"], transB=s["trans_b"])}
    if s["direction"] == "weight_grad":
        return {"db": eng.gemm_grouped_bf16_wgrad(s["dc"], s["a"], s["offsets"])}
    return {"c": eng.gemm_grouped_bf16(s["a"], s["offsets"], s["b"], transB=s["direction"] == "forward")}


def _e4m3_rows(h):
    """e4m3 with a scale for each 128 of a row."""
    rows, cols = h.shape
    blocks = _padded(h, 1, BLOCK).view(rows, -1, BLOCK)
    scale = _scale_of(blocks.abs().amax(dim=2))
    q = (blocks / scale[:, :, None]).clamp(-E4M3_MAX, E4M3_MAX).view(rows, -1)[:, :cols]
    return q.to(torch.float8_e4m3fn), scale


def _spread(scale, rows, cols, shape):
    """Scales of blocks of `rows` x `cols` at every element."""
    return scale.repeat_interleave(rows, 0)[: shape[0]].repeat_interleave(cols, 1)[:, : shape[1]]


def _block_product(a, sa, b, sb, trans_b):
    a32 = a.float() * _spread(sa, 1, BLOCK, a.shape)
    b32 = b.float() * _spread(sb, BLOCK, BLOCK, b.shape)
    return a32 @ (b32.t() if trans_b else b32)


def _run_plain(s):
    op = s["op"]
    if op == "norm" and s["direction"] == "forward":
        total = s["x"].float() if s["r"] is None else s["x"].float() + s["r"].float()
        rstd = torch.rsqrt(total.square().mean(dim=1) + EPS)
        h = total * rstd[:, None] * s["weight"].float()
        y, scales = _e4m3_rows(h) if s["out"] == "e4m3" else (h.to(torch.bfloat16), None)
        return {"y": y, "scales": scales, "summed": s["x"] if s["r"] is None else total.to(torch.bfloat16), "rstd": rstd}
    if op == "norm":
        n = s["summed"].float() * s["rstd"][:, None]
        dy = s["dy"].float()
        g = dy * s["weight"].float()
        dx = s["rstd"][:, None] * (g - n * (g * n).mean(dim=1, keepdim=True))
        return {"dx": (dx if s["dr"] is None else dx + s["dr"].float()).to(torch.bfloat16), "dw": (dy * n).sum(dim=0)}
    if op == "fp8":
        return {"c": _block_product(s["a"], s["sa"], s["b"], s["sb"], s["trans_b"]).to(torch.bfloat16)}
    if op == "experts_fp8":
        parts = zip(s["a"].split(s["sizes"]), s["sa"].split(s["sizes"]), s["b"], s["sb"])
        c = torch.cat([_block_product(a, sa, b, sb, s["trans_b"]) for a, sa, b, sb in parts])
        if s["swiglu"]:
            gate, up = c.chunk(2, dim=1)
            q, scales = _e4m3_rows(gate / (1.0 + torch.exp(-gate)) * up)
            return {"h": q, "scales": scales}
        return {"c": c.to(torch.bfloat16)}
    if s["direction"] == "weight_grad":
        parts = zip(s["dc"].split(s["sizes"]), s["a"].split(s["sizes"]))
        return {"db": torch.stack([(dc.float().t() @ a.float()).to(torch.bfloat16) for dc, a in parts])}
    parts = zip(s["a"].split(s["sizes"]), s["b"])
    forward = s["direction"] == "forward"
    return {"c": torch.cat([a.float() @ (b.float().t() if forward else b.float()) for a, b in parts]).to(torch.bfloat16)}


def run(state):
    return _run_own(state) if own else _run_plain(state)


# ---- what a pass cannot do without --------------------------------------------------------------
def work(case):
    op = case["op"]
    if op == "norm":
        T, N = case["T"], case["N"]
        w = N * (2 if case["w"] == "bf16" else 4)
        if case["direction"] == "backward":  # dy, the stream, 1 / rms, w (and the residual's gradient) in; dx and dw out
            return {"bytes": T * N * (8 if case["residual"] else 6) + 4 * T + w + 4 * N, "flops": 9 * T * N}
        out = T * N + 4 * T * -(-N // BLOCK) if case["out"] == "e4m3" else 2 * T * N
        return {"bytes": T * N * (6 if case["residual"] else 2) + out + 4 * T + w, "flops": 6 * T * N}
    if op == "fp8":
        M, N, K = case["M"], case["N"], case["K"]
        scales = 4 * (M * -(-K // BLOCK) + -(-N // BLOCK) * -(-K // BLOCK))
        return {"bytes": M * K + N * K + scales + 2 * M * N, "flops": 2 * M * N * K}
    T, G, N, K = case["T"], case["G"], case["N"], case["K"]
    active = sum(n > 0 for n in _sizes(case))
    if op == "experts_fp8":
        cols = 2 * N if case["swiglu"] else N
        weights = active * (cols * K + 4 * -(-cols // BLOCK) * -(-K // BLOCK))
        out = T * N + 4 * T * -(-N // BLOCK) if case["swiglu"] else 2 * T * N
        return {"bytes": weights + T * K + 4 * T * -(-K // BLOCK) + 4 * (G + 1) + out, "flops": 2 * T * cols * K}
    if case["direction"] == "weight_grad":
        return {"bytes": 2 * T * (N + K) + 2 * G * N * K + 4 * (G + 1), "flops": 2 * T * N * K}
    return {"bytes": 2 * T * (N + K) + 2 * active * N * K + 4 * (G + 1), "flops": 2 * T * N * K}


# ---- the values in 64 bits ----------------------------------------------------------------------
def _exact_quant(h):
    """Blocks of 128 along a row, each divided by amax / 448 (1 where that is no normal number) and rounded to e4m3."""
    T, N = h.shape
    nb = (N + BLOCK - 1) // BLOCK
    wide = h.new_zeros(T, nb * BLOCK)
    wide[:, :N] = h
    wide = wide.unflatten(1, (nb, BLOCK))
    peak = torch.linalg.vector_norm(wide, float("inf"), dim=2) / 448
    peak = peak.masked_fill(peak < 2.0 ** -126, 1.0)
    return (wide / peak.unsqueeze(2)).clamp(-448, 448).flatten(1)[:, :N].to(torch.float8_e4m3fn).double(), peak


def _exact_operand(q, scale, rows):
    """The real numbers that an e4m3 matrix with a scale for each block of `rows` x 128 stands for."""
    i = torch.arange(q.shape[0], device=q.device) // rows
    j = torch.arange(q.shape[1], device=q.device) // BLOCK
    return q.double() * scale.double()[i[:, None], j[None, :]]


def exact(case, seed):
    s = prepare(case, seed)
    op = case["op"]
    if op == "norm":
        w = s["weight"].double()
        if case["direction"] == "forward":
            total = s["x"].double()
            if case["residual"]:
                total = total + s["r"].double()
            rms = torch.sqrt(torch.linalg.vector_norm(total, dim=1) ** 2 / case["N"] + EPS)
            h = total / rms[:, None] * w
            y, scales = _exact_quant(h) if case["out"] == "e4m3" else (h, None)
            return {"y": y, "scales": scales, "summed": total, "rstd": 1 / rms}
        z, rstd, dy = s["summed"].double(), s["rstd"].double().unsqueeze(1), s["dy"].double()
        # d/dz of z * rstd(z) * w applied to dy: rstd w dy - z rstd^3 (z . w dy) / N
        along = torch.einsum("tn,tn,n->t", z, dy, w).unsqueeze(1) / case["N"]
        dx = rstd * dy * w - z * rstd ** 3 * along
        return {"dx": dx + s["dr"].double() if case["residual"] else dx, "dw": torch.einsum("tn,tn,t->n", dy, z, rstd.squeeze(1))}
    if op == "fp8":
        a = _exact_operand(s["a"], s["sa"], 1)
        b = _exact_operand(s["b"], s["sb"], BLOCK)
        return {"c": torch.matmul(a, b.mT if case["trans_b"] else b)}
    first, out = 0, []
    for e, n in enumerate(s["sizes"]):
        rows = slice(first, first + n)
        first += n
        if op == "experts_fp8":
            a, b = _exact_operand(s["a"][rows], s["sa"][rows], 1), _exact_operand(s["b"][e], s["sb"][e], BLOCK)
            out.append(torch.matmul(a, b.mT if case["trans_b"] else b))
        elif case["direction"] == "weight_grad":
            out.append(torch.matmul(s["dc"][rows].double().mT, s["a"][rows].double()))
        else:
            b = s["b"][e].double()
            out.append(torch.matmul(s["a"][rows].double(), b.mT if case["direction"] == "forward" else b))
    if op == "experts" and case["direction"] == "weight_grad":
        return {"db": torch.stack(out)}
    c = torch.cat(out)
    if op == "experts_fp8" and case["swiglu"]:
        N = case["N"]
        h, scales = _exact_quant(c[:, :N] * torch.sigmoid(c[:, :N]) * c[:, N:])
        return {"h": h, "scales": scales}
    return {"c": c}
