"""GPU: a pointer that is no multiple of its elements' size is refused before anything is launched, by every entry point
around a feed-forward layer's products and for each of its operands."""
import pytest
import torch

import open64_b200 as o

pytestmark = pytest.mark.gpu


def sweep(call, args, elements):
    assert call(*args.values()) == o.OK
    torch.cuda.synchronize()
    for name, size in elements.items():
        for off in range(1, size):
            assert call(*{**args, name: args[name] + off}.values()) == o.ERR_ALIGN, (name, off)
    torch.cuda.synchronize()


@pytest.fixture
def memory():
    return [torch.zeros(1 << 16, device="cuda") for _ in range(9)]


def test_rms_norm(eng, memory):
    L, s, m = eng.lib, torch.cuda.current_stream().cuda_stream, [t.data_ptr() for t in memory]
    for f32, kind in ((1, o.OUT_BF16), (0, o.OUT_E4M3)):
        args = dict(h=eng._h, T=4, N=256, X=m[0], ldx=256, R=m[1], ldr=256, S=m[2], lds=256, W=m[3], f=f32, eps=1e-6, kind=kind, block=128, Y=m[4],
                    ldy=256, sc=m[5], ldsc=2, rstd=m[6], st=s)
        sweep(L.o64_rmsnorm_bf16, args, dict(X=2, R=2, S=2, W=4 if f32 else 2, Y=2 if kind == o.OUT_BF16 else 1, sc=4, rstd=4))
        args = dict(h=eng._h, T=4, N=256, dY=m[0], lddy=256, S=m[1], lds=256, W=m[2], f=f32, rstd=m[3], dR=m[4], lddr=256, dX=m[5], lddx=256, dW=m[6],
                    ws=m[7], st=s)
        sweep(L.o64_rmsnorm_bf16_backward, args, dict(dY=2, S=2, W=4 if f32 else 2, rstd=4, dR=2, dX=2, dW=4, ws=4))


def test_block_scaled_products(eng, memory):
    L, s, m = eng.lib, torch.cuda.current_stream().cuda_stream, [t.data_ptr() for t in memory]
    args = dict(h=eng._h, M=4, N=256, K=256, A=m[0], lda=256, sa=m[1], ldsa=2, B=m[2], ldb=256, t=1, sb=m[3], ldsb=2, C=m[4], ldc=256, st=s)
    sweep(L.o64_gemm_fp8_block, args, dict(A=16, sa=4, B=16, sb=4, C=2))
    for kind in (o.OUT_BF16, o.OUT_E4M3):
        args = dict(h=eng._h, M=4, N=128, K=256, A=m[0], lda=256, sa=m[1], ldsa=2, B=m[2], ldb=256, sb=m[3], ldsb=2, H=m[4], ldh=128, kind=kind, sh=m[5],
                    ldsh=1, st=s)
        sweep(L.o64_gemm_fp8_block_swiglu, args, dict(A=16, sa=4, B=16, sb=4, H=2 if kind == o.OUT_BF16 else 1, **({} if kind == o.OUT_BF16 else dict(sh=4))))


def test_grouped_products(eng, memory):
    L, s, m = eng.lib, torch.cuda.current_stream().cuda_stream, [t.data_ptr() for t in memory]
    args = dict(h=eng._h, G=2, T=4, N=64, K=64, A=m[0], lda=64, off=m[1], B=m[2], ldb=64, sb=4096, t=1, C=m[3], ldc=64, st=s)
    sweep(L.o64_gemm_grouped_bf16, args, dict(A=16, off=4, B=16, C=2))
    for kind, size in ((o.OUT_BF16, 2), (o.OUT_F32, 4)):
        args = dict(h=eng._h, G=2, T=4, N=64, K=64, dC=m[0], lddc=64, A=m[1], lda=64, off=m[2], dB=m[3], lddb=64, sdb=4096, kind=kind, st=s)
        sweep(L.o64_gemm_grouped_bf16_wgrad, args, dict(dC=16, A=16, off=4, dB=size))
    args = dict(h=eng._h, G=2, T=4, N=64, K=64, A=m[0], lda=64, sa=m[1], ldsa=1, off=m[2], B=m[3], ldb=64, sb=4096, t=1, scb=m[4], ldsb=1, ssb=1, C=m[5],
                ldc=64, st=s)
    sweep(L.o64_gemm_grouped_fp8_block, args, dict(A=16, sa=4, off=4, B=16, scb=4, C=2))
    args = dict(h=eng._h, G=2, T=4, N=128, K=64, A=m[0], lda=64, sa=m[1], ldsa=1, off=m[2], B=m[3], ldb=64, sb=16384, scb=m[4], ldsb=1, ssb=2, H=m[5],
                ldh=128, kind=o.OUT_E4M3, sh=m[6], ldsh=1, st=s)
    sweep(L.o64_gemm_grouped_fp8_block_swiglu, args, dict(A=16, sa=4, off=4, B=16, scb=4, sh=4))
