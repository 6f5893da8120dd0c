"""CPU: the entry points around a feed-forward layer refuse calls without a handle, and their workspace query
needs no device."""
import open64_b200 as o


def test_no_handle_is_refused(built):
    L = o.lib()
    assert L.o64_rmsnorm_bf16(None, 4, 64, None, 64, None, 0, None, 0, None, 1, 1e-6, o.OUT_BF16, 128, None, 64, None, 0, None, None) == o.ERR_RANK
    assert L.o64_rmsnorm_bf16_backward(None, 4, 64, None, 64, None, 64, None, 1, None, None, 0, None, 64, None, None, None) == o.ERR_RANK
    assert L.o64_gemm_fp8_block(None, 1, 1, 16, None, 16, None, 1, None, 16, 1, None, 1, None, 16, None) == o.ERR_RANK
    assert L.o64_gemm_fp8_block_swiglu(None, 1, 128, 16, None, 16, None, 1, None, 16, None, 1, None, 128, o.OUT_E4M3, None, 1, None) == o.ERR_RANK
    assert L.o64_gemm_fp8_block_swiglu(None, 1, 128, 16, None, 16, None, 1, None, 16, None, 1, None, 128, o.OUT_S8, None, 1, None) == o.ERR_DTYPE
    assert L.o64_gemm_grouped_bf16(None, 1, 1, 8, 8, None, 8, None, None, 8, 64, 1, None, 8, None) == o.ERR_RANK
    assert L.o64_gemm_grouped_bf16_wgrad(None, 1, 1, 8, 8, None, 8, None, 8, None, None, 8, 64, o.OUT_BF16, None) == o.ERR_RANK
    assert L.o64_gemm_grouped_fp8_block(None, 1, 1, 8, 16, None, 16, None, 1, None, None, 16, 128, 1, None, 1, 1, None, 8, None) == o.ERR_RANK
    assert L.o64_gemm_grouped_fp8_block_swiglu(None, 1, 1, 128, 16, None, 16, None, 1, None, None, 16, 4096, None, 1, 2, None, 128, o.OUT_E4M3, None, 1,
                                               None) == o.ERR_RANK


def test_backward_workspace(built):
    need = o.lib().o64_rmsnorm_bf16_backward_workspace
    assert need(0, 64) == 0 and need(64, 0) == 0 and need(64, 32769) == 0
    assert need(1, 4096) == 4096 * 4  # one row: one partial row
    sizes = [need(1 << 20, n) for n in (64, 1000, 4096, 5003, 32768)]
    assert all(s > 0 and s % 4 == 0 for s in sizes) and max(sizes) <= 444 * 32768 * 4
