"""Refusals of the block-scaled FP8 entry points, at the C boundary: every one returns before it touches the device, so a
made-up context and made-up (aligned) addresses do."""

import ctypes

import pytest

CTX, BUF = ctypes.c_void_p(0x1000), 0x100000


@pytest.fixture(scope="module")
def lib():
    from xax_b200 import _lib

    return _lib.load()


def refused(lib, rc, word):
    from xax_b200 import _lib

    assert rc in (_lib.BAD_ARGUMENT, _lib.UNSUPPORTED)
    assert word in lib.xaxb_last_error().decode()


@pytest.mark.parametrize("change,word", [
    (dict(x=None), "aligned"), (dict(x=BUF + 8), "aligned"), (dict(q=BUF + 4), "aligned"), (dict(inv=None), "aligned"),
    (dict(block_rows=2), "block_rows"), (dict(block_rows=0), "block_rows"), (dict(rows=0), "rows"), (dict(rows=-1), "rows"),
    (dict(cols=0), "multiple of 16"), (dict(cols=8), "multiple of 16"), (dict(cols=4100), "multiple of 16"),
    (dict(rows=1 << 28, cols=4096), "2^31"), (dict(block_rows=128, cols=1 << 24), "65535"),
])
def test_quantize_blocks_refuses(lib, change, word):
    a = dict(x=BUF, rows=4, cols=256, block_rows=1, q=BUF, inv=BUF) | change
    refused(lib, lib.xaxb_quantize_blocks(CTX, None, a["x"], a["rows"], a["cols"], a["block_rows"], a["q"], a["inv"]), word)


@pytest.mark.parametrize("change,word", [
    (dict(x=BUF + 2), "aligned"), (dict(weight=None), "aligned"), (dict(sum=None), "sum"), (dict(residual=None), "sum"),
    (dict(residual=BUF + 8), "aligned"), (dict(sum=BUF + 8), "aligned"), (dict(cols=40), "multiple of 16"),
    (dict(rows=0), "rows"), (dict(cols=32784), "32768"),
])
def test_rmsnorm_blocks_refuses(lib, change, word):
    a = dict(x=BUF, residual=BUF, weight=BUF, rows=4, cols=256, sum=BUF, q=BUF, inv=BUF) | change
    refused(lib, lib.xaxb_rmsnorm_blocks(CTX, None, a["x"], a["residual"], a["weight"], 1e-6, a["rows"], a["cols"], a["sum"],
                                         a["q"], a["inv"]), word)


@pytest.mark.parametrize("change,word", [
    (dict(gu=BUF + 8), "aligned"), (dict(ld=500), "ld"), (dict(ld=516), "ld"), (dict(dim=24, ld=48), "multiple of 16"),
    (dict(rows=0), "rows"), (dict(dim=0), "multiple of 16"),
])
def test_silu_mul_blocks_refuses(lib, change, word):
    a = dict(gu=BUF, ld=512, rows=4, dim=256, q=BUF, inv=BUF) | change
    refused(lib, lib.xaxb_silu_mul_blocks(CTX, None, a["gu"], a["ld"], a["rows"], a["dim"], a["q"], a["inv"]), word)


@pytest.mark.parametrize("change,word", [
    (dict(a=None), "null"), (dict(b_inv=None), "null"), (dict(M=0), "non-positive"), (dict(K=0), "non-positive"),
    (dict(K=264, lda=272, ldb=272), "multiples of 16"), (dict(lda=264), "multiples of 16"), (dict(ldb=240), "row strides"),
    (dict(N=100), "of 8"), (dict(ldo=252), "of 8"), (dict(ldo=248), "row strides"), (dict(ldr=8), "row strides"),
    (dict(a=BUF + 8), "aligned"), (dict(out=BUF + 8), "aligned"), (dict(bias=BUF + 2), "aligned"),
    (dict(M=(1 << 30) + 1), "M"),
])
def test_gemm_fp8_blocks_refuses(lib, change, word):
    a = dict(a=BUF, lda=256, a_inv=BUF, b=BUF, ldb=256, b_inv=BUF, M=4, N=256, K=256, bias=BUF, residual=BUF, ldr=256, out=BUF,
             ldo=256) | change
    refused(lib, lib.xaxb_gemm_fp8_blocks(CTX, None, a["a"], a["lda"], a["a_inv"], a["b"], a["ldb"], a["b_inv"], a["M"], a["N"],
                                          a["K"], a["bias"], a["residual"], a["ldr"], a["out"], a["ldo"]), word)


def test_wrappers_refuse_cpu_tensors():
    import torch

    from xax_b200 import ops

    x, w = torch.zeros((4, 256), dtype=torch.bfloat16), torch.zeros((256,), dtype=torch.bfloat16)
    q, inv = torch.zeros((4, 256), dtype=torch.float8_e4m3fn), torch.ones((4, 2))
    for call in (lambda: ops.quantize_blocks(x), lambda: ops.rmsnorm_blocks(x, w, 1e-6), lambda: ops.silu_mul_blocks(x, 128),
                 lambda: ops.gemm_fp8_blocks(q, q, inv, inv)):
        with pytest.raises(ValueError, match="CUDA"):
            call()
