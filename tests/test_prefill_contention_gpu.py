"""Prefill attention whose loads are held up: its loader may come late to any barrier, by more than a tile, and must neither
miss a phase nor change a bit of the result."""

import pytest
import torch

pytestmark = pytest.mark.gpu

BF16 = torch.bfloat16


@pytest.mark.parametrize("head_dim", [64, 128])
def test_prefill_beside_copies(head_dim):
    from xax_b200 import _lib, ops

    B, T, Hq, Hkv = 2, 1000, 16, 4
    gen = torch.Generator(device="cuda").manual_seed(head_dim)

    def rand(*shape):
        return torch.randn(shape, generator=gen, device="cuda").to(BF16)

    q, k, v = rand(B * T, Hq, head_dim), rand(B, 1024, Hkv, head_dim), rand(B, 1024, Hkv, head_dim)
    pos = torch.zeros((B,), dtype=torch.int32, device="cuda")
    want = ops.attn_prefill(q, k, v, pos, B, T)
    src, dst = (torch.zeros((64 << 20,), device="cuda") for _ in range(2))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for _ in range(60):
            dst.copy_(src)
    outs = [ops.attn_prefill(q, k, v, pos, B, T) for _ in range(100)]
    torch.cuda.synchronize()
    _lib.device_status()
    for out in outs:
        assert torch.equal(out, want)
