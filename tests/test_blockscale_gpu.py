"""Block-scaled FP8 operators against plain implementations in 64 bits.

Tolerances.  A value cast to e4m3 is off by at most half a step: 2^-4 of itself, or 2^-10 of the multiplier where e4m3 is
subnormal (its smallest step is 2^-9).  The float32 arithmetic in front of the cast may move the value, and the
multiplier, by a relative ``d`` that is counted per operator:

* plain cast: inv = fl(amax * fl(1/448)) is two roundings, 1/inv and the product with it one each: d = 4 * 2^-24;
* RMSNorm: at most 64 squares summed in sequence per thread and ten additions across threads, each 2^-24 of a sum of
  positive numbers, halved by the square root; then a division, an addition, rsqrt (2 units) and two products, and the
  plain cast: d = (37 + 2 * 2 + 5 + 4) * 2^-24 < 2^-18;
* SiLU * up: exp (2 units), an addition, a division (2 units), a product, and the plain cast: d < 16 * 2^-24 = 2^-20;
* product: K additions of exact products, each off by at most one unit of the running sum (the tensor core may cut off
  instead of rounding), 2^-23 of the sum of magnitudes; two roundings of the combined multiplier and one for each block's
  addition; the result is rounded to bf16 once, 2^-8 of itself (with the same of the error).
"""

import pytest
import torch

pytestmark = pytest.mark.gpu

BF16, E4M3, F64 = torch.bfloat16, torch.float8_e4m3fn, torch.float64
D_CAST, D_NORM, D_SILU = 4 * 2.0**-24, 2.0**-18, 2.0**-20


def blocks(n):
    return -(-n // 128)


def gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def activations(rows, cols, seed, scale=1.0):
    x = torch.randn((rows, cols), generator=gen(seed), device="cuda")
    x[:, :: max(1, cols // 7)] *= 30.0
    return (x * scale).to(BF16)


def spread(inv, block_rows, shape):
    """inv per element, float64."""
    return inv.to(F64).repeat_interleave(block_rows, 0)[: shape[0]].repeat_interleave(128, 1)[:, : shape[1]]


def block_amax(y, block_rows):
    rows, cols = y.shape
    v = torch.zeros((-(-rows // block_rows) * block_rows, blocks(cols) * 128), dtype=F64, device=y.device)
    v[:rows, :cols] = y.abs()
    return v.reshape(-1, block_rows, blocks(cols), 128).amax(dim=(1, 3))


def check_cast(y, q, inv, block_rows, d):
    """(q, inv) is the cast of the float64 values y."""
    rows, cols = y.shape
    assert q.dtype == E4M3 and q.shape == (rows, cols) and inv.dtype == torch.float32
    assert inv.shape == (-(-rows // block_rows), blocks(cols))
    amax = block_amax(y, block_rows)
    want = torch.where(amax > 0, torch.clamp(amax / 448.0, min=2.0**-126), torch.ones_like(amax))
    assert ((inv.to(F64) - want).abs() <= (d + 2.0**-24) * want).all()
    s = spread(inv, block_rows, y.shape)
    off = (q.to(F64) * s - y).abs()
    assert (off <= torch.maximum(2.0**-4 * y.abs(), 2.0**-10 * s) * (1 + 4 * d) + 2 * d * y.abs()).all(), float(off.max())


def plain_cast32(x, block_rows):
    """The definition in float32, operation by operation: the kernel's bits."""
    rows, cols = x.shape
    v = torch.zeros((-(-rows // block_rows) * block_rows, blocks(cols) * 128), device=x.device)
    v[:rows, :cols] = x.float()
    v = v.reshape(-1, block_rows, blocks(cols), 128)
    amax = v.abs().amax(dim=(1, 3))
    inv = torch.clamp(amax * torch.tensor(1.0 / 448.0, device=x.device), min=2.0**-126)
    inv = torch.where((amax > 0) & torch.isfinite(amax), inv, torch.ones_like(inv))
    q = torch.clamp(v * (1.0 / inv)[:, None, :, None], -448, 448).to(E4M3)
    return q.reshape(-1, blocks(cols) * 128)[:rows, :cols], inv


def same_bytes(q, want):
    nan = want.float().isnan()
    assert torch.equal(q.float().isnan(), nan)
    assert torch.equal(q.view(torch.uint8)[~nan], want.contiguous().view(torch.uint8)[~nan])


# ---------------------------------------------------------------------------------------
# cast


@pytest.mark.parametrize("block_rows", [1, 128])
@pytest.mark.parametrize("rows,cols", [(1, 16), (1, 128), (3, 144), (7, 4096), (128, 256), (129, 272), (333, 5648), (1024, 2048)])
def test_quantize_blocks(rows, cols, block_rows):
    from xax_b200 import ops

    x = activations(rows, cols, rows + cols)
    q, inv = ops.quantize_blocks(x, block_rows)
    check_cast(x.to(F64), q, inv, block_rows, D_CAST)
    want_q, want_inv = plain_cast32(x, block_rows)
    assert torch.equal(inv, want_inv)
    same_bytes(q, want_q)


@pytest.mark.parametrize("block_rows", [1, 128])
def test_quantize_blocks_special_values(block_rows):
    """Zero, infinite and NaN blocks keep a multiplier of 1; tiny and huge ones stay finite; neighbours are untouched."""
    from xax_b200 import ops

    x = activations(256, 128 * 9, 5)
    big = float(torch.finfo(BF16).max)
    tiny = 2.0**-133  # the smallest bf16 subnormal
    for i, fill in enumerate((0.0, float("inf"), float("nan"), big, tiny, 2.0**-118, -0.0)):
        blk = x[:128, i * 128:(i + 1) * 128]
        if fill != fill or fill in (float("inf"),):
            blk[5, 7] = fill  # one such value among ordinary ones (some above 448)
            blk[5, 8] = 1000.0
        else:
            blk.fill_(fill)
    q, inv = ops.quantize_blocks(x, block_rows)
    want_q, want_inv = plain_cast32(x, block_rows)
    assert torch.equal(inv, want_inv) and torch.isfinite(inv).all()
    same_bytes(q, want_q)
    assert (inv[0, 0] == 1) and not q[:128, :128].float().any()
    row = 5 if block_rows == 1 else 0
    assert inv[row, 1] == 1 and inv[row, 2] == 1
    assert q[5, 128 + 7].float() == 448 and q[5, 128 + 8].float() == 448 and q[5, 256 + 7].float().isnan()
    assert q[0, 3 * 128].float() == 448
    fine = torch.ones_like(x, dtype=torch.bool)
    fine[:128, 128:384] = False
    y = torch.where(fine, x.to(F64), 0.0)
    s = spread(inv, block_rows, x.shape)
    off = ((q.to(F64) * s) - y).abs()[fine]
    lim = (torch.maximum(2.0**-4 * y.abs(), 2.0**-10 * s) * (1 + 2.0**-20))[fine]
    assert (off <= lim).all()


# ---------------------------------------------------------------------------------------
# RMSNorm and SiLU * up


@pytest.mark.parametrize("with_residual", [False, True])
@pytest.mark.parametrize("rows,cols", [(1, 16), (5, 128), (3, 2000), (64, 2048), (17, 4096), (9, 5648), (130, 8192), (3, 16384),
                                       (2, 32768)])
def test_rmsnorm_blocks(rows, cols, with_residual):
    from xax_b200 import ops

    x = activations(rows, cols, 1)
    r = activations(rows, cols, 2, 0.5) if with_residual else None
    w = (1 + 0.1 * torch.randn((cols,), generator=gen(3), device="cuda")).to(BF16)
    total, q, inv = ops.rmsnorm_blocks(x, w, 1e-6, residual=r)
    t = x.to(F64) if r is None else x.to(F64) + r.to(F64)
    if r is None:
        assert total is None
    else:
        assert torch.equal(total, (x.float() + r.float()).to(BF16))
    y = t * torch.rsqrt((t * t).mean(dim=1, keepdim=True) + 1e-6) * w.to(F64)
    # x + residual in float32 is off by 2^-24 of itself where the two are far apart
    check_cast(y, q, inv, 1, D_NORM + 2.0**-24)


def test_rmsnorm_blocks_rows_stand_alone():
    """A zero row stays zero (its multipliers 1), a NaN row does not reach its neighbours, tiny rows do not divide by zero."""
    from xax_b200 import ops

    x = activations(6, 512, 4)
    x[1] = 0
    x[2, 3] = float("nan")
    x[3] = 2.0**-100
    w = torch.ones((512,), dtype=BF16, device="cuda")
    _, q, inv = ops.rmsnorm_blocks(x, w, 1e-6)
    assert not q[1].float().any() and (inv[1] == 1).all()
    assert q[2].float().isnan().all()
    keep = [0, 3, 4, 5]
    t = x[keep].to(F64)
    check_cast(t * torch.rsqrt((t * t).mean(1, keepdim=True) + 1e-6), q[keep], inv[keep], 1, D_NORM)


@pytest.mark.parametrize("rows,dim", [(1, 16), (2, 128), (5, 2000), (128, 14336), (33, 5632), (700, 272)])
def test_silu_mul_blocks(rows, dim):
    from xax_b200 import ops

    gu = activations(rows, 2 * dim, rows, 2.0)
    q, inv = ops.silu_mul_blocks(gu, dim)
    g, u = gu[:, :dim].to(F64), gu[:, dim:].to(F64)
    check_cast(g * torch.sigmoid(g) * u, q, inv, 1, D_SILU)


def test_silu_mul_blocks_extreme_gates():
    """Gates whose exponential overflows give zero (negative) or pass up through (positive); zeros stay zero."""
    from xax_b200 import ops

    dim = 256
    gu = torch.zeros((2, 2 * dim), dtype=BF16, device="cuda")
    gu[0, :8] = torch.tensor([-1e30, -200.0, -100.0, -88.0, 0.0, 88.0, 200.0, 3e4], device="cuda").to(BF16)
    gu[0, dim:dim + 8] = 1.0
    q, inv = ops.silu_mul_blocks(gu, dim)
    got = q[0, :8].to(F64) * inv[0, 0].to(F64)
    assert not got[:5].any() and torch.isfinite(got).all()
    assert abs(float(got[7]) / float(gu[0, 7]) - 1) <= 2.0**-4
    assert not q[1].float().any() and (inv[1] == 1).all() and inv[0, 1] == 1


# ---------------------------------------------------------------------------------------
# product


def operands(M, N, K, seed):
    from xax_b200 import ops

    a_q, a_inv = ops.quantize_blocks(activations(M, K, seed))
    b_q, b_inv = ops.quantize_blocks(activations(N, K, seed + 1, 0.02), 128)
    return a_q, a_inv, b_q, b_inv


def check_product(out, a_q, a_inv, b_q, b_inv, bias=None, residual=None):
    M, K = a_q.shape
    N = b_q.shape[0]
    a, b = a_q.to(F64) * spread(a_inv, 1, (M, K)), b_q.to(F64) * spread(b_inv, 128, (N, K))
    want, size = a @ b.T, a.abs() @ b.abs().T
    for t in (bias, residual):
        if t is not None:
            want, size = want + t.to(F64), size + t.to(F64).abs()
    assert out.dtype == BF16 and out.shape == (M, N)
    err = (K + blocks(K) + 4) * 2.0**-23 * size
    off = (out.to(F64) - want).abs()
    assert (off <= err * (1 + 2.0**-8) + 2.0**-8 * want.abs()).all(), float((off - err - 2.0**-8 * want.abs()).max())
    # the bound above is a worst case over the order of the sum; errors of independent additions stay far below it
    assert float((out.to(F64) - want).norm() / want.norm()) < 3e-3  # uniform bf16 rounding: 2^-8 / sqrt(3) = 2.3e-3 at most


SHAPES = [(1, 8, 16), (1, 128, 128), (1, 4096, 2048), (2, 256, 144), (5, 2504, 5648), (15, 512, 1024), (16, 1000, 4096),
          (17, 2048, 5632), (33, 640, 384), (64, 2048, 5632), (65, 392, 2064), (100, 4096, 1024), (128, 6144, 4096),
          (129, 256, 512), (200, 1288, 1040), (256, 4096, 4096), (333, 2504, 5648), (500, 5632, 2048), (1000, 264, 528),
          (1024, 11264, 2048), (2048, 8192, 2048), (2500, 2056, 656)]


@pytest.mark.parametrize("M,N,K", SHAPES)
def test_gemm_fp8_blocks(M, N, K):
    from xax_b200 import _lib, ops

    a_q, a_inv, b_q, b_inv = operands(M, N, K, M + N)
    bias = torch.randn((N,), generator=gen(7), device="cuda").to(BF16)
    residual = activations(M, N, 8)
    check_product(ops.gemm_fp8_blocks(a_q, b_q, a_inv, b_inv), a_q, a_inv, b_q, b_inv)
    out = ops.gemm_fp8_blocks(a_q, b_q, a_inv, b_inv, bias, residual)
    check_product(out, a_q, a_inv, b_q, b_inv, bias, residual)
    assert torch.equal(out, ops.gemm_fp8_blocks(a_q, b_q, a_inv, b_inv, bias, residual))  # no order of sums is left to chance
    _lib.device_status()


@pytest.mark.parametrize("M,N,K", [(1, 256, 512), (20, 2504, 1040), (128, 4096, 1024), (300, 512, 640), (2048, 4096, 512)])
def test_gemm_fp8_blocks_exact_integers(M, N, K):
    """Small integers with power-of-two multipliers: products and sums are exact in float32, so the result is the
    bf16 rounding of the integer result and every multiplier has to sit on its own block."""
    from xax_b200 import ops

    g = gen(M)
    a = torch.randint(-2, 3, (M, K), generator=g, device="cuda").float()
    b = torch.randint(-2, 3, (N, K), generator=g, device="cuda").float()
    a_inv = torch.exp2(torch.randint(-3, 4, (M, blocks(K)), generator=g, device="cuda").float())
    b_inv = torch.exp2(torch.randint(-3, 4, (blocks(N), blocks(K)), generator=g, device="cuda").float())
    out = ops.gemm_fp8_blocks(a.to(E4M3), b.to(E4M3), a_inv, b_inv)
    want = (a.to(F64) * spread(a_inv, 1, a.shape)) @ (b.to(F64) * spread(b_inv, 128, b.shape)).T
    assert torch.equal(out, want.float().to(BF16))


@pytest.mark.parametrize("M", [3, 130, 1030])
def test_gemm_fp8_blocks_strides_and_guard(M):
    """Row strides wider than the rows on every side; nothing beside the result is written."""
    from xax_b200 import ops

    N, K = 392, 656
    a_q, a_inv, b_q, b_inv = operands(M, N, K, 3)
    wide = lambda t, extra: torch.empty((t.shape[0], t.shape[1] + extra), dtype=t.dtype, device="cuda")  # noqa: E731
    a_w, b_w = wide(a_q, 48).view(torch.uint8).fill_(0x7F).view(E4M3), wide(b_q, 16).view(torch.uint8).fill_(0x7F).view(E4M3)
    a_w.view(torch.uint8)[:, :K], b_w.view(torch.uint8)[:, :K] = a_q.view(torch.uint8), b_q.view(torch.uint8)
    residual = activations(M, N + 24, 5)
    out = torch.full((M + 2, N + 16), 7.0, dtype=BF16, device="cuda")
    view = out[1:M + 1, 8:8 + N]
    got = ops.gemm_fp8_blocks(a_w[:, :K], b_w[:, :K], a_inv, b_inv, None, residual[:, :N], out=view)
    assert got.data_ptr() == view.data_ptr()
    check_product(view, a_q, a_inv, b_q, b_inv, None, residual[:, :N])
    out[1:M + 1, 8:8 + N] = 7.0
    assert (out == 7.0).all()


@pytest.mark.parametrize("M", [4, 300])
def test_gemm_fp8_blocks_special_values(M):
    """NaN in a row of A or B reaches that row or column alone, zero multipliers give zero, sums that pass bf16 are infinite."""
    from xax_b200 import ops

    N, K = 264, 384
    a_q, a_inv, b_q, b_inv = operands(M, N, K, 9)
    a_q.view(torch.uint8)[1, 5] = 0x7F
    b_q.view(torch.uint8)[9, 300] = 0x7F
    a_inv[2] = 0.0
    a_inv[3] = 3e38
    out = ops.gemm_fp8_blocks(a_q, b_q, a_inv, b_inv)
    nan = out.float().isnan()
    assert nan[1].all() and nan[:, 9].all()
    nan[1], nan[:, 9] = False, False
    nan[3] = False
    assert not nan.any()
    keep = torch.ones((N,), dtype=torch.bool, device="cuda")
    keep[9] = False
    assert not out[2][keep].any()
    rows = [r for r in range(M) if r not in (1, 2, 3)]
    a = a_q[rows].to(F64) * spread(a_inv[rows], 1, (len(rows), K))
    b = (b_q.to(F64) * spread(b_inv, 128, (N, K)))[keep]
    off = (out[rows][:, keep].to(F64) - a @ b.T).abs()
    assert (off <= 2 * (K + 8) * 2.0**-23 * (a.abs() @ b.abs().T) + 2.0**-8 * (a @ b.T).abs()).all()


# ---------------------------------------------------------------------------------------
# all of them, as a layer uses them


def mlp(ops, x, delta, w, gate_up, down):
    total, q, inv = ops.rmsnorm_blocks(x, w, 1e-6, residual=delta)
    gu = ops.gemm_fp8_blocks(q, gate_up[0], inv, gate_up[1])
    hq, h_inv = ops.silu_mul_blocks(gu, gate_up[0].shape[0] // 2)
    out = ops.gemm_fp8_blocks(hq, down[0], h_inv, down[1], None, total)
    return total, q, inv, gu, hq, h_inv, out


@pytest.mark.parametrize("tokens,H,F", [(1, 2048, 5632), (37, 1024, 1424), (600, 2048, 5632)])
def test_mlp_chain_eager_and_captured(tokens, H, F):
    """The MLP half of a block: every stage against 64 bits on what the stage before it gave; then the same calls captured
    into a graph, replayed on new inputs while eager calls run between, with the eager bits."""
    from xax_b200 import _lib, ops

    x, delta = activations(tokens, H, 1), activations(tokens, H, 2)
    w = (1 + 0.1 * torch.randn((H,), generator=gen(3), device="cuda")).to(BF16)
    gate_up = ops.quantize_blocks(activations(2 * F, H, 4, 0.02), 128)
    down = ops.quantize_blocks(activations(H, F, 5, 0.02), 128)
    total, q, inv, gu, hq, h_inv, out = mlp(ops, x, delta, w, gate_up, down)
    t = x.to(F64) + delta.to(F64)
    check_cast(t * torch.rsqrt((t * t).mean(1, keepdim=True) + 1e-6) * w.to(F64), q, inv, 1, D_NORM + 2.0**-24)
    check_product(gu, q, inv, *gate_up)
    g, u = gu[:, :F].to(F64), gu[:, F:].to(F64)
    check_cast(g * torch.sigmoid(g) * u, hq, h_inv, 1, D_SILU)
    check_product(out, hq, h_inv, *down, None, total)

    xs, ds = x.clone(), delta.clone()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        mlp(ops, xs, ds, w, gate_up, down)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured = mlp(ops, xs, ds, w, gate_up, down)
    for seed in (11, 12):
        x2, d2 = activations(tokens, H, seed), activations(tokens, H, seed + 50)
        xs.copy_(x2), ds.copy_(d2)
        graph.replay()
        want = mlp(ops, x2, d2, w, gate_up, down)
        for got, exp in zip(captured, want):
            assert torch.equal(got.view(torch.uint8), exp.view(torch.uint8))
    _lib.device_status()


def test_two_streams_at_once():
    """The operators keep no state between calls: two streams interleave without touching each other's results."""
    from xax_b200 import ops

    work = [operands(64, 2048, 4096, s) for s in (1, 2)]
    want = [ops.gemm_fp8_blocks(a, b, ai, bi) for a, ai, b, bi in work]
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    torch.cuda.synchronize()
    got = [[], []]
    for _ in range(20):
        for i, (a, ai, b, bi) in enumerate(work):
            with torch.cuda.stream(streams[i]):
                got[i].append(ops.gemm_fp8_blocks(a, b, ai, bi))
    torch.cuda.synchronize()
    for i in range(2):
        assert all(torch.equal(g, want[i]) for g in got[i])


def test_offsets_past_32_bits():
    """Tensors of more than 2^31 values: the last rows come out as they do alone."""
    from xax_b200 import ops

    def tail_matches(whole, part):
        for w, p in zip(whole, part):
            assert torch.equal(w[-p.shape[0]:].view(torch.uint8), p.view(torch.uint8))

    rows, cols, last = 131100, 16416, 5  # 2.15e9 values; a width that is no multiple of 128
    x = torch.empty((rows, cols), dtype=BF16, device="cuda")
    x[:-last] = 1.0
    x[-last:] = activations(last, cols, 1)
    end = x[-last:].clone()
    tail_matches(ops.quantize_blocks(x), ops.quantize_blocks(end))
    w = torch.ones((cols,), dtype=BF16, device="cuda")
    tail_matches(ops.rmsnorm_blocks(x, w, 1e-6, residual=x), ops.rmsnorm_blocks(end, w, 1e-6, residual=end))
    tail_matches(ops.silu_mul_blocks(x, cols // 2), ops.silu_mul_blocks(end, cols // 2))
    del x
    M, N, K = 262300, 8200, 144  # 2.15e9 results
    a_q, a_inv, b_q, b_inv = operands(300, N, K, 1)
    big_q, big_inv = a_q.view(torch.uint8)[:1].expand(M, K).contiguous().view(E4M3), a_inv[:1].expand(M, 2).contiguous()
    big_q.view(torch.uint8)[-300:], big_inv[-300:] = a_q.view(torch.uint8), a_inv
    residual = torch.ones((M, N), dtype=BF16, device="cuda")
    out = ops.gemm_fp8_blocks(big_q, b_q, big_inv, b_inv, None, residual)
    check_product(out[-300:], a_q, a_inv, b_q, b_inv, None, residual[-300:])
    check_product(out[:2], big_q[:2], big_inv[:2], b_q, b_inv, None, residual[:2])


# ---------------------------------------------------------------------------------------
# refusals and small calls


def test_empty_and_copied_inputs():
    from xax_b200 import ops

    x = torch.empty((0, 256), dtype=BF16, device="cuda")
    q, inv = ops.quantize_blocks(x)
    assert q.shape == (0, 256) and inv.shape == (0, 2)
    w = torch.ones((256,), dtype=BF16, device="cuda")
    assert ops.rmsnorm_blocks(x, w, 1e-6, residual=x)[0].shape == (0, 256)
    assert ops.silu_mul_blocks(x, 128)[0].shape == (0, 128)
    b_q, b_inv = ops.quantize_blocks(activations(264, 256, 1), 128)
    assert ops.gemm_fp8_blocks(q, b_q, inv, b_inv).shape == (0, 264)
    # a transposed or sliced input is copied, like the other operators do it
    y = activations(256, 64, 3)
    odd = y.reshape(-1)[4:4 + 512].reshape(2, 256)  # contiguous, 8 bytes off the boundary that the kernels load at
    for view in (y.t(), y[:, 16:48], activations(8, 512, 4)[:, ::2], odd):
        got, want = ops.quantize_blocks(view), ops.quantize_blocks(view.contiguous())
        same_bytes(got[0], want[0])
        assert torch.equal(got[1], want[1])
    w = torch.ones((257,), dtype=BF16, device="cuda")
    for got, want in zip(ops.rmsnorm_blocks(odd, w[1:], 1e-6, residual=odd),
                         ops.rmsnorm_blocks(odd.clone(), w[:256], 1e-6, residual=odd.clone())):
        assert torch.equal(got.view(torch.uint8), want.view(torch.uint8))
    for got, want in zip(ops.silu_mul_blocks(odd, 128), ops.silu_mul_blocks(odd.clone(), 128)):
        assert torch.equal(got.view(torch.uint8), want.view(torch.uint8))


def test_arguments_are_checked():
    from xax_b200 import ops

    x = activations(4, 256, 1)
    w = torch.ones((256,), dtype=BF16, device="cuda")
    a_q, a_inv = ops.quantize_blocks(x)
    b_q, b_inv = ops.quantize_blocks(activations(264, 256, 2), 128)
    bad = [
        lambda: ops.quantize_blocks(x.float()), lambda: ops.quantize_blocks(x[0]), lambda: ops.quantize_blocks(x, 64),
        lambda: ops.quantize_blocks(x[:, :24].contiguous()), lambda: ops.quantize_blocks(x[:, :0]),
        lambda: ops.rmsnorm_blocks(x, w[:128], 1e-6), lambda: ops.rmsnorm_blocks(x, w.float(), 1e-6),
        lambda: ops.rmsnorm_blocks(x, w, 1e-6, residual=x[:2]),
        lambda: ops.silu_mul_blocks(x, 256), lambda: ops.silu_mul_blocks(x, 0), lambda: ops.silu_mul_blocks(x, 100),
        lambda: ops.gemm_fp8_blocks(x, b_q, a_inv, b_inv), lambda: ops.gemm_fp8_blocks(a_q, b_q, a_inv[:, :1], b_inv),
        lambda: ops.gemm_fp8_blocks(a_q, b_q, a_inv, b_inv[:1]), lambda: ops.gemm_fp8_blocks(a_q[:, :128], b_q, a_inv, b_inv),
        lambda: ops.gemm_fp8_blocks(a_q, b_q, a_inv.double(), b_inv),
        lambda: ops.gemm_fp8_blocks(a_q, b_q, a_inv, b_inv, w), lambda: ops.gemm_fp8_blocks(a_q, b_q, a_inv, b_inv, None, x),
        lambda: ops.gemm_fp8_blocks(a_q, b_q[:260], a_inv, b_inv),  # N not a multiple of 8
        lambda: ops.gemm_fp8_blocks(a_q, b_q, a_inv, b_inv, out=torch.empty((4, 264), device="cuda")),
        lambda: ops.gemm_fp8_blocks(a_q.cpu(), b_q, a_inv, b_inv),
    ]
    for call in bad:
        with pytest.raises(ValueError):
            call()


def test_silu_mul_blocks_where_the_sigmoid_is_denormal():
    """Gates from -87.3 down have a sigmoid below the smallest normal float32; their product with a large up counts."""
    from xax_b200 import ops

    gu = torch.empty((4, 512), dtype=BF16, device="cuda")
    gu[:, :256] = torch.linspace(-88.5, -84.0, 256, device="cuda")  # (e^88.5 is the last that float32 holds)
    gu[:, 256:] = torch.tensor([1.0, 1e10, 1e30, 3e38], device="cuda")[:, None]
    q, inv = ops.silu_mul_blocks(gu, 256)
    g, u = gu[:, :256].to(F64), gu[:, 256:].to(F64)
    check_cast(g * torch.sigmoid(g) * u, q, inv, 1, D_SILU)
