"""Cases of the block-scaled FP8 operators: what a linear layer with one scale per block of 128 is made of.

A block-scaled tensor is a pair: e4m3 values ``q`` and float32 multipliers ``inv``, one per block, so that the tensor
stands for ``q * inv``.  Activations [rows, cols] have a block per row and 128 columns, weights [out, in] one per 128 x
128 square; the last block of a row or column of blocks may be smaller.

  cast   bf16 [rows, cols] -> (q, inv)
  norm   RMSNorm of x (+ residual), cast -> (x + residual in bf16, q, inv)
  silu   silu(gate) * up, cast -> (q, inv)
  gemm   (q_a, inv_a) [M, K] times (q_b, inv_b) [N, K], transposed, + bias + residual -> bf16 [M, N]
"""

import torch

own = False

BLOCK = 128
TOP = 448.0  # the largest e4m3 value
EPS = 1e-6


def listed():
    return [
        # the attention output of one decode step of 16 sequences, cast for the output projection: the smallest call
        {"name": "cast_decode_16", "op": "cast", "rows": 16, "cols": 4096, "block_rows": 1},
        # the same cast for a prefill of 8192 tokens
        {"name": "cast_prefill_8192", "op": "cast", "rows": 8192, "cols": 4096, "block_rows": 1},
        # one gate weight, cast when a bf16 model is loaded
        {"name": "cast_weight", "op": "cast", "rows": 14336, "cols": 4096, "block_rows": 128},
        # gate | up of one sequence's next token: all of the weight is read for one row
        {"name": "gemm_decode_1", "op": "gemm", "m": 1, "n": 28672, "k": 4096, "bias": False, "residual": False},
        # down projection of a decode step of 64 sequences of a small model
        {"name": "gemm_decode_64", "op": "gemm", "m": 64, "n": 2048, "k": 5632, "bias": False, "residual": True},
        # down projection of a decode step of 128 sequences
        {"name": "gemm_decode_128", "op": "gemm", "m": 128, "n": 4096, "k": 14336, "bias": False, "residual": True},
        # a ragged prompt against a weight whose last blocks are cut off on both sides
        {"name": "gemm_ragged", "op": "gemm", "m": 333, "n": 2504, "k": 5648, "bias": True, "residual": False},
        # gate | up of a prefill of 4096 tokens: the largest product of a layer
        {"name": "gemm_prefill_4096", "op": "gemm", "m": 4096, "n": 28672, "k": 4096, "bias": False, "residual": False},
        # the norm between attention and MLP in a decode step of 64 sequences of a small model
        {"name": "norm_decode_64", "op": "norm", "rows": 64, "cols": 2048, "residual": True},
        # the same norm in a prefill of 8192 tokens
        {"name": "norm_prefill_8192", "op": "norm", "rows": 8192, "cols": 4096, "residual": True},
        # between gate | up and down in a decode step of 128 sequences
        {"name": "silu_decode_128", "op": "silu", "rows": 128, "cols": 14336},
        # the same in a prefill whose number of tokens is odd
        {"name": "silu_prefill_4099", "op": "silu", "rows": 4099, "cols": 5632},
    ]


def _spread(rng, lo, hi):
    """A whole number in lo .. hi, even over the logarithm."""
    return max(lo, min(hi, int(round(lo * (hi / lo) ** rng.random()))))


def draw(rng):
    op = rng.choice(["cast", "gemm", "gemm", "norm", "silu"])
    if op == "gemm":
        while True:
            m, n, k = _spread(rng, 1, 4096), 8 * _spread(rng, 16, 3584), 16 * _spread(rng, 8, 896)
            if m * n * k <= 4096 * 28672 * 4096:
                return {"op": op, "m": m, "n": n, "k": k, "bias": rng.random() < 0.5, "residual": rng.random() < 0.5}
    if op == "norm":
        return {"op": op, "rows": _spread(rng, 1, 8192), "cols": 16 * _spread(rng, 16, 512), "residual": rng.random() < 0.7}
    if op == "silu":
        return {"op": op, "rows": _spread(rng, 1, 4099), "cols": 16 * _spread(rng, 16, 896)}
    return {"op": op, "rows": _spread(rng, 1, 8192), "cols": 16 * _spread(rng, 16, 896), "block_rows": rng.choice([1, 1, 128])}


def _blocks(n):
    return -(-n // BLOCK)


def _activations(gen, rows, cols):
    """Unit-scale activations with a few channels that stick out, as a residual stream has them."""
    x = torch.randn((rows, cols), generator=gen, device="cuda")
    gain = torch.exp(0.5 * torch.randn((cols,), generator=gen, device="cuda"))
    gain[torch.rand((cols,), generator=gen, device="cuda") < 0.002] *= 20.0
    return (x * gain).to(torch.bfloat16)


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    op = case["op"]
    if op == "gemm":
        m, n, k = case["m"], case["n"], case["k"]
        a_q, a_inv = _plain_cast(_activations(gen, m, k), 1)
        b_q, b_inv = _plain_cast((0.02 * torch.randn((n, k), generator=gen, device="cuda")).to(torch.bfloat16), BLOCK)
        bias = (0.1 * torch.randn((n,), generator=gen, device="cuda")).to(torch.bfloat16) if case["bias"] else None
        residual = _activations(gen, m, n) if case["residual"] else None
        return {"op": op, "a_q": a_q, "a_inv": a_inv, "b_q": b_q, "b_inv": b_inv, "bias": bias, "residual": residual}
    rows, cols = case["rows"], case["cols"]
    if op == "norm":
        residual = _activations(gen, rows, cols) if case["residual"] else None
        weight = (1.0 + 0.1 * torch.randn((cols,), generator=gen, device="cuda")).to(torch.bfloat16)
        return {"op": op, "x": _activations(gen, rows, cols), "residual": residual, "weight": weight}
    if op == "silu":
        return {"op": op, "gate_up": _activations(gen, rows, 2 * cols), "cols": cols}
    x = _activations(gen, rows, cols)
    if case["block_rows"] == BLOCK:
        x = x * 0.02
    return {"op": op, "x": x, "block_rows": case["block_rows"]}


def _plain_cast(x, block_rows):
    """q = e4m3(x / inv), inv = max|x| / 448 of the block (1 where the maximum is 0 or not finite)."""
    rows, cols = x.shape
    down, right = -(-rows // block_rows), _blocks(cols)
    v = torch.nn.functional.pad(x.float(), (0, right * BLOCK - cols, 0, down * block_rows - rows))
    v = v.reshape(down, block_rows, right, BLOCK)
    amax = v.abs().amax(dim=(1, 3))
    inv = torch.clamp(amax * (1.0 / TOP), min=2.0**-126)
    inv = torch.where((amax > 0) & torch.isfinite(amax), inv, torch.ones_like(inv))
    q = torch.clamp(v * (1.0 / inv)[:, None, :, None], -TOP, TOP).to(torch.float8_e4m3fn)
    return q.reshape(down * block_rows, right * BLOCK)[:rows, :cols].contiguous(), inv


def _plain(state):
    op = state["op"]
    if op == "gemm":
        a_q, b_q = state["a_q"], state["b_q"]
        k, n = a_q.shape[1], b_q.shape[0]
        a = a_q.float() * state["a_inv"].repeat_interleave(BLOCK, dim=1)[:, :k]
        b = b_q.float() * state["b_inv"].repeat_interleave(BLOCK, dim=1)[:, :k].repeat_interleave(BLOCK, dim=0)[:n]
        out = a @ b.t()
        if state["bias"] is not None:
            out = out + state["bias"].float()
        if state["residual"] is not None:
            out = out + state["residual"].float()
        return out.to(torch.bfloat16)
    if op == "norm":
        x = state["x"].float()
        if state["residual"] is not None:
            x = x + state["residual"].float()
        y = x * torch.rsqrt((x * x).mean(dim=1, keepdim=True) + EPS) * state["weight"].float()
        q, inv = _plain_cast(y, 1)
        return {"q": q, "inv": inv} if state["residual"] is None else {"sum": x.to(torch.bfloat16), "q": q, "inv": inv}
    if op == "silu":
        gate, up = state["gate_up"].float().split(state["cols"], dim=1)
        return _plain_cast(gate / (1.0 + torch.exp(-gate)) * up, 1)
    return _plain_cast(state["x"], state["block_rows"])


def run(state):
    if own:
        from xax_b200 import ops

        op = state["op"]
        if op == "gemm":
            return ops.gemm_fp8_blocks(state["a_q"], state["b_q"], state["a_inv"], state["b_inv"], state["bias"], state["residual"])
        if op == "norm":
            total, q, inv = ops.rmsnorm_blocks(state["x"], state["weight"], EPS, residual=state["residual"])
            return {"q": q, "inv": inv} if total is None else {"sum": total, "q": q, "inv": inv}
        if op == "silu":
            return ops.silu_mul_blocks(state["gate_up"], state["cols"])
        return ops.quantize_blocks(state["x"], state["block_rows"])
    return _plain(state)


def work(case):
    """Each input read once, each output written once; two operations a multiply-add."""
    op = case["op"]
    if op == "gemm":
        m, n, k = case["m"], case["n"], case["k"]
        scales = 4 * (m + _blocks(n)) * _blocks(k)
        extra = (2 * n if case["bias"] else 0) + (2 * m * n if case["residual"] else 0)
        return {"bytes": m * k + n * k + scales + extra + 2 * m * n, "flops": 2 * m * n * k}
    rows, cols = case["rows"], case["cols"]
    if op == "norm":
        return {"bytes": rows * cols * ((2 + 2 + 2 if case["residual"] else 2) + 1) + 4 * rows * _blocks(cols) + 2 * cols,
                "flops": 8 * rows * cols}
    if op == "silu":
        return {"bytes": rows * cols * (4 + 1) + 4 * rows * _blocks(cols), "flops": 8 * rows * cols}
    return {"bytes": rows * cols * (2 + 1) + 4 * -(-rows // case["block_rows"]) * _blocks(cols), "flops": 3 * rows * cols}


def _nearest_e4m3(v):
    """The e4m3 value nearest to each float64, ties to even: 3 bits of fraction down to 2^-6, steps of 2^-9 below."""
    _, e = torch.frexp(v)
    step = torch.exp2(torch.clamp(e - 1, min=-6).double() - 3)
    return torch.clamp(torch.round(v / step) * step, -TOP, TOP)


def _exact_cast(y, block_rows):
    rows, cols = y.shape
    down, right = -(-rows // block_rows), _blocks(cols)
    full = torch.zeros((down * block_rows, right * BLOCK), dtype=torch.float64, device=y.device)
    full[:rows, :cols] = y
    tiles = full.unflatten(1, (right, BLOCK)).unflatten(0, (down, block_rows)).permute(0, 2, 1, 3)
    amax = tiles.abs().flatten(2).max(dim=2).values
    inv = torch.where(amax > 0, amax / TOP, torch.ones_like(amax))
    q = _nearest_e4m3(tiles / inv[:, :, None, None]).permute(0, 2, 1, 3).reshape(down * block_rows, right * BLOCK)
    return q[:rows, :cols], inv


def exact(case, seed):
    state = prepare(case, seed)
    op = state["op"]
    if op == "gemm":
        def values(q, inv, block_rows):
            down = torch.arange(q.shape[0], device=q.device) // block_rows
            right = torch.arange(q.shape[1], device=q.device) // BLOCK
            return inv.double()[down][:, right].mul_(q.double())

        out = values(state["a_q"], state["a_inv"], 1) @ values(state["b_q"], state["b_inv"], BLOCK).mT
        for more in (state["bias"], state["residual"]):
            if more is not None:
                out += more.double()
        return out
    if op == "norm":
        total = state["x"].double() + (0 if state["residual"] is None else state["residual"].double())
        y = total / (total.square().sum(dim=1, keepdim=True) / total.shape[1] + EPS).sqrt() * state["weight"].double()
        q, inv = _exact_cast(y, 1)
        return {"q": q, "inv": inv} if state["residual"] is None else {"sum": total, "q": q, "inv": inv}
    if op == "silu":
        both = state["gate_up"].double()
        gate, up = both[:, :state["cols"]], both[:, state["cols"]:]
        return _exact_cast(gate * torch.sigmoid(gate) * up, 1)
    return _exact_cast(state["x"].double(), state["block_rows"])
