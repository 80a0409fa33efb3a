"""The module API on block-scaled FP8: Fp8BlockLinear, SwiGLU, self-attention, the transformer block, a whole LLM and
block-quantised checkpoints.  The operators are held to 64 bits elsewhere; here modules must be exactly the operators they are
made of, and a block must be as near to its bf16 self as the casts allow.

How near: an e4m3 rounding is off by at most 2^-4 of the value, uniformly spread 2^-4 / sqrt(3) = 0.036 in the mean at
the top of a binade and half that at the bottom, 0.027 over all; activations and weights each bring that into a product whose
terms' errors are independent, so the output of one linear layer is off by about sqrt(2) * 0.027 = 0.038 of its norm and never
more than the two worst cases together, 2 * 2^-4 (plus their product) of the sum of magnitudes.  Three such stages in a row
(RMSNorm's own cast counts to its product): sqrt(3) * 0.038 = 0.066; 0.1 is the bound used."""

import json

import pytest
import torch

pytestmark = pytest.mark.gpu

BF16, E4M3 = torch.bfloat16, torch.float8_e4m3fn


def randn(*shape, seed=0, std=1.0):
    return (torch.randn(shape, generator=torch.Generator(device="cuda").manual_seed(seed), device="cuda") * std).to(BF16)


def rel(a, b):
    return float((a.double() - b.double()).norm() / b.double().norm())


def values(layer):
    w = layer.weight.double()
    inv = layer.weight_inv.double().repeat_interleave(128, 0)[:w.shape[0]].repeat_interleave(128, 1)[:, :w.shape[1]]
    return w * inv


def same(a, b):
    return a.dtype == b.dtype and torch.equal(a.contiguous().view(torch.uint8), b.contiguous().view(torch.uint8))


def test_linear():
    from xax_b200 import Fp8BlockLinear, apply_linear, ops

    w, b, x = randn(392, 656, seed=1, std=0.02), randn(392, seed=2), randn(2, 5, 656, seed=3)
    layer = Fp8BlockLinear(656, 392, weight=w, bias=b)
    q, inv = ops.quantize_blocks(w, 128)
    assert same(layer.weight, q) and same(layer.weight_inv, inv) and layer.weight_inv.shape == (4, 6)
    out = layer(x)
    assert out.shape == (2, 5, 392)
    want = x.double() @ values(layer).T + b.double()
    assert rel(out, want) < 0.04  # the activations' cast alone: 0.027 in the mean
    assert rel(out, x.double() @ w.double().T + b.double()) < 0.1
    residual = randn(2, 5, 392, seed=4)
    assert same(apply_linear(x, layer, residual=residual), layer(x, residual=residual))
    assert same(layer(x)[1, 2], layer(x[1, 2]))  # a token stands alone, batched or not
    again = Fp8BlockLinear(656, 392, weight=q, weight_inv=inv, bias=b)
    assert same(again(x), out)


def test_linear_refusals():
    from xax_b200 import Fp8BlockLinear, chunked_cross_entropy_loss, loraize_linear

    w = randn(64, 256)
    layer = Fp8BlockLinear(256, 64, weight=w)
    bad = [lambda: Fp8BlockLinear(250, 64), lambda: Fp8BlockLinear(256, 60), lambda: Fp8BlockLinear(256, 64, weight=w.t()),
           lambda: Fp8BlockLinear(256, 64, weight=layer.weight), lambda: layer(randn(3, 128)),
           lambda: Fp8BlockLinear(256, 64, weight=layer.weight, weight_inv=layer.weight_inv[:, :1]),
           lambda: Fp8BlockLinear(256, 64, weight=w, weight_inv=layer.weight_inv), lambda: loraize_linear(layer, 8),
           lambda: chunked_cross_entropy_loss(randn(3, 256), torch.zeros(3, dtype=torch.int32, device="cuda"), layer)]
    for call in bad:
        with pytest.raises(ValueError):
            call()


@pytest.mark.parametrize("hidden", [512, 368])  # whole squares (one stacked product) and cut ones (a product each)
@pytest.mark.parametrize("tokens", [1, 7, 200])
def test_swiglu(tokens, hidden):
    from xax_b200 import SwiGLU, ops
    from xax_b200.arch.attention import Linear

    m = SwiGLU.build(256, hidden, key=3, fp8_blocks=True)
    x = randn(tokens, 256, seed=5)
    q, inv = ops.quantize_blocks(x)
    gu = torch.cat([m.gate.forward_quantized(q, inv), m.up.forward_quantized(q, inv)], dim=1)
    want = m.down.forward_quantized(*ops.silu_mul_blocks(gu, hidden))
    assert same(m(x), want)
    g, u = x.double() @ values(m.gate).T, x.double() @ values(m.up).T
    assert rel(m(x), (g * torch.sigmoid(g) * u) @ values(m.down).T) < 0.1
    # another weight in the same layer object is seen
    m.gate.weight_inv = m.gate.weight_inv * 2
    assert not same(m(x), want)
    # layers of several kinds still make an MLP
    m.up = Linear(256, hidden, use_bias=False, weight=randn(hidden, 256, seed=6, std=0.06))
    assert m(x).shape == (tokens, 256) and torch.isfinite(m(x).float()).all()


def bf16_twin(block):
    """The same transformer block with bf16 layers that hold the cast weights' values."""
    import copy

    from xax_b200.arch.attention import Linear, SwiGLU

    lin = lambda m: Linear(m.in_features, m.out_features, use_bias=m.bias is not None, weight=values(m).to(BF16), bias=m.bias)  # noqa: E731
    t = copy.copy(block)
    t.self_attn = copy.copy(block.self_attn)
    t.self_attn._fused = None
    for n in ("q_proj", "k_proj", "v_proj", "output_proj"):
        setattr(t.self_attn, n, lin(getattr(block.self_attn, n)))
    f = block.feed_forward
    t.feed_forward = SwiGLU(lin(f.gate), lin(f.up), lin(f.down))
    return t


@pytest.mark.parametrize("kv_heads,head_dim", [(2, 64), (4, 64), (1, 128)])
def test_transformer_block_prefill_and_decode(kv_heads, head_dim):
    from xax_b200 import TransformerBlock, ops

    H, B, T = 256, 3, 37
    block = TransformerBlock.build(H, 4, 656, key=1, num_kv_heads=kv_heads, head_dim=head_dim, causal=True, use_rotary_embeddings=True,
                                   norm_type="rmsnorm", feedforward_type="swiglu", fp8_blocks=True)
    assert block.self_attn.is_fp8_blocks() and block.feed_forward.is_fp8_blocks()
    twin = bf16_twin(block)
    caches = [{"k": torch.zeros((B, 64, kv_heads, head_dim), dtype=BF16, device="cuda"),
               "v": torch.zeros((B, 64, kv_heads, head_dim), dtype=BF16, device="cuda"),
               "position": torch.zeros((B,), dtype=torch.int32, device="cuda")} for _ in range(2)]
    for step, t in enumerate((T, 1, 1)):
        x = randn(B * t, H, seed=10 + step)
        got, caches[0] = block.forward_tokens(x, B, t, cache=caches[0])
        want, caches[1] = twin.forward_tokens(x, B, t, cache=caches[1])
        assert got.shape == (B * t, H)
        assert rel(got.double() - x.double(), want.double() - x.double()) < 0.1  # what the block adds to the stream
    # the block is its operators: redo the last step's MLP half from the attention half
    a, f = block.self_attn, block.feed_forward
    _, q, inv = ops.rmsnorm_blocks(x, block.attn_norm.weight_bf16(), block.attn_norm.eps)
    cache = {k: v.clone() for k, v in caches[0].items()}
    cache["position"] -= 1
    o, _ = a.forward_tokens(x, B, 1, cache=cache, y_q=(q, inv))
    x1, q, inv = ops.rmsnorm_blocks(o, block.mlp_norm.weight_bf16(), block.mlp_norm.eps, residual=x)
    assert same(x1, (o.float() + x.float()).to(BF16))
    assert same(got, f.forward_tokens(x1, B, 1, residual=x1, y_q=(q, inv)))
    # the one-sequence entry points take the same path
    y, _ = block(randn(5, H, seed=20))
    assert y.shape == (5, H)
    # a block with only its MLP block-scaled, and one with only its attention
    for part in ("self_attn", "feed_forward"):
        mixed = bf16_twin(block)
        setattr(mixed, part, getattr(block, part))
        z, _ = mixed.forward_tokens(randn(B * 4, H, seed=30), B, 4)
        w, _ = twin.forward_tokens(randn(B * 4, H, seed=30), B, 4)
        assert rel(z, w) < 0.1


def config():
    from xax_b200 import LLMConfig

    return LLMConfig(vocab_size=256, embed_dim=256, q_heads=4, kv_heads=2, head_dim=64, num_layers=2, max_tsz=64, mlp_hidden_dim=656)


def test_llm_generates_the_same_with_and_without_a_graph():
    from xax_b200 import LLM, _lib, llm_generate_batch

    m = LLM.build(config(), key=3, fp8_blocks=True, init_std=0.08)
    toks = torch.randint(0, 256, (3, 9), dtype=torch.int32, device="cuda", generator=torch.Generator(device="cuda").manual_seed(1))
    a, _ = llm_generate_batch(m, toks, 12, use_graph=True)
    b, _ = llm_generate_batch(m, toks, 12, use_graph=False)
    assert torch.equal(a, b)
    # cached decoding agrees with one pass over the finished sequence wherever its choice is not a near tie
    logits, _ = m.forward_batch(a[:, :-1].contiguous())
    top = logits[:, 8:].float().topk(2, dim=-1).values
    clear = top[..., 0] - top[..., 1] > 0.05 * logits.float().std()
    assert (logits[:, 8:].float().argmax(-1) == a[:, 9:])[clear].float().mean() > 0.9
    _lib.device_status()
    with pytest.raises(ValueError, match="tensor-parallel"):
        LLM.build(config(), key=3, fp8_blocks=True, tp_size=2)


def checkpoint(m, path, quantised=True, size=(128, 128)):
    from safetensors.torch import save_file

    st = {"model.embed_tokens.weight": m.embed.weight, "model.norm.weight": m.norm.weight_bf16(), "lm_head.weight": m.lm_head.weight}
    for i, b in enumerate(m.blocks):
        a, f, pre = b.self_attn, b.feed_forward, f"model.layers.{i}"
        for name, lin in (("self_attn.q_proj", a.q_proj), ("self_attn.k_proj", a.k_proj), ("self_attn.v_proj", a.v_proj),
                          ("self_attn.o_proj", a.output_proj), ("mlp.gate_proj", f.gate), ("mlp.up_proj", f.up), ("mlp.down_proj", f.down)):
            if quantised:
                st[f"{pre}.{name}.weight"], st[f"{pre}.{name}.weight_scale_inv"] = lin.weight, lin.weight_inv
            else:
                st[f"{pre}.{name}.weight"] = values(lin).to(BF16)
        st[f"{pre}.input_layernorm.weight"] = b.attn_norm.weight_bf16()
        st[f"{pre}.post_attention_layernorm.weight"] = b.mlp_norm.weight_bf16()
    save_file({k: v.cpu().contiguous() for k, v in st.items()}, str(path / "model.safetensors"))
    c = m.config
    cfg = {"hidden_size": c.embed_dim, "num_attention_heads": c.q_heads, "num_key_value_heads": c.kv_heads, "head_dim": c.head_dim,
           "num_hidden_layers": c.num_layers, "vocab_size": c.vocab_size, "intermediate_size": c.mlp_hidden_dim}
    if quantised:
        cfg["quantization_config"] = {"quant_method": "fp8", "weight_block_size": list(size)}
    (path / "config.json").write_text(json.dumps(cfg))


def test_block_quantised_checkpoint(tmp_path):
    from xax_b200 import LLM, Fp8BlockLinear, build_pretrained_llm
    from xax_b200.arch.attention import Linear

    m = LLM.build(config(), key=5, fp8_blocks=True, init_std=0.08)
    checkpoint(m, tmp_path)
    toks = torch.arange(12, dtype=torch.int32, device="cuda").reshape(2, 6)
    want, _ = m.forward_batch(toks)
    loaded = build_pretrained_llm(str(tmp_path))
    assert isinstance(loaded.blocks[0].feed_forward.down, Fp8BlockLinear)
    assert torch.equal(loaded.forward_batch(toks)[0], want)
    # other layers get the dequantised weight
    plain = build_pretrained_llm(str(tmp_path), use_fp8=False)
    assert type(plain.blocks[0].self_attn.q_proj) is Linear
    assert same(plain.blocks[0].self_attn.q_proj.weight, values(m.blocks[0].self_attn.q_proj).to(BF16))
    # a bf16 checkpoint is cast on the way in
    (tmp_path / "bf16").mkdir()
    checkpoint(m, tmp_path / "bf16", quantised=False)
    cast = build_pretrained_llm(str(tmp_path / "bf16"), fp8_blocks=True)
    assert rel(cast.forward_batch(toks)[0], want) < 0.1
    checkpoint(m, tmp_path, size=(64, 128))
    with pytest.raises(ValueError, match="weight_block_size"):
        build_pretrained_llm(str(tmp_path))


def test_stacked_weights_are_the_layers_own():
    """Layers that the library builds share one operand: no second copy, no stale one, and layers of the user's stay theirs."""
    from xax_b200 import Fp8BlockLinear, SwiGLU, ops

    x = randn(9, 256, seed=1)
    xq, x_inv = ops.quantize_blocks(x)

    def each(mlp):
        return torch.cat([m.forward_quantized(xq, x_inv) for m in (mlp.gate, mlp.up)], 1)

    mlp = SwiGLU.build(256, 384, key=3, use_bias=True, fp8_blocks=True)
    assert mlp.gate.weight.untyped_storage().data_ptr() == mlp.up.weight.untyped_storage().data_ptr()
    assert mlp._gate_up_stack()._weights()[0].data_ptr() == mlp.gate.weight.data_ptr()
    assert same(mlp._gate_up_stack()(xq, x_inv), each(mlp))
    other, other_inv = ops.quantize_blocks(randn(384, 256, seed=5, std=0.05), 128)
    for write in (lambda: mlp.up.weight.data.copy_(other), lambda: mlp.up.weight_inv.data.copy_(other_inv),
                  lambda: setattr(mlp.gate, "weight", other), lambda: mlp.gate.bias.data.zero_(),
                  lambda: setattr(mlp.up, "bias", None)):
        before = mlp._gate_up_stack()(xq, x_inv)
        write()
        after = mlp._gate_up_stack()(xq, x_inv)
        assert same(after, each(mlp)) and not same(after, before)

    gate, up = (Fp8BlockLinear(256, 384, key=k, use_bias=False) for k in (1, 2))
    held = gate.weight
    with torch.inference_mode():
        mine = SwiGLU(gate, up, Fp8BlockLinear(384, 256, key=4, use_bias=False))
        first = mine.forward_tokens(x, 1, 9)
    held.copy_(other)
    assert gate.weight is held and not same(mine.forward_tokens(x, 1, 9), first)
    assert same(mine._gate_up_stack()(xq, x_inv), each(mine))


def test_first_call_captured():
    """A module whose first call is captured answers alike before, in and after the replay."""
    from xax_b200 import Fp8BlockLinear, SwiGLU

    x = randn(9, 256, seed=1)
    warm, mlp = (SwiGLU.build(256, 384, key=3, fp8_blocks=True) for _ in range(2))
    want = warm.forward_tokens(x, 1, 9)
    own = SwiGLU(*(Fp8BlockLinear(i, o, key=k, use_bias=False) for i, o, k in ((256, 384, 4), (256, 384, 5), (384, 256, 6))))
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got, got_own = mlp.forward_tokens(x, 1, 9), own.forward_tokens(x, 1, 9)
    eager, eager_own = mlp.forward_tokens(x, 1, 9), own.forward_tokens(x, 1, 9)
    graph.replay()
    assert same(eager, want) and same(got, want)
    assert same(got_own, eager_own)


def test_transformer_on_block_scaled_layers():
    """The token-in, logits-out module: batched self-attention casts its input once, sequence by sequence alike, and a token
    does not depend on those behind it (every scale belongs to one token)."""
    from xax_b200 import Transformer, apply_linear, ops

    model = Transformer.build(64, 256, 4, 512, 2, 64, key=1, causal=True, use_rotary_embeddings=True, use_fp8=True, fp8_blocks=True)
    assert all(b.self_attn.is_fp8_blocks() and b.feed_forward.is_fp8_blocks() for b in model.layers.layers)
    attn = model.layers.layers[0].self_attn
    assert not attn.use_fp8
    x = randn(2, 9, 256, seed=3)
    out = attn(x)
    assert out.shape == x.shape and same(out[1], attn(x[1:])[0])
    assert same(attn.q_proj.forward_quantized(*ops.quantize_blocks(x.reshape(18, 256))),
                apply_linear(x, attn.q_proj).reshape(18, 256))
    tokens = torch.arange(16, device="cuda", dtype=torch.int32)
    logits, _ = model.forward(tokens)
    assert logits.shape == (16, 64) and torch.isfinite(logits).all()
    hidden, x = model.encode(tokens)[0], model.token_embedding(tokens[0]).reshape(1, 256)
    for block in model.layers.layers:  # the first token, alone through the blocks
        x, _ = block.forward(x)
    assert rel(model.layer_norm(x), hidden[:1]) < 2.0**-6  # (a few bf16 and e4m3 roundings may fall the other way)
