"""Decode steps with 4-bit weights and an 8-bit cache: fast-transformer_amd/decode.py over kernels/w4.py and cache_q8.py.

The step is compared bit for bit with its operators called one by one, and a step whose weights alone are in 4 bits with
transformers' float32 model over the same dequantised weights (the bar of the BF16 step's own test: 2e-2 + 1e-2 |ref|).
"""

import copy

import pytest
import torch

import qwen3_tiny as Q

import decode as D
from kernels import argmax, cache_q8, rmsnorm, w4

pytestmark = pytest.mark.gpu


def setup(batch, dims=Q.SMALL, seed=5, length=5):
    m = Q.model(dims)
    gpu = copy.deepcopy(m).to("cuda", torch.bfloat16)
    prompt = torch.randint(0, m.config.vocab_size, (batch, length), generator=torch.Generator().manual_seed(seed))
    return m, gpu, prompt


@pytest.mark.parametrize("batch,group", [(1, 128), (3, 64)])
def test_four_bit_weights_against_transformers(cuda, batch, group):
    m, gpu, prompt = setup(batch)
    dec = D.Decoder(gpu, batch, 24, weight_bits=4, weight_group=group)
    ids, logits = dec.generate(prompt, 5)

    def value(t):
        # the codes and scales of quantize_w4, whose products stay in float32 here
        wide = t.float().unflatten(1, (-1, group))
        s = (wide.abs().amax(dim=2, keepdim=True) / 7).to(torch.bfloat16).float()
        return ((wide / s).round().clamp(-8, 7) * s).flatten(1)

    with torch.no_grad():
        for layer in m.model.layers:
            for p in (*layer.self_attn.parameters(), *layer.mlp.parameters()):
                if p.dim() == 2:
                    p.copy_(value(p))
        tokens = torch.cat([prompt, ids[:, :-1].cpu()], dim=1)
        want = m(tokens).logits.numpy()
    assert Q.close(logits.float().cpu().numpy(), want)


@pytest.mark.parametrize("kind", [torch.float8_e4m3fn, torch.int8])
@pytest.mark.parametrize("bits", [4, 16])
def test_the_step_is_its_operators_in_turn(cuda, kind, bits):
    if bits == 16:
        from kernels import linear as L
        from kernels import swiglu as S
    batch, capacity = 2, 40
    m, gpu, prompt = setup(batch, length=7)
    dec = D.Decoder(gpu, batch, capacity, weight_bits=bits, cache_dtype=kind, cache_block=16)
    assert dec.cache.store.dtype == kind and not dec.fused_rope
    ids, logits = dec.generate(prompt, 14)
    base = gpu.model
    packed = [D.PackedLayer(layer) for layer in base.layers]
    if bits == 4:
        packed = [p.quantize(128) for p in packed]
    dims = (batch, m.config.num_key_value_heads, capacity, m.config.head_dim)
    caches = [cache_q8.new_cache_q8(*dims, block=16, dtype=kind, device=cuda) for _ in packed]
    phases = torch.zeros((batch, 1), dtype=torch.int64, device=cuda)
    tokens = torch.cat([prompt.to(cuda), ids[:, :-1]], dim=1)
    for t in range(tokens.shape[1]):
        at = torch.full((batch,), t, dtype=torch.int64, device=cuda)
        r = None
        for i, (p, c) in enumerate(zip(packed, caches)):
            gain, eps = p.input_norm.weight, p.input_norm.variance_epsilon
            if bits == 4:
                if i == 0:
                    n, r = rmsnorm.embed_rms_norm(tokens[:, t].contiguous(), dec.embed, gain, eps)
                    qkv = w4.linear_w4(n, p.qkv_weight)
                else:
                    qkv = w4.rms_norm_linear_w4(r, gain, eps, p.qkv_weight)
            elif i == 0:
                qkv, r = L.embed_rms_norm_linear(tokens[:, t].contiguous(), dec.embed, gain, eps, p.qkv_weight)
            else:
                qkv = L.rms_norm_linear(r, gain, eps, p.qkv_weight)
            q = cache_q8.qk_rope_cache_q8(qkv.view(batch, 1, -1), p.q_norm, p.k_norm, dec.cos, dec.sin, at, *c, p.q_heads,
                                          rows=True, phases=phases)
            a = cache_q8.decode_attention_q8(q, *c, at, p.scaling).view(batch, -1)
            gain, eps = p.post_norm.weight, p.post_norm.variance_epsilon
            if bits == 4:
                r = w4.linear_residual_w4(a, p.o_weight, r)
                r = w4.linear_residual_w4(w4.gate_up_swiglu_w4(r, p.gate_up_weight, gain, eps), p.down_weight, r)
            else:
                r = L.linear_residual(a, p.o_weight, r)
                r = L.linear_residual(S.gate_up_swiglu(r, p.gate_up_weight, gain, eps), p.down_weight, r)
        _, want = argmax.lm_head_argmax(r, dec.lm_head, base.norm.weight, base.norm.variance_epsilon)
        assert torch.equal(logits[:, t], want), t
    for i, (keys, values, ks, vs) in enumerate(caches):
        n = tokens.shape[1]
        for mine, theirs in ((keys, dec.cache.keys[i]), (values, dec.cache.values[i])):
            assert torch.equal(mine.view(torch.uint8)[:, :, :n], theirs.view(torch.uint8)[:, :, :n])
        assert torch.equal(ks, dec.cache.k_scales[i]) and torch.equal(vs, dec.cache.v_scales[i])


@pytest.mark.parametrize("bits,kind", [(4, torch.float8_e4m3fn), (4, torch.bfloat16), (16, torch.int8)])
def test_graph_replays_give_the_eager_bits(cuda, bits, kind):
    _, gpu, prompt = setup(2, seed=9)
    args = dict(weight_bits=bits, cache_dtype=kind, cache_block=16)
    e_ids, e_logits = D.Decoder(gpu, 2, 32, **args).generate(prompt, 20)
    dec = D.Decoder(gpu, 2, 32, **args)
    for _ in range(2):  # the second replays the same graph from position 0
        ids, logits = dec.generate(prompt, 20, graph=True)
        assert torch.equal(ids, e_ids) and torch.equal(logits, e_logits)


def test_refusals(cuda):
    _, gpu, _ = setup(1)
    with pytest.raises(ValueError, match="weight_bits"):
        D.Decoder(gpu, 1, 16, weight_bits=8)
    with pytest.raises(ValueError, match="8-bit"):
        D.Decoder(gpu, 1, 16, cache_dtype=torch.float16)
    with pytest.raises(ValueError, match="8-bit"):
        D.Decoder(gpu, 1, 16, cache_dtype=torch.int8, cache_block=48)


def test_custom_ops_equal_the_functions(cuda):
    import kernels.ops  # noqa: F401

    g = torch.Generator(device=cuda).manual_seed(3)
    weight = w4.quantize_w4(torch.randn((256, 512), generator=g, device=cuda).to(torch.bfloat16), 64)
    both = w4.quantize_w4(torch.randn((256, 512), generator=g, device=cuda).to(torch.bfloat16), 64, gate_up=True)
    x = torch.randn((3, 512), generator=g, device=cuda).to(torch.bfloat16)
    gain = torch.ones(512, dtype=torch.bfloat16, device=cuda)
    ops = torch.ops.ftk
    assert torch.equal(ops.linear_w4(x, weight.codes, weight.scales, None, 256, 512, 64), w4.linear_w4(x, weight))
    assert torch.equal(ops.gate_up_swiglu_w4(x, both.codes, both.scales, None, 256, 512, 64, gain, 1e-6),
                       w4.gate_up_swiglu_w4(x, both, gain, 1e-6))
    caches = [cache_q8.new_cache_q8(2, 2, 64, 64, block=16, device=cuda) for _ in range(2)]
    packed = torch.randn((2, 1, 8 * 64), generator=g, device=cuda).to(torch.bfloat16)
    head = torch.ones(64, dtype=torch.bfloat16, device=cuda)
    table = torch.randn((64, 64), generator=g, device=cuda).to(torch.bfloat16)
    at, phases = torch.tensor([3, 60], device=cuda), torch.zeros((2, 1), dtype=torch.int64, device=cuda)
    norm = kernels.ops._Norm(head, 1e-6)
    q = cache_q8.qk_rope_cache_q8(packed, norm, norm, table, table, at, *caches[0], 4, rows=True, phases=phases)
    got = ops.qk_rope_cache_q8(packed, head, head, 1e-6, 1e-6, table, table, at, *caches[1], 4, phases)
    assert torch.equal(got.transpose(1, 2), q)
    for a, b in zip(*caches):
        assert torch.equal(a.view(torch.uint8), b.view(torch.uint8))
    q = q.contiguous()
    assert torch.equal(ops.decode_attention_q8(q, *caches[0], at, 0.125), cache_q8.decode_attention_q8(q, *caches[0], at, 0.125))
    torch.library.opcheck(ops.linear_w4.default, (x, weight.codes, weight.scales, None, 256, 512, 64),
                          test_utils=("test_schema", "test_faketensor"))
    whole = cache_q8.new_cache_q8(2, 2, 64, 64, block=16, dtype=torch.int8, device=cuda)  # (opcheck compares no e4m3)
    torch.library.opcheck(ops.decode_attention_q8.default, (q, *whole, at, 0.125),
                          test_utils=("test_schema", "test_faketensor"))
