"""Greedy decode steps of a Qwen3 causal LM, one token per row, through this library's kernels.

The caller side of the path: engine/decode.py:165-297 (optimize_model,
KVCache, forward_last for a decode token) and engine/layers.py:13-102
(PackedAttention, PackedMLP), restated over the fused forms of ``kernels``.
One step, per row b at its device-side position p_b:

  layer 0   qkv, r = embed_rms_norm_linear(ids, E, ln1, W_qkv)   embedding gather + norm + QKV, one launch
  layer l   qkv    = rms_norm_linear(r, ln1, W_qkv)               norm + QKV, one launch
            a      = rope_attend(qkv, ...)                        head norms + RoPE, K, V into slot p_b,
                                                                  decode attention over slots 0..p_b
            r      = linear_residual(a, W_o, r)                   O, the residual add in its epilogue
            act    = gate_up_swiglu(r, W_gu, ln2)                 norm + gate/up + SwiGLU
            r      = linear_residual(act, W_down, r)              down, the residual add in its epilogue
  final     ids, logits = lm_head_argmax(r, W_lm, norm)           norm + lm_head + argmax

The reference adds each sublayer's output to the residual stream in the next
norm (add_rms_norm, decode.py:236-243, :258-261, :291-296); here the add runs
in the epilogue of the projection that produces it, which stores the same BF16
sum, so no norm prologue has to read a second [rows, H] stream. The head
norms, RoPE and the cache update run in the attention kernel's prologue
(rope_attend) where it takes the head layout (head_dim 128, at most 4 query
heads per KV head; otherwise qk_rope_cache and decode attention launch
apart). That is 5 launches per layer (6 with a merge of attention splits)
and one for the vocabulary. The weights are the model's own tensors (BF16, on the GPU),
packed once as the reference packs them ([Wq; Wk; Wv], [Wg; Wu],
layers.py:23-26, :92-95). Positions, input ids and the RoPE phase live on the
device, so one captured graph serves every step (``Decoder.capture``), the way
the reference replays its decode graph (decode.py:650-668).

``weight_bits=4`` holds the layers' projections in 4 bits (kernels/w4.py) and ``cache_dtype=torch.float8_e4m3fn`` or
``torch.int8`` the cache in 8 (kernels/cache_q8.py): the same step over the same operators' few-bits forms. The
embedding and the vocabulary stay BF16.

  layer l   qkv    = rms_norm_linear_w4(r, ln1, W_qkv)            (layer 0: embed_rms_norm, then linear_w4)
            a      = decode_attention_q8(qk_rope_cache_q8(qkv))   the block of slot p_b re-scaled where it must be
            r      = linear_residual_w4(a, W_o, r)
            act    = gate_up_swiglu_w4(r, W_gu, ln2)
            r      = linear_residual_w4(act, W_down, r)

A prompt is fed one token per step: each prompt token attends to the slots
before it, which is what a causal prefill computes. A batched prefill
(grouped SDPA over the whole prompt, layers.py:66-71) is not part of this
library.
"""

import torch

from kernels import _native
from kernels import argmax as _argmax
from kernels import cache_q8 as _q8
from kernels import decode_attention as _attention
from kernels import linear as _linear
from kernels import qk_rope as _rope
from kernels import rmsnorm as _rmsnorm
from kernels import swiglu as _swiglu
from kernels import w4 as _w4


class KVCache:
    """Layer-local BF16 [batch, kv_heads, capacity, head_dim] caches in one allocation (engine/decode.py:176-213).

    ``store`` is [key/value, layer, B, Hkv, C, D]; ``keys[l]`` and
    ``values[l]`` are contiguous views of one layer.
    """

    def __init__(self, config, batch, capacity, device, dtype=torch.bfloat16):
        head_dim = getattr(config, "head_dim", None) or config.hidden_size // config.num_attention_heads
        shape = (batch, config.num_key_value_heads, capacity, head_dim)
        layers = config.num_hidden_layers
        self.store = torch.zeros((2, layers, *shape), dtype=dtype, device=device)
        self.keys = [self.store[0, layer] for layer in range(layers)]
        self.values = [self.store[1, layer] for layer in range(layers)]


class KVCacheQ8:
    """The same caches held in 8 bits: ``store`` [key/value, layer, B, Hkv, C, D] codes (float8_e4m3fn or int8) and
    ``scales`` [key/value, layer, B, Hkv, ceil(C / block)] FP32, with one layer's views ``keys[l]``, ``values[l]``,
    ``k_scales[l]`` and ``v_scales[l]``."""

    def __init__(self, config, batch, capacity, device, dtype, block):
        if dtype not in _q8.TYPES or block not in _q8.BLOCKS:
            raise ValueError(f"an 8-bit cache is float8_e4m3fn or int8 in blocks of {_q8.BLOCKS}, got {dtype}, {block}")
        head_dim = getattr(config, "head_dim", None) or config.hidden_size // config.num_attention_heads
        layers, heads = config.num_hidden_layers, config.num_key_value_heads
        self.store = torch.zeros((2, layers, batch, heads, capacity, head_dim), dtype=torch.uint8,
                                 device=device).view(dtype)
        self.scales = torch.ones((2, layers, batch, heads, -(-capacity // block)), device=device)
        self.keys, self.values = ([self.store[i, layer] for layer in range(layers)] for i in range(2))
        self.k_scales, self.v_scales = ([self.scales[i, layer] for layer in range(layers)] for i in range(2))


class PackedLayer:
    """One decoder layer's weights as the step reads them (engine/layers.py:13-30, :92-98)."""

    def __init__(self, layer):
        attention, mlp = layer.self_attn, layer.mlp
        with torch.no_grad():
            self.qkv_weight = torch.cat((attention.q_proj.weight, attention.k_proj.weight,
                                         attention.v_proj.weight), dim=0).contiguous()
            self.gate_up_weight = torch.cat((mlp.gate_proj.weight, mlp.up_proj.weight), dim=0).contiguous()
        self.o_weight = attention.o_proj.weight.detach()
        self.down_weight = mlp.down_proj.weight.detach()
        self.input_norm = layer.input_layernorm
        self.post_norm = layer.post_attention_layernorm
        self.q_norm, self.k_norm = attention.q_norm, attention.k_norm
        self.q_heads = attention.q_proj.out_features // attention.head_dim
        self.scaling = attention.scaling

    def quantize(self, group):
        """The projections in 4 bits instead (W4Weights in place of the tensors)."""
        with torch.no_grad():
            self.qkv_weight = _w4.quantize_w4(self.qkv_weight, group)
            self.gate_up_weight = _w4.quantize_w4(self.gate_up_weight, group, gate_up=True)
            self.o_weight = _w4.quantize_w4(self.o_weight, group)
            self.down_weight = _w4.quantize_w4(self.down_weight, group)
        return self


class Decoder:
    """Decode state for ``batch`` rows of a transformers Qwen3ForCausalLM held in BF16 on the GPU.

    ``token_ids`` [B] and ``position`` [B] (int64, on the device) are the
    step's inputs; ``step()`` returns (ids [B] int64, logits [B, V] BF16) and
    writes each layer's key and value at slot ``position[b]`` of row b.
    ``weight_bits`` 4 quantises the layers' projections (round to nearest, a
    BF16 scale per ``weight_group`` columns); ``cache_dtype`` float8_e4m3fn or
    int8 holds the cache in 8 bits, a scale per ``cache_block`` slots.
    """

    def __init__(self, model, batch, capacity, fused_rope=True, weight_bits=16, weight_group=128,
                 cache_dtype=torch.bfloat16, cache_block=64):
        base = model.model
        embed = base.embed_tokens.weight
        if embed.dtype != torch.bfloat16 or embed.device.type != "cuda":
            raise ValueError("the model must be BF16 on a GPU (model.to('cuda', torch.bfloat16))")
        _native.require_gpu(embed)
        self.batch, self.capacity = batch, capacity
        self.embed = embed.detach()
        self.lm_head = model.lm_head.weight.detach()
        self.norm = base.norm
        if weight_bits not in (4, 16):
            raise ValueError(f"weight_bits {weight_bits}: 16 (BF16) or 4")
        self.weight_bits = weight_bits
        self.layers = []
        for layer in base.layers:
            packed = PackedLayer(layer)
            self.layers.append(packed.quantize(weight_group) if weight_bits == 4 else packed)
        #: The cache in 8 bits.
        self.cache_q8 = cache_dtype != torch.bfloat16
        self.cache = KVCacheQ8(model.config, batch, capacity, embed.device, cache_dtype, cache_block) if self.cache_q8 \
            else KVCache(model.config, batch, capacity, embed.device)
        device = embed.device
        with torch.no_grad():
            # Full tables [capacity, D]: the kernel reads row position[b] + phase on the device.
            cos, sin = base.rotary_emb(embed.new_empty((1, 1, embed.shape[1])),
                                       torch.arange(capacity, device=device).unsqueeze(0))
        self.cos, self.sin = cos[0].contiguous(), sin[0].contiguous()
        self.phases = torch.zeros((batch, 1), dtype=torch.int64, device=device)
        self.position = torch.zeros((batch,), dtype=torch.int64, device=device)
        self.token_ids = torch.zeros((batch,), dtype=torch.int64, device=device)
        self._graph = None
        first = self.layers[0]
        gains = [t for layer in self.layers for t in (layer.q_norm.weight, layer.k_norm.weight)]
        #: Head norms + RoPE in the attention launch (else the separate qk_rope_cache launch).
        self.fused_rope = bool(fused_rope) and not self.cache_q8 and _attention.rope_attention_supported(
            first.q_heads, self.cache.keys[0].shape[1], self.cache.keys[0].shape[3], capacity=capacity) and \
            all(t.is_contiguous() and t.data_ptr() % 16 == 0 for t in [self.cos, self.sin, self.cache.store, *gains])

    def step(self):
        """One decode token per row at ``position`` (engine/decode.py:215-297 for a one-token step)."""
        batch = self.batch
        residual = None
        for index, layer in enumerate(self.layers):
            qkv, residual = self._qkv(index, layer, residual)
            attention = self._attend(index, layer, qkv).view(batch, -1)
            if self.weight_bits == 4:
                residual = _w4.linear_residual_w4(attention, layer.o_weight, residual)
                act = _w4.gate_up_swiglu_w4(residual, layer.gate_up_weight, layer.post_norm.weight,
                                            layer.post_norm.variance_epsilon)
                residual = _w4.linear_residual_w4(act, layer.down_weight, residual)
                continue
            residual = _linear.linear_residual(attention, layer.o_weight, residual)
            act = _swiglu.gate_up_swiglu(residual, layer.gate_up_weight, layer.post_norm.weight,
                                         layer.post_norm.variance_epsilon)
            residual = _linear.linear_residual(act, layer.down_weight, residual)
        return _argmax.lm_head_argmax(residual, self.lm_head, self.norm.weight, self.norm.variance_epsilon)

    def _qkv(self, index, layer, residual):
        """(packed QKV rows, the residual stream) of a layer; layer 0 gathers the embedding."""
        norm, eps = layer.input_norm.weight, layer.input_norm.variance_epsilon
        if self.weight_bits == 4:
            if index == 0:
                normalized, residual = _rmsnorm.embed_rms_norm(self.token_ids, self.embed, norm, eps)
                return _w4.linear_w4(normalized, layer.qkv_weight), residual
            return _w4.rms_norm_linear_w4(residual, norm, eps, layer.qkv_weight), residual
        if index == 0:
            return _linear.embed_rms_norm_linear(self.token_ids, self.embed, norm, eps, layer.qkv_weight)
        return _linear.rms_norm_linear(residual, norm, eps, layer.qkv_weight), residual

    def _attend(self, index, layer, qkv):
        """The layer's attention output [B, 1, Hq, D], its key and value heads written to the cache."""
        batch, cache = self.batch, self.cache
        keys, values = cache.keys[index], cache.values[index]
        if self.cache_q8:
            scales = cache.k_scales[index], cache.v_scales[index]
            query = _q8.qk_rope_cache_q8(qkv.view(batch, 1, -1), layer.q_norm, layer.k_norm, self.cos, self.sin,
                                         self.position, keys, values, *scales, layer.q_heads, rows=True,
                                         phases=self.phases)
            return _q8.decode_attention_q8(query, keys, values, *scales, self.position, layer.scaling)
        if self.fused_rope:
            return _attention.rope_attend(qkv, layer.q_norm, layer.k_norm, self.cos, self.sin, self.position, keys,
                                          values, layer.q_heads, layer.scaling, phases=self.phases)
        query = _rope.qk_rope_cache(qkv.view(batch, 1, -1), layer.q_norm, layer.k_norm, self.cos, self.sin,
                                    self.position, keys, values, layer.q_heads, rows=True, phases=self.phases)
        return _attention.attend(query.reshape(batch, layer.q_heads, -1), keys, values, self.position, layer.scaling)

    def advance(self, ids):
        """Feed ``ids`` as the next tokens and move every row one slot on (device-side, capturable)."""
        self.token_ids.copy_(ids)
        self.position.add_(1)

    def capture(self):
        """Record ``step`` + ``advance`` in one graph; returns the graph's (ids, logits) outputs.

        One eager step first sizes the workspaces the kernels share (capture
        allocates nothing of its own); it writes slot ``position`` of the
        caches, which the next real step at that position rewrites.
        """
        self.step()
        stream = torch.cuda.Stream(device=self.embed.device)
        stream.wait_stream(torch.cuda.current_stream(self.embed.device))
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.stream(stream):
            with torch.cuda.graph(graph, stream=stream):
                ids, logits = self.step()
                self.advance(ids)
        torch.cuda.current_stream(self.embed.device).wait_stream(stream)
        self._graph = (graph, ids, logits)
        return ids, logits

    def generate(self, prompt, steps, graph=False):
        """Greedy continuation of ``prompt`` [B, P] int64: ([B, steps] ids, [B, P + steps - 1, V] logits).

        The prompt goes through one step per token (positions 0..P-1); the
        last of them gives the first new token, and ``steps - 1`` more steps
        follow. ``graph`` replays one captured step instead of launching each.
        """
        batch, length = prompt.shape
        if batch != self.batch:
            raise ValueError(f"prompt has {batch} rows, the decoder {self.batch}")
        if length < 1 or steps < 1 or length + steps - 1 > self.capacity:
            raise ValueError(f"{length} prompt tokens + {steps} steps do not fit {self.capacity} cache slots")
        prompt = prompt.to(self.token_ids.device)
        if graph and self._graph is None:
            self.position.zero_()
            self.token_ids.copy_(prompt[:, 0])
            self.capture()
        self.position.zero_()
        out, logits = [], []
        for t in range(length + steps - 1):
            if t < length:
                self.token_ids.copy_(prompt[:, t])
            if graph:
                g, ids, step_logits = self._graph
                g.replay()
            else:
                ids, step_logits = self.step()
                self.advance(ids)
            logits.append(step_logits.clone())
            if t >= length - 1:
                out.append(ids.clone())
        return torch.stack(out, dim=1), torch.stack(logits, dim=1)
