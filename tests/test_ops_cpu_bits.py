"""The few-bits custom ops register and give the output shapes under FakeTensorMode (no kernel runs)."""

import torch
from torch._subclasses.fake_tensor import FakeTensorMode

import kernels.ops  # noqa: F401


def test_fake_shapes():
    bf, q8 = torch.bfloat16, torch.float8_e4m3fn
    with FakeTensorMode():
        x, g = torch.empty(2, 5, 4096, dtype=bf), torch.empty(4096, dtype=bf)
        codes = torch.empty(64, 32, 64, 4, dtype=torch.int32)
        scales = torch.empty(64, 32, 16, 1, dtype=bf)
        assert torch.ops.ftk.linear_w4(x, codes, scales, None, 1024, 4096, 128).shape == (2, 5, 1024)
        assert torch.ops.ftk.gate_up_swiglu_w4(x, codes, scales, None, 1024, 4096, 128, g, 1e-6).shape == (2, 5, 512)
        q = torch.empty(2, 32, 1, 128, dtype=bf)
        cache, s = torch.empty(2, 8, 64, 128, dtype=q8), torch.empty(2, 8, 4)
        pos = torch.empty(2, dtype=torch.int64)
        assert torch.ops.ftk.decode_attention_q8(q, cache, cache, s, s, pos, 0.088).shape == (2, 1, 32, 128)
        packed, gain = torch.empty(2, 1, 48 * 128, dtype=bf), torch.empty(128, dtype=bf)
        table, phases = torch.empty(64, 128, dtype=bf), torch.empty(2, 1, dtype=torch.int64)
        out = torch.ops.ftk.qk_rope_cache_q8(packed, gain, gain, 1e-6, 1e-6, table, table, pos, cache,
                                             torch.empty_like(cache), s, torch.empty_like(s), 32, phases)
        assert out.shape == (2, 1, 32, 128) and out.dtype == bf
