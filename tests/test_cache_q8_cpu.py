"""The 8-bit cache's sizes, interval counts and argument checks, on the CPU."""

from types import SimpleNamespace

import pytest
import torch

from kernels import _native
from kernels import cache_q8 as C


def test_block_of_inverts_the_scale_count():
    for capacity in (1, 15, 16, 17, 100, 128, 129, 777, 4096, 32768, 1000003):
        for block in C.BLOCKS:
            found = C.block_of(capacity, -(-capacity // block))
            assert found == block or (capacity <= 128 and -(-capacity // found) == -(-capacity // block))
            if found != block:  # two sizes give as many scales: then every slot has the same scale in both
                assert all(t // found == t // block for t in range(capacity))
    with pytest.raises(ValueError, match="scales"):
        C.block_of(4096, 5)


def test_new_cache():
    keys, values, ks, vs = C.new_cache_q8(2, 3, 100, 64, block=32, dtype=torch.int8, device="cpu")
    assert keys.shape == values.shape == (2, 3, 100, 64) and ks.shape == vs.shape == (2, 3, 4)
    assert keys.dtype == torch.int8 and not keys.any() and torch.all(ks == 1)
    assert keys.data_ptr() != values.data_ptr() and ks.data_ptr() != vs.data_ptr()
    with pytest.raises(ValueError, match="block"):
        C.new_cache_q8(1, 1, 16, 64, block=48, device="cpu")
    with pytest.raises(ValueError, match="type"):
        C.new_cache_q8(1, 1, 16, 64, dtype=torch.bfloat16, device="cpu")


def test_intervals_fill_the_device_and_no_more():
    lib = _native.lib()
    for batch, kv, capacity in ((1, 8, 32768), (1, 1, 16), (32, 8, 16384), (4, 2, 777), (1000, 8, 131072), (1, 1, (1 << 30) - 1)):
        splits = lib.ftk_decode_attention_q8_splits(batch, 4 * kv, kv, capacity, 128, 256)
        assert 1 <= splits <= 1024 and splits <= -(-capacity // 64)
        need = lib.ftk_decode_attention_q8_workspace_bytes(batch, 4 * kv, kv, 128, splits)
        assert need == (0 if splits == 1 else batch * 4 * kv * splits * 130 * 4)
    for bad in ((0, 8, 8, 64, 128), (1, 9, 8, 64, 128), (1, 17, 1, 64, 128), (1, 8, 8, 0, 128), (1, 8, 8, 64, 96)):
        assert lib.ftk_decode_attention_q8_splits(*bad, 256) == -1
    assert lib.ftk_decode_attention_q8_workspace_bytes(1, 8, 8, 128, 0) == -1
    assert lib.ftk_decode_attention_q8_workspace_bytes(1, 8, 8, 128, 1025) == -1


def cache(**kw):
    return C.new_cache_q8(2, 2, 64, 64, block=16, device="cpu", **kw)


def test_attention_refusals():
    keys, values, ks, vs = cache()
    q = torch.zeros((2, 4, 1, 64), dtype=torch.bfloat16)
    p = torch.zeros(2, dtype=torch.int64)

    def refused(match, q=q, keys=keys, values=values, ks=ks, vs=vs, p=p):
        with pytest.raises(ValueError, match=match):
            C.decode_attention_q8(q, keys, values, ks, vs, p, 1.0)

    refused("GPU")
    refused("BF16", q=q.float())
    refused("BF16", q=q[:1])
    refused("BF16", q=torch.zeros((2, 4, 2, 64), dtype=torch.bfloat16))
    refused("heads", q=q[:, :3])
    refused("heads", q=q.repeat(1, 10, 1, 1))
    refused("heads", q=q[:, :0])
    refused("8-bit", keys=keys.to(torch.bfloat16))
    refused("8-bit", values=values.view(torch.int8))
    refused("8-bit", ks=ks.double())
    refused("fit", values=values[:, :1])
    refused("fit", ks=ks[:, :, :2])
    refused("contiguous", ks=ks.expand(2, 2, 4).transpose(0, 1), vs=vs)
    refused("scales", ks=torch.ones((2, 2, 3)), vs=torch.ones((2, 2, 3)))
    refused("contiguous", keys=keys.view(torch.uint8).transpose(0, 1).view(keys.dtype))
    refused("position", p=p.int())
    refused("position", p=torch.zeros(3, dtype=torch.int64))
    refused("position", p=torch.zeros((2, 1), dtype=torch.int64))
    wide = torch.zeros((2, 2, 64, 96), dtype=torch.int8)
    refused("head_dim", keys=wide, values=wide)


def test_write_refusals():
    keys, values, ks, vs = cache()
    norm = SimpleNamespace(weight=torch.ones(64, dtype=torch.bfloat16), variance_epsilon=1e-6)
    packed = torch.zeros((2, 3, 8 * 64), dtype=torch.bfloat16)
    table = torch.zeros((64, 64), dtype=torch.bfloat16)
    phases = torch.zeros((2, 3), dtype=torch.int64)
    position = torch.zeros(2, dtype=torch.int64)

    def refused(match, packed=packed, norm=norm, cos=table, sin=table, position=position, rows=True, phases=phases, **kw):
        with pytest.raises(ValueError, match=match):
            C.qk_rope_cache_q8(packed, norm, norm, cos, sin, position, keys, values, ks, vs, 4, rows=rows, phases=phases,
                               **kw)

    refused("GPU")
    refused("packed", packed=packed[:, :, :448])
    refused("packed", packed=packed[:1])
    refused("BF16", packed=packed.float())
    refused("BF16", cos=table.float())
    refused("BF16", norm=SimpleNamespace(weight=torch.ones(64), variance_epsilon=1e-6))
    refused("gains", norm=SimpleNamespace(weight=torch.ones(128, dtype=torch.bfloat16), variance_epsilon=1e-6))
    refused("contiguous", packed=packed.transpose(1, 2).contiguous().transpose(1, 2))
    refused("prompt", prefill=True)
    refused("phases", rows=False)
    refused("phases", phases=phases.int())
    refused("tables", cos=table[:, :32].contiguous())
    refused("rows of", phases=None)
    refused("position", position=position[:1])
    refused("position", position=position.int())
    refused("tokens", packed=torch.zeros((2, 65, 512), dtype=torch.bfloat16), phases=None)


def test_entry_points_refuse_bad_calls():
    lib, p = _native.lib(), 1 << 12

    def attend(q=p, k=p, out=p, positions=1, b=2, hq=8, hkv=2, c=64, d=128, block=16, kind=0, splits=1, ws=None, size=0):
        return lib.ftk_decode_attention_q8(q, k, p, p, p, p, positions, out, b, hq, hkv, c, d, block, kind, 1.0, splits,
                                           ws, size, None)

    invalid, unsupported = _native.FTK_ERR_INVALID, _native.FTK_ERR_UNSUPPORTED
    assert attend(q=None) == attend(b=0) == attend(hq=7) == attend(c=0) == attend(block=24) == attend(kind=2) == invalid
    assert attend(positions=3) == attend(splits=-1) == attend(splits=1025) == attend(hkv=0) == invalid
    assert attend(d=96) == attend(hq=34) == attend(q=p + 2) == attend(k=p + 8) == attend(out=p + 8) == unsupported
    assert attend(splits=2) == attend(splits=2, ws=p, size=2 * 8 * 2 * 130 * 4 - 1) == _native.FTK_ERR_WORKSPACE
    assert attend(splits=2, ws=p + 8, size=1 << 20) == _native.FTK_ERR_WORKSPACE

    def write(packed=p, query=p, keys=p, position=p, phases=None, b=2, t=3, hq=4, hkv=2, c=64, d=64, block=16, kind=0,
              mode=0, rows=64):
        return lib.ftk_qk_rope_cache_q8(packed, p, p, 1e-6, 1e-6, p, p, rows, position, phases, query, keys, p, p, p, b, t,
                                        hq, hkv, c, d, block, kind, mode, None)

    assert write(packed=None) == write(position=None) == write(t=0) == write(t=65) == write(block=256) == invalid
    assert write(kind=-1) == write(mode=8) == write(mode=_native.ROPE_TABLE) == write(rows=2) == invalid
    assert write(mode=_native.ROPE_ROWS, rows=5) == write(mode=_native.ROPE_ROWS | _native.ROPE_PREFILL) == invalid
    assert write(d=32) == write(packed=p + 1) == write(query=p + 2) == write(keys=p + 8) == unsupported


@pytest.mark.parametrize("splits", [-1, 1025, (1 << 32) + 1])
def test_interval_counts_refused(splits):
    with pytest.raises(ValueError):
        C._launch(0, 1, 8, 2, 64, 128, splits)
