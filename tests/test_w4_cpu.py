"""The 4-bit weights' packed layout and argument checks, on the CPU."""

import numpy as np
import pytest
import torch

from kernels import _native, w4


def unpack(weight):
    """(codes, scales, zeros) [rows, columns] of a W4Weight, by the layout's definition in include/ftk.h."""
    codes = weight.codes.numpy().view(np.uint32)
    tiles, chunks = codes.shape[:2]
    n, k = tiles * 16, chunks * 128
    q, s, z = np.zeros((n, k)), np.zeros((n, k)), np.full((n, k), 8.0)
    scales = weight.scales.float().numpy()
    for t in range(tiles):
        for c in range(chunks):
            for lane in range(64):
                li, g = lane % 16, lane // 16
                for step in range(4):
                    for e in range(8):
                        col = 128 * c + 32 * step + 8 * g + e
                        at = (32 * step + 8 * g) // weight.group
                        q[16 * t + li, col] = (codes[t, c, lane, step] >> (4 * (e // 2) + 16 * (e % 2))) & 15
                        s[16 * t + li, col] = scales[t, c, li, at]
                        if weight.zeros is not None:
                            z[16 * t + li, col] = weight.zeros[t, c, li, at]
    if weight.gate_up:
        half = weight.rows // 2
        order = [t * 16 + r for part in (0, 8) for t in range(tiles) for r in range(part, part + 8) if 8 * t + r - part < half]
    else:
        order = list(range(weight.rows))
    return tuple(a[order][:, : weight.columns] for a in (q, s, z))


def parts(n, k, group, zeros, seed=0, dtype=torch.bfloat16):
    g = torch.Generator().manual_seed(seed)
    groups = -(-k // group)
    codes = torch.randint(0, 16, (n, k), generator=g, dtype=torch.uint8)
    scales = (torch.rand((n, groups), generator=g) + 0.5).to(dtype)
    z = torch.randint(0, 16, (n, groups), generator=g, dtype=torch.uint8) if zeros else None
    return codes, scales, z


@pytest.mark.parametrize("n,k,group,zeros,gate_up", [
    (16, 128, 128, False, False), (17, 130, 32, True, False), (33, 257, 64, False, False), (1, 1, 32, True, False),
    (20, 300, 256, True, False), (18, 200, 200, False, False), (34, 140, 64, True, True), (2, 128, 128, False, True),
    (48, 384, 128, True, True), (40, 50, 64, False, True)])
def test_packed_layout_is_the_documented_one(n, k, group, zeros, gate_up):
    codes, scales, z = parts(n, k, group, zeros)
    q, s, zz = unpack(w4.pack_w4(codes, scales, z, group, gate_up))
    wide = np.arange(k) // group
    assert np.array_equal(q, codes.numpy())
    assert np.array_equal(s, scales.float().numpy()[:, wide])
    assert np.array_equal(zz, np.full((n, k), 8.0) if z is None else z.numpy()[:, wide])


@pytest.mark.parametrize("gate_up", [False, True])
def test_packing_in_slabs_is_packing_at_once(monkeypatch, gate_up):
    codes, scales, z = parts(150, 300, 32, True)
    whole = w4.pack_w4(codes, scales, z, 32, gate_up)
    monkeypatch.setattr(w4, "_SLAB", 3 * 16 * 384)
    assert torch.equal(whole.codes, w4.pack_w4(codes, scales, z, 32, gate_up).codes)


def test_round_to_nearest_codes():
    weight = (torch.randn(24, 300, generator=torch.Generator().manual_seed(1))).to(torch.bfloat16)
    weight[3, :128] = 0
    q, s, z = unpack(w4.quantize_w4(weight, 128))
    value = (q - z) * s
    # Half a step, and what the scale's own rounding (2^-8 of 7 steps) can clip off the largest value.
    assert np.all(np.abs(value - weight.float().numpy()) <= s * (0.5 + 7 * 2**-8) + 1e-30)
    assert np.all(value[3, :128] == 0)


def test_refusals():
    codes, scales, z = parts(8, 256, 128, True)
    with pytest.raises(ValueError, match="group"):
        w4.pack_w4(codes, scales, None, 96)
    with pytest.raises(ValueError, match="group"):
        w4.pack_w4(codes, scales, None, 0)
    with pytest.raises(ValueError, match="scales"):
        w4.pack_w4(codes, scales[:, :1], None, 128)
    with pytest.raises(ValueError, match="scales"):
        w4.pack_w4(codes, scales.float(), None, 128)
    with pytest.raises(ValueError, match="zeros"):
        w4.pack_w4(codes, scales, z[:4], 128)
    with pytest.raises(ValueError, match="0..15"):
        w4.pack_w4(codes + 1, scales, None, 128)
    with pytest.raises(ValueError, match="uint8"):
        w4.pack_w4(codes.int(), scales, None, 128)
    with pytest.raises(ValueError, match="even"):
        w4.pack_w4(codes[:7], scales[:7], None, 128, gate_up=True)
    rows, gate_up = w4.pack_w4(codes, scales, z, 128), w4.pack_w4(codes, scales, z, 128, gate_up=True)
    x = torch.zeros((2, 256), dtype=torch.bfloat16)
    with pytest.raises(ValueError, match="gate_up"):
        w4.linear_w4(x, gate_up)
    with pytest.raises(ValueError, match="gate_up"):
        w4.gate_up_swiglu_w4(x, rows)
    with pytest.raises(ValueError, match="BF16"):
        w4.linear_w4(x.float(), rows)
    with pytest.raises(ValueError, match="columns"):
        w4.linear_w4(x[:, :128], rows)
    with pytest.raises(ValueError, match="GPU"):
        w4.linear_w4(x, rows)


def test_entry_point_refuses_bad_handles():
    lib = _native.lib()
    codes, scales, _ = parts(16, 128, 128, False)
    weight = w4.pack_w4(codes, scales)

    def status(m=1, x=1 << 12, y=1 << 12, gamma=None, stride=128, residual=None, **change):
        h = _native.W4()
        for name, _ in _native.W4._fields_:
            setattr(h, name, getattr(weight._handle, name))
        for name, value in change.items():
            setattr(h, name, value)
        return lib.ftk_w4_project_bf16(x, stride, gamma, 1e-6, h, residual, y, m, None)

    assert status(m=0) == status(m=33) == _native.FTK_ERR_INVALID
    assert status(x=None) == status(y=None) == status(codes=None) == status(scales=None) == _native.FTK_ERR_INVALID
    assert status(group=96) == status(scale_type=2) == status(layout=2) == status(N=0) == _native.FTK_ERR_INVALID
    assert status(layout=_native.W4_GATE_UP, N=15) == _native.FTK_ERR_INVALID
    assert status(layout=_native.W4_GATE_UP, residual=1 << 12) == _native.FTK_ERR_INVALID
    assert status(m=2, stride=127) == _native.FTK_ERR_INVALID
    assert status(codes=1 << 12 | 8) == status(x=(1 << 12) + 1) == _native.FTK_ERR_UNSUPPORTED
    assert lib.ftk_w4_project_bf16(1 << 12, 128, None, 1e-6, None, None, 1 << 12, 1, None) == _native.FTK_ERR_INVALID
    assert lib.ftk_w4_dequantize_bf16(weight._handle, None, None) == _native.FTK_ERR_INVALID


@pytest.mark.parametrize("shape,group", [((4, 64), 0), ((4, 64), -32), ((0, 64), 32), ((4, 0), 32)])
def test_quantize_refusals(shape, group):
    with pytest.raises(ValueError):
        w4.quantize_w4(torch.ones(shape, dtype=torch.bfloat16), group)
