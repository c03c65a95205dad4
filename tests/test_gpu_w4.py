"""Projections over 4-bit weights against the definition in 64 bits.

Bounds. With integer x, power-of-two scales and every partial sum below 2^24 the FP32 sums are exact, so the output
is the exact result rounded once: compared bit for bit. Otherwise an output may be off by half a BF16 step (2^-8 of it)
and by the FP32 sums: a group of at most 128 columns takes up to 8 matrix instructions of at most 4 roundings each,
of partial sums of at most (143 + 143) sum |x|, and every group's scaled sum is added with one rounding.
"""

import pytest
import torch
from torch.nn import functional as F

from kernels import _native, w4

pytestmark = pytest.mark.gpu


def make(n, k, group, zeros, cuda, seed=0, dtype=torch.bfloat16, exact=False, gate_up=False):
    g = torch.Generator(device=cuda).manual_seed(seed)
    groups = -(-k // group)
    codes = torch.randint(0, 16, (n, k), generator=g, device=cuda, dtype=torch.uint8)
    if exact:
        scales = torch.exp2(torch.randint(-3, 1, (n, groups), generator=g, device=cuda).float()).to(dtype)
    else:
        scales = ((torch.rand((n, groups), generator=g, device=cuda) + 0.5) * 0.004).to(dtype)
    z = torch.randint(0, 16, (n, groups), generator=g, device=cuda, dtype=torch.uint8) if zeros else None
    return w4.pack_w4(codes, scales, z, group, gate_up), codes, scales, z, group


def wide(codes, scales, z, group):
    at = torch.arange(codes.shape[1], device=codes.device) // group
    s = scales.double()[:, at]
    return s * (codes.double() - (8.0 if z is None else z.double()[:, at])), s


def inputs(m, k, cuda, seed=1, exact=False):
    g = torch.Generator(device=cuda).manual_seed(seed)
    if exact:
        return torch.randint(-4, 5, (m, k), generator=g, device=cuda).to(torch.bfloat16)
    return torch.randn((m, k), generator=g, device=cuda).to(torch.bfloat16)


def slack(x, s):
    """The FP32 part of the bound for x [M, K] and per-element scales s [N, K]."""
    groups = x.shape[1] // 32 + 2
    return 2.0**-24 * (32 * 286 + 15 * groups) * (x.double().abs() @ s.t().contiguous())


SHAPES = [(1, 16, 128), (1, 4096, 1024), (3, 130, 257), (16, 256, 4096), (17, 100, 640), (32, 1040, 1531), (5, 9497, 96),
          (8, 1, 1), (2, 15, 7), (31, 33, 12288), (16, 4096, 2048), (24, 512, 8)]


@pytest.mark.parametrize("group", [32, 64, 128])
@pytest.mark.parametrize("zeros", [False, True])
@pytest.mark.parametrize("m,n,k", SHAPES)
def test_linear_exact_sums(cuda, m, n, k, zeros, group):
    weight, *parts = make(n, k, group, zeros, cuda, exact=True)
    x = inputs(m, k, cuda, exact=True)
    want = x.double() @ wide(*parts)[0].t().contiguous()
    assert torch.equal(w4.linear_w4(x, weight), want.to(torch.bfloat16))
    r = inputs(m, n, cuda, 2, exact=True)
    assert torch.equal(w4.linear_residual_w4(x, weight, r), (want + r.double()).to(torch.bfloat16))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("group", [32, 64, 128, 256, 100000])
@pytest.mark.parametrize("m,n,k", [(1, 4096, 1024), (4, 1000, 2570), (16, 640, 4096), (27, 272, 3000)])
def test_linear_random(cuda, m, n, k, group, dtype):
    weight, *parts = make(n, k, group, m % 2 == 0, cuda, dtype=dtype)
    x = inputs(m, k, cuda)
    value, s = wide(*parts)
    want = x.double() @ value.t().contiguous()
    off = (w4.linear_w4(x, weight).double() - want).abs()
    assert torch.all(off <= 2.0**-8 * want.abs() + slack(x, s))


@pytest.mark.parametrize("m,inter,k,group,zeros", [(1, 1536, 1024, 128, False), (5, 100, 640, 64, True), (16, 9, 2048, 32, True),
                                                   (24, 520, 1000, 128, True), (32, 64, 4096, 128, False), (1, 1, 8, 32, False)])
@pytest.mark.parametrize("norm", [False, True])
def test_gate_up_swiglu(cuda, m, inter, k, group, zeros, norm):
    weight, *parts = make(2 * inter, k, group, zeros, cuda, gate_up=True)
    x = inputs(m, k, cuda)
    gain = (inputs(1, k, cuda, 3)[0].float() * 0.1 + 1).to(torch.bfloat16) if norm else None
    value, s = wide(*parts)
    if norm:  # the norm's own roundings: bf16(bf16(x / rms) gain)
        from kernels.rmsnorm import rms_norm
        xn = rms_norm(x, gain, 1e-6)
    else:
        xn = x
    sums = xn.double() @ value.t().contiguous()
    err = slack(xn, s)
    if norm:  # a prologue may sum a row's squares in another order: x / rms lands on the other side of a rounding
        err = err + 2.0**-7 * (xn.double().abs() @ value.abs().t().contiguous()) * 2.0**-4
    gate, up = sums.chunk(2, dim=1)
    eg, eu = err.chunk(2, dim=1)
    want = F.silu(gate) * up
    # silu' is below 1.1 everywhere; silu itself is at most |gate|, and its FP32 exp and division add 2^-21 of it.
    bound = 1.1 * eg * (up.abs() + eu) + gate.abs() * eu + 2.0**-21 * want.abs() + 2.0**-8 * want.abs()
    got = w4.gate_up_swiglu_w4(x, weight, gain, 1e-6)
    assert got.shape == (m, inter)
    assert torch.all((got.double() - want).abs() <= bound + 1e-30)


#: Rows and columns on every path of a launch: one row or several, x held in registers or read in passes, one block of
#: operand rows or two, one row block or two.
LAUNCHES = [(1, 512, 1024), (7, 100, 2570), (16, 272, 4096), (32, 33, 512), (1, 40, 9000), (1, 100, 12288), (1, 33, 25000),
            (2, 40, 9000), (3, 17, 12288), (5, 40, 6200), (9, 40, 4096), (12, 50, 9000), (17, 30, 4096), (24, 64, 12288),
            (32, 20, 5000), (4, 40, 4700), (8, 24, 8192)]


# Enough tiles that a workgroup takes two blocks of operand rows (3 or 4 chunks to a wave), at odd sizes and, for 17 rows
# and 24 under a norm, with row blocks of unequal rows.
@pytest.mark.parametrize("norm", [False, True])
@pytest.mark.parametrize("m,n,k,group", [(17, 19001, 2200, 128), (24, 25003, 3130, 64), (32, 18800, 4096, 128)])
def test_two_blocks_of_rows(m, n, k, group, norm, cuda):
    check_rows(m, n, k, group, norm, cuda)


# Short walks with four chunks to each of eight waves, which 16 waves take: whole and ragged rows, idle waves.
@pytest.mark.parametrize("norm", [False, True])
@pytest.mark.parametrize("group", [32, 64, 128])
@pytest.mark.parametrize("m,n,k", [(2, 333, 3201), (7, 6150, 4096), (9, 40, 3977), (32, 1000, 3400)])
def test_sixteen_waves(m, n, k, group, norm, cuda):
    check_rows(m, n, k, group, norm, cuda)


# Rows of several passes whose walks take two tiles, a batch and one more, two batches and more (32 rows under a norm and
# without: a workgroup walks n / 1024 and n / 2048 tiles).
@pytest.mark.parametrize("norm", [False, True])
@pytest.mark.parametrize("m,n,k,group", [(32, 1500, 8300, 128), (32, 8700, 6200, 64), (32, 17003, 4300, 32),
                                         (9, 4200, 12288, 128)])
def test_batches_of_passes(m, n, k, group, norm, cuda):
    check_rows(m, n, k, group, norm, cuda)


def check_rows(m, n, k, group, norm, cuda):
    weight, *parts = make(n, k, group, group == 64, cuda)
    x, r = inputs(m, k, cuda), inputs(m, n, cuda, 4)
    gain = (inputs(1, k, cuda, 3)[0].float() * 0.1 + 1).to(torch.bfloat16)
    value, s = wide(*parts)
    wx = x.double()
    if norm:
        wx = wx / torch.sqrt((wx * wx).mean(-1, keepdim=True) + 1e-6) * gain.double()
        got = w4.rms_norm_linear_w4(x, gain, 1e-6, weight, residual=r)
    else:
        got = w4.linear_residual_w4(x, weight, r)
    want = wx @ value.t().contiguous() + r.double()
    # (The norm itself: FP32 sums of squares and a root, some roundings of 2^-24 each, within the slack's 2^-16.)
    assert torch.all((got.double() - want).abs() <= 2.0**-8 * want.abs() + slack(wx, s) + 2.0**-20 * want.abs())


@pytest.mark.parametrize("group", [32, 64, 128])
@pytest.mark.parametrize("m,n,k", LAUNCHES)
def test_rms_norm_linear(cuda, m, n, k, group):
    from kernels.rmsnorm import rms_norm

    weight, *parts = make(n, k, group, group == 64, cuda)
    x, r = inputs(m, k, cuda), inputs(m, n, cuda, 4)
    gain = (inputs(1, k, cuda, 3)[0].float() * 0.1 + 1).to(torch.bfloat16)
    xn = rms_norm(x, gain, 1e-6)
    value, s = wide(*parts)
    want = xn.double() @ value.t().contiguous()
    # A sixteenth of the elements, at most, on the other side of a rounding (one step, 2^-7): see above.
    err = slack(xn, s) + 2.0**-11 * (xn.double().abs() @ value.abs().t().contiguous())
    assert torch.all((w4.rms_norm_linear_w4(x, gain, 1e-6, weight).double() - want).abs() <= 2.0**-8 * want.abs() + err)
    both = want + r.double()
    got = w4.rms_norm_linear_w4(x, gain, 1e-6, weight, residual=r)
    assert torch.all((got.double() - both).abs() <= 2.0**-8 * both.abs() + err)


def test_views_strides_and_leading_dimensions(cuda):
    weight, *parts = make(100, 258, 64, True, cuda, exact=True)
    value = wide(*parts)[0].t().contiguous()
    base = inputs(12, 600, cuda, exact=True)
    for x in (base[:, 1:259], base[::3, 7:265], base[:3, 300:558], base[:1].expand(4, 600)[:, 5:263],
              base.t().contiguous().t()[:, :258], base[:6, :258].reshape(2, 3, 258)):
        got = w4.linear_w4(x, weight)
        assert got.shape == (*x.shape[:-1], 100) and got.is_contiguous()
        assert torch.equal(got.reshape(-1, 100), (x.reshape(-1, 258).double() @ value).to(torch.bfloat16))


def test_no_row_leaks_into_another(cuda):
    """A row's outputs do not depend on the other rows, bit for bit, NaN rows included."""
    weight, *_ = make(272, 1000, 32, True, cuda)
    x = inputs(20, 1000, cuda)
    alone = torch.cat([w4.linear_w4(x[i : i + 1], weight) for i in range(20)])
    full = w4.linear_w4(x, weight)
    assert torch.equal(full[:16], w4.linear_w4(x[:16], weight))
    assert (alone.float() - full.float()).abs().max() <= 2.0**-7 * full.float().abs().max()
    x[3] = float("nan")
    got = w4.linear_w4(x, weight)
    keep = [i for i in range(20) if i != 3]
    assert torch.equal(got[keep], full[keep]) and got[3].isnan().all()


def test_infinite_and_huge_activations(cuda):
    """An infinite activation gives that infinity with the sign of q - z (NaN where q = z); 128 x may overflow
    (2^121: beside it the other terms, at most 300 x 60, vanish)."""
    n, k = 64, 300
    weight, *parts = make(n, k, 32, True, cuda, exact=True)
    value = wide(*parts)[0]
    some = value[:, 130] != 0
    for big in (float("inf"), -float("inf"), 2.0**121, -(2.0**121)):
        x = inputs(3, k, cuda, exact=True)
        x[1, 130] = big
        got = w4.linear_w4(x, weight)
        want = x.double() @ value.t().contiguous()
        assert torch.equal(got[[0, 2]], want[[0, 2]].to(torch.bfloat16))
        large = value[:, 130] * big
        assert torch.allclose(got[1][some].double(), large[some], rtol=2.0**-8, atol=0)
        if big in (float("inf"), -float("inf")):
            assert got[1][~some].isnan().all()


def test_empty_and_prompt_rows(cuda):
    weight, *parts = make(272, 256, 128, False, cuda, exact=True)
    assert w4.linear_w4(torch.empty((0, 256), device=cuda, dtype=torch.bfloat16), weight).shape == (0, 272)
    value = wide(*parts)[0]
    x = inputs(77, 256, cuda, exact=True)
    assert torch.equal(w4.linear_w4(x, weight), (x.double() @ value.t().contiguous()).to(torch.bfloat16))
    assert w4.linear_w4(x.view(7, 11, 256), weight).shape == (7, 11, 272)


@pytest.mark.parametrize("n,k,group,zeros,gate_up", [(272, 256, 128, False, False), (33, 130, 32, True, False),
                                                     (34, 200, 64, True, True), (2, 5, 32, False, True)])
def test_dequantize(cuda, n, k, group, zeros, gate_up):
    weight, *parts = make(n, k, group, zeros, cuda, gate_up=gate_up)
    assert torch.equal(w4.dequantize_w4(weight), wide(*parts)[0].to(torch.bfloat16))


def test_captured_and_on_another_stream(cuda):
    weight, *_ = make(1024, 1024, 128, False, cuda)
    x, r = inputs(4, 1024, cuda), inputs(4, 1024, cuda, 5)
    want = w4.linear_residual_w4(x, weight, r)
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.stream(stream):
        assert torch.equal(w4.linear_residual_w4(x, weight, r), want)
        with torch.cuda.graph(graph, stream=stream):
            y = w4.linear_residual_w4(x, weight, r)
    torch.cuda.current_stream().wait_stream(stream)
    for seed in (6, 7, 8):
        x.copy_(inputs(4, 1024, cuda, seed))
        graph.replay()
        assert torch.equal(y, w4.linear_residual_w4(x, weight, r))
