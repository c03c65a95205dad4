"""The 8-bit cache's writer and its attention against their definitions in 64 bits.

Writer bounds. A code is its value over the block's scale rounded to nearest: off by half a step of the code, and by
the FP32 chain before it (norm, gain, two products and a sum: under 16 roundings, 2^-20 of the largest term). Scales
are powers of two and equal. Re-scaled slots are the old codes times a power of two rounded once: equal.
Attention bounds: see ``attend_bound``.
"""

from types import SimpleNamespace

import pytest
import torch

from kernels import cache_q8 as C

pytestmark = pytest.mark.gpu
EPS = 1e-6
TOP = {torch.float8_e4m3fn: 448.0, torch.int8: 127.0}
KINDS = [torch.float8_e4m3fn, torch.int8]


def power(amax, kind):
    """The smallest power of two s >= 2^-126 with amax <= top s, by trial."""
    s = torch.exp2(torch.floor(torch.log2(amax.clamp(min=2.0**-140) / TOP[kind])) - 1)
    for _ in range(3):
        s = torch.where(amax > TOP[kind] * s, 2 * s, s)
    return s.clamp(min=2.0**-126)


def encode(x, kind):
    x = torch.where(x.isnan(), x, x.clamp(-TOP[kind], TOP[kind]))
    return x.nan_to_num(0.0).round().to(kind) if kind == torch.int8 else x.float().to(kind)


def half_step(x, kind):
    if kind == torch.int8:
        return torch.full_like(x, 0.5)
    return torch.exp2(torch.floor(torch.log2(x.abs().clamp(min=2.0**-6))) - 4)


def rope(x, gain, cos, sin):
    """[..., D] in 64 bits, and the largest term of each element."""
    n = x / (x.pow(2).mean(dim=-1, keepdim=True) + EPS).sqrt() * gain
    a, b = n.chunk(2, dim=-1)
    rot = torch.cat((-b, a), dim=-1)
    return n * cos + rot * sin, torch.maximum((n * cos).abs(), (rot * sin).abs())


class Writer:
    def __init__(self, cuda, batch, kv, capacity, dim, block, kind, q_heads, seed=0):
        self.gen = torch.Generator(device=cuda).manual_seed(seed)
        self.cuda, self.kv, self.q_heads, self.dim, self.block, self.kind = cuda, kv, q_heads, dim, block, kind
        self.cache = C.new_cache_q8(batch, kv, capacity, dim, block, kind, cuda)
        self.q_norm, self.k_norm = (SimpleNamespace(weight=self.randn((dim,), 0.1, 1.0), variance_epsilon=EPS)
                                    for _ in range(2))
        angles = torch.arange(capacity, device=cuda)[:, None] * 1e4 ** (-torch.arange(0, dim, 2, device=cuda) / dim)
        angles = torch.cat((angles, angles), dim=1)
        self.cos, self.sin = angles.cos().to(torch.bfloat16), angles.sin().to(torch.bfloat16)

    def randn(self, shape, scale=1.0, shift=0.0):
        return (torch.randn(shape, generator=self.gen, device=self.cuda) * scale + shift).to(torch.bfloat16)

    def packed(self, tokens, scale=1.0):
        batch = self.cache[0].shape[0]
        return self.randn((batch, tokens, (self.q_heads + 2 * self.kv) * self.dim), scale)

    def check(self, packed, position, **kw):
        """One call against the definition; ``position`` a list of each row's first slot (None: a prompt)."""
        keys, values, ks, vs = self.cache
        batch, tokens = packed.shape[:2]
        capacity = keys.shape[2]
        before = [t.clone() for t in self.cache]
        table, phases = None, None
        if position is None:
            first, pos = [0] * batch, torch.arange(tokens, device=self.cuda)
            table = torch.arange(tokens, device=self.cuda).expand(batch, tokens)
            cos, sin = self.cos[:tokens].contiguous(), self.sin[:tokens].contiguous()
            args = dict(prefill=True)
        elif "phases" in kw:
            first, pos, phases = position, torch.tensor(position, device=self.cuda), kw["phases"]
            table, cos, sin = pos[:, None] + phases, self.cos, self.sin
            args = dict(rows=True, phases=phases)
        elif len(position) == 1 and batch > 1:
            first, pos = position * batch, torch.tensor(position, device=self.cuda)
            table = torch.arange(tokens, device=self.cuda).expand(batch, tokens)
            cos, sin = self.cos[:tokens].contiguous(), self.sin[:tokens].contiguous()
            args = dict()
        else:
            first, pos = position, torch.tensor(position, device=self.cuda)
            table = torch.arange(batch * tokens, device=self.cuda).view(batch, tokens)
            cos, sin = (t[table.flatten() % capacity].contiguous() for t in (self.cos, self.sin))
            args = dict(rows=True)
        query = C.qk_rope_cache_q8(packed, self.q_norm, self.k_norm, cos, sin, pos, keys, values, ks, vs, self.q_heads, **args)
        assert query.shape == (batch, self.q_heads, tokens, self.dim)
        good = (table >= 0) & (table < cos.numel() // self.dim)
        at = table.clamp(0, cos.numel() // self.dim - 1)
        c, s = (t.double().view(-1, self.dim)[at][:, :, None] for t in (cos, sin))
        heads = packed.double().view(batch, tokens, -1, self.dim)
        q, q_term = rope(heads[:, :, : self.q_heads], self.q_norm.weight.double(), c, s)
        k, k_term = rope(heads[:, :, self.q_heads : self.q_heads + self.kv], self.k_norm.weight.double(), c, s)
        v = heads[:, :, self.q_heads + self.kv :]
        off = (query.transpose(1, 2).double() - q).abs()
        assert torch.all((off <= 2.0**-8 * q.abs() + 2.0**-20 * q_term)[good])
        for new, term, codes, scales, old, old_scales in ((k, k_term, keys, ks, before[0], before[2]),
                                                          (v, torch.zeros_like(v), values, vs, before[1], before[3])):
            want, want_scales = old.clone(), old_scales.clone()
            raw = want.view(torch.uint8)
            fresh = torch.zeros(old.shape[:3], dtype=torch.bool, device=self.cuda)
            for b in range(batch):
                slots = [(first[b] + t, t) for t in range(tokens) if 0 <= first[b] + t < capacity]
                begin = max(first[b], 0)
                for blk in sorted({slot // self.block for slot, _ in slots}):
                    mine = [(slot, t) for slot, t in slots if slot // self.block == blk and bool(good[b, t])]
                    if not mine:
                        continue
                    low = max(begin, blk * self.block)
                    values_in = torch.stack([new[b, t] for _, t in mine], dim=1)  # [Hkv, slots, D]
                    finite = torch.where(values_in.isfinite(), values_in.abs(), 0.0)
                    scale = power(finite.amax(dim=(1, 2)), self.kind)
                    if low > blk * self.block:
                        was = old_scales[b, :, blk].double()
                        scale = torch.maximum(scale, was)
                        part = old[b, :, blk * self.block : low].double() * (was / scale)[:, None, None]
                        grown = (scale > was)[:, None, None]
                        raw[b, :, blk * self.block : low] = torch.where(
                            grown, encode(part, self.kind).view(torch.uint8), raw[b, :, blk * self.block : low])
                    want_scales[b, :, blk] = scale.float()
                    for slot, t in mine:
                        fresh[b, :, slot] = True
                        code = new[b, t] / scale[:, None]
                        code = torch.where(code.isnan(), code, code.clamp(-TOP[self.kind], TOP[self.kind]))
                        if self.kind == torch.int8:
                            code = code.nan_to_num(0.0)
                        got = codes[b, :, slot].double()
                        slack = 2.0**-20 * term[b, t] / scale[:, None]
                        ok = (got - code).abs() <= half_step(code, self.kind) * (1 + 2.0**-10) + slack
                        assert torch.all(ok | (got.isnan() & code.isnan())), (b, slot)
            assert torch.equal(scales, want_scales)
            same = codes.view(torch.uint8) == raw
            nan = codes.double().isnan() & want.double().isnan()
            assert torch.all((same | nan)[~fresh])  # everything that was not written, and what was re-scaled


SHAPES = [(1, 1, 64, 64, 16, 1), (2, 2, 100, 128, 16, 4), (3, 1, 200, 64, 32, 14), (2, 3, 300, 128, 64, 5),
          (1, 8, 400, 128, 128, 32), (4, 2, 260, 64, 128, 6)]


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("batch,kv,capacity,dim,block,q_heads", SHAPES)
def test_prompt_then_tokens(cuda, batch, kv, capacity, dim, block, q_heads, kind):
    w = Writer(cuda, batch, kv, capacity, dim, block, kind, q_heads)
    w.check(w.packed(min(capacity, 2 * block + 3)), None)
    at = min(capacity, 2 * block + 3)
    for i in range(6):  # tokens that grow: the blocks' scales rise and their earlier slots are re-scaled
        if at + i < capacity:
            w.check(w.packed(1, 2.0**i), [at + i], **({} if batch > 1 else {"phases": torch.zeros((1, 1), dtype=torch.int64, device=cuda)}))


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("batch,kv,capacity,dim,block,q_heads", SHAPES[1:4] + SHAPES[5:])
def test_rows_at_their_own_places(cuda, batch, kv, capacity, dim, block, q_heads, kind):
    """Per-row positions: inside blocks, at their starts, across their ends, before and past the cache."""
    w = Writer(cuda, batch, kv, capacity, dim, block, kind, q_heads, seed=1)
    w.check(w.packed(capacity), None)
    for tokens, places in ((1, [0, block, block - 1, capacity - 1]), (3, [block - 1, 5, capacity - 2, -2]),
                           (block + 1, [block - 2, 1, capacity - 1, capacity]), (2 * block, [7, 0, -block, -5])):
        if tokens <= capacity:
            zeros = torch.zeros((batch, tokens), dtype=torch.int64, device=cuda) + torch.arange(tokens, device=cuda)
            w.check(w.packed(tokens, 4.0), places[:batch], phases=zeros)
            w.check(w.packed(tokens, 8.0), places[:batch])
    far = torch.zeros((batch, 1), dtype=torch.int64, device=cuda)
    w.check(w.packed(1), [2**62, -(2**62), -1, capacity][:batch], phases=far)


@pytest.mark.parametrize("kind", KINDS)
def test_tokens_without_a_table_row_are_skipped(cuda, kind):
    w = Writer(cuda, 2, 2, 96, 64, 16, kind, 4, seed=2)
    w.check(w.packed(90), None)
    phases = torch.tensor([[0, 1, 10**6, 3], [-1000, -1000, -1000, -1000]], device=cuda)
    w.check(w.packed(4), [40, 50], phases=phases)


@pytest.mark.parametrize("kind", KINDS)
def test_values_that_are_not_finite(cuda, kind):
    """Infinities saturate and do not set the scale; NaN stays in e4m3 and is 0 in int8; zeros have the least scale."""
    w = Writer(cuda, 2, 2, 64, 64, 16, kind, 2, seed=3)
    packed = w.packed(20)
    heads = packed.view(2, 20, 6, 64)
    heads[0, 3, 4, 5], heads[0, 9, 5, 60], heads[1, 4, 4, 0] = float("inf"), -float("inf"), float("nan")
    heads[1, 16:, 5] = 0
    w.check(packed, None)
    assert w.cache[3][1, 1, 1] == 2.0**-126


def test_int8_growth_costs_less_than_a_step(cuda):
    """A token's code after any number of re-scalings is within one step of its value over the final scale."""
    w = Writer(cuda, 1, 1, 16, 128, 16, torch.int8, 1, seed=4)
    phases = torch.zeros((1, 1), dtype=torch.int64, device=cuda)
    tokens = [w.packed(1, 2.0 ** (i / 2)) for i in range(16)]
    for i, packed in enumerate(tokens):
        w.check(packed, [i], phases=phases)
    value = torch.cat([p.view(3, 128)[2:] for p in tokens]).double() / w.cache[3].double().view(1)
    assert torch.all((w.cache[1].double().view(16, 128) - value).abs() <= 1)


def test_write_captured(cuda):
    w = Writer(cuda, 2, 2, 64, 64, 16, torch.float8_e4m3fn, 4, seed=5)
    other = Writer(cuda, 2, 2, 64, 64, 16, torch.float8_e4m3fn, 4, seed=5)
    packed, position = w.packed(1), torch.zeros(2, dtype=torch.int64, device=cuda)
    phases = torch.zeros((2, 1), dtype=torch.int64, device=cuda)

    def step(w):
        return C.qk_rope_cache_q8(packed, w.q_norm, w.k_norm, w.cos, w.sin, position, *w.cache, 4, rows=True, phases=phases)

    step(w)
    stream, graph = torch.cuda.Stream(), torch.cuda.CUDAGraph()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream), torch.cuda.graph(graph, stream=stream):
        query = step(w)
    torch.cuda.current_stream().wait_stream(stream)
    for i in range(20):
        packed.copy_(w.packed(1, 1 + i))
        position.copy_(torch.tensor([i, 2 * i], device=cuda))
        graph.replay()
        assert torch.equal(query, step(other))
        for a, b in zip(w.cache, other.cache):
            assert torch.equal(a.view(torch.uint8), b.view(torch.uint8))


# ---- attention ----------------------------------------------------------------------------------


def make(cuda, batch, q_heads, kv, capacity, dim, block, kind, seed=0):
    g = torch.Generator(device=cuda).manual_seed(seed)
    q = torch.randn((batch, q_heads, 1, dim), generator=g, device=cuda).to(torch.bfloat16)
    out = [q]
    for _ in range(2):
        if kind == torch.int8:
            codes = torch.randint(-127, 128, (batch, kv, capacity, dim), generator=g, device=cuda, dtype=torch.int8)
        else:
            codes = (torch.randn((batch, kv, capacity, dim), generator=g, device=cuda) * 100).clamp(-448, 448).to(kind)
        out.append(codes)
    for _ in range(2):  # any positive scales, powers of two or not
        scale = torch.rand((batch, kv, -(-capacity // block)), generator=g, device=cuda) + 0.5
        out.append(scale / (64.0 if kind == torch.int8 else 100.0))
    return out


def check_attention(cuda, q, keys, values, ks, vs, position, scale, block, splits=0):
    """out against softmax(q k) v in 64 bits.

    The bound: half a BF16 step of the output, 2^-8, and of sum p |v| / sum p: p's 16 bits (2^-16), its exp2
    (2^-21), FP32 sums over the slots (n + 64 roundings at worst, far fewer as they are summed by parts), and twice
    the error of a score, 24 roundings of at most sum |q| |k| scale each and two of its products.
    """
    got = C.decode_attention_q8(q, keys, values, ks, vs, position, scale, splits=splits)
    batch, q_heads, _, dim = q.shape
    kv, capacity = keys.shape[1:3]
    share = q_heads // kv
    assert got.shape == (batch, 1, q_heads, dim) and got.is_contiguous()
    for b in range(batch):
        n = min(int(position[b if len(position) > 1 else 0]), capacity - 1) + 1
        if n <= 0:
            assert not got[b].any()
            continue
        at = torch.arange(n, device=cuda) // block
        k = keys[b, :, :n].double() * ks[b].double()[:, at, None]
        v = values[b, :, :n].double() * vs[b].double()[:, at, None]
        qb = q[b, :, 0].double().view(kv, share, dim)
        kt = k.transpose(1, 2).contiguous()
        p = torch.softmax(qb @ kt * scale, dim=-1)
        want = (p @ v).view(q_heads, dim)
        size = (p @ v.abs()).view(q_heads, dim)
        score = 26 * 2.0**-24 * float((qb.abs() @ kt.abs()).max()) * scale
        bound = 2.0**-8 * want.abs() + (2.0**-16 + 2.0**-20 + 2.0**-24 * (n**0.5 * 8 + 64) + 2 * score) * size
        assert torch.all((got[b, 0].double() - want).abs() <= bound), b
    return got


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("dim,block", [(64, 16), (64, 128), (128, 32), (128, 64)])
@pytest.mark.parametrize("capacity", [1, 15, 16, 17, 63, 64, 65, 255, 257, 1000, 4096])
def test_attention_lengths(cuda, capacity, dim, block, kind):
    q, *cache = make(cuda, 3, 8, 2, capacity, dim, block, kind, seed=capacity)
    for p in (torch.tensor([capacity - 1], device=cuda), torch.tensor([0, capacity // 2, capacity - 1], device=cuda),
              torch.tensor([-1, capacity + 5, capacity // 3], device=cuda)):
        check_attention(cuda, q, *cache, p, dim**-0.5, block)


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("share", [1, 2, 3, 5, 7, 8, 12, 16])
def test_attention_heads(cuda, share, dim, kind):
    q, *cache = make(cuda, 2, 3 * share, 3, 700, dim, 64, kind, seed=share)
    check_attention(cuda, q, *cache, torch.tensor([650, 3], device=cuda), 0.125, 64)


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("splits", [1, 2, 3, 7, 16, 64, 1024])
def test_attention_intervals(cuda, splits, kind):
    q, *cache = make(cuda, 2, 8, 2, 3001, 128, 16, kind, seed=splits)
    check_attention(cuda, q, *cache, torch.tensor([3000, 700], device=cuda), 128**-0.5, 16, splits)
    check_attention(cuda, q, *cache, torch.tensor([-1, 0], device=cuda), 128**-0.5, 16, splits)


def test_attention_ignores_what_lies_past_the_position(cuda):
    """NaN codes and NaN scales after the position, also inside the last visible block and unit."""
    q, keys, values, ks, vs = make(cuda, 3, 8, 2, 500, 128, 16, torch.float8_e4m3fn, seed=9)
    position = torch.tensor([0, 203, 499], device=cuda)
    want = check_attention(cuda, q, keys, values, ks, vs, position, 0.09, 16)
    for b, p in enumerate(position.tolist()):
        keys.view(torch.uint8)[b, :, p + 1 :] = 0x7F
        values.view(torch.uint8)[b, :, p + 1 :] = 0xFF
        ks[b, :, p // 16 + 1 :] = float("nan")
        vs[b, :, p // 16 + 1 :] = float("nan")
    assert torch.equal(C.decode_attention_q8(q, keys, values, ks, vs, position, 0.09), want)
    keys.view(torch.uint8)[1, 0, 203, 5] = 0x7F  # a NaN the row does see
    got = C.decode_attention_q8(q, keys, values, ks, vs, position, 0.09)
    assert got[1, 0, :4].isnan().all() and torch.equal(got[1, 0, 4:], want[1, 0, 4:]) and torch.equal(got[[0, 2]], want[[0, 2]])


def test_attention_extreme_scores(cuda):
    """Scores far apart (one slot takes all), all equal, and scales that are tiny or huge."""
    q, keys, values, ks, vs = make(cuda, 1, 4, 1, 300, 64, 32, torch.int8, seed=10)
    p = torch.tensor([299], device=cuda)
    check_attention(cuda, q, keys, values, ks, vs, p, 0.0, 32)
    for s in (2.0**-100, 2.0**60):
        check_attention(cuda, q, keys, values, ks, vs * s, p, 0.125, 32)
    keys[0, 0, 137] = torch.where(q[0, 0, 0] > 0, 127, -127).to(torch.int8)
    got = C.decode_attention_q8(q, keys, values, ks * 100, vs, p, 1.0)
    want = values[0, 0, 137].double() * vs[0, 0, 137 // 32].double()
    assert torch.allclose(got[0, 0, 0].double(), want, rtol=2.0**-8, atol=0)


def test_attention_unaligned_query_and_views(cuda):
    q, *cache = make(cuda, 2, 4, 2, 100, 64, 16, torch.int8, seed=11)
    p = torch.tensor([99, 50], device=cuda)
    want = C.decode_attention_q8(q, *cache, p, 0.125)
    store = torch.empty(q.numel() + 1, dtype=torch.bfloat16, device=cuda)
    odd = store[1:].view(q.shape)
    odd.copy_(q)
    wide = torch.empty((2, 1, 4, 96), dtype=torch.bfloat16, device=cuda)
    wide[:, 0, :, 7:71] = q[:, :, 0]
    assert torch.equal(C.decode_attention_q8(odd, *cache, p, 0.125), want)
    assert torch.equal(C.decode_attention_q8(wide[:, :, :, 7:71].transpose(1, 2), *cache, p, 0.125), want)


def test_attention_empty_batch(cuda):
    q, *cache = make(cuda, 2, 4, 2, 100, 64, 16, torch.int8)
    got = C.decode_attention_q8(q[:0], *(t[:0].contiguous() for t in cache), torch.zeros(1, dtype=torch.int64, device=cuda), 1.0)
    assert got.shape == (0, 1, 4, 64)


def test_offsets_past_32_bits(cuda):
    """66 x 8 heads x 65536 slots x 128: 4.4 GB of codes each. The last rows' writes and reads land in their own slots."""
    batch, kv, capacity, dim, block = 66, 8, 65536, 128, 64
    cache = C.new_cache_q8(batch, kv, capacity, dim, block, torch.float8_e4m3fn, cuda)
    small = C.new_cache_q8(2, kv, 256, dim, block, torch.float8_e4m3fn, cuda)
    g = torch.Generator(device=cuda).manual_seed(12)
    packed = torch.randn((batch, 200, (8 + 2 * kv) * dim), generator=g, device=cuda).to(torch.bfloat16)
    norm = SimpleNamespace(weight=torch.ones(dim, dtype=torch.bfloat16, device=cuda), variance_epsilon=EPS)
    table = torch.rand((200, dim), generator=g, device=cuda).to(torch.bfloat16)
    position = torch.arange(200, device=cuda)
    q = C.qk_rope_cache_q8(packed, norm, norm, table, table, position, *cache, 8, prefill=True)
    pick = torch.tensor([0, batch - 1], device=cuda)
    q2 = C.qk_rope_cache_q8(packed[pick].contiguous(), norm, norm, table, table, position, *small, 8, prefill=True)
    assert torch.equal(q[pick], q2)
    for a, b in zip(cache[:2], small[:2]):
        assert torch.equal(a.view(torch.uint8)[pick][:, :, :256], b.view(torch.uint8))
    at = torch.tensor([199], device=cuda)
    one = q[:, :, -1:].contiguous()
    got = C.decode_attention_q8(one, *cache, at, 0.09)
    want = C.decode_attention_q8(one[pick].contiguous(), *small, at, 0.09)
    assert (got[pick].float() - want.float()).abs().max() <= 2.0**-7 * want.float().abs().max()


def test_two_captured_graphs_side_by_side(cuda):
    """Two graphs of split attention replayed on two streams at once: each keeps partials of its own."""
    graphs, outs, wants = [], [], []
    for seed in (13, 14):
        q, *cache = make(cuda, 1, 8, 2, 9000, 128, 64, torch.float8_e4m3fn, seed=seed)
        p = torch.tensor([8999], device=cuda)
        wants.append(C.decode_attention_q8(q, *cache, p, 0.09))
        stream, graph = torch.cuda.Stream(), torch.cuda.CUDAGraph()
        stream.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(stream), torch.cuda.graph(graph, stream=stream):
            outs.append(C.decode_attention_q8(q, *cache, p, 0.09))
        graphs.append((graph, stream, q, cache, p))
    torch.cuda.synchronize()
    for _ in range(20):
        for graph, stream, *_ in graphs:
            with torch.cuda.stream(stream):
                graph.replay()
        torch.cuda.synchronize()
        for out, want in zip(outs, wants):
            assert torch.equal(out, want)
            out.zero_()
        torch.cuda.synchronize()


def test_written_cache_attends_like_the_bf16_one(cuda):
    """Prompt and tokens through the writer, then attention: near the same steps over the BF16 cache (8-bit keys and
    values are off by 2^-4 of themselves at most, averaged over 64 or more dimensions and slots), and exactly the
    attention over the written values."""
    from kernels import decode_attention as A
    from kernels import qk_rope as R

    w = Writer(cuda, 2, 2, 300, 128, 64, torch.float8_e4m3fn, 8, seed=15)
    keys, values = (torch.zeros((2, 2, 300, 128), dtype=torch.bfloat16, device=cuda) for _ in range(2))
    packed = w.packed(200)
    position = torch.arange(200, device=cuda)
    cos, sin = w.cos[:200].contiguous(), w.sin[:200].contiguous()
    C.qk_rope_cache_q8(packed, w.q_norm, w.k_norm, cos, sin, position, *w.cache, 8, prefill=True)
    R.qk_rope_cache(packed, w.q_norm, w.k_norm, cos, sin, position, keys, values, 8, prefill=True)
    for t in range(200, 210):
        packed, at = w.packed(1), torch.tensor([t, t], device=cuda)
        phases = torch.zeros((2, 1), dtype=torch.int64, device=cuda)
        q = C.qk_rope_cache_q8(packed, w.q_norm, w.k_norm, w.cos, w.sin, at, *w.cache, 8, rows=True, phases=phases)
        q16 = R.qk_rope_cache(packed, w.q_norm, w.k_norm, w.cos, w.sin, at, keys, values, 8, rows=True, phases=phases)
        got = check_attention(cuda, q, *w.cache, at, 128**-0.5, 64)
        want = A.attend(q16.reshape(2, 8, 128).contiguous(), keys, values, at, 128**-0.5)
        assert (got.float() - want.float()).norm() <= 2.0**-4 * want.float().norm()
