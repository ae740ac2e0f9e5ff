"""Calls of the decode operators at the edges of what they take, on the GPU."""
import pytest
import torch

from nnr_b200 import ops
from test_gpu_decode import HALF, TYPES, attention_ref, filled, generator, layout, near, values, weights

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module", autouse=True)
def device(cuda_dev):
    yield cuda_dev
    torch.cuda.synchronize()
    assert ops.device_status() == 0


def test_attention_of_an_empty_batch_behind_a_prefix():
    cache = ops.KVCache(4, 16, 2, 64)
    table = torch.zeros(1, 2, dtype=torch.int32, device="cuda")
    lens = torch.ones(1, dtype=torch.int32, device="cuda")
    q = torch.zeros(1, 3, 4, 64, device="cuda", dtype=torch.bfloat16)
    y = ops.KVAttention(cache, 4).exec(q[:0], table[:0], lens[:0], prefix_table=table[0], prefix_len=20)
    assert y.shape == (0, 3, 4, 64) and y.dtype == torch.bfloat16


@pytest.mark.parametrize("t", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("kind,batch,prefix,window", [((8, 0, 128, 2, 16), 2, 0, 60), ((4, 32, 128, 2, 16), 2, 0, 60),
                                                      ((8, 0, 256, 1, 16), 2, 0, 60), ((8, 32, 96, 2, 16), 2, 0, 60),
                                                      ((8, 0, 128, 2, 16), 40, 203, 150)])
@pytest.mark.parametrize("zeros", [False, True])
@pytest.mark.parametrize("large", [1e6, 1e38])
def test_attention_large_scales_of_unseen_values(kind, batch, prefix, window, zeros, large, t):
    """Keys that lie in a tile with the window's first, or behind a sequence's
    end, and are not seen: their values' scales do not matter however large they
    are, not even where all that is seen is zero."""
    cache = filled(kind, batch * 7 + 15, 5)
    table, prefix_table = layout(cache, batch, 100, prefix, 4)
    lens = torch.full((batch,), 90, dtype=torch.int32, device="cuda")
    lens[1] = 33
    seen = torch.zeros(cache.pages, 16, dtype=torch.bool, device="cuda")
    for b in range(batch):
        held = int(lens[b])
        for at in range(max(0, prefix + held - 1 - window), prefix + held):
            page = table[b, (at - prefix) // 16] if at >= prefix else prefix_table[at // 16]
            seen[int(page), at % 16 if at < prefix else (at - prefix) % 16] = True
    if zeros:
        cache.v_scale.zero_()
    q = torch.randn(batch, 2, 8, kind[2], generator=generator(4), device="cuda").to(TYPES[t])
    op = ops.KVAttention(cache, 8, window=window)
    want = op.exec(q, table, lens, max_len=100, prefix_table=prefix_table, prefix_len=prefix)
    assert torch.isfinite(want).all() and bool((want == 0).all()) == zeros
    cache.v_scale.copy_(torch.where(seen[:, None, :, None], cache.v_scale, large))
    got = op.exec(q, table, lens, max_len=100, prefix_table=prefix_table, prefix_len=prefix)
    assert torch.equal(got, want)


@pytest.mark.parametrize("t", ["f32", "bf16"])
@pytest.mark.parametrize("q_len,prefix", [(4, 0), (4, 40), (12, 40)])
@pytest.mark.parametrize("window", [2 ** 31 - 1, 2 ** 31 - 3, 1 << 30])
def test_attention_window_past_every_position(q_len, prefix, window, t):
    """A window that hides nothing, on sequences with fewer tokens than queries too."""
    kind = (8, 0, 64, 2, 16)
    cache = filled(kind, 6 * 2 + 5, 1)
    table, prefix_table = layout(cache, 6, 30, prefix, 2)
    lens = torch.tensor([0, 1, 2, 3, 13, 30], dtype=torch.int32, device="cuda")
    q = torch.randn(6, q_len, 8, 64, generator=generator(3), device="cuda").to(TYPES[t])
    kw = dict(max_len=30, prefix_table=prefix_table, prefix_len=prefix)
    want = ops.KVAttention(cache, 8).exec(q, table, lens, **kw)
    ref, slack = attention_ref(cache, q, table, lens, prefix_table, prefix, 0, 64 ** -0.5, t)
    near(want, ref, slack, t)
    assert torch.equal(ops.KVAttention(cache, 8, window=window).exec(q, table, lens, **kw), want)


def test_matmul_nbits_refuses_another_device():
    """Weights on another device than the current one are not read. (There is
    one device here: the operator is told that its weights are elsewhere.)"""
    op = ops.MatMulNBits(torch.zeros(8, 2, 16, dtype=torch.uint8), torch.ones(8, 2, dtype=torch.bfloat16), 64)
    a = torch.zeros(2, 64, device="cuda", dtype=torch.bfloat16)
    assert op.exec(a).shape == (2, 8)
    op._device += 1
    with pytest.raises(ValueError, match="weights are on cuda:1"):
        op.exec(a)


def test_attention_takes_a_scale_and_a_window_set_anew():
    cache = filled((8, 0, 64, 1, 16), 9, 1)
    table, _ = layout(cache, 2, 60, 0, 1)
    lens = torch.tensor([60, 41], dtype=torch.int32, device="cuda")
    q = torch.randn(2, 1, 2, 64, generator=generator(2), device="cuda").bfloat16()
    op = ops.KVAttention(cache, 2)
    seen = [op.exec(q, table, lens)]
    for kw in (dict(scale=1.0), dict(scale=-0.5, window=7), dict(window=3), dict()):
        op.scale, op.window = kw.get("scale", 64 ** -0.5), kw.get("window", 0)
        y = op.exec(q, table, lens)
        assert torch.equal(y, ops.KVAttention(cache, 2, **kw).exec(q, table, lens))
        seen.append(y)
    assert torch.equal(seen[0], seen[4])
    assert all(not torch.equal(seen[i], seen[j]) for i in range(4) for j in range(i))


def test_numbers_past_32_bits_are_refused():
    """Not answered as what is left of them in 32 bits."""
    cache = filled((8, 0, 64, 2, 16), 9, 1)
    table, prefix_table = layout(cache, 2, 60, 16, 1)
    lens = torch.tensor([60, 41], dtype=torch.int32, device="cuda")
    q = torch.randn(2, 1, 4, 64, generator=generator(2), device="cuda").bfloat16()
    op = ops.KVAttention(cache, 4)
    kw = dict(max_len=60, prefix_table=prefix_table, prefix_len=16)
    for bad in (dict(max_len=2 ** 32 + 60), dict(prefix_len=2 ** 32 + 16), dict(prefix_len=-2 ** 32)):
        with pytest.raises(ValueError, match="32 bits"):
            op.exec(q, table, lens, **{**kw, **bad})
    op.window = 2 ** 32 + 5
    with pytest.raises(ValueError, match="32 bits"):
        op.exec(q, table, lens, **kw)
    for bad in (dict(pages=2 ** 32 + 9), dict(heads=2 ** 32 + 2), dict(group=2 ** 32)):
        with pytest.raises(ValueError, match="32 bits"):
            ops.KVCache(**{**dict(pages=9, page_size=16, heads=2, head_dim=64), **bad},
                        buffers={n: getattr(cache, n) for n in ("k", "k_scale", "v", "v_scale")})
    linear = ops.MatMulNBits(torch.zeros(1, 1, 16, dtype=torch.uint8), torch.ones(1, 1, dtype=torch.half), 1)
    a = torch.empty(2 ** 32 + 5, 1, dtype=torch.half, device="cuda")
    with pytest.raises(ValueError, match="32 bits"):
        linear.exec(a)


def test_matmul_nbits_of_the_most_rows():
    """2^31 - 1 rows, which pass 2^31 when they are rounded up to a block's."""
    op = ops.MatMulNBits(torch.full((1, 1, 16), 0x99, dtype=torch.uint8), torch.ones(1, 1, dtype=torch.half), 1)
    a = torch.empty(2 ** 31 - 1, 1, dtype=torch.half, device="cuda").uniform_(-1, 1, generator=generator(1))
    y = torch.full_like(a, float("nan"))
    op.exec(a, y=y)
    assert torch.equal(y, a)  # a weight of 9 - 8 times 1
    del a, y
    torch.cuda.empty_cache()


def near_by_weight(got, cache, q, table, lens, prefix_table, prefix, scale, t):
    """As test_gpu_decode.near for one query a sequence, but what a weight p_j r_j
    loses (its fp16 steps of 2^-24, half of one, in units in which the row's
    largest weight is at least 2^6: 2^-31 of that) is counted against the largest
    weight and not against the largest value. (Twice, since the largest code of
    that key may be less than the type's.)"""
    batch, _, q_heads, dim = q.shape
    k, v = (values(cache, p) for p in "kv")
    for b in range(batch):
        rows = [torch.cat((x[prefix_table.long()].flatten(0, 1)[:prefix], x[table[b].long()].flatten(0, 1)[:int(lens[b])]))
                for x in (k, v)]
        kk, vv = (r.repeat_interleave(q_heads // cache.heads, 1).transpose(0, 1) for r in rows)
        qq = q[b, 0].double()[:, :, None] * scale
        x = (kk @ qq)[..., 0]
        p = torch.softmax(x, -1)
        want = (p[:, None] @ vv)[:, 0]
        n, terms = p.shape[1], (kk.abs() @ qq.abs())[..., 0].amax(-1, keepdim=True)
        loose = HALF[t] + 2 * (dim / 16 + 16) * 2.0 ** -23 * terms + 2.0 ** -20 + (n / 16 + 64) * 2.0 ** -23
        slack = loose * (p[:, None] @ vv.abs())[:, 0]
        slack += n * 2.0 ** -31 * (p * vv.abs().amax(-1)).amax(-1, keepdim=True) * 2
        near(got[b, 0], want, slack, t)


@pytest.mark.parametrize("t", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("kind,batch,longest,prefix", [
    ((8, 0, 64, 1, 16), 2, 120, 0), ((8, 0, 64, 1, 16), 40, 40, 200), ((4, 32, 128, 1, 16), 2, 300, 0),
    ((8, 0, 256, 1, 16), 2, 300, 0), ((8, 0, 128, 1, 16), 1, 9000, 0), ((8, 0, 128, 4, 16), 40, 20, 12000),
    ((4, 0, 64, 4, 16), 40, 20, 12000)])
@pytest.mark.parametrize("power", [0, 16, 24, 40])
def test_attention_large_values_that_weigh_next_to_nothing(kind, batch, longest, prefix, power, t):
    """Keys whose values are 2^power times the others', and which no query gives
    a weight of 2^-60: the others keep their precision."""
    bits, group, dim, heads, page = kind
    per, shared = -(-longest // page), -(-prefix // page)
    cache = filled(kind, batch * per + shared, 3)
    pages = torch.arange(cache.pages, dtype=torch.int32, device="cuda")
    prefix_table, table = pages[:shared].contiguous(), pages[shared:].view(batch, per)
    q = torch.randn(batch, 1, heads * 4, dim, generator=generator(9), device="cuda").to(TYPES[t])
    q[..., 0] = 16
    for page_of in ([table[b, i] for b in range(batch) for i in (0, per // 2)] if longest >= 40 else
                    [prefix_table[i] for i in (0, 2, shared // 2, shared - 2)]):
        at = (int(page_of), slice(None), 7)
        # a code of -127 (-7) in channel 0, where every query is 16, and zeros elsewhere
        cache.k[at] = 0 if bits == 8 else 0x88
        cache.k[at[0], :, 7, 0] = -127 if bits == 8 else 0x81
        cache.k_scale[at] = 60 * dim ** 0.5 / (16 * (127 if bits == 8 else 7))  # a logit of -60
        cache.v_scale[at] *= 2.0 ** power
    lens = torch.full((batch,), longest, dtype=torch.int32, device="cuda")
    got = ops.KVAttention(cache, heads * 4).exec(q, table, lens, prefix_table=prefix_table, prefix_len=prefix)
    near_by_weight(got, cache, q, table, lens, prefix_table, prefix, dim ** -0.5, t)


@pytest.mark.parametrize("t", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("kind,batch,longest,prefix", [
    ((8, 0, 64, 1, 16), 2, 120, 0), ((8, 0, 128, 1, 16), 1, 9000, 0), ((4, 32, 128, 4, 16), 8, 6000, 0),
    ((8, 0, 128, 4, 16), 40, 20, 12000), ((8, 0, 64, 4, 16), 20, 20, 16000)])
@pytest.mark.parametrize("back", [False, True])
@pytest.mark.parametrize("period", [32, 200, 1 << 20])
def test_attention_values_that_fall_as_logits_rise(kind, batch, longest, prefix, period, back, t):
    """Over each `period` keys (or all) logits rise by 60, which is a factor of
    2^86 in p, and values fall by 2^40, or the other way round."""
    bits, group, dim, heads, page = kind
    per, shared = -(-longest // page), -(-prefix // page)
    cache = filled(kind, batch * per + shared, 3)
    pages = torch.arange(cache.pages, dtype=torch.int32, device="cuda")
    prefix_table, table = pages[:shared].contiguous(), pages[shared:].view(batch, per)
    q = torch.randn(batch, 1, heads * 4, dim, generator=generator(9), device="cuda").to(TYPES[t])
    q[..., 0] = 16
    top = 127 if bits == 8 else 7
    cache.k.fill_(0 if bits == 8 else 0x88)
    cache.k[..., 0] = top if bits == 8 else 0x8F
    n = (shared if prefix else per) * page
    at = (torch.arange(n, device="cuda") % period / min(n, period)).view(-1, 1, page, 1)
    rise = 1 - at if back else at
    for row in [prefix_table] if prefix else list(table):
        cache.k_scale[row.long()] = (60 * dim ** 0.5 / (16 * top) * rise).expand(-1, heads, -1, cache.k_scale.shape[-1])
        cache.v_scale[row.long()] *= 2.0 ** (-40 * rise)
    if prefix:  # what follows the prefix has logits of 0 and weighs nothing
        cache.k_scale[shared:] = 0
        cache.v_scale[shared:] *= 2.0 ** -40
    lens = torch.full((batch,), longest, dtype=torch.int32, device="cuda")
    got = ops.KVAttention(cache, heads * 4).exec(q, table, lens, prefix_table=prefix_table, prefix_len=prefix)
    near_by_weight(got, cache, q, table, lens, prefix_table, prefix, dim ** -0.5, t)


@pytest.mark.parametrize("t", ["f32", "bf16"])
@pytest.mark.parametrize("kind,batch,longest,prefix", [
    ((8, 0, 64, 1, 16), 2, 120, 0), ((4, 32, 128, 1, 16), 2, 900, 0), ((8, 0, 256, 1, 16), 2, 900, 0),
    ((8, 0, 128, 8, 16), 1, 9000, 0), ((8, 0, 128, 4, 16), 40, 20, 6000), ((8, 0, 64, 4, 16), 3, 20, 6000)])
def test_attention_of_values_near_the_largest(kind, batch, longest, prefix, t):
    """A mean of values is no larger than they are, however large their sum."""
    bits, group, dim, heads, page = kind
    per, shared = -(-longest // page), -(-prefix // page)
    cache = filled(kind, batch * per + shared, 3)
    pages = torch.arange(cache.pages, dtype=torch.int32, device="cuda")
    prefix_table, table = pages[:shared].contiguous(), pages[shared:].view(batch, per)
    cache.v_scale.fill_(2.6e36 if bits == 8 else 4.7e37)  # values up to 3.3e38
    cache.v.clamp_(min=1) if bits == 8 else cache.v.bitwise_or_(0x99)
    cache.k_scale *= 0.1  # many keys of about the same weight
    lens = torch.full((batch,), longest, dtype=torch.int32, device="cuda")
    q = torch.randn(batch, 1, heads * 4, dim, generator=generator(9), device="cuda").to(TYPES[t])
    got = ops.KVAttention(cache, heads * 4).exec(q, table, lens, prefix_table=prefix_table, prefix_len=prefix)
    near_by_weight(got, cache, q, table, lens, prefix_table, prefix, dim ** -0.5, t)


@pytest.mark.parametrize("t", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("kind,batch,prefix", [((8, 0, 64, 1, 16), 2, 0), ((8, 0, 64, 1, 16), 40, 500),
                                               ((4, 32, 128, 1, 16), 2, 0), ((8, 0, 256, 1, 16), 2, 0)])
@pytest.mark.parametrize("size", [1e3, 1e4, 3e4])
@pytest.mark.parametrize("scale", [None, -0.3, 1.7, 0.0])
def test_attention_logits_far_past_fp32_steps_of_one(kind, batch, prefix, size, scale, t):
    """Queries and keys of 1e4 have logits of 1e8, where fp32 has steps of 8 and
    more: the largest alone is left, and its value comes out."""
    cache = filled(kind, batch * 8 + 34, 3)
    cache.k_scale.mul_(size)
    table, prefix_table = layout(cache, batch, 120, prefix, 3)
    lens = torch.full((batch,), 120, dtype=torch.int32, device="cuda")
    q = torch.randn(batch, 1, 4, kind[2], generator=generator(9), device="cuda").clamp(-2, 2)
    q = (q * size).to(TYPES[t])
    got = ops.KVAttention(cache, 4, scale=scale).exec(q, table, lens, prefix_table=prefix_table, prefix_len=prefix)
    scale = kind[2] ** -0.5 if scale is None else scale
    want, slack = attention_ref(cache, q, table, lens, prefix_table, prefix, 0, scale, t)
    near(got, want, slack, t)


@pytest.mark.parametrize("t", ["f32", "bf16"])
@pytest.mark.parametrize("kind,batch,q_len,prefix,window", [((8, 0, 128, 2, 16), 2, 2, 0, 60), ((8, 0, 64, 2, 5), 3, 1, 0, 40),
                                                           ((4, 32, 128, 2, 16), 2, 3, 0, 1), ((8, 0, 128, 2, 16), 40, 1, 203, 150),
                                                           ((8, 0, 64, 1, 16), 2, 48, 0, 7)])
def test_attention_pages_that_no_window_reaches_may_be_gone(kind, batch, q_len, prefix, window, t):
    """A table may hold -1 for a page that every window has left behind, and
    beyond a sequence's end; that is no error."""
    page = kind[4]
    per, shared = -(-100 // page), -(-prefix // page)
    cache = filled(kind, batch * per + shared + 3, 5)
    table, prefix_table = layout(cache, batch, 100, prefix, 4)
    table = table.contiguous()
    lens = torch.randint(70, 101, (batch,), generator=generator(6), device="cuda", dtype=torch.int32)
    q = torch.randn(batch, q_len, 8, kind[2], generator=generator(4), device="cuda").to(TYPES[t])
    op = ops.KVAttention(cache, 8, window=window)
    kw = dict(max_len=100, prefix_len=prefix)
    want = op.exec(q, table, lens, prefix_table=prefix_table, **kw)
    first = prefix + lens - q_len - window + 1  # the first position that a sequence's first query sees
    for b in range(batch):
        table[b, :max(0, int(first[b]) - prefix) // page] = -1
        table[b, -(-int(lens[b]) // page):] = -1
    prefix_table[:min(prefix, max(0, int(first.min()))) // page] = -1
    assert (table == -1).any()
    assert torch.equal(op.exec(q, table, lens, prefix_table=prefix_table, **kw), want)
    torch.cuda.synchronize()
    assert ops.device_status() == 0


@pytest.mark.parametrize("kind,batch,prefix", [((8, 0, 128, 2, 16), 3, 0), ((4, 0, 64, 2, 16), 40, 300)])
def test_a_step_in_a_cuda_graph_and_on_two_streams(kind, batch, prefix):
    """A projection, the cache's write and attention, captured and replayed with
    other inputs and lengths; and two such steps at once."""
    bits, group, dim, heads, page = kind
    hidden, q_heads = 96, heads * 4
    cache = filled(kind, batch * 4 + 30, 3)
    table, prefix_table = layout(cache, batch, 60, prefix, 1)
    b, s, z, c = weights((q_heads + 2 * heads) * dim, hidden, 32, "bf16", True, True, 1)
    linear, attention = ops.MatMulNBits(b, s * 0.1, hidden, zero_points=z, bias=c), ops.KVAttention(cache, q_heads)
    x = torch.randn(batch, hidden, generator=generator(2), device="cuda").bfloat16()
    lens = torch.full((batch,), 7, dtype=torch.int32, device="cuda")

    def slots():
        at = lens.long() - 1
        return table.gather(1, (at // page)[:, None])[:, 0].long() * page + at % page

    def step(x, stream=None):
        qkv = linear.exec(x, stream=stream).view(batch, -1, dim)
        cache.write(qkv[:, q_heads:q_heads + heads], qkv[:, q_heads + heads:], to, stream=stream)
        return attention.exec(qkv[:, None, :q_heads], table, lens, max_len=60, prefix_table=prefix_table,
                              prefix_len=prefix, stream=stream)

    to = slots()
    step(x)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y = step(x)
    for held in (7, 20, 60):
        lens.fill_(held)
        to.copy_(slots())
        x.normal_(generator=generator(held))
        graph.replay()
        assert torch.equal(y, step(x))
    want, other = step(x), torch.randn(batch, hidden, generator=generator(3), device="cuda").bfloat16()
    q = [linear.exec(a).view(batch, -1, dim)[:, None, :q_heads] for a in (x, other)]
    kw = dict(max_len=60, prefix_table=prefix_table, prefix_len=prefix)
    wants = [attention.exec(a, table, lens, **kw) for a in q]
    streams = [torch.cuda.Stream() for _ in q]
    torch.cuda.synchronize()
    for _ in range(20):
        got = [attention.exec(a, table, lens, stream=st, **kw) for a, st in zip(q, streams)]
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, wants))
    assert torch.equal(wants[0], want)


@pytest.mark.parametrize("kind,batch,longest,prefix", [
    ((8, 0, 128, 2, 16), 3, 1, 0), ((8, 0, 64, 1, 16), 5, 3, 0), ((4, 32, 128, 2, 16), 3, 300, 0), ((8, 32, 64, 2, 16), 2, 40, 0),
    ((4, 0, 256, 1, 16), 2, 100, 0), ((8, 0, 128, 2, 16), 40, 2, 500), ((8, 0, 64, 2, 16), 40, 2, 130),
    ((4, 0, 128, 4, 16), 40, 20, 9000), ((4, 0, 64, 4, 16), 70, 20, 9000)])
def test_attention_in_fp16_is_off_by_its_rounding_only(kind, batch, longest, prefix):
    """As test_gpu_decode's bound, but with weights of 22 bits, not of fp16's 11."""
    bits, group, dim, heads, page = kind
    per, shared = -(-longest // page), -(-prefix // page)
    cache = filled(kind, batch * per + shared, 11)
    table, prefix_table = layout(cache, batch, longest, prefix, 4)
    lens = torch.full((batch,), longest, dtype=torch.int32, device="cuda")
    q = torch.randn(batch, 1, heads * 4, dim, generator=generator(4), device="cuda").half()
    got = ops.KVAttention(cache, heads * 4).exec(q, table, lens, prefix_table=prefix_table, prefix_len=prefix)
    want, slack = attention_ref(cache, q, table, lens, prefix_table, prefix, 0, dim ** -0.5, "f32")
    near(got, want, slack, "f16")  # fp32's slack has 2^-20 for exp and the weights
    if longest == 1 and not prefix:
        v = values(cache, "v")[table[:, 0].long(), 0].half()
        assert torch.equal(got[:, 0], v.repeat_interleave(4, 1))


@pytest.mark.parametrize("kind,batch,longest", [((8, 0, 128, 8, 64), 8, 8192), ((8, 0, 128, 5, 48), 1, 30000),
                                                ((8, 0, 256, 2, 48), 3, 200), ((4, 0, 64, 8, 16), 8, 9000),
                                                ((4, 32, 128, 4, 16), 8, 6000)])
@pytest.mark.parametrize("seed", [1, 2, 3])
def test_attention_in_fp32_is_off_by_few_roundings(kind, batch, longest, seed):
    """In the norm of the output. A logit of up to 16 has steps of 2^-20 (half of
    one is 2^-21 of its p), exp2 is off by 2^-22 and so are operands of 22 bits:
    together less than 2^-20, if the sums of both products add nothing."""
    bits, group, dim, heads, page = kind
    per = -(-longest // page)
    cache = filled(kind, batch * per, seed)
    table, _ = layout(cache, batch, longest, 0, seed)
    lens = torch.full((batch,), longest, dtype=torch.int32, device="cuda")
    q = torch.randn(batch, 1, heads, dim, generator=generator(seed), device="cuda") * 1.25
    got = ops.KVAttention(cache, heads).exec(q, table, lens).double()
    want, _ = attention_ref(cache, q, table, lens, None, 0, 0, dim ** -0.5, "f32")
    assert (got - want).norm() <= want.norm() * 2.0 ** -20
