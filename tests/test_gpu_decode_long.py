"""The decode operators where a block has much to do: several items with more
spans of k than the ring has stages, several units of many tiles that are cut
at uneven places (tolerances: tests/test_gpu_decode.py)."""
import pytest
import torch

from nnr_b200 import ops
from test_gpu_decode import TYPES, attention_ref, filled, generator, layout, near, product, weights

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module", autouse=True)
def device(cuda_dev):
    yield cuda_dev
    torch.cuda.synchronize()
    assert ops.device_status() == 0
    torch.cuda.empty_cache()


def sms():
    return torch.cuda.get_device_properties(0).multi_processor_count


# m, n, k: by tiles of 16 outputs a warp takes one or two at once, and 8 or 16
# warps share k. On 148 SMs each of these gives blocks two items or more, and
# not all the same number, but (5, 4100, 2077), which has one and a long row.
LONG = [(1, 14600, 1500), (16, 9617, 2077), (33, 4817, 2900), (60, 4100, 6000), (5, 4100, 2077), (9, 2000, 12000),
        (70, 1900, 9000)]


@pytest.mark.parametrize("t", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("m,n,k", LONG)
@pytest.mark.parametrize("block", [32, 128])
@pytest.mark.parametrize("zero", [False, True])
def test_matmul_nbits_long(m, n, k, block, zero, t):
    b, s, z, c = weights(n, k, block, t, zero, zero, m + n)
    a = torch.randn(m, k, generator=generator(1), device="cuda").to(TYPES[t])
    op = ops.MatMulNBits(b, s, k, zero_points=z, bias=c)
    y = op.exec(a)
    want, terms = product(a, b, s, z, c, k, block)
    near(y, want, terms * (k / 16 + 64) * 2.0 ** -24, t)
    assert torch.equal(y, op.exec(a))


ATTEND = [  # kind of cache, batch, q_len, query heads a cache head, longest, prefix, window
    ((8, 0, 128, 8, 64), 32, 1, 4, 6000, 0, 0),      # blocks of 8 rows,
    ((8, 0, 64, 8, 48), 24, 3, 5, 6000, 0, 0),       # of 16
    ((8, 0, 128, 8, 16), 20, 3, 7, 5000, 0, 0),      # and of 24
    ((4, 32, 128, 8, 48), 20, 3, 7, 5000, 0, 3001),
    ((4, 0, 96, 8, 16), 24, 2, 4, 5000, 0, 0),
    ((8, 32, 64, 8, 64), 24, 2, 6, 5000, 0, 0),
    ((8, 0, 256, 8, 64), 16, 2, 5, 5000, 0, 0),
    ((4, 32, 256, 8, 33), 16, 1, 3, 5000, 0, 0),
    ((8, 0, 128, 8, 64), 40, 1, 4, 300, 9000, 0),    # of 128, for 16-bit tensors
    ((4, 0, 128, 8, 64), 40, 1, 4, 300, 9001, 0),
    ((8, 0, 64, 8, 48), 40, 1, 4, 300, 9000, 0),
    ((4, 0, 64, 8, 16), 30, 2, 3, 300, 12345, 0),
    ((8, 0, 128, 8, 64), 40, 2, 4, 300, 9000, 4000),
    ((8, 0, 128, 8, 64), 12, 30, 2, 3000, 0, 0),
]


def quads(held, heads, blocks):
    """Stretches of 128 keys of all units."""
    return sum(max(1, -(-n // 128)) for n in held) * heads * blocks


@pytest.mark.parametrize("t", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("kind,batch,q_len,share,longest,prefix,window", ATTEND)
def test_attention_long(kind, batch, q_len, share, longest, prefix, window, t):
    bits, group, dim, heads, page = kind
    per, shared = -(-longest // page), -(-prefix // page)
    cache = filled(kind, batch * per + shared + 2, longest + dim)
    table, prefix_table = layout(cache, batch, longest, prefix, 2)
    g = generator(longest)
    lens = torch.randint(longest // 3, longest + 1, (batch,), generator=g, device="cuda", dtype=torch.int32)
    lens[0], lens[1], lens[2] = longest, 0, 1
    # a block has more than one stretch of keys: more of them than blocks run at once
    rows = q_len * share
    many = t != "f32" and not group and dim in (64, 128)
    n, held = (rows * batch, [prefix]) if prefix else (rows, [min(int(x), window or longest) for x in lens])
    of, at_once = (128, sms()) if many and n >= 40 else (8 if dim > 128 else 24, 4 * sms())
    assert quads(held, heads, -(-n // of)) > 1.5 * at_once
    q = torch.randn(batch, q_len, heads * share, dim, generator=g, device="cuda").to(TYPES[t])
    op = ops.KVAttention(cache, heads * share, window=window)
    kw = dict(max_len=longest, prefix_table=prefix_table, prefix_len=prefix)
    got = op.exec(q, table, lens, **kw)
    want, slack = attention_ref(cache, q, table, lens, prefix_table, prefix, window, dim ** -0.5, t)
    near(got, want, slack, t)
    for _ in range(3):
        assert torch.equal(got, op.exec(q, table, lens, **kw))


@pytest.mark.parametrize("t", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("kind,batch,longest,prefix", [((8, 0, 64, 8, 16), 24, 5000, 0), ((4, 32, 128, 8, 16), 24, 5000, 0),
                                                       ((8, 0, 64, 8, 16), 40, 30, 12000),
                                                       ((8, 0, 128, 8, 16), 40, 30, 9000)])
@pytest.mark.parametrize("back", [False, True])
def test_attention_long_with_growing_logits_and_values(kind, batch, longest, prefix, back, t):
    """The largest logit and the largest value scale rise (or fall) by 2^20 and
    more on the way along the keys, so that sums are rescaled again and again."""
    bits, group, dim, heads, page = kind
    per, shared = -(-longest // page), -(-prefix // page)
    cache = filled(kind, batch * per + shared, 7)
    pages = torch.arange(cache.pages, dtype=torch.int32, device="cuda")
    prefix_table, table = pages[:shared].contiguous(), pages[shared:].view(batch, per)
    at = torch.arange(max(longest, prefix) + page, device="cuda") / max(longest, prefix)
    if back:
        at = 1 - at
    for n, rows in [(shared, prefix_table[None])] if prefix else [(per, table)]:
        rise = at[:n * page].view(n, 1, page, 1)
        for row in rows:
            cache.k_scale[row.long()] *= 0.05 + 3 * rise
            cache.v_scale[row.long()] *= 2.0 ** (20 * rise - 20)
    lens = torch.randint(longest // 2, longest + 1, (batch,), generator=generator(1), device="cuda", dtype=torch.int32)
    q = torch.randn(batch, 1, heads * 4, dim, generator=generator(2), device="cuda").to(TYPES[t])
    op = ops.KVAttention(cache, heads * 4)
    got = op.exec(q, table, lens, prefix_table=prefix_table, prefix_len=prefix)
    want, slack = attention_ref(cache, q, table, lens, prefix_table, prefix, 0, dim ** -0.5, t)
    near(got, want, slack, t)
