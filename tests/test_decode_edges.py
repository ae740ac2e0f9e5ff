"""Calls of the decode operators at the edges of what they take, which need no GPU."""
import subprocess
import sys
from pathlib import Path

import pytest
import torch

from nnr_b200 import ops

ROOT = Path(__file__).resolve().parent.parent

EMPTY = """
import ctypes as C
from nnr_b200 import _lib
cache = _lib.KvCacheDesc(pages=4, page_size=16, heads=2, head_dim={dim}, bits=8, group=0)
desc = _lib.KvAttentionDesc(batch=0, q_len=1, q_heads=4, dtype=1, q_batch_stride=256, q_token_stride=256,
                            q_head_stride=64, table_pages=2, table_stride=2, max_len=32, prefix_len={prefix},
                            prefix_pages=4, window=0, scale=0.125)
n = C.c_size_t(77)
assert _lib.lib.nnrcu_kv_attention_workspace(C.byref(cache), C.byref(desc), C.byref(n)) == 0
assert n.value == 0
assert _lib.lib.nnrcu_kv_attention_workspace(C.byref(cache), C.byref(desc), None) == -1
"""


@pytest.mark.parametrize("dim", [64, 256])
@pytest.mark.parametrize("prefix", [0, 50])
def test_an_empty_batch_needs_no_workspace(dim, prefix):
    # in a process of its own: a division by zero would end it
    r = subprocess.run([sys.executable, "-c", EMPTY.format(dim=dim, prefix=prefix)], cwd=ROOT, capture_output=True,
                       text=True)
    assert r.returncode == 0, (r.returncode, r.stderr)


@pytest.mark.parametrize("kind,names", [
    (ops.MatMulNBits, ("n", "k", "block_size", "dtype")),
    (ops.KVCache, ("pages", "page_size", "heads", "head_dim", "bits", "group", "desc", "k", "k_scale", "v", "v_scale")),
    (ops.KVAttention, ("cache", "q_heads"))])
def test_what_calls_rely_on_is_set_once(kind, names):
    """Descriptions hold sizes and addresses: a cache whose k is replaced would
    write to the old one's freed memory."""
    x = kind.__new__(kind)
    for name in names:
        setattr(x, name, 1)
        with pytest.raises(AttributeError, match=name):
            setattr(x, name, 2)
        assert getattr(x, name) == 1


def test_a_buffer_may_be_changed_in_place():
    cache = ops.KVCache.__new__(ops.KVCache)
    cache.k_scale = buffer = torch.ones(3)
    cache.k_scale *= 2
    assert cache.k_scale is buffer and (buffer == 2).all()
    with pytest.raises(AttributeError):
        cache.k_scale = cache.k_scale * 2
