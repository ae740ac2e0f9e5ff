"""Calls of the decode operators at the edges of what they take, which need no GPU."""
import subprocess
import sys
from pathlib import Path

import pytest

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
