"""The 4-bit KV cache's attention where lengths, tables and q do not fit each other, and where
values span many orders of magnitude, against tests/kv4_ref.py.  Bounds as in test_gpu_kv4.py."""
import numpy as np
import pytest
import torch

from csed499ii_amd import marlin
from tests import kv4_ref as ref
from tests.test_gpu_kv4 import DEV, _check, _problem, ints

pytestmark = pytest.mark.gpu

# query and kv heads: rows for the kernel of few rows, and for that of prompts
KERNELS = [(4, 2), (34, 17)]


def _wider(table, pages):
    """The table with ``pages`` entries a row, those added no page: for the reference, which
    knows no width."""
    return np.pad(table, ((0, 0), (0, pages - table.shape[1])), constant_values=-1)


@pytest.mark.parametrize("Hq,Hkv", KERNELS)
@pytest.mark.parametrize("D,g", [(128, -1), (64, 32)])
def test_new_tokens_past_the_table_keep_their_positions(Hq, Hkv, D, g):
    """A table of 64 tokens for requests of 80, 64, 200 and 20: the tokens that it covers see
    what lies up to them, those past it all that it covers."""
    T, new, kv = 16, [50, 3, 60, 20], [80, 64, 200, 20]
    q, cache, table, cut, cu, G = _problem(new, [min(n, 64) for n in kv], Hq, Hkv, D, g, T, torch.float16, seed=201)
    want = ref.attention(q.double().numpy(), cache, _wider(table, 13), kv, cu, D, G, T)
    out, lse = marlin.kv4_attention(q.to(DEV), torch.from_numpy(cache).to(DEV), ints(table), ints(kv), ints(cu),
                                    max_q=60, max_kv=200, groupsize=g, return_lse=True)
    _check(out, lse, want, torch.float16, "cut by the table")


@pytest.mark.parametrize("Hq,Hkv", KERNELS)
def test_fewer_rows_of_q_than_new_tokens(Hq, Hkv):
    """cu_q counts 90 new tokens, q has the first 65: each at its own position."""
    T, D, new, kv = 16, 128, [20, 70], [33, 90]
    q, cache, table, kvs, cu, G = _problem(new, kv, Hq, Hkv, D, -1, T, torch.float16, seed=202)
    want = [x[:65] for x in ref.attention(q.double().numpy(), cache, table, kv, cu, D, G, T)]
    out, lse = marlin.kv4_attention(q[:65].to(DEV), torch.from_numpy(cache).to(DEV), ints(table), ints(kv), ints(cu),
                                    max_q=70, max_kv=90, return_lse=True)
    _check(out, lse, want, torch.float16, "cut by q")
