"""Attention over an 8-bit cache (attention8.hip): what a call takes of scratch and launches, where its bounds are far above its lengths."""
import numpy as np
import pytest
import torch

from plain_cache8 import attention
from test_cache8_gpu import TYPES, attend, close, filled, host, ints, items_of, tables
from vosti_amd.kernels import kernels_for

pytestmark = pytest.mark.gpu


WINDOWS = [
    # (type, rows, keys, nq, nkv, d, P, window): items of one tile of columns, of two by two waves, of more by four; of 32 bits
    ("bf16", [1, 1, 1, 1], [1, 512, 1025, 3000], 4, 2, 128, 64, 1),
    ("bf16", [2, 1], [513, 2049], 4, 2, 64, 16, 512),
    ("bf16", [3, 2, 3], [514, 1537, 2600], 8, 2, 128, 64, 512),
    ("bf16", [3, 3], [1026, 2050], 16, 2, 128, 32, 513),
    ("bf16", [5, 4], [1028, 2563], 8, 1, 64, 64, 511),
    ("bf16", [7, 7], [1536, 2055], 8, 1, 128, 16, 1000),
    ("bf16", [16], [1551], 4, 1, 256, 64, 1025),
    ("bf16", [9, 1], [700, 1600], 6, 1, 192, 64, 2),
    ("f32", [2, 2], [1025, 2000], 8, 2, 64, 16, 512),
    ("f32", [4, 4], [515, 2051], 8, 1, 128, 64, 510),
]


@pytest.mark.parametrize("case", range(len(WINDOWS)))
def test_a_windows_scratch_does_not_grow_with_the_bound(case):
    """A recorded step's bound of 131,072 keys: the sums of two segments more than a window has, nothing behind them written, and a row's bits those of a call with a bound of its length."""
    name, rows, keys, nq, nkv, d, P, window = WINDOWS[case]
    k, most, bound = kernels_for(name), max(rows), 131072
    rng = np.random.default_rng(40 + case)
    table, pages = tables(rng, keys, P)
    cache = filled(rng, pages, nkv, P, d)
    q = torch.from_numpy(rng.standard_normal((sum(rows), nq, d))).to(TYPES[name]).cuda()
    wide = np.full((len(keys), bound // P), -1)
    wide[:, :table.shape[1]] = table
    need = k.attn8_scratch_floats(len(keys), most, nq, d, bound, window=window)
    segments = (window + most - 1 + 510) // 512 + 1                # most that so many neighbouring keys touch
    assert need == (len(keys) * most * nq * (d + 2) * segments if segments > 1 else 0)
    scratch = torch.full((need + 4096,), 77.0, device="cuda")
    want = attend(k, q, cache, table, rows, keys, most, window)
    assert torch.equal(attend(k, q, cache, wide, rows, keys, most, window, max_k_len=bound, scratch=scratch), want)
    assert scratch[need:].eq(77.0).all()
    close(want, attention(host(q), *map(host, cache), table, np.concatenate([[0], np.cumsum(rows)]), keys, d ** -0.5, window), name, d)
    # Lengths that say more than the bound: the keys below it that the window leaves.
    attend(k, q, cache, wide, rows, [2 ** 31 - 1 - i for i in range(len(keys))], most, window, max_k_len=bound, scratch=scratch)
    attend(k, q, cache, wide, rows, [bound + window // 2] * len(keys), most, window, max_k_len=bound, scratch=scratch)
    assert scratch[need:].eq(77.0).all()
