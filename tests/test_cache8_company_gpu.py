"""Rows of attention over an 8-bit cache (attention8.hip) in calls of many sequences, where a workgroup takes several segments and walks more pages than it reads at once, and in calls of
their own."""
import numpy as np
import pytest
import torch

from plain_cache8 import attention
from test_cache8_gpu import E4M3, TYPES, attend, close, host, tables
from vosti_amd.kernels import kernels_for

pytestmark = pytest.mark.gpu


COMPANY = [
    # (type, rows, keys, nq, nkv, d, P, window, rows of an item): sequences with lengths of their own; more than four segments a workgroup in the first ones
    ("bf16", [1] * 150, [1900 + i for i in range(150)], 8, 8, 128, 16, 0, 1),
    ("bf16", [2] * 150, [2050 - 7 * i for i in range(150)], 16, 8, 128, 16, 1300, 2),
    ("bf16", [1] * 150, [1700 + 3 * i for i in range(150)], 8, 8, 256, 16, 0, 1),
    ("bf16", [3] * 150, [2100 - i for i in range(150)], 8, 8, 192, 16, 1500, 3),
    ("f32", [2] * 150, [1800 + 2 * i for i in range(150)], 8, 8, 128, 16, 0, 2),
    ("f32", [1] * 150, [1800 - 5 * i for i in range(150)], 8, 8, 256, 16, 1100, 1),
    # Every way through LDS: two waves, four, whole rows; with and without a window; a page a tile, and four.
    ("bf16", [8, 3, 8], [700, 90, 1500], 8, 2, 64, 64, 0, 8),
    ("bf16", [7, 7, 2], [600, 1200, 40], 16, 4, 128, 16, 555, 7),
    ("bf16", [16, 5, 16], [530, 1100, 16], 8, 1, 256, 64, 0, 16),
    ("bf16", [20, 150, 64], [20, 700, 300], 8, 2, 128, 64, 0, 128),
    ("bf16", [33, 130], [333, 1200], 6, 2, 64, 16, 200, 64),
    ("f32", [6, 2], [900, 33], 8, 1, 64, 64, 0, 6),
    ("f32", [40, 22], [300, 40], 4, 2, 128, 32, 0, 40),
]


def filled(seed, pages, nkv, P, d):
    g = torch.Generator(device="cuda").manual_seed(seed)
    kc, vc = (torch.randn(pages, nkv, *shape, device="cuda", generator=g).mul_(90).clamp_(-448, 448).to(E4M3) for shape in ((P, d), (d, P)))
    return kc, vc, torch.exp2(torch.randint(-9, -4, (pages, nkv, 2), device="cuda", generator=g).float())


@pytest.mark.parametrize("case", range(len(COMPANY)))
def test_a_sequence_is_the_formula_and_the_same_bits_alone(case):
    name, rows, keys, nq, nkv, d, P, window, most = COMPANY[case]
    k, cu = kernels_for(name), np.concatenate([[0], np.cumsum(rows)])
    rng = np.random.default_rng(60 + case)
    table, pages = tables(rng, keys, P)
    cache = filled(60 + case, pages, nkv, P, d)
    q = torch.from_numpy(rng.standard_normal((sum(rows), nq, d))).to(TYPES[name]).cuda()
    got = attend(k, q, cache, table, rows, keys, most, window)
    assert torch.equal(got, attend(k, q, cache, table, rows, keys, most, window))
    for s in sorted({0, 1, len(rows) // 2, len(rows) - 1}):
        mine = slice(cu[s], cu[s + 1])
        alone = attend(k, q[mine].contiguous(), cache, table[s:s + 1], rows[s:s + 1], keys[s:s + 1], most, window)
        assert torch.equal(got[mine], alone)
        used = table[s, :-(-keys[s] // P)]
        close(alone, attention(host(q[mine]), *(host(t[used.tolist()]) for t in cache), np.arange(len(used))[None], [0, rows[s]], keys[s:s + 1], d ** -0.5, window), name, d)
