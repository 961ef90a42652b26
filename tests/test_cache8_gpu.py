"""Append to an 8-bit cache (store8.hip) and attention over it (attention8.hip) against their formulas in 64 bits."""
import numpy as np
import pytest
import torch

from plain_cache8 import attention, store
from vosti_amd.kernels import KernelError, kernels_for

pytestmark = pytest.mark.gpu
E4M3 = torch.float8_e4m3fn
TYPES = {"bf16": torch.bfloat16, "f32": torch.float32}


def host(t):
    return None if t is None else t.detach().to(torch.float64).cpu().numpy()


def ints(values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


def tables(rng, keys, P, spare=3, width=None):
    """Pages of every sequence in any order, and a table that holds page numbers of nothing behind them."""
    used = [-(-k // P) for k in keys]
    order = rng.permutation(sum(used) + spare)
    W = max(max(used, default=0), 1) if width is None else width
    table, at = np.full((len(keys), W), 10 ** 9), 0
    for s, n in enumerate(used):
        table[s, :n] = order[at:at + n]
        at += n
    return table, sum(used) + spare


def rotation(places, half, dtype):
    angle = torch.arange(places, dtype=torch.float64)[:, None] * 1e4 ** (-torch.arange(half, dtype=torch.float64) / half)
    return torch.cos(angle).to(dtype).cuda(), torch.sin(angle).to(dtype).cuda()


def filled(rng, pages, nkv, P, d, low=-9, high=-4):
    """A cache whose entries use their range, NaN in none."""
    def entries(*shape):
        return torch.from_numpy(np.clip(rng.standard_normal(shape) * 90, -448, 448)).to(torch.float32).to(E4M3).cuda()
    scales = torch.from_numpy(2.0 ** rng.integers(low, high, (pages, nkv, 2))).to(torch.float32).cuda()
    return entries(pages, nkv, P, d), entries(pages, nkv, d, P), scales


STORES = [
    # (type, rows, keys, nq, nkv, d, P, norm, rotated entries)
    ("bf16", [1], [1], 2, 1, 16, 16, True, 16),
    ("bf16", [1, 1, 1], [64, 65, 100], 8, 2, 128, 64, True, 128),
    ("bf16", [130], [130], 4, 2, 128, 64, True, 128),
    ("bf16", [5, 0, 200, 1, 17], [70, 9, 200, 128, 33], 6, 2, 64, 32, True, 64),
    ("bf16", [40, 3], [50, 259], 3, 3, 80, 16, False, 40),
    ("bf16", [300, 2], [301, 5], 2, 1, 256, 256, True, 256),
    ("bf16", [33], [40], 5, 1, 192, 128, True, 96),
    ("bf16", [7] * 70, [7 + 3 * i for i in range(70)], 2, 1, 32, 16, True, 20),
    ("f32", [1, 1], [16, 17], 4, 2, 64, 16, True, 64),
    ("f32", [90, 0, 31], [95, 0, 64], 4, 4, 96, 32, True, 48),
    ("f32", [21, 300], [21, 300], 2, 2, 256, 128, False, 0),
    ("f32", [5], [300], 2, 1, 16, 256, True, 8),
    # No more rows than sequences, and yet several of one.
    ("bf16", [21, 0, 1] + [0] * 25, [50, 7, 3] + [9] * 25, 2, 2, 64, 16, True, 64),
]


@pytest.mark.parametrize("case", range(len(STORES)))
def test_append_is_the_formula(case):
    """Entries and scales to the bit (they are computed in 64 bits and rounded once); q off by its rounding and a few 32-bit ones, of sums of d squares and two products:
    half a step of the type and 2^-24 (d / 64 + 12) of the two entries that a rotation mixes."""
    name, rows, keys, nq, nkv, d, P, norm, turned = STORES[case]
    dtype, k = TYPES[name], kernels_for(name)
    rng = np.random.default_rng(case)
    T = sum(rows) + 2                                          # two rows behind the last sequence
    qkv = torch.from_numpy(rng.standard_normal((T, (nq + 2 * nkv) * d)) * 2.0 ** rng.integers(-3, 4, (T, 1))).to(dtype).cuda()
    table, pages = tables(rng, keys, P)
    kc, vc, scales = filled(rng, pages, nkv, P, d)
    q_w = k_w = cos = sin = None
    if norm:
        q_w, k_w = (torch.from_numpy(rng.uniform(0.5, 1.5, d)).to(dtype).cuda() for _ in range(2))
    if turned:
        cos, sin = rotation(max(keys) + 3, turned // 2, dtype)
    cu = np.concatenate([[0], np.cumsum(rows)])
    want_k, want_v, want_s = host(kc), host(vc), host(scales)
    want = store(host(qkv), nq, nkv, d, want_k, want_v, want_s, host(q_w), host(k_w), 1e-5, host(cos), host(sin), table, cu, keys)
    out = torch.full((T, nq, d), 77.0, dtype=dtype, device="cuda")
    got = k.qkv_post8(qkv, nq=nq, nkv=nkv, d=d, k_cache=kc, v_cache=vc, scales=scales, q_w=q_w, k_w=k_w, eps=1e-5, cos=cos, sin=sin, block_table=ints(table),
                      cu_q=ints(cu), k_len=ints(keys), max_k_len=max(keys), q_out=out)
    assert got is out
    assert np.array_equal(host(scales), want_s)
    assert np.array_equal(host(kc), want_k)
    assert np.array_equal(host(vc), want_v)
    got = host(got)
    assert (got[sum(rows):] == 77.0).all()
    got, want = got[:sum(rows)], want[:sum(rows)]
    most = np.abs(want).max(-1, keepdims=True)
    assert (np.abs(got - want) <= torch.finfo(dtype).eps / 2 * np.abs(want) * (1 + 1e-3) + 2.0 ** -24 * (d / 64 + 12) * most).all()


def append(k, x, kc, vc, scales, table, keys, rows=None, d=64, nkv=1):
    rows = [1] * len(keys) if rows is None else rows
    k.qkv_post8(x, nq=0, nkv=nkv, d=d, k_cache=kc, v_cache=vc, scales=scales, q_w=None, k_w=None, eps=0.0, cos=None, sin=None, block_table=ints(table),
                cu_q=ints(np.concatenate([[0], np.cumsum(rows)])), k_len=ints(keys), max_k_len=max(keys))


@pytest.mark.parametrize("name", ["bf16", "f32"])
def test_a_page_appended_token_by_token_is_the_page_appended_at_once(name):
    """Entries of at least 2^-14 of the largest: whatever order their scale grew in."""
    k, d, P = kernels_for(name), 64, 32
    rng = np.random.default_rng(3)
    x = torch.from_numpy(rng.standard_normal((P, 2 * d)).clip(-3, 3) * 2.0 ** rng.integers(-4, 5, (P, 1))).to(TYPES[name])
    x = torch.where(x.abs() < 2.0 ** -6, torch.zeros_like(x), x).cuda()
    one, many = k.empty_cache8(2, 1, P, d), k.empty_cache8(2, 1, P, d)
    append(k, x, *one, [[1]], [P], [P])
    for i in range(P):
        append(k, x[i:i + 1], *many, [[1]], [i + 1])
    for a, b in zip(one, many):
        assert np.array_equal(host(a), host(b))


def test_what_is_not_finite_is_stored_as_nan_and_does_not_set_the_scale():
    k, d = kernels_for("bf16"), 64
    x = torch.ones(3, 2 * d, dtype=torch.bfloat16, device="cuda")
    x[0, 3], x[1, 5], x[2, d + 7] = float("inf"), float("nan"), -float("inf")
    kc, vc, scales = k.empty_cache8(1, 1, 16, d)
    append(k, x, kc, vc, scales, [[0]], [3], [3])
    assert scales.tolist() == [[[2.0 ** -8, 2.0 ** -8]]]
    kf, vf = kc[0, 0, :3].float(), vc[0, 0, :, :3].float().T
    assert torch.isnan(kf).nonzero().tolist() == [[0, 3], [1, 5]] and torch.isnan(vf).nonzero().tolist() == [[2, 7]]
    assert torch.nan_to_num(kf, nan=256.0).eq(256.0).all() and torch.nan_to_num(vf, nan=256.0).eq(256.0).all()


def test_zeros_extremes_and_pages_that_are_none():
    """A page of zeros has the smallest scale; the largest number of the type fits; -1 and a number beyond the cache keep nothing; a sequence that exceeds the
    bound is left out."""
    k, d = kernels_for("f32"), 16
    kc, vc, scales = k.empty_cache8(4, 1, 16, d)
    x = torch.zeros(5, 2 * d, device="cuda")
    x[1] = torch.finfo(torch.float32).max
    x[2:] = 1.0
    k.qkv_post8(x, nq=0, nkv=1, d=d, k_cache=kc, v_cache=vc, scales=scales, q_w=None, k_w=None, eps=0.0, cos=None, sin=None,
                block_table=ints([[0, 9], [1, 9], [-1, 9], [4, 9], [3, 3]]), cu_q=ints([0, 1, 2, 3, 4, 5]), k_len=ints([1, 1, 1, 1, 30]), max_k_len=20)
    assert scales[0].tolist() == [[2.0 ** -64] * 2] and scales[1].tolist() == [[2.0 ** 120] * 2]
    assert kc[1, 0, 0].float().tolist() == [256.0] * d          # 2^128 - 2^104 in 2^120, to four digits
    assert not scales[2:].any() and not kc[2:].float().any() and not vc[2:].float().any()


def test_rows_of_a_wider_tensor_and_either_half_alone():
    k, nq, nkv, d, P = kernels_for("bf16"), 4, 2, 64, 16
    rng = np.random.default_rng(5)
    wide = torch.from_numpy(rng.standard_normal((9, (nq + 2 * nkv) * d + 24))).to(torch.bfloat16).cuda()
    rows = wide[:, 16:16 + (nq + 2 * nkv) * d]
    cos, sin = rotation(16, d // 2, torch.bfloat16)
    common = dict(d=d, q_w=None, k_w=None, eps=0.0, cos=cos, sin=sin, block_table=ints([[1]]), cu_q=ints([0, 9]), k_len=ints([9]), max_k_len=9)
    one, two = k.empty_cache8(2, nkv, P, d), k.empty_cache8(2, nkv, P, d)
    q = k.qkv_post8(rows, nq=nq, nkv=nkv, k_cache=one[0], v_cache=one[1], scales=one[2], **common)
    q2 = k.qkv_post8(rows[:, :nq * d], nq=nq, nkv=0, k_cache=None, v_cache=None, scales=None, **common)
    assert k.qkv_post8(rows[:, nq * d:].contiguous(), nq=0, nkv=nkv, k_cache=two[0], v_cache=two[1], scales=two[2], **common) is None
    assert torch.equal(q, q2)
    for a, b in zip(one, two):
        assert np.array_equal(host(a), host(b))


# ------------------------------------------------------------------------------------------------------ attention
def close(got, plain, name, d):
    """A result is off by half a step of its type; by the weights' rounding, in the sum of weights times values and in that of weights alike: weights w (1 + e) with |e| at most half a
    step of sixteen-bit floating point, 2^-11, move it by at most 2^-11 of the mean of |v - out|, at most that of |v| and |out|; those below 2^-24 of the largest are off by up
    to 2^-25 of it, which moves it by 2^-25 of the sum of |v - out|; and by the scores', sums of d products in 32 bits: (d + 16) 2^-24 of the largest sum of |q k|, twice
    (numerator and denominator), and 2^-20 for the exponentials."""
    out, weighted, most, flushed = plain
    dtype = TYPES[name]
    score = 2 * (d + 16) * 2.0 ** -24 * most + 2.0 ** -20
    weights = 2.0 ** -11 if name == "bf16" else 2.0 ** -20
    bound = torch.finfo(dtype).eps / 2 * np.abs(out) * 1.01 + (weighted + np.abs(out)) * weights + weighted * score + (2.0 ** -25 if name == "bf16" else 0.0) * flushed + 1e-30
    got = host(got)
    assert np.array_equal(np.isnan(got), np.isnan(out)), np.argwhere(np.isnan(got) != np.isnan(out))[:5]
    fine = ~np.isnan(out)
    off = np.abs(got - out)[fine] / bound[fine]
    assert off.size == 0 or off.max() <= 1, (off.max(), got[fine][off.argmax()], out[fine][off.argmax()])


def items_of(rows, most):
    return ints([(s, a) for s, n in enumerate(rows) for a in range(0, n, most)] or np.zeros((0, 2)))


def attend(k, q, cache, table, rows, keys, most, window=0, scale=None, max_k_len=None, **kw):
    return k.paged_attention8(q, *cache, ints(table), ints(np.concatenate([[0], np.cumsum(rows)])), ints(keys), items_of(rows, most), item_rows=most,
                              scale=q.shape[2] ** -0.5 if scale is None else scale, window=window, max_k_len=max(keys) if max_k_len is None else max_k_len, **kw)


ATTENDS = [
    # (type, rows, keys, nq, nkv, d, P, window, rows of an item)
    ("bf16", [1], [1], 2, 1, 16, 16, 0, 1),
    ("bf16", [1, 1, 1, 1], [63, 64, 65, 1030], 8, 2, 128, 64, 0, 1),
    ("bf16", [1, 1], [300, 2000], 16, 2, 64, 16, 0, 1),
    ("bf16", [5, 3, 1], [5, 259, 700], 10, 2, 128, 64, 0, 5),
    ("bf16", [9, 16], [9, 300], 16, 2, 80, 32, 0, 16),
    ("bf16", [16], [513], 64, 1, 128, 128, 0, 16),
    ("bf16", [4, 1, 2], [900, 3, 600], 8, 8, 256, 64, 0, 4),
    ("bf16", [3, 2], [400, 64], 6, 1, 192, 256, 0, 3),
    ("bf16", [2, 5, 1], [700, 300, 40], 12, 4, 96, 16, 100, 5),
    ("bf16", [1, 3], [600, 520], 4, 2, 128, 64, 1, 3),
    ("bf16", [17], [17], 4, 2, 128, 64, 0, 128),
    ("bf16", [150, 20, 1], [150, 333, 70], 8, 2, 128, 64, 0, 128),
    ("bf16", [130, 60], [200, 60], 5, 1, 64, 16, 33, 128),
    ("bf16", [70], [200], 3, 3, 256, 32, 0, 64),
    ("bf16", [40], [41], 14, 2, 192, 128, 0, 40),
    ("bf16", [33, 18], [100, 18], 6, 2, 32, 16, 7, 33),
    ("f32", [1, 1], [64, 515], 8, 2, 64, 16, 0, 1),
    ("f32", [4, 2], [300, 7], 16, 2, 128, 64, 0, 4),
    ("f32", [7], [260], 8, 1, 256, 32, 50, 7),
    ("f32", [3], [70], 2, 2, 192, 16, 0, 3),
    ("f32", [66, 20], [100, 300], 4, 2, 80, 16, 0, 128),
    ("f32", [30], [90], 4, 1, 256, 64, 20, 30),
    ("f32", [140], [140], 2, 1, 64, 64, 0, 128),
    ("f32", [25], [50], 3, 1, 128, 64, 0, 25),
    # Columns (rows of an item times q heads of a kv head) from one tile to more than a workgroup takes at once, for every width of a head.
    ("bf16", [8, 3], [700, 40], 8, 2, 64, 64, 0, 8),
    ("bf16", [12, 7], [530, 1100], 8, 2, 48, 16, 90, 12),
    ("bf16", [16, 1], [100, 600], 4, 1, 64, 32, 0, 16),
    ("bf16", [16, 9], [620, 30], 5, 1, 32, 64, 0, 16),
    ("bf16", [4, 2], [1040, 300], 16, 2, 128, 64, 0, 4),
    ("bf16", [3, 3], [70, 600], 8, 1, 112, 16, 65, 3),
    ("bf16", [5, 2], [513, 90], 8, 1, 128, 128, 0, 5),
    ("bf16", [4], [600], 8, 1, 192, 64, 0, 4),
    ("bf16", [7], [130], 8, 1, 144, 32, 40, 7),
    ("bf16", [2, 2], [520, 33], 16, 1, 256, 64, 0, 2),
    ("bf16", [11], [700], 8, 1, 208, 16, 0, 11),
    ("bf16", [100], [140], 8, 8, 160, 64, 0, 100),
    ("f32", [4, 1], [600, 20], 8, 1, 64, 64, 0, 4),
    ("f32", [3], [530], 8, 1, 128, 16, 0, 3),
    ("f32", [6], [90], 8, 1, 96, 64, 30, 6),
    ("f32", [3], [520], 8, 1, 176, 32, 0, 3),
    ("f32", [2, 5], [30, 513], 10, 1, 256, 64, 0, 5),
    ("f32", [9], [65], 1, 1, 256, 256, 0, 9),
    # So many sequences that a workgroup takes several segments of one, among them more than 64 pages; the last ones without a key in it.
    ("bf16", [1] * 300, [1930 - 6 * i for i in range(300)], 4, 4, 16, 16, 0, 1),
    ("bf16", [2] * 300, [130 + 7 * i for i in range(300)], 8, 4, 16, 32, 300, 2),
    ("f32", [4] * 90, [1500 - 15 * i for i in range(90)], 32, 4, 32, 16, 0, 4),
    # Prompts on more than 64 pages.
    ("bf16", [40], [2500], 4, 1, 64, 16, 0, 128),
    ("bf16", [140, 20], [1400, 3000], 2, 1, 128, 16, 1500, 128),
    ("bf16", [30], [4300], 2, 2, 256, 32, 0, 64),
    ("f32", [20], [1300], 2, 1, 64, 16, 0, 128),
]


@pytest.mark.parametrize("case", range(len(ATTENDS)))
def test_attention_is_the_formula(case):
    name, rows, keys, nq, nkv, d, P, window, most = ATTENDS[case]
    k = kernels_for(name)
    rng = np.random.default_rng(100 + case)
    table, pages = tables(rng, keys, P)
    cache = filled(rng, pages, nkv, P, d)
    q = torch.from_numpy(rng.standard_normal((sum(rows), nq, d)) * 1.5).to(TYPES[name]).cuda()
    got = attend(k, q, cache, table, rows, keys, most, window)
    close(got, attention(host(q), *map(host, cache), table, np.concatenate([[0], np.cumsum(rows)]), keys, d ** -0.5, window), name, d)
    # A larger bound changes nothing (the table is wider, the launch covers more keys).
    wide = np.full((len(keys), table.shape[1] + 9), -1)
    wide[:, :table.shape[1]] = table
    assert torch.equal(got, attend(k, q, cache, wide, rows, keys, most, window, max_k_len=wide.shape[1] * P))


@pytest.mark.parametrize("name", ["bf16", "f32"])
@pytest.mark.parametrize("most", [6, 40])
def test_nan_is_seen_where_it_is_visible_and_nowhere_else(name, most):
    """NaN in keys that only later rows see, in keys before the window, behind the last key and in pages of nobody; in keys and in values."""
    k, P, d, nkv, nq, window = kernels_for(name), 32, 64, 2, 4, 70
    rng = np.random.default_rng(8)
    rows, keys = [most, 3], [100 + most, 80]
    table, pages = tables(rng, keys, P)
    kc, vc, scales = filled(rng, pages, nkv, P, d)
    nan = float("nan")
    kf, vf = kc.float(), vc.float()
    kf[table[0, 3], 0, (100 + most // 2) % P] = nan                 # seen by the rows from the middle one on (both fall in the fourth page)
    vf[table[0, 3], 1, 5, (100 + most // 2) % P] = nan
    kf[table[0, 0]] = nan                                           # keys 0..31: before every row's window
    vf[table[0, 0]] = nan
    vf[table[0, 1], 0, 9, 1] = nan                                  # key 33: seen by the first rows alone
    last = keys[1] % P                                              # behind sequence 1's last key
    kf[table[1, 2], :, last:] = nan
    vf[table[1, 2], :, :, last:] = nan
    kc, vc = kf.to(E4M3), vf.to(E4M3)
    q = torch.from_numpy(rng.standard_normal((sum(rows), nq, d))).to(TYPES[name]).cuda()
    got = attend(k, q, (kc, vc, scales), table, rows, keys, most, window)
    plain = attention(host(q), host(kc), host(vc), host(scales), table, np.concatenate([[0], np.cumsum(rows)]), keys, d ** -0.5, window)
    assert np.isnan(plain[0]).any() and not np.isnan(plain[0]).all(axis=(1, 2)).all()
    close(got, plain, name, d)


@pytest.mark.parametrize("most", [1, 20])
def test_rows_without_keys_are_zero_and_rows_of_no_item_stay(most):
    k, P, d = kernels_for("bf16"), 16, 64
    rng = np.random.default_rng(9)
    rows, keys = [most, most, most], [0, most + 30, most]
    table, pages = tables(rng, [16, 64, 32], P)
    table[2] = -1                                                   # pages of nothing: no keys
    cache = filled(rng, pages, 2, P, d)
    q = torch.from_numpy(rng.standard_normal((sum(rows) + 2, 4, d))).to(torch.bfloat16).cuda()
    out = torch.full_like(q, 7.0)
    cu = ints(np.concatenate([[0], np.cumsum(rows)]))
    k.paged_attention8(q, *cache, ints(table), cu, ints(keys), ints([(0, 0), (1, 0), (2, 0), (3, 0), (-1, 0), (1, most), (1, -1)]), item_rows=most, scale=0.1, max_k_len=most + 30, out=out)
    got = host(out)
    assert (got[:most] == 0).all() and (got[2 * most:3 * most] == 0).all() and (got[3 * most:] == 7).all()
    close(out[most:2 * most], attention(host(q[most:2 * most]), *map(host, cache), table[1:2], [0, most], keys[1:2], 0.1), "bf16", d)


@pytest.mark.parametrize("name,most", [("bf16", 4), ("bf16", 30), ("f32", 4), ("f32", 30)])
def test_pages_of_very_different_scales(name, most):
    """Scales 2^-40 to 2^20 beside one another: values relative to their neighbours' lose what lies 2^-24 below the largest page's and less."""
    k, P, d = kernels_for(name), 16, 64
    rng = np.random.default_rng(11)
    rows, keys = [most], [300]
    table, pages = tables(rng, keys, P)
    kc, vc, scales = filled(rng, pages, 1, P, d)
    scales[:, :, 1] = torch.from_numpy(2.0 ** rng.integers(-40, 20, (pages, 1))).to(torch.float32)
    q = torch.from_numpy(rng.standard_normal((most, 4, d))).to(TYPES[name]).cuda()
    got = attend(k, q, (kc, vc, scales), table, rows, keys, most)
    plain = attention(host(q), host(kc), host(vc), host(scales), table, [0, most], keys, d ** -0.5)
    close(got, plain, name, d)


@pytest.mark.parametrize("name", ["bf16", "f32"])
def test_a_row_is_the_same_bits_in_any_company(name):
    """Few rows: whatever other sequences, items and bounds are in the call, and on every repetition."""
    k, P, d, nq, nkv = kernels_for(name), 64, 128, 8, 2
    rng = np.random.default_rng(12)
    rows, keys = [3, 1, 3, 2], [1500, 90, 700, 2]
    table, pages = tables(rng, keys, P)
    cache = filled(rng, pages, nkv, P, d)
    q = torch.from_numpy(rng.standard_normal((sum(rows), nq, d))).to(TYPES[name]).cuda()
    got = attend(k, q, cache, table, rows, keys, 3)
    assert torch.equal(got, attend(k, q, cache, table, rows, keys, 3))
    at = 0
    for s, n in enumerate(rows):
        alone = attend(k, q[at:at + n].contiguous(), cache, table[s:s + 1], [n], keys[s:s + 1], 3, max_k_len=1500)
        assert torch.equal(got[at:at + n], alone)
        at += n


def test_arrays_that_say_more_than_there_is():
    """Lengths beyond the bound, rows and sequences that the arrays do not have, a table of numbers of nothing: what exists is computed, the rest left as it was."""
    k, P, d = kernels_for("bf16"), 16, 64
    rng = np.random.default_rng(21)
    cache = filled(rng, 6, 1, P, d)
    table = np.array([[0, 1, 2, 3], [4, -7, 10 ** 9, 6], [5, 5, 5, 5], [1, 1, 1, 1], [2, 2, 2, 2]])
    for rows in (3, 30):
        q = torch.from_numpy(rng.standard_normal((4 * rows, 2, d))).to(torch.bfloat16).cuda()
        cu = ints([0, rows, 2 * rows, 3 * rows, 2 ** 31 - 1, -2 ** 31])
        keys = ints([2 ** 31 - 1, 40, -2 ** 31, 9, 9])
        out = torch.full_like(q, 7.0)
        items = ints([(0, 0), (1, 0), (2, 0), (3, 0), (4, 0), (0, 2 ** 31 - 1), (5, 0), (-2 ** 31, 0), (2, rows - 1)])
        k.paged_attention8(q, *cache, ints(table), cu, keys, items, item_rows=rows, scale=0.1, max_k_len=50, out=out)
        # Sequence 0's rows stand far behind the bound and see all 50 keys below it; 1 has the keys of its one page; 2 has none; 3 and 4 do not exist.
        kk = host(cache[0])[[0, 1, 2, 3], 0] * host(cache[2])[[0, 1, 2, 3], 0, 0][:, None, None]
        vv = host(cache[1])[[0, 1, 2, 3], 0].swapaxes(1, 2) * host(cache[2])[[0, 1, 2, 3], 0, 1][:, None, None]
        kk, vv = kk.reshape(-1, d)[:50], vv.reshape(-1, d)[:50]
        w = np.exp(0.1 * host(q[:rows]) @ kk.T)
        want = (w / w.sum(-1, keepdims=True)) @ vv
        assert np.abs(host(out[:rows]) - want).max() <= 2.0 ** -7 * np.abs(vv).max()
        close(out[rows:2 * rows], attention(host(q[rows:2 * rows]), *map(host, cache), table[1:2], [0, rows], [40], 0.1), "bf16", d)
        assert not out[2 * rows:3 * rows].any() and out[3 * rows:].eq(7.0).all()
    before = [host(t) for t in cache]
    x = torch.ones(12, 2 * d, dtype=torch.bfloat16, device="cuda")
    k.qkv_post8(x, nq=0, nkv=1, d=d, k_cache=cache[0], v_cache=cache[1], scales=cache[2], q_w=None, k_w=None, eps=0.0, cos=None, sin=None, block_table=ints(table),
                cu_q=ints([0, 3, 6, 2 ** 31 - 1, -2 ** 31, -1]), k_len=ints([2 ** 31 - 1, 2, 9, 9, -2 ** 31]), max_k_len=60)
    for a, b in zip(cache, before):
        assert np.array_equal(host(a), b)


def test_scales_before_the_window_do_not_matter():
    """A page that lies before every row's window has been given to another sequence, with a scale of another size."""
    k, P, d, window = kernels_for("bf16"), 16, 64, 20
    rng = np.random.default_rng(22)
    for most in (2, 24):
        rows, keys = [most], [110]
        table, pages = tables(rng, keys, P)
        kc, vc, scales = filled(rng, pages, 1, P, d)
        q = torch.from_numpy(rng.standard_normal((most, 4, d))).to(torch.bfloat16).cuda()
        want = attend(k, q, (kc, vc, scales), table, rows, keys, most, window)
        first = (110 - most - window + 1) // P
        scales[table[0, :first]] = 2.0 ** 100
        scales[table[0, 0]] = float("nan")
        assert torch.equal(want, attend(k, q, (kc, vc, scales), table, rows, keys, most, window))
        table[0, :first] = -1
        assert torch.equal(want, attend(k, q, (kc, vc, scales), table, rows, keys, most, window))


@pytest.mark.parametrize("d", (64, 128, 256))
@pytest.mark.parametrize("rows", (1, 5, 20))
def test_heads_of_small_and_large_entries(d, rows):
    """q whose entries lie far apart, the largest against keys that are 0 there.  Heads of 128 and 256 are held by two numbers of four digits: entries below 2^-14 of the largest's power of two are off by
    up to 2^-22 of it, which moves a score by that times the sum of |k|, and a result by twice that (numerator and denominator) of the mean of |v - out|, at most that of |v| and |out|."""
    k, P, nq, nkv, keys = kernels_for("bf16"), 64, 4, 2, 150
    rng = np.random.default_rng(d + rows)
    table, pages = tables(rng, [keys], P)
    kc, vc, scales = filled(rng, pages, nkv, P, d, -9, -6)
    kc[..., 3] = 0
    q = rng.standard_normal((rows, nq, d)) * 2.0 ** rng.integers(-16, 2, (rows, nq, d))
    for at, size in enumerate((2.0 ** 9, 2.0 ** 14, 2.0 ** 40, 0.0)):
        q[:, at, 3] = size
    q = torch.from_numpy(q).to(torch.bfloat16).cuda()
    got = host(attend(k, q, (kc, vc, scales), table, [rows], [keys], 16 if rows < 16 else 128))
    out, weighted, most, flushed = attention(host(q), *map(host, (kc, vc, scales)), table, [0, rows], [keys], d ** -0.5)
    power = 2.0 ** np.floor(np.log2(np.abs(host(q)).max(-1, keepdims=True)))
    size = (np.abs(host(kc)).sum(-1) * host(scales)[:, :, None, 0]).max() * d ** -0.5
    moved = 2.0 ** -22 * power * size + 2 * (d + 16) * 2.0 ** -24 * most + 2.0 ** -20
    bound = 2.0 ** -8 * 1.01 * np.abs(out) + (weighted + np.abs(out)) * (2.0 ** -11 + 2 * moved) + 2.0 ** -25 * flushed + 1e-30
    assert (np.abs(got - out) <= bound)[:, [0, 1, 3]].all()
    assert np.isfinite(got[:, 2]).all() and np.abs(got[:, 2]).max() <= np.abs(host(vc) * host(scales)[:, :, 1, None, None]).max() * 1.01
    q[0, 1, d - 1] = float("nan")
    more = host(attend(k, q, (kc, vc, scales), table, [rows], [keys], 16 if rows < 16 else 128))
    assert np.isnan(more[0, 1]).all()
    more[0, 1] = got[0, 1]
    assert np.array_equal(more, got)


@pytest.mark.parametrize("name", ["bf16", "f32"])
@pytest.mark.parametrize("rows", (1, 9, 20))
@pytest.mark.parametrize("d", (64, 128))
def test_scores_that_32_bits_hold_to_a_hundred(name, rows, d):
    """Scores of 2^30 and more: a weight is what 32 bits make of it, but no more than 1 beside the largest, so that a result lies among the values; and where one key is ahead by far it is that key's."""
    k, P, nq, nkv, keys = kernels_for(name), 64, 4, 2, 700
    rng = np.random.default_rng(rows + d)
    table, pages = tables(rng, [keys], P)
    kc, vc, scales = filled(rng, pages, nkv, P, d)
    scales[..., 0] = 2.0 ** 12
    q = torch.from_numpy(rng.standard_normal((rows, nq, d)) * 2.0 ** 14).to(TYPES[name]).cuda()
    most = 16 if rows < 16 else 128
    got = host(attend(k, q, (kc, vc, scales), table, [rows], [keys], most))
    vv = host(vc) * host(scales)[:, :, 1, None, None]
    assert np.isfinite(got).all() and np.abs(got).max() <= np.abs(vv).max() * (1 + 2.0 ** -8)
    # Beside such heads another one is what it is beside small ones.
    small = torch.from_numpy(rng.standard_normal((rows, nq, d)) * 2.0 ** -16).to(TYPES[name]).cuda()
    beside = q.clone()
    beside[:, 1] = small[:, 1]
    assert torch.equal(attend(k, beside, (kc, vc, scales), table, [rows], [keys], most)[:, 1], attend(k, small, (kc, vc, scales), table, [rows], [keys], most)[:, 1])
    # Place 5 of the sequence along q's first row's heads, its other places across them.
    kc[:] = torch.zeros((), device="cuda").to(E4M3)
    page = int(table[0, 0])
    q[:] = 0
    q[..., 0] = 2.0 ** 14
    kc[page, :, 5, 0] = torch.tensor(256.0, device="cuda").to(E4M3)
    got = host(attend(k, q, (kc, vc, scales), table, [rows], [keys], most))
    want = vv[page, :, :, 5].repeat(nq // nkv, 0)[None]
    assert (np.abs(got - want) <= torch.finfo(TYPES[name]).eps / 2 * np.abs(want) + 2.0 ** -20 * np.abs(want).max()).all()


@pytest.mark.parametrize("most", (16, 128))
def test_a_window_longer_than_the_keys_hides_none(most):
    """Among rows that stand before the first key, where a window's begin could leave 32 bits."""
    k, P, d = kernels_for("bf16"), 32, 64
    rng = np.random.default_rng(23)
    rows, keys = [40, 3], [25, 60]
    table, pages = tables(rng, keys, P)
    cache = filled(rng, pages, 2, P, d)
    q = torch.from_numpy(rng.standard_normal((43, 4, d))).to(torch.bfloat16).cuda()
    want = attend(k, q, cache, table, rows, keys, most)
    assert not want[:15].any() and want[15:].abs().amax(-1).gt(0).all()
    for window in (60, 64, 2 ** 31 - 1):
        assert torch.equal(want, attend(k, q, cache, table, rows, keys, most, window))


def test_on_streams_of_their_own():
    """Two calls at once, each with its own memory, in either order."""
    k, P, d = kernels_for("bf16"), 64, 128
    rng = np.random.default_rng(23)
    work = []
    for keys in ([3000, 200], [900, 1500]):
        table, pages = tables(rng, keys, P)
        cache = filled(rng, pages, 2, P, d)
        q = torch.from_numpy(rng.standard_normal((4, 8, d))).to(torch.bfloat16).cuda()
        work.append((q, cache, table, keys, attend(k, q, cache, table, [2, 2], keys, 2)))
    streams = [torch.cuda.Stream() for _ in work]
    torch.cuda.synchronize()
    for _ in range(5):
        got = []
        for (q, cache, table, keys, _), st in zip(work, streams):
            with torch.cuda.stream(st):
                got.append(attend(k, q, cache, table, [2, 2], keys, 2))
        torch.cuda.synchronize()
        for (*_, want), g in zip(work, got):
            assert torch.equal(want, g)


def test_offsets_beyond_32_bits():
    """Pages whose entries lie beyond 4 GiB, written and read."""
    k, P, d, nkv = kernels_for("bf16"), 64, 128, 8
    pages = 70000                                                   # 4.6 GB of keys, as much of values
    kc, vc, scales = k.empty_cache8(pages, nkv, P, d)
    rng = np.random.default_rng(13)
    table = np.array([[pages - 1, 3, pages - 7]])
    x = torch.from_numpy(rng.standard_normal((150, 3 * nkv * d))).to(torch.bfloat16).cuda()
    q = k.qkv_post8(x, nq=nkv, nkv=nkv, d=d, k_cache=kc, v_cache=vc, scales=scales, q_w=None, k_w=None, eps=0.0, cos=None, sin=None, block_table=ints(table),
                    cu_q=ints([0, 150]), k_len=ints([150]), max_k_len=150)
    small = k.empty_cache8(10, nkv, P, d)
    k.qkv_post8(x, nq=nkv, nkv=nkv, d=d, k_cache=small[0], v_cache=small[1], scales=small[2], q_w=None, k_w=None, eps=0.0, cos=None, sin=None,
                block_table=ints([[9, 3, 5]]), cu_q=ints([0, 150]), k_len=ints([150]), max_k_len=150)
    for big, little in zip((kc, vc, scales), small):
        for a, b in ((pages - 1, 9), (3, 3), (pages - 7, 5)):
            assert np.array_equal(host(big[a]), host(little[b]))
    for most in (16, 128):
        assert torch.equal(attend(k, q, (kc, vc, scales), table, [150], [150], most), attend(k, q, small, [[9, 3, 5]], [150], [150], most))


def test_refusals():
    k = kernels_for("bf16")
    kc, vc, sc = k.empty_cache8(4, 2, 16, 64)
    q = torch.zeros(3, 4, 64, dtype=torch.bfloat16, device="cuda")
    x = torch.zeros(3, 8 * 64, dtype=torch.bfloat16, device="cuda")
    table, cu, kl, it = ints([[0, 1]]), ints([0, 3]), ints([3]), ints([[0, 0]])

    def att(q=q, kc=kc, vc=vc, sc=sc, table=table, cu=cu, kl=kl, it=it, **kw):
        return k.paged_attention8(q, kc, vc, sc, table, cu, kl, it, **{**dict(item_rows=3, scale=0.1, max_k_len=32), **kw})

    def put(x=x, **kw):
        return k.qkv_post8(x, **{**dict(nq=4, nkv=2, d=64, k_cache=kc, v_cache=vc, scales=sc, q_w=None, k_w=None, eps=0.0, cos=None, sin=None, block_table=table, cu_q=cu,
                                        k_len=kl, max_k_len=32), **kw})
    att(), put()
    for bad in (dict(q=q.float()), dict(q=q[:, :, :32]), dict(q=q.cpu()), dict(q=q[:, :3].contiguous()), dict(kc=kc.float()), dict(vc=kc), dict(sc=sc[:, :1]), dict(table=table.long()),
                dict(cu=ints([0])), dict(kl=ints([3, 3])), dict(it=ints([0, 0])), dict(item_rows=0), dict(item_rows=129), dict(window=-1), dict(max_k_len=33),
                dict(out=q[:2]), dict(max_k_len=-1), dict(item_rows=-1), dict(window=2 ** 32 + 5), dict(max_k_len=2 ** 32 + 5)):
        with pytest.raises(KernelError):
            att(**bad)
    small = k.empty_cache8(4, 2, 8, 64), k.empty_cache8(2, 2, 512, 64), k.empty_cache8(2, 2, 48, 64)
    for c in small:
        with pytest.raises(KernelError):
            att(kc=c[0], vc=c[1], sc=c[2])
        with pytest.raises(KernelError):
            put(k_cache=c[0], v_cache=c[1], scales=c[2])
    with pytest.raises(KernelError):                                # scratch too small
        att(table=ints([list(range(4)) * 10]), max_k_len=600, scratch=torch.empty(8, device="cuda"))
    cos = torch.zeros(32, 32, dtype=torch.bfloat16, device="cuda")
    put(cos=cos, sin=cos)
    for bad in (dict(x=x[:, 1:]), dict(x=x.float()), dict(x=x.t()), dict(nq=3), dict(d=24, x=x[:, :192].contiguous()), dict(cos=cos[:31], sin=cos[:31]), dict(cos=cos, sin=cos.float()),
                dict(cos=torch.zeros(32, 33, dtype=torch.bfloat16, device="cuda"), sin=torch.zeros(32, 33, dtype=torch.bfloat16, device="cuda")), dict(q_w=x[0, :32]),
                dict(q_w=x[0, :64].contiguous(), k_w=torch.zeros(64, device="cuda")), dict(max_k_len=33), dict(max_k_len=2 ** 32 + 5), dict(max_k_len=-1), dict(q_out=q[:2]), dict(k_cache=vc), dict(scales=sc.double())):
        with pytest.raises(KernelError):
            put(**bad)
    unaligned = torch.zeros(3 * 512 + 1, dtype=torch.bfloat16, device="cuda")[1:].view(3, 512)
    with pytest.raises(KernelError):
        put(x=unaligned)
