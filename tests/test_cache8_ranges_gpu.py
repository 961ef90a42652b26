"""Attention over an 8-bit cache (attention8.hip) where numbers lie far apart: scales of neighbouring pages, weights of neighbouring keys."""
import numpy as np
import pytest
import torch

from plain_cache8 import attention
from test_cache8_gpu import TYPES, attend, close, filled, host, tables
from vosti_amd.kernels import kernels_for

pytestmark = pytest.mark.gpu


def case(name, d, P, rows, keys, seed, nq=4, nkv=2, size=1.0):
    rng = np.random.default_rng(seed)
    table, pages = tables(rng, [keys], P)
    q = torch.from_numpy(rng.standard_normal((rows, nq, d)) * size).to(TYPES[name]).cuda()
    return table, filled(rng, pages, nkv, P, d, -6, -4), q


def check(name, q, cache, table, rows, keys, window=0, without=()):
    """The bounds of `close`, which hold each row to the values that it sees itself; `without`: pages of the sequence that weigh nothing and are none to the plain form and its bounds."""
    got = attend(kernels_for(name), q, cache, table, [rows], [keys], 16 if rows <= 16 else 128, window)
    seen = table.copy()
    seen[0, list(without)] = -1
    close(got, attention(host(q), *map(host, cache), seen, [0, rows], [keys], q.shape[2] ** -0.5, window), name, q.shape[2])


@pytest.mark.parametrize("up", (15, 16, 30, 60))
@pytest.mark.parametrize("P", (16, 64))
@pytest.mark.parametrize("name,d,rows", [("bf16", 64, 5), ("bf16", 64, 20), ("bf16", 128, 5), ("bf16", 128, 11), ("bf16", 128, 20), ("bf16", 256, 20), ("f32", 64, 5), ("f32", 64, 20)])
def test_a_large_page_that_one_row_sees_leaves_the_others(name, d, rows, P, up):
    """A page whose values stand 2^up above the others': seen by the first row alone, the window of the next ones beginning behind it; and by the last row alone, which stands in its first place."""
    window, at = 70, 6
    keys = P * at + P - 1 + window - 1 + rows                  # row 0 sees the last place of page `at`
    table, (kc, vc, scales), q = case(name, d, P, rows, keys, d + rows + P + up)
    scales[..., 1] = 2.0 ** -5
    scales[int(table[0, at]), :, 1] = 2.0 ** (up - 5)
    check(name, q, (kc, vc, scales), table, rows, keys, window)
    keys = P * at + 1                                          # the last row sees the first place of page `at`
    scales[..., 1] = 2.0 ** -5
    scales[int(table[0, at]), :, 1] = 2.0 ** (up - 5)
    check(name, q, (kc, vc, scales), table, rows, keys)


@pytest.mark.parametrize("up", (15, 30))
@pytest.mark.parametrize("P", (16, 32, 64))
@pytest.mark.parametrize("name,d,rows", [("bf16", 64, 1), ("bf16", 64, 20), ("bf16", 128, 1), ("bf16", 128, 9), ("bf16", 128, 20), ("bf16", 192, 9), ("f32", 128, 9)])
def test_a_large_page_of_no_weight_leaves_the_others(name, d, rows, P, up):
    """Pages 2^up above the others in whose keys every score is some 90 powers of two behind, which leaves 2^-40 of nothing: the first, one in the middle, the last but one."""
    keys = 300
    table, (kc, vc, scales), q = case(name, d, P, rows, keys, d + rows + P + up)
    scales[..., 0], scales[..., 1] = 2.0 ** -6, 2.0 ** -5
    kf = kc.float()
    kf[..., 0] = 0.0
    q[..., 0] = 8.0
    used = -(-keys // P)
    large = (0, used // 2, used - 2)
    for at in large:
        page = int(table[0, at])
        kf[page] = 0.0
        kf[page, ..., 0] = -round(90 * np.log(2) * d ** 0.5 / 8 * 2 ** 2)
        scales[page, :, 0], scales[page, :, 1] = 2.0 ** -2, 2.0 ** (up - 5)
    assert kf.abs().max() <= 448
    check(name, q, (kf.to(kc.dtype), vc, scales), table, rows, keys, without=large)


def test_a_small_page_beside_large_ones_is_exact():
    """The smallest entries there are, in pages of every distance from the one in front of them that another row sees: one key's value, to the bit."""
    k, d, P = kernels_for("bf16"), 64, 16
    for rows in (2, 20):
        for down in (1, 8, 14, 15, 16, 17, 22, 40):
            keys = 32 + rows - 1
            table, (kc, vc, scales), q = case("bf16", d, P, rows, keys, down)
            window = rows - 1                                 # the last row sees keys 32 .. 30 + rows, the first one 33 - rows .. 31
            scales[..., 1] = 1.0
            scales[table[0, 2:].tolist(), :, 1] = 2.0 ** -down
            kc[:] = torch.zeros((), device="cuda").to(kc.dtype)
            least = torch.full(vc.shape, 2.0 ** -9, device="cuda")
            least[:, :, ::2] *= 3
            vc = least.to(vc.dtype)
            got = host(attend(k, q, (kc, vc, scales), table, [rows], [keys], 16 if rows <= 16 else 128, window))[-1]
            assert np.array_equal(got, np.broadcast_to(host(least)[0, 0, :, 0] * 2.0 ** -down, got.shape)), (rows, down)


@pytest.mark.parametrize("behind", (20, 25, 29))
@pytest.mark.parametrize("name,d,P,rows,keys", [("bf16", 64, 64, 20, 4096), ("bf16", 64, 16, 20, 4000), ("bf16", 128, 64, 33, 2100), ("bf16", 256, 64, 17, 700), ("bf16", 128, 64, 1, 3000),
                                                ("bf16", 128, 64, 12, 1500), ("f32", 64, 64, 20, 4096)])
def test_weights_far_behind_one_key_of_no_value(name, d, P, rows, keys, behind):
    """The first key is 2^behind ahead of all others and its value is 0: what is left of the result is theirs.  A weight is off by 2^-11 of itself, or by 2^-32 of the largest (half of 2^-24 where the largest
    is 2^7 or more); otherwise the bounds are those of `close`."""
    table, (kc, vc, scales), q = case(name, d, P, rows, keys, d + keys + behind, size=0.25)
    scales[..., 0] = 2.0 ** -6
    scales[int(table[0, 0]), :, 0] = 1.0                       # (its other keys are zeros)
    kf, vf = kc.float(), vc.float().abs()
    kf[..., 0], q[..., 0] = 0.0, 8.0
    kf[int(table[0, 0])] = 0.0
    kf[int(table[0, 0]), :, 0, 0] = round(behind * np.log(2) * d ** 0.5 / 8)
    vf[int(table[0, 0]), :, :, 0] = 0.0
    kc, vc = kf.to(kc.dtype), vf.to(vc.dtype)
    got = host(attend(kernels_for(name), q, (kc, vc, scales), table, [rows], [keys], 16 if rows <= 16 else 128))
    out, weighted, most, flushed = attention(host(q), *map(host, (kc, vc, scales)), table, [0, rows], [keys], d ** -0.5)
    weights = 2.0 ** -11 if name == "bf16" else 2.0 ** -20
    score = 2 * (d + 16) * 2.0 ** -24 * most + 2.0 ** -20
    bound = torch.finfo(TYPES[name]).eps / 2 * out * 1.01 + (weighted + out) * weights + weighted * score + (2.0 ** -32 if name == "bf16" else 0.0) * flushed
    assert (np.abs(got - out) <= bound).all(), (np.abs(got - out) / bound).max()
    assert behind > 25 or (bound < 0.1 * out).all()            # the bounds say something


@pytest.mark.parametrize("name,d,rows,keys", [("bf16", 64, 1, 400), ("bf16", 64, 1, 700), ("bf16", 128, 2, 1200), ("bf16", 64, 8, 700), ("bf16", 128, 16, 300), ("bf16", 128, 20, 700), ("f32", 64, 2, 700)])
def test_values_near_the_largest_numbers(name, d, rows, keys):
    """Values to 2^114, and a key in the second tile of a wave's whose weight is 2^7.9 times that of the keys in the first: sums of weights times values leave 32 bits where a weight may be 2^15."""
    table, (kc, vc, scales), q = case(name, d, 64, rows, keys, d + keys)
    scales[..., 0], scales[..., 1] = 2.0 ** -6, 2.0 ** 105
    kf, vf = kc.float(), vc.float()
    kf[:], q[..., 0] = 0.0, 8.0
    page, place = int(table[0, 260 // 64]), 260 % 64
    scales[page, :, 0] = 2.0 ** -3
    kf[page, :, place, 0] = round(7.9 * np.log(2) * d ** 0.5)
    vf[page, :, :, place] = 448.0
    check(name, q, (kf.to(kc.dtype), vf.to(vc.dtype), scales), table, rows, keys)


@pytest.mark.parametrize("d", (48, 64, 80, 112, 144, 192, 208))
@pytest.mark.parametrize("rows", (1, 20))
def test_which_heads_take_q_whole(d, rows):
    """q with one entry far above the others, against keys that are 0 there.  Heads to 64 and of 129 to 192 entries take it whole and are held to the bounds of `close`; others hold entries below 2^-14 of the
    largest's power of two to 2^-22 of it, which moves a score by that times the sum of |k|, and a result by twice that of the mean of |v - out|, at most that of |v| and |out|."""
    k, keys = kernels_for("bf16"), 150
    table, (kc, vc, scales), q = case("bf16", d, 64, rows, keys, d + rows)
    kc[..., 3] = torch.zeros((), device="cuda").to(kc.dtype)
    q *= torch.from_numpy(2.0 ** np.random.default_rng(d).integers(-16, 1, tuple(q.shape))).to(q.dtype).cuda()
    q[..., 3] = torch.tensor([2.0 ** 9, 2.0 ** 14, 2.0 ** 9, 2.0 ** 14], device="cuda").to(q.dtype)
    if not 64 < d <= 128 and d <= 192:
        return check("bf16", q, (kc, vc, scales), table, rows, keys)
    got = host(attend(k, q, (kc, vc, scales), table, [rows], [keys], 16 if rows <= 16 else 128))
    out, weighted, most, flushed = attention(host(q), *map(host, (kc, vc, scales)), table, [0, rows], [keys], d ** -0.5)
    power = 2.0 ** np.floor(np.log2(np.abs(host(q)).max(-1, keepdims=True)))
    size = (np.abs(host(kc)).sum(-1) * host(scales)[:, :, None, 0]).max() * d ** -0.5
    moved = 2.0 ** -22 * power * size + 2 * (d + 16) * 2.0 ** -24 * most + 2.0 ** -20
    assert (np.abs(got - out) <= 2.0 ** -8 * 1.01 * np.abs(out) + (weighted + np.abs(out)) * (2.0 ** -11 + 2 * moved) + 2.0 ** -25 * flushed + 1e-30).all()


@pytest.mark.parametrize("order", ((0, -20, -40, -60), (-60, -40, -20, 0), (-20, -60, 0, -40)))
@pytest.mark.parametrize("name,d,rows", [("bf16", 64, 2), ("bf16", 128, 12), ("bf16", 128, 70), ("bf16", 256, 16), ("bf16", 192, 100), ("f32", 64, 70)])
def test_every_page_of_a_tile_in_a_scale_of_its_own(name, d, rows, order):
    """Pages of 16 keys in steps of 2^20 to 2^60, and windows of a key to two pages: each row is held to the values that it sees, in as many passes as a tile has pages."""
    for window in (1, 5, 16, 31):
        for keys in (70, 200 + rows):
            keys = max(keys, rows)
            table, (kc, vc, scales), q = case(name, d, 16, rows, keys, d + rows + window)
            for at in range(-(-keys // 16)):
                scales[int(table[0, at]), :, 1] = 2.0 ** order[at % 4]
            check(name, q, (kc, vc, scales), table, rows, keys, window)
