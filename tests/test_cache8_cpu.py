"""The refusals of the 8-bit cache's and the verification's C entries, which come before any launch, and the 64-bit formulas that the GPU tests compare with."""
import ctypes
import math
import re
from pathlib import Path

import numpy as np
import pytest

from plain_cache8 import attention, chances, e4m3, e4m3_numbers, exponent_for, store, verify
from vosti_amd.kernels import build
from vosti_amd.kernels.ops import ABI_VERSION, Kernels

GOOD = 1 << 20            # an address that nothing looks at


@pytest.fixture(scope="module", params=["bf16", "f32"])
def kernels(request):
    return Kernels(request.param)


def test_both_callers_ask_for_the_librarys_interface(kernels):
    """The native engine refuses a library of another number than its own, and so does the Python package."""
    source = (Path(build.__file__).parents[1] / "csrc" / "engine" / "gpu.cpp").read_text()
    assert kernels.lib.vk_abi_version() == ABI_VERSION == int(re.search(r"KERNEL_ABI = (\d+);", source).group(1))


def refused(kernels, fn, *args):
    assert fn(*args) != 0
    return kernels.lib.vk_last_error().decode()


def put(kernels, qkv=GOOD, stride=512, q_out=GOOD, kc=GOOD, vc=GOOD, scales=GOOD, cos=None, sin=None, half=0, W=4, T=3, S=1, nq=4, nkv=2, d=64, P=16, pages=4, max_k_len=32):
    return (kernels.lib.vk_qkv_post8, qkv, stride, q_out, kc, vc, scales, None, None, 0, cos, sin, half, GOOD, W, GOOD, GOOD, T, S, nq, nkv, d, P, pages, max_k_len, 1e-6, None)


@pytest.mark.parametrize("bad", [dict(T=-1), dict(S=-1), dict(nq=0, nkv=0), dict(nkv=-1), dict(d=24), dict(d=0), dict(d=272), dict(P=8), dict(P=48), dict(P=512), dict(stride=511),
                                 dict(stride=514), dict(cos=GOOD), dict(cos=GOOD, sin=GOOD, half=33), dict(cos=GOOD, sin=GOOD, half=0), dict(kc=None), dict(vc=None),
                                 dict(scales=None), dict(pages=0), dict(W=0), dict(q_out=None), dict(max_k_len=65), dict(max_k_len=-1), dict(qkv=GOOD + 2), dict(kc=GOOD + 8),
                                 dict(T=2 ** 31 - 1, nkv=64, nq=1, stride=129 * 64, S=1)])
def test_append_refuses(kernels, bad):
    assert "qkv_post8" in refused(kernels, *put(kernels, **bad))


def att(kernels, out=GOOD, q=GOOD, W=4, n=2, rows=3, scratch=None, floats=0, T=3, S=1, nq=4, nkv=2, d=64, P=16, pages=4, max_k_len=32, window=0, scale=0.125):
    return (kernels.lib.vk_paged_attention8, out, q, GOOD, GOOD, GOOD, GOOD, W, GOOD, GOOD, GOOD, n, rows, scratch, floats, T, S, nq, nkv, d, P, pages, max_k_len, window, scale, None)


@pytest.mark.parametrize("bad", [dict(T=-1), dict(n=-1), dict(nq=3), dict(nkv=0), dict(d=8), dict(d=100), dict(d=288), dict(P=8), dict(P=24), dict(P=1024), dict(rows=0), dict(rows=129),
                                 dict(pages=0), dict(W=0), dict(max_k_len=65), dict(max_k_len=-1), dict(window=-1), dict(scale=0.0), dict(scale=-0.1), dict(scale=math.nan), dict(scale=math.inf), dict(q=GOOD + 4), dict(out=GOOD + 8),
                                 dict(W=64, max_k_len=1000), dict(W=64, max_k_len=1000, scratch=GOOD, floats=100), dict(W=64, max_k_len=1000, scratch=GOOD + 4, floats=1 << 20),
                                 dict(W=2 ** 30, P=16, max_k_len=32)])
def test_attention_refuses(kernels, bad):
    assert "attention8" in refused(kernels, *att(kernels, **bad))


def test_scratch_of_attention(kernels):
    f = kernels.attn8_scratch_floats
    assert f(5, 17, 32, 128, 100000) == 0 and f(5, 4, 32, 128, 512) == 0 and f(0, 1, 32, 128, 5000) == 0
    assert f(5, 4, 32, 128, 513) == 5 * 4 * 32 * 2 * 130
    assert f(512, 16, 128, 256, 1 << 20) == 512 * 16 * 128 * 2048 * 258          # beyond 32 bits


def ver(kernels, tokens=GOOD, logits=GOOD, ids=GOOD, temps=None, au=None, du=None, scratch=GOOD, size=1 << 30, R=3, D=2, S=1, V=100):
    return (kernels.lib.vk_verify, tokens, GOOD, GOOD, logits, ids, GOOD, None, temps, au, du, scratch, size, R, D, S, V, None)


@pytest.mark.parametrize("bad", [dict(R=-1), dict(D=-1), dict(S=-1), dict(V=0), dict(V=1 << 30), dict(temps=GOOD), dict(temps=GOOD, du=GOOD), dict(temps=GOOD, au=GOOD), dict(tokens=None),
                                 dict(logits=None), dict(ids=None), dict(scratch=None), dict(scratch=GOOD + 8), dict(size=100), dict(V=(1 << 30) - 1, size=1 << 60)])
def test_verification_refuses(kernels, bad):
    assert "verify" in refused(kernels, *ver(kernels, **bad))


def test_nothing_to_do_is_no_error(kernels):
    for call in (put(kernels, T=0), put(kernels, S=0), att(kernels, n=0), att(kernels, T=0), att(kernels, S=0), ver(kernels, S=0)):
        assert call[0](*call[1:]) == 0


def test_tensors_on_the_cpu_are_refused(kernels):
    import torch
    from vosti_amd.kernels import KernelError
    x = torch.zeros(3, 512, dtype=kernels.dtype)
    with pytest.raises(KernelError):
        kernels.verify(x, torch.zeros(2, dtype=torch.int32), torch.zeros(2, dtype=torch.int32))
    with pytest.raises(KernelError):
        kernels.qkv_post8(x, nq=8, nkv=0, d=64, k_cache=None, v_cache=None, scales=None, q_w=None, k_w=None, eps=0.0, cos=None, sin=None,
                          block_table=torch.zeros(1, 1, dtype=torch.int32), cu_q=torch.zeros(2, dtype=torch.int32), k_len=torch.zeros(1, dtype=torch.int32), max_k_len=1)


# ------------------------------------------------------------------------------------------- the formulas themselves
def test_e4m3_is_torchs():
    import torch
    bits = torch.arange(256, dtype=torch.uint8).view(torch.float8_e4m3fn).double()
    assert np.array_equal(bits[:127].numpy(), e4m3_numbers()) and math.isnan(bits[127])
    x = torch.cat([bits[:127], (bits[:126] + bits[1:127]) / 2, torch.rand(5000, dtype=torch.float64, generator=torch.Generator().manual_seed(0)) * 448])
    x = torch.cat([x, -x]).float()                                        # the middles are 32-bit numbers
    assert np.array_equal(e4m3(x.double().numpy()), x.to(torch.float8_e4m3fn).double().numpy())


def test_exponents():
    assert [exponent_for(v) for v in (0.0, 448.0, 448.0001, 1.75, 1.76, 2.0 ** -80, 3.4e38)] == [-64, 0, 1, -8, -7, -64, 120]


def test_a_long_store_holds_what_attention_reads():
    """Attention over a cache that was filled in two calls, against softmax over the rows themselves, within what e4m3 keeps."""
    rng = np.random.default_rng(0)
    nq, nkv, d, P, n = 2, 1, 16, 16, 40
    x = rng.standard_normal((n, (nq + 2 * nkv) * d))
    k, v, s = np.zeros((4, 1, P, d)), np.zeros((4, 1, d, P)), np.zeros((4, 1, 2))
    table = np.array([[2, 0, 3]])
    q = [store(x[a:b], nq, nkv, d, k, v, s, None, None, 0.0, None, None, table, [0, b - a], [b]) for a, b in ((0, 21), (21, 40))]
    out = attention(np.concatenate(q), k, v, s, table, [0, n], [n], 0.25)[0]
    kk, vv = x[:, nq * d:(nq + 1) * d], x[:, (nq + 1) * d:]
    for r in range(n):
        for h in range(nq):
            w = np.exp(0.25 * kk[:r + 1] @ x[r, h * d:(h + 1) * d])
            assert np.abs(out[r, h] - w @ vv[:r + 1] / w.sum()).max() < 0.15


def test_verified_tokens_are_the_targets_distribution():
    """Over many numbers, drafts drawn from q and verified against p are p: the frequency of each first token within five standard deviations."""
    rng = np.random.default_rng(1)
    V, N = 6, 20000
    p, q = rng.standard_normal((2, V)) * 1.5, rng.standard_normal((1, V)) * 1.5
    ids = rng.choice(V, N, p=chances(q[0], 1.0))
    seen = np.zeros(V)
    u, w = rng.random((2, N))
    for i in range(N):
        seen[verify(p, ids[i:i + 1], [0, 2], q, [1.0], u[i:i + 1], w[i:i + 1])[0][0]] += 1
    want = chances(p[0], 1.0)
    assert (np.abs(seen / N - want) <= 5 * np.sqrt(want * (1 - want) / N)).all()


@pytest.mark.parametrize("window,rows,segments", [(1, 1, 1), (2, 1, 2), (1, 2, 2), (512, 1, 2), (513, 1, 2), (514, 1, 3), (510, 4, 2), (512, 16, 3), (1024, 5, 4), (5000, 1, 10), (4999, 1, 10), (0, 1, 10)])
def test_scratch_of_attention_with_a_window(kernels, window, rows, segments):
    """So many segments of 512 as that many neighbouring keys touch, of a bound of 5,000."""
    keys = window + rows - 1
    if 0 < window < 5000:
        touched = max((a + keys - 1) // 512 - a // 512 + 1 for a in range(1024))
        assert segments == min(touched, 10)
    assert kernels.attn8_scratch_floats(3, rows, 8, 64, 5000, window) == (3 * rows * 8 * 66 * segments if segments > 1 else 0)
