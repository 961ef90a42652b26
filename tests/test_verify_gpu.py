"""Verification of drafted tokens (verify.hip) against its definition in 64 bits, and a step over an 8-bit cache with drafted tokens as a whole."""
import numpy as np
import pytest
import torch

from plain_cache8 import attention, chances, store, verify
from vosti_amd.kernels import KernelError, kernels_for

pytestmark = pytest.mark.gpu
TYPES = {"bf16": torch.bfloat16, "f32": torch.float32}


def host(t):
    return None if t is None else t.detach().to(torch.float64).cpu().numpy()


def ints(values):
    return torch.tensor(np.asarray(values), dtype=torch.int32, device="cuda")


def floats(values):
    return torch.tensor(np.asarray(values, dtype=np.float32), device="cuda")


def check(name, logits, ids, cu, draft_logits=None, temps=None, accept_u=None, draw_u=None):
    """Tokens and counts are the definition's; the chances are off by their rounding to 32 bits and by the exponentials' 1.1e-12."""
    k = kernels_for(name)
    dev = lambda x: None if x is None else floats(x)   # noqa: E731
    got = k.verify(logits, ints(ids), ints(cu), draft_logits=draft_logits, temps=dev(temps), accept_uniforms=dev(accept_u), draw_uniforms=dev(draw_u))
    f32 = lambda x: None if x is None else np.asarray(x, dtype=np.float32).astype(np.float64)   # noqa: E731
    want = verify(host(logits), ids, cu, host(draft_logits), f32(temps), f32(accept_u), f32(draw_u))
    last = max(cu)
    assert got[0].cpu().numpy()[:last].tolist() == want[0][:last].tolist()
    assert got[1].cpu().numpy().tolist() == want[1].tolist()
    accept = got[2].cpu().numpy().astype(np.float64)
    told = ~np.isnan(want[2])
    assert (np.abs(accept - want[2])[told] <= 2.0 ** -24 * want[2][told] + 1e-12).all()
    return got


CASES = [
    # (type, drafts of each sequence, vocabulary, draft logits)
    ("bf16", [0], 1, False),
    ("bf16", [1, 0, 2], 2, True),
    ("bf16", [4], 503, True),
    ("bf16", [3, 0, 7, 1], 8191, True),
    ("bf16", [2, 5], 8193, False),
    ("bf16", [1] * 70 + [0, 3], 257, True),
    ("bf16", [4, 4, 0], 40007, True),
    ("bf16", [17], 20000, False),
    ("f32", [4, 0, 2], 503, True),
    ("f32", [1, 6], 16385, False),
    ("f32", [3, 3], 30001, True),
    # More pieces of sequences than a few rounds of workgroups: what stands is decided in a launch of its own.
    ("bf16", [2, 0, 1] * 300, 5000, True),
    ("f32", [1, 0, 17] + [1] * 300, 16385, False),
]


@pytest.mark.parametrize("case", range(len(CASES)))
def test_tokens_are_the_definitions(case):
    name, drafts, V, drawn = CASES[case]
    rng = np.random.default_rng(case)
    cu = np.concatenate([[0], np.cumsum(np.array(drafts) + 1)])
    R, D, S = cu[-1], sum(drafts), len(drafts)
    logits = torch.from_numpy(rng.standard_normal((R + 2, V)) * 3).to(TYPES[name]).cuda()      # two rows behind the last sequence
    of = np.arange(D) + np.repeat(np.arange(S), drafts)
    near = (logits[torch.from_numpy(of).long()].float() + torch.from_numpy(rng.standard_normal((D, V))).float().cuda()).to(TYPES[name])
    for temp in (0.7, 1.0, 0.0):
        for again in range(3):
            temps = np.where(rng.random(S) < 0.25, 0.0, temp)
            t = np.repeat(temps, drafts)
            ids = np.array([rng.choice(V, p=chances(host(near[i]) if drawn else host(logits[of[i]]), t[i])) for i in range(D)], dtype=int)
            check(name, logits, ids, cu, near if drawn else None, temps, rng.random(D), rng.random(S))
    check(name, logits, ids, cu, near if drawn else None)


def test_a_sequence_is_the_same_in_any_company():
    """Alone, and among so many that another launch decides."""
    k, V, S = kernels_for("bf16"), 5000, 900
    g = torch.Generator().manual_seed(3)
    logits, near = (torch.randn(n, V, generator=g).mul(2).to(torch.bfloat16).cuda() for n in (3 * S, 2 * S))
    ids, u, w = torch.randint(0, V, (2 * S,), generator=g, dtype=torch.int32).cuda(), torch.rand(2 * S, generator=g).mul(0.01).cuda(), torch.rand(S, generator=g).cuda()
    run = lambda a, b: k.verify(logits[3 * a:3 * b], ids[2 * a:2 * b], ints([3 * i for i in range(b - a + 1)]), draft_logits=near[2 * a:2 * b],   # noqa: E731
                                temps=torch.ones(b - a, device="cuda"), accept_uniforms=u[2 * a:2 * b], draw_uniforms=w[a:b])
    tokens, counts, accept = run(0, S)
    assert counts.unique().numel() > 1
    for s in (0, 1, 63, 64, 500, S - 1):
        one = run(s, s + 1)
        assert torch.equal(one[0], tokens[3 * s:3 * s + 3]) and torch.equal(one[1], counts[s:s + 1]) and torch.equal(one[2], accept[2 * s:2 * s + 2])


@pytest.mark.parametrize("name", ["bf16", "f32"])
def test_borders_of_the_random_numbers(name):
    """0, the smallest and the largest number below 1; drafts from the target's own distribution always stand; a draft that the target rules out never does."""
    rng = np.random.default_rng(1)
    V, n = 300, 6
    logits = torch.from_numpy(rng.standard_normal((n + 1, V)) * 4).to(TYPES[name]).cuda()
    logits[:, 17] = -float("inf")
    ids = rng.integers(18, V, n)
    one = np.float32(1) - np.float32(2.0 ** -24)
    for u in (0.0, 1e-30, float(one)):
        check(name, logits, ids, [0, n + 1], logits[:n].contiguous(), [1.0], [u] * n, [u])
        check(name, logits, ids, [0, n + 1], None, [1.0], [u] * n, [u])
        got = check(name, logits, [17] * n, [0, n + 1], None, [1.0], [u] * n, [u])
        assert got[1].tolist() == [1]
    got = check(name, logits, ids, [0, n + 1], logits[:n].contiguous(), [1.0], [float(one)] * n, [0.5])
    assert got[1].tolist() == [n + 1]


@pytest.mark.parametrize("name", ["bf16", "f32"])
def test_logits_that_are_not_finite_and_odd_temperatures(name):
    rng = np.random.default_rng(2)
    V, drafts = 9000, [2] * 8
    cu = np.concatenate([[0], np.cumsum(np.array(drafts) + 1)])
    logits = torch.from_numpy(rng.standard_normal((cu[-1], V)) * 2).to(TYPES[name]).cuda()
    near = (logits[torch.tensor([i + i // 2 for i in range(16)])].float() + 0.3).to(TYPES[name])
    nan, inf = float("nan"), float("inf")
    logits[0, 8500] = nan
    logits[0, 8700] = nan
    logits[3, 4] = inf
    logits[4, :] = -inf
    logits[6, 100:] = -inf
    near[4, 8200] = nan
    near[5, 8300] = inf
    near[6, :] = -inf
    logits[15, 7] = logits[15, 8900] = 50.0
    ids = rng.integers(0, 100, 16)
    ids[0], ids[2], ids[4], ids[10] = 8500, 4, 8200, 7
    temps = [1.0, 1.0, 0.8, 1.0, inf, nan, -1.0, 1e-40]
    for _ in range(4):
        check(name, logits, ids, cu, near, temps, rng.random(16), rng.random(8))
        check(name, logits, ids, cu, None, temps, rng.random(16), rng.random(8))


def test_ids_outside_the_vocabulary_and_sequences_without_rows():
    rng = np.random.default_rng(3)
    V = 100
    logits = torch.from_numpy(rng.standard_normal((9, V))).to(torch.bfloat16).cuda()
    near = torch.from_numpy(rng.standard_normal((6, V))).to(torch.bfloat16).cuda()
    cu = [0, 0, 3, 3, 7, 8, 8]
    for ids in ([1, 2, 3, 4, 5, 6], [-1, 2, 3, V, 5, 6], [1, -2 ** 31, 2 ** 31 - 1, 4, 5, 6]):
        for d in (None, near):
            for _ in range(3):
                check("bf16", logits, np.array(ids), cu, d, [0.9] * 6, rng.random(6), rng.random(6))
    assert kernels_for("bf16").verify(logits, ints(np.zeros(0)), ints([0]))[1].shape == (0,)
    # Sequences that the arrays do not hold: no tokens.
    for cu in ([0, 3, 10], [-1, 3], [0, 2 ** 31 - 1, -2 ** 31], [5, 2], [0, 9]):
        counts = kernels_for("bf16").verify(logits, ints([1, 2, 3]), ints(cu))[1].tolist()
        assert counts == {(0, 3, 10): [counts[0], 0]}.get(tuple(cu), [0] * (len(cu) - 1)) and 0 <= counts[0] <= 3


def test_refusals():
    k = kernels_for("bf16")
    logits = torch.zeros(3, 50, dtype=torch.bfloat16, device="cuda")
    ids, cu, temps, u, w = ints([1, 2]), ints([0, 3]), floats([1.0]), floats([0.1, 0.2]), floats([0.3])
    k.verify(logits, ids, cu, temps=temps, accept_uniforms=u, draw_uniforms=w)
    for args, kw in (((logits.float(), ids, cu), {}), ((logits[:, ::2], ids, cu), {}), ((logits[0], ids, cu), {}), ((logits, ids.long(), cu), {}), ((logits, ids, cu.cpu()), {}),
                     ((logits, ids, cu[:0]), {}), ((logits, ids, cu), dict(draft_logits=logits)), ((logits, ids, cu), dict(draft_logits=logits[:2, :40].contiguous())),
                     ((logits, ids, cu), dict(temps=temps)), ((logits, ids, cu), dict(temps=temps, accept_uniforms=u)),
                     ((logits, ids, cu), dict(temps=u, accept_uniforms=u, draw_uniforms=w)), ((logits, ids, cu), dict(temps=temps, accept_uniforms=w, draw_uniforms=w)),
                     ((logits, ids, cu), dict(temps=temps, accept_uniforms=u, draw_uniforms=u))):
        with pytest.raises(KernelError):
            k.verify(*args, **kw)


# -------------------------------------------------------------------------------------------- a step as a whole
class Step:
    """Two attention layers' caches and a head, a step's buffers, and the calls of a step in their order."""

    def __init__(self, name, seed, drafts=3):
        self.name, self.k, self.dtype = name, kernels_for(name), TYPES[name]
        self.nq, self.nkv, self.d, self.P, self.V, self.n = 4, 2, 64, 16, 700, drafts
        g = torch.Generator().manual_seed(seed)
        rnd = lambda *s: torch.randn(*s, generator=g).to(self.dtype).cuda()   # noqa: E731
        self.S, self.width = 3, (self.nq + 2 * self.nkv) * self.d
        self.T = self.S * (drafts + 1)
        self.caches = [self.k.empty_cache8(40, self.nkv, self.P, self.d) for _ in range(2)]
        self.table = ints(np.random.default_rng(seed).permutation(39).reshape(3, 13))
        self.w = [rnd(self.width, 128) / 4 for _ in range(2)]
        self.wo = [rnd(128, self.nq * self.d) / 8 for _ in range(2)]
        self.head, self.emb = rnd(self.V, 128), rnd(self.V, 128)
        angle = torch.arange(208, dtype=torch.float64)[:, None] * 1e4 ** (-torch.arange(32, dtype=torch.float64) / 32)
        self.cos, self.sin = torch.cos(angle).to(self.dtype).cuda(), torch.sin(angle).to(self.dtype).cuda()
        self.norm = torch.ones(self.d, dtype=self.dtype, device="cuda")
        self.cu = ints([i * (drafts + 1) for i in range(self.S + 1)])
        self.items = ints([(s, 0) for s in range(self.S)])
        self.ids, self.k_len = ints(np.zeros(self.T)), ints(np.zeros(self.S))
        self.drafts, self.temps = ints(np.zeros(self.S * drafts)), floats([0.0, 0.8, 1.1])
        self.u, self.w_draw = floats(np.zeros(self.S * drafts)), floats(np.zeros(self.S))

    def forward(self):
        k, x = self.k, self.k.embedding(self.emb, self.ids)
        for (kc, vc, sc), w, wo in zip(self.caches, self.w, self.wo):
            q = k.qkv_post8(k.gemm(x, w), nq=self.nq, nkv=self.nkv, d=self.d, k_cache=kc, v_cache=vc, scales=sc, q_w=self.norm, k_w=self.norm, eps=1e-6, cos=self.cos,
                            sin=self.sin, block_table=self.table, cu_q=self.cu, k_len=self.k_len, max_k_len=208)
            o = k.paged_attention8(q, kc, vc, sc, self.table, self.cu, self.k_len, self.items, item_rows=self.n + 1, scale=0.125, max_k_len=208)
            x = k.gemm(o.view(self.T, -1), wo)
        logits = k.gemm(x, self.head)
        return (logits, *k.verify(logits, self.drafts, self.cu, temps=self.temps, accept_uniforms=self.u, draw_uniforms=self.w_draw))

    def set(self, state, rng):
        """The next step's inputs: the last token of each sequence and drafted ones, at the sequence's length."""
        ids = np.stack([np.concatenate([[last], rng.integers(0, self.V, self.n)]) for last, _ in state])
        self.ids.copy_(ints(ids.reshape(-1)))
        self.drafts.copy_(ints(ids[:, 1:].reshape(-1)))
        self.k_len.copy_(ints([length + self.n + 1 for _, length in state]))
        self.u.copy_(floats(rng.random(self.u.numel()) * 0.002))
        self.w_draw.copy_(floats(rng.random(self.S)))

    @staticmethod
    def next(state, tokens, counts):
        """Rejected places are written again by the next step."""
        rows = tokens.cpu().numpy().reshape(len(state), -1)
        return [(int(rows[s, c - 1]), length + c) for s, ((_, length), c) in enumerate(zip(state, counts.tolist()))]


@pytest.mark.parametrize("name", ["bf16", "f32"])
def test_steps_with_drafted_tokens_are_the_formulas(name):
    """Six steps, their caches by the formula from the very rows that the kernels are given, their rejected places written again."""
    m, rng = Step(name, 5), np.random.default_rng(6)
    state = [(1, 0), (2, 0), (3, 0)]
    mirror = [[host(t) for t in c] for c in m.caches]
    for _ in range(6):
        m.set(state, rng)
        k_len, cu, table = m.k_len.tolist(), m.cu.tolist(), m.table.cpu().numpy()
        x = m.k.embedding(m.emb, m.ids)
        for layer in range(2):
            qkv = m.k.gemm(x, m.w[layer])
            kc, vc, sc = m.caches[layer]
            q = m.k.qkv_post8(qkv, nq=m.nq, nkv=m.nkv, d=m.d, k_cache=kc, v_cache=vc, scales=sc, q_w=m.norm, k_w=m.norm, eps=1e-6, cos=m.cos, sin=m.sin,
                              block_table=m.table, cu_q=m.cu, k_len=m.k_len, max_k_len=208)
            store(host(qkv), m.nq, m.nkv, m.d, *mirror[layer], host(m.norm), host(m.norm), 1e-6, host(m.cos), host(m.sin), table, cu, k_len)
            for a, b in zip(m.caches[layer], mirror[layer]):
                assert np.array_equal(host(a), b)
            o = m.k.paged_attention8(q, kc, vc, sc, m.table, m.cu, m.k_len, m.items, item_rows=m.n + 1, scale=0.125, max_k_len=208)
            want = attention(host(q), *mirror[layer], table, cu, k_len, 0.125)[0]
            assert np.abs(host(o) - want).max() <= (2.0 ** -7 if name == "bf16" else 2.0 ** -18) * np.abs(want).max()
            x = m.k.gemm(o.view(m.T, -1), m.wo[layer])
        logits = m.k.gemm(x, m.head)
        _, tokens, counts, _ = (logits, *m.k.verify(logits, m.drafts, m.cu, temps=m.temps, accept_uniforms=m.u, draw_uniforms=m.w_draw))
        want = verify(host(logits), m.drafts.cpu().numpy(), cu, None, host(m.temps), host(m.u), host(m.w_draw))
        assert tokens.tolist() == want[0].tolist() and counts.tolist() == want[1].tolist()
        state = m.next(state, tokens, counts)


@pytest.mark.parametrize("name", ["bf16", "f32"])
def test_a_recorded_step_is_the_step(name):
    """Captured once, replayed for six steps with eager work in between, each replay against the eager step; on a stream of its own."""
    eager, m = Step(name, 7), Step(name, 7)
    other = Step(name, 8)
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        m.set([(1, 0), (2, 0), (3, 0)], np.random.default_rng(1))
        m.forward()
    torch.cuda.current_stream().wait_stream(stream)
    graph, twin = torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = m.forward()
    with torch.cuda.graph(twin, pool=graph.pool()):
        m.forward()
    for c in m.caches:
        for t in c:
            t.zero_()
    rngs = np.random.default_rng(9), np.random.default_rng(9)
    states = [[(1, 0), (2, 0), (3, 0)] for _ in range(2)]
    for step in range(6):
        eager.set(states[0], rngs[0])
        want = eager.forward()
        states[0] = eager.next(states[0], want[1], want[2])
        m.set(states[1], rngs[1])
        graph.replay()
        other.set(states[0], np.random.default_rng(step))
        other.forward()
        for a, b in zip(out, want):
            assert torch.equal(a, b)
        twin.replay()                                           # the other recording shares its memory with the first, and appends what is there
        graph.replay()
        for a, b in zip(out, want):
            assert torch.equal(a, b)
        for c, e in zip(m.caches, eager.caches):
            for a, b in zip(c, e):
                assert np.array_equal(host(a), host(b))
        states[1] = m.next(states[1], out[1], out[2])
        torch.cuda.synchronize()


@pytest.mark.parametrize("drawn", (False, True))
def test_a_sequence_beside_one_that_the_arrays_do_not_hold(drawn):
    """Its tokens, count and chances are those of the definition, whatever the next one's rows are said to be."""
    k, V, rng = kernels_for("bf16"), 100, np.random.default_rng(31)
    logits = torch.from_numpy(rng.standard_normal((9, V)) * 3).to(torch.bfloat16).cuda()
    near = torch.from_numpy(rng.standard_normal((3, V))).to(torch.bfloat16).cuda() if drawn else None
    seen = set()
    for again in range(12):
        ids, u, w = rng.integers(0, V, 3), rng.random(3).astype(np.float32) * 0.02, rng.random(2).astype(np.float32)
        want = verify(host(logits)[:3], ids[:2], [0, 3], host(near[:2]) if drawn else None, [float(np.float32(0.9))], u[:2].astype(np.float64), w[:1].astype(np.float64))
        for cu in ([0, 3, 10], [0, 3, 2], [0, 3, 2 ** 31 - 1], [0, 3, -1]):
            tokens, counts, accept = k.verify(logits, ints(ids), ints(cu), draft_logits=near, temps=floats([0.9, 0.9]), accept_uniforms=floats(u), draw_uniforms=floats(w))
            assert tokens[:3].tolist() == want[0].tolist() and counts.tolist() == [want[1][0], 0]
            assert (np.abs(accept[:2].cpu().numpy() - want[2]) <= 2.0 ** -24 * want[2] + 1e-12).all()
        seen.add(int(want[1][0]))
    assert len(seen) > 1


def test_a_batch_whose_sequences_have_no_rows():
    """No logits at all: no tokens, and no error."""
    k = kernels_for("bf16")
    tokens, counts, accept = k.verify(torch.zeros(0, 700, dtype=torch.bfloat16, device="cuda"), ints(np.zeros(0)), ints([0, 0, 0]))
    assert tokens.shape == (0,) and accept.shape == (0,) and counts.tolist() == [0, 0]
