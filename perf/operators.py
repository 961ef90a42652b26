"""Serving from a cache of 8-bit keys and values, with several drafted tokens a step: the three operators of such a step, and what they are
measured on.

``store8``: what happens to the projections' rows in front of attention (head norm, rotation) with the append of keys and values to pages of
8-bit entries, a power-of-two scale a page and head.  ``attend8``: attention of a step's rows (one token, a few drafted ones, a prompt) over
such pages.  ``verify``: which drafted tokens stand against the target's probabilities, and the token that follows them, from given random
numbers.

A case is one call; heads, head sizes, pages and vocabularies are those of the Qwen3 shapes and of this repository's tests.
"""
from __future__ import annotations

import math

import numpy as np
import torch

own = False

F32, F64, E4M3 = torch.float32, torch.float64, torch.float8_e4m3fn
LOWEST = -64            # a page's scale is 2^LOWEST at least


# -------------------------------------------------------------------------------------------------- the cases
def store(name, dtype, seqs, rows, held, nq, nkv, d, page, ragged=False, norm=True, rot=1.0):
    """seqs sequences bring `rows` tokens each on top of `held` cached ones (ragged: down to a quarter of both)."""
    return {"name": name, "op": "store8", "dtype": dtype, "seqs": seqs, "rows": rows, "held": held, "ragged": ragged, "nq": nq, "nkv": nkv, "d": d,
            "page": page, "norm": norm, "rot": rot}


def attend(name, dtype, seqs, rows, held, nq, nkv, d, page, ragged=False, window=0):
    """The same, its rows looking at all keys or at the last `window`."""
    return {"name": name, "op": "attend8", "dtype": dtype, "seqs": seqs, "rows": rows, "held": held, "ragged": ragged, "nq": nq, "nkv": nkv, "d": d,
            "page": page, "window": window}


def check(name, dtype, seqs, drafts, vocab, ragged=False, drafted="logits"):
    """`drafts` tokens a sequence (ragged: 0 to that many), drawn by a draft model whose logits are at hand or looked up in the text so far."""
    return {"name": name, "op": "verify", "dtype": dtype, "seqs": seqs, "drafts": drafts, "vocab": vocab, "ragged": ragged, "drafted": drafted}


def listed():
    return [
        # A decoding step of a full batch: one row a sequence, in the middle of its page.
        store("store a token each", "bfloat16", 64, 1, 2047, 32, 8, 128, 64),
        # A prompt into an empty cache.
        store("store a prompt", "bfloat16", 1, 4096, 0, 32, 8, 128, 64),
        # Portions of prompts that begin and end inside pages, pages of 16, the 32-bit build.
        store("store portions float32", "float32", 7, 333, 45, 16, 8, 64, 16, ragged=True),
        # One short request: latency.
        attend("attend one token", "bfloat16", 1, 1, 332, 16, 8, 128, 64),
        # A full batch at long contexts: the cache's bytes.
        attend("attend a token each", "bfloat16", 64, 1, 8191, 32, 8, 128, 64),
        # Drafted tokens of a few requests of unequal lengths, the largest group of heads a key head has.
        attend("attend drafts", "bfloat16", 13, 5, 4091, 64, 8, 128, 64, ragged=True),
        # A prompt over its own keys: matrix products.
        attend("attend a prompt", "bfloat16", 1, 4096, 0, 32, 8, 128, 64),
        # Portions of prompts on cached contexts, five heads a key head, a window, pages of 16.
        attend("attend portions window", "bfloat16", 5, 700, 1301, 40, 8, 128, 16, ragged=True, window=1024),
        # The 32-bit build, as it is used to check the other.
        attend("attend drafts float32", "float32", 3, 4, 1500, 16, 8, 64, 32, ragged=True),
        # One request's four drafted tokens over the whole vocabulary: latency.
        check("verify one", "bfloat16", 1, 4, 151936),
        # A full batch's.
        check("verify a batch", "bfloat16", 64, 4, 151936),
        # Tokens looked up in the text, unequal numbers of them, an odd vocabulary.
        check("verify lookups float32", "float32", 24, 7, 32771, ragged=True, drafted="lookup"),
    ]


def spread(rng, lo, hi):
    return max(lo, min(hi, round(math.exp(rng.uniform(math.log(lo), math.log(hi + 0.49))))))


def draw(rng):
    """One more case: 1 to 64 sequences; contexts to 8,192 keys, prompts to 4,096 tokens in all; heads of 16 to 256, groups of 1 to 8, pages of 16 to
    128; 0 to 8 drafted tokens, vocabularies of 256 to 151,936."""
    op = rng.choice(["store8", "attend8", "attend8", "verify"])
    dtype = "float32" if rng.random() < 0.25 else "bfloat16"
    ragged = rng.random() < 0.6
    if op == "verify":
        seqs = spread(rng, 1, 64 if dtype == "bfloat16" else 32)
        c = check("", dtype, seqs, rng.randrange(0, 9) if ragged else rng.randrange(1, 6), spread(rng, 256, 151936), ragged, rng.choice(["logits", "lookup"]))
        while c["seqs"] * (c["drafts"] + 1) > 320:
            c["seqs"] //= 2
        del c["name"]
        return c
    nkv, group, d = rng.choice([1, 2, 4, 8]), rng.choice([1, 2, 3, 4, 5, 8]), rng.choice([16, 32, 64, 80, 96, 128, 128, 128, 192, 256])
    page = rng.choice([16, 32, 64, 64, 128])
    kind = rng.choice(["decode", "drafts", "prompt"])
    if kind == "prompt":
        total = spread(rng, 17, 4096)
        seqs = spread(rng, 1, min(8, total // 17))
        rows = max(17, total // seqs)
        held = rng.choice([0, spread(rng, 1, 2048)])
        if dtype == "float32":
            rows, held = min(rows, 1024), min(held, 1024)
    else:
        seqs = spread(rng, 1, 64)
        rows = 1 if kind == "decode" else rng.randrange(2, 10)
        held = spread(rng, 1, 8000)
        if dtype == "float32" or d > 128:
            held, seqs = min(held, 2000), min(seqs, 32)
    if op == "store8":
        c = store("", dtype, seqs, rows, held, nkv * group, nkv, d, page, ragged, rng.random() < 0.7, rng.choice([0.0, 0.5, 1.0, 1.0]))
    else:
        c = attend("", dtype, seqs, rows, held, nkv * group, nkv, d, page, ragged, rng.choice([0, 0, spread(rng, 1, 2048)]))
        while c["seqs"] > 1 and c["seqs"] * c["rows"] * (c["rows"] + c["held"]) * c["nq"] > 500e6:
            c["seqs"] -= 1
    del c["name"]
    return c


def lengths(c):
    """(new rows, keys with them) of each sequence."""
    n, out = c["seqs"], []
    for i in range(n):
        part = (lambda v: v - (i * v * 3) // (4 * n)) if c["ragged"] else (lambda v: v)
        rows = max(1, part(c["rows"]))
        out.append((rows, rows + part(c["held"])))
    return out


def draft_counts(c):
    n = c["seqs"]
    return [c["drafts"] - (i * (c["drafts"] + 1)) // n if c["ragged"] else c["drafts"] for i in range(n)]


def element(c):
    return getattr(torch, c["dtype"])


# --------------------------------------------------------------------------------------- what a program has in hand
def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return (prepare_verify if case["op"] == "verify" else prepare_cache)(case, g)


def prepare_cache(c, g):
    """The step's rows, the pages as earlier steps left them (in any order in the cache), and where everything is.  Entries are near normal; a page's
    scale is what entries of normal size need, give or take a power of two, so that some pages' grow."""
    dtype, S, P, nq, nkv, d = element(c), c["seqs"], c["page"], c["nq"], c["nkv"], c["d"]
    both = lengths(c)
    rows, keys = [r for r, _ in both], [k for _, k in both]
    W = -(-max(keys) // P)
    used = [-(-k // P) for k in keys]
    order = torch.randperm(sum(used), device="cuda", generator=g).to(torch.int32)
    table = torch.zeros(S, W, dtype=torch.int32, device="cuda")
    at = 0
    for s, n in enumerate(used):
        table[s, :n] = order[at:at + n]
        at += n

    def entries(shape):
        x = torch.randn(shape, dtype=torch.bfloat16, device="cuda", generator=g)
        return x.mul_(64).clamp_(-448, 448).to(E4M3)
    scales = two_to(torch.randint(-8, -5, (at, nkv, 2), device="cuda", generator=g)).to(F32)
    s = {"case": c, "k": entries((at, nkv, P, d)), "v": entries((at, nkv, d, P)), "scales": scales, "table": table,
         "cu": torch.tensor(np.concatenate([[0], np.cumsum(rows)]), dtype=torch.int32, device="cuda"),
         "k_len": torch.tensor(keys, dtype=torch.int32, device="cuda"), "max_k_len": max(keys), "max_rows": max(rows)}
    T = sum(rows)
    if c["op"] == "attend8":
        s["q"] = (torch.randn(T, nq, d, device="cuda", generator=g) * 1.5).to(dtype)
        most = 128 if max(rows) > 16 else max(rows)        # rows of an item
        items = [(i, a) for i, r in enumerate(rows) for a in range(0, r, most)]
        s["items"], s["item_rows"] = torch.tensor(items, dtype=torch.int32, device="cuda"), most
        return s
    s["qkv"] = torch.randn(T, (nq + 2 * nkv) * d, device="cuda", generator=g).to(dtype)
    s["q_w"] = s["k_w"] = s["cos"] = s["sin"] = None
    if c["norm"]:
        s["q_w"], s["k_w"] = ((0.8 + 0.4 * torch.rand(d, device="cuda", generator=g)).to(dtype) for _ in range(2))
    half = int(c["rot"] * d) // 2
    if half:
        angle = torch.arange(max(keys), device="cuda", dtype=F64)[:, None] * 1e6 ** (-torch.arange(half, device="cuda", dtype=F64) / half)
        s["cos"], s["sin"] = torch.cos(angle).to(dtype), torch.sin(angle).to(dtype)
    # The pages that the step writes to, for the plain form.
    touched = [(i, j) for i, (r, k) in enumerate(both) for j in range((k - r) // P, (k - 1) // P + 1)]
    at = torch.tensor(touched, device="cuda")
    s["touched"] = table[at[:, 0], at[:, 1]].long()
    return s


def prepare_verify(c, g):
    """Logits of a model that is fairly sure of a few tokens, a draft model's that are near them, and tokens drawn from the latter (or some of the
    likely ones, looked up).  A fifth of the sequences is greedy."""
    dtype, S, V = element(c), c["seqs"], c["vocab"]
    counts = draft_counts(c)
    D, R = sum(counts), sum(counts) + S
    logits = torch.randn(R, V, device="cuda", generator=g).mul_(2.0)
    likely = torch.randint(0, V, (R, 4), device="cuda", generator=g)
    logits.scatter_add_(1, likely, 12.0 + 3.0 * torch.randn(R, 4, device="cuda", generator=g))
    cu = np.concatenate([[0], np.cumsum(np.array(counts) + 1)])
    of = np.repeat(np.arange(S), counts)                                    # sequence of each draft
    temps = torch.where(torch.rand(S, device="cuda", generator=g) < 0.2, 0.0, 0.6 + 0.6 * torch.rand(S, device="cuda", generator=g))
    s = {"case": c, "logits": logits.to(dtype), "cu": torch.tensor(cu, dtype=torch.int32, device="cuda"), "temps": temps, "most": max(counts),
         "accept_u": torch.rand(D, device="cuda", generator=g), "draw_u": torch.rand(S, device="cuda", generator=g), "draft_logits": None}
    rows = torch.tensor(np.arange(D) + of, dtype=torch.long, device="cuda")  # row of the target's logits of each draft
    if c["drafted"] == "logits":
        draft = logits[rows].add_(torch.randn(D, V, device="cuda", generator=g).mul_(0.7)).to(dtype)
        t = temps[torch.tensor(of, dtype=torch.long, device="cuda")].clamp(min=1e-3)[:, None]
        noise = -torch.log(-torch.log(torch.rand(D, V, device="cuda", generator=g).clamp(1e-12, 1 - 1e-7)))
        s["draft_ids"] = (draft.float() / t + noise).argmax(1).to(torch.int32) if D else torch.zeros(0, dtype=torch.int32, device="cuda")
        s["draft_logits"] = draft
    else:
        which = torch.randint(0, 4, (D, 1), device="cuda", generator=g)
        s["draft_ids"] = likely[rows].gather(1, which)[:, 0].to(torch.int32)
    return s


# ------------------------------------------------------------------------------------------------------ one pass
def run(s):
    if own:
        return run_own(s)
    return {"store8": plain_store, "attend8": plain_attend, "verify": plain_verify}[s["case"]["op"]](s)


def run_own(s):
    from vosti_amd.kernels import kernels_for
    c = s["case"]
    k = kernels_for(c["dtype"])
    if c["op"] == "store8":
        q = k.qkv_post8(s["qkv"], nq=c["nq"], nkv=c["nkv"], d=c["d"], k_cache=s["k"], v_cache=s["v"], scales=s["scales"], q_w=s["q_w"], k_w=s["k_w"], eps=1e-6,
                        cos=s["cos"], sin=s["sin"], block_table=s["table"], cu_q=s["cu"], k_len=s["k_len"], max_k_len=s["max_k_len"])
        return {"q": q, "k": s["k"], "v": s["v"], "scales": s["scales"]}
    if c["op"] == "attend8":
        return k.paged_attention8(s["q"], s["k"], s["v"], s["scales"], s["table"], s["cu"], s["k_len"], s["items"], item_rows=s["item_rows"], scale=c["d"] ** -0.5,
                                  window=c["window"], max_k_len=s["max_k_len"])
    tokens, counts, accept = k.verify(s["logits"], s["draft_ids"], s["cu"], draft_logits=s["draft_logits"], temps=s["temps"], accept_uniforms=s["accept_u"],
                                      draw_uniforms=s["draw_u"])
    return {"tokens": tokens, "counts": counts, "accept": accept}


def places(s, T):
    """Sequence and place in it of each of the step's rows."""
    t = torch.arange(T, device="cuda")
    cu = s["cu"].long()
    seq = torch.bucketize(t, cu[1:], right=True)
    return seq, s["k_len"].long()[seq] - cu[seq + 1] + t


def two_to(e):
    """2^e, to the bit."""
    return ((e.long() + 1023) << 52).view(F64)


def least_exponent(x):
    """The least e with |x| <= 448 * 2^e, entry by entry."""
    m, e = torch.frexp(x)
    return torch.where(x == 0, LOWEST, e - 9 + (m.abs() > 0.875).int()).clamp(min=LOWEST)


def to_e4m3(x):
    """64-bit numbers of at most 448 to the nearest e4m3 value, ties to the even one: four binary digits, steps of 2^-9 at least."""
    e = torch.frexp(x)[1].clamp(min=-5) - 4
    return (torch.round(x * two_to(-e)) * two_to(e)).to(E4M3)


def plain_store(s):
    """In 64 bits: an entry next to the border between two e4m3 values goes to the one that its formula says."""
    c = s["case"]
    T, nq, nkv, d, P = len(s["qkv"]), c["nq"], c["nkv"], c["d"], c["page"]
    x = s["qkv"].view(T, nq + 2 * nkv, d).to(F64)
    q, k, v = x[:, :nq], x[:, nq:nq + nkv], x[:, nq + nkv:]
    seq, place = places(s, T)

    def normed(x, w):
        return x * torch.rsqrt((x * x).mean(-1, keepdim=True) + 1e-6) * w.to(F64)

    def turned(x):
        h = s["cos"].shape[1]
        cos, sin = (t[place].to(F64)[:, None] for t in (s["cos"], s["sin"]))
        a, b = x[..., :h], x[..., h:2 * h]
        return torch.cat([a * cos - b * sin, b * cos + a * sin, x[..., 2 * h:]], -1)
    if s["q_w"] is not None:
        q, k = normed(q, s["q_w"]), normed(k, s["k_w"])
    if s["cos"] is not None:
        q, k = turned(q), turned(k)
    new = torch.stack([k, v], 2)                                               # [T, nkv, 2, d]
    page, off = s["table"].long()[seq, place // P], place % P
    old = torch.frexp(s["scales"])[1] - 1                                      # exponents [pages, nkv, 2]
    fresh = old.new_zeros(len(old)).scatter_reduce(0, page, (off == 0).to(old.dtype), "amax")   # pages that begin with this step
    kept = torch.where(fresh[:, None, None] > 0, LOWEST, old)
    need = least_exponent(new.abs().amax(-1))
    now = kept.scatter_reduce(0, page[:, None, None].expand_as(need), need.to(kept.dtype), "amax")
    s["scales"].copy_(two_to(now))
    at = s["touched"]
    down = (old - now)[at].clamp(max=0)
    kb, vb = s["k"].view(torch.uint8), s["v"].view(torch.uint8)                # the same bytes, for indexing
    kb[at] = to_e4m3(s["k"][at].to(F64) * two_to(down[:, :, 0, None, None])).view(torch.uint8)
    vb[at] = to_e4m3(s["v"][at].to(F64) * two_to(down[:, :, 1, None, None])).view(torch.uint8)
    held = to_e4m3(new * two_to(-now[page][..., None])).view(torch.uint8)
    kb[page, :, off] = held[:, :, 0]
    vb[page, :, :, off] = held[:, :, 1]
    return {"q": q.to(element(c)), "k": s["k"], "v": s["v"], "scales": s["scales"]}


def plain_attend(s):
    """All sequences at once, their rows and keys filled up to the longest one's."""
    c = s["case"]
    S, T, nq, nkv, d, P, R = c["seqs"], len(s["q"]), c["nq"], c["nkv"], c["d"], c["page"], s["max_rows"]
    table = s["table"].long()
    W = table.shape[1]
    scales = s["scales"][table]
    k = s["k"].view(torch.uint8)[table].view(E4M3).to(F32) * scales[..., 0, None, None]
    v = s["v"].view(torch.uint8)[table].view(E4M3).to(F32) * scales[..., 1, None, None]
    k = k.transpose(1, 2).reshape(S, nkv, W * P, d)
    v = v.permute(0, 2, 1, 4, 3).reshape(S, nkv, W * P, d)
    cu, k_len = s["cu"].long(), s["k_len"].long()
    row = torch.arange(R, device="cuda")
    q = s["q"].to(F32)[(cu[:-1, None] + row).clamp(max=T - 1)]                 # [S, R, nq, d]
    q = q.view(S, R, nkv, nq // nkv, d).permute(0, 2, 3, 1, 4).reshape(S, nkv, -1, d)
    scores = torch.matmul(q, k.transpose(2, 3)).mul_(d ** -0.5).view(S, nkv, nq // nkv, R, W * P)
    pos = (k_len - (cu[1:] - cu[:-1]))[:, None] + row                          # [S, R]
    key = torch.arange(W * P, device="cuda")
    hidden = key > pos[..., None]
    if c["window"]:
        hidden |= key <= pos[..., None] - c["window"]
    scores.masked_fill_(hidden[:, None, None], -math.inf)
    scores.sub_(scores.amax(-1, keepdim=True)).exp_()
    total = scores.sum(-1, keepdim=True)
    out = torch.matmul(scores.view(S, nkv, -1, W * P), v).view(S, nkv, nq // nkv, R, d) / total
    out = out.permute(0, 3, 1, 2, 4).reshape(S * R, nq, d)
    t = torch.arange(T, device="cuda")
    seq = torch.bucketize(t, cu[1:], right=True)
    return out[seq * R + t - cu[seq]].to(element(c))


def plain_verify(s):
    """In 64 bits: a token is the one in whose share of the line the random number lies."""
    R, V = s["logits"].shape
    S, D = len(s["temps"]), len(s["draft_ids"])
    cu, ids = s["cu"].long(), s["draft_ids"].long()
    first = cu - torch.arange(S + 1, device="cuda")                            # first draft of each sequence
    of_row = torch.bucketize(torch.arange(R, device="cuda"), cu[1:], right=True)
    of_draft = torch.bucketize(torch.arange(D, device="cuda"), first[1:], right=True)
    column = torch.arange(V, device="cuda")

    def chances(logits, of):
        x, t = logits.to(F64), s["temps"].to(F64)[of][:, None]
        top = x.amax(1, keepdim=True)
        best = torch.where(x == top, column, V).amin(1, keepdim=True)
        p = torch.exp((x - top) / torch.where(t > 0, t, 1.0))
        return torch.where(t > 0, p / p.sum(1, keepdim=True), (column == best).to(F64))
    p = chances(s["logits"], of_row)
    q = chances(s["draft_logits"], of_draft) if s["draft_logits"] is not None else (column == ids[:, None]).to(F64)
    n = torch.arange(D, device="cuda")
    pd, qd = p[n + of_draft, ids], q[n, ids]
    stands = torch.zeros(S, s["most"] + 1, dtype=torch.bool, device="cuda")
    stands[of_draft, n - first[of_draft]] = s["accept_u"].to(F64) * qd < pd
    accepted = stands.int().cumprod(1).sum(1)
    row = cu[:-1] + accepted
    weights = p[row]
    if D:
        less = (weights - q[(first[:-1] + accepted).clamp(max=D - 1)]).clamp(min=0)
        refused = (accepted < first[1:] - first[:-1]) & (less.sum(1) > 0)
        weights = torch.where(refused[:, None], less, weights)
    line = weights.cumsum(1)
    target = s["draw_u"].to(F64)[:, None] * line[:, -1:]
    last = torch.where(weights > 0, column, 0).amax(1)
    drawn = torch.minimum((line <= target).sum(1), last)
    place = torch.arange(R, device="cuda") - cu[of_row]
    draft = torch.cat([ids, ids.new_zeros(1)])[(torch.arange(R, device="cuda") - of_row).clamp(max=D)]
    tokens = torch.where(place < accepted[of_row], draft, torch.where(place == accepted[of_row], drawn[of_row], -1))
    ratio = torch.where(qd > 0, pd / torch.where(qd > 0, qd, 1.0), (pd > 0).to(F64)).clamp(max=1)
    return {"tokens": tokens.int(), "counts": (accepted + 1).int(), "accept": ratio.to(F32)}


# ------------------------------------------------------------------------------------------------- in 64 bits
def exact(case, seed):
    s = prepare(case, seed)
    return {"store8": exact_store, "attend8": exact_attend, "verify": exact_verify}[case["op"]](s)


def exact_store(s):
    """Sequence by sequence and page by page, with a list of the e4m3 numbers."""
    c = s["case"]
    nq, nkv, d, P = c["nq"], c["nkv"], c["d"], c["page"]
    numbers = np.array([m * 2.0 ** -9 for m in range(8)] + [(8 + m) * 2.0 ** (e - 10) for e in range(1, 16) for m in range(8)])[:127]
    middles = (numbers[1:] + numbers[:-1]) / 2

    def nearest(x):
        a = np.abs(x)
        i = np.searchsorted(middles, a, side="left")
        tie = (i < 126) & (a == middles[np.minimum(i, 125)])
        i = i + (tie & (i % 2 == 1))
        return np.copysign(numbers[i], x)
    host = {n: (s[n].to(F64).cpu().numpy() if s[n] is not None else None) for n in ("qkv", "k", "v", "scales", "q_w", "k_w", "cos", "sin")}
    table = s["table"].cpu().numpy()
    x = host["qkv"].reshape(-1, nq + 2 * nkv, d)
    kc, vc, scales = host["k"], host["v"], host["scales"]
    q_out = np.empty((len(x), nq, d))
    t = 0
    for i, (n, keys) in enumerate(lengths(c)):
        mine, at = x[t:t + n], np.arange(keys - n, keys)

        def heads(y, w):
            if w is not None:
                y = y / np.sqrt(np.square(y).sum(-1, keepdims=True) / d + 1e-6) * w
            if host["cos"] is None:
                return y
            cos, sin = host["cos"][at][:, None], host["sin"][at][:, None]
            h, y = cos.shape[-1], y.copy()
            a, b = y[..., :h].copy(), y[..., h:2 * h].copy()
            y[..., :h], y[..., h:2 * h] = a * cos - b * sin, a * sin + b * cos
            return y
        q_out[t:t + n] = heads(mine[:, :nq], host["q_w"])
        new = heads(mine[:, nq:nq + nkv], host["k_w"]), mine[:, nq + nkv:]
        for j in range((keys - n) // P, (keys - 1) // P + 1):
            a, b = max(j * P, keys - n), min((j + 1) * P, keys)
            page, o = table[i, j], a - j * P
            for which, cache in ((0, kc), (1, np.swapaxes(vc, 2, 3))):
                part = new[which][a - keys + n:b - keys + n].transpose(1, 0, 2)          # [nkv, rows, d]
                scale = np.full(nkv, 2.0 ** LOWEST) if o == 0 else scales[page, :, which].copy()
                top = np.abs(part).max((1, 2))
                while (grow := top > 448 * scale).any():
                    scale[grow] *= 2
                cache[page] = nearest(cache[page] * np.minimum(scales[page, :, which] / scale, 1.0)[:, None, None])
                cache[page][:, o:o + b - a] = nearest(part / scale[:, None, None])
                scales[page, :, which] = scale
        t += n
    return {"q": q_out, "k": kc, "v": vc, "scales": scales}


def exact_attend(s):
    """Sequence by sequence and key head by key head."""
    c = s["case"]
    nq, nkv, d, P = c["nq"], c["nkv"], c["d"], c["page"]
    group, out, t = nq // nkv, torch.empty(s["q"].shape, dtype=F64, device="cuda"), 0
    for i, (n, keys) in enumerate(lengths(c)):
        pages = s["table"][i, :-(-keys // P)].tolist()
        j, r = torch.arange(keys, device="cuda"), torch.arange(n, device="cuda")[:, None]
        seen = j <= keys - n + r
        if c["window"]:
            seen &= j > keys - n + r - c["window"]
        for h in range(nkv):
            k = torch.cat([s["k"][p, h].to(F64) * s["scales"][p, h, 0].double() for p in pages])[:keys]
            v = torch.cat([s["v"][p, h].to(F64).T * s["scales"][p, h, 1].double() for p in pages])[:keys]
            for m in range(h * group, (h + 1) * group):
                e = torch.exp(s["q"][t:t + n, m].to(F64) @ k.T / math.sqrt(d)) * seen
                out[t:t + n, m] = e @ v / e.sum(1, keepdim=True)
        t += n
    return out


def exact_verify(s):
    """Sequence by sequence, as the definition says it."""
    c = s["case"]
    host = {n: s[n].to(F64).cpu().numpy() for n in ("logits", "temps", "accept_u", "draw_u")}
    ids, cu = s["draft_ids"].cpu().numpy(), s["cu"].cpu().numpy()
    drafts = s["draft_logits"].to(F64).cpu().numpy() if s["draft_logits"] is not None else None
    V = c["vocab"]

    def chances(x, t):
        if t <= 0:
            y = np.zeros(V)
            y[int(np.argmax(x))] = 1.0
            return y
        y = np.exp(x / t - np.max(x) / t)
        return y / y.sum()
    tokens, counts, accept = np.full(len(host["logits"]), -1, np.int32), np.zeros(c["seqs"], np.int32), np.zeros(len(ids))
    for i in range(c["seqs"]):
        t, going, n = host["temps"][i], True, cu[i + 1] - cu[i] - 1
        for a in range(n + 1):
            r, m = cu[i] + a, cu[i] - i + a
            p = chances(host["logits"][r], t)
            left = p
            if a < n:
                if drafts is not None:
                    q = chances(drafts[m], t)
                else:
                    q = np.zeros(V)
                    q[ids[m]] = 1.0
                x, y = p[ids[m]], q[ids[m]]
                accept[m] = min(1.0, x / y) if y > 0 else float(x > 0)
                if not going:
                    continue
                if host["accept_u"][m] * y < x:
                    tokens[r] = ids[m]
                    continue
                left = np.maximum(p - q, 0)
                if left.sum() == 0:
                    left = p
            if going:
                line = np.cumsum(left)
                tokens[r] = min(int(np.searchsorted(line, host["draw_u"][i] * line[-1], side="right")), int(np.nonzero(left)[0][-1]))
                counts[i], going = a + 1, False
    return {"tokens": tokens, "counts": counts, "accept": accept}


# -------------------------------------------------------------------------------------------------------- its work
def work(c):
    """Each row, entry, scale and logit that the call needs read once, each output written once."""
    e = 4 if c["dtype"] == "float32" else 2
    if c["op"] == "verify":
        D, R, V = sum(draft_counts(c)), sum(draft_counts(c)) + c["seqs"], c["vocab"]
        rows = R + (D if c["drafted"] == "logits" else 0)
        return {"bytes": e * rows * V + 4 * (2 * D + R) + 16 * c["seqs"], "flops": 4 * rows * V}
    nq, nkv, d, P = c["nq"], c["nkv"], c["d"], c["page"]
    both = lengths(c)
    T = sum(r for r, _ in both)
    if c["op"] == "store8":
        pages = sum((k - 1) // P - (k - r) // P + 1 for r, k in both)
        half = int(c["rot"] * d) // 2
        return {"bytes": T * ((2 * nq + 2 * nkv) * d * e + 2 * nkv * d + 2 * half * e) + 16 * nkv * pages, "flops": T * ((nq + nkv) * d * (4 * c["norm"] + 3 * c["rot"]) + 4 * nkv * d)}
    w = c["window"] or 1 << 30
    seen = sum(sum(min(p + 1, w) for p in range(k - r, k)) for r, k in both)
    keys = sum(min(k, r - 1 + w) for r, k in both)
    return {"bytes": 2 * nkv * d * keys + 8 * nkv * -(-keys // P) + 2 * T * nq * d * e, "flops": 4 * nq * d * seen}
