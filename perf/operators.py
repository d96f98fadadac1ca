"""Performance cases of the serving operators: rotary positions, a paged cache with a prefix that requests share, and the
verification of drafted tokens.

``rotate``     ``rope.rotate``: positions put into queries or keys, or taken out of them
``append``     ``paged.append``: a pass's keys and values into the pages of their requests, rotated on the way
``attention``  ``paged.attention``: a pass's queries over the pages of a shared prefix and of their own requests
``verify``     ``verify.verify_tokens``: how many drafted tokens stand, and the token behind them

Head counts, head sizes, frequency bases and vocabularies are those of the presets of the benchmark configurations.  With
``own`` false ``run`` computes the same in elementary torch operations.
"""
import math
import random

import torch

own = False
DEVICE = "cuda"
TYPES = {"fp16": torch.float16, "bf16": torch.bfloat16, "fp32": torch.float32}
SIZE = {"fp16": 2, "bf16": 2, "fp32": 4}
# query heads, key heads, head size, base of the rotation
HEADS = {"0.5b": (14, 2, 64, 1e6), "1b": (32, 8, 64, 5e5), "7b": (28, 4, 128, 1e6), "8b": (32, 8, 128, 5e5), "70b": (64, 8, 128, 5e5)}
VOCABULARIES = (128256, 151936, 152064)
LLAMA3 = dict(rope_type="llama3", factor=8.0, low_freq_factor=1.0, high_freq_factor=4.0, original_max_position_embeddings=8192)


# --------------------------------------------------------------------------------------------------- the cases
def listed():
    return [
        # the queries of one token of a draft-sized model: all latency
        dict(name="rotate 1 token", kind="rotate", tokens=1, heads=14, dim=64, rotary=64, dtype="fp16", interleaved=False, inverse=False,
             scaled=False, far=4096),
        # the queries of a long prompt chunk, half of each head rotated, neighbours paired, frequencies rescaled for far positions
        dict(name="rotate 4099 far", kind="rotate", tokens=4099, heads=32, dim=128, rotary=64, dtype="bf16", interleaved=True,
             inverse=False, scaled=True, far=131072),
        # positions taken out of single-precision rows again (the gradient of a rotation)
        dict(name="rotate 1021 back", kind="rotate", tokens=1021, heads=28, dim=128, rotary=128, dtype="fp32", interleaved=False,
             inverse=True, scaled=False, far=32768),
        # the next token of a few requests
        dict(name="append 16 tokens", kind="append", model="7b", requests=16, rows=1, ragged=False, page=16, own=700, prefix=1000,
             dtype="fp16", scaled=False, interleaved=False),
        # prompts of several requests in one pass, none as long as another
        dict(name="append ragged prompts", kind="append", model="8b", requests=12, rows=1200, ragged=True, page=64, own=1500, prefix=8192,
             dtype="bf16", scaled=True, interleaved=False),
        # the next token of a few requests on a small model behind a short system prompt: latency
        dict(name="attend 4 short", kind="attention", model="0.5b", requests=4, rows=1, ragged=False, page=16, own=60, prefix=200,
             dtype="fp16", tree=False),
        # the next token of many requests behind a long prefix
        dict(name="attend 64 long prefix", kind="attention", model="8b", requests=64, rows=1, ragged=False, page=16, own=1024,
             prefix=16384, dtype="fp16", tree=False),
        # a tree of drafted tokens of each of several requests, groups of seven heads
        dict(name="attend 8 trees", kind="attention", model="7b", requests=8, rows=16, ragged=True, page=32, own=777, prefix=8003,
             dtype="bf16", tree=True),
        # pieces of prompts behind a prefix of a book: many queries, the tensor cores' work
        dict(name="attend prompt pieces", kind="attention", model="8b", requests=16, rows=64, ragged=False, page=64, own=512,
             prefix=32768, dtype="bf16", tree=False),
        # one request, a short draft
        dict(name="verify 1x3", kind="verify", requests=1, drafts=3, vocab=128256, dtype="fp32", drawn=True, ragged=False),
        # a full batch of sampled drafts, not all of one length
        dict(name="verify 64x7", kind="verify", requests=64, drafts=7, vocab=152064, dtype="fp32", drawn=True, ragged=True),
        # drafts that were not drawn (the likeliest token, a lookup), probabilities in 16 bits
        dict(name="verify 16x15 not drawn", kind="verify", requests=16, drafts=15, vocab=151936, dtype="bf16", drawn=False, ragged=False),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["rotate", "append", "attention", "attention", "verify"])
    if kind == "rotate":
        dim = rng.choice([64, 96, 128])
        return dict(kind=kind, tokens=_log(rng, 1, 8192), heads=rng.randint(1, 64), dim=dim, rotary=rng.choice([dim, dim, dim // 2, 24]),
                    dtype=rng.choice(["fp16", "bf16", "fp32"]), interleaved=rng.random() < 0.5, inverse=rng.random() < 0.3,
                    scaled=rng.random() < 0.5, far=_log(rng, 4096, 262144))
    if kind == "append":
        rows = rng.choice([1, _log(rng, 2, 32), _log(rng, 33, 1024)])
        return dict(kind=kind, model=rng.choice(sorted(HEADS)), requests=_log(rng, 1, 64 if rows <= 32 else 8), rows=rows, ragged=rng.random() < 0.5,
                    page=rng.choice([8, 16, 32, 64, 128]), own=rows + _log(rng, 1, 2000), prefix=rng.choice([0, _log(rng, 64, 32768)]),
                    dtype=rng.choice(["fp16", "bf16"]), scaled=rng.random() < 0.5, interleaved=rng.random() < 0.3)
    if kind == "attention":
        rows = rng.choice([1, 1, _log(rng, 2, 32), _log(rng, 33, 128)])
        requests = _log(rng, 1, 64 if rows <= 32 else 8)
        return dict(kind=kind, model=rng.choice(sorted(HEADS)), requests=requests, rows=rows, ragged=rng.random() < 0.5,
                    page=rng.choice([8, 16, 32, 64, 128]), own=rows + _log(rng, 1, 2000), prefix=rng.choice([0, _log(rng, 64, 16384), _log(rng, 64, 16384)]),
                    dtype=rng.choice(["fp16", "bf16"]), tree=1 < rows <= 32 and rng.random() < 0.5)
    return dict(kind=kind, requests=_log(rng, 1, 48), drafts=rng.randint(1, 8), vocab=rng.choice(VOCABULARIES + (_log(rng, 1000, 150000),)),
                dtype=rng.choice(["fp32", "fp32", "fp16", "bf16"]), drawn=rng.random() < 0.7, ragged=rng.random() < 0.5)


# --------------------------------------------------------------------------------------------------- sizes
def _counts(case):
    """New rows of each request, and the rows in its own pages with them: what the case says, or spread between that and little."""
    rng = random.Random(f"{case['requests']} {case['rows']} {case['own']}")
    n, length = [], []
    for _ in range(case["requests"]):
        n.append(rng.randint(1, case["rows"]) if case["ragged"] else case["rows"])
        length.append(n[-1] + rng.randint(0, case["own"] - case["rows"]))
    return n, length


def _drafts(case):
    rng = random.Random(f"{case['requests']} {case['drafts']}")
    return [rng.randint(0, case["drafts"]) if case["ragged"] else case["drafts"] for _ in range(case["requests"])]


def work(case):
    kind = case["kind"]
    if kind == "rotate":
        n = case["tokens"] * case["heads"]
        return {"bytes": 2 * n * case["dim"] * SIZE[case["dtype"]] + 8 * case["tokens"], "flops": 3 * n * case["rotary"]}
    if kind == "verify":
        # Refused drafts: the rows of both distributions at the first; all stand: the target's row behind the last.  Some 0.7 of drawn
        # tokens stand.
        rows = sum(2 - 0.7 ** k for k in _drafts(case)) if case["drawn"] else case["requests"]
        return {"bytes": int(rows * case["vocab"] * SIZE[case["dtype"]]), "flops": int(3 * rows * case["vocab"])}
    hq, hk, dim, _ = HEADS[case["model"]]
    n, length = _counts(case)
    tokens = sum(n)
    if kind == "append":
        return {"bytes": 2 * tokens * (hq + 2 * hk) * dim * 2 + 8 * tokens, "flops": 3 * tokens * (hq + hk) * dim}
    seen = sum(a * (case["prefix"] + b) - a * (a - 1) // 2 for a, b in zip(n, length))
    return {"bytes": 2 * tokens * hq * dim * 2 + 2 * (case["prefix"] + sum(length)) * hk * dim * 2, "flops": 4 * hq * dim * seen}


# --------------------------------------------------------------------------------------------------- inputs
def _frequencies(dim, base, scaled):
    """Rotation frequencies in single precision, rescaled where a model was stretched to longer contexts."""
    f = base ** (-torch.arange(0, dim, 2, dtype=torch.float64) / dim)
    if scaled:
        turns = LLAMA3["original_max_position_embeddings"] * f / (2 * math.pi)
        lo, hi = LLAMA3["low_freq_factor"], LLAMA3["high_freq_factor"]
        smooth = ((turns - lo) / (hi - lo)).clamp(0, 1)
        f = f * (smooth + (1 - smooth) / LLAMA3["factor"])
    return f.float().to(DEVICE)


def _normal(shape, dtype, g):
    return torch.randn(shape, generator=g, device=DEVICE, dtype=TYPES[dtype] if dtype != "fp32" else torch.float32)


def _ints(values, dtype=torch.int32):
    return torch.tensor(values, dtype=dtype, device=DEVICE)


def _starts(n):
    return [sum(n[:i]) for i in range(len(n) + 1)]


def _masks(n, g):
    """Ancestor masks of random trees: word ``i`` has a bit for each of the request's new rows that row ``i`` sees, itself among them."""
    words = []
    rng = random.Random(int(torch.randint(0, 1 << 30, (1,), generator=g, device=DEVICE)))
    for count in n:
        rows = []
        for i in range(count):
            rows.append((rows[rng.randrange(i)] if i else 0) | 1 << i)
        words += rows
    return _ints(words, torch.int64)


def prepare(case, seed):
    g = torch.Generator(device=DEVICE).manual_seed(int(seed))
    kind, dtype = case["kind"], case["dtype"]
    s = dict(case=case)
    if kind == "rotate":
        # rows of a fused projection's result: the queries, keys and values of a token behind one another
        s["x"] = _normal((case["tokens"], case["heads"] + 2, case["dim"]), dtype, g)[:, : case["heads"]]
        first = int(torch.randint(0, max(1, case["far"] - case["tokens"]), (1,), generator=g, device=DEVICE))
        s["positions"] = torch.arange(first, first + case["tokens"], dtype=torch.int32, device=DEVICE)
        s["inv_freqs"] = _frequencies(case["rotary"], 5e5, case["scaled"])
        s["magnitude"] = 1.1 if case["scaled"] else 1.0
        return s
    if kind == "verify":
        b, k, v = case["requests"], case["drafts"], case["vocab"]
        logits = 3.0 * torch.randn(b, k + 1, v, generator=g, device=DEVICE)
        near = logits[:, :k] + 0.8 * torch.randn(b, k, v, generator=g, device=DEVICE)
        s["target"] = torch.softmax(logits, -1).to(TYPES[dtype])
        if case["drawn"]:
            q = torch.softmax(near, -1)
            s["draft"] = q.to(TYPES[dtype])
            s["tokens"] = torch.multinomial(q.reshape(b * k, v), 1, generator=g).reshape(b, k).int()
        else:
            s["draft"] = None
            s["tokens"] = logits[:, :k].argmax(-1).int()
        s["uniforms"] = torch.rand(b, k + 1, generator=g, device=DEVICE)
        s["lengths"] = _ints(_drafts(case)) if case["ragged"] else None
        return s
    hq, hk, dim, base = HEADS[case["model"]]
    n, length = _counts(case)
    page, prefix = case["page"], case["prefix"]
    own_pages = [(c + page - 1) // page for c in length]
    shared = (prefix + page - 1) // page
    pages = shared + sum(own_pages) + 3
    order = torch.randperm(pages, generator=g, device=DEVICE).int()          # pages come as they were freed
    table = torch.zeros(len(n), max(own_pages), dtype=torch.int32, device=DEVICE)
    at = shared
    for b, count in enumerate(own_pages):
        table[b, :count] = order[at: at + count]
        at += count
    cache = _normal((2, pages, hk, page, dim), dtype, g)
    s.update(k_pages=cache[0], v_pages=cache[1], table=table, prefix_pages=order[:shared].contiguous() if prefix else None, prefix=prefix,
             lengths=_ints(length), starts=_ints(_starts(n)), n=n, length=length)
    if kind == "append":
        qkv = _normal((sum(n), hq + 2 * hk, dim), dtype, g)
        s.update(q=qkv[:, :hq], k=qkv[:, hq: hq + hk], v=qkv[:, hq + hk:], inv_freqs=_frequencies(dim, base, case["scaled"]))
        return s
    s.update(q=2 * _normal((sum(n), hq, dim), dtype, g), mask=_masks(n, g) if case["tree"] else None)
    return s


# --------------------------------------------------------------------------------------------------- one pass
def run(s):
    return (_own if own else _plain)[s["case"]["kind"]](s)


def _own_rotate(s):
    import b200_eagle as be
    return be.rope.rotate(s["x"], s["positions"], s["inv_freqs"], magnitude=s["magnitude"], interleaved=s["case"]["interleaved"],
                          inverse=s["case"]["inverse"])


def _own_append(s):
    import b200_eagle as be
    q = be.paged.append(s["q"], s["k"], s["v"], s["k_pages"], s["v_pages"], s["table"], s["lengths"], s["starts"], s["inv_freqs"],
                        prefix_length=s["prefix"], interleaved=s["case"]["interleaved"])
    return q, s["k_pages"], s["v_pages"]


def _own_attention(s):
    import b200_eagle as be
    return be.paged.attention(s["q"], s["k_pages"], s["v_pages"], s["table"], s["lengths"], s["starts"], prefix_pages=s["prefix_pages"],
                              prefix_length=s["prefix"], mask=s["mask"])


def _own_verify(s):
    import b200_eagle as be
    return be.verify.verify_tokens(s["tokens"], s["target"], s["uniforms"], draft_probs=s["draft"], draft_lengths=s["lengths"])


_own = dict(rotate=_own_rotate, append=_own_append, attention=_own_attention, verify=_own_verify)


def _rotated(x, positions, inv_freqs, interleaved, inverse=False, magnitude=1.0):
    """Angles in double precision, the rest in single."""
    angle = positions.double()[:, None] * inv_freqs.double()
    c, sn = (magnitude * angle.cos()).float()[:, None], (magnitude * angle.sin()).float()[:, None]
    if inverse:
        sn = -sn
    r = 2 * inv_freqs.numel()
    y = x.float().clone()
    a, b = (x[..., 0:r:2].float(), x[..., 1:r:2].float()) if interleaved else (x[..., : r // 2].float(), x[..., r // 2: r].float())
    u, w = a * c - b * sn, a * sn + b * c
    if interleaved:
        y[..., 0:r:2], y[..., 1:r:2] = u, w
    else:
        y[..., : r // 2], y[..., r // 2: r] = u, w
    return y.to(x.dtype)


def _plain_rotate(s):
    return _rotated(s["x"], s["positions"], s["inv_freqs"], s["case"]["interleaved"], s["case"]["inverse"], s["magnitude"])


def _plain_append(s):
    page = s["case"]["page"]
    tokens = torch.arange(s["q"].shape[0], device=DEVICE)
    starts, lengths = s["starts"].long(), s["lengths"].long()
    req = (tokens[:, None] >= starts[None, 1:]).sum(1)
    row = lengths[req] - starts[req + 1] + tokens
    at, inside = s["table"][req, row // page].long(), row % page
    positions = s["prefix"] + row
    s["k_pages"][at, :, inside] = _rotated(s["k"], positions, s["inv_freqs"], s["case"]["interleaved"])
    s["v_pages"][at, :, inside] = s["v"]
    return _rotated(s["q"], positions, s["inv_freqs"], s["case"]["interleaved"]), s["k_pages"], s["v_pages"]


def _plain_attention(s):
    page, prefix = s["case"]["page"], s["prefix"]
    tokens, hq, dim = s["q"].shape
    hk = s["k_pages"].shape[1]
    scale = dim ** -0.5
    q = s["q"].float().reshape(tokens, hk, hq // hk, dim)
    # own rows, padded to the longest request
    b, most, width = len(s["n"]), max(s["n"]), s["table"].shape[1] * page
    starts, n, length = s["starts"][:-1].long(), s["starts"].diff().long(), s["lengths"].long()
    new = torch.arange(most, device=DEVICE)
    at = (starts[:, None] + new).clamp(max=tokens - 1)
    keys = s["k_pages"][s["table"].long()].float().transpose(2, 3).reshape(b, width, hk, dim)
    values = s["v_pages"][s["table"].long()].float().transpose(2, 3).reshape(b, width, hk, dim)
    scores = torch.einsum("bnhgd,bkhd->bhgnk", q[at], keys) * scale
    key = torch.arange(width, device=DEVICE)
    behind = key[None, None] - (length - n)[:, None, None]                        # which of the new rows, negative: an older one
    if s["mask"] is None:
        seen = behind <= new[None, :, None]
    else:
        seen = (behind < 0) | ((s["mask"][at][:, :, None] >> behind.clamp(0, 63)) & 1 == 1)
    seen = (seen & (key < length[:, None])[:, None])[:, None, None]
    scores = scores.masked_fill(~seen, float("-inf"))
    top = scores.amax(-1, keepdim=True)
    pad = (new < n[:, None])[:, None, None, :, None]
    if prefix:
        pk = s["k_pages"][s["prefix_pages"].long()].float().transpose(1, 2).reshape(-1, hk, dim)[:prefix]
        pv = s["v_pages"][s["prefix_pages"].long()].float().transpose(1, 2).reshape(-1, hk, dim)[:prefix]
        shared = torch.einsum("thgd,khd->thgk", q, pk) * scale
        top = torch.maximum(top, shared.amax(-1)[at].permute(0, 2, 3, 1)[..., None])
        mine = torch.where(pad, top, 0.0).permute(0, 3, 1, 2, 4)                  # the maxima of the tokens, laid out as their queries
        flat = torch.zeros(tokens, hk, hq // hk, 1, device=DEVICE).index_add_(0, at.reshape(-1), mine.reshape(b * most, hk, hq // hk, 1))
        e = torch.exp(shared - flat)
        psum, pout = e.sum(-1, keepdim=True), torch.einsum("thgk,khd->thgd", e, pv)
        del e, shared
    e = torch.exp(scores - top)
    out = torch.einsum("bhgnk,bkhd->bnhgd", e, values)
    total = e.sum(-1, keepdim=True).permute(0, 3, 1, 2, 4)
    if prefix:
        out, total = out + pout[at], total + psum[at]
    valid = (new < n[:, None]).reshape(-1)
    return (out / total).reshape(b * most, hq, dim)[valid].to(s["q"].dtype)


def _plain_verify(s):
    b, k = s["tokens"].shape
    v = s["target"].shape[-1]
    tokens = s["tokens"].long()
    lengths = torch.full((b,), k, device=DEVICE) if s["lengths"] is None else s["lengths"].long()
    step = torch.arange(k, device=DEVICE)
    p = torch.gather(s["target"][:, :k], 2, tokens[..., None])[..., 0].double()
    q = torch.ones_like(p) if s["draft"] is None else torch.gather(s["draft"], 2, tokens[..., None])[..., 0].double()
    stands = (s["uniforms"][:, :k].double() * q < p) & (step < lengths[:, None])
    accepted = stands.int().cumprod(1).sum(1)
    rows = torch.arange(b, device=DEVICE)
    weights = s["target"][rows, accepted].double()
    refused = accepted < lengths
    last = accepted.clamp(max=max(k - 1, 0))
    if s["draft"] is None:
        rest = weights.clone()
        rest[rows, tokens[rows, last]] = 0.0
    else:
        rest = (weights - s["draft"][rows, last].double()).clamp(min=0.0)
    weights = torch.where(refused[:, None], rest, weights)
    sums = weights.cumsum(1)
    drawn = (sums <= s["uniforms"][:, k:].double() * sums[:, -1:]).sum(1).clamp(max=v - 1)
    out = torch.full((b, k + 1), -1, dtype=torch.int32, device=DEVICE)
    out[:, :k] = torch.where(step < accepted[:, None], s["tokens"], out[:, :k])
    out[rows, accepted] = drawn.int()
    return out, accepted.int()


_plain = dict(rotate=_plain_rotate, append=_plain_append, attention=_plain_attention, verify=_plain_verify)


# --------------------------------------------------------------------------------------------------- in 64 bits
def _turned(x, positions, inv_freqs, interleaved, sign=1.0, magnitude=1.0):
    """The rotation as a product of complex numbers."""
    r = 2 * inv_freqs.numel()
    turn = torch.polar(torch.full((1,), float(magnitude), dtype=torch.float64, device=DEVICE),
                       sign * torch.outer(positions.double(), inv_freqs.double()))[:, None]
    x = x.double()
    pairs = x[..., :r].unflatten(-1, (r // 2, 2)) if interleaved else x[..., :r].unflatten(-1, (2, r // 2)).transpose(-1, -2)
    z = torch.view_as_real(torch.view_as_complex(pairs.contiguous()) * turn)
    return torch.cat([(z if interleaved else z.transpose(-1, -2)).flatten(-2), x[..., r:]], -1)


def exact(case, seed):
    kind = case["kind"]
    if kind == "verify":
        return None                                            # whole numbers
    s = prepare(case, seed)
    if kind == "rotate":
        return _turned(s["x"], s["positions"], s["inv_freqs"], case["interleaved"], -1.0 if case["inverse"] else 1.0, s["magnitude"])
    page, prefix, at = case["page"], case["prefix"], 0
    table = s["table"].tolist()
    if kind == "append":
        q, k, v = [], s["k_pages"].double(), s["v_pages"].double()
        for b, (count, length) in enumerate(zip(s["n"], s["length"])):
            rows = torch.arange(length - count, length, device=DEVICE)
            q.append(_turned(s["q"][at: at + count], prefix + rows, s["inv_freqs"], case["interleaved"]))
            kr, vr = _turned(s["k"][at: at + count], prefix + rows, s["inv_freqs"], case["interleaved"]), s["v"][at: at + count].double()
            for p in range((length - count) // page, (length - 1) // page + 1):
                lo, hi = max(p * page, length - count), min((p + 1) * page, length)
                i = slice(lo - (length - count), hi - (length - count))
                k[table[b][p], :, lo - p * page: hi - p * page] = kr[i].transpose(0, 1)
                v[table[b][p], :, lo - p * page: hi - p * page] = vr[i].transpose(0, 1)
            at += count
        return torch.cat(q), k, v
    hq, hk, dim, _ = HEADS[case["model"]]
    out = torch.empty(sum(s["n"]), hq, dim, dtype=torch.float64, device=DEVICE)

    def rows_of(cache, pages, count, head):
        return cache[pages.long(), head].reshape(-1, dim)[:count].double()

    for head in range(hk):
        mine = slice(head * (hq // hk), (head + 1) * (hq // hk))
        pk = rows_of(s["k_pages"], s["prefix_pages"], prefix, head) if prefix else torch.empty(0, dim, dtype=torch.float64, device=DEVICE)
        pv = rows_of(s["v_pages"], s["prefix_pages"], prefix, head) if prefix else pk
        at = 0
        for b, (count, length) in enumerate(zip(s["n"], s["length"])):
            k = torch.cat([pk, rows_of(s["k_pages"], s["table"][b], length, head)])
            v = torch.cat([pv, rows_of(s["v_pages"], s["table"][b], length, head)])
            visible = torch.ones(count, prefix + length, dtype=torch.bool, device=DEVICE)
            new = visible[:, prefix + length - count:]
            if s["mask"] is None:
                new.copy_(new.tril())
            else:
                words = s["mask"][at: at + count]
                for j in range(count):
                    new[:, j] = (words >> j) & 1 == 1
            score = torch.einsum("ngd,kd->gnk", s["q"][at: at + count, mine].double(), k) / math.sqrt(dim)
            out[at: at + count, mine] = torch.einsum("gnk,kd->ngd", torch.softmax(score.masked_fill(~visible, -math.inf), -1), v)
            at += count
    return out
