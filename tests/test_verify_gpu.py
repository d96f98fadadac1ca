"""Verification of drafted tokens from given random numbers, against the rule written out request by request in 64 bits: the same tokens."""
import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu


def rule(tokens, p, u, q=None, lengths=None):
    out, accepted = [], []
    B, K = tokens.shape
    V = p.shape[-1]
    for b in range(B):
        n = K if lengths is None else min(max(int(lengths[b]), 0), K)
        length = n
        for i in range(length):
            x = int(tokens[b, i])
            if not (0 <= x < V and float(u[b, i]) * (1.0 if q is None else float(q[b, i, x])) < float(p[b, i, x])):
                n = i
                break
        w = p[b, n].astype(np.float64)
        full = np.where(w > 0, w, 0.0)
        if n < length:
            if q is None:
                w = w.copy()
                if 0 <= tokens[b, n] < V:
                    w[tokens[b, n]] = 0.0
            else:
                w = w - q[b, n].astype(np.float64)
        w = np.where(w > 0, w, 0.0)
        if not w.sum() > 0:
            w = full
        s = np.cumsum(w)
        over = np.nonzero((s > float(u[b, K]) * s[-1]) & (w > 0))[0]
        some = np.nonzero(w > 0)[0]
        token = int(over[0]) if len(over) else (int(some[-1]) if len(some) else 0)
        out.append([int(t) for t in tokens[b, :n]] + [token] + [-1] * (K - n))
        accepted.append(n)
    return out, accepted


def check(be, cuda, tokens, p, u, q=None, lengths=None):
    want = rule(tokens.numpy(), p.float().numpy(), u.numpy(), None if q is None else q.float().numpy(), None if lengths is None else lengths.numpy())
    got = be.verify_tokens(tokens.to(cuda), p.to(cuda), u.to(cuda), draft_probs=None if q is None else q.to(cuda),
                           draft_lengths=None if lengths is None else lengths.to(cuda))
    assert got[0].dtype == got[1].dtype == torch.int32
    assert got[1].tolist() == want[1] and got[0].tolist() == want[0]
    return want


@pytest.mark.parametrize("drawn", [True, False])
@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16], ids=str)
@pytest.mark.parametrize("B,K,V", [(1, 0, 1), (2, 1, 2), (5, 3, 7), (3, 2, 1000), (40, 7, 4099), (9, 40, 521), (2, 5, 151936), (300, 2, 33)])
def test_the_same_tokens_as_the_rule(be, cuda, B, K, V, dtype, drawn):
    g = torch.Generator().manual_seed(B * 1000 + V)
    logits = 2.0 * torch.randn(B, K + 1, V, generator=g)
    p = torch.softmax(logits, -1).to(dtype)
    full = torch.softmax(logits[:, :K] + 0.7 * torch.randn(B, K, V, generator=g), -1)
    tokens = torch.multinomial(full.reshape(-1, V), 1, generator=g).reshape(B, K).int() if K else torch.zeros(B, 0, dtype=torch.int32)
    u = torch.rand(B, K + 1, generator=g)
    lengths = torch.randint(-1, K + 2, (B,), generator=g).int()
    for n in (None, lengths):
        want = check(be, cuda, tokens, p, u, full.to(dtype) if drawn else None, n)
    if B >= 40 and drawn:
        assert len(set(want[1])) > 2


def test_borders_are_exact(be, cuda):
    """Weights of quarters and random numbers on the borders between them: a border belongs to the token behind it; u q = p refuses."""
    p = torch.tensor([0.25, 0.0, 0.25, 0.5]).repeat(8, 2, 1)
    u = torch.tensor([0.0, 0.25, 0.5, 0.75, 2.0 ** -24, 0.25 - 2.0 ** -26, 0.5 + 2.0 ** -24, 1 - 2.0 ** -24])
    uniforms = torch.stack([torch.full((8,), 0.99), u], 1)
    tokens = torch.full((8, 1), 1, dtype=torch.int32)
    want = check(be, cuda, tokens, p, uniforms)                          # token 1 cannot stand: drawn from p without it
    assert [t[0] for t in want[0]] == [0, 2, 3, 3, 0, 0, 3, 3]
    q = torch.tensor([0.5, 0.5, 0.0, 0.0]).repeat(8, 1, 1)
    uniforms = torch.stack([torch.full((8,), 0.5), u], 1)                # 0.5 * 0.5 = p(0): refused; left: 0, 0, 0.25, 0.5
    want = check(be, cuda, torch.zeros(8, 1, dtype=torch.int32), p, uniforms, q)
    assert want[1] == [0] * 8 and {t[0] for t in want[0]} == {2, 3}
    uniforms[:, 0] = torch.nextafter(torch.tensor(0.5), torch.tensor(0.0))
    assert check(be, cuda, torch.zeros(8, 1, dtype=torch.int32), p, uniforms, q)[1] == [1] * 8


def test_what_leaves_nothing(be, cuda):
    """p = q refused by u = 1 (a caller's rounding): drawn from p.  An empty row: token 0.  NaN and negative values weigh nothing.  Tokens outside
    the vocabulary are refused, whatever the random number."""
    g = torch.Generator().manual_seed(1)
    p = torch.softmax(torch.randn(4, 3, 50, generator=g), -1)
    q = p[:, :2].clone()
    tokens = torch.randint(0, 50, (4, 2), generator=g).int()
    u = torch.rand(4, 3, generator=g)
    u[:, 0] = 1.0
    check(be, cuda, tokens, p, u, q)
    p[1, 0] = 0.0
    p[2, 0, 10:] = float("nan")
    p[3, 0, :20] = -1.0
    check(be, cuda, tokens, p, u, q)
    check(be, cuda, tokens, p, u)
    tokens[0, 0], tokens[1, 0], tokens[2, 1] = -1, 50, 2 ** 31 - 1
    u[:, 0] = 0.0
    check(be, cuda, tokens, p, u, q)
    check(be, cuda, tokens, p, u)
    u[:, 2] = torch.tensor([1.0, float("nan"), -0.5, 1.5])               # outside [0, 1): some token of the row all the same
    t, n = be.verify_tokens(tokens.to(cuda), p.to(cuda), u.to(cuda), draft_probs=q.to(cuda))
    last = t[torch.arange(4), n.long()]
    assert ((0 <= last) & (last < 50)).all()


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=str)
def test_strides_and_unaligned_rows(be, cuda, dtype):
    g = torch.Generator().manual_seed(2)
    B, K, V = 6, 4, 3001
    big = torch.softmax(2 * torch.randn(K + 1, B, V, generator=g), -1).to(dtype)
    p, q = big.transpose(0, 1), torch.softmax(2 * torch.randn(B, 2 * K, V, generator=g), -1).to(dtype)[:, ::2]
    tokens = torch.randint(0, V, (B, 2 * K), generator=g).int()[:, :K]
    u = torch.rand(B, 9, generator=g)[:, :K + 1]
    u[:, :K] *= 1e-3
    want = rule(tokens.numpy(), p.float().numpy(), u.numpy(), q.float().numpy())
    base = torch.empty(K + 1, B, V + 3, dtype=dtype, device=cuda)
    base[..., 3:] = big.to(cuda)
    for pd in (big.to(cuda).transpose(0, 1), base[..., 3:].transpose(0, 1)):
        qd = torch.empty(B, 2 * K, V, dtype=dtype, device=cuda)[:, ::2]
        qd.copy_(q)
        td, ud = torch.zeros(B, 2 * K, dtype=torch.int32, device=cuda)[:, :K], torch.zeros(B, 9, device=cuda)[:, :K + 1]
        td.copy_(tokens), ud.copy_(u)
        got = be.verify_tokens(td, pd, ud, draft_probs=qd)
        assert got[1].tolist() == want[1] and got[0].tolist() == want[0]


def test_tokens_are_distributed_as_the_target(be, cuda):
    """60 000 requests of one pair of distributions: the first token that comes out, drafted or drawn, follows p.  Chi-square with 11 degrees of
    freedom, 99.9th percentile 31.3; the seed is fixed."""
    g = torch.Generator(device=cuda).manual_seed(4)
    V, n = 12, 60000
    p, q = torch.softmax(1.5 * torch.randn(2, V, device=cuda, generator=g), -1)
    tokens = torch.multinomial(q, n, replacement=True, generator=g).int()[:, None]
    u = torch.rand(n, 2, device=cuda, generator=g)
    t, a = be.verify_tokens(tokens, p.expand(n, 2, V), u, draft_probs=q.expand(n, 1, V))
    count = torch.bincount(t[:, 0].long(), minlength=V).double()
    want = n * p.double() / p.double().sum()
    assert ((count - want) ** 2 / want).sum() < 31.3
    share = torch.minimum(p, q).sum().item()
    assert abs(a.double().mean().item() - share) < 5 * (0.25 / n) ** 0.5


def test_repeated_captured_and_on_another_stream(be, cuda):
    g = torch.Generator(device=cuda).manual_seed(6)
    B, K, V = 33, 3, 20011
    p = torch.softmax(2 * torch.randn(B, K + 1, V, device=cuda, generator=g), -1)
    q = torch.softmax(p[:, :K].log() + 0.5 * torch.randn(B, K, V, device=cuda, generator=g), -1)
    tokens = torch.multinomial(q.reshape(-1, V), 1, generator=g).reshape(B, K).int()
    u = torch.rand(B, K + 1, device=cuda, generator=g)
    want = [t.clone() for t in be.verify_tokens(tokens, p, u, draft_probs=q)]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        other = be.verify_tokens(tokens, p, u, draft_probs=q)
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(a, b) for a, b in zip(want, other))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = be.verify_tokens(tokens, p, u, draft_probs=q)
    u.copy_(u.flip(0).clone())
    graph.replay()
    again = be.verify_tokens(tokens, p, u, draft_probs=q)
    assert all(torch.equal(a, b) for a, b in zip(got, again)) and not torch.equal(want[0], again[0])


def test_verify_refusals(be, cuda):
    p, q = torch.rand(2, 4, 10, device=cuda), torch.rand(2, 3, 10, device=cuda)
    tokens, u, n = torch.zeros(2, 3, dtype=torch.int32, device=cuda), torch.rand(2, 4, device=cuda), torch.zeros(2, dtype=torch.int32, device=cuda)
    v = be.verify_tokens
    calls = [lambda: v(tokens.long(), p, u), lambda: v(tokens, p[0], u), lambda: v(tokens, p, u[:, :3]), lambda: v(tokens, p.cpu(), u),
             lambda: v(tokens, p, u.double()), lambda: v(tokens, p.double(), u), lambda: v(tokens, p, u, draft_probs=q.half()),
             lambda: v(tokens, p, u, draft_probs=p), lambda: v(tokens, p, u, draft_lengths=n.long()), lambda: v(tokens, p, u, draft_lengths=n[:1]),
             lambda: v(tokens, p.transpose(1, 2), u), lambda: v(tokens[:, :2], p, u), lambda: v(tokens, p[:, :, :0], u), lambda: v(tokens.cpu(), p, u)]
    for call in calls:
        with pytest.raises(be._lib.B200Error):
            call()
    assert v(tokens[:0], p[:0], u[:0])[0].shape == (0, 4)
