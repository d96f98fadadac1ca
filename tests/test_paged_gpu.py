"""A paged cache behind a prefix that requests share: append and attention against their definitions in 64 bits.

Tolerance of the attention, e = eps / 2 of the type, A = sum of p |v| per output: a probability is rounded to the type (e p), and the sum uses the
rounded ones (e A more, after division); the result is rounded (e |o|).  Scores are fp32 sums of 16-bit products, off by at most 2^-20 of
S = scale * sum |q k| (128 terms, 2^-24 each, and as much again for a sum that truncates), which moves a probability by twice that
relatively (its own and the sum's), as do the roundings of exp2 and of the running sums, 2^-18 together for up to 2^14 rows.  fp16
probabilities below 2^-14 are off by up to 2^-25 in place of e p, relative to the largest: a row of n keys by n 2^-25 max |v| at most, over a sum of
at least 1."""
import ctypes
import math
import pathlib
import re

import pytest
import torch

pytestmark = pytest.mark.gpu

HALF, BF = torch.float16, torch.bfloat16


class Batch:
    """Requests with `new` tokens each behind `old` rows, pages in random order, everything that is nobody's poisoned."""

    def __init__(self, cuda, heads, kv, hd, page, prefix, old, new, dtype=HALF, seed=0, order="hnd", poison=float("nan"), spread=2.0, pad=0):
        g = torch.Generator().manual_seed(seed)
        self.heads, self.kv, self.hd, self.page, self.prefix, self.old, self.new = heads, kv, hd, page, prefix, old, new
        lengths = [o + n for o, n in zip(old, new)]
        need = [(x + page - 1) // page for x in lengths]
        shared = (prefix + page - 1) // page
        pages = shared + sum(need) + 2
        perm = torch.randperm(pages, generator=g).int()
        self.prefix_pages = perm[:shared].to(cuda)
        table = torch.full((len(old), max(need + [1]) + 1), -7, dtype=torch.int32)
        at = shared
        for b, n in enumerate(need):
            table[b, :n] = perm[at:at + n]
            at += n
        self.table = table.to(cuda)
        shape = (2, pages, kv, page, hd) if order == "hnd" else (2, pages, page, kv, hd)
        data = torch.full(shape, poison).to(dtype).to(cuda)
        self.data = data if order == "hnd" else data.transpose(2, 3)
        self.k_pages, self.v_pages = self.data[0], self.data[1]
        self.lengths = torch.tensor(lengths, dtype=torch.int32, device=cuda)
        self.row_starts = torch.tensor([sum(new[:i]) for i in range(len(new) + 1)], dtype=torch.int32, device=cuda)
        self.tokens = sum(new) + pad
        # dense rows: the prefix's, then each request's
        draw = lambda n: torch.randn(2, kv, n, hd, generator=g).to(dtype).to(cuda)
        self.shared = draw(prefix)
        self.rows = [draw(x) for x in lengths]
        self._put(self.prefix_pages.tolist(), self.shared)
        for b, r in enumerate(self.rows):
            self._put(self.table[b].tolist(), r)
        self.q = (spread * torch.randn(self.tokens, heads, hd, generator=g)).to(dtype).to(cuda)
        self.mask = None

    def _put(self, pages, rows):
        for i in range(0, rows.shape[2], self.page):
            n = min(self.page, rows.shape[2] - i)
            self.data[:, pages[i // self.page], :, :n] = rows[:, :, i:i + n]

    def tree(self, seed=1, empty=False):
        g = torch.Generator().manual_seed(seed)
        words = []
        for n in self.new:
            mine = []
            for i in range(n):
                parent = mine[int(torch.randint(0, i, (1,), generator=g))] if i else 0
                mine.append(parent | 1 << i)
            words += mine
        words += [0] * (self.tokens - len(words))
        if empty:
            words[::2] = [0] * len(words[::2])
        words = [w & (1 << 64) - 1 for w in words]                       # (bits of the first 64 new rows)
        self.mask = torch.tensor([w - (1 << 64) if w >= 1 << 63 else w for w in words], dtype=torch.int64).to(self.q.device)
        return self

    def run(self, be, **kw):
        args = dict(prefix_pages=self.prefix_pages if self.prefix else None, prefix_length=self.prefix, mask=self.mask)
        args.update(kw)
        return be.paged.attention(self.q, self.k_pages, self.v_pages, self.table, self.lengths, self.row_starts, **args)

    def exact(self, scale=None):
        """(o, tolerance) in 64 bits; tokens that are nobody's are NaN."""
        scale = self.hd ** -0.5 if scale is None else scale
        dtype = self.q.dtype
        e = torch.finfo(dtype).eps / 2
        group = self.heads // self.kv
        out = torch.full(self.q.shape, math.nan, dtype=torch.float64, device=self.q.device)
        tol = torch.zeros_like(out)
        at = 0
        for b, n in enumerate(self.new):
            if n == 0:
                continue
            old, rows = self.old[b], torch.cat([self.shared, self.rows[b]], 2).double()
            k, v = rows[0].repeat_interleave(group, 0), rows[1].repeat_interleave(group, 0)              # (heads, keys, hd)
            q = self.q[at:at + n].double().transpose(0, 1)
            seen = torch.ones(n, rows.shape[2], dtype=torch.bool, device=self.q.device)
            for j in range(n):
                col = self.prefix + old + j
                seen[:, col] = torch.arange(n, device=seen.device) >= j if self.mask is None else \
                    (((self.mask[at:at + n] >> j) & 1 == 1) if j < 64 else torch.zeros(n, dtype=torch.bool, device=seen.device))
            s = (scale * q @ k.transpose(1, 2)).masked_fill(~seen, -math.inf)
            p = torch.softmax(s, -1)
            p = torch.where(seen.any(-1)[:, None], p, torch.zeros_like(p))
            o, a = p @ v, p @ v.abs()
            big = float((abs(scale) * q.abs() @ k.abs().transpose(1, 2)).max()) if rows.shape[2] else 0.0
            small = rows.shape[2] * 2.0 ** -25 * float(v.abs().max()) if dtype == HALF and rows.shape[2] else 0.0
            out[at:at + n] = o.transpose(0, 1)
            tol[at:at + n] = (e * o.abs() + (2 * e + 2 * 2.0 ** -20 * big + 2.0 ** -18) * a).transpose(0, 1) + small + (2.0 ** -25 if dtype == HALF else 0.0)
            at += n
        return out, tol

    def check(self, be, scale=None, **kw):
        got = self.run(be, **({} if scale is None else dict(scale=scale)), **kw)
        want, tol = self.exact(scale)
        n = sum(self.new)
        assert got.dtype == self.q.dtype
        bad = ~((got[:n].double() - want[:n]).abs() <= tol[:n])
        assert not bad.any(), (int(bad.sum()), bad.nonzero()[0].tolist(), got[:n][bad][:4].tolist(), want[:n][bad][:4].tolist())
        assert be.paged.attention_error(self.q.device) == 0
        return got


SHAPES = [(14, 2, 64), (8, 2, 128), (9, 3, 128), (4, 4, 64), (32, 1, 128), (160, 1, 64)]
BATCHES = [
    # prefix, old rows, new tokens
    (0, [0], [1]),
    (0, [5, 0, 127, 128, 129], [1, 1, 1, 1, 1]),
    (1, [0, 0], [1, 3]),
    (127, [3], [2]),
    (128, [1000, 0, 64], [1, 7, 0]),
    (129, [0, 250], [130, 2]),
    (1000, [700] * 9, [1] * 9),
    (4099, [10, 300, 0, 45, 1], [1, 2, 33, 16, 5]),
    (700, [0] * 40, [4] * 40),
    (20000, [100, 2500], [1, 1]),
]


@pytest.mark.parametrize("batch", BATCHES, ids=lambda b: f"{b[0]}-{len(b[1])}x{max(b[2])}")
@pytest.mark.parametrize("shape", SHAPES, ids=lambda s: "x".join(map(str, s)))
def test_attention_is_the_definition(be, cuda, shape, batch):
    dtype = BF if len(batch[1]) % 2 else HALF
    Batch(cuda, *shape, 16, *batch, dtype=dtype).check(be)
    Batch(cuda, *shape, 128, *batch, dtype=HALF if dtype == BF else BF, order="nhd", seed=1).check(be)


@pytest.mark.parametrize("hd,prefix,new", [(64, 700, [350, 350]), (128, 1500, [700]), (128, 330, [256, 1, 400, 0, 31]), (64, 2900, [1100])])
def test_many_tiles_share_a_prefix(be, cuda, hd, prefix, new):
    """So many tiles of queries that a worker's stretch of a prefix is more than half of it, or all, or several."""
    Batch(cuda, 32, 8, hd, 64, prefix, [5] * len(new), new, dtype=BF if hd == 64 else HALF).check(be)
    Batch(cuda, 12, 2, hd, 16, prefix, [200] * len(new), new, seed=2).check(be)


@pytest.mark.parametrize("page", [8, 16, 32, 64, 128, 256, 384])
@pytest.mark.parametrize("order", ["hnd", "nhd"])
@pytest.mark.parametrize("hd", [64, 128])
def test_pages_of_any_size_and_order(be, cuda, page, order, hd):
    Batch(cuda, 8, 2, hd, page, 777, [3, 515, 0], [1, 6, 9], order=order).check(be)


@pytest.mark.parametrize("dtype", [HALF, BF], ids=str)
@pytest.mark.parametrize("prefix,old,new", [(0, [0, 7, 130], [5, 64, 31]), (300, [100, 0], [64, 17]), (513, [65, 126, 1], [3, 64, 2]), (0, [40], [90])])
@pytest.mark.parametrize("shape", [(14, 2, 64), (8, 2, 128)], ids=lambda s: "x".join(map(str, s)))
def test_masks_of_drafted_trees(be, cuda, shape, prefix, old, new, dtype):
    Batch(cuda, *shape, 32, prefix, old, new, dtype=dtype).tree().check(be)
    got = Batch(cuda, *shape, 32, prefix, old, new, dtype=dtype).tree(empty=True).check(be)
    if prefix == 0 and old[0] == 0:
        assert (got[0] == 0).all()                                       # a token that sees nothing


@pytest.mark.parametrize("spread,scale", [(30.0, None), (2.0, 1.0), (2.0, 0.0)])
def test_peaked_and_flat_scales(be, cuda, spread, scale):
    for dtype in (HALF, BF):
        Batch(cuda, 8, 2, 128, 16, 600, [50, 600], [3, 2], dtype=dtype, spread=spread).check(be, scale=scale)


def test_growing_scores_leave_earlier_maxima_far_behind(be, cuda):
    b = Batch(cuda, 8, 2, 64, 16, 2000, [900, 10], [2, 40])
    ramp = lambda n: torch.linspace(0.1, 4.0, n, device=cuda)[:, None]
    b.shared[0] = (b.shared[0].float().abs() * ramp(2000)).half()
    for r in b.rows:
        r[0] = (r[0].float().abs() * 2 * ramp(r.shape[2])).half()
    b._put(b.prefix_pages.tolist(), b.shared)
    for i, r in enumerate(b.rows):
        b._put(b.table[i].tolist(), r)
    b.q = b.q.abs()
    b.check(be)


@pytest.mark.parametrize("dtype", [HALF, BF], ids=str)
@pytest.mark.parametrize("tree", [False, True])
@pytest.mark.parametrize("hd,prefix,old,new", [(64, 0, [0, 3], [9, 1]), (128, 300, [125, 700, 1], [7, 1, 40]), (128, 0, [60], [130])])
def test_nan_and_infinities_reach_those_who_see_them(be, cuda, hd, prefix, old, new, tree, dtype):
    """New rows whose values or keys are not finite: a token that does not see them (a later row, another branch of the tree) gets what it
    gets without them, within the tolerance; one that does is not finite in those dims, or, for a key, NaN in all."""
    def batch():
        b = Batch(cuda, 8, 2, hd, 16, prefix, old, new, dtype=dtype)
        return b.tree(empty=True) if tree else b
    b = batch()
    want = b.run(be)
    exact, tol = b.exact()
    at, hit = 0, torch.zeros(sum(new), 8, hd, dtype=torch.bool, device=cuda)
    for r, n in enumerate(new):
        for j, head, what, key in ((n - 1, 0, math.inf, False), (n // 2, 1, math.nan, False), (n // 3, 0, -math.inf, False), (n - 2, 1, math.nan, True)):
            if j < 0:
                continue
            dims = slice(0, hd) if key else slice(3 * j % hd, 3 * j % hd + 1)
            b.rows[r][0 if key else 1, head, old[r] + j, 7 if key else dims] = what
            for i in range(n):
                sees = j <= i if not tree else j < 64 and bool((int(b.mask[at + i]) >> j) & 1)
                if sees:
                    hit[at + i, 4 * head: 4 * head + 4, dims] = True
        at += n
        b._put(b.table[r].tolist(), b.rows[r])
    got = b.run(be)
    assert not got[hit].isfinite().any() and ((got.double() - exact).abs() <= tol)[~hit].all()
    b = batch()                                                          # and nothing of it is left for the next call
    assert torch.equal(b.run(be), want) and be.paged.attention_error(cuda) == 0


def test_a_prefix_counts_like_rows_of_its_own(be, cuda):
    """The same keys as a shared prefix, and copied into every request's pages: the same within two roundings."""
    a = Batch(cuda, 8, 2, 128, 16, 333, [20, 90], [2, 5])
    b = Batch(cuda, 8, 2, 128, 16, 0, [353, 423], [2, 5], seed=1)
    for i, r in enumerate(b.rows):
        r.copy_(torch.cat([a.shared, a.rows[i]], 2))
        b._put(b.table[i].tolist(), r)
    b.q = a.q
    got = a.check(be), b.check(be)
    _, tol = a.exact()
    assert ((got[0].double() - got[1].double()).abs() <= 2 * tol).all()


def test_padding_is_left_alone_and_strided_operands_are_taken(be, cuda):
    b = Batch(cuda, 8, 2, 128, 16, 100, [20, 0, 90], [2, 0, 5], pad=4)
    wide = torch.zeros(b.tokens, 12, 256, dtype=HALF, device=cuda)
    wide[:, 2:10, :128] = b.q
    b.q = wide[:, 2:10, :128]
    out = torch.full((8, b.tokens, 128), 7.0, dtype=HALF, device=cuda).transpose(0, 1)
    assert b.check(be, out=out) is out
    assert (out[7:] == 7.0).all()
    b.row_starts += 2                                                     # tokens ahead of the first request are nobody's either
    b.q = torch.cat([b.q[:2], b.q[:9]])
    out = torch.full((11, 8, 128), 7.0, dtype=HALF, device=cuda)
    b.run(be, out=out)
    assert (out[:2] == 7.0).all() and (out[9:] == 7.0).all() and (out[2:9] != 7.0).all()


def test_page_numbers_outside_the_cache_stand_for_zeros(be, cuda):
    b = Batch(cuda, 8, 2, 64, 16, 64, [100], [1])
    want = Batch(cuda, 8, 2, 64, 16, 64, [100], [1])
    want.rows[0][:, :, 16:32] = 0
    want.rows[0][:, :, 64:80] = 0
    want.shared[:, :, 32:48] = 0
    b.shared, b.rows = want.shared, want.rows
    b.table[0, 1], b.table[0, 4], b.prefix_pages[2] = b.k_pages.shape[0], -1, 2 ** 31 - 1
    b.check(be)
    b.lengths.fill_(-5)                                                   # no rows, as the lengths say: the prefix is left
    b.run(be)
    b.lengths.fill_(10 ** 6)                                              # more rows than the table has: those it has, the poisoned ones among them
    assert b.run(be).isnan().all() and be.paged.attention_error(cuda) == 0


def test_append_then_attention_is_a_step(be, cuda):
    """Steps of several requests, captured once and replayed with other lengths, against attention over the rows in 64 bits; rows the pass
    does not write stay as they are."""
    heads, kv, hd, page, prefix, B, T = 8, 2, 128, 16, 200, 3, 4
    g = torch.Generator(device=cuda).manual_seed(0)
    cache = be.PagedKVCache(2, 64, page, kv, hd, device=cuda)
    shared = cache.take(prefix)
    own = [cache.take(100) for _ in range(B)]
    prefix_pages, table = torch.tensor(shared, dtype=torch.int32, device=cuda), torch.tensor(own, dtype=torch.int32, device=cuda)
    cache.data.normal_(generator=g)
    inv, scaling, mag = be.rope.frequencies(hd, 1e4, dict(type="yarn", factor=4.0, original_max_position_embeddings=4096), device=cuda)
    lengths = torch.tensor([4, 20, 61], dtype=torch.int32, device=cuda)
    starts = torch.arange(0, B * T + 1, T, dtype=torch.int32, device=cuda)
    qkv = torch.randn(B * T, heads + 2 * kv, hd, device=cuda, generator=g).half()
    kw = dict(scaling_factor=scaling, magnitude=mag)

    def step():
        out = []
        for layer in range(2):
            k_pages, v_pages = cache.layer(layer)
            q = be.paged.append(qkv[:, :heads], qkv[:, heads:heads + kv], qkv[:, heads + kv:], k_pages, v_pages, table, lengths, starts, inv, prefix_length=prefix, **kw)
            out.append((q, be.paged.attention(q, k_pages, v_pages, table, lengths, starts, prefix_pages=prefix_pages, prefix_length=prefix)))
        return out

    step()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    for turn in range(3):
        qkv.normal_(generator=g)
        before, old = cache.data.clone(), lengths.tolist()
        graph.replay()
        pos = torch.cat([torch.arange(prefix + n - T, prefix + n) for n in old]).to(cuda)
        for layer, (q, o) in enumerate(out):
            assert torch.equal(q, be.rope.rotate(qkv[:, :heads], pos, inv, **kw))
            kr, want = be.rope.rotate(qkv[:, heads:heads + kv], pos, inv, **kw), before[layer].clone()
            for b in range(B):
                for j in range(T):
                    r = old[b] - T + j
                    want[0, own[b][r // page], :, r % page] = kr[b * T + j]
                    want[1, own[b][r // page], :, r % page] = qkv[b * T + j, heads + kv:]
            assert torch.equal(cache.data[layer], want)
            m = Batch(cuda, heads, kv, hd, page, prefix, [n - T for n in old], [T] * B)
            rows = lambda pages, n: want[:, pages].transpose(2, 3).reshape(2, -1, kv, hd)[:, :n].transpose(1, 2)
            m.shared, m.rows, m.q = rows(shared, prefix), [rows(own[b], old[b]) for b in range(B)], q
            exact, tol = m.exact()
            assert ((o.double() - exact).abs() <= tol).all()
        lengths += T
    cache.give(shared)
    with pytest.raises(be._lib.B200Error):
        cache.give(shared)


@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("dtype", [HALF, BF], ids=str)
@pytest.mark.parametrize("hd,rotary,page,order", [(64, 64, 16, "hnd"), (128, 64, 8, "nhd"), (96, 40, 32, "hnd"), (70, 6, 128, "nhd"), (128, 128, 64, "hnd")])
def test_append_writes_its_rows_and_no_other(be, cuda, hd, rotary, page, order, dtype, interleaved):
    g = torch.Generator().manual_seed(hd)
    new = [1, 0, 40, 3, 700]
    old = [0, 9, 100, 15, 4]
    heads, kv, B, pad = 6, 2, 5, 3
    b = Batch(cuda, heads, kv, hd, page, 0, old, new, dtype=dtype, order=order, poison=3.0, pad=pad)
    b.data.copy_(torch.randn(b.data.shape, generator=g))
    qkv = torch.randn(b.tokens, heads + 2 * kv, hd, generator=g).to(dtype).to(cuda)
    q, k, v = qkv[:, :heads], qkv[:, heads:heads + kv], qkv[:, heads + kv:]
    inv, _, _ = be.rope.frequencies(rotary, 5e5, device=cuda)
    n = sum(new)
    rows = torch.cat([torch.arange(o, o + x) for o, x in zip(old, new)]).to(cuda)
    for positions, prefix in ((None, 1000), (torch.randint(0, 9999, (b.tokens,), generator=g).to(cuda), 0), (torch.arange(b.tokens, device=cuda).int(), 5)):
        before = b.data.clone()
        out = torch.full(q.shape, 7.0, dtype=dtype, device=cuda)
        be.paged.append(q, k, v, b.k_pages, b.v_pages, b.table, b.lengths, b.row_starts, inv, positions=positions, prefix_length=prefix, magnitude=0.75,
                        interleaved=interleaved, q_out=out)
        pos = rows + prefix if positions is None else positions[:n].long()
        kw = dict(magnitude=0.75, interleaved=interleaved)
        assert torch.equal(out[:n], be.rope.rotate(q[:n], pos, inv, **kw)) and (out[n:] == 7.0).all()
        kr = be.rope.rotate(k[:n], pos, inv, **kw)
        req = torch.repeat_interleave(torch.arange(B), torch.tensor(new)).to(cuda)
        at = b.table[req, rows // page].long()
        before[0][at, :, rows % page] = kr
        before[1][at, :, rows % page] = v[:n]
        assert torch.equal(b.data, before)
    same = qkv.clone()
    got = be.paged.append(same[:, :heads], k, v, b.k_pages, b.v_pages, b.table, b.lengths, b.row_starts, inv, q_out=same[:, :heads], interleaved=interleaved)
    assert torch.equal(got[:n], be.rope.rotate(q[:n], rows, inv, interleaved=interleaved)) and torch.equal(same[:, heads:], qkv[:, heads:])


def test_append_drops_rows_without_a_page(be, cuda):
    b = Batch(cuda, 4, 2, 64, 16, 0, [14, 0, 30], [4, 2, 6])
    inv, _, _ = be.rope.frequencies(64, device=cuda)
    k = torch.randn(12, 2, 64, device=cuda).half()
    b.data.zero_()
    b.table[0, 1] = b.k_pages.shape[0]                                    # request 0: two of four rows dropped
    b.table[1, 0] = -1                                                    # request 1: both
    b.lengths[2] = 10 ** 9                                                # request 2: behind the table's end
    out = be.paged.append(b.q, k, k, b.k_pages, b.v_pages, b.table, b.lengths, b.row_starts, inv)
    assert out.isfinite().all()
    assert int((b.data[1] != 0).any(-1).any(1).sum()) == 2
    b.lengths.fill_(1)                                                    # fewer rows than new tokens: what lies ahead of row 0 is dropped
    b.data.zero_()
    b.table.fill_(0)
    be.paged.append(b.q, k, k, b.k_pages, b.v_pages, b.table[:, :1], b.lengths, b.row_starts, inv)
    assert int((b.data[1] != 0).any(-1).any(1).sum()) == 1


def test_paged_refusals(be, cuda):
    b = Batch(cuda, 4, 2, 64, 16, 20, [14, 0], [4, 2])
    E, at, ap = be._lib.B200Error, be.paged.attention, be.paged.append
    inv, _, _ = be.rope.frequencies(64, device=cuda)
    k = torch.randn(6, 2, 64, device=cuda).half()
    base = [b.q, b.k_pages, b.v_pages, b.table, b.lengths, b.row_starts]

    def changed(i, t):
        return base[:i] + [t] + base[i + 1:]

    calls = [lambda: at(*changed(0, b.q.cpu())), lambda: at(*changed(0, b.q.bfloat16())), lambda: at(*changed(0, b.q[0])), lambda: at(*changed(0, b.q[:, :3])),
             lambda: at(*changed(1, b.k_pages[:, :1])), lambda: at(*changed(2, b.v_pages.transpose(1, 2).contiguous().transpose(1, 2))),
             lambda: at(*changed(3, b.table.long())), lambda: at(*changed(3, b.table[:1])), lambda: at(*changed(4, b.lengths.long())),
             lambda: at(*changed(5, b.row_starts[:2])), lambda: at(*base, prefix_length=5), lambda: at(*base, prefix_pages=b.prefix_pages, prefix_length=33),
             lambda: at(*base, prefix_length=-1), lambda: at(*base, scale=-0.1), lambda: at(*base, scale=math.nan), lambda: at(*base, mask=torch.zeros(5, dtype=torch.int64, device=cuda)),
             lambda: at(*base, mask=torch.zeros(6, dtype=torch.int32, device=cuda)), lambda: at(*base, out=b.q[:5]), lambda: at(*base, out=b.q.float()),
             lambda: at(*changed(0, b.q[:1].expand(6, 4, 64))), lambda: at(*changed(0, torch.zeros(6, 4, 68, device=cuda).half()[..., 1:65])),
             lambda: at(b.q[..., :32], b.k_pages[..., :32], b.v_pages[..., :32], *base[3:]),
             lambda: at(b.q, b.k_pages[:, :, :12], b.v_pages[:, :, :12], *base[3:]),
             lambda: ap(b.q, k[:5], k, *base[1:], inv), lambda: ap(b.q, k, k[:, :1], *base[1:], inv), lambda: ap(b.q, k, k, *base[1:], inv[:0]),
             lambda: ap(b.q, k, k, *base[1:], inv, prefix_length=-1), lambda: ap(b.q, k, k, *base[1:], inv, positions=torch.zeros(5, device=cuda).int()),
             lambda: ap(b.q, k, k, *base[1:], inv, q_out=b.q[:5]), lambda: be.PagedKVCache(1, 4, 24, 2, 64, device=cuda)]
    for call in calls:
        with pytest.raises(E):
            call()
    empty = torch.zeros(0, 4, 64, device=cuda).half()
    none = dict(page_table=b.table[:0], lengths=b.lengths[:0], row_starts=b.row_starts[:1])
    assert at(empty, b.k_pages, b.v_pages, **none).shape == (0, 4, 64)


@pytest.mark.parametrize("shape", [(8, 2, 128), (14, 2, 64)], ids=str)
def test_calls_at_once_captured_and_in_place(be, cuda, shape):
    """Passes side by side on two streams, by calls and by two graphs replayed in turn and at once, have a workspace each: bit for bit what
    one call after the other gives; so has a result that takes the queries' place."""
    heads, kv, hd = shape
    a = Batch(cuda, heads, kv, hd, 16, 5000, [700, 90, 0], [3, 40, 1])
    b = Batch(cuda, heads, kv, hd, 32, 1000, [300] * 5, [4] * 5, seed=1).tree()
    want = [x.check(be).clone() for x in (a, b)]
    here, side = torch.cuda.current_stream(), torch.cuda.Stream()
    side.wait_stream(here)
    got = []
    for _ in range(5):
        got.append((0, a.run(be)))
        with torch.cuda.stream(side):
            got.append((1, b.run(be)))
    graphs, out = [], []
    torch.cuda.synchronize()
    for x in (a, b):
        graphs.append(torch.cuda.CUDAGraph())
        with torch.cuda.graph(graphs[-1]):
            out.append(x.run(be))
    for turn in range(4):
        for o in out:
            o.zero_()
        side.wait_stream(here)
        graphs[0].replay()
        with torch.cuda.stream(side if turn % 2 else here):
            graphs[1].replay()
        here.wait_stream(side)
        got += [(0, out[0].clone()), (1, out[1].clone())]
    torch.cuda.synchronize()
    for i, o in got:
        assert torch.equal(o, want[i])
    for x, w in zip((a, b), want):
        assert x.run(be, out=x.q) is x.q and torch.equal(x.q, w)
    assert be.paged.attention_error(cuda) == 0


def test_the_first_attention_is_not_captured(be, cuda, monkeypatch):
    b = Batch(cuda, 4, 2, 64, 16, 20, [14, 0], [4, 2])
    want = b.run(be)
    monkeypatch.setattr(be.paged, "_errors", {})
    with pytest.raises(be._lib.B200Error, match="captured"):
        with torch.cuda.graph(torch.cuda.CUDAGraph()):
            b.run(be)
    assert torch.equal(b.run(be), want)


def test_as_many_requests_as_are_taken(be, cuda):
    Batch(cuda, 4, 1, 64, 8, 100, [i % 11 for i in range(1024)], [1 + (i % 7 == 0) for i in range(1024)]).check(be)
    Batch(cuda, 4, 1, 64, 8, 0, [0] * 1024, [i % 2 for i in range(1024)]).check(be)
    more = Batch(cuda, 4, 1, 64, 8, 0, [0] * 1025, [1] * 1025)
    with pytest.raises(be._lib.B200Error):
        more.run(be)


def test_scores_of_minus_infinity_weigh_nothing(be, cuda):
    """A key whose scores are minus infinity, first of a request without a prefix, counts as if it were hidden; also where a value that is not
    seen makes the row be looked at again."""
    b = Batch(cuda, 4, 2, 64, 16, 0, [3], [2])
    b.q[..., 0] = 1.0
    b.rows[0][0, :, 0, 0] = -math.inf
    b.rows[0][1, :, 4, 5] = math.inf                                     # (of the last token, which the one before it does not see)
    b._put(b.table[0].tolist(), b.rows[0])
    got = b.run(be)
    q, (k, v) = b.q[0].double(), b.rows[0][:, :, 1:4].double()
    k, v = k.repeat_interleave(2, 0), v.repeat_interleave(2, 0)
    p = torch.softmax(torch.einsum("hd,hnd->hn", q, k) / 8, -1)
    want, size = torch.einsum("hn,hnd->hd", p, v), torch.einsum("hn,hnd->hd", p, v.abs())
    big = float(torch.einsum("hd,hnd->hn", q.abs(), k.abs()).max()) / 8
    tol = 2.0 ** -11 * want.abs() + (2 * 2.0 ** -11 + 2 * 2.0 ** -20 * big + 2.0 ** -18) * size + 2.0 ** -25 * (1 + 5 * float(v.abs().max()))
    assert ((got[0].double() - want).abs() <= tol).all()
    assert got[1, :, 5].isinf().all() and got[1, :, 6:].isfinite().all()


@pytest.mark.parametrize("interleaved", [False, True])
def test_speculation_writes_what_plain_steps_write(be, cuda, interleaved):
    """Requests behind a shared prompt, drafts of mixed quality: append, attention and verification together give the tokens that a model in 64
    bits without a cache gives, and accept just the drafts that agree.  (The best logit is ahead by more than 0.1 at every place, by the 64-bit model.
    Here half-step roundings of q, k, probabilities and results move an output by 6e-4, as a standard deviation, and a logit of 384 of them by 0.012.)"""
    heads, kv, hd, page, V, prompt, B, K, total = 6, 2, 64, 16, 61, 43, 3, 3, 24
    g = torch.Generator().manual_seed(9)
    table_of = torch.randn(V, heads + 2 * kv, hd, generator=g).half()
    W = torch.randn(heads * hd, V, generator=g).half()
    inv, scaling, mag = be.rope.frequencies(hd, 1e4)
    text = torch.randint(0, V, (prompt,), generator=g).tolist()
    starts = torch.randint(0, V, (B,), generator=g).tolist()

    def turn(x):
        pos = torch.arange(x.shape[0], dtype=torch.float64)[:, None] * inv.double()
        c, s = pos.cos()[:, None], pos.sin()[:, None]
        a, b = (x[..., ::2], x[..., 1::2]) if interleaved else (x[..., :hd // 2], x[..., hd // 2:])
        y = (a * c - b * s, b * c + a * s)
        return torch.stack(y, -1).flatten(-2) if interleaved else torch.cat(y, -1)

    def after(tokens):
        x = table_of[tokens].double()
        q, k = turn(x)[-1, :heads], turn(x)[:, heads:heads + kv].repeat_interleave(heads // kv, 1)
        p = torch.softmax(torch.einsum("hd,nhd->hn", q, k) / 8, -1)
        logits = torch.einsum("hn,nhd->hd", p, x[:, heads + kv:].repeat_interleave(heads // kv, 1)).flatten() @ W.double()
        best = logits.topk(2).values
        assert best[0] - best[1] > 0.1
        return int(logits.argmax())

    want = []
    for b in range(B):
        mine = [starts[b]]
        for _ in range(total + K + 1):
            mine.append(after(text + mine))
        want.append(mine)

    cache = be.PagedKVCache(1, 32, page, kv, hd, device=cuda)
    k_pages, v_pages = cache.layer(0)
    ints = lambda x: torch.tensor(x, dtype=torch.int32, device=cuda)
    prefix = ints(cache.take(prompt))
    table = ints([cache.take(total + 2 * K + 2) for _ in range(B)])
    E, proj = table_of.to(cuda), W.float().to(cuda)
    inv = inv.to(cuda)

    def put(tokens, pages, lengths, row_starts, ahead):
        x = E[tokens.long()]
        return be.paged.append(x[:, :heads], x[:, heads:heads + kv], x[:, heads + kv:], k_pages, v_pages, pages, lengths, row_starts, inv, prefix_length=ahead,
                               interleaved=interleaved)

    put(ints(text), prefix[None], ints([prompt]), ints([0, prompt]), 0)
    written, rnd = [1] * B, torch.Generator().manual_seed(0)
    row_starts = torch.arange(0, B * (K + 1) + 1, K + 1, dtype=torch.int32, device=cuda)
    while min(written) < total:
        right = torch.randint(0, K + 1, (B,), generator=rnd).tolist()
        drafts = [[want[b][written[b] + i] if i != right[b] else (want[b][written[b] + i] + 1) % V for i in range(K)] if written[b] < total else [0] * K
                  for b in range(B)]
        agree = [next((i for i in range(K) if written[b] + i >= len(want[b]) or drafts[b][i] != want[b][written[b] + i]), K) for b in range(B)]
        pas = ints([[want[b][written[b] - 1]] + drafts[b] for b in range(B)]).flatten()
        lengths = ints([w + K for w in written])                         # rows: the tokens written, the last of them in this pass, and the drafts
        q = put(pas, table, lengths, row_starts, prompt)
        o = be.paged.attention(q, k_pages, v_pages, table, lengths, row_starts, prefix_pages=prefix, prefix_length=prompt)
        probs = torch.softmax(1000 * (o.float().flatten(1) @ proj), -1).view(B, K + 1, V)
        tokens, accepted = be.verify_tokens(ints(drafts), probs, torch.full((B, K + 1), 0.5, device=cuda))
        for b in range(B):
            if written[b] >= total:                                      # (a request that is done stays where it is)
                continue
            n = int(accepted[b])
            assert n == agree[b], (b, written[b], drafts[b], want[b][written[b]:written[b] + K + 1], tokens[b].tolist())
            assert tokens[b, :n + 1].tolist() == want[b][written[b]:written[b] + n + 1] and (tokens[b, n + 1:] == -1).all()
            written[b] += n + 1
    assert be.paged.attention_error(cuda) == 0


def test_sizes_beyond_32_bits_are_refused(be, cuda):
    """Not cut to what is left of them."""
    b = Batch(cuda, 4, 2, 64, 16, 20, [14, 0], [4, 2])
    inv, _, _ = be.rope.frequencies(64, device=cuda)
    k = torch.randn(6, 2, 64, device=cuda).half()
    base = [b.k_pages, b.v_pages, b.table, b.lengths, b.row_starts]
    far = (1 << 32) + 5
    calls = [lambda: be.paged.append(b.q, k, k, *base, inv, prefix_length=far), lambda: be.paged.attention(b.q, *base, prefix_pages=b.prefix_pages, prefix_length=far),
             lambda: be.paged.append(b.q[:1].expand(far, 4, 64), k[:1].expand(far, 2, 64), k[:1].expand(far, 2, 64), *base, inv),
             lambda: be.rope.rotate(b.q[:1].expand(far, 4, 64), torch.zeros(6, device=cuda).int(), inv)]
    for call in calls:
        with pytest.raises(be._lib.B200Error):
            call()


@pytest.mark.parametrize("shape", [(8, 4, 128), (14, 2, 64)], ids=str)
def test_workers_of_many_pieces(be, cuda, shape):
    """Segments of a block or two, a dozen to a worker: the sum of a piece and the maxima of the next, which begins at once, are told apart, so that
    every run gives the same bits, those of the definition."""
    n = 900
    b = Batch(cuda, *shape, 16, 40, [(37 * i) % 200 for i in range(n)], [1 + i % 3 for i in range(n)])
    want = b.check(be)
    for _ in range(30):
        assert torch.equal(b.run(be), want)


@pytest.mark.parametrize("ahead", [0, 16, 32, 48])
def test_a_workspace_may_begin_at_any_16_bytes(be, cuda, ahead):
    """By the C entry, in just the bytes that it asks for: the same bits wherever it begins, and nothing behind it is written."""
    b = Batch(cuda, 8, 2, 128, 16, 1500, [700, 90, 0], [3, 140, 1])
    want = b.check(be)
    lib, ptr = be._lib.lib(), be._lib.ptr
    c = be.paged._paged(b.q, b.k_pages, b.v_pages, b.table, b.lengths, b.row_starts)
    room = lib.b200_paged_attention_workspace_bytes(ctypes.byref(c))
    ws = torch.full((room + 128,), 113, dtype=torch.uint8, device=cuda)
    assert ws.data_ptr() % 64 == 0
    out, err = torch.empty_like(b.q), torch.zeros(1, dtype=torch.int32, device=cuda)
    rc = lib.b200_paged_attention(ctypes.byref(c), ptr(b.q), *b.q.stride()[:2], ptr(out), *out.stride()[:2], ptr(b.prefix_pages), b.prefix, None,
                                  128 ** -0.5, ptr(ws[ahead:]), room, ptr(err), be._lib.stream_ptr(cuda))
    assert rc == 0 and torch.equal(out, want) and int(err) == 0
    assert (ws[:ahead] == 113).all() and (ws[ahead + room:] == 113).all()


def test_the_error_word_is_read_back(be, cuda):
    """Set by the host, in the place of a wait that ran out, and found by every name of the device."""
    b = Batch(cuda, 4, 2, 64, 16, 20, [14, 0], [4, 2])
    b.run(be)
    word = be.paged._errors[b.q.device.index]
    try:
        word.fill_(31)
        for name in ("cuda", torch.device("cuda"), b.q.device.index, f"cuda:{b.q.device.index}", b.q.device):
            assert be.paged.attention_error(name) == 31
    finally:
        word.zero_()
    b.check(be)


def test_the_error_word_is_clear_for_every_stream(be, cuda, monkeypatch):
    """Made by a call on a stream that has work ahead of it, and read on another at once: its zero is there, not what the memory held."""
    b = Batch(cuda, 4, 2, 64, 16, 20, [14, 0], [4, 2])
    want = b.run(be)
    monkeypatch.setattr(be.paged, "_errors", {})
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        used = torch.full((1,), 77, dtype=torch.int32, device=cuda)      # (the allocator's next block of this size)
        torch.cuda.current_stream().synchronize()
        del used
        torch.cuda._sleep(40_000_000)                                    # 20 ms
        be.paged._error_word(b.q.device)                                 # (as the first attention does)
    assert be.paged.attention_error(b.q.device) == 0
    with torch.cuda.stream(side):
        got = b.run(be)
    torch.cuda.synchronize()
    assert torch.equal(got, want)


@pytest.mark.parametrize("prefix,old,new", [(20000, [100, 2500], [1, 1]), (3000, [5, 5], [300, 400])])
def test_a_short_wait_limit_changes_no_result_and_the_error_word_clears(be, cuda, prefix, old, new):
    """A limit of one poll, for calls and captured ones.  (A poll takes some 4 us, and all that a wait here is for comes within two, so that the word stays
    clear by itself: the host sets it.)"""
    lib = be._lib.lib()
    b = Batch(cuda, 8, 2, 128, 16, prefix, old, new)
    want = b.check(be)
    word, graph = be.paged._errors[b.q.device.index], torch.cuda.CUDAGraph()
    try:
        lib.b200_set_wait_limit(1)
        word.fill_(31)
        assert torch.equal(b.run(be), want)
        with torch.cuda.graph(graph):
            got = b.run(be)
    finally:
        lib.b200_set_wait_limit(0)
    graph.replay()
    assert torch.equal(got, want)
    assert be.paged.attention_error(cuda) == be.paged.attention_error(cuda, clear=True) == 31 and be.paged.attention_error(cuda) == 0
    b.check(be)


@pytest.mark.parametrize("prefix,old,new", [(20000, [3], [1]), (2000, [100, 3], [40, 2]), (900, [7] * 20, [30] * 20)])
def test_values_of_weights_that_are_too_small_for_a_number_reach_the_row(be, cuda, prefix, old, new):
    """The prefix's scores lie 144 below the own rows', so that its weights are 0: its NaN and infinities make NaN of a row's dims all the same, whichever
    piece of the line they are in, and the other dims are what the own rows make them."""
    b = Batch(cuda, 8, 2, 64, 16, prefix, old, new)
    own = Batch(cuda, 8, 2, 64, 16, 0, old, new)
    b.q.fill_(3.0)
    b.shared[0] = -3.0
    for r, o in zip(b.rows, own.rows):
        r[0] = 3.0
        o.copy_(r)
    own.q = b.q
    b.shared[1, 0, 0, 5], b.shared[1, 0, prefix // 2, 9], b.shared[1, 1, prefix - 1, 11] = math.nan, math.inf, -math.inf
    b._put(b.prefix_pages.tolist(), b.shared)
    for i, r in enumerate(b.rows):
        b._put(b.table[i].tolist(), r)
    got = b.run(be)
    want, tol = own.exact()
    hit = torch.zeros_like(got, dtype=torch.bool)
    hit[:, :4, 5] = hit[:, :4, 9] = hit[:, 4:, 11] = True
    assert got[hit].isnan().all() and ((got.double() - want).abs() <= tol)[~hit].all()


@pytest.mark.parametrize("prefix,old,new,heads", [(300, [30000], [1], 8), (300, [20000] * 8, [40] * 8, 8)])
def test_nan_in_the_prefix_costs_no_walk_over_the_own_rows(be, cuda, prefix, old, new, heads):
    """All see it, so that a row's own rows have nothing to tell apart: results as they are, in about the time of other values (row by row, 30000 own rows took
    a hundred times that)."""
    b = Batch(cuda, heads, 2, 128, 64, prefix, old, new)
    want = b.check(be)

    def time():
        took = []
        for _ in range(5):
            start, end = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
            torch.cuda._sleep(200_000)                                   # (the host gets ahead)
            start.record()
            got = b.run(be)
            end.record()
            end.synchronize()
            took.append(start.elapsed_time(end))
        return min(took), got

    usual = time()[0]
    b.shared[1, 1, 5, 3], b.shared[0, 0, 7, 2] = math.nan, math.nan
    b._put(b.prefix_pages.tolist(), b.shared)
    longer, got = time()
    want[:, heads // 2:, 3] = want[:, :heads // 2] = math.nan
    assert torch.equal(got.isnan(), want.isnan()) and torch.equal(got.nan_to_num(), want.nan_to_num())
    assert longer < 4 * usual, (usual, longer)


def test_the_documented_calls_run(be, cuda):
    """The block of the documentation that serves requests over pages, line by line as it stands."""
    root = pathlib.Path(__file__).resolve().parent.parent
    blocks = [b for f in sorted(root.glob("*.md")) for b in re.findall(r"```python\n(.*?)```", f.read_text(), re.S)
              if all(f"be.{name}(" in b for name in ("PagedKVCache", "rope.frequencies", "paged.append", "paged.attention", "verify_tokens"))]
    assert blocks
    g = torch.Generator(device=cuda).manual_seed(4)
    ints = lambda *x: torch.tensor(x, dtype=torch.int32, device=cuda)
    heads, kv, P, n, V = 8, 2, 40, 7, 50
    rand = lambda *shape: torch.randn(*shape, device=cuda, generator=g).half()
    for text in blocks:
        names = dict(be=be, layers=2, pages=16, kv_heads=kv, config=dict(rope_scaling=dict(type="linear", factor=2.0)), i=1, q=rand(n, heads, 128), k=rand(n, kv, 128),
                     v=rand(n, kv, 128), page_table=ints(3, 4, 5, 6).view(2, 2), lengths=ints(20, 3), row_starts=ints(0, 4, 7), P=P, prefix=ints(7, 8, 9),
                     x=rand(n, heads, 128), positions=torch.arange(n, device=cuda), draft_tokens=torch.zeros(2, 3, dtype=torch.int32, device=cuda),
                     target_probs=torch.rand(2, 4, V, device=cuda, generator=g), draft_probs=torch.rand(2, 3, V, device=cuda, generator=g),
                     uniforms=torch.rand(2, 4, device=cuda, generator=g))
        exec(text, names)
        assert names["o"].shape == (n, heads, 128) and names["o"].isfinite().all() and names["x"].shape == (n, heads, 128) and names["tokens"].shape == (2, 4)
    torch.cuda.synchronize()
