"""Rotary positions in general form, and the append to a paged cache, against the formula in 64 bits.

Tolerance: of a rotated pair (a, b), magnitude m: the angle is off by at most 2^-25 (its fraction of a turn rounded to fp32 in an eighth of a turn to
either side), sine and cosine by two units of 2^-24, m times them, two products and their sum by half a unit each: below 2^-21 m (|a| + |b|)
in all, and the result's rounding: half a step of its type, or of the smallest fp16 numbers, 2^-25."""
import math
from fractions import Fraction

import pytest
import torch

pytestmark = pytest.mark.gpu

HALF, BF, F32 = torch.float16, torch.bfloat16, torch.float32


def turned(x, positions, inv_freqs, scaling=1.0, magnitude=1.0, interleaved=False, inverse=False):
    """(result, |a| + |b| of each value's pair) in 64 bits."""
    r = 2 * inv_freqs.numel()
    angle = positions.double()[:, None] * (inv_freqs.double() * scaling)
    c, s = magnitude * angle.cos()[:, None], magnitude * angle.sin()[:, None] * (-1.0 if inverse else 1.0)
    x = x.double()
    out, size = x.clone(), torch.zeros_like(x)
    lo, hi = (slice(0, r, 2), slice(1, r, 2)) if interleaved else (slice(0, r // 2), slice(r // 2, r))
    a, b = x[..., lo], x[..., hi]
    out[..., lo], out[..., hi] = a * c - b * s, a * s + b * c
    size[..., lo] = size[..., hi] = magnitude * (a.abs() + b.abs())
    return out, size


def close(got, want, size, dtype):
    tol = 2.0 ** -21 * size + torch.finfo(dtype).eps / 2 * want.abs() + (2.0 ** -25 if dtype == HALF else 0.0)
    tol = torch.where(size > 0, tol, torch.zeros_like(tol))              # what passes through is copied
    assert got.dtype == dtype and ((got.double() - want).abs() <= tol).all()


@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("dtype", [HALF, BF, F32], ids=str)
@pytest.mark.parametrize("tokens,heads,dim,rotary", [(1, 1, 64, 64), (3, 5, 128, 64), (130, 7, 96, 24), (700, 4, 128, 128), (5, 3, 80, 80), (2, 3, 7, 2), (9, 70, 33, 6),
                                                     (1300, 1, 256, 256), (4, 2, 2048, 2048)])
def test_rotate_is_the_formula(be, cuda, tokens, heads, dim, rotary, dtype, interleaved):
    g = torch.Generator().manual_seed(tokens)
    x = torch.randn(tokens, heads, dim, generator=g).to(dtype).to(cuda)
    pos = torch.randint(-5000, 1 << 20, (tokens,), generator=g).to(cuda)
    inv, scaling, _ = be.rope.frequencies(rotary, 5e5, device=cuda)
    for p in (pos, pos.int()):
        for inverse in (False, True):
            got = be.rope.rotate(x, p, inv, scaling_factor=1 / 3, magnitude=1.25, interleaved=interleaved, inverse=inverse)
            close(got, *turned(x, pos, inv, 1 / 3, 1.25, interleaved, inverse), dtype)


def test_far_positions_keep_their_angles(be, cuda):
    """2^31 rows on, at a frequency of one, a product in single precision would be off by more than a turn."""
    x = torch.randn(6, 2, 64, device=cuda)
    pos = torch.tensor([0, 1, 131071, 1 << 24, (1 << 31) - 1, -(1 << 31)], device=cuda)
    inv, _, _ = be.rope.frequencies(64, 1e4, device=cuda)
    close(be.rope.rotate(x, pos, inv), *turned(x, pos, inv), F32)


@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("offset", [0, 1])
def test_strided_rows_in_place_and_into_a_slice(be, cuda, interleaved, offset):
    """Slices of a fused projection; with an offset no row starts at 16 bytes."""
    g = torch.Generator().manual_seed(3)
    fused = torch.randn(37, 9, 64 + 2 * offset, generator=g).half().to(cuda)
    before = fused.clone()
    pos = torch.arange(37, device=cuda)
    inv, _, _ = be.rope.frequencies(48, 1e4, device=cuda)
    x = fused[:, 2:7, offset:offset + 64]
    want, size = turned(x, pos, inv, interleaved=interleaved)
    got = be.rope.rotate(x, pos, inv, interleaved=interleaved)
    assert got.is_contiguous()
    close(got, want, size, HALF)
    other = torch.zeros(5, 37, 70, dtype=HALF, device=cuda).transpose(0, 1)[..., offset:offset + 64]
    assert be.rope.rotate(x, pos, inv, interleaved=interleaved, out=other) is other and torch.equal(other, got)
    be.rope.rotate(x, pos, inv, interleaved=interleaved, out=x)
    assert torch.equal(x, got)
    before[:, 2:7, offset:offset + 64] = got
    assert torch.equal(fused, before)


def test_broadcast_heads_empty_calls_and_infinities(be, cuda):
    inv, _, _ = be.rope.frequencies(32, 1e4, device=cuda)
    x = torch.randn(4, 1, 64, device=cuda).half()
    pos = torch.arange(4, device=cuda)
    assert torch.equal(be.rope.rotate(x.expand(4, 6, 64), pos, inv), be.rope.rotate(x, pos, inv).expand(4, 6, 64))
    assert be.rope.rotate(x[:0], pos[:0], inv).shape == (0, 1, 64)
    assert be.rope.rotate(x[:, :0], pos, inv).shape == (4, 0, 64)
    x[1, 0, 3], x[2, 0, 63], x[3, 0, 40] = float("inf"), float("nan"), float("-inf")
    got = be.rope.rotate(x, pos, inv)
    bad = ~got.isfinite()
    assert bad.nonzero().tolist() == [[1, 0, 3], [1, 0, 19], [2, 0, 63], [3, 0, 40]]


@pytest.mark.parametrize("interleaved", [False, True])
def test_the_inverse_is_the_gradient(be, cuda, interleaved):
    """Against the formula's own gradient, by torch in 64 bits, and against differences: the rotation is linear, so a difference of any length
    is exact up to rounding."""
    g = torch.Generator().manual_seed(5)
    x, dy, d = (torch.randn(11, 3, 64, generator=g).to(cuda) for _ in range(3))
    pos = torch.arange(100, 111, device=cuda)
    inv, _, _ = be.rope.frequencies(40, 1e4, device=cuda)
    kw = dict(magnitude=1.5, interleaved=interleaved)
    grad = be.rope.rotate(dy, pos, inv, inverse=True, **kw)
    leaf = x.double().requires_grad_()
    r = 20
    angle = pos.double()[:, None] * inv.double()
    c, s = 1.5 * angle.cos()[:, None], 1.5 * angle.sin()[:, None]
    a, b = (leaf[..., 0:40:2], leaf[..., 1:40:2]) if interleaved else (leaf[..., :r], leaf[..., r:40])
    u, w = a * c - b * s, a * s + b * c
    da, db = (dy[..., 0:40:2], dy[..., 1:40:2]) if interleaved else (dy[..., :r], dy[..., r:40])
    ((u * da).sum() + (w * db).sum() + (leaf[..., 40:] * dy[..., 40:]).sum()).backward()
    close(grad, leaf.grad, turned(dy, pos, inv, 1.0, 1.5, interleaved, True)[1], F32)
    slope = ((be.rope.rotate(x + d, pos, inv, **kw).double() - be.rope.rotate(x, pos, inv, **kw).double()) * dy.double()).sum()
    # (about 2000 terms of size one, each off by a few units of 2^-24)
    assert abs(slope - (grad.double() * d.double()).sum()) <= 2000 * 2.0 ** -20


def test_scaled_frequencies(be):
    """Against each rule written out pair by pair."""
    import math
    f, scaling, mag = be.rope.frequencies(64, 1e4, dict(type="linear", factor=4.0))
    assert scaling == 0.25 and mag == 1.0 and f[0] == 1.0 and f[16].item() == pytest.approx(1e-2, rel=1e-6)
    f, scaling, mag = be.rope.frequencies(128, 5e5, dict(rope_type="llama3", factor=8.0))
    for i in range(64):
        base = 5e5 ** (-2 * i / 128)
        turns = 8192 * base / (2 * math.pi)
        want = base if turns > 4 else base / 8 if turns < 1 else base / 8 * (4 - turns) / 3 + base * (turns - 1) / 3
        assert f[i].item() == pytest.approx(want, rel=1e-6)
    model = be.ModelArgs(**{**be.shape_preset("llama3-8b").__dict__, "rope_scaling": dict(type="llama3", factor=8.0)})
    assert torch.allclose(f, be.llama.rope_inv_freqs(model)[0], rtol=1e-5, atol=0.0)
    f, scaling, mag = be.rope.frequencies(128, 1e6, dict(type="yarn", factor=4.0, original_max_position_embeddings=32768))
    assert mag == pytest.approx(1 + 0.1 * math.log(4.0)) and scaling == 1.0
    for i in range(64):
        base = 1e6 ** (-2 * i / 128)
        turns = 32768 * base / (2 * math.pi)
        if turns > 32 * 1.25:                                            # (a pair's frequency is 1.24 times the next one's)
            assert f[i].item() == pytest.approx(base, rel=1e-6)
        elif turns < 1 / 1.25:
            assert f[i].item() == pytest.approx(base / 4, rel=1e-6)
        else:
            assert base / 4 * (1 - 1e-6) <= f[i].item() <= base * (1 + 1e-6)
    for bad in (dict(type="dynamic", factor=2.0),):
        with pytest.raises(be._lib.B200Error):
            be.rope.frequencies(64, 1e4, bad)
    with pytest.raises(be._lib.B200Error):
        be.rope.frequencies(63)


def test_rotate_refusals(be, cuda):
    x, pos, (inv, _, _) = torch.zeros(4, 2, 64, device=cuda).half(), torch.arange(4, device=cuda), be.rope.frequencies(64, device=cuda)
    E = be._lib.B200Error
    calls = [lambda: be.rope.rotate(x.cpu(), pos, inv), lambda: be.rope.rotate(x, pos.cpu(), inv), lambda: be.rope.rotate(x, pos[:3], inv),
             lambda: be.rope.rotate(x, pos.float(), inv), lambda: be.rope.rotate(x.double(), pos, inv), lambda: be.rope.rotate(x[0], pos, inv),
             lambda: be.rope.rotate(x, pos, inv.double()), lambda: be.rope.rotate(x[..., :32], pos, inv), lambda: be.rope.rotate(x, pos, inv[:0]),
             lambda: be.rope.rotate(x.transpose(1, 2), pos, inv[:1]), lambda: be.rope.rotate(x, pos, inv, out=x[:, :1]),
             lambda: be.rope.rotate(x, pos, inv, out=x.float()), lambda: be.rope.rotate(x, pos, inv, out=x[:, :1].expand(4, 2, 64)),
             lambda: be.rope.rotate(x, None, inv)]
    for call in calls:
        with pytest.raises(E):
            call()


def test_calls_on_two_streams_and_replayed(be, cuda):
    """Rotations side by side and from a graph, with positions that change: the same bits as one call after the other."""
    inv, _, _ = be.rope.frequencies(128, device=cuda)
    xs = [torch.randn(n, 6, 128, device=cuda).half() for n in (1, 300, 3000)]
    pos = [torch.arange(7, 7 + x.shape[0], device=cuda) for x in xs]
    want = [be.rope.rotate(x, p, inv) for x, p in zip(xs, pos)]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    got = []
    for _ in range(3):
        for i, (x, p) in enumerate(zip(xs, pos)):
            got.append((i, be.rope.rotate(x, p, inv)))
            with torch.cuda.stream(side):
                got.append((i, be.rope.rotate(x, p, inv)))
    torch.cuda.synchronize()
    assert all(torch.equal(y, want[i]) for i, y in got)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = [be.rope.rotate(x, p, inv) for x, p in zip(xs, pos)]
    for p in pos:
        p += 1000
    graph.replay()
    assert all(torch.equal(y, be.rope.rotate(x, p, inv)) for x, p, y in zip(xs, pos, out))
    assert not torch.equal(out[1], want[1])


def test_positions_beyond_32_bits_keep_their_angles(be, cuda):
    """Against angles reduced in fractions of 80 digits.  Up to 2^37 rows an angle is off by 2^-24 more than near ones (half of 2^-23), where the tolerance has
    room: 2^-25 + 2 units of 2^-24, 2 products and a sum make 1.75 x 2^-23 (and 0.5 now) of the 4 x 2^-23 that it is."""
    turn = Fraction(1) / (2 * Fraction("3.14159265358979323846264338327950288419716939937510582097494459230781640628620899"))
    pos = [p + d for p in (1 << 31, 1 << 34, (1 << 37) - 3000, -(1 << 36)) for d in (-1, 0, 777, 2049)]
    x = torch.randn(len(pos), 2, 128, generator=torch.Generator().manual_seed(2)).to(cuda)
    inv, _, _ = be.rope.frequencies(128, 5e5)
    for scaling in (1.0, 1 / 3):
        angle = torch.empty(len(pos), 64, dtype=torch.float64)
        for j, f in enumerate(inv.tolist()):
            for i, p in enumerate(pos):
                angle[i, j] = 2 * math.pi * float(Fraction(f) * Fraction(scaling) * p * turn % 1)
        c, s, (a, b) = angle.cos().to(cuda)[:, None], angle.sin().to(cuda)[:, None], x.double().chunk(2, -1)
        size = (a.abs() + b.abs()).repeat(1, 1, 2)
        close(be.rope.rotate(x, torch.tensor(pos, device=cuda), inv.to(cuda), scaling_factor=scaling), torch.cat([a * c - b * s, a * s + b * c], -1), size, F32)
