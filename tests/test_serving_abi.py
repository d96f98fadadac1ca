"""Refusals of the serving operators' C entries, which come ahead of any CUDA call, so that they run without a GPU; and the operators of
Python on tensors that are not on one."""
import ctypes

import pytest
import torch


def _memory():
    buf = (ctypes.c_char * 128)()
    base = ctypes.addressof(buf)
    return buf, base + (-base) % 16


def _cache(be, base, **kw):
    args = dict(dtype=0, requests=2, tokens=3, heads=4, kv_heads=2, head_dim=64, pages=4, page_size=16, table_width=2, page_table=base, table_stride=2,
                lengths=base, row_starts=base, k_pages=base, v_pages=base, page_stride=2048, head_stride=1024, row_stride=64)
    return be._lib.Paged(**{**args, **kw})


def _rotary(be, base, **kw):
    args = dict(positions=base, inv_freqs=base, scaling=1.0, magnitude=1.0, positions_64=0, rotary_dim=64, interleaved=0, inverse=0)
    return be._lib.Rotary(**{**args, **kw})


def test_rotate_entry(be):
    lib, (buf, base) = be._lib.lib(), _memory()

    def call(r, x=base, out=base, dtype=0, tokens=3, heads=4, dim=64):
        return lib.b200_rotate(ctypes.byref(r) if r is not None else None, x, 256, 64, out, 256, 64, dtype, tokens, heads, dim, None)

    assert call(None) == call(_rotary(be, base), x=None) == call(_rotary(be, base), out=None) == -1
    assert call(_rotary(be, base, rotary_dim=63)) == call(_rotary(be, base, rotary_dim=0)) == call(_rotary(be, base, rotary_dim=66)) == -1
    assert call(_rotary(be, base, positions=None)) == call(_rotary(be, base, inv_freqs=None)) == -1
    assert call(_rotary(be, base), tokens=-1) == call(_rotary(be, base), dim=4096) == call(_rotary(be, base), heads=1 << 17) == -1
    assert call(_rotary(be, base), dtype=3) == -3
    assert call(_rotary(be, base), tokens=0) == call(_rotary(be, base), heads=0) == 0


def test_append_entry(be):
    lib, (buf, base) = be._lib.lib(), _memory()

    def call(c, r=None, q=base):
        r = _rotary(be, base) if r is None else r
        return lib.b200_paged_append(ctypes.byref(c), ctypes.byref(r), q, 256, 64, base, base, 128, 64, base, 256, 64, 0, None)

    for kw in (dict(kv_heads=3), dict(kv_heads=0), dict(pages=0), dict(page_size=0), dict(tokens=-1), dict(requests=-1), dict(k_pages=None),
               dict(v_pages=None), dict(lengths=None), dict(row_starts=None), dict(page_table=None), dict(table_width=-1), dict(head_dim=4096)):
        assert call(_cache(be, base, **kw)) == -1, kw
    assert call(_cache(be, base, dtype=2)) == -3
    assert call(_cache(be, base, table_width=1 << 28)) == -6
    assert call(_cache(be, base), r=_rotary(be, base, inverse=1)) == call(_cache(be, base), r=_rotary(be, base, rotary_dim=128)) == -1
    assert call(_cache(be, base), q=None) == -1
    assert call(_cache(be, base, tokens=0)) == call(_cache(be, base, requests=0)) == 0


def test_attention_entry(be):
    lib, (buf, base) = be._lib.lib(), _memory()

    def call(c, q=base, q_token=256, prefix=None, length=0, ws=base, room=1 << 40, error=base, scale=0.125):
        return lib.b200_paged_attention(ctypes.byref(c), q, q_token, 64, base, 256, 64, prefix, length, None, scale, ws, room, error, None)

    assert lib.b200_paged_attention_workspace_bytes(ctypes.byref(_cache(be, base))) > 0
    assert lib.b200_paged_attention_workspace_bytes(ctypes.byref(_cache(be, base, kv_heads=3))) == 0
    for kw in (dict(head_dim=96), dict(page_size=12), dict(page_size=4), dict(page_size=192)):
        assert call(_cache(be, base, **kw)) == -1, kw
    assert call(_cache(be, base, requests=1025)) == call(_cache(be, base, table_width=(1 << 26) + 1)) == -6
    assert call(_cache(be, base), prefix=base, length=(1 << 30) + 1) == call(_cache(be, base), prefix=base, length=0x7fffffff) == -6
    assert call(_cache(be, base), length=5) == call(_cache(be, base), prefix=base, length=-1) == -1
    assert call(_cache(be, base), q=None) == call(_cache(be, base), ws=None) == call(_cache(be, base), error=None) == -1
    assert call(_cache(be, base), scale=-1.0) == call(_cache(be, base), scale=float("nan")) == -1
    assert call(_cache(be, base), room=0) == -4
    assert call(_cache(be, base), q=base + 2) == call(_cache(be, base), q_token=257) == call(_cache(be, base, row_stride=65)) == -2
    assert call(_cache(be, base, tokens=0)) == 0


def test_verify_entry(be):
    lib, (buf, base) = be._lib.lib(), _memory()

    def call(target=base, dtype=2, requests=2, drafts=3, vocab=10, tokens=base, out=base):
        return lib.b200_verify_tokens(tokens, 3, target, 40, 10, base, 30, 10, base, 4, None, dtype, requests, drafts, vocab, out, base, None)

    assert call(target=None) == call(out=None) == call(tokens=None) == call(drafts=-1) == call(drafts=1025) == call(vocab=0) == call(requests=-1) == -1
    assert call(dtype=5) == -3
    assert call(requests=65536) == call(vocab=(1 << 30) + 1) == -6
    assert call(requests=0) == 0


def test_no_cpu_path(be):
    x, pos, inv = torch.zeros(2, 4, 64).half(), torch.zeros(2, dtype=torch.int32), torch.zeros(32)
    pages = torch.zeros(4, 2, 16, 64).half()
    table, n, starts = torch.zeros(1, 2, dtype=torch.int32), torch.ones(1, dtype=torch.int32), torch.zeros(2, dtype=torch.int32)
    for call in (lambda: be.rope.rotate(x, pos, inv), lambda: be.paged.append(x, x[:, :2], x[:, :2], pages, pages, table, n, starts, inv),
                 lambda: be.paged.attention(x, pages, pages, table, n, starts), lambda: be.verify_tokens(table, torch.zeros(1, 3, 8), torch.zeros(1, 3))):
        with pytest.raises(be._lib.B200Error, match="CUDA"):
            call()


def test_scalings_that_are_not_known_are_refused(be):
    yarn = dict(type="yarn", factor=4.0, original_max_position_embeddings=4096)
    assert be.rope.frequencies(64, 1e4, yarn)[2] > 1.0
    for bad in (dict(type="linear"), dict(type="linear", factor=0.0), dict(type="llama3"), dict(type="llama3", factor=8.0, low_freq_factor=4.0),
                dict(type="yarn", factor=4.0), dict(yarn, factor=-1.0), dict(yarn, mscale=0.7), dict(yarn, truncate=False), dict(type="longrope", factor=2.0)):
        with pytest.raises(be._lib.B200Error):
            be.rope.frequencies(64, 1e4, bad)
    with pytest.raises(be._lib.B200Error):
        be.rope.frequencies(64, 1.0, yarn)


def test_pages_of_the_pool_are_handed_out_once(be):
    cache = be.PagedKVCache(1, 6, 16, 2, 64, device="cpu")
    a, b = cache.take(33), cache.take(1)
    assert len(a) == 3 and len(b) == 1 and not set(a) & set(b) and cache.free == 2
    with pytest.raises(be._lib.B200Error):
        cache.take(33)
    assert cache.take(0) == []
    cache.give(a)
    assert cache.free == 5
    for pages in (a, [b[0], b[0]], [99]):
        with pytest.raises(be._lib.B200Error):
            cache.give(pages)
    assert cache.layer(0)[0].shape == (6, 2, 16, 64)


def test_the_error_word_is_found_however_its_device_is_named(be, monkeypatch):
    monkeypatch.setattr(be.paged, "_errors", {0: torch.tensor([31], dtype=torch.int32), 1: torch.tensor([0], dtype=torch.int32)})
    for current, words in ((0, 31), (1, 0)):
        monkeypatch.setattr(torch.cuda, "current_device", lambda: current)
        assert be.paged.attention_error("cuda") == be.paged.attention_error(torch.device("cuda")) == words
    for name in (0, "cuda:0", torch.device("cuda", 0)):
        assert be.paged.attention_error(name) == 31
    assert be.paged.attention_error("cuda:1") == be.paged.attention_error("cuda:2") == 0
    assert be.paged.attention_error(0, clear=True) == 31 and be.paged.attention_error(0) == 0
    monkeypatch.setattr(be.paged, "_errors", {})
    assert be.paged.attention_error("cuda") == 0


def test_a_page_of_more_rows_than_are_counted_is_refused(be):
    """Also where no table makes more of them."""
    lib, (buf, base) = be._lib.lib(), _memory()
    c = _cache(be, base, page_size=(1 << 30) + 128, table_width=0, page_table=None)
    assert lib.b200_paged_attention(ctypes.byref(c), base, 256, 64, base, 256, 64, base, 5, None, 0.125, base, 1 << 40, base, None) == -6
