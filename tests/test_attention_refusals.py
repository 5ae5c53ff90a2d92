"""The paged attention, append, page copy and sampling entries refuse what they do not take, with
a reason, before they look at the device (no GPU needed)."""
import ctypes as C

import numpy as np
import pytest

from sabrewing_amd import backend as B

A = 1 << 20                                        # an aligned address that nothing reads


@pytest.fixture(scope="module")
def lib():
    return B.load_library()


def cache(**kw):
    d = dict(k=A, v=2 * A, type="bf16", n_pages=4, page_size=16, n_heads=2, head_dim=64)
    strides = kw.pop("strides", None)
    t = kw.pop("raw_type", None)
    d.update(kw)
    c = B.Backend.kv_cache(strides=strides, **d)
    if t is not None:
        c.type = t
    return c


def rows(**kw):
    d = dict(pos_dev=A, table_dev=A, n_seqs=8, max_pages=4, seq_dev=None)
    d.update(kw)
    return B.Backend.kv_rows(**d)


def rope_call(lib, c=None, r=None, rope=None, qkv=A, ld=512, Hq=4, q_out=64 * A, S=3):
    return lib.lag_hip_qk_rope_append(c or cache(), r or rows(), rope, qkv, ld, None, None, 1e-6, Hq, q_out, S)


def attn_call(lib, c=None, r=None, q=A, Hq=4, window=0, out=64 * A, S=3):
    return lib.lag_hip_attn_paged(c or cache(), r or rows(), q, Hq, 0.125, window, out, S)


def refused(lib, rc, word):
    assert rc == -1
    msg = lib.lag_hip_last_error().decode()
    assert word in msg, msg


BAD_CACHES = [
    (dict(k=0), "no pools"), (dict(v=0), "no pools"), (dict(raw_type=3), "type"), (dict(raw_type=-1), "type"),
    (dict(n_pages=0), "count"), (dict(n_heads=0), "count"), (dict(head_dim=0), "head_dim"), (dict(head_dim=48), "head_dim"),
    (dict(head_dim=288), "head_dim"), (dict(page_size=0), "page_size"), (dict(page_size=4), "page_size"),
    (dict(page_size=24), "page_size"), (dict(page_size=8192), "page_size"), (dict(k=A + 8), "16 bytes"),
    (dict(strides=(2048, 1024, 68)), "16 bytes"), (dict(strides=(2048, 1024, 32)), "overlap"),
    (dict(strides=(2048, 512, 64)), "overlap"), (dict(strides=(1024, 1024, 64)), "overlap"),
    (dict(strides=(-2048, 1024, 64)), "overlap"), (dict(strides=(1 << 60, 1024, 64)), "overlap"),
    (dict(strides=(0, 0, 0)), "overlap"),
]


@pytest.mark.parametrize("kw,word", BAD_CACHES)
def test_bad_caches(lib, kw, word):
    c = cache(**kw)
    refused(lib, rope_call(lib, c), word)
    refused(lib, attn_call(lib, c), word)
    one = np.zeros(1, np.int32)
    refused(lib, lib.lag_hip_kv_copy_pages((B.LagHipKvCache * 1)(c), 1, one.ctypes.data, one.ctypes.data, 1), word)


@pytest.mark.parametrize("kw,word", [
    (dict(pos_dev=0), "no positions"), (dict(table_dev=0), "no positions"), (dict(n_seqs=0), "count"), (dict(max_pages=0), "count"),
    (dict(n_seqs=2), "more rows than sequences"), (dict(max_pages=(1 << 26) + 1), "2^30")])
def test_bad_rows(lib, kw, word):
    refused(lib, rope_call(lib, r=rows(**kw)), word)
    refused(lib, attn_call(lib, r=rows(**kw)), word)


def test_bad_append(lib):
    for kw, word in [(dict(qkv=0), "aligned"), (dict(qkv=A + 4), "aligned"), (dict(q_out=0), "aligned"), (dict(ld=514), "aligned"),
                     (dict(q_out=64 * A + 8), "aligned"), (dict(Hq=3), "n_q_heads"), (dict(Hq=0), "n_q_heads"), (dict(Hq=2048), "n_q_heads"),
                     (dict(ld=508), "ld"), (dict(S=0), "count"), (dict(S=-1), "count"), (dict(q_out=A), "overlap"),
                     (dict(q_out=A + 512 * 4 * 3 - 16), "overlap"), (dict(rope=B.LagHipRope(A, 66, 0, 1.0)), "rope"),
                     (dict(rope=B.LagHipRope(A, 31, 0, 1.0)), "rope"), (dict(rope=B.LagHipRope(A, -2, 0, 1.0)), "rope"),
                     (dict(rope=B.LagHipRope(None, 64, 0, 1.0)), "rope")]:
        refused(lib, rope_call(lib, **kw), word)


def test_bad_attention(lib):
    for kw, word in [(dict(q=0), "aligned"), (dict(q=A + 4), "aligned"), (dict(out=0), "aligned"), (dict(Hq=5), "n_q_heads"),
                     (dict(window=-1), "window"), (dict(S=0), "count"), (dict(out=A), "overlap"),
                     (dict(out=A + 3 * 4 * 64 * 4 - 16), "overlap"), (dict(out=A - 16), "overlap")]:
        refused(lib, attn_call(lib, **kw), word)


def copy_call(lib, src, dst, layers=None, n=None):
    s, d = np.asarray(src, np.int32), np.asarray(dst, np.int32)
    layers = layers or [cache(), cache(k=3 * A, v=4 * A)]
    arr = (B.LagHipKvCache * len(layers))(*layers)
    return lib.lag_hip_kv_copy_pages(arr, len(layers), s.ctypes.data, d.ctypes.data, len(src) if n is None else n)


def test_bad_copies(lib):
    for src, dst, word in [([0], [4], "outside"), ([4], [0], "outside"), ([-1], [0], "outside"), ([0], [-1], "outside"),
                           ([0, 0], [1, 1], "twice"), ([0, 1], [1, 2], "source"), ([1], [1], "source"),
                           ([0, 1], [2, 0], "source"), ([0] * 5, [1, 2, 3, 1, 2], "twice")]:
        refused(lib, copy_call(lib, src, dst), word)
    refused(lib, copy_call(lib, [0], [1], n=-1), "no layers")
    refused(lib, copy_call(lib, [0], [1], layers=[cache(), cache(page_size=32)]), "geometry")
    refused(lib, copy_call(lib, [0], [1], layers=[cache(), cache(raw_type=2)]), "geometry")
    assert lib.lag_hip_kv_copy_pages(None, 1, None, None, 0) == -1
    with pytest.raises(ValueError):
        B.Backend.kv_copy_pages(None, None, [0, 1], [2])


def test_bad_sampling(lib):
    for args, word in [((0, 2, 8, None, A, A), "no logits"), ((A, 0, 8, None, A, A), "no logits"), ((A, 2, 0, None, A, A), "no logits"),
                       ((A, 2, 8, None, 0, A), "no logits"), ((A, 2, 8, None, A, 0), "no logits"),
                       ((A, 1, (1 << 20) + 1, None, A, A), "2^20")]:
        refused(lib, lib.lag_hip_sample(*args), word)


def test_bad_sums(lib):
    for args, word in [((0, A, 8), "no values"), ((A, 0, 8), "no values"), ((A, 2 * A, 0), "no values"), ((A, A + 4, 8), "overlap"), ((A, A - 28, 8), "overlap")]:
        lib.lag_hip_sample(0, 1, 1, None, A, A)        # (leaves another reason)
        refused(lib, lib.lag_hip_add(*args), word)
    if not lib.lag_hip_alloc(16):                      # (none is initialised in this process)
        for args in [(A, A, 8), (A, A + 32, 8), (A + 32, A, 8)]:
            refused(lib, lib.lag_hip_add(*args), "not initialised")


def test_good_arguments_reach_the_device(lib):
    """the same calls with nothing wrong are refused for want of a device alone (run where none is initialised)"""
    if lib.lag_hip_alloc(16):
        pytest.skip("a device is initialised in this process")
    ok = [rope_call(lib), attn_call(lib), copy_call(lib, [0, 0, 1], [2, 3], n=2), lib.lag_hip_sample(A, 2, 1 << 20, None, A, A),
          attn_call(lib, c=cache(strides=(2048, 64, 128))), attn_call(lib, c=cache(strides=(64, 4096, 256))),
          attn_call(lib, c=cache(n_heads=1, strides=(1024, 0, 64)))]
    assert ok == [-1] * len(ok)
    assert "not initialised" in lib.lag_hip_last_error().decode()
    for f in (lambda: rope_call(lib), lambda: attn_call(lib), lambda: copy_call(lib, [0], [1])):
        refused(lib, f(), "not initialised")


def test_too_many_cells(lib):
    """64 rows of tables of 2^30 cells are refused, one is not"""
    r = dict(n_seqs=64, max_pages=1 << 26)
    refused(lib, attn_call(lib, r=rows(**r), S=64, out=1024 * A), "2^30")
    assert attn_call(lib, r=rows(**r), S=1) == -1 and "2^30" not in lib.lag_hip_last_error().decode()


def test_cells_that_round_up_to_too_many(lib):
    """a row of 2^30 - 8 cells is 2^26 chunks where they are of 16 tokens, and 64 such rows no number of 32 bits; one page
    less is, and so are chunks of 32"""
    if lib.lag_hip_alloc(16):
        pytest.skip("a device is initialised in this process")
    n, out = 1 << 27, 1024 * A
    for kw in (dict(type="f32", head_dim=64), dict(type="f16", head_dim=192), dict(type="bf16", head_dim=192)):
        c = cache(page_size=8, **kw)
        refused(lib, attn_call(lib, c, rows(n_seqs=64, max_pages=n - 1), S=64, out=out), "2^30")
        refused(lib, attn_call(lib, c, rows(n_seqs=300, max_pages=n - 1), S=300, out=out), "2^30")
        for S, pages in ((64, n - 2), (63, n - 1), (1, n)):
            assert attn_call(lib, c, rows(n_seqs=64, max_pages=pages), S=S, out=out) == -1
            assert "2^30" not in lib.lag_hip_last_error().decode()
    assert attn_call(lib, cache(page_size=8), rows(n_seqs=64, max_pages=n - 1), S=64, out=out) == -1
    assert "2^30" not in lib.lag_hip_last_error().decode()
