"""The entries for trees of drafted tokens and for latent attention refuse what they do not take, with a reason, before they look at the
device (no GPU needed)."""
import pytest

from sabrewing_amd import backend as B
from test_attention_refusals import A, BAD_CACHES, cache, lib, refused, rows  # noqa: F401  (lib: the fixture)

FAR = 1 << 36


def trees(**kw):
    d = dict(first_dev=A, base_dev=2 * A, sees_dev=3 * A, table_dev=4 * A, n_trees=2, n_seqs=8, max_pages=4, max_nodes=16, seq_dev=5 * A, pos_dev=6 * A)
    d.update(kw)
    return B.Backend.trees(**d)


def tree_call(lib, c=None, t=None, q=FAR, Hq=4, window=0, out=2 * FAR, S=3):
    return lib.lag_hip_attn_tree(c or cache(), t or trees(), q, Hq, 0.125, window, out, S)


def at_call(lib, c=None, r=None, at=A, qkv=FAR, q_out=2 * FAR, S=3):
    return lib.lag_hip_qk_rope_append_at(c or cache(), r or rows(), at, None, qkv, 512, None, None, 1e-6, 4, q_out, S)


def commit_call(lib, layers=None, t=None, parent=7 * A, draft=8 * A, tok=9 * A, path=10 * A, count=11 * A, nxt=12 * A, S=3):
    layers = layers or [cache(), cache(k=3 * A, v=4 * A)]
    return lib.lag_hip_tree_commit((B.LagHipKvCache * len(layers))(*layers), len(layers), t or trees(), parent, draft, tok, path, count, nxt, S)


@pytest.mark.parametrize("kw,word", BAD_CACHES)
def test_bad_caches(lib, kw, word):
    c = cache(**kw)
    refused(lib, tree_call(lib, c), word)
    refused(lib, at_call(lib, c), word)
    refused(lib, commit_call(lib, [c]), word)


@pytest.mark.parametrize("kw,word", [
    (dict(first_dev=0), "no rows"), (dict(base_dev=0), "no rows"), (dict(table_dev=0), "no rows"), (dict(n_trees=0), "count"), (dict(n_trees=-1), "count"),
    (dict(n_trees=65536), "count"), (dict(n_seqs=0), "count"), (dict(max_pages=0), "count"), (dict(max_nodes=0), "max_nodes"), (dict(max_nodes=65), "max_nodes"),
    (dict(seq_dev=None, n_trees=9), "more trees"), (dict(max_pages=(1 << 26) + 1), "2^30")])
def test_bad_trees(lib, kw, word):
    refused(lib, tree_call(lib, t=trees(**kw)), word)
    refused(lib, commit_call(lib, t=trees(**kw)), word)


def test_bad_tree_attention(lib):
    n = 3 * 4 * 64 * 4
    for kw, word in [(dict(q=0), "aligned"), (dict(q=FAR + 4), "aligned"), (dict(out=0), "aligned"), (dict(out=2 * FAR + 8), "aligned"), (dict(Hq=5), "n_q_heads"),
                     (dict(Hq=0), "n_q_heads"), (dict(Hq=2048), "n_q_heads"), (dict(window=-1), "window"), (dict(S=0), "count"), (dict(out=FAR), "overlap"),
                     (dict(out=FAR + n - 16), "overlap"), (dict(out=FAR - n + 16), "overlap"), (dict(t=trees(sees_dev=None)), "attend"),
                     (dict(t=trees(pos_dev=None), window=5), "positions")]:
        refused(lib, tree_call(lib, **kw), word)
    assert lib.lag_hip_attn_tree(None, trees(), FAR, 4, 0.1, 0, 2 * FAR, 3) == -1
    assert lib.lag_hip_attn_tree(cache(), None, FAR, 4, 0.1, 0, 2 * FAR, 3) == -1
    refused(lib, at_call(lib, at=0), "positions")


def test_bad_commits(lib):
    for kw, word in [(dict(parent=0), "no parents"), (dict(draft=0), "no parents"), (dict(tok=0), "no parents"), (dict(path=0), "no place"), (dict(count=0), "no place"),
                     (dict(nxt=0), "no place"), (dict(S=0), "count"), (dict(path=7 * A), "overlap"), (dict(path=7 * A - 124), "overlap"), (dict(count=8 * A + 8), "overlap"),
                     (dict(nxt=A + 8), "overlap"), (dict(count=2 * A + 4), "overlap"), (dict(count=10 * A + 124), "overlap"), (dict(nxt=11 * A + 4), "overlap")]:
        refused(lib, commit_call(lib, **kw), word)
    refused(lib, commit_call(lib, [cache(), cache(page_size=32)]), "geometry")
    refused(lib, lib.lag_hip_tree_commit(None, 1, trees(), A, A, A, A, A, A, 3), "no layers")


def latents(**kw):
    d = dict(c=A, type="bf16", n_pages=4, page_size=16, rank=128, rope_dims=64)
    strides, t = kw.pop("strides", None), kw.pop("raw_type", None)
    d.update(kw)
    c = B.Backend.latent_cache(strides=strides, **d)
    if t is not None:
        c.type = t
    return c


heads = B.Backend.heads


def append_call(lib, c=None, r=None, rope=B.LagHipRope(A, 64, 0, 1.0), ckv=FAR, ld_c=192, q=2 * FAR, ld_q=384, H=4, nope=32, qn=heads(3 * FAR, 768, 192),
                qr=heads(3 * FAR + 256, 768, 192), S=3):
    return lib.lag_hip_latent_append(c or latents(), r or rows(), rope, ckv, ld_c, None, 1e-6, q, ld_q, H, nope, qn, qr, S)


def heads_call(lib, type=B.KV_TYPES["bf16"], x=heads(A, 512, 128), W=FAR, H=4, n_in=128, n_out=64, y=heads(2 * FAR, 256, 64), f32=0, S=3):
    return lib.lag_hip_latent_heads(type, x, W, H, n_in, n_out, y, f32, S)


def latent_call(lib, c=None, r=None, q=FAR, H=4, out=2 * FAR, S=3):
    return lib.lag_hip_attn_latent(c or latents(), r or rows(), q, H, 0.1, out, S)


def prompt_call(lib, c=None, pages=A, n=4, start=5, wk=FAR, wv=2 * FAR, nope=64, vd=64, q=3 * FAR, H=4, out=4 * FAR, f32=0, S=3):
    return lib.lag_hip_attn_latent_prompt(c or latents(), pages, n, start, wk, wv, nope, vd, q, H, 0.1, out, f32, S)


@pytest.mark.parametrize("kw,word", [
    (dict(c=0), "no pool"), (dict(raw_type=0), "type"), (dict(raw_type=3), "type"), (dict(n_pages=0), "page count"), (dict(page_size=4), "page_size"),
    (dict(page_size=24), "page_size"), (dict(page_size=8192), "page_size"), (dict(rank=64), "rank"), (dict(rank=640), "rank"), (dict(rank=200), "rank"),
    (dict(rope_dims=8), "rope_dims"), (dict(rope_dims=80), "rope_dims"), (dict(rope_dims=-16), "rope_dims"), (dict(c=A + 8), "16 bytes"),
    (dict(strides=(4096, 196)), "16 bytes"), (dict(strides=(4096, 184)), "overlap"), (dict(strides=(3064, 192)), "overlap"), (dict(strides=(-4096, 192)), "overlap"),
    (dict(strides=(1 << 60, 192)), "overlap"), (dict(strides=(184, 4096)), "overlap")])
def test_bad_latent_caches(lib, kw, word):
    c = latents(**kw)
    for call in (append_call, latent_call, prompt_call):
        refused(lib, call(lib, c), word)


def test_bad_latent_rows(lib):
    for kw, word in [(dict(pos_dev=0), "no positions"), (dict(table_dev=0), "no positions"), (dict(n_seqs=0), "count"), (dict(max_pages=0), "count"),
                     (dict(n_seqs=2), "more rows"), (dict(max_pages=(1 << 26) + 1), "2^30")]:
        refused(lib, append_call(lib, r=rows(**kw)), word)
        refused(lib, latent_call(lib, r=rows(**kw)), word)


def test_bad_latent_appends(lib):
    for kw, word in [(dict(ckv=0), "ckv"), (dict(ckv=FAR + 4), "ckv"), (dict(ld_c=194), "ckv"), (dict(ld_c=188), "ld_c"), (dict(rope=B.LagHipRope(A, 32, 0, 1.0)), "rope"),
                     (dict(rope=B.LagHipRope(None, 64, 0, 1.0)), "rope"), (dict(H=-1), "n_heads"), (dict(H=1025), "n_heads"), (dict(nope=24), "nope"), (dict(nope=0), "nope"),
                     (dict(nope=272), "nope"), (dict(q=0), "q must"), (dict(q=2 * FAR + 8), "q must"), (dict(ld_q=386), "q must"), (dict(ld_q=380), "ld_q"),
                     (dict(qn=None), "no heads"), (dict(qr=None), "no heads"), (dict(qn=heads(3 * FAR + 8, 768, 192)), "16 bytes"), (dict(qn=heads(3 * FAR, 768, 180)), "16 bytes"),
                     (dict(qn=heads(3 * FAR, 768, 24)), "overlap"), (dict(qn=heads(3 * FAR, 600, 192)), "overlap"), (dict(qr=heads(3 * FAR + 48, 768, 192)), "overlap"),
                     (dict(qr=heads(3 * FAR + 256, 1536, 384)), "overlap"), (dict(qn=heads(FAR, 768, 192)), "overlap what"), (dict(qr=heads(2 * FAR + 64, 768, 192)), "overlap what"),
                     (dict(qn=heads(3 * FAR, -768, 192)), "strides"), (dict(S=0), "count")]:
        refused(lib, append_call(lib, **kw), word)


def test_bad_latent_heads(lib):
    for kw, word in [(dict(type=0), "type"), (dict(type=5), "type"), (dict(S=0), "count"), (dict(H=0), "count"), (dict(H=1025), "count"), (dict(n_in=48), "n_in"), (dict(n_in=0), "n_in"),
                     (dict(n_in=1056), "n_in"), (dict(n_out=16), "n_in"), (dict(n_out=1056), "n_in"), (dict(W=0), "W"), (dict(W=FAR + 8), "W"), (dict(x=None), "no heads"),
                     (dict(y=None), "no heads"), (dict(y=heads(2 * FAR, 256, 32)), "overlap"), (dict(y=heads(2 * FAR, 192, 64)), "overlap"), (dict(y=heads(A, 256, 64)), "overlap what"),
                     (dict(y=heads(FAR, 256, 64)), "overlap what"), (dict(y=heads(FAR - 2 * 640, 256, 64)), "overlap what")]:
        refused(lib, heads_call(lib, **kw), word)


def test_bad_latent_attention(lib):
    for kw, word in [(dict(q=0), "aligned"), (dict(q=FAR + 8), "aligned"), (dict(out=0), "aligned"), (dict(H=0), "n_heads"), (dict(H=1025), "n_heads"), (dict(S=0), "count"),
                     (dict(out=FAR), "overlap"), (dict(out=FAR + 3 * 4 * 192 * 2 - 16), "overlap")]:
        refused(lib, latent_call(lib, **kw), word)
    for kw, word in [(dict(pages=0), "no pages"), (dict(n=0), "no pages"), (dict(S=0), "tokens"), (dict(start=-1), "tokens"), (dict(start=(1 << 22) - 2), "tokens"), (dict(H=0), "n_heads"),
                     (dict(H=1025), "n_heads"), (dict(nope=48), "nope"), (dict(nope=288), "nope"), (dict(vd=16), "nope"), (dict(wk=0), "aligned"), (dict(wv=2 * FAR + 8), "aligned"),
                     (dict(q=0), "aligned"), (dict(out=4 * FAR + 8), "aligned"), (dict(out=3 * FAR), "overlap"), (dict(out=FAR), "overlap"), (dict(out=2 * FAR), "overlap")]:
        refused(lib, prompt_call(lib, **kw), word)


def test_good_arguments_reach_the_device(lib):
    if lib.lag_hip_alloc(16):
        pytest.skip("a device is initialised in this process")
    for call in (tree_call, at_call, commit_call, append_call, heads_call, latent_call, prompt_call):
        refused(lib, call(lib), "not initialised")
    for ok in (lambda: tree_call(lib, t=trees(pos_dev=None)), lambda: tree_call(lib, t=trees(seq_dev=None, n_trees=8), window=3),
               lambda: commit_call(lib, t=trees(sees_dev=None, pos_dev=None)), lambda: append_call(lib, H=0, q=None, qn=None, qr=None), lambda: append_call(lib, rope=None),
               lambda: append_call(lib, latents(rope_dims=0), rope=None, qr=None), lambda: heads_call(lib, x=heads(A, 128, 0)),
               lambda: heads_call(lib, y=heads(2 * FAR, 64, 192), f32=1), lambda: latent_call(lib, latents(strides=(192, 1024))),
               lambda: prompt_call(lib, start=(1 << 22) - 3)):
        refused(lib, ok(), "not initialised")
