"""What a stack with attention refuses, and what it keeps, before anything runs on the device: every call of
the stand-in below records itself and computes nothing."""
import numpy as np
import pytest

from sabrewing_amd import configs as cf
from sabrewing_amd.attention import AttnConfig, DeviceAttention, PagedCache, Rope
from sabrewing_amd.backend import Backend
from sabrewing_amd.stack import DeviceStack


class Buf:
    def __init__(self, addr):
        self.addr, self.freed = addr, False

    def __int__(self):
        assert not self.freed
        return self.addr

    def free(self):
        self.freed = True


class Recorder:
    kv_cache, kv_caches, kv_rows, rope = (staticmethod(getattr(Backend, n)) for n in ("kv_cache", "kv_caches", "kv_rows", "rope"))

    def __init__(self):
        self.next, self.calls, self.bufs = 4096, [], []

    def alloc(self, n):
        self.bufs.append(Buf(self.next))
        self.next += n + 4096
        return self.bufs[-1]

    def upload(self, a):
        return self.alloc(np.asarray(a).nbytes)

    def router_upload(self, a, bf16):
        return self.upload(a)

    def __getattr__(self, name):
        return lambda *a: self.calls.append(name)


class Layer:
    def weights(self):
        return None

    def free(self):
        pass


A = AttnConfig(4, 2, 32, 32)


def attention(be, acfg, D, rope):
    u16, f32 = (lambda *s: np.zeros(s, np.uint16)), (lambda *s: np.ones(s, np.float32))
    return DeviceAttention.from_host(be, acfg, D, f32(D), u16(acfg.qkv_rows, D), u16(D, acfg.n_q * acfg.head_dim),
                                     f32(acfg.head_dim), f32(acfg.head_dim), rope)


def stack(be, acfgs, D=None):
    cfg = cf.scaled(cf.C5_LAYER, D=512, E=32, K=8, I=384)
    st = DeviceStack(be, cfg, 1000)
    st.layers, st.norms = [Layer() for _ in acfgs], [be.alloc(4 * cfg.D) for _ in acfgs]
    st.final_norm, st.head = be.alloc(4), be.alloc(4)
    rope = Rope(be, acfgs[0])
    return st.add_attention(acfgs[0], [attention(be, a, D or cfg.D, rope) for a in acfgs])


def step(be, st, cache, rows, S):
    st.step(be.alloc(4), be.alloc(4), be.alloc(4), be.alloc(4), S, cache=cache, rows=rows)


def test_steps_that_do_not_fit():
    be = Recorder()
    st = stack(be, [A, A])
    cache = PagedCache(be, 2, 8, 8, 2, 32, max_seqs=3)
    step(be, st, cache, cache.desc, 3)
    assert be.calls.count("attn_paged") == 2
    for bad in (PagedCache(be, 2, 8, 8, 1, 32, max_seqs=3), PagedCache(be, 2, 8, 8, 2, 64, max_seqs=3), PagedCache(be, 1, 8, 8, 2, 32), None):
        be.calls.clear()
        with pytest.raises(ValueError):
            step(be, st, bad, cache.desc, 3)
        assert not be.calls
    with pytest.raises(ValueError):
        step(be, st, cache, cache.desc, 4)             # the row arrays end at three
    with pytest.raises(ValueError):
        step(be, st, cache, None, 3)
    # layers whose heads, or width, are not the first one's
    for acfgs, D in (([A, AttnConfig(8, 2, 32, 32)], None), ([A, AttnConfig(4, 4, 32, 32)], None), ([A, A], 640)):
        with pytest.raises(ValueError):
            step(be, stack(be, acfgs, D), cache, cache.desc, 2)
    step(be, stack(be, [A, AttnConfig(4, 2, 32, 32, window=8)]), cache, cache.desc, 2)


def test_attention_is_added_once():
    be = Recorder()
    st = stack(be, [A])
    with pytest.raises(ValueError):
        st.add_attention(A, st.attn)
    st2 = DeviceStack(be, st.cfg, 10)
    st2.layers = [Layer(), Layer()]
    with pytest.raises(ValueError):
        st2.add_attention(A, st.attn)
    assert not st2.attn


def test_scratch_outlives_its_growth():
    """a recorded step of three rows goes on replaying over its scratch after a step of five"""
    be = Recorder()
    st = stack(be, [A])
    cache = PagedCache(be, 1, 8, 8, 2, 32, max_seqs=8)
    step(be, st, cache, cache.desc, 3)
    old = st.scratch
    step(be, st, cache, cache.desc, 5)
    assert st.scratch is not old and not any(b.freed for b in (old.qkv, old.q, old.ctx, old.out))
    step(be, st, cache, cache.desc, 2)
    new = st.scratch
    st.free()
    assert all(b.freed for s in (old, new) for b in (s.qkv, s.q, s.ctx, s.out))


@pytest.mark.parametrize("second,D", [(AttnConfig(8, 2, 32, 32), None), (AttnConfig(4, 4, 32, 32), None), (AttnConfig(4, 2, 64, 32), None),
                                      (A, 640)], ids=str)
def test_layers_of_other_shapes_run_nothing(second, D):
    """they are refused before a first layer has changed h or appended its keys and values"""
    be = Recorder()
    cache = PagedCache(be, 2, 8, 8, 2, 32, max_seqs=3)
    cfg = cf.scaled(cf.C5_LAYER, D=512, E=32, K=8, I=384)
    rope = Rope(be, A)
    layers = [attention(be, A, D or cfg.D, rope), attention(be, second, D or cfg.D, rope)]
    st = DeviceStack(be, cfg, 1000)
    st.layers, st.norms = [Layer(), Layer()], [be.alloc(4 * cfg.D) for _ in range(2)]
    st.final_norm, st.head = be.alloc(4), be.alloc(4)
    be.calls.clear()
    with pytest.raises(ValueError):
        st.add_attention(A, layers)
        step(be, st, cache, cache.desc, 2)
    assert not be.calls
