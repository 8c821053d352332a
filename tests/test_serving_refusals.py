"""not-gpu: what the serving operators refuse, on the host before any launch (C-ABI with addresses that are never used), the page bookkeeping of
PagedKVCache, and that there is no CPU path."""
import pytest
import torch

from dsrg_amd import _lib, kernels as K
from dsrg_amd._lib import DsrgHipError


def _cache(**kw):
    a = dict(k_pool=64, v_pool=64, k_scale=None, v_scale=None, n_pages=4, page_size=32, n_kv_heads=2, head_dim=64, dtype=_lib.BF16)
    a.update(kw)
    c = _lib.KvCache()
    for k, v in a.items():
        setattr(c, k, v)
    return c


BAD = [(dict(k_pool=None), b'NULL'), (dict(dtype=7), b'dtype'), (dict(head_dim=96), b'head dim'), (dict(page_size=48), b'page size'), (dict(page_size=16), b'page size'),
       (dict(n_pages=0), b'pages'), (dict(n_kv_heads=0), b'heads'), (dict(dtype=_lib.I8), b'scale'), (dict(k_scale=64, v_scale=64), b'scale'), (dict(v_pool=72), b'aligned'),
       (dict(dtype=_lib.E4M3, k_scale=64), b'scale')]


@pytest.mark.parametrize('kw,word', BAD)
def test_bad_caches(kw, word):
    lib, c = _lib.load(), _cache(**kw)
    for rc in (lib.dsrg_kv_append(c, 64, 128, 128, 64, 128, 128, _lib.BF16, 64, 4, 4, 64, None, 1, 1, None),
               lib.dsrg_kv_read(c, 64, 128, 128, 64, 128, 128, _lib.BF16, 64, 4, 4, 64, 64, 1, 1, None),
               lib.dsrg_attention_paged(c, 64, 128, 128, 64, 128, 128, None, 64, 4, 4, 64, 1, 2, 1, 0.125, 0, 0, None, 0, _lib.BF16, None),
               lib.dsrg_attention_paged_workspace(c, 4, 1, 2, 1, 0)):
        assert rc == -1 and word in lib.dsrg_last_error()


def test_append_and_read_refusals():
    lib, c = _lib.load(), _cache()

    def app(k=64, kb=128, kr=128, dt=_lib.BF16, table=64, ld=4, width=4, start=64, B=1, T=1, cache=c):
        return lib.dsrg_kv_append(cache, k, kb, kr, 64, 128, 128, dt, table, ld, width, start, None, B, T, None)

    def read(k=64, kb=128, kr=128, dt=_lib.BF16, table=64, ld=4, width=4, count=64, B=1, n=1, cache=c):
        return lib.dsrg_kv_read(cache, k, kb, kr, 64, 128, 128, dt, table, ld, width, 64, count, B, n, None)

    assert app(B=0) == 0 and app(T=0) == 0 and read(B=0) == 0 and read(n=0) == 0          # nothing to do: no launch
    for f in (app, read):
        assert f(k=None) == -1 and f(B=-1) == -1 and f(table=None) == -1 and f(width=0) == -1 and f(ld=2, B=2) == -1
        assert f(dt=_lib.F32) == -1 and b'dtype' in lib.dsrg_last_error()
        assert f(dt=_lib.I8) == -1
        assert f(k=66) == -1 and b'aligned' in lib.dsrg_last_error()
        assert f(kr=129) == -1 and f(kb=4) == -1
        assert f(width=(1 << 25) + 1) == -1 and b'table' in lib.dsrg_last_error()
        assert f(B=70000, T=8) == -1 if f is app else f(B=70000) == -1
    assert app(start=None) == -1 and read(count=None) == -1 and app(T=-3) == -1 and read(n=-3) == -1


def test_attention_refusals():
    lib, c = _lib.load(), _cache()

    def att(q=64, qr=128, nh=2, Nq=1, causal=0, window=0, ws=None, wsb=0, dt=_lib.BF16, B=1, width=4, lens=64, table=64, cache=c):
        return lib.dsrg_attention_paged(cache, q, 128, qr, 64, 128, 128, None, table, width, width, lens, B, nh, Nq, 0.125, causal, window, ws, wsb, dt, None)

    assert att(B=0) == 0 and att(Nq=0) == 0
    assert att(nh=3) == -1 and b'heads' in lib.dsrg_last_error()
    assert att(dt=_lib.F32) == -1 and b'dtype' in lib.dsrg_last_error()
    assert att(dt=_lib.BF16, cache=_cache(dtype=_lib.F32)) == -1
    assert att(window=5) == -1 and b'causal' in lib.dsrg_last_error()
    assert att(causal=1, window=-5) == -1
    assert att(q=None) == -1 and att(lens=None) == -1 and att(table=None) == -1 and att(B=-2) == -1 and att(Nq=-1) == -1 and att(B=70000) == -1
    assert att(q=72) == -1 and att(qr=132) == -1 and b'aligned' in lib.dsrg_last_error()
    need = lib.dsrg_attention_paged_workspace(c, 4000, 1, 2, 1, 0)
    assert need > 0
    assert att(width=4000) == -1 and b'workspace' in lib.dsrg_last_error()
    assert att(width=4000, ws=64, wsb=need - 1) == -1 and att(width=4000, ws=65, wsb=need) == -1
    # a short window needs no split, however long the table
    assert lib.dsrg_attention_paged_workspace(c, 4000, 1, 2, 1, 32) == 0
    assert lib.dsrg_attention_paged_workspace(c, 4000, 0, 2, 1, 0) == 0
    assert lib.dsrg_attention_paged_workspace(c, 0, 1, 2, 1, 0) == -1
    assert lib.dsrg_attention_paged_workspace(c, 4, 1, 2, 1 << 21, 0) == -1


def test_sample_refusals():
    lib = _lib.load()

    def s(logits=64, ld=100, dt=_lib.F32, u=64, T=1.0, k=0, p=1.0, m=0.0, token=64, logp=64, B=2, V=100):
        return lib.dsrg_sample_rows(logits, ld, dt, u, None, T, None, k, None, p, None, m, token, logp, B, V, None)

    assert s(B=0) == 0
    assert s(dt=_lib.I8) == -1 and s(V=0) == -1 and s(V=(1 << 19) + 1, ld=1 << 20) == -1 and s(B=-1) == -1
    assert s(logits=None) == -1 and s(u=None) == -1 and s(token=None) == -1 and s(logp=None) == -1 and s(ld=99) == -1
    nan, inf = float('nan'), float('inf')
    for bad, word in ((dict(T=-1.0), b'temperature'), (dict(T=nan), b'temperature'), (dict(T=inf), b'temperature'), (dict(k=-1), b'top_k'), (dict(p=-0.5), b'top_p'),
                      (dict(p=nan), b'top_p'), (dict(m=1.5), b'min_p'), (dict(m=-0.1), b'min_p'), (dict(m=nan), b'min_p')):
        assert s(**bad) == -1 and word in lib.dsrg_last_error()


def test_page_bookkeeping_and_shapes():
    from dsrg_amd.kvcache import PagedKVCache
    c = PagedKVCache(6, 2, 64, device='cpu', dtype=torch.int8)
    assert c.k_pool.shape == (6, 2, 2, 8, 16, 8) and c.v_pool.shape == (6, 2, 1, 4, 4, 16, 2, 4) and c.k_scale.shape == (6, 2, 32)
    t = c.table([33, 0, 64])
    assert t.shape == (3, 2) and t.dtype == torch.int32 and (t[1] == -1).all() and (t[[0, 2]] >= 0).all() and t[[0, 2]].unique().numel() == 4 and c.free_pages == 2
    with pytest.raises(DsrgHipError, match='free'):
        c.table([97])
    assert c.free_pages == 2
    with pytest.raises(DsrgHipError, match='negative'):
        c.table([-1])
    c.release(t[:1])
    assert c.free_pages == 4
    for again in (t[:1], t[[2, 2]], torch.tensor([[6]])):
        with pytest.raises(DsrgHipError, match='not taken'):
            c.release(again)
    c.release(t[1:])
    assert c.free_pages == 6 and c.table([]).shape == (0, 1)
    f = PagedKVCache(2, 1, 128, device='cpu', dtype=torch.float32, page_size=64)
    assert f.k_pool.shape == (2, 1, 4, 32, 16, 4) and f.v_pool.shape == (2, 1, 4, 8, 4, 16, 4) and f.k_scale is None
    for kw in (dict(page_size=48), dict(head_dim=80), dict(dtype=torch.float16), dict(n_pages=0), dict(n_kv_heads=0)):
        with pytest.raises(DsrgHipError):
            PagedKVCache(**{**dict(n_pages=2, n_kv_heads=1, head_dim=64, device='cpu'), **kw})


@pytest.mark.skipif(torch.cuda.is_available(), reason='CPU-only check')
def test_no_cpu_path():
    from dsrg_amd.kvcache import PagedKVCache
    c = PagedKVCache(2, 1, 64, device='cpu')
    x, i, t = torch.zeros(1, 1, 64, dtype=torch.bfloat16), torch.zeros(1, dtype=torch.int32), torch.zeros(1, 1, dtype=torch.int32)
    for call in (lambda: c.append(x, x, t, i), lambda: c.read(t, i, i, 1), lambda: c.attend(x, t, i, 1), lambda: K.sample_rows(torch.zeros(1, 4), torch.zeros(1))):
        with pytest.raises(DsrgHipError, match='device tensors'):
            call()
    with pytest.raises(DsrgHipError, match='no backward'):
        c.attend(x.requires_grad_(), t, i, 1)


def test_inputs_that_ask_for_a_gradient():
    """no serving operator has a backward: such an input is refused (before any other look at it), not detached; under no_grad it is one like any other"""
    ks, vs = K.kv_pool_shapes(2, 32, 1, 64, torch.bfloat16)
    kp, vp = torch.zeros(ks, dtype=torch.bfloat16), torch.zeros(vs, dtype=torch.bfloat16)
    x, i, t = torch.zeros(1, 1, 64, dtype=torch.bfloat16), torch.zeros(1, dtype=torch.int32), torch.zeros(1, 1, dtype=torch.int32)
    r, one = x.clone().requires_grad_(), torch.ones(1)
    grad = lambda y: y.clone().requires_grad_()          # noqa: E731
    calls = [('k', lambda: K.kv_append(r, x, kp, vp, t, i)), ('v', lambda: K.kv_append(x, r, kp, vp, t, i)), ('q', lambda: K.attention_paged(r, kp, vp, t, i, 1)),
             ('k_pool', lambda: K.attention_paged(x, grad(kp), vp, t, i, 1)), ('v_pool', lambda: K.kv_read(kp, grad(vp), t, i, i, 1)),
             ('logits', lambda: K.sample_rows(grad(torch.zeros(1, 4)), one)), ('temperature', lambda: K.sample_rows(torch.zeros(1, 4), one, grad(one))),
             ('top_p', lambda: K.sample_rows(torch.zeros(1, 4), one, top_p=grad(one))), ('min_p', lambda: K.sample_rows(torch.zeros(1, 4), one, min_p=grad(one)))]
    for name, call in calls:
        with pytest.raises(DsrgHipError, match='no backward and %s asks' % name):
            call()
        if not torch.cuda.is_available():
            with torch.no_grad(), pytest.raises(DsrgHipError, match='device tensors'):
                call()


def test_pages_too_large_are_refused_where_the_pools_are_made():
    """the kernels take pages of up to 65536 tokens: a larger cache could be made and then not used"""
    from dsrg_amd.kvcache import PagedKVCache
    assert _lib.load().dsrg_attention_paged_workspace(_cache(page_size=1 << 16), 4, 1, 2, 1, 0) >= 0
    assert _lib.load().dsrg_attention_paged_workspace(_cache(page_size=1 << 17), 4, 1, 2, 1, 0) == -1 and b'65536' in _lib.load().dsrg_last_error()
    assert K.kv_pool_shapes(1, 1 << 16, 1, 64, torch.int8)[0] == (1, 1, 4096, 8, 16, 8)
    for f in (lambda: K.kv_pool_shapes(1, 1 << 17, 1, 64, torch.int8), lambda: PagedKVCache(1, 1, 64, device='cpu', dtype=torch.int8, page_size=1 << 17)):
        with pytest.raises(DsrgHipError, match='65536'):
            f()
