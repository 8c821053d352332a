"""gpu: the serving operators - paged key / value cache (write with quantisation, read back), attention over it, sampling - against plain
64-bit implementations, at the sizes, masks and orders where they can go wrong.

Tolerances count roundings (half a step relative to the value: bf16 2^-8, fp32 2^-24): _bound() for attention; reads of bf16 / fp32 caches
are exact; 8-bit codes and scales are compared bit for bit with the same IEEE fp32 formula in numpy."""
import math
import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu

F32, BF16, I8, E4M3 = torch.float32, torch.bfloat16, torch.int8, torch.float8_e4m3fn
IO = {F32: F32, BF16: BF16, I8: BF16, E4M3: BF16}


@pytest.fixture(scope='module')
def K():
    assert torch.cuda.is_available(), 'GPU tests need an MI355X'
    from dsrg_amd import kernels
    return kernels


def _g(seed):
    return torch.Generator(device='cpu').manual_seed(seed)


def _fill(t, byte=0xff):
    """every byte of t set: NaN in bf16, fp32 and e4m3, -1 in int8"""
    t.view(torch.uint8).fill_(byte) if t.is_contiguous() else None
    return t


def _cache(K, P, S, H, D, dtype):
    """pools full of bytes that no result may show (NaN patterns), scales NaN"""
    ks, vs = K.kv_pool_shapes(P, S, H, D, dtype)
    c = dict(k_pool=_fill(torch.empty(ks, device='cuda', dtype=dtype)), v_pool=_fill(torch.empty(vs, device='cuda', dtype=dtype)), k_scale=None, v_scale=None)
    if dtype in (I8, E4M3):
        c.update(k_scale=torch.full((P, H, S), float('nan'), device='cuda'), v_scale=torch.full((P, H, S), float('nan'), device='cuda'))
    return c


def _table(B, width, P, seed, spare=1):
    """random distinct pages from `spare` on"""
    return (torch.randperm(P - spare, generator=_g(seed))[:B * width] + spare).to(torch.int32).view(B, width).cuda()


def _i(*v):
    return torch.tensor(v, dtype=torch.int32, device='cuda')


def _stored(x, dtype, H):
    """x [.., H*D] on the CPU -> (codes float32, scale float32 [.., H]) by the documented formula in IEEE fp32, or the values themselves"""
    if dtype in (F32, BF16):
        return x.float(), None
    y = x.float().reshape(*x.shape[:-1], H, -1).numpy()
    most = np.float32(127 if dtype == I8 else 448)
    scale = np.maximum(np.abs(y).max(-1, keepdims=True) * np.float32(1.0 / float(most)), np.float32(2.0 ** -126))
    z = np.clip(y / scale, -most, most)
    codes = np.rint(z) if dtype == I8 else torch.from_numpy(z).to(E4M3).float().numpy()
    return torch.from_numpy(codes.astype(np.float32)).reshape(x.shape), torch.from_numpy(scale[..., 0])


def _rows_from_pool(c, table, b, n, S, D, dtype):
    """tokens 0..n-1 of sequence b from the pools by the documented index formulas -> k, v codes [n, H, D] and scales (CPU)"""
    kp, vp = ((p.view(torch.uint8).cpu().view(E4M3) if dtype == E4M3 else p.cpu()).float() for p in (c['k_pool'], c['v_pool']))
    H, e = kp.shape[1], 4 if dtype == F32 else 8
    pg, r = table[b].cpu().long()[torch.arange(n) // S][:, None, None], (torch.arange(n) % S)[:, None, None]
    h, d = torch.arange(H)[None, :, None], torch.arange(D)[None, None]
    k = kp[pg, h, r // 16, d // e, r % 16, d % e]
    v = vp[pg, h, r // 16, d // 16, r % 16 // 4, d % 16, r % 4] if dtype == F32 else vp[pg, h, r // 32, d // 16, r % 16 // 4, d % 16, r % 32 // 16, r % 4]
    sc = [None if s is None else s.cpu()[pg[..., 0], h[..., 0], r[..., 0]] for s in (c['k_scale'], c['v_scale'])]
    return k, v, sc


@pytest.mark.parametrize('dtype', [BF16, F32, I8, E4M3])
@pytest.mark.parametrize('H,D,S', [(12, 64, 32), (3, 128, 64), (1, 64, 128)])
def test_append_layout_and_read(K, dtype, H, D, S):
    """ragged appends in two calls (starts inside a 16- and a 32-token group, one sequence with nothing to write, rows past the table dropped):
    pools by the layout's formulas, read back whole, everything not written left as it was."""
    B, T, width = 4, 45, 3
    P = B * width + 2
    io = IO[dtype]
    c = _cache(K, P, S, H, D, dtype)
    table = _table(B, width, P, 1)
    before = [None if t is None else t.view(torch.uint8).clone() for t in c.values()]
    want = {}
    start, count = [0, 7, 19, width * S - 20], [45, 0, 31, 45]      # the second writes nothing, from inside a block; the last one runs past its table: 20 rows fit
    for call in range(2):
        g = _g(10 + call)
        packed = torch.randn(B, T, 2, H * D, generator=g) * torch.exp(torch.randn(B, T, 1, 1, generator=g))
        packed = packed.to(io)
        dev = packed.cuda()
        K.kv_append(dev[:, :, 0], dev[:, :, 1], table=table, start=_i(*start), count=_i(*count), **c)
        for b in range(B):
            for t in range(count[b]):
                if start[b] + t < width * S:
                    want[b, start[b] + t] = packed[b, t]
        start = [45, 7, 50, 0]
        count = [1, 40, 0, 13]
    written = torch.zeros(P, S, dtype=torch.bool)
    for b in range(B):
        k, v, sc = _rows_from_pool(c, table, b, width * S, S, D, dtype)
        for (bb, t), row in want.items():
            if bb != b:
                continue
            written[table[b, t // S].item(), t % S] = True
            for x, got, s in ((row[0], k[t], sc[0]), (row[1], v[t], sc[1])):
                codes, scale = _stored(x, dtype, H)
                assert torch.equal(got.reshape(-1), codes), (b, t)
                if s is not None:
                    assert torch.equal(s[t], scale)
    # what was not written keeps its bytes: K rows by token, V by token
    for name, now, old in zip(c, c.values(), before):
        if now is None:
            continue
        now, old = now.view(torch.uint8), old
        if name == 'k_pool':
            shape = (P, H, S // 16, -1, 16, 16 if dtype in (F32, BF16) else 8)
            same = (now.view(shape) == old.view(shape)).all(-1).all(3).cpu().permute(0, 2, 3, 1).reshape(P, S, H).all(-1)
        elif name == 'v_pool':
            sz = {F32: 4, BF16: 2}.get(dtype, 1)
            if dtype == F32:
                same = (now.view(P, H, S // 16, D // 16, 4, 16, 4, sz) == old.view(P, H, S // 16, D // 16, 4, 16, 4, sz)).all(-1).all(5).all(3).all(1).cpu().reshape(P, S)
            else:
                eq = (now.view(P, H, S // 32, D // 16, 4, 16, 2, 4, sz) == old.view(P, H, S // 32, D // 16, 4, 16, 2, 4, sz)).all(-1).all(5).all(3).all(1).cpu()
                same = eq.permute(0, 1, 3, 2, 4).reshape(P, S)
        else:
            same = (now.view(P, H, S, 4) == old.view(P, H, S, 4)).all(-1).all(1).cpu()
        assert same[~written].all(), name
    # read back: from the middle too, past the written part rows are zero
    for out_dt in ([F32, BF16] if dtype in (I8, E4M3) else [io]):
        rs, rc, n = [0, 7, 19, 0], [46, 40, 31, 13], 50
        k, v = K.kv_read(c['k_pool'], c['v_pool'], table, _i(*rs), _i(*rc), n, c['k_scale'], c['v_scale'], out_dt)
        assert k.dtype == out_dt and k.shape == (B, n, H * D)
        for b in range(B):
            assert (k[b, rc[b]:] == 0).all() and (v[b, rc[b]:] == 0).all()
            for t in range(rc[b]):
                for i, got in enumerate((k[b, t], v[b, t])):
                    codes, scale = _stored(want[b, rs[b] + t][i], dtype, H)
                    val = codes if scale is None else (codes.reshape(H, D) * scale[:, None]).reshape(-1)
                    assert torch.equal(got.cpu(), val.to(out_dt)), (b, t, i)


@pytest.mark.parametrize('dtype', [I8, E4M3])
def test_quantised_rows_that_are_special(K, dtype):
    """zeros, the smallest magnitudes, a row with one huge value, rows with infinities and NaN (they read back as NaN, their neighbours do not)"""
    H, D = 2, 64
    x = torch.randn(1, 8, H * D, generator=_g(3))
    x[0, 0] = 0
    x[0, 1] *= 1e-38
    x[0, 2, 5] = 3e38
    x[0, 3, 7] = float('inf')
    x[0, 4, 70] = float('nan')
    x[0, 5, 3] = float('-inf')
    x[0, 6] = torch.linspace(-1, 1, H * D)
    c = _cache(K, 2, 32, H, D, dtype)
    d = x.cuda()
    K.kv_append(d, d, table=_i(1)[None], start=_i(0), **c)
    k, v = K.kv_read(c['k_pool'], c['v_pool'], _i(1)[None], _i(0), _i(8), 8, c['k_scale'], c['v_scale'], F32)
    assert torch.equal(torch.nan_to_num(k, nan=7e37), torch.nan_to_num(v, nan=7e37))
    k = k.cpu().view(8, H, D)
    bad = ~torch.isfinite(x.view(8, H, D)).all(-1)
    assert bad.sum() == 3 and torch.isnan(k[bad]).all() and torch.isfinite(k[~bad]).all()
    codes, scale = _stored(torch.where(bad[..., None], 0, x.view(8, H, D)).reshape(1, 8, H * D), dtype, H)
    want = codes.view(8, H, D) * scale.view(8, H, 1)
    assert torch.equal(k[~bad], want[~bad])
    # half a step of the code: int8 half a scale; e4m3 2^-4 relative, half its smallest step (2^-10) of a scale near zero.  The division and
    # the product add 2^-23 of the value; scales near 2^-126 lose their own lower bits (2^-149 a product)
    lim = 0.5 * scale.view(8, H, 1) if dtype == I8 else torch.maximum(x.view(8, H, D).abs() * 2.0 ** -4, scale.view(8, H, 1) * 2.0 ** -10)
    err = (k - x.view(8, H, D)).abs()
    assert (err[~bad] <= (lim * (1 + 2.0 ** -20) + x.view(8, H, D).abs() * 2.0 ** -22 + 2.0 ** -126)[~bad]).all()


def test_append_and_read_bad_pages_and_positions(K):
    """pages outside the pool and negative positions: nothing is written, reads are zero, attention does not see the tokens"""
    H, D, S, P = 2, 64, 32, 3
    c = _cache(K, P, S, H, D, BF16)
    x = torch.randn(2, 96, H * D, generator=_g(5)).to(BF16).cuda()
    table = torch.tensor([[1, -1, 2], [P, 0, 1 << 30]], dtype=torch.int32, device='cuda')
    K.kv_append(x, x, table=table, start=_i(0, 0), **c)
    K.kv_append(x, x, table=table, start=_i(-200, 96), **c)              # wholly outside
    k, v = K.kv_read(c['k_pool'], c['v_pool'], table, _i(0, 0), _i(96, 96), 96)
    live = torch.zeros(2, 96, dtype=torch.bool, device='cuda')
    live[0, :32] = live[0, 64:] = live[1, 32:64] = True
    want = torch.where(live[..., None], x, 0)
    assert torch.equal(k, want) and torch.equal(v, want)
    q = torch.randn(2, 1, H * D, generator=_g(6)).to(BF16).cuda()
    o = K.attention_paged(q, table=table, lens=_i(96, 1000), nh=H, **c)
    for b in range(2):
        ref, _, tol, _ = _ref(q[b].double(), x[b][live[b]].double(), x[b][live[b]].double(), H, H, 0.125, torch.ones(1, int(live[b].sum()), dtype=torch.bool, device='cuda'), BF16)
        assert ((o[b].double() - ref).abs() <= tol).all()
    dead = torch.full((2, 3), -1, dtype=torch.int32, device='cuda')
    o, lse = K.attention_paged(q, table=dead, lens=_i(96, 3), nh=H, want_lse=True, **c)
    assert (o == 0).all() and (lse == float('-inf')).all()


def _ref(q, k, v, nh, H, scale, ok, dtype):
    """q [Nq, nh*D], k, v [n, H*D] (64 bits), ok [Nq, n] -> o [Nq, nh*D], lse [nh, Nq], bounds of both.

    With A = sum p |v| and B = max sum |q k| scale: fp32 dot products of D terms are off by (D + 4) 2^-24 B (the multiplication by scale * log2 e
    and the exponential included), p by twice that and the maximum's own share; sums of n terms by n 2^-24; P is rounded once (bf16 caches:
    2^-8; 8-bit caches the same, after the value's scale), O once."""
    Nq, D, n = q.shape[0], q.shape[1] // nh, k.shape[0]
    q_, k_, v_ = q.view(Nq, nh, D), k.view(n, H, D).repeat_interleave(nh // H, 1), v.view(n, H, D).repeat_interleave(nh // H, 1)
    s = torch.stack([q_[:, h] @ k_[:, h].T for h in range(nh)]) * scale                     # [nh, Nq, n]
    B = (torch.stack([q_[:, h].abs() @ k_[:, h].abs().T for h in range(nh)]) * abs(scale)).amax(-1) if n else torch.zeros(nh, Nq, device=q.device, dtype=torch.float64)
    s = s.masked_fill(~ok, float('-inf'))
    lse = torch.logsumexp(s, -1) if n else torch.full((nh, Nq), float('-inf'), device=q.device, dtype=torch.float64)
    p = torch.exp(s - lse.masked_fill(lse == float('-inf'), 0)[..., None])
    o = torch.stack([p[h] @ v_[:, h] for h in range(nh)], 1)
    A = torch.stack([p[h] @ v_[:, h].abs() for h in range(nh)], 1)
    ds = (D + 8) * 2.0 ** -24 * B + 2.0 ** -22                                              # of a score
    step = 2.0 ** -24 if dtype == F32 else 2.0 ** -8
    tol = A * (2 * ds.T[..., None] + (n + 64) * 2.0 ** -23 + step) + o.abs() * step + 1e-30
    return o.reshape(Nq, -1), lse, tol.reshape(Nq, -1), ds + (n + 64) * 2.0 ** -23 + lse.abs().nan_to_num(posinf=0) * 2.0 ** -22


def _seen(n, Nq, causal, window, dev='cuda'):
    at = torch.arange(n, device=dev)
    last = n - Nq + torch.arange(Nq, device=dev)[:, None] if causal else torch.full((Nq, 1), n - 1, device=dev)
    ok = at <= last
    return ok & (at > last - window) if window else ok


def _dense(K, c, table, lens, n, dtype):
    B = table.shape[0]
    return K.kv_read(c['k_pool'], c['v_pool'], table, torch.zeros(B, dtype=torch.int32, device='cuda'), lens, n, c['k_scale'], c['v_scale'], F32 if dtype in (I8, E4M3) else None)


def _attend_case(K, dtype, B, Nq, nh, H, D, S, lens, causal=False, window=0, scale=None, seed=0, spread=1.0):
    width = max(1, -(-max(lens) // S)) + 1
    P = B * width + 1
    c = _cache(K, P, S, H, D, dtype)
    table = _table(B, width, P, seed + 1)
    io, n = IO[dtype], max(max(lens), 1)
    x = (torch.randn(B, n, 2, H * D, generator=_g(seed)) * spread).to(io).cuda()
    L = _i(*lens)
    K.kv_append(x[:, :, 0], x[:, :, 1], table=table, start=torch.zeros_like(L), count=L, **c)
    q = (torch.randn(B, Nq, nh * D, generator=_g(seed + 2)) * spread).to(io).cuda()
    o, lse = K.attention_paged(q, table=table, lens=L, nh=nh, causal=causal, window=window, scale=scale, want_lse=True, **c)
    k, v = _dense(K, c, table, L, n, dtype)          # (checked on its own above)
    for b in range(B):
        m = lens[b]
        ref, rl, tol, tl = _ref(q[b].double(), k[b, :m].double(), v[b, :m].double(), nh, H, D ** -0.5 if scale is None else scale, _seen(m, Nq, causal, window), dtype)
        err = (o[b].double() - ref).abs()
        assert (err <= tol).all(), (b, m, (err / tol).max().item())
        none = rl == float('-inf')
        assert torch.equal(lse[b] == float('-inf'), none)
        assert (o[b].view(Nq, nh, D).transpose(0, 1)[none] == 0).all()
        assert ((lse[b].double() - rl).abs() <= tl)[~none].all()
    return q, c, table, L, o


@pytest.mark.parametrize('dtype', [BF16, F32, I8, E4M3])
@pytest.mark.parametrize('nh,H,D', [(12, 12, 64), (8, 2, 128), (5, 1, 64), (48, 2, 128)])
@pytest.mark.parametrize('Nq,causal,window', [(1, False, 0), (3, False, 0), (1, True, 0), (4, True, 0), (1, True, 37), (6, True, 50), (20, True, 1)])
def test_attention_paged(K, dtype, nh, H, D, Nq, causal, window):
    """lengths of zero and one, below, at and past tiles and pages, fewer tokens than rows; head layouts (own, shared, one, more rows than a
    tile's 16 columns); pools hold NaN wherever nothing was written"""
    _attend_case(K, dtype, 9, Nq, nh, H, D, 32, [0, 1, 2, 15, 31, 32, 33, 129, 300], causal, window)


@pytest.mark.parametrize('dtype', [BF16, I8])
def test_attention_paged_window_over_everything(K, dtype):
    """windows at and past the table's reach are none at all"""
    for window in (128, 4096, 2 ** 31 - 1):
        _attend_case(K, dtype, 4, 5, 8, 2, 64, 32, [0, 3, 70, 96], True, window, seed=9)


@pytest.mark.parametrize('dtype', [BF16, F32, I8, E4M3])
def test_attention_paged_split(K, dtype):
    """few sequences, long: the tokens are split over workgroups and joined; one sequence is empty, one ends inside the first split"""
    _attend_case(K, dtype, 3, 1, 8, 2, 128, 64, [9001, 0, 5], seed=3)
    _attend_case(K, dtype, 1, 2, 12, 12, 64, 32, [4097], causal=True, window=3000, seed=4)
    _attend_case(K, dtype, 2, 1, 2, 1, 64, 128, [20000, 128], seed=5)


@pytest.mark.parametrize('dtype,B,Nq,nh,H,D,causal', [(I8, 37, 1, 12, 12, 64, False), (BF16, 64, 2, 16, 8, 128, True), (F32, 2, 1, 160, 160, 64, False), (E4M3, 33, 1, 8, 8, 64, False),
                                                        (I8, 64, 1, 12, 12, 64, False), (F32, 8, 1, 80, 80, 64, False), (E4M3, 61, 3, 12, 12, 64, True), (BF16, 41, 9, 16, 8, 64, True),
                                                        (F32, 33, 20, 8, 8, 128, False)])
def test_attention_paged_ragged_batches(K, dtype, B, Nq, nh, H, D, causal):
    """more workgroups than CUs over sequences of very different lengths, which are taken longest first: equal lengths, empty ones and the longest in
    any place, full and partial rounds of workgroups"""
    lens = torch.randint(0, 1400, (B,), generator=_g(B)).tolist()
    lens[-1] = 1500
    lens[0] = 0
    lens[B // 2:B // 2 + 5] = [700] * len(lens[B // 2:B // 2 + 5])
    lens[-1] = 1500
    _attend_case(K, dtype, B, Nq, nh, H, D, 64, lens, causal=causal, seed=B)


@pytest.mark.parametrize('dtype', [BF16, F32, I8, E4M3])
@pytest.mark.parametrize('Nq,causal', [(1, False), (3, True)])
def test_attention_paged_nan_scores_show(K, dtype, Nq, causal):
    """a NaN among the scores that a row sees makes its o and lse NaN, also where a wave (a workgroup) saw nothing else; other heads, other
    sequences and rows that do not see it stay as they are"""
    nh, H, D, S, lens, at = 4, 2, 64, 32, [1, 40, 5000, 5000, 70], [0, 39, 4990, 3, None]
    B, n, io = len(lens), max(lens), IO[dtype]
    width = -(-n // S)
    P = B * width + 1
    c, table, L = _cache(K, P, S, H, D, dtype), _table(B, width, P, 1), _i(*lens)
    x = torch.randn(B, n, 2, H * D, generator=_g(2)).to(io).cuda()
    K.kv_append(x[:, :, 0], x[:, :, 1], table=table, start=torch.zeros_like(L), count=L, **c)
    q = torch.randn(B, Nq, nh * D, generator=_g(3)).to(io).cuda()
    q[4, Nq - 1, 3 * D + 5] = float('nan')            # one row's last head
    for b, t in enumerate(at):
        if t is None:
            continue
        k = x[b:b + 1, t:t + 1, 0].clone()
        k[..., :D] = float('nan')                     # the first key / value head
        K.kv_append(k, x[b:b + 1, t:t + 1, 1], table=table[b:b + 1], start=_i(t), **c)
    o, lse = K.attention_paged(q, table=table, lens=L, nh=nh, causal=causal, want_lse=True, **c)
    o = o.view(B, Nq, nh, D)
    for b in range(B):
        for i in range(Nq):
            last = lens[b] - Nq + i if causal else lens[b] - 1
            for h in range(nh):
                bad = (at[b] is not None and h < nh // H and at[b] <= last) or (b == 4 and i == Nq - 1 and h == 3)
                assert torch.isnan(o[b, i, h]).all() if bad else torch.isfinite(o[b, i, h]).all(), (b, i, h)
                assert lse[b, h, i].isnan() if bad else (lse[b, h, i].isfinite() if last >= 0 else lse[b, h, i] == float('-inf')), (b, i, h)


@pytest.mark.parametrize('dtype', [I8, E4M3])
@pytest.mark.parametrize('nh', [2, 16])
def test_attention_paged_hidden_rows_without_a_scale(K, dtype, nh):
    """8-bit keys and values of a token that only the last row sees, written from NaN and infinities: the other rows do not notice"""
    H, D, n = 2, 64, 40
    x = torch.randn(1, n, 2, H * D, generator=_g(5)).to(BF16).cuda()
    bad = x.clone()
    bad[0, n - 1, :, 3], bad[0, n - 1, :, D + 7], bad[0, n - 1, :, D + 9] = float('nan'), float('inf'), float('-inf')
    q = torch.randn(1, 3, nh * D, generator=_g(6)).to(BF16).cuda()
    table, L, got = _i(2, 1)[None], _i(n), []
    for rows in (x, bad):
        c = _cache(K, 3, 32, H, D, dtype)
        K.kv_append(rows[:, :, 0], rows[:, :, 1], table=table, start=_i(0), **c)
        got.append(K.attention_paged(q, table=table, lens=L, nh=nh, causal=True, want_lse=True, **c))
    assert torch.equal(got[0][0][:, :2], got[1][0][:, :2]) and torch.equal(got[0][1][..., :2], got[1][1][..., :2])
    assert torch.isfinite(got[0][0]).all() and torch.isnan(got[1][0][:, 2]).all() and torch.isnan(got[1][1][..., 2]).all()


def test_attention_paged_scales_and_large_scores(K):
    """scores of hundreds (one token takes the whole row), a scale of its own, a negative one"""
    _attend_case(K, BF16, 2, 2, 4, 2, 64, 32, [700, 90], seed=6, spread=8.0)
    _attend_case(K, F32, 2, 2, 4, 2, 64, 32, [700, 90], seed=7, spread=8.0)
    _attend_case(K, F32, 2, 1, 4, 4, 128, 32, [70, 90], seed=8, scale=-0.3)


@pytest.mark.parametrize('dtype', [BF16, F32])
def test_attention_paged_masked_values_may_be_anything(K, dtype):
    """infinities and NaN in tokens that a row does not see leave it alone; a row that sees them shows them (as the sum does)"""
    H, D, S, n, Nq = 2, 64, 32, 70, 8
    c = _cache(K, 4, S, H, D, dtype)
    table = _i(1, 2, 3)[None]
    k, v = (torch.randn(1, n, H * D, generator=_g(s)).to(dtype) for s in (1, 2))
    q = torch.randn(1, Nq, H * D, generator=_g(3)).to(dtype).cuda()
    clean_k, clean_v = k.clone(), v.clone()
    k[0, 66, :D] = float('nan')                    # token 66 is the row 4's own: rows 4.. see it
    v[0, 67, 3] = float('inf')
    v[0, 68, D + 1] = float('nan')
    v[0, 2, 7] = float('nan')                      # outside every window below
    k[0, 3, 9] = float('-inf')
    K.kv_append(k.cuda(), v.cuda(), table=table, start=_i(0), **c)
    o = K.attention_paged(q, table=table, lens=_i(n), nh=H, causal=True, window=40, **c)
    c2 = _cache(K, 4, S, H, D, dtype)
    K.kv_append(clean_k.cuda(), clean_v.cuda(), table=table, start=_i(0), **c2)
    o2 = K.attention_paged(q, table=table, lens=_i(n), nh=H, causal=True, window=40, **c2)
    o, o2 = o.view(Nq, H, D), o2.view(Nq, H, D)
    assert torch.equal(o[:4], o2[:4]) and torch.isfinite(o2).all()
    assert torch.isnan(o[4:, 0]).all()                                             # K's NaN: the head's whole row
    assert torch.equal(o[4:6, 1], o2[4:6, 1])
    assert not torch.isfinite(o[5:, 0, 3]).any()
    assert torch.isnan(o[6:, 1, 1]).all() and torch.equal(o[6:, 1, 2:], o2[6:, 1, 2:]) and torch.equal(o[6:, 1, 0], o2[6:, 1, 0])


def test_paged_offsets_past_32_bits(K):
    """pages whose elements lie past 2^31 (bytes past 2^32) in the pool"""
    H, D, S = 8, 128, 64
    P = (1 << 31) // (H * D * S) + 600                   # 33,368 pages of 128 KiB a pool
    ks, vs = K.kv_pool_shapes(P, S, H, D, BF16)
    c = dict(k_pool=torch.empty(ks, device='cuda', dtype=BF16), v_pool=torch.empty(vs, device='cuda', dtype=BF16), k_scale=None, v_scale=None)
    table = _i(P - 1, 3, P - 500)[None]
    lens = _i(150)
    x = torch.randn(1, 150, 2, H * D, generator=_g(1)).to(BF16).cuda()
    K.kv_append(x[:, :, 0], x[:, :, 1], table=table, start=_i(0), **c)
    k, v = K.kv_read(c['k_pool'], c['v_pool'], table, _i(0), lens, 150)
    assert torch.equal(k, x[:, :, 0]) and torch.equal(v, x[:, :, 1])
    q = torch.randn(1, 1, H * D, generator=_g(2)).to(BF16).cuda()
    o = K.attention_paged(q, table=table, lens=lens, nh=H, **c)
    ref, _, tol, _ = _ref(q[0].double(), k[0].double(), v[0].double(), H, H, D ** -0.5, _seen(150, 1, False, 0), BF16)
    assert ((o[0].double() - ref).abs() <= tol).all()


def test_strides_orders_and_streams(K):
    """views with other strides, unaligned ones (copied), a table that is a slice of a wider one, another stream"""
    H, D, S, B = 4, 64, 32, 3
    c, c2 = _cache(K, 20, S, H, D, BF16), _cache(K, 20, S, H, D, BF16)
    wide = torch.zeros(B, 7, dtype=torch.int32, device='cuda')
    wide[:, 2:5] = _table(B, 3, 20, 1)
    table = wide[:, 2:5]
    x = torch.randn(70, B, 3 * H * D + 3, generator=_g(1)).to(BF16).cuda()
    k, v = x[..., 1:1 + H * D].transpose(0, 1), x[..., 2 + H * D:2 + 2 * H * D].transpose(0, 1)       # tokens first, rows not 16-byte aligned
    start, count = _i(0, 5, 9), _i(70, 61, 1)
    K.kv_append(k, v, table=table, start=start, count=count, **c)
    K.kv_append(k.contiguous(), v.contiguous(), table=table.contiguous(), start=start, count=count, **c2)
    assert torch.equal(c['k_pool'].view(torch.uint8), c2['k_pool'].view(torch.uint8)) and torch.equal(c['v_pool'].view(torch.uint8), c2['v_pool'].view(torch.uint8))
    qq = torch.randn(2, B, 2, H * D, generator=_g(2)).to(BF16).cuda()
    q = qq.permute(1, 0, 2, 3)[:, :, 1]
    lens = _i(70, 66, 10)
    bits = lambda t: t.view(torch.int16)      # (sequences 1 and 2 were written from tokens 5 and 9 on: their rows show the NaN before those)  # noqa: E731
    want = bits(K.attention_paged(q.contiguous(), table=table.contiguous(), lens=lens, nh=H, **c))
    assert torch.equal(bits(K.attention_paged(q, table=table, lens=lens, nh=H, **c)), want)
    st = torch.cuda.Stream()
    st.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(st):
        other = bits(K.attention_paged(q, table=table, lens=lens, nh=H, **c))
    torch.cuda.current_stream().wait_stream(st)
    assert torch.equal(other, want)


def test_empty_calls(K):
    H, D, S = 2, 64, 32
    c = _cache(K, 2, S, H, D, BF16)
    e = torch.empty(0, 1, H * D, device='cuda', dtype=BF16)
    none = torch.empty(0, dtype=torch.int32, device='cuda')
    t0 = torch.empty(0, 1, dtype=torch.int32, device='cuda')
    K.kv_append(e, e, table=t0, start=none, **c)
    assert K.attention_paged(e, table=t0, lens=none, nh=H, **c).shape == (0, 1, H * D)
    assert K.attention_paged(torch.empty(1, 0, H * D, device='cuda', dtype=BF16), table=_i(1)[None], lens=_i(0), nh=H, **c).shape == (1, 0, H * D)
    k, v = K.kv_read(c['k_pool'], c['v_pool'], _i(1)[None], _i(0), _i(0), 0)
    assert k.shape == (1, 0, H * D)
    tok, lp = K.sample_rows(torch.empty(0, 5, device='cuda'), torch.empty(0, device='cuda'))
    assert tok.shape == lp.shape == (0,)


# ---- sampling ----------------------------------------------------------------------------------------------------------------

def _sample_ref(x, u, T, k, p, m):
    """one row, 64 bits, from the definition -> (token, logp, kept indices)"""
    x = x.double().cpu()
    x = torch.where(torch.isnan(x), float('-inf'), x)
    cand = [j for j in torch.argsort(x, descending=True, stable=True).tolist() if x[j] > float('-inf')]
    if not cand:
        return -1, float('-inf'), []
    top = x[cand[0]]
    if not T > 0:
        return cand[0], 0.0, cand[:1]
    if k > 0:
        cand = cand[:k]
    z = torch.where(x == top, torch.zeros_like(x), (x - top) / T)
    w = torch.exp(z)
    if p < 1:
        run = torch.cumsum(w[cand], 0)
        cand = cand[:max(1, int((run < p * run[-1]).sum()) + (1 if p > 0 else 0))]
    cand = [cand[0]] + [j for j in cand[1:] if w[j] >= m]
    cand = sorted(cand)
    run = torch.cumsum(w[cand], 0)
    j = min(int((run <= float(u) * run[-1]).sum()), len(cand) - 1)
    return cand[j], float(z[cand[j]] - torch.log(run[-1])), cand


def _check_rows(K, logits, u, T=1.0, k=0, p=1.0, m=0.0):
    B, V = logits.shape
    tok, lp = K.sample_rows(logits, u, T, k, p, m)
    assert tok.dtype == torch.int64 and lp.dtype == torch.float32
    at = lambda a, b: a[b].item() if isinstance(a, torch.Tensor) else a if isinstance(a, int) else float(np.float32(a))      # (numbers are fp32 too)  # noqa: E731
    for b in range(B):
        rt, rl, _ = _sample_ref(logits[b], u[b].item(), at(T, b), at(k, b), at(p, b), at(m, b))
        assert tok[b].item() == rt, (b, V, tok[b].item(), rt)
        if rt < 0:
            assert lp[b].item() == float('-inf')
        else:      # one rounding to fp32 (2^-24), weights of 2^-45 an entry
            assert abs(lp[b].item() - rl) <= abs(rl) * 2.0 ** -23 + V * 2.0 ** -44 + 1e-12, (b, lp[b].item(), rl)
    return tok


@pytest.mark.parametrize('dtype', [F32, BF16])
@pytest.mark.parametrize('V', [1, 2, 63, 64, 65, 100, 257, 1000, 1025, 4096, 4097, 30522, 131071])
def test_sample_rows_sizes(K, dtype, V):
    B = 6
    g = _g(V)
    logits = (torch.randn(B, V, generator=g) * 3).to(dtype).cuda()
    u = torch.rand(B, generator=g).cuda()
    _check_rows(K, logits, u)
    _check_rows(K, logits, u, 0.7, 0, 0.9, 0.0)
    _check_rows(K, logits, u, 1.3, 50, 1.0, 0.0)
    _check_rows(K, logits, u, 0.9, 40, 0.8, 0.05)
    par = dict(T=torch.rand(B, generator=g) + 0.3, k=torch.randint(0, V + 3, (B,), generator=g, dtype=torch.int32), p=torch.rand(B, generator=g) * 1.2, m=torch.rand(B, generator=g) * 0.1)
    _check_rows(K, logits, u, **{n: t.cuda() for n, t in par.items()})


@pytest.mark.parametrize('dtype', [F32, BF16])
@pytest.mark.parametrize('V', [50, 900, 5000, 40001])
def test_sample_rows_ties_and_flat_rows(K, dtype, V):
    """equal values rank by index, also by the thousand; narrow rows fall into one bin; signed zeros are one value"""
    g = _g(V + 1)
    rows = [torch.zeros(V), torch.full((V,), -7.25), torch.randint(0, 3, (V,), generator=g).float(), torch.randn(V, generator=g) * 1e-4,
            1000 + torch.randn(V, generator=g) * 1e-3, torch.where(torch.rand(V, generator=g) < 0.5, -0.0, 0.0), torch.randn(V, generator=g) * 1e-30,
            torch.linspace(-40, 40, V)]
    logits = torch.stack(rows).to(dtype).cuda()
    B = logits.shape[0]
    for i, (k, p, m) in enumerate([(0, 1.0, 0.0), (V // 3 + 1, 1.0, 0.0), (0, 0.37, 0.0), (V // 2 + 1, 0.61, 0.0), (1, 0.5, 0.5), (V - 1, 0.999, 0.9), (0, 0.0, 0.0)]):
        _check_rows(K, logits, torch.rand(B, generator=_g(i)).cuda(), 0.8, k, p, m)


def test_sample_rows_masks_and_special_values(K):
    inf, nan = float('inf'), float('nan')
    V = 300
    x = torch.randn(8, V, generator=_g(1))
    x[0] = -inf                                    # nothing to draw
    x[1] = nan
    x[2, :] = -inf
    x[2, 217] = -3e38                              # one candidate, at the type's lowest values
    x[3, ::2] = nan
    x[4, 1:] = -inf
    x[5, 7] = x[5, 200] = inf                      # infinities share the row
    x[6] = -3.4e38                                 # a mask of the lowest value is a value like any other
    x[6, 100:] = torch.randn(200, generator=_g(2))
    u = torch.tensor([0.3, 0.3, 0.9, 0.5, 0.0, 0.6, 0.99, 0.2]).cuda()
    x = x.cuda()
    for args in [(1.0, 0, 1.0, 0.0), (0.5, 3, 0.7, 0.1), (2.0, 250, 0.95, 0.0), (0.0, 0, 1.0, 0.0), (1e-30, 0, 0.9, 0.0), (1e30, 0, 0.9, 0.3)]:
        _check_rows(K, x, u, *args)
    tok, lp = K.sample_rows(x, u)
    assert tok[0] == -1 and tok[1] == -1 and lp[0] == -inf and tok[5] == 200 and tok[4] == 0
    # given numbers at the ends of [0, 1)
    lo, hi = torch.zeros(8, device='cuda'), torch.full((8,), 1 - 2.0 ** -24, device='cuda')
    _check_rows(K, x, lo)
    _check_rows(K, x, hi)


@pytest.mark.parametrize('V', [40, 3000, 20000, 70000])
def test_sample_rows_min_p_alone_and_parameters_out_of_range(K, V):
    """min-p without the other cuts (few and many entries left); tensors may hold what a number may not: min-p over 1 (the largest alone), NaN and
    negative values (no cut; temperature: the largest), top-p of 0 and below, top-k over the row"""
    B = 8
    logits = (torch.randn(B, V, generator=_g(V)) * 1.5).cuda()
    u = torch.rand(B, generator=_g(1)).cuda()
    for m in (0.9, 0.3, 0.01, 1e-5):
        _check_rows(K, logits, u, 0.9, 0, 1.0, m)
    t = lambda *v: torch.tensor(v, device='cuda')        # noqa: E731
    nan = float('nan')
    T = t(1.0, 1.0, nan, -1.0, 0.7, 0.7, 2.0, 0.7)
    k = t(0, V + 5, 3, 3, -4, 300, 700, 2000).int()
    p = t(0.5, -0.5, 0.9, 0.9, nan, 0.0, 0.8, 0.9)
    m = t(1.7, 0.0, 0.1, 0.1, nan, 0.2, -1.0, 5.0)
    tok, lp = K.sample_rows(logits, u, T, k, p, m)
    for b in range(B):
        pb, mb = p[b].item(), m[b].item()
        rt, rl, _ = _sample_ref(logits[b], u[b].item(), T[b].item(), k[b].item(), 1.0 if pb != pb else pb, 0.0 if mb != mb else mb)
        assert tok[b].item() == rt, b
        assert abs(lp[b].item() - rl) <= abs(rl) * 2.0 ** -23 + V * 2.0 ** -44 + 1e-12, b


@pytest.mark.parametrize('V', [2000, 6000, 30522, 70000])
@pytest.mark.parametrize('start,width,T', [(0.0, 0.003, 1.0), (0.0, 0.00397, 1.0), (5.0, 0.01, 1.0), (300.0, 90.0, 100.0), (700.0, 2.0, 1.0)])
def test_sample_rows_crowded_bins(K, V, start, width, T):
    """thousands of different values, and some equal ones, close together behind the largest: near it, in the middle, far away"""
    B = 4
    x = -(start + width * torch.rand(B, V, generator=_g(V)))
    x[:, 5:40] = x[:, 50:51]
    x[:, 77] = 0.0
    logits, u = x.cuda(), torch.rand(B, generator=_g(3)).cuda()
    for k, p, m in [(0, 0.7, 0.0), (V // 2, 1.0, 0.0), (V // 3, 0.4, 0.0), (0, 0.3, 1e-3)]:
        _check_rows(K, logits, u, T, k, p, m)


@pytest.mark.parametrize('V', [40, 3000, 20000])
def test_sample_rows_infinite_temperature(K, V):
    """(a tensor may hold one; as a number it is refused) every candidate weighs the same, so min-p of 1 keeps them all"""
    logits, u = torch.randn(4, V, generator=_g(V)).cuda(), torch.rand(4, generator=_g(2)).cuda()
    for k, p, m in [(0, 1.0, 0.0), (0, 1.0, 1.0), (17, 1.0, 1.0), (0, 0.5, 1.0)]:
        _check_rows(K, logits, u, torch.full((4,), float('inf'), device='cuda'), k, p, m)


@pytest.mark.parametrize('dtype', [F32, BF16])
def test_sample_rows_strided_rows(K, dtype):
    """rows that begin anywhere, and end anywhere in front of numbers that are larger than any of theirs"""
    big = torch.randn(5, 1000, generator=_g(4))
    big[:, :3] = big[:, 903:] = 50
    big = big.to(dtype).cuda()
    u = torch.rand(5, generator=_g(5)).cuda()
    a = _check_rows(K, big[:, 3:903], u, 0.9, 30, 0.9)
    assert torch.equal(a, K.sample_rows(big[:, 3:903].contiguous(), u, 0.9, 30, 0.9)[0])


def test_sample_rows_follows_the_distribution(K):
    """20,000 draws from one row: each kept entry's share is within 5 standard deviations, no other entry is drawn"""
    V, n = 200, 20000
    row = torch.randn(V, generator=_g(9)) * 2
    u = (torch.arange(n) + 0.5) / n
    tok, _ = K.sample_rows(row.expand(n, V).contiguous().cuda(), u[torch.randperm(n, generator=_g(1))].cuda(), 0.9, 30, 0.9, 0.01)
    _, _, kept = _sample_ref(row, 0.5, 0.9, 30, 0.9, 0.01)
    p = torch.softmax(row.double()[kept] / 0.9, 0)
    share = torch.bincount(tok.cpu(), minlength=V).double()[kept] / n
    assert share.sum() == 1 and ((share - p).abs() <= 1.5 / n).all()        # (an even grid of numbers: exact to its step)


# ---- together ----------------------------------------------------------------------------------------------------------------

@pytest.mark.parametrize('dtype', [BF16, I8, E4M3, F32])
def test_a_decoding_loop(K, dtype):
    """what a serving loop does, step by step: prompts of different lengths written at once, then per step one new token appended, attended and
    drawn - through PagedKVCache; each step against 64 bits on the tokens drawn so far; pages go back at the end"""
    from dsrg_amd.kvcache import PagedKVCache
    B, H, D, V, steps = 5, 2, 64, 211, 40
    io = IO[dtype]
    g = _g(1)
    emb, wq, wk, wv, wo = (torch.randn(*s, generator=g).to(io).cuda() for s in ((V, 64), (64, 4 * D), (64, H * D), (64, H * D), (4 * D, V)))
    prompt = [1, 17, 32, 33, 90]
    cache = PagedKVCache(64, H, D, dtype=dtype)
    free = cache.free_pages
    table = cache.table([n + steps for n in prompt])
    ids = torch.randint(0, V, (B, max(prompt)), generator=g).cuda()
    x = emb[ids]
    lens = _i(*prompt)
    cache.append(x @ wk, x @ wv, table, torch.zeros_like(lens), lens)
    tok = ids.gather(1, (lens.long() - 1)[:, None])[:, 0]
    for step in range(steps):
        x = emb[tok][:, None]
        q, k, v = x @ wq, x @ wk, x @ wv
        cache.append(k, v, table, lens)
        lens = lens + 1
        o = cache.attend(q, table, lens, nh=4, causal=True)
        n = int(lens.max())
        kd, vd = cache.read(table, torch.zeros_like(lens), lens, n, F32 if dtype != BF16 else None)
        for b in (0, step % B):
            m = int(lens[b])
            ref, _, tol, _ = _ref(q[b].double(), kd[b, :m].double(), vd[b, :m].double(), 4, H, D ** -0.5, _seen(m, 1, True, 0), dtype)
            assert ((o[b].double() - ref).abs() <= tol).all()
        logits = (o[:, 0].float() @ wo.float()) * 0.3
        u = torch.rand(B, generator=_g(step)).cuda()
        tok, _ = K.sample_rows(logits, u, 0.9, 50, 0.95)
        if step % 10 == 0:
            _check_rows(K, logits, u, 0.9, 50, 0.95)
    cache.release(table)
    assert cache.free_pages == free


def test_captured_loops_share_nothing(K):
    """append + attend (split: with its workspace) + draw captured into two graphs, replayed in turn and at once on two streams, with eager calls
    of the same operators between the replays: every replay gives the eager result"""
    H, D, S, nh, V = 2, 128, 64, 8, 3000
    sets = []
    for i in range(2):
        c = _cache(K, 70, S, H, D, BF16)
        table = _table(1, 60, 70, i)
        n = 3000 + 500 * i
        x = torch.randn(1, n, 2, H * D, generator=_g(i)).to(BF16).cuda()
        K.kv_append(x[:, :, 0], x[:, :, 1], table=table, start=_i(0), **c)
        s = dict(c=c, table=table, start=_i(n), lens=_i(n + 1), k=torch.empty(1, 1, H * D, device='cuda', dtype=BF16), v=torch.empty(1, 1, H * D, device='cuda', dtype=BF16),
                 q=torch.empty(1, 1, nh * D, device='cuda', dtype=BF16), w=torch.randn(nh * D, V, generator=_g(7 + i)).cuda() * 0.3, u=torch.empty(1, device='cuda'))
        sets.append(s)

    def step(s):
        K.kv_append(s['k'], s['v'], table=s['table'], start=s['start'], **s['c'])
        o = K.attention_paged(s['q'], table=s['table'], lens=s['lens'], nh=nh, **s['c'])
        logits = o[:, 0].float() @ s['w']
        return o, logits, *K.sample_rows(logits, s['u'], 0.8, 100, 0.9, 0.01)

    def feed(s, seed):
        g = _g(seed)
        for name in 'kvq':
            s[name].copy_(torch.randn(s[name].shape, generator=g).to(BF16))
        s['u'].copy_(torch.rand(1, generator=g))

    graphs, outs = [], []
    for i, s in enumerate(sets):
        feed(s, i)
        step(s)
        torch.cuda.synchronize()
        gr = torch.cuda.CUDAGraph()
        with torch.cuda.graph(gr):
            outs.append(step(s))
        graphs.append(gr)
    streams = [torch.cuda.Stream() for _ in range(2)]
    for rep in range(6):
        for i, s in enumerate(sets):
            feed(s, 100 * rep + i)
        torch.cuda.synchronize()
        want = [[t.clone() for t in step(s)] for s in sets]
        torch.cuda.synchronize()
        for i in range(2):
            with torch.cuda.stream(streams[i] if rep % 2 else torch.cuda.current_stream()):
                graphs[i].replay()
        torch.cuda.synchronize()
        for o, w in zip(outs, want):
            for a, b in zip(o, w):
                assert torch.equal(a, b), rep
