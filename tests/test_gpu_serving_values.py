"""gpu: attention over the paged cache where values or scores are not finite: what a row sees shows, whatever it weighs and whichever wave, workgroup
or block holds it; what it does not see does not."""
import pytest
import torch

from tests.test_gpu_serving import BF16, E4M3, F32, I8, IO, _cache, _g, _i, _table

pytestmark = pytest.mark.gpu


@pytest.fixture(scope='module')
def K():
    assert torch.cuda.is_available(), 'GPU tests need an MI355X'
    from dsrg_amd import kernels
    return kernels


def _with_and_without(K, dtype, n, Nq, nh, H, D, S, top, bad, value, reach=0):
    """One sequence of n tokens whose token `top` has a score of about 1000 and the others of less than 200 (so that they weigh 0), with and without
    `value` in dim 3 of head 0's values at token `bad` -> ((o, lse) with, (o, lse) without), o [Nq, nh, D]"""
    io = IO[dtype]
    x = torch.randn(1, n, 2, H * D, generator=_g(n + top)).to(io)
    q = torch.full((1, Nq, nh * D), 8.0, dtype=io)
    x[0, top, 0] = 8.0 * 2 * (64 / D) ** 0.5          # 8 * 16 * 64 / 8 (D = 64); the others: 8 * N(0, 64) / 8, |.| < 60
    width = max(-(-n // S), reach)
    got = []
    for rows in (x.clone(), x):
        if not got:
            rows[0, bad, 1, 3] = value
        c, table = _cache(K, width + 1, S, H, D, dtype), _table(1, width, width + 1, 1)
        d = rows.cuda()
        K.kv_append(d[:, :, 0], d[:, :, 1], table=table, start=_i(0), **c)
        o, lse = K.attention_paged(q.cuda(), table=table, lens=_i(n), nh=nh, causal=True, want_lse=True, **c)
        got.append((o.view(Nq, nh, D), lse[0]))
    return got


def _check(got, dtype, n, Nq, nh, H, bad):
    (o, lse), (o2, lse2) = got
    G = nh // H
    assert torch.isfinite(o2).all() and torch.equal(lse, lse2)
    assert torch.equal(o[:, G:], o2[:, G:])                                   # the other key / value heads
    for i in range(Nq):
        if bad > n - Nq + i:
            assert torch.equal(o[i], o2[i]), i
        elif dtype in (I8, E4M3):                                             # (the row has no scale: all its values are NaN)
            assert torch.isnan(o[i, :G]).all(), i
        else:
            assert not torch.isfinite(o[i, :G, 3]).any(), i
            keep = [d for d in range(o.shape[2]) if d != 3]
            assert torch.equal(o[i, :G][:, keep], o2[i, :G][:, keep]), i


@pytest.mark.parametrize('dtype', [BF16, F32, I8, E4M3])
@pytest.mark.parametrize('value', [float('inf'), float('nan')])
@pytest.mark.parametrize('n,top,bad', [(200, 5, 40), (200, 150, 7), (190, 40, 64), (9001, 4, 8000), (9001, 8990, 3), (9001, 8000, 40)])
def test_values_without_weight_show_across_waves_and_splits(K, dtype, value, n, top, bad):
    """token `bad` lies in a block that is seen whole, in another wave or workgroup than the token that takes all the weight"""
    for Nq, nh, H, D in ((1, 2, 2, 64), (1, 8, 2, 128), (3, 12, 2, 64)):
        _check(_with_and_without(K, dtype, n, Nq, nh, H, D, 32, top, bad, value), dtype, n, Nq, nh, H, bad)


@pytest.mark.parametrize('dtype', [BF16, F32, I8, E4M3])
@pytest.mark.parametrize('value', [float('inf'), float('nan')])
@pytest.mark.parametrize('n,top,bad', [(200, 5, 196), (200, 197, 193), (190, 40, 188), (9001, 4, 8995), (33, 1, 32), (20, 3, 11)])
def test_values_without_weight_show_in_blocks_seen_in_part(K, dtype, value, n, top, bad):
    """token `bad` lies in the last, incomplete block (of some, only the later rows see it)"""
    for Nq, nh, H, D in ((1, 2, 2, 64), (1, 8, 2, 128), (3, 12, 2, 64), (3, 16, 2, 128)):
        _check(_with_and_without(K, dtype, n, Nq, nh, H, D, 32, top, bad, value), dtype, n, Nq, nh, H, bad)
