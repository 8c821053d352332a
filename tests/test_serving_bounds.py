"""Attention over the paged cache against 64 bits within a bound that counts the kernel's own roundings, and a check on the CPU that the bound is tight
enough: an output that misses one block of 32 tokens, or whose weights were rounded once to bf16, lies outside it.

The bound, first order in the roundings (one is 2^-24 of the value, half a step of fp32; an addition inside a matrix instruction is counted as 2^-23,
a whole step, as its order and rounding are the hardware's):
  score s_t of a token: D products and additions, the scales and the exponential's argument: ds_t = (D + 8) 2^-23 sum_d |q_d k_td| scale + 2^-22;
  o = sum p_t v_t: a relative error e_t of a weight moves o by at most sum p_t e_t |v_t| + |o| sum p_t e_t (the second from the sum of weights);
  sums: a wave adds T tokens in turn (with P in two parts 2 T products), is rescaled at most once in 32 of them (2 roundings each, for O and the sum),
        then up to 16 waves and up to 32 workgroups are joined (2 each): C = 2 T + 4 T / 32 + 96 steps of 2^-23;
  P: two bf16 numbers, the second with half a step of the first's remainder: 2^-8 2^-8 (fp32 caches: not rounded);
  o: rounded once to its type (half a step: 2^-8, 2^-24).
T is what the rule of how a sequence is shared gives (the table's reach in blocks over the workgroups and their waves)."""
import pytest
import torch

from tests.test_gpu_serving import BF16, E4M3, F32, I8, IO, _cache, _dense, _g, _i, _seen, _stored, _table

# name: (sequences' lengths, Nq, nh, H, D, page, causal, window, T)
CASES = {
    'short': ([2, 33, 40, 50, 65, 300], 1, 12, 12, 64, 32, False, 0, 32),
    'rows': ([40, 70, 2500], 6, 16, 2, 128, 64, True, 0, 96),
    'split': ([9001, 0, 5], 1, 8, 2, 128, 64, False, 0, 96),
    'window': ([4097], 2, 12, 12, 64, 32, True, 3000, 64),
    'long': ([20000, 128], 1, 2, 1, 64, 128, False, 0, 96),
    'batch': ([1500, 0, 700, 700, 31] + list(range(100, 1280, 20)), 1, 12, 12, 64, 64, False, 0, 416),
}


def _bound(q, k, v, nh, H, ok, dtype, T):
    """q [Nq, nh*D], k, v [n, H*D] in 64 bits, ok [Nq, n] -> o, lse [nh, Nq], their bounds, and p [nh, Nq, n]"""
    Nq, D, n = q.shape[0], q.shape[1] // nh, k.shape[0]
    q_ = q.view(Nq, nh, D).transpose(0, 1)
    k_, v_ = (x.view(n, H, D).repeat_interleave(nh // H, 1).transpose(0, 1) for x in (k, v))
    s = torch.matmul(q_, k_.transpose(1, 2).contiguous()) * D ** -0.5
    ds = (D + 8) * 2.0 ** -23 * torch.matmul(q_.abs(), k_.abs().transpose(1, 2).contiguous()) * D ** -0.5 + 2.0 ** -22
    s = s.masked_fill(~ok, float('-inf'))
    lse = torch.logsumexp(s, -1)
    p = torch.exp(s - lse.masked_fill(lse == float('-inf'), 0)[..., None])
    o, A, E, S = torch.matmul(p, v_), torch.matmul(p, v_.abs()), torch.matmul(p * ds, v_.abs()), (p * ds).sum(-1, keepdim=True)
    C = (2 * T + 4 * T / 32 + 96) * 2.0 ** -23
    tol = E + o.abs() * S + (A + o.abs()) * C + (0 if dtype == F32 else A * 2.0 ** -16)
    tol = tol + (o.abs() + tol) * (2.0 ** -24 if dtype == F32 else 2.0 ** -8) + 1e-30
    back = lambda x: x.transpose(0, 1).reshape(Nq, nh * D)      # noqa: E731
    n_ = torch.log(torch.tensor(max(n, 1), dtype=torch.float64))
    return back(o), lse, back(tol), S[..., 0] + C + (lse.abs() + n_ + 1) * 2.0 ** -22, p


def _inputs(case, dtype, seed):
    lens, Nq, nh, H, D = CASES[case][:5]
    x = torch.randn(len(lens), max(lens), 2, H * D, generator=_g(seed)).to(IO[dtype])
    return x, torch.randn(len(lens), Nq, nh * D, generator=_g(seed + 1)).to(IO[dtype])


@pytest.mark.parametrize('dtype', [BF16, F32, I8, E4M3])
@pytest.mark.parametrize('case', list(CASES))
def test_the_bound_shows_a_lost_block_and_weights_of_one_rounding(case, dtype):
    lens, Nq, nh, H, D, _, causal, window, T = CASES[case]
    x, q = _inputs(case, dtype, 1)
    n, once = lens[0] if case != 'short' else lens[-1], False
    b = lens.index(n)
    k, v = x[b, :n].unbind(1)
    if dtype in (I8, E4M3):
        k, v = ((codes.view(n, H, D) * scale[..., None]).reshape(n, H * D) for codes, scale in (_stored(y, dtype, H) for y in (k, v)))
    k, v, q = k.double(), v.double(), q.double()
    ok = _seen(n, Nq, causal, window, 'cpu')
    o, lse, tol, tl, p = _bound(q[b], k, v, nh, H, ok, dtype, T)
    assert ((o.to(IO[dtype]).double() - o).abs() <= tol).all()
    lost = (n - 1) // 64 * 32                              # a block in the middle (rows that see none of it are left out below)
    gone = ok.clone()
    gone[:, lost:lost + 32] = False
    rows = (ok != gone).any(1)
    o1, lse1 = _bound(q[b], k, v, nh, H, gone, dtype, T)[:2]
    err = (o1.to(IO[dtype]).double() - o).abs()
    assert (err[rows].view(-1, nh, D) > tol[rows].view(-1, nh, D)).any(-1).all()                 # in every row and head
    assert ((lse1 - lse).abs() > tl)[:, rows].all()
    v0 = v.clone()
    v0[lost:lost + 32] = 0
    o2 = _bound(q[b], k, v0, nh, H, ok, dtype, T)[0]
    assert ((o2.to(IO[dtype]).double() - o).abs()[rows].view(-1, nh, D) > tol[rows].view(-1, nh, D)).any(-1).all()
    if case == 'short' and dtype != F32:
        v_ = v.view(n, H, D).repeat_interleave(nh // H, 1).transpose(0, 1)
        top = p.amax(-1, keepdim=True)                     # (the kernel's weights are relative to the largest)
        w = (p / top).to(BF16).double() * top
        o3 = torch.matmul(w, v_).transpose(0, 1).reshape(Nq, nh * D)
        assert ((o3.to(IO[dtype]).double() - o).abs() > tol).any()


@pytest.mark.gpu
@pytest.mark.parametrize('dtype', [BF16, F32, I8, E4M3])
@pytest.mark.parametrize('case', list(CASES))
def test_attention_paged_within_its_own_roundings(case, dtype):
    from dsrg_amd import kernels as K
    lens, Nq, nh, H, D, S, causal, window, T = CASES[case]
    x, q = _inputs(case, dtype, 1)
    x, q, L = x.cuda(), q.cuda(), _i(*lens)
    width = -(-max(lens) // S)
    c, table = _cache(K, len(lens) * width + 1, S, H, D, dtype), _table(len(lens), width, len(lens) * width + 1, 2)
    K.kv_append(x[:, :, 0], x[:, :, 1], table=table, start=torch.zeros_like(L), count=L, **c)
    o, lse = K.attention_paged(q, table=table, lens=L, nh=nh, causal=causal, window=window, want_lse=True, **c)
    k, v = _dense(K, c, table, L, max(lens), dtype)
    for b, n in enumerate(lens):
        if n == 0:
            assert (o[b] == 0).all() and (lse[b] == float('-inf')).all()
            continue
        ref, rl, tol, tl, _ = _bound(q[b].double(), k[b, :n].double(), v[b, :n].double(), nh, H, _seen(n, Nq, causal, window), dtype, T)
        err = (o[b].double() - ref).abs()
        assert (err <= tol).all(), (b, n, (err / tol).max().item())
        assert ((lse[b].double() - rl).abs() <= tl).all(), (b, n, ((lse[b].double() - rl).abs() / tl).max().item())
