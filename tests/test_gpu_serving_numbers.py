"""gpu: the numbers that sample_rows documents as "off" (or as the largest entry) are taken as numbers and as tensors, with the same answers."""
import numpy as np
import pytest
import torch

from dsrg_amd._lib import DsrgHipError
from tests.test_gpu_serving import BF16, F32, _check_rows, _g, _sample_ref

pytestmark = pytest.mark.gpu


@pytest.fixture(scope='module')
def K():
    assert torch.cuda.is_available(), 'GPU tests need an MI355X'
    from dsrg_amd import kernels
    return kernels


@pytest.mark.parametrize('V', [100, 3000])
@pytest.mark.parametrize('kw', [dict(top_k=-1), dict(top_k=-2 ** 31), dict(temperature=-1.0), dict(temperature=float('-inf')), dict(temperature=0), dict(min_p=-0.1),
                                dict(top_p=1.5), dict(temperature=-0.5, top_k=-7, top_p=2, min_p=-1)])
def test_sample_rows_numbers_that_switch_off(K, kw, V):
    B = 6
    logits, u = torch.randn(B, V, generator=_g(V)).cuda(), torch.rand(B, generator=_g(1)).cuda()
    tensors = {n: torch.full((B,), x, device='cuda', dtype=torch.int32 if n == 'top_k' else F32) for n, x in kw.items()}
    got, want = K.sample_rows(logits, u, **kw), K.sample_rows(logits, u, **tensors)
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    full = {**dict(temperature=1.0, top_k=0, top_p=1.0, min_p=0.0), **kw}
    assert torch.equal(got[0], _check_rows(K, logits, u, full['temperature'], max(full['top_k'], 0), float(full['top_p']), float(full['min_p'])))


def test_sample_rows_numbers_that_are_refused(K):
    logits, u = torch.zeros(2, 5, device='cuda'), torch.zeros(2, device='cuda')
    nan, inf = float('nan'), float('inf')
    for kw in (dict(temperature=nan), dict(temperature=inf), dict(top_p=nan), dict(top_p=-0.5), dict(min_p=nan), dict(min_p=1.5)):
        with pytest.raises(DsrgHipError, match=next(iter(kw))):
            K.sample_rows(logits, u, **kw)


@pytest.mark.parametrize('dtype', [F32, BF16])
@pytest.mark.parametrize('V', [1, 2, 50, 160, 161, 689, 4096, 4097, 20000, 70000])
def test_sample_rows_of_one_candidate(K, dtype, V):
    """top-k of 1 without top-p (the largest entry), with and without min-p; rows of one candidate; a few candidates and a k that is no smaller"""
    B = 9
    logits, u = (torch.randn(B, V, generator=_g(V)) * 3).to(dtype).cuda(), torch.rand(B, generator=_g(1)).cuda()
    top = torch.tensor([_sample_ref(row, 0.5, 0.0, 0, 1.0, 0.0)[0] for row in logits]).cuda()
    for m in (0.0, 0.2, 1.0):
        for k in (1, torch.ones(B, dtype=torch.int32, device='cuda')):
            tok, lp = K.sample_rows(logits, u, 0.9, k, 1.0, m)
            assert torch.equal(tok, top) and (lp == 0).all()
    for left in (1, 2, 3):
        rows, at = torch.full_like(logits, float('-inf')), V // 2
        rows[:, at:at + left] = logits[:, at:at + left]
        for k in (0, 1, 2, 3, 4):
            for p, m in ((1.0, 0.0), (0.7, 0.1)):
                tok, lp = K.sample_rows(rows, u, 0.9, k, p, m)
                for b in range(B):
                    rt, rl, _ = _sample_ref(rows[b, at:at + left], u[b].item(), float(np.float32(0.9)), k, float(np.float32(p)), float(np.float32(m)))
                    assert tok[b].item() == at + rt and abs(lp[b].item() - rl) <= abs(rl) * 2.0 ** -23 + V * 2.0 ** -44 + 1e-12, (left, k, p, b)
