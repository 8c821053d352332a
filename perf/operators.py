"""The serving operators of a rollout - the paged key / value cache, the attention that reads it, and the draw of an action or
word from the logits - as measured workloads: their cases, their inputs, what they cost at least, and what they compute.

`run` with `own` false computes them from elementary torch operations in 32 bits; with `own` true it calls dsrg_amd.kernels.

How the cache lies in memory (P pages of S tokens, Hkv key / value heads of D values; e values make 16 bytes of bf16 or fp32,
and the 8-bit types take bf16's e = 8):
  k_pool [P, Hkv, S/16, D/e, 16, e]                token 16 t + r, value e c + j           at [p, h, t, c, r, j]
  v_pool [P, Hkv, S/32, D/16, 4, 16, 2, 4]         token 32 t + 16 m + 4 g + i, value 16 c + d   at [p, h, t, c, g, d, m, i]
  v_pool [P, Hkv, S/16, D/16, 4, 16, 4]   (fp32)   token 16 t + 4 g + i, value 16 c + d    at [p, h, t, c, g, d, i]
  k_scale, v_scale [P, Hkv, S] fp32 (8-bit types): a stored code times its token's and head's scale is the value.
Token t of sequence b lies in page table[b, t // S]."""
import math

import torch

own = False

TYPES = {'bf16': torch.bfloat16, 'fp32': torch.float32, 'int8': torch.int8, 'e4m3': torch.float8_e4m3fn}
SIZE = {'bf16': 2, 'fp32': 4, 'int8': 1, 'e4m3': 1}
TINY = 2.0 ** -126          # the smallest scale: a row of zeros has this one


def listed():
    attend = lambda name, **k: dict(name=name, op='attend', **k)      # noqa: E731
    store = lambda name, **k: dict(name=name, op='store', **k)        # noqa: E731
    sample = lambda name, **k: dict(name=name, op='sample', **k)      # noqa: E731
    return [
        # one episode, one new token over an instruction of full length (200 words): latency alone counts
        attend('attend_one', kv='bf16', B=1, Nq=1, nh=12, nkv=12, D=64, S=32, longest=200, shortest=200, causal=False, window=0),
        # a nav-step's cross-attention: the 20 local tokens of 64 episodes over ragged instructions of up to 80 words
        attend('attend_nav_step', kv='bf16', B=64, Nq=20, nh=12, nkv=12, D=64, S=32, longest=80, shortest=17, causal=False, window=0),
        # the same heads over long histories kept in 8 bits
        attend('attend_int8', kv='int8', B=64, Nq=1, nh=12, nkv=12, D=64, S=64, longest=2011, shortest=1, causal=False, window=0),
        # exact arithmetic (the parity mode's type)
        attend('attend_fp32', kv='fp32', B=16, Nq=1, nh=12, nkv=12, D=64, S=32, longest=999, shortest=333, causal=False, window=0),
        # a few new tokens at once (a drafted continuation) over shared heads, the last 1500 positions only
        attend('attend_window', kv='bf16', B=48, Nq=5, nh=32, nkv=8, D=128, S=64, longest=4097, shortest=3, causal=True, window=1500),
        # few long sequences in 8 bits: little to share out but the length itself
        attend('attend_long_e4m3', kv='e4m3', B=3, Nq=1, nh=32, nkv=8, D=128, S=64, longest=60001, shortest=40000, causal=False, window=0),
        # the largest: a full batch of long ragged sequences
        attend('attend_largest', kv='bf16', B=32, Nq=1, nh=64, nkv=8, D=128, S=64, longest=32768, shortest=1000, causal=False, window=0),
        # one new token of 64 episodes written as it is
        store('store_step', kv='bf16', B=64, T=1, ragged=False, back=False, nkv=12, D=64, S=32, longest=200, shortest=1),
        # the same in 8 bits, then the sequences read back as they stand
        store('store_step_e4m3', kv='e4m3', B=24, T=1, ragged=False, back=True, nkv=12, D=64, S=32, longest=777, shortest=5),
        # whole prompts written in 8 bits and read back
        store('store_prompt_int8', kv='int8', B=32, T=1031, ragged=True, back=True, nkv=8, D=128, S=64, longest=1100, shortest=1),
        # an action of each of 64 episodes among up to 100 graph nodes, most of them masked
        sample('sample_action', B=64, V=100, dtype='fp32', masked=0.7, spread=2.0, k=0, p=0.9, m=0.0),
        # a word of the instruction's vocabulary for each of 256 rows, every filter on
        sample('sample_word', B=256, V=30522, dtype='fp32', masked=0.0, spread=2.5, k=60, p=0.92, m=0.02),
    ]


def draw(rng):
    def logly(lo, hi):
        return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))

    op = rng.choice(('attend', 'attend', 'store', 'sample'))
    if op == 'sample':
        B = logly(1, 512)
        V = logly(2, min(131072, 20_000_000 // B))
        return dict(op=op, B=B, V=V, dtype=rng.choice(('fp32', 'bf16')), masked=rng.choice((0.0, 0.0, 0.5)), spread=round(rng.uniform(0.5, 4.0), 2),
                    k=rng.choice((0, logly(1, 2000))), p=rng.choice((1.0, round(rng.uniform(0.3, 0.99), 3))), m=rng.choice((0.0, round(rng.uniform(0.001, 0.2), 4))))
    kv = rng.choice(('bf16', 'bf16', 'int8', 'e4m3', 'fp32'))
    D = rng.choice((64, 128))
    nkv = rng.choice((1, 2, 4, 8, 12))
    S = rng.choice((32, 64, 128))
    if op == 'store':
        B, T = logly(1, 96), rng.choice((1, logly(2, 900)))
        longest = T + logly(1, 1200)
        return dict(op=op, kv=kv, B=B, T=T, ragged=rng.random() < 0.5, back=True, nkv=nkv, D=D, S=S, longest=longest, shortest=rng.randint(1, longest))
    nh = nkv * rng.choice((1, 1, 2, 3, 4, 7, 8))
    Nq = rng.choice((1, 1, 1, rng.randint(2, 24)))
    B = logly(1, 64)
    longest = logly(1, max(1, min(60000, 400_000_000 // (B * nkv * D), 60_000_000 // (B * nh * Nq))))
    causal = rng.random() < 0.4
    return dict(op=op, kv=kv, B=B, Nq=Nq, nh=nh, nkv=nkv, D=D, S=S, longest=longest, shortest=rng.randint(0, longest),
                causal=causal, window=rng.choice((0, rng.randint(1, longest))) if causal else 0)


# ---- what a case costs at least ----------------------------------------------------------------------------------------

def _lengths(c):
    """The batch's lengths, spread evenly from the shortest to the longest (which sequence has which goes by the seed)."""
    B, lo, hi = c['B'], c['shortest'], c['longest']
    return [hi if B == 1 else int(round(lo + (hi - lo) * i / (B - 1))) for i in range(B)]


def _counts(c):
    """How many of the T rows of each sequence are real (the first has them all)."""
    B, T = c['B'], c['T']
    return [T if not c['ragged'] or B == 1 else max(0, int(round(T * (1 - i / (B - 1))))) for i in range(B)]


def work(c):
    if c['op'] == 'sample':
        return {'bytes': float(c['B'] * c['V'] * SIZE[c['dtype']] + c['B'] * 32), 'flops': float(6 * c['B'] * c['V'])}
    size, row = SIZE[c['kv']], c['nkv'] * c['D']
    extra = 4 * c['nkv'] if c['kv'] in ('int8', 'e4m3') else 0
    wide = 4 if c['kv'] == 'fp32' else 2
    if c['op'] == 'store':
        new = sum(_counts(c))
        moved = new * (row * wide + row * size + extra) * 2
        if c['back']:
            moved += sum(_ends(c)) * (row * size + extra + row * wide) * 2
        return {'bytes': float(moved), 'flops': float(4 * new * row)}
    seen = pairs = 0
    for n in _lengths(c):
        if c['causal'] and c['window']:
            seen += min(n, c['window'] + c['Nq'] - 1)
        else:
            seen += n
        if c['causal']:
            for i in range(c['Nq']):
                pos = n - c['Nq'] + i + 1
                pairs += max(0, min(pos, c['window']) if c['window'] else pos)
        else:
            pairs += n * c['Nq']
    rows = c['B'] * c['Nq'] * c['nh'] * c['D']
    return {'bytes': float(seen * 2 * (row * size + extra) + 2 * rows * wide), 'flops': float(4 * pairs * c['nh'] * c['D'])}


def _ends(c):
    """Length of each sequence after the write: what is read back."""
    return [min(n, c['longest'] - t) + t for n, t in zip(_lengths(c), _counts(c))]


# ---- inputs ------------------------------------------------------------------------------------------------------------

def _shapes(c, P):
    kv, H, S, D = c['kv'], c['nkv'], c['S'], c['D']
    e = 4 if kv == 'fp32' else 8
    return (P, H, S // 16, D // e, 16, e), ((P, H, S // 16, D // 16, 4, 16, 4) if kv == 'fp32' else (P, H, S // 32, D // 16, 4, 16, 2, 4))


def _pages(c, gen):
    """Pools full of a cache's values, and the page tables of the batch: pages are dealt out at random, page 0 to nobody."""
    S, B = c['S'], c['B']
    width = max(1, -(-c['longest'] // S))
    P = B * width + 1
    table = (torch.randperm(P - 1, generator=gen, device='cuda') + 1).to(torch.int32).view(B, width)

    def pool(shape):
        if c['kv'] in ('bf16', 'fp32'):
            return torch.randn(shape, generator=gen, device='cuda', dtype=TYPES[c['kv']]), None
        scale = torch.rand((P, c['nkv'], S), generator=gen, device='cuda') * 0.02 + 0.015
        codes = torch.randint(-127, 128, shape, generator=gen, device='cuda', dtype=torch.int8)
        if c['kv'] == 'int8':
            return codes, scale
        codes = codes.view(torch.uint8)
        codes = torch.where((codes & 127) >= 120, codes & 0xB7, codes).view(torch.float8_e4m3fn)        # codes up to 208, no NaN
        return codes, scale * 0.5

    ks, vs = _shapes(c, P)
    (k_pool, k_scale), (v_pool, v_scale) = pool(ks), pool(vs)
    return dict(k_pool=k_pool, v_pool=v_pool, k_scale=k_scale, v_scale=v_scale, table=table)


def _shuffled(values, gen):
    v = torch.tensor(values, dtype=torch.int32, device='cuda')
    return v[torch.randperm(len(values), generator=gen, device='cuda')]


def prepare(case, seed):
    c, gen = dict(case), torch.Generator(device='cuda')
    gen.manual_seed(int(seed) * 7919 + 17)
    if c['op'] == 'sample':
        B, V = c['B'], c['V']
        logits = torch.randn(B, V, generator=gen, device='cuda') * c['spread']
        if c['masked']:
            out = torch.rand(B, V, generator=gen, device='cuda') < c['masked']
            out[:, 0] = False
            logits.masked_fill_(out, float('-inf'))
        par = lambda lo, hi: torch.rand(B, generator=gen, device='cuda') * (hi - lo) + lo        # noqa: E731
        return dict(case=c, logits=logits.to(TYPES[c['dtype']]), u=torch.rand(B, generator=gen, device='cuda'), temperature=par(0.6, 1.3),
                    top_k=torch.full((B,), c['k'], dtype=torch.int32, device='cuda'), top_p=torch.full((B,), c['p'], device='cuda'),
                    min_p=torch.full((B,), c['m'], device='cuda'))
    s = dict(case=c, **_pages(c, gen))
    wide = torch.float32 if c['kv'] == 'fp32' else torch.bfloat16
    if c['op'] == 'attend':
        s['lens'] = _shuffled(_lengths(c), gen)
        s['q'] = torch.randn(c['B'], c['Nq'], c['nh'] * c['D'], generator=gen, device='cuda', dtype=wide)
        return s
    order = torch.randperm(c['B'], generator=gen, device='cuda')
    t = torch.tensor([[min(n, c['longest'] - t), t] for n, t in zip(_lengths(c), _counts(c))], dtype=torch.int32, device='cuda')[order]
    s['start'], s['count'] = t[:, 0].contiguous(), t[:, 1].contiguous()
    s['zero'], s['end'] = torch.zeros_like(s['start']), s['start'] + s['count']
    # keys and values as a packed projection gives them: [B, T, keys | values]
    kv = torch.randn(c['B'], c['T'], 2, c['nkv'] * c['D'], generator=gen, device='cuda', dtype=wide)
    s['k'], s['v'] = kv[:, :, 0], kv[:, :, 1]
    return s


# ---- the operators -----------------------------------------------------------------------------------------------------

def run(s):
    c = s['case']
    if c['op'] == 'sample':
        return _own_sample(s) if own else _sample(s['logits'], s['u'], s['temperature'], s['top_k'], s['top_p'], s['min_p'])
    if c['op'] == 'attend':
        return _own_attend(s) if own else _attend(s)
    return _own_store(s) if own else _store(s)


def _own_sample(s):
    from dsrg_amd import kernels as K
    return K.sample_rows(s['logits'], s['u'], s['temperature'], s['top_k'], s['top_p'], s['min_p'])


def _own_attend(s):
    from dsrg_amd import kernels as K
    c = s['case']
    return K.attention_paged(s['q'], s['k_pool'], s['v_pool'], s['table'], s['lens'], c['nh'], k_scale=s['k_scale'], v_scale=s['v_scale'],
                             causal=c['causal'], window=c['window'])


def _own_store(s):
    from dsrg_amd import kernels as K
    c = s['case']
    K.kv_append(s['k'], s['v'], s['k_pool'], s['v_pool'], s['table'], s['start'], s['count'], k_scale=s['k_scale'], v_scale=s['v_scale'])
    if not c['back']:
        return s['k_pool'], s['v_pool']
    return K.kv_read(s['k_pool'], s['v_pool'], s['table'], s['zero'], s['end'], c['longest'], k_scale=s['k_scale'], v_scale=s['v_scale'])


def _take(pool, table):
    return pool[table] if pool.dtype != torch.float8_e4m3fn else pool.view(torch.uint8)[table].view(torch.float8_e4m3fn)


def _dense(s, to=torch.float32):
    """The sequences' keys and values as [B, Hkv, tokens, D], in 32 bits."""
    c, table = s['case'], s['table'].long()
    B, H, D, n = c['B'], c['nkv'], c['D'], table.shape[1] * c['S']
    k = _take(s['k_pool'], table).permute(0, 2, 1, 3, 5, 4, 6).reshape(B, H, n, D).to(to)
    v = _take(s['v_pool'], table)
    v = (v.permute(0, 2, 1, 3, 5, 7, 4, 6) if c['kv'] == 'fp32' else v.permute(0, 2, 1, 3, 7, 5, 8, 4, 6)).reshape(B, H, n, D).to(to)
    if s['k_scale'] is not None:
        k = k * s['k_scale'][table].transpose(1, 2).reshape(B, H, n, 1).to(to)
        v = v * s['v_scale'][table].transpose(1, 2).reshape(B, H, n, 1).to(to)
    return k, v


def _seen(c, lens, n):
    """[B, 1 or Nq, n]: the positions that each query row sees."""
    at = torch.arange(n, device='cuda')
    last = (lens[:, None] - c['Nq'] + torch.arange(c['Nq'], device='cuda') if c['causal'] else lens[:, None] - 1)[..., None]
    ok = at <= last
    if c['window']:
        ok = ok & (at > last - c['window'])
    return ok


def _attend(s):
    c, q = s['case'], s['q']
    B, Nq, nh, H, D = c['B'], c['Nq'], c['nh'], c['nkv'], c['D']
    G = nh // H
    k, v = _dense(s)
    rows = q.float().view(B, Nq, H, G, D).permute(0, 2, 3, 1, 4).reshape(B, H, G * Nq, D)
    x = torch.matmul(rows, k.transpose(2, 3)) * D ** -0.5
    ok = _seen(c, s['lens'], k.shape[2])[:, None, None]
    x = x.view(B, H, G, Nq, -1).masked_fill(~ok, float('-inf'))
    top = x.amax(-1, keepdim=True).clamp_min(-3e38)
    e = torch.exp(x - top)
    o = torch.matmul(e.view(B, H, G * Nq, -1), v).view(B, H, G, Nq, D) / e.sum(-1, keepdim=True).clamp_min(1e-38)
    return o.permute(0, 3, 1, 2, 4).reshape(B, Nq, nh * D).to(q.dtype)


def _codes(x, kv):
    """[.., D] -> what is stored of it and its scale: the largest magnitude of a row takes the type's largest value."""
    if kv in ('bf16', 'fp32'):
        return x, None
    x = x.float()
    most = 127.0 if kv == 'int8' else 448.0
    scale = (x.abs().amax(-1, keepdim=True) * (1.0 / most)).clamp_min(TINY)
    y = (x / scale).clamp(-most, most)
    return (y.round().to(torch.int8) if kv == 'int8' else y.to(torch.float8_e4m3fn)), scale[..., 0]


def _raw(x):
    return x.view(torch.uint8) if x.dtype == torch.float8_e4m3fn else x


def _store(s):
    c, S = s['case'], s['case']['S']
    B, T, H, D = c['B'], c['T'], c['nkv'], c['D']
    t = torch.arange(T, device='cuda')
    pos = (s['start'][:, None] + t).long()
    real = t < s['count'][:, None]
    page = s['table'].long().gather(1, (pos // S).clamp_max(s['table'].shape[1] - 1))
    page = torch.where(real, page, 0)[..., None]                       # padding rows go to page 0, which is nobody's
    h, at = torch.arange(H, device='cuda'), (pos % S)[..., None]
    e = 4 if c['kv'] == 'fp32' else 8
    k, ks = _codes(s['k'].view(B, T, H, D), c['kv'])
    v, vs = _codes(s['v'].view(B, T, H, D), c['kv'])
    _raw(s['k_pool'])[page, h, at // 16, :, at % 16] = _raw(k).view(B, T, H, D // e, e)
    v = _raw(v).view(B, T, H, D // 16, 16)
    if c['kv'] == 'fp32':
        _raw(s['v_pool'])[page, h, at // 16, :, at % 16 // 4, :, at % 4] = v
    else:
        _raw(s['v_pool'])[page, h, at // 32, :, at % 16 // 4, :, at % 32 // 16, at % 4] = v
    if ks is not None:
        s['k_scale'][page, h, at] = ks
        s['v_scale'][page, h, at] = vs
    if not c['back']:
        return s['k_pool'], s['v_pool']
    k, v = _dense(s)
    n = c['longest']
    live = (torch.arange(n, device='cuda') < s['end'][:, None])[..., None]
    return tuple(torch.where(live, x[:, :, :n].transpose(1, 2).reshape(B, n, H * D), 0).to(s['k'].dtype) for x in (k, v))


def _sample(logits, u, temperature, top_k, top_p, min_p):
    """A row's candidates in falling order (ties: the lowest index first) are cut after the k-th, then after the first whose
    running share of what is left reaches p, then where the weight falls under m of the largest; one is drawn by the given
    number, in the order of their indices.  Sums are of 64 bits: a number next to a border must not fall to its other side."""
    x = logits.double()
    x = torch.where(torch.isnan(x), float('-inf'), x)
    top = x.amax(1, keepdim=True)
    w = torch.exp((x - top) / temperature.double()[:, None])
    order = torch.sort(x, dim=1, descending=True, stable=True).indices
    ws = w.gather(1, order)
    rank = torch.arange(x.shape[1], device=x.device)
    k = torch.where(top_k > 0, top_k, x.shape[1])[:, None]
    ws = torch.where(rank < k, ws, 0)
    run_ = ws.cumsum(1)
    p = top_p.double()[:, None]
    keep = (ws > 0) & ((run_ - ws < p * run_[:, -1:]) | (p >= 1) | (rank == 0)) & ((ws >= min_p.double()[:, None]) | (rank == 0))
    w = torch.where(torch.zeros_like(keep).scatter(1, order, keep), w, 0)
    cdf = w.cumsum(1)
    token = (cdf > u.double()[:, None] * cdf[:, -1:]).to(torch.uint8).argmax(1)
    logp = torch.log(w.gather(1, token[:, None])[:, 0] / cdf[:, -1])
    return token, logp.float()


# ---- the definitions, in 64 bits ---------------------------------------------------------------------------------------

def exact(case, seed):
    c = dict(case)
    s = prepare(c, seed)
    if c['op'] == 'sample':
        return _exact_sample(s)
    if c['op'] == 'store' and not c['back']:
        return None                                 # values are moved, none is computed
    return _exact_store(s) if c['op'] == 'store' else _exact_attend(s)


def _token_rows(s, b, n):
    """Keys and values of the first n tokens of sequence b, [n, Hkv, D] in 64 bits, by the layout's own indices."""
    c = s['case']
    t = torch.arange(n, device='cuda')
    page, r, h = s['table'][b].long()[t // c['S']], t % c['S'], torch.arange(c['nkv'], device='cuda')
    d = torch.arange(c['D'], device='cuda')
    e = 4 if c['kv'] == 'fp32' else 8
    P, R, Hh, Dd = page[:, None, None], r[:, None, None], h[None, :, None], d[None, None, :]
    wide = lambda x: x.double() if x.dtype != torch.float8_e4m3fn else x.float().double()        # noqa: E731
    get = lambda pool, *at: wide(pool[at] if pool.dtype != torch.float8_e4m3fn else pool.view(torch.uint8)[at].view(torch.float8_e4m3fn))     # noqa: E731
    k = get(s['k_pool'], P, Hh, R // 16, Dd // e, R % 16, Dd % e)
    if c['kv'] == 'fp32':
        v = get(s['v_pool'], P, Hh, R // 16, Dd // 16, R % 16 // 4, Dd % 16, R % 4)
    else:
        v = get(s['v_pool'], P, Hh, R // 32, Dd // 16, R % 16 // 4, Dd % 16, R % 32 // 16, R % 4)
    if s['k_scale'] is not None:
        k = k * s['k_scale'][P, Hh, R].double()
        v = v * s['v_scale'][P, Hh, R].double()
    return k, v


def _exact_attend(s):
    c = s['case']
    Nq, nh, H, D = c['Nq'], c['nh'], c['nkv'], c['D']
    out = torch.zeros(c['B'], Nq, nh, D, dtype=torch.float64, device='cuda')
    for b, n in enumerate(s['lens'].tolist()):
        if n == 0:
            continue
        k, v = _token_rows(s, b, n)
        q = s['q'][b].double().view(Nq, nh, D)
        for i in range(Nq):
            last = n - Nq + i if c['causal'] else n - 1
            first = max(0, last - c['window'] + 1) if c['window'] else 0
            if last < 0:
                continue
            kk, vv = k[first:last + 1], v[first:last + 1]
            x = (kk[:, :, None] * q[i].view(1, H, nh // H, D)).sum(-1) / math.sqrt(D) if kk.shape[0] * nh * D < 30_000_000 else \
                torch.stack([kk[:, h] @ q[i].view(H, nh // H, D)[h].T for h in range(H)], 1) / math.sqrt(D)
            p = torch.softmax(x, 0)                              # [tokens, Hkv, group]
            out[b, i] = torch.stack([p[:, h].T @ vv[:, h] for h in range(H)], 0).reshape(nh, D)
    return out.view(c['B'], Nq, nh * D)


def _exact_store(s):
    c = s['case']
    H, D, n = c['nkv'], c['D'], c['longest']
    outs = [torch.zeros(c['B'], n, H, D, dtype=torch.float64, device='cuda') for _ in range(2)]
    e4m3 = torch.arange(127, dtype=torch.uint8, device='cuda').view(torch.float8_e4m3fn).double() if c['kv'] == 'e4m3' else None
    for b, (start, count) in enumerate(zip(s['start'].tolist(), s['count'].tolist())):
        old = _token_rows(s, b, start)
        for out, was, new in zip(outs, old, (s['k'][b], s['v'][b])):
            x = new[:count].double().view(count, H, D)
            if c['kv'] == 'int8':
                scale = x.abs().amax(-1, keepdim=True) / 127
                x = torch.round(x / scale.clamp_min(TINY)) * scale
            elif c['kv'] == 'e4m3':
                scale = x.abs().amax(-1, keepdim=True) / 448
                y = (x / scale.clamp_min(TINY)).abs()
                at = torch.bucketize(y, (e4m3[1:] + e4m3[:-1]) / 2)      # the nearest of the type's values
                x = torch.sign(x) * e4m3[at] * scale
            out[b, :start], out[b, start:start + count] = was, x
    return tuple(o.view(c['B'], n, H * D) for o in outs)


def _exact_sample(s):
    tokens, logps = [], []
    for b in range(s['case']['B']):
        x = s['logits'][b].double()
        T, u = s['temperature'][b].double(), s['u'][b].double()
        kept = torch.argsort(x, descending=True, stable=True)
        kept = kept[x[kept] > float('-inf')]
        if int(s['top_k'][b]) > 0:
            kept = kept[:int(s['top_k'][b])]
        logw = (x - x.max()) / T
        w = torch.exp(logw)
        if float(s['top_p'][b]) < 1:
            run_ = torch.cumsum(w[kept], 0)
            kept = kept[:int((run_ < s['top_p'][b].double() * run_[-1]).sum()) + 1]
        kept = torch.cat([kept[:1], kept[1:][w[kept[1:]] >= s['min_p'][b].double()]])
        kept = torch.sort(kept).values
        run_ = torch.cumsum(w[kept], 0)
        j = min(int((run_ <= u * run_[-1]).sum()), kept.numel() - 1)
        tokens.append(kept[j])
        logps.append(logw[kept[j]] - torch.log(run_[-1]))
    return torch.stack(tokens), torch.stack(logps)
