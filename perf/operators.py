"""Work items of the attention answer decoder: cross attention to region states, attention with a learned relative position bias,
and the vocabulary loss of a linear layer without its logits.

Every case is one pass a user's program makes: a forward step (``step`` / ``eval``) or a forward with its gradients (``train``).
``own`` selects between the plain torch formulas (float32 throughout, rounded once at the end) and the framework's operators.
"""
import math

import numpy as np
import torch

own = False

DTYPES = {'f32': torch.float32, 'bf16': torch.bfloat16, 'f16': torch.float16}
SIZE = {'f32': 4, 'bf16': 2, 'f16': 2}


# --------------------------------------------------------------------------- cases
def listed():
    return [
        # one answer token of 64 image pairs over the 52 + 52 region states of a pair, 4 heads of 256: a decode step, latency counts
        dict(name='cross_step_regions_f32', op='cross', grad=False, dtype='f32', B=64, H=4, KV=4, dh=256, Lq=1, Lk=104, ragged=True, mask=False),
        # one new token per sample over long encoder states, heads sharing keys 4 : 1, ragged lengths: bound by reading the states
        dict(name='cross_step_long_bf16', op='cross', grad=False, dtype='bf16', B=16, H=32, KV=8, dh=128, Lq=1, Lk=8192, ragged=True, mask=False),
        # the answer decoder's training pass at the framework's own widths: 90 answer tokens over 104 regions, undetected regions masked
        dict(name='cross_train_regions_f32', op='cross', grad=True, dtype='f32', B=64, H=4, KV=4, dh=256, Lq=90, Lk=104, ragged=False, mask=True),
        # training over long states of another length, odd query length, shared keys
        dict(name='cross_train_long_bf16', op='cross', grad=True, dtype='bf16', B=8, H=16, KV=4, dh=64, Lq=1021, Lk=2048, ragged=True, mask=False),
        # one new token against the decoder's own cache, bias by distance
        dict(name='rel_step_cache_f16', op='rel', grad=False, dtype='f16', B=32, H=16, KV=16, dh=64, Lq=1, Lk=4096, ragged=True, mask=False,
             causal=True, nb=32, md=128),
        # the 20 question words of 256 pairs, both directions, 8 heads of 64
        dict(name='rel_train_question_f32', op='rel', grad=True, dtype='f32', B=256, H=8, KV=8, dh=64, Lq=20, Lk=20, ragged=True, mask=False,
             causal=False, nb=32, md=128),
        # a decoder's own tokens in training, long and causal
        dict(name='rel_train_causal_bf16', op='rel', grad=True, dtype='bf16', B=4, H=16, KV=16, dh=128, Lq=2048, Lk=2048, ragged=False, mask=False,
             causal=True, nb=32, md=128),
        # the framework's own answer head: 64 pairs x 90 steps, 512 wide, 148 words
        dict(name='loss_train_answers_f32', op='loss', grad=True, dtype='f32', B=64, T=90, D=512, V=148, bias=True),
        # a subword vocabulary in full precision
        dict(name='loss_train_subword_f32', op='loss', grad=True, dtype='f32', B=16, T=90, D=512, V=10007, bias=True),
        # evaluation: the loss alone over a large vocabulary
        dict(name='loss_eval_large_f16', op='loss', grad=False, dtype='f16', B=64, T=90, D=512, V=50021, bias=False),
        # training over a large vocabulary, odd sizes
        dict(name='loss_train_large_bf16', op='loss', grad=True, dtype='bf16', B=9, T=511, D=1024, V=32003, bias=True),
        # the largest: a long batch, wide states
        dict(name='loss_train_wide_bf16', op='loss', grad=True, dtype='bf16', B=16, T=1024, D=2048, V=65536, bias=False),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    """One more case of the listed cases' ranges."""
    top = {}
    for c in listed():
        w = work(c)
        for k in w:
            top[k] = max(top.get(k, 0), w[k])
    while True:
        op = rng.choice(['cross', 'rel', 'loss'])
        dtype = rng.choice(['f32', 'bf16', 'f16'])
        grad = rng.random() < 0.6
        if op == 'loss':
            c = dict(op=op, grad=grad, dtype=dtype, B=_log_int(rng, 2, 64), T=_log_int(rng, 16, 1024), D=64 * _log_int(rng, 4, 32),
                     V=_log_int(rng, 148, 65536), bias=rng.random() < 0.5)
            limit = 0.15 if dtype == 'f32' else 0.8
        else:
            KV = rng.choice([1, 2, 4, 8, 16])
            c = dict(op=op, grad=grad, dtype=dtype, B=_log_int(rng, 1, 64), H=KV * rng.choice([1, 1, 2, 4]), KV=KV,
                     dh=rng.choice([32, 64, 64, 128, 128, 256]), Lq=1 if not grad else _log_int(rng, 8, 2048), Lk=_log_int(rng, 16, 8192 if not grad else 2048),
                     ragged=rng.random() < 0.6, mask=rng.random() < 0.3)
            if op == 'rel':
                c.update(causal=rng.random() < 0.5, nb=rng.choice([16, 32]), md=rng.choice([64, 128]))
                if grad:
                    c['Lk'] = c['Lq']
            limit = 0.01 if dtype == 'f32' else 0.02            # of the widest loss: attention passes stay near the listed ones
        w = work(c)
        if w['flops'] <= limit * top['flops'] and w['bytes'] <= top['bytes'] and w['bytes'] >= 1e5:
            if op == 'loss' or c['B'] * c['H'] * c['Lq'] * c['Lk'] <= 2 ** 28:        # the plain form keeps its scores
                return c


def _lengths(c, n, full):
    """Valid lengths of the case's samples, the same multiset for every seed: spread evenly over 30 ... 100 % of ``full``."""
    return [max(1, int(round(full * (0.3 + 0.7 * (i + 1) / n)))) for i in range(n)]


def _pairs(c):
    """(query, key) pairs a case attends over, valid key rows."""
    lens = _lengths(c, c['B'], c['Lk']) if c['ragged'] else [c['Lk']] * c['B']
    pairs = keys = 0
    for n in lens:
        if c.get('causal'):
            p0 = n - 1 if c['Lq'] == 1 else 0
            pairs += sum(min(n, p0 + i + 1) for i in range(c['Lq']))
        else:
            pairs += n * c['Lq']
        keys += n
    return pairs * (0.9 if c['mask'] else 1.0), keys


def work(case):
    c = case
    s = SIZE[c['dtype']]
    if c['op'] == 'loss':
        rows = sum(_lengths(c, c['B'], c['T']))
        x, w = rows * c['D'] * s, c['V'] * c['D'] * s
        return {'bytes': (2 if c['grad'] else 1) * (x + w) + 12 * c['B'] * c['T'], 'flops': (6 if c['grad'] else 2) * rows * c['D'] * c['V']}
    pairs, keys = _pairs(c)
    q, kv = c['B'] * c['Lq'] * c['H'] * c['dh'] * s, keys * c['KV'] * c['dh'] * s
    if not c['grad']:
        return {'bytes': 2 * q + 2 * kv, 'flops': 4 * c['dh'] * c['H'] * pairs}
    return {'bytes': 4 * q + 4 * kv, 'flops': 14 * c['dh'] * c['H'] * pairs}


# --------------------------------------------------------------------------- inputs
def prepare(case, seed):
    c = case
    dev, dt = 'cuda', DTYPES[c['dtype']]
    g = torch.Generator(device=dev).manual_seed(seed)
    h = np.random.RandomState(seed % (1 << 31))

    def randn(*shape, scale=1.0):
        return (torch.randn(*shape, generator=g, device=dev) * scale).to(dt)

    st = {'case': c}
    if c['op'] == 'loss':
        lens = torch.tensor(h.permutation(_lengths(c, c['B'], c['T'])), device=dev)
        st['x'] = randn(c['B'], c['T'], c['D'])
        st['weight'] = randn(c['V'], c['D'], scale=1.5 / math.sqrt(c['D']))
        st['bias'] = randn(c['V'], scale=0.5) if c['bias'] else None
        # frequent words first, as a vocabulary sorted by frequency has them
        u = torch.rand(c['B'], c['T'], generator=g, device=dev)
        st['target'] = (torch.exp(u * math.log(c['V'] + 1.0)) - 1.0).long().clamp_(0, c['V'] - 1)
        st['mask'] = (torch.arange(c['T'], device=dev)[None, :] < lens[:, None]).float()
        if c['grad']:
            for k in ('x', 'weight', 'bias'):
                if st[k] is not None:
                    st[k].requires_grad_(True)
            st['dout'] = torch.ones((), device=dev)
        return st
    B, H, KV, dh, Lq, Lk = (c[k] for k in ('B', 'H', 'KV', 'dh', 'Lq', 'Lk'))
    st['q'], st['k'], st['v'] = randn(B, Lq, H * dh, scale=1.3), randn(B, Lk, KV * dh), randn(B, Lk, KV * dh)
    lens = h.permutation(_lengths(c, B, Lk)) if c['ragged'] else np.full(B, Lk)
    st['k_len'] = torch.tensor(lens, device=dev, dtype=torch.int32) if c['ragged'] else None
    st['key_mask'] = None
    if c['mask']:                                # a tenth of the keys missing; from eight samples on, one sample without any
        m = torch.rand(B, Lk, generator=g, device=dev) >= 0.1
        if B >= 8:
            m[int(h.randint(B))] = False
        st['key_mask'] = m
    if c['op'] == 'rel':
        st['table'] = torch.randn(c['nb'], H, generator=g, device=dev) * 0.7
        st['q_pos'] = torch.tensor(lens - 1, device=dev, dtype=torch.int32) if Lq == 1 else None
    if c['grad']:
        st['dout'] = randn(B, Lq, H * dh)
        for k in ('q', 'k', 'v') + (('table',) if c['op'] == 'rel' else ()):
            st[k].requires_grad_(True)
    return st


# --------------------------------------------------------------------------- one pass
def run(state):
    c = state['case']
    if own:
        return _own(state, c)
    with torch.no_grad():
        return _plain_loss(state, c) if c['op'] == 'loss' else _plain_attention(state, c)


def _own(st, c):
    from ekaid_amd import ops
    if c['op'] == 'loss':
        loss = ops.linear_lm_loss(st['x'], st['weight'], st['bias'], st['target'], st['mask'])
        leaves = [st[k] for k in ('x', 'weight', 'bias') if st[k] is not None]
        return [loss.detach()] + (list(torch.autograd.grad(loss, leaves, st['dout'])) if c['grad'] else [])
    if c['op'] == 'cross':
        out = ops.cross_attention(st['q'], st['k'], st['v'], c['H'], kv_heads=c['KV'], k_len=st['k_len'], key_mask=st['key_mask'])
        leaves = [st['q'], st['k'], st['v']]
    else:
        out = ops.relative_attention(st['q'], st['k'], st['v'], st['table'], c['H'], kv_heads=c['KV'], k_len=st['k_len'], key_mask=st['key_mask'],
                                     q_pos=st['q_pos'], causal=c['causal'], max_distance=c['md'])
        leaves = [st['q'], st['k'], st['v'], st['table']]
    return [out.detach()] + (list(torch.autograd.grad(out, leaves, st['dout'])) if c['grad'] else [])


def _plain_loss(st, c):
    D, V, dt = c['D'], c['V'], DTYPES[c['dtype']]
    x, w = st['x'].float().reshape(-1, D), st['weight'].float()
    z = x @ w.t()
    if st['bias'] is not None:
        z = z + st['bias'].float()
    m = z.max(1, keepdim=True).values
    e = torch.exp(z - m)
    total = e.sum(1, keepdim=True)
    t, mask = st['target'].reshape(-1), st['mask'].reshape(-1)
    denom = mask.sum()
    nll = (m + torch.log(total)).squeeze(1) - z.gather(1, t[:, None]).squeeze(1)
    loss = (nll * mask).sum() / denom
    if not c['grad']:
        return [loss]
    dz = e / total
    del z, e
    dz[torch.arange(t.numel(), device=t.device), t] -= 1.0
    dz = dz * (st['dout'] * mask / denom)[:, None]
    out = [loss, (dz @ w).view(st['x'].shape).to(dt), (dz.t() @ x).to(dt)]
    if st['bias'] is not None:
        out.append(dz.sum(0).to(dt))
    return out


def _bucket(rel, nb, md, bidirectional):
    """Bucket of the offset key - query, logarithms in float64 (the nudge keeps exact borders on their upper side)."""
    base = torch.zeros_like(rel)
    if bidirectional:
        nb //= 2
        base = (rel > 0).long() * nb
        d = rel.abs()
    else:
        d = (-rel).clamp_min(0)
    e = nb // 2
    far = e + torch.floor(torch.log(d.clamp_min(1).double() / e) / math.log(md / e) * (nb - e) + 1e-9).long()
    return base + torch.where(d < e, d, far.clamp_max(nb - 1))


def _valid(st, c):
    """(B, 1, Lq or 1, Lk) truth of attended places, and the offsets key - query (B or 1, Lq, Lk) of the relative form."""
    B, Lq, Lk, dev = c['B'], c['Lq'], c['Lk'], st['q'].device
    j = torch.arange(Lk, device=dev)
    ok = torch.ones(B, 1, 1, Lk, dtype=torch.bool, device=dev)
    if st['k_len'] is not None:
        ok = ok & (j < st['k_len'][:, None])[:, None, None, :]
    if st['key_mask'] is not None:
        ok = ok & st['key_mask'][:, None, None, :]
    rel = None
    if c['op'] == 'rel':
        i = torch.arange(Lq, device=dev)[None, :] + (st['q_pos'].long()[:, None] if st['q_pos'] is not None else 0)
        rel = j[None, None, :] - i[:, :, None]
        if c['causal']:
            ok = ok & (rel <= 0)[:, None]
    return ok, rel


def _plain_attention(st, c):
    B, H, KV, dh, Lq, Lk = (c[k] for k in ('B', 'H', 'KV', 'dh', 'Lq', 'Lk'))
    dt, scale, G = DTYPES[c['dtype']], 1.0 / math.sqrt(dh), H // KV

    def heads(t, n, L):
        return t.float().view(B, L, n, dh).transpose(1, 2).contiguous()

    q = heads(st['q'], H, Lq)
    k, v = (heads(st[n], KV, Lk).repeat_interleave(G, 1) for n in ('k', 'v'))
    ok, rel = _valid(st, c)
    s = (q @ k.transpose(2, 3).contiguous()) * scale
    if rel is not None:
        bk = _bucket(rel, c['nb'], c['md'], not c['causal'])
        s = s + st['table'][bk].permute(0, 3, 1, 2)
    s = s.masked_fill(~ok, float('-inf'))
    m = s.max(3, keepdim=True).values
    p = torch.exp(s - torch.where(m == float('-inf'), torch.zeros_like(m), m))
    total = p.sum(3, keepdim=True)
    p = p / torch.where(total == 0, torch.ones_like(total), total)
    del s
    o = p @ v

    def rows(t, n, L):
        return t.transpose(1, 2).reshape(B, L, n * dh)

    out = [rows(o, H, Lq).to(dt)]
    if not c['grad']:
        return out
    do = heads(st['dout'], H, Lq)
    dv = p.transpose(2, 3).contiguous() @ do
    ds = p * (do @ v.transpose(2, 3).contiguous() - (do * o).sum(3, keepdim=True))
    dq = (ds @ k) * scale
    dk = (ds.transpose(2, 3).contiguous() @ q) * scale
    dk, dv = (t.view(B, KV, G, Lk, dh).sum(2) for t in (dk, dv))
    out += [rows(dq, H, Lq).to(dt), rows(dk, KV, Lk).to(dt), rows(dv, KV, Lk).to(dt)]
    if rel is not None:
        # the offsets are the same for every sample of a training pass: sums along the diagonals (millions of terms, in float64), rows of a
        # skewed copy, then over the offsets of a bucket
        skew = torch.zeros(H, Lq, Lq + Lk, device=q.device, dtype=torch.float64)
        skew[:, :, :Lk] = ds.sum(0, dtype=torch.float64).flip(1)
        diag = skew.view(H, -1)[:, :Lq * (Lq + Lk - 1)].view(H, Lq, Lq + Lk - 1).sum(1)
        off = torch.arange(1 - Lq, Lk, device=q.device)
        dtab = torch.zeros(c['nb'], H, device=q.device, dtype=torch.float64)
        dtab.index_add_(0, _bucket(off, c['nb'], c['md'], not c['causal']), diag.t().contiguous())
        out.append(dtab.float())
    return out


# --------------------------------------------------------------------------- float64 from the definitions
def exact(case, seed):
    st = prepare(case, seed)
    with torch.no_grad():
        return _exact_loss(st, case) if case['op'] == 'loss' else _exact_attention(st, case)


def _exact_loss(st, c):
    D, V = c['D'], c['V']
    w = st['weight'].detach().double()
    b = st['bias'].detach().double() if st['bias'] is not None else None
    x, t, wt = st['x'].detach().double().view(-1, D), st['target'].view(-1), st['mask'].double().view(-1)
    num = torch.zeros((), dtype=torch.float64, device=x.device)
    dx, dw, db = torch.zeros_like(x), torch.zeros_like(w), torch.zeros(V, dtype=torch.float64, device=x.device)
    for r0 in range(0, x.shape[0], 2048):
        xr, tr, wr = x[r0:r0 + 2048], t[r0:r0 + 2048], wt[r0:r0 + 2048] / wt.sum()
        logits = torch.mm(xr, w.t()) if b is None else torch.addmm(b, xr, w.t())
        logp = logits - torch.logsumexp(logits, 1, keepdim=True)
        del logits
        num -= (logp.gather(1, tr.view(-1, 1)).view(-1) * wr).sum()
        if c['grad']:
            d = logp.exp_().mul_(wr.view(-1, 1))
            d.scatter_add_(1, tr.view(-1, 1), -wr.view(-1, 1))
            dx[r0:r0 + 2048] = torch.mm(d, w)
            dw += torch.mm(d.t(), xr)
            db += d.sum(0)
    if not c['grad']:
        return [num]
    return [num, dx.view(st['x'].shape), dw] + ([db] if b is not None else [])


def _bucket_exact(r, nb, md, bidirectional):
    """Bucket of one integer offset, decided with whole numbers: (d/e)^n >= (md/e)^s as d^n e^s >= md^s e^n."""
    off = 0
    if bidirectional:
        nb //= 2
        off, d = (nb if r > 0 else 0), abs(r)
    else:
        d = max(-r, 0)
    e = nb // 2
    n = nb - e
    if d < e:
        return off + d
    s = 0
    while s + 1 < n and d ** n * e ** (s + 1) >= md ** (s + 1) * e ** n:
        s += 1
    return off + e + s


def _exact_attention(st, c):
    B, H, KV, dh, Lq, Lk = (c[k] for k in ('B', 'H', 'KV', 'dh', 'Lq', 'Lk'))
    dev = st['q'].device
    Q, K, V = (st[n].detach().double() for n in ('q', 'k', 'v'))
    O, dQ, dK, dV = torch.zeros_like(Q), torch.zeros_like(Q), torch.zeros_like(K), torch.zeros_like(V)
    lens = st['k_len'].tolist() if st['k_len'] is not None else [Lk] * B
    pos = st['q_pos'].tolist() if st.get('q_pos') is not None else [0] * B
    if c['op'] == 'rel':
        tab = st['table'].detach().double()
        dtab = torch.zeros_like(tab)
        reach = Lq + Lk + 1 + max(pos)
        lut = torch.tensor([_bucket_exact(r, c['nb'], c['md'], not c['causal']) if abs(r) <= 2 * c['md'] else -1 for r in range(-reach, reach + 1)], device=dev)
        far = [_bucket_exact(sgn * 2 * c['md'], c['nb'], c['md'], not c['causal']) for sgn in (-1, 1)]
        r_all = torch.arange(-reach, reach + 1, device=dev)
        lut = torch.where(lut >= 0, lut, torch.where(r_all < 0, torch.full_like(lut, far[0]), torch.full_like(lut, far[1])))
    for b in range(B):
        keep = torch.arange(Lk, device=dev) < lens[b]
        if st['key_mask'] is not None:
            keep = keep & st['key_mask'][b]
        idx = keep.nonzero().view(-1)
        if idx.numel() == 0:
            continue
        qb = Q[b].view(Lq, H, dh).permute(1, 0, 2)
        share = torch.arange(H, device=dev) // (H // KV)
        kb, vb = (t[b, idx].view(-1, KV, dh).permute(1, 0, 2)[share].contiguous() for t in (K, V))
        logits = torch.bmm(qb.contiguous(), kb.transpose(1, 2).contiguous()) / math.sqrt(dh)
        if c['op'] == 'rel':
            off = idx[None, :] - (pos[b] + torch.arange(Lq, device=dev))[:, None]
            cls = lut[off + reach]
            logits += tab.t()[:, cls.view(-1)].view(H, Lq, -1)
            if c['causal']:
                logits.masked_fill_((off > 0)[None], float('-inf'))
        none = (logits == float('-inf')).all(2, keepdim=True)
        w = torch.softmax(logits.masked_fill(none, 0.0), 2).masked_fill(none, 0.0)
        ob = torch.bmm(w, vb)
        O[b] = ob.permute(1, 0, 2).reshape(Lq, H * dh)
        if not c['grad']:
            continue
        gb = st['dout'][b].double().view(Lq, H, dh).permute(1, 0, 2).contiguous()
        gw = torch.bmm(gb, vb.transpose(1, 2).contiguous())
        gl = w * (gw - (w * gw).sum(2, keepdim=True))
        dQ[b] = (torch.bmm(gl, kb) / math.sqrt(dh)).permute(1, 0, 2).reshape(Lq, H * dh)
        gk = torch.bmm(gl.transpose(1, 2).contiguous(), qb.contiguous()) / math.sqrt(dh)
        gv = torch.bmm(w.transpose(1, 2).contiguous(), gb)
        for dst, src in ((dK, gk), (dV, gv)):
            dst[b, idx] = torch.zeros(KV, idx.numel(), dh, dtype=torch.float64, device=dev).index_add_(0, share, src).permute(1, 0, 2).reshape(-1, KV * dh)
        if c['op'] == 'rel':
            for i in range(c['nb']):
                dtab[i] += (gl * (cls == i)).sum((1, 2))
    if not c['grad']:
        return [O]
    return [O, dQ, dK, dV] + ([dtab] if c['op'] == 'rel' else [])
