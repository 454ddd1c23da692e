"""Cross attention and relative-bias attention against the definition in float64, element by element.

Every bound is derived, none is fitted: u = 2^-24 for arithmetic in f32, h = half a step of the tensors' type where a value is rounded to
it.  A score carries (dh + 3) u S (S = scale * sum |q||k|), a probability twice that plus (Lk + 8) u relative; probabilities and score
gradients are rounded to the type (h relative; f16 also 2^-25 absolute below its normal range, score gradients after their power-of-two
scaling) where they enter a product; delta = <dout, out> uses the output before its rounding -- formed from rounded probabilities, which reaches dq; with a bias table the rest of the
backward takes delta as the f32 sum of P dP -- and the result is rounded once (h)."""
import ctypes
import math

import pytest
import torch

F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16
DEV = 'cuda'
gpu = pytest.mark.gpu


def bucket(rel, side, md, bidirectional):
    """Definition by whole numbers, one offset."""
    off, d = (side if rel > 0 else 0, abs(rel)) if bidirectional else (0, max(-rel, 0))
    e = side // 2
    if d < e:
        return off + d
    s = 0
    while s + 1 < side - e and d ** (side - e) * e ** (s + 1) >= md ** (s + 1) * e ** (side - e):
        s += 1
    return off + e + s


def make(dtype, B, H, KV, dh, Lq, Lk, seed=0, nb=0, md=0, scale_out=1.0, table_dtype=F32):
    g = torch.Generator().manual_seed(seed + 7 * Lq + Lk + dh)
    r = lambda *s: torch.randn(*s, generator=g)                                    # noqa: E731
    t = dict(q=r(B, Lq, H * dh) * 1.2, k=r(B, Lk, KV * dh), v=r(B, Lk, KV * dh), dout=r(B, Lq, H * dh) * scale_out)
    t = {n: x.to(dtype) for n, x in t.items()}
    if nb:
        t['table'] = (r(nb, H) * 0.8).to(table_dtype)
    return t


def reference(t, H, KV, dh, k_len=None, key_mask=None, q_pos=None, causal=False, bidirectional=None, md=0, scale=None, keep=None):
    """(values, bounds) in float64: out, dq, dk, dv (, dtable)."""
    dtype = t['q'].dtype
    B, Lq, Lk = t['q'].shape[0], t['q'].shape[1], t['k'].shape[1]
    G, u = H // KV, 2.0 ** -24
    h = torch.finfo(dtype).eps / 2
    tiny = 2.0 ** -25 if dtype == F16 else 0.0
    hp = 0.0 if dtype == F32 else h
    scale = dh ** -0.5 if scale is None else scale
    ok = torch.ones(B, 1, Lq, Lk, dtype=torch.bool)
    if k_len is not None:
        ok &= (torch.arange(Lk)[None] < k_len.cpu().clamp(0, Lk)[:, None])[:, None, None]
    if key_mask is not None:
        ok &= key_mask.cpu()[:, None, None]
    row_ok = ok[:, 0, 0] if Lq else torch.zeros(B, Lk, dtype=torch.bool)
    split = lambda x, n: x.double().reshape(B, -1, n, dh).permute(0, 2, 1, 3)        # noqa: E731
    q, do = split(t['q'], H), split(t['dout'], H)
    clean = lambda x: torch.where(row_ok[:, :, None], x.double(), torch.zeros(()).double())    # noqa: E731
    k, v = (split(clean(t[n]), KV).repeat_interleave(G, 1) for n in ('k', 'v'))
    s = scale * (q @ k.transpose(2, 3))
    S = abs(scale) * (q.abs() @ k.abs().transpose(2, 3))
    bk = None
    if 'table' in t:
        bidirectional = (not causal) if bidirectional is None else bidirectional
        side = t['table'].shape[0] // 2 if bidirectional else t['table'].shape[0]
        pos = torch.arange(Lq)[None] + (q_pos.cpu()[:, None] if q_pos is not None else 0)
        rel = (torch.arange(Lk)[None, None] - pos[:, :, None]).expand(B, Lq, Lk)
        lo, hi = (int(rel.min()), int(rel.max())) if rel.numel() else (0, 0)
        lut = torch.tensor([bucket(r, side, md, bidirectional) for r in range(lo, hi + 1)])
        bk = lut[rel - lo]
        bias = t['table'].double()[bk].permute(0, 3, 1, 2)
        s = s + bias
        S = S + bias.abs()
        if causal:
            ok = ok & (rel <= 0)[:, None]
    elif causal:
        raise AssertionError
    s = s.masked_fill(~ok, -math.inf)
    m = s.max(3, keepdim=True).values if Lk else torch.zeros(B, H, Lq, 1).double()
    m = torch.where(m.isinf(), torch.zeros_like(m), m)
    p = torch.exp(s - m)
    tot = p.sum(3, keepdim=True)
    p = torch.where(tot > 0, p / tot.clamp_min(1e-300), torch.zeros_like(p))
    keep = torch.ones_like(p) if keep is None else keep.double().cpu().view(B, H, Lq, Lk)
    pd = p * keep
    # the largest magnitude of a score decides the rounding of the power of two's argument
    ep = 2 * (dh + 6) * u * (S.amax(3, keepdim=True) if Lk else m * 0) + (Lk + 8) * u
    o = pd @ v
    eo32 = (pd * (ep + hp) + tiny * keep) @ v.abs()               # before the result is rounded
    eo = eo32 + h * o.abs()
    dpr = do @ v.transpose(2, 3)
    delta = (do * o).sum(3, keepdim=True)
    edelta = (do.abs() * (eo32 + u * (dh + 1) * o.abs())).sum(3, keepdim=True)
    ds = p * (dpr * keep - delta)
    absd = p * ((do.abs() @ v.abs().transpose(2, 3)) * keep + (do.abs() * o.abs()).sum(3, keepdim=True))
    nrm = do.norm(dim=3, keepdim=True)
    under = tiny * nrm / 8
    eds = absd * (ep + 2 * dh * u) + p * edelta                   # of ds in f32
    edq = scale * ((eds + hp * ds.abs() + under) @ k.abs())
    if 'table' in t:
        eds = absd * (ep + 2 * dh * u) + p * (absd * (ep + 2 * dh * u + Lk * u)).sum(3, keepdim=True)
    dq = scale * (ds @ k)
    share = lambda x: x.view(B, KV, G, Lk, dh).sum(2)               # noqa: E731
    dk = share(scale * (ds.transpose(2, 3) @ q))
    under_k = tiny * nrm.amax((1, 2), keepdim=True) / 8 if Lq else under
    edk = share(scale * ((eds + hp * ds.abs() + under_k).transpose(2, 3) @ q.abs()))
    dv = share(pd.transpose(2, 3) @ do)
    edv = share((pd * (ep + hp) + tiny * keep).transpose(2, 3) @ do.abs())
    acc = (Lk + Lq * G + 8) * u                                      # order of the sums over keys / rows
    join = lambda x: x.permute(0, 2, 1, 3).reshape(B, x.shape[2], -1)              # noqa: E731
    vals = [join(o), join(dq), join(dk), join(dv)]
    sub = 2.0 ** -25 if dtype == F16 else 0.0
    bnds = [join(eo) + acc * join(pd @ v.abs()), join(edq) + h * join(dq).abs() + acc * join(abs(scale) * (ds.abs() @ k.abs())),
            join(edk) + h * join(dk).abs() + acc * join(share(abs(scale) * (ds.abs().transpose(2, 3) @ q.abs()))),
            join(edv) + h * join(dv).abs() + acc * join(share(pd.transpose(2, 3) @ do.abs()))]
    bnds = [b + sub for b in bnds]
    if 'table' in t:
        nb = t['table'].shape[0]
        dt, et = torch.zeros(nb, H).double(), torch.zeros(nb, H).double()
        for c in range(nb):
            sel = (bk == c)[:, None]
            dt[c] = (ds * sel).sum((0, 2, 3))
            et[c] = ((eds + (Lq + Lk + 64) * u * absd) * sel).sum((0, 2, 3))
        vals.append(dt)
        bnds.append(et + torch.finfo(t['table'].dtype).eps / 2 * dt.abs() + sub)
    return vals, bnds


def run(t, H, KV, backward=True, md=0, **kw):
    from ekaid_amd import ops
    d = {n: x.detach().to(DEV) for n, x in t.items()}
    names = ['q', 'k', 'v'] + (['table'] if 'table' in t else [])
    for n in names:
        d[n].requires_grad_(backward)
    if 'table' in t:
        out = ops.relative_attention(d['q'], d['k'], d['v'], d['table'], H, kv_heads=KV, max_distance=md, **kw)
    else:
        out = ops.cross_attention(d['q'], d['k'], d['v'], H, kv_heads=KV, **kw)
    if not backward:
        return [out.detach()]
    return [out.detach()] + list(torch.autograd.grad(out, [d[n] for n in names], d['dout']))


def compare(got, vals, bnds, what=''):
    for n, a, w, b in zip(('out', 'dq', 'dk', 'dv', 'dtable'), got, vals, bnds):
        a = a.double().cpu()
        assert a.shape == w.shape, (n, a.shape, w.shape)
        if a.numel() == 0:
            continue
        assert torch.isfinite(a).all(), '%s %s: non-finite' % (what, n)
        over = ((a - w).abs() / (b + 1e-30))
        assert float(over.max()) <= 1.0, '%s %s: %.3g times the bound (err %.3e, bound %.3e)' % (
            what, n, float(over.max()), float((a - w).abs().view(-1)[over.argmax()]), float(b.reshape(-1)[over.argmax()]))


def dev(x):
    return None if x is None else x.to(DEV)


# --------------------------------------------------------------------------- cross attention
CROSS = [
    # B, H, KV, dh, Lq, Lk
    (2, 3, 3, 8, 1, 1), (1, 2, 1, 40, 1, 7), (2, 4, 4, 256, 5, 104), (2, 4, 2, 64, 33, 65), (1, 2, 2, 128, 129, 67), (1, 4, 1, 96, 20, 300),
    (3, 2, 2, 64, 90, 52), (1, 2, 2, 256, 70, 129), (1, 1, 1, 64, 300, 20), (1, 8, 2, 128, 1, 777), (2, 1, 1, 32, 16, 16), (1, 2, 1, 128, 17, 33),
]


@gpu
@pytest.mark.parametrize('dtype', [F32, BF16, F16], ids=['f32', 'bf16', 'f16'])
@pytest.mark.parametrize('shape', CROSS, ids=lambda s: 'x'.join(map(str, s)))
def test_cross_attention(shape, dtype):
    B, H, KV, dh, Lq, Lk = shape
    t = make(dtype, B, H, KV, dh, Lq, Lk)
    vals, bnds = reference(t, H, KV, dh)
    compare(run(t, H, KV), vals, bnds)
    compare(run(t, H, KV, backward=False), vals, bnds, 'no grad')


@gpu
@pytest.mark.parametrize('dtype', [F32, BF16, F16], ids=['f32', 'bf16', 'f16'])
@pytest.mark.parametrize('index', [torch.int32, torch.int64], ids=['i32', 'i64'])
def test_ragged_lengths_and_masks(dtype, index):
    """Lengths 0, 1, full and beyond, a key mask with an empty sample; masked states hold NaN and infinities."""
    B, H, KV, dh, Lq, Lk = 6, 4, 2, 64, 37, 150
    t = make(dtype, B, H, KV, dh, Lq, Lk)
    k_len = torch.tensor([0, 1, 150, 97, 64, 500], dtype=index)
    mask = torch.rand(B, Lk, generator=torch.Generator().manual_seed(3)) > 0.3
    mask[4] = False
    mask[2, :64] = False                                   # a whole tile
    dead = (torch.arange(Lk)[None] >= k_len[:, None]) | ~mask
    t['k'][dead] = float('nan')
    t['v'][dead] = float('inf')
    vals, bnds = reference(t, H, KV, dh, k_len=k_len, key_mask=mask)
    got = run(t, H, KV, k_len=dev(k_len), key_mask=dev(mask))
    compare(got, vals, bnds)
    for b in (0, 4):
        for x in got:
            assert (x[b] == 0).all()
    t2 = {n: x[:, :1] if n in ('q', 'dout') else x for n, x in t.items()}
    vals, bnds = reference(t2, H, KV, dh, k_len=k_len, key_mask=mask)
    compare(run(t2, H, KV, k_len=dev(k_len), key_mask=dev(mask)), vals, bnds, 'one token')


@gpu
@pytest.mark.parametrize('dtype', [F32, BF16], ids=['f32', 'bf16'])
@pytest.mark.parametrize('B,Lq,Lk', [(0, 3, 4), (2, 0, 5), (2, 3, 0), (2, 1, 0)])
def test_empty_axes(dtype, B, Lq, Lk):
    for nb in (0, 8):
        t = make(dtype, B, 2, 1, 16, Lq, Lk, nb=nb)
        got = run(t, 2, 1, md=20 if nb else 0)
        for n, x in zip(('q', 'q', 'k', 'v', 'table'), got):
            assert x.shape == t[n].shape and (x == 0).all()


@gpu
@pytest.mark.parametrize('dtype', [F32, BF16, F16], ids=['f32', 'bf16', 'f16'])
def test_strided_and_unaligned_operands(dtype):
    """Slices of one packed projection, a transposed batch, an odd storage offset: the same results as contiguous tensors."""
    from ekaid_amd import ops
    B, H, dh, Lq, Lk = 3, 2, 32, 9, 70
    D = H * dh
    g = torch.Generator().manual_seed(1)
    packed = torch.randn(Lk, B, 2 * D, generator=g).to(dtype).to(DEV)
    k, v = packed[..., :D].transpose(0, 1), packed[..., D:].transpose(0, 1)
    flat = torch.randn(B * Lq * D + 3, generator=g).to(dtype).to(DEV)
    q = flat[3:].view(B, Lq, D)
    wide = torch.randn(B, Lq, D + 5, generator=g).to(dtype).to(DEV)[..., 1:D + 1]
    shared = torch.randn(1, Lk, D, generator=g).to(dtype).to(DEV).expand(B, Lk, D)
    for a, b, c in ((q, k, v), (wide, k, v), (q, shared, v), (q, k[:, ::2], v[:, ::2])):
        want = ops.cross_attention(a.clone(memory_format=torch.contiguous_format), b.clone(memory_format=torch.contiguous_format), c.clone(memory_format=torch.contiguous_format), H)
        assert torch.equal(ops.cross_attention(a, b, c, H), want)
    base = torch.randn(1, Lk, D, generator=g).to(dtype).to(DEV).requires_grad_(True)       # a broadcast input: its gradient is the sum
    dout = torch.randn(B, Lq, D, generator=g).to(dtype).to(DEV)
    (gb,) = torch.autograd.grad(ops.cross_attention(q, base.expand(B, Lk, D), v, H), [base], dout)
    full = base.detach().expand(B, Lk, D).contiguous().requires_grad_(True)
    (gf,) = torch.autograd.grad(ops.cross_attention(q, full, v, H), [full], dout)
    assert torch.equal(gb, gf.sum(0, keepdim=True).to(dtype))


@gpu
def test_offsets_beyond_32_bits():
    """Rows so far apart that a 32-bit offset would wrap: one new token over a cache kept inside a 9 GB buffer."""
    from ekaid_amd import ops
    H, dh, Lk, row = 2, 64, 70000, 1 << 16
    big = torch.empty(Lk * row, device=DEV, dtype=BF16)
    view = big.view(1, Lk, row)[..., :2 * H * dh]
    g = torch.Generator(device=DEV).manual_seed(5)
    view.copy_(torch.randn(1, Lk, 2 * H * dh, generator=g, device=DEV))
    k, v = view[..., :H * dh], view[..., H * dh:]
    q = torch.randn(1, 1, H * dh, generator=g, device=DEV).to(BF16)
    assert (Lk - 1) * row > 1 << 32
    assert torch.equal(ops.cross_attention(q, k, v, H), ops.cross_attention(q, k.contiguous(), v.contiguous(), H))


@gpu
@pytest.mark.parametrize('dtype', [F32, F16], ids=['f32', 'f16'])
def test_small_and_large_incoming_gradients(dtype):
    """A gradient of 1e-4 of the usual size (a loss divided by thousands of tokens) and one of 300 times: relative accuracy as usual."""
    for scale_out in (1e-4, 300.0):
        t = make(dtype, 1, 2, 2, 64, 70, 260, scale_out=scale_out)
        t['dout'][:, :20] *= 2.0 ** -3
        vals, bnds = reference(t, 2, 2, 64)
        compare(run(t, 2, 2), vals, bnds, str(scale_out))


@gpu
def test_scores_out_of_the_usual_range():
    """Scores of several hundred (one key takes everything) and a table of the type's lowest value: no overflow, no NaN."""
    t = make(F32, 1, 2, 2, 64, 40, 80)
    t['q'] *= 30
    vals, bnds = reference(t, 2, 2, 64)
    compare(run(t, 2, 2), vals, bnds)
    t = make(F32, 1, 2, 2, 64, 40, 80, nb=8)
    t['table'][3] = torch.finfo(F32).min
    t['table'][5] = -math.inf
    vals, _ = reference(t, 2, 2, 64, md=16)
    t2 = dict(t, table=t['table'].clamp_min(-1e4))
    vals, bnds = reference(t2, 2, 2, 64, md=16)
    got = run(t, 2, 2, md=16)
    S = 64 * 2.0 ** -24 * 40 + 200 * 2.0 ** -24                   # the bound of the unmasked places (|scores| < 40)
    for a, w in zip(got, vals):
        assert torch.isfinite(a).all()
        assert float((a.double().cpu() - w).abs().max()) <= 8 * S * float(w.abs().max())
    t['table'][:] = -math.inf                                      # every score of every row: empty rows
    for x in run(t, 2, 2, md=16):
        assert (x == 0).all()


@gpu
@pytest.mark.parametrize('dtype', [F32, BF16], ids=['f32', 'bf16'])
@pytest.mark.parametrize('shape', [(2, 4, 2, 32, 40, 70), (1, 2, 1, 64, 1, 200)], ids=str)
def test_dropout_of_the_probabilities(dtype, shape):
    from ekaid_amd import ops
    B, H, KV, dh, Lq, Lk = shape
    p = 0.3
    t = make(dtype, B, H, KV, dh, Lq, Lk, nb=8)
    ops.manual_seed(11)
    keep = ops.dropout(torch.ones(B * H * Lq * Lk, device=DEV), p, True)           # the mask of the seed the call will draw
    assert 0.2 < float((keep == 0).float().mean()) < 0.4
    vals, bnds = reference(t, H, KV, dh, md=20, keep=keep)
    ops.manual_seed(11)
    compare(run(t, H, KV, md=20, p=p, training=True), vals, bnds)
    vals, bnds = reference(t, H, KV, dh, md=20)
    compare(run(t, H, KV, md=20, p=p, training=False), vals, bnds, 'eval')


@gpu
def test_equals_the_frameworks_equal_length_attention():
    from ekaid_amd import ops
    g = torch.Generator().manual_seed(2)
    q, k, v = (torch.randn(4, 52, 256, generator=g).to(DEV) for _ in range(3))
    a, b = ops.cross_attention(q, k, v, 4), ops.head_attention(q, k, v, 4)
    assert float((a - b).abs().max()) <= 2 * (64 + 52 + 20) * 2.0 ** -24 * 40 * float(v.abs().max())


# --------------------------------------------------------------------------- relative bias
def test_borders_are_exact():
    from ekaid_amd.ops import relative_borders
    for side, md in ((16, 128), (32, 128), (8, 64), (5, 20), (2, 2), (32, 1000), (16, 9)):
        b = relative_borders(side, md)
        assert len(b) == side - 1
        for d in range(0, md + 50):
            assert sum(x <= d for x in b) == bucket(-d, side, md, False), (side, md, d)
    assert relative_borders(16, 128) == (1, 2, 3, 4, 5, 6, 7, 8, 12, 16, 23, 32, 46, 64, 91)


REL = [
    # B, H, KV, dh, Lq, Lk, nb, md, causal
    (2, 3, 3, 64, 20, 20, 32, 128, False), (1, 2, 2, 64, 150, 150, 32, 128, True), (2, 2, 1, 32, 70, 130, 16, 40, False),
    (1, 2, 2, 128, 300, 300, 32, 50, True), (1, 4, 4, 256, 33, 90, 8, 20, False), (1, 2, 2, 16, 1, 1, 4, 9, True), (1, 1, 1, 64, 520, 260, 16, 64, False),
    (1, 2, 2, 64, 40, 700, 16, 64, True),
]


@gpu
@pytest.mark.parametrize('dtype', [F32, BF16, F16], ids=['f32', 'bf16', 'f16'])
@pytest.mark.parametrize('shape', REL, ids=lambda s: 'x'.join(map(str, s)))
def test_relative_attention(shape, dtype):
    B, H, KV, dh, Lq, Lk, nb, md, causal = shape
    t = make(dtype, B, H, KV, dh, Lq, Lk, nb=nb)
    vals, bnds = reference(t, H, KV, dh, causal=causal, md=md)
    got = run(t, H, KV, md=md, causal=causal)
    compare(got, vals, bnds)
    again = run(t, H, KV, md=md, causal=causal)
    assert all(torch.equal(a, b) for a, b in zip(got, again))


@gpu
@pytest.mark.parametrize('dtype', [F32, BF16, F16], ids=['f32', 'bf16', 'f16'])
@pytest.mark.parametrize('shape', [(1, 3, 64, 2, 1300), (2, 2, 128, 70, 1200), (1, 2, 256, 80, 1090), (2, 6, 64, 1150, 70)], ids=lambda s: 'x'.join(map(str, s)))
def test_largest_reach(shape, dtype):
    """The last bucket begins at the largest distance that is taken: the tables and sums in LDS at their full size."""
    from ekaid_amd import ops
    KV, H, dh, Lq, Lk = shape
    md = max(m for m in range(900, 2000) if ops.relative_borders(64, m)[-1] <= 1024)
    assert ops.relative_borders(64, md)[-1] == 1024
    for two in (False, True):
        t = make(dtype, 1, H, KV, dh, Lq, Lk, seed=3, nb=128 if two else 64, md=md)
        kw = dict(bidirectional=two, causal=not two)
        if Lq < Lk:
            kw['q_pos'] = torch.tensor([Lk - Lq])
        vals, bnds = reference(t, H, KV, dh, md=md, **kw)
        compare(run(t, H, KV, md=md, **{n: dev(x) if torch.is_tensor(x) else x for n, x in kw.items()}), vals, bnds, str(two))


@gpu
@pytest.mark.parametrize('bidirectional', [True, False])
@pytest.mark.parametrize('causal', [True, False])
def test_positions_masks_and_directions(bidirectional, causal):
    """Query positions ahead of, behind and before the keys, ragged lengths, masked first keys (empty causal rows), a 16-bit table."""
    B, H, KV, dh, Lq, Lk = 4, 4, 2, 64, 45, 200
    t = make(BF16, B, H, KV, dh, Lq, Lk, nb=16, table_dtype=BF16)
    q_pos = torch.tensor([0, 155, -30, 400])
    k_len = torch.tensor([200, 200, 180, 33], dtype=torch.int32)
    mask = torch.ones(B, Lk, dtype=torch.bool)
    mask[0, :10] = False
    kw = dict(q_pos=q_pos, k_len=k_len, key_mask=mask, causal=causal, bidirectional=bidirectional)
    vals, bnds = reference(t, H, KV, dh, md=30, **kw)
    got = run(t, H, KV, md=30, **{n: dev(x) if torch.is_tensor(x) else x for n, x in kw.items()})
    compare(got, vals, bnds)
    if causal:
        assert (got[0][0, :10] == 0).all() and (got[1][0, :10] == 0).all() and (got[0][2, :30] == 0).all()


@gpu
@pytest.mark.parametrize('dtype', [F32, BF16, F16], ids=['f32', 'bf16', 'f16'])
def test_new_token_equals_the_row_of_the_whole_sequence(dtype):
    """A decoder's step over its cache is the last row of the same call over the whole sequence, sample by sample (bounds of both)."""
    from ekaid_amd import ops
    B, H, KV, dh, L = 3, 4, 2, 64, 333
    t = make(dtype, B, H, KV, dh, L, L, nb=16)
    vals, bnds = reference(t, H, KV, dh, causal=True, md=100)
    lens = torch.tensor([333, 17, 128])
    last = torch.stack([t['q'][b, n - 1:n] for b, n in enumerate(lens.tolist())])
    got = ops.relative_attention(dev(last), dev(t['k']), dev(t['v']), dev(t['table']), H, kv_heads=KV, k_len=dev(lens), q_pos=dev(lens - 1), causal=True, max_distance=100)
    for b, n in enumerate(lens.tolist()):
        assert ((got[b, 0].double().cpu() - vals[0][b, n - 1]).abs() <= bnds[0][b, n - 1]).all()


@gpu
def test_gradients_against_differences():
    """d(loss)/d(direction) of the f32 operator against central differences of the float64 formula along the same direction."""
    t = make(F32, 2, 2, 1, 16, 21, 34, nb=8)
    kw = dict(md=20, causal=False)
    got = run(t, 2, 1, **kw)
    w = t['dout'].double()
    for n, gr in zip(('q', 'k', 'v', 'table'), got[1:]):
        e = torch.randn(t[n].shape, generator=torch.Generator().manual_seed(9))
        step = 2.0 ** -9
        f = [float((reference({**{a: b.double() for a, b in t.items()}, n: t[n].double() + s * step * e.double()}, 2, 1, 16, **kw)[0][0] * w).sum()) for s in (1, -1)]
        # central difference: third derivatives ~ step^2; the operator: relative 1e-6 of sums of 1e3 terms
        assert abs(float((gr.double().cpu() * e).sum()) - (f[0] - f[1]) / (2 * step)) <= 1e-3 * max(1.0, abs(f[0] - f[1]) / (2 * step))


# --------------------------------------------------------------------------- streams, graphs, refusals
@gpu
def test_two_streams_at_once_and_captured_replays():
    """Two different calls on two streams at once; the same passes captured, replayed with eager work between, other inputs in place."""
    from ekaid_amd import ops
    cases = [make(BF16, 1, 4, 2, 64, 1, 900, nb=16), make(BF16, 2, 4, 4, 64, 130, 190, nb=16, seed=4)]
    eager = [run(t, 4, KV, md=64) for t, KV in zip(cases, (2, 4))]
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    torch.cuda.synchronize()
    got = []
    for _ in range(5):
        for st, t, KV in zip(streams, cases, (2, 4)):
            with torch.cuda.stream(st):
                got.append(run(t, 4, KV, md=64))
    torch.cuda.synchronize()
    for i, g in enumerate(got):
        assert all(torch.equal(a, b) for a, b in zip(g, eager[i % 2]))
    graphs = []
    for t, KV in zip(cases, (2, 4)):
        d = {n: x.to(DEV) for n, x in t.items()}
        leaves = [d[n].requires_grad_(True) for n in ('q', 'k', 'v', 'table')]
        gr = torch.cuda.CUDAGraph()
        torch.cuda.synchronize()
        with torch.cuda.graph(gr):
            out = ops.relative_attention(d['q'], d['k'], d['v'], d['table'], 4, kv_heads=KV, max_distance=64)
            res = [out] + list(torch.autograd.grad(out, leaves, d['dout']))
        graphs.append((gr, [x.detach() for x in res], d))
    for rep in range(3):
        for (gr, res, d), t, KV in zip(graphs, cases, (2, 4)):
            with torch.no_grad():
                d['q'].mul_(1.0 if rep == 0 else -0.5)
            gr.replay()
            torch.cuda.synchronize()
            want = run({n: x.detach() for n, x in d.items()}, 4, KV, md=64)
            assert all(torch.equal(a, b) for a, b in zip(res, want))


@gpu
def test_second_derivatives_and_changed_inputs_are_errors():
    from ekaid_amd import ops
    q, k, v = (torch.randn(1, 4, 16, device=DEV, requires_grad=True) for _ in range(3))
    (gq,) = torch.autograd.grad(ops.cross_attention(q, k, v, 1).sum(), [q], create_graph=True)
    with pytest.raises(RuntimeError):
        gq.sum().backward()
    out = ops.cross_attention(q, k, v, 1).sum()
    with torch.no_grad():
        k.add_(1.0)
    with pytest.raises(RuntimeError):
        out.backward()


@gpu
def test_refusals():
    from ekaid_amd import ops
    from ekaid_amd.hip import EkaidError
    z = lambda *s, dt=F32: torch.zeros(*s, device=DEV, dtype=dt)            # noqa: E731
    q, k, tab = z(2, 3, 64), z(2, 5, 64), z(8, 2)
    bad = [
        lambda: ops.cross_attention(q.cpu(), k.cpu(), k.cpu(), 2), lambda: ops.cross_attention(q[0], k, k, 2), lambda: ops.cross_attention(q.double(), k.double(), k.double(), 2),
        lambda: ops.cross_attention(q, k.half(), k, 2), lambda: ops.cross_attention(q, k, k, 3), lambda: ops.cross_attention(q, k, k, 2, kv_heads=3),
        lambda: ops.cross_attention(q, k, k, 16), lambda: ops.cross_attention(z(2, 3, 512), z(2, 5, 512), z(2, 5, 512), 1), lambda: ops.cross_attention(q, k, k[:, :4], 2),
        lambda: ops.cross_attention(q, z(3, 5, 64), z(3, 5, 64), 2), lambda: ops.cross_attention(q, k, k, 2, kv_heads=1), lambda: ops.cross_attention(q, k, k, 0),
        lambda: ops.cross_attention(q, k, k, 2, k_len=z(2)), lambda: ops.cross_attention(q, k, k, 2, k_len=z(3, dt=torch.int32)),
        lambda: ops.cross_attention(q, k, k, 2, k_len=torch.zeros(2, dtype=torch.int32)), lambda: ops.cross_attention(q, k, k, 2, key_mask=z(2, 5)),
        lambda: ops.cross_attention(q, k, k, 2, key_mask=z(2, 4, dt=torch.bool)), lambda: ops.cross_attention(q, k, k, 2, scale=float('nan')),
        lambda: ops.cross_attention(q, k, k, 2, p=1.0, training=True), lambda: ops.relative_attention(q, k, k, None, 2), lambda: ops.relative_attention(q, k, k, z(8, 3), 2),
        lambda: ops.relative_attention(q, k, k, z(8, 2, dt=BF16), 2), lambda: ops.relative_attention(q, k, k, z(7, 2), 2), lambda: ops.relative_attention(q, k, k, z(2, 2), 2),
        lambda: ops.relative_attention(q, k, k, tab, 2, max_distance=2), lambda: ops.relative_attention(q, k, k, tab, 2, max_distance=10 ** 7),
        lambda: ops.relative_attention(q, k, k, z(300, 2), 2, max_distance=1000), lambda: ops.relative_attention(q, k, k, tab, 2, q_pos=z(2)),
    ]
    for i, f in enumerate(bad):
        with pytest.raises(EkaidError):
            f()
            raise AssertionError('call %d was taken' % i)


def test_c_entry_refuses_bad_descriptors():
    """The C entries check before they touch the device: bad sizes, strides, alignment, borders and workspaces are error codes."""
    from ekaid_amd import hip
    L = hip.load()

    def desc(**kw):
        d = hip.Attn()
        d.q = d.k = d.v = d.out = d.dout = d.lse = d.dq = d.dk = d.dv = 1 << 20
        d.B, d.H, d.KV, d.dh, d.Lq, d.Lk = 2, 4, 2, 64, 8, 16
        d.q_batch, d.q_row, d.k_batch, d.k_row, d.v_batch, d.v_row = 2048, 256, 2048, 128, 2048, 128
        d.scale = 1.0
        for n, x in kw.items():
            setattr(d, n, x)
        return d
    bad = [dict(dtype=3), dict(B=-1), dict(H=5), dict(KV=0), dict(dh=60), dict(dh=264), dict(dh=0), dict(Lq=-1), dict(Lk=-2), dict(q=(1 << 20) + 4), dict(q_row=258),
           dict(k_batch=-4), dict(drop_p=1.0), dict(drop_p=float('nan')), dict(table=1 << 20, reach=0), dict(table=1 << 20, reach=5000), dict(table=1 << 20, reach=4, n_border=128),
           dict(table=1 << 20, reach=1, n_border=1), dict(B=1 << 14, H=1 << 14, KV=1 << 14)]
    for kw in bad:
        d = desc(**kw)
        for entry in (L.ekaid_attn_fwd, L.ekaid_attn_bwd):
            rc = entry(ctypes.byref(d), 1 << 20, 1 << 40, None)
            assert rc < 0 and hip.last_error(), kw
        assert L.ekaid_attn_workspace_bytes(ctypes.byref(d), 1) == 0
    d = desc(table=1 << 20, dtable=1 << 20, reach=9, n_border=2)
    d.border[0], d.border[1] = 5, 3
    assert L.ekaid_attn_fwd(ctypes.byref(d), None, 0, None) < 0
    d = desc()
    assert L.ekaid_attn_bwd(ctypes.byref(d), None, 0, None) < 0 and 'workspace' in hip.last_error()
    for name in ('q', 'k', 'v', 'out', 'lse', 'dout', 'dq', 'dk', 'dv'):
        d = desc(**{name: None})
        assert L.ekaid_attn_bwd(ctypes.byref(d), 1 << 20, 1 << 40, None) < 0
    assert L.ekaid_attn_fwd(None, None, 0, None) < 0
    assert ctypes.sizeof(hip.Attn) > 0


@gpu
def test_forward_mode_derivatives_are_errors():
    """An operand that carries a tangent: refused, as every operator without a forward derivative does, not a result that has lost it."""
    import torch.autograd.forward_ad as fw
    from ekaid_amd import ops
    q, k, v, tab = (torch.randn(*s, device=DEV) for s in ((1, 4, 16), (1, 6, 16), (1, 6, 16), (4, 1)))
    want = ops.relative_attention(q, k, v, tab, 1, max_distance=9)
    with fw.dual_level():
        for i in range(4):
            a = [fw.make_dual(x, torch.ones_like(x)) if i == n else x for n, x in enumerate((q, k, v, tab))]
            with pytest.raises(NotImplementedError):
                ops.relative_attention(*a, 1, max_distance=9)
            if i < 3:
                with pytest.raises(NotImplementedError):
                    ops.cross_attention(*a[:3], 1)
        assert torch.equal(ops.relative_attention(q, k, v, tab, 1, max_distance=9), want)


@gpu
def test_max_distance_that_is_no_whole_number_is_refused():
    from ekaid_amd import ops
    from ekaid_amd.hip import EkaidError
    q, k, tab = torch.zeros(2, 3, 64, device=DEV), torch.zeros(2, 5, 64, device=DEV), torch.zeros(8, 2, device=DEV)
    for md in (math.inf, -math.inf, math.nan, 9.5, None, '9'):
        with pytest.raises(EkaidError):
            ops.relative_attention(q, k, k, tab, 2, max_distance=md)
    import numpy as np
    assert torch.equal(ops.relative_attention(q, k, k, tab, 2, max_distance=np.int64(9)), ops.relative_attention(q, k, k, tab, 2, max_distance=9))
    assert torch.equal(ops.relative_attention(q, k, k, tab, 2, max_distance=9.0), ops.relative_attention(q, k, k, tab, 2, max_distance=9))


@gpu
@pytest.mark.parametrize('dtype', [F32, BF16, F16], ids=['f32', 'bf16', 'f16'])
@pytest.mark.parametrize('Lq', [1, 16, 17, 70, 130])
def test_causal_rows_read_nothing_behind_the_last_position(Lq, dtype):
    """A chunk of rows over a cache without lengths: what stands behind the last row's position (NaN, Inf) reaches no result."""
    B, H, KV, dh, Lk = 2, 4, 2, 64, 300
    t = make(dtype, B, H, KV, dh, Lq, Lk, nb=16)
    q_pos = torch.tensor([3, 141])
    behind = torch.arange(Lk)[None] >= (q_pos + Lq)[:, None]
    res = []
    for kx, vx in ((0.0, 0.0), (float('nan'), float('nan')), (1.0, float('inf'))):
        t['k'][behind], t['v'][behind] = kx, vx
        res.append(run(t, H, KV, md=30, causal=True, q_pos=dev(q_pos)))
    for other in res[1:]:
        for n, a, b in zip(('out', 'dq', 'dk', 'dv', 'dtable'), res[0], other):
            assert torch.equal(a, b), n
    assert (res[0][2][behind] == 0).all() and (res[0][3][behind] == 0).all()


@gpu
@pytest.mark.parametrize('Lq', [1, 40, 90])
@pytest.mark.parametrize('dtype,table_dtype,low', [(F32, F32, -1e9), (F32, F32, -6e4), (F32, F32, torch.finfo(F32).min), (BF16, BF16, -1e9), (BF16, BF16, torch.finfo(BF16).min),
                                                   (F16, F16, torch.finfo(F16).min), (F16, F32, -1e5)], ids=str)
def test_lowest_entries_of_the_table_close_their_distances(dtype, table_dtype, low, Lq):
    """A table with a large negative entry in place of -inf: the same results, rows that see nothing but such distances among them."""
    B, H, KV, dh, Lk = 3, 2, 1, 64, 80
    t = make(dtype, B, H, KV, dh, Lq, Lk, nb=8, table_dtype=table_dtype)
    q_pos = torch.tensor([0, 400, 30])                            # the second sample's keys all lie in the farthest bucket behind
    res = []
    for x in (-math.inf, low):
        t['table'][3] = x
        res.append(run(t, H, KV, md=16, q_pos=dev(q_pos)))
    for n, a, b in zip(('out', 'dq', 'dk', 'dv', 'dtable'), *res):
        assert torch.isfinite(a).all() and torch.equal(a, b), n
    for x in res[1][:4]:
        assert (x[1] == 0).all() and not (x[2] == 0).all()


def f16_score_gradient_floor(t, H, KV, dh, inv_keep=1.0):
    """What f16 score gradients lose below the normal range, in dq and dk: they are stored with 2 |dout| max |v| inv_keep brought to at least
    2^13, so half a step is 2^-25 of a 2^13th of that."""
    split = lambda x, n: x.double().view(x.shape[0], x.shape[1], n, dh)                 # noqa: E731
    do, v = split(t['dout'], H).norm(dim=3).amax((1, 2)), split(t['v'], KV).norm(dim=3).amax((1, 2))
    lost = (2.0 ** -25 * 2 * inv_keep / 2 ** 13 * do * v * dh ** -0.5)[:, None, None]
    kq = split(t['k'], KV).abs().sum(1).repeat_interleave(H // KV, 1).flatten(1)[:, None]
    qk = split(t['q'], H).abs().sum(1).view(-1, KV, H // KV, dh).sum(2).flatten(1)[:, None]
    return lost * kq, lost * qk


@gpu
@pytest.mark.parametrize('shape', [(1, 2, 1, 256, 40, 150), (2, 2, 2, 128, 70, 90), (1, 4, 2, 64, 200, 200), (2, 2, 2, 64, 5, 33)], ids=str)
def test_f16_values_of_thousands(shape):
    """Values up to half of f16's range, sharp rows: the score gradients of such rows pass f16's range many times over, no gradient does."""
    B, H, KV, dh, Lq, Lk = shape
    t = make(F16, B, H, KV, dh, Lq, Lk, scale_out=2e-3)
    t['q'], t['v'] = t['q'] * 4, (t['v'].float() * 7000).half()
    vals, bnds = reference(t, H, KV, dh)
    eq, ek = f16_score_gradient_floor(t, H, KV, dh)
    compare(run(t, H, KV), vals, [bnds[0], bnds[1] + eq, bnds[2] + ek, bnds[3]])


@gpu
@pytest.mark.parametrize('p', [0.5, 0.98])
def test_f16_dropout(p):
    """Kept probabilities of up to fifty times their size beside values of some thirty: score gradients stay in range."""
    from ekaid_amd import ops
    B, H, KV, dh, Lq, Lk = 2, 4, 2, 64, 40, 90
    t = make(F16, B, H, KV, dh, Lq, Lk, scale_out=0.05)
    t['q'], t['v'] = t['q'] * 3, (t['v'].float() * 30).half()
    ops.manual_seed(5)
    keep = ops.dropout(torch.ones(B * H * Lq * Lk, device=DEV), p, True)
    vals, bnds = reference(t, H, KV, dh, keep=keep)
    eq, ek = f16_score_gradient_floor(t, H, KV, dh, 1 / (1 - p))
    ops.manual_seed(5)
    compare(run(t, H, KV, p=p, training=True), vals, [bnds[0], bnds[1] + eq, bnds[2] + ek, bnds[3]])


@gpu
def test_f16_value_gradients_of_many_keys():
    """818400 equal keys: a probability of 1.2e-6 lies between two of f16's smallest numbers.  Every score is exactly 0, every power 1 and
    the sum exact, so a value's gradient is sum_i dout_i / 818400: rounding of the probability (h), of the result (h), 24 f32 additions and a
    logarithm of 20 in f32 (2^-24 * 20, twice)."""
    from ekaid_amd import ops
    Lk, Lq, dh = 818400, 24, 8
    g = torch.Generator(device=DEV).manual_seed(1)
    q = torch.zeros(1, Lq, dh, device=DEV, dtype=F16, requires_grad=True)
    k, v = (torch.rand(1, Lk, dh, generator=g, device=DEV).half().requires_grad_(True) for _ in range(2))
    dout = (torch.rand(1, Lq, dh, generator=g, device=DEV) * 200 + 100).half()
    (dv,) = torch.autograd.grad(ops.cross_attention(q, k, v, 1), [v], dout)
    want = dout.double().sum(1, keepdim=True) / Lk
    assert float(((dv.double() - want).abs() / want).max()) <= 2 * 2.0 ** -11 + (24 + 2 * 20 + 10) * 2.0 ** -24


@gpu
@pytest.mark.parametrize('shape', [(1, 16, 16, 32, 64, 1024), (8, 16, 16, 32, 1, 8192)], ids=str)
def test_f16_dropout_that_keeps_almost_nothing(shape):
    """One probability in 2^17 is kept, 2^17 times its size, which f16 does not hold; output and gradients it holds."""
    from ekaid_amd import ops
    B, H, KV, dh, Lq, Lk = shape
    p = 1 - 2.0 ** -17
    t = make(F16, B, H, KV, dh, Lq, Lk, scale_out=0.05)
    t['q'], t['v'] = t['q'] * 0.25, (t['v'].float() * 0.1).half()
    seed = 0
    while True:
        ops.manual_seed(seed)
        keep = ops.dropout(torch.ones(B * H * Lq * Lk, device=DEV), p, True)
        if int((keep != 0).sum()) >= 4:
            break
        seed += 1
    vals, bnds = reference(t, H, KV, dh, keep=keep)
    eq, ek = f16_score_gradient_floor(t, H, KV, dh, 2.0 ** 17)
    ops.manual_seed(seed)
    compare(run(t, H, KV, p=p, training=True), vals, [bnds[0], bnds[1] + eq, bnds[2] + ek, bnds[3]])


def test_c_entry_refuses_more_threads_than_a_launch_counts():
    from ekaid_amd import hip
    L = hip.load()
    for kw in (dict(B=1 << 12, H=1 << 12), dict(B=1 << 10, H=64, Lq=1 << 14), dict(B=1 << 10, H=64, Lk=1 << 14), dict(B=1, H=1 << 18, table=1 << 20, reach=9)):
        d = hip.Attn()
        d.q = d.k = d.v = d.out = d.dout = d.lse = d.dq = d.dk = d.dv = d.dtable = 1 << 20
        d.B, d.H, d.KV, d.dh, d.Lq, d.Lk, d.scale = 2, 1, 1, 8, 1, 1, 1.0
        for n, x in kw.items():
            setattr(d, n, x)
        d.KV = d.H
        for entry in (L.ekaid_attn_fwd, L.ekaid_attn_bwd):
            assert entry(ctypes.byref(d), 1 << 20, 1 << 50, None) < 0 and 'too many' in hip.last_error(), kw
        assert L.ekaid_attn_workspace_bytes(ctypes.byref(d), 0) == 0
        d.B, d.H, d.KV, d.Lq, d.Lk = 1, max(1, d.H >> 2), max(1, d.H >> 2), max(1, d.Lq >> 2), max(1, d.Lk >> 2)
        assert L.ekaid_attn_workspace_bytes(ctypes.byref(d), 1) > 0, kw


@gpu
@pytest.mark.parametrize('dtype', [F32, BF16, F16], ids=['f32', 'bf16', 'f16'])
@pytest.mark.parametrize('Lq', [1, 20, 70, 130])
def test_gradients_of_samples_without_states_are_zero_whatever_comes_in(Lq, dtype):
    """Two samples attend nothing, by their length and by their mask, and NaN and Inf come in for them: zeros there, nothing changes elsewhere."""
    B, H, KV, dh, Lk = 4, 4, 2, 64, 150
    t = make(dtype, B, H, KV, dh, Lq, Lk, nb=16)
    k_len, mask = torch.tensor([150, 0, 100, 150]), torch.ones(B, Lk, dtype=torch.bool)
    mask[2] = False
    res = []
    for bad in (0.0, float('nan'), float('inf')):
        t['dout'][1:3] = bad
        res.append([run(t, H, KV, md=30, k_len=dev(k_len), key_mask=dev(mask)), run({n: x for n, x in t.items() if n != 'table'}, H, KV, k_len=dev(k_len), key_mask=dev(mask))])
    for other in res[1:]:
        for a, b in zip(res[0], other):
            for n, x, y in zip(('out', 'dq', 'dk', 'dv', 'dtable'), a, b):
                assert torch.equal(x, y), n
            for x in b[:4]:
                assert (x[1:3] == 0).all()
