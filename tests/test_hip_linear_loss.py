"""Vocabulary loss of a linear layer without its logits, against the definition in float64, element by element.

Bounds: u = 2^-24; a logit carries (D + 8) u sum |x||w| (f32 products of the split arithmetics: another 2^-21 of it, and 2^-39 of the
largest magnitudes for values far below them); a probability twice the largest logit error of its row plus the sum over words
((300 + V / 64) u); 16-bit types round each logit gradient once (h = half a step; f16 also 2^-39 absolute, its scale being 2^14) where it
enters a product, and each result once (h)."""
import ctypes
import math

import pytest
import torch

F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16
DEV = 'cuda'
gpu = pytest.mark.gpu
IDS = ['f32', 'bf16', 'f16']


def make(dtype, B, T, D, V, seed=0, bias=True, xs=1.0):
    g = torch.Generator().manual_seed(seed + D + V + T)
    r = lambda *s: torch.randn(*s, generator=g)                                   # noqa: E731
    t = dict(x=(r(B, T, D) * xs).to(dtype).to(DEV), weight=(r(V, D) * 1.5 / math.sqrt(D)).to(dtype).to(DEV), bias=r(V).mul(0.5).to(dtype).to(DEV) if bias else None,
             target=torch.randint(0, V, (B, T), generator=g).to(DEV))
    lens = torch.randint(1, T + 1, (B,), generator=g)
    t['mask'] = (torch.arange(T)[None] < lens[:, None]).float().to(DEV)
    return t


def reference(t, denom=None, dloss=1.0):
    """(values, bounds) in float64 on the device (2-D products only): loss, dx, dweight, dbias."""
    dtype = t['x'].dtype
    B, T, D = t['x'].shape
    V = t['weight'].shape[0]
    u, h = 2.0 ** -24, torch.finfo(dtype).eps / 2
    hp, tiny = (0.0 if dtype == F32 else h), (2.0 ** -39 if dtype == F16 else 0.0)
    k3 = 2.0 ** -21 if dtype == F32 else 0.0
    far = 2.0 ** -39 if dtype == F32 else 0.0
    m = t['mask'][:, :T].double().reshape(-1)
    on = (m != 0).nonzero().view(-1)
    x, w = t['x'].double().reshape(-1, D)[on], t['weight'].double()
    b = t['bias'].double() if t['bias'] is not None else torch.zeros(V, device=DEV).double()
    tg, mo = t['target'][:, :T].reshape(-1)[on], m[on]
    den = m.sum() if denom is None else denom.double()
    z = x @ w.t() + b
    S = x.abs() @ w.abs().t()
    top = far * D * x.abs().amax(1, keepdim=True) * w.abs().max()
    ez = ((D + 8) * u + k3) * S.amax(1, keepdim=True) + top + 4 * u * z.abs().amax(1, keepdim=True)
    lse = torch.logsumexp(z, 1, keepdim=True)
    es = (300 + V / 64) * u
    nll = lse.view(-1) - z.gather(1, tg[:, None]).view(-1)
    loss = (nll * mo).sum() / den
    eloss = ((2 * ez.view(-1) + es + 4 * u * lse.abs().view(-1)) * mo.abs()).sum() / den.abs() + 2 * u * loss.abs() + 1100 * u * (nll * mo).abs().sum() / den.abs()
    g = dloss / den
    p = torch.exp(z - lse)
    dz = p.clone()
    dz[torch.arange(on.numel(), device=DEV), tg] -= 1
    edz = p * (2 * ez + es + 8 * u * (1 + lse.abs())) + (hp + 4 * u) * dz.abs() + tiny
    wr = (g * mo).view(-1, 1)
    dz, edz = dz * wr, edz * wr.abs()
    R = on.numel()
    ax, aw = dz.abs() @ w.abs(), dz.abs().t() @ x.abs()
    sub = 2.0 ** -25 if dtype == F16 else 0.0
    dx, dw, db = dz @ w, dz.t() @ x, dz.sum(0)
    ex = edz @ w.abs() + ((V + 8) * u + k3) * ax + far * V * (dz.abs().amax(1, keepdim=True) if R else 0) * w.abs().amax(0) + h * dx.abs() + sub
    ew = edz.t() @ x.abs() + ((R + 8) * u + k3) * aw + h * dw.abs() + sub
    if R:
        ew = ew + far * R * dz.abs().amax(0)[:, None] * x.abs().amax(0)
    eb = edz.sum(0) + (R + 8) * u * dz.abs().sum(0) + h * db.abs() + sub
    full, efull = torch.zeros(B * T, D, device=DEV).double(), torch.zeros(B * T, D, device=DEV).double()
    full[on], efull[on] = dx, ex
    return [loss, full.view(B, T, D), dw, db], [eloss, efull.view(B, T, D), ew, eb]


def run(t, denom=None, dloss=1.0):
    from ekaid_amd import ops
    leaves = {n: t[n].detach().requires_grad_(True) for n in ('x', 'weight', 'bias') if t[n] is not None}
    loss = ops.linear_lm_loss(leaves['x'], leaves['weight'], leaves.get('bias'), t['target'], t['mask'], denom)
    return [loss.detach()] + list(torch.autograd.grad(loss, list(leaves.values()), torch.tensor(dloss, device=DEV)))


def compare(got, want, what=''):
    vals, bnds = want
    for n, a, w, b in zip(('loss', 'dx', 'dweight', 'dbias'), got, vals, bnds):
        assert a.shape == w.shape, (n, a.shape, w.shape)
        assert torch.isfinite(a).all(), '%s %s: non-finite' % (what, n)
        over = (a.double() - w).abs() / (b + 1e-30)
        assert float(over.max()) <= 1.0, '%s %s: %.3g times the bound (err %.3e)' % (what, n, float(over.max()), float((a.double() - w).abs().max()))


SHAPES = [
    # B, T, D, V
    (2, 3, 8, 1), (1, 1, 64, 2), (2, 5, 64, 7), (3, 37, 72, 300), (4, 90, 512, 148), (2, 300, 136, 1000), (2, 300, 64, 12811), (5, 103, 1024, 517),
]


@gpu
@pytest.mark.parametrize('dtype', [F32, BF16, F16], ids=IDS)
@pytest.mark.parametrize('shape', SHAPES, ids=lambda s: 'x'.join(map(str, s)))
def test_loss_and_gradients(shape, dtype):
    t = make(dtype, *shape)
    got = run(t)
    compare(got, reference(t))
    assert all(torch.equal(a, b) for a, b in zip(got, run(t)))
    t['bias'] = None
    compare(run(t, dloss=3.0), reference(t, dloss=3.0), 'no bias')


@gpu
@pytest.mark.parametrize('shape', [(1, 1, 4, 1), (3, 7, 4, 4), (2, 33, 60, 60), (2, 40, 68, 65), (7, 97, 132, 129), (2, 33, 60, 40), (7, 97, 132, 113), (2, 20, 16, 16), (9, 40, 20, 3), (3, 50, 256, 256), (64, 90, 512, 148), (5, 61, 1028, 200)],
                         ids=lambda s: 'x'.join(map(str, s)))
def test_few_words(shape):
    """No more words, in whole sixteens, than the width (f32: whole rows of logits in one workgroup), and sizes just beside that: whatever stands
    in rows that do not count, weighted rows; each gradient alone is the one of the full call; a weight gradient into an unaligned slot."""
    from ekaid_amd import ops
    B, T, D, V = shape
    t = make(F32, *shape)
    t['mask'] = t['mask'] * (torch.arange(B * T, device=DEV).view(B, T) % 5 + 1) / 4
    if B > 1:
        t['mask'][:B // 2 + 1].mul_(torch.tensor(0.0, device=DEV))
    off = t['mask'] == 0
    t['x'][off] = float('nan')
    t['target'][off] = 10 ** 12
    want = reference(t, dloss=0.5)
    got = run(t, dloss=0.5)
    if off.all():                                             # nothing counts (two samples, both masked): loss 0 / 0, gradients 0
        assert torch.isnan(want[0][0]) and torch.isnan(got[0])
        assert all(float(g.abs().max()) == 0 for g in got[1:])
    else:
        compare(got, want)
    for k, name in enumerate(('x', 'weight', 'bias')):
        leaf = {n: t[n].detach().requires_grad_(n == name) for n in ('x', 'weight', 'bias')}
        loss = ops.linear_lm_loss(leaf['x'], leaf['weight'], leaf['bias'], t['target'], t['mask'])
        alone = torch.autograd.grad(loss, leaf[name], torch.tensor(0.5, device=DEV))[0]
        if (V + 15) // 16 * 16 <= D:
            assert torch.equal(alone, got[1 + k]), name
        else:                                                 # the other route: a bias gradient alone is summed in another order, within its bound
            assert bool(((alone.double() - want[0][1 + k]).abs() <= want[1][1 + k] + 1e-30).all()), name
    flat = torch.zeros(V * D + 1, device=DEV)                 # the weight's gradient into a slot of a flat buffer that is no whole vector
    ops._grad_slots[t['weight'].data_ptr()] = (t['weight'], flat, 1, V * D, (V, D))
    try:
        run(t, dloss=0.5)
    finally:
        del ops._grad_slots[t['weight'].data_ptr()]
        ops._grad_claimed.discard(t['weight'].data_ptr())
    assert torch.equal(flat[1:].view(V, D), got[2])
    t['weight'][V // 2, 0] = float('inf')
    assert not torch.isfinite(run(t)[0])


@gpu
@pytest.mark.parametrize('mode', ['f32', 'bf16x3', 'f16x2'])
def test_f32_arithmetics_and_odd_widths(mode):
    """Every product arithmetic, a width that is no whole vector, a size that takes the operand bounds of the two-term split."""
    from ekaid_amd import ops
    old = ops.get_gemm_mode()
    ops.set_gemm_mode(dict(f32=ops.GEMM_F32_MFMA, bf16x3=ops.GEMM_BF16_SPLIT, f16x2=ops.GEMM_F16X2)[mode])
    try:
        for shape in ((2, 21, 37, 203), (8, 256, 512, 6001), (8, 256, 516, 6001)):
            t = make(F32, *shape)
            compare(run(t), reference(t), str(shape))
    finally:
        ops.set_gemm_mode(old)


@gpu
@pytest.mark.parametrize('dtype,V,mode', [(F32, 8300, None), (F32, 8300, 1), (BF16, 9001, None), (BF16, 17001, None)], ids=['f32', 'f32-bf16x3', 'bf16', 'bf16-2'])
def test_vocabulary_in_several_pieces(dtype, V, mode):
    from ekaid_amd import ops
    old = ops.get_gemm_mode()
    ops.set_gemm_mode(old if mode is None else mode)
    try:
        t = make(dtype, 4, 4100, 16, V)
        compare(run(t), reference(t))
    finally:
        ops.set_gemm_mode(old)


@gpu
@pytest.mark.parametrize('xs', [1.0, 25.0])
def test_f32_terms_of_uneven_magnitudes(xs):
    """Rows and words whose magnitudes differ by powers of ten, rows decided by one word: every output element within its own bound."""
    t = make(F32, 6, 200, 256, 8111, xs=xs)
    g = torch.Generator().manual_seed(12)
    t['x'] = t['x'] * (10.0 ** torch.randint(-4, 1, (6, 200, 1), generator=g)).to(DEV)
    t['weight'] = t['weight'] * (10.0 ** torch.randint(-3, 1, (8111, 1), generator=g)).to(DEV)
    t['weight'][5] = 0
    compare(run(t), reference(t))


@gpu
@pytest.mark.parametrize('dtype', [F32, BF16, F16], ids=IDS)
def test_masks(dtype):
    """Weights, a large common factor, one row alone, a supplied denominator; rows that do not count hold NaN and targets out of range."""
    base = make(dtype, 4, 70, 64, 333)
    g = torch.Generator().manual_seed(8)
    for what in ('weights', 'large', 'one', 'denom'):
        t = dict(base)
        t['mask'] = base['mask'].clone()
        denom = None
        if what == 'weights':
            t['mask'] = torch.rand(4, 70, generator=g).to(DEV) * (torch.rand(4, 70, generator=g).to(DEV) > 0.4)
            t['mask'][2, 3] = -0.5
        elif what == 'large':
            t['mask'] = t['mask'] * 1e6
        elif what == 'one':
            t['mask'] = torch.zeros(4, 70, device=DEV)
            t['mask'][1, 17] = 1.0
        else:
            denom = torch.tensor(311.0, device=DEV)
        dead = t['mask'] == 0
        t['x'] = t['x'].clone()
        t['target'] = t['target'].clone()
        want = reference(t, denom)
        t['x'][dead] = float('nan')
        t['target'][dead] = torch.where(torch.rand(4, 70, generator=g).to(DEV)[dead] > 0.5, -100, 1 << 40)
        got = run(t, denom)
        compare(got, want, what)
        assert (got[1][dead] == 0).all()


@gpu
@pytest.mark.parametrize('dtype', [F32, BF16], ids=['f32', 'bf16'])
def test_nothing_counts_and_targets_outside(dtype):
    t = make(dtype, 2, 9, 64, 50)
    t['mask'] = torch.zeros(2, 9, device=DEV)
    got = run(t)
    assert torch.isnan(got[0]) and all((x == 0).all() for x in got[1:])
    got = run(t, denom=torch.tensor(4.0, device=DEV))
    assert got[0] == 0 and all((x == 0).all() for x in got[1:])
    got = run(t, denom=torch.tensor(4.0, device=DEV), dloss=float('inf'))
    assert all((x == 0).all() for x in got[1:])
    for bad in (-1, 50, 1 << 40):
        t = make(dtype, 2, 9, 64, 50)
        t['mask'][:] = 1
        t['target'][1, 4] = bad
        assert torch.isnan(run(t)[0])
    from ekaid_amd import ops
    x = torch.zeros(0, 5, 64, device=DEV, dtype=dtype, requires_grad=True)
    w = torch.zeros(50, 64, device=DEV, dtype=dtype, requires_grad=True)
    loss = ops.linear_lm_loss(x, w, None, torch.zeros(0, 5, device=DEV, dtype=torch.int64), torch.zeros(0, 5, device=DEV))
    gx, gw = torch.autograd.grad(loss, [x, w])
    assert torch.isnan(loss) and gx.shape == x.shape and (gw == 0).all()


@gpu
@pytest.mark.parametrize('dtype', [F32, BF16, F16], ids=IDS)
def test_extreme_logits(dtype):
    """Logits of several hundred (a row decided by one word), a word of bias -inf (excluded), incoming gradients of 2^-14 and 2^14."""
    t = make(dtype, 2, 40, 64, 500, xs=60.0)
    compare(run(t), reference(t))
    t = make(dtype, 2, 40, 64, 500)
    t['bias'][7] = -math.inf
    t['target'][t['target'] == 7] = 8
    got = run(t)
    t2 = dict(t, bias=t['bias'].clone())
    t2['bias'][7] = -3e4
    compare(got, reference(t2))
    assert (got[2][7] == 0).all() and got[3][7] == 0
    t = make(dtype, 2, 40, 64, 500)
    for d in (2.0 ** -14, 2.0 ** 14):
        compare(run(t, dloss=d), reference(t, dloss=d), str(d))


@gpu
@pytest.mark.parametrize('dtype', [F32, BF16], ids=['f32', 'bf16'])
def test_strided_operands(dtype):
    """Time-major states, a column slice, an odd storage offset, labels and masks cut from wider tensors."""
    t = make(dtype, 3, 11, 64, 100)
    want = run(t)
    labels = torch.zeros(3, 15, dtype=torch.int64, device=DEV)
    masks = torch.ones(3, 15, device=DEV)
    labels[:, 1:12], masks[:, 1:12] = t['target'], t['mask']
    alt = dict(t, target=labels[:, 1:], mask=masks[:, 1:])
    tb = t['x'].transpose(0, 1).contiguous().transpose(0, 1)
    wide = torch.zeros(3, 11, 72, device=DEV, dtype=dtype)
    wide[..., :64] = t['x']
    odd = torch.zeros(3 * 11 * 64 + 1, device=DEV, dtype=dtype)
    odd[1:] = t['x'].reshape(-1)
    for x in (tb, wide[..., :64], odd[1:].view(3, 11, 64)):
        got = run(dict(alt, x=x))
        assert all(torch.equal(a, b) for a, b in zip(got, want))
    got = run(dict(t, weight=t['weight'].t().contiguous().t(), target=t['target'].t().contiguous().t(), mask=t['mask'].t().contiguous().t()))
    assert all(torch.equal(a, b) for a, b in zip(got, want))


@gpu
def test_equals_the_frameworks_chain():
    """lm_loss(log_softmax(linear)) of the framework, its criterion class and a gradient slot of the optimizer's flat buffer."""
    from ekaid_amd import ops
    from ekaid_amd.models.fc import Linear
    from ekaid_amd.utils.utils import LanguageModelCriterion, LinearLanguageModelCriterion
    t = make(F32, 6, 20, 512, 148)
    layer = Linear(512, 148).to(DEV)
    with torch.no_grad():
        layer.weight.copy_(t['weight'])
        layer.bias.copy_(t['bias'])
    res = []
    for fused in (False, True):
        layer.zero_grad(set_to_none=True)
        x = t['x'].clone().requires_grad_(True)
        loss = LinearLanguageModelCriterion()(x, layer, t['target'], t['mask']) if fused else LanguageModelCriterion()(ops.log_softmax(layer(x)), t['target'], t['mask'])
        loss.backward()
        res.append([loss.detach(), x.grad, layer.weight.grad, layer.bias.grad])
    want = reference(t)
    for r in res:
        compare(r, want)
    layer.zero_grad(set_to_none=True)
    flat = torch.zeros(148 * 512, device=DEV)
    ops.register_grad_slot(layer.weight, flat, 0)
    try:
        ops.clear_grad_claims()
        LinearLanguageModelCriterion()(t['x'], layer, t['target'], t['mask']).backward()
        assert layer.weight.grad.data_ptr() == flat.data_ptr() and torch.equal(flat.view(148, 512), res[1][2])
    finally:
        ops._grad_slots.pop(layer.weight.data_ptr())
        ops.clear_grad_claims()


@gpu
def test_gradient_against_differences():
    t = make(F32, 2, 12, 40, 90)
    got = run(t)
    for n, gr in zip(('x', 'weight', 'bias'), got[1:]):
        e = torch.randn(t[n].shape, generator=torch.Generator().manual_seed(4)).to(DEV)
        step = 2.0 ** -10
        f = [float(reference({**{a: (b.double() if b.is_floating_point() else b) for a, b in t.items()}, n: t[n].double() + s * step * e.double()})[0][0]) for s in (1, -1)]
        want = (f[0] - f[1]) / (2 * step)
        assert abs(float((gr.double() * e).sum()) - want) <= 1e-3 * max(1.0, abs(want))


@gpu
def test_streams_and_captured_replays():
    from ekaid_amd import ops
    cases = [make(BF16, 3, 50, 64, 700), make(F32, 2, 60, 128, 900), make(F16, 2, 300, 64, 12811)]
    eager = [run(t) for t in cases]
    streams = [torch.cuda.Stream() for _ in cases]
    torch.cuda.synchronize()
    got = []
    for _ in range(4):
        for i, t in enumerate(cases):
            with torch.cuda.stream(streams[i]):
                got.append(run(t))
    torch.cuda.synchronize()
    for i, g in enumerate(got):
        assert all(torch.equal(a, b) for a, b in zip(g, eager[i % 3]))
    for t, want in zip(cases, eager):
        x, w, b = (t[n].detach().clone().requires_grad_(True) for n in ('x', 'weight', 'bias'))
        one = torch.ones((), device=DEV)
        gr = torch.cuda.CUDAGraph()
        torch.cuda.synchronize()
        with torch.cuda.graph(gr):
            loss = ops.linear_lm_loss(x, w, b, t['target'], t['mask'])
            res = [loss] + list(torch.autograd.grad(loss, [x, w, b], one))
        for rep in range(3):
            with torch.no_grad():
                x.mul_(1.0 if rep == 0 else -1.5)
            gr.replay()
            torch.cuda.synchronize()
            again = run(dict(t, x=x.detach(), weight=w.detach(), bias=b.detach()))
            assert all(torch.equal(p, q) for p, q in zip([r.detach() for r in res], again))
            if rep == 0:
                assert all(torch.equal(p, q) for p, q in zip([r.detach() for r in res], want))


@gpu
@pytest.mark.parametrize('dtype', [F32, BF16], ids=['f32', 'bf16'])
def test_single_gradients(dtype):
    """Each gradient asked for alone (a frozen layer, frozen states) is the one of the full call."""
    from ekaid_amd import ops
    t = make(dtype, 3, 40, 64, 333)
    want = reference(t)
    for n in ('x', 'weight', 'bias'):
        leaf = t[n].detach().requires_grad_(True)
        a = dict(t, **{n: leaf})
        (g,) = torch.autograd.grad(ops.linear_lm_loss(a['x'], a['weight'], a['bias'], t['target'], t['mask']), [leaf])
        i = ('x', 'weight', 'bias').index(n) + 1
        compare([want[0][0].float(), *[w.to(dtype) if k != i else g for k, w in enumerate(want[0])][1:]], want, n)


@gpu
def test_refusals():
    from ekaid_amd import ops
    from ekaid_amd.hip import EkaidError
    z = lambda *s, dt=F32: torch.zeros(*s, device=DEV, dtype=dt)           # noqa: E731
    x, w, b, tg, m = z(2, 3, 16), z(5, 16), z(5), z(2, 3, dt=torch.int64), z(2, 3)
    bad = [
        lambda: ops.linear_lm_loss(x.cpu(), w.cpu(), None, tg.cpu(), m.cpu()), lambda: ops.linear_lm_loss(x[0], w, b, tg, m), lambda: ops.linear_lm_loss(x, z(5, 8), b, tg, m),
        lambda: ops.linear_lm_loss(x.double(), w.double(), None, tg, m), lambda: ops.linear_lm_loss(x, w.half(), None, tg, m), lambda: ops.linear_lm_loss(x, w, b.half(), tg, m),
        lambda: ops.linear_lm_loss(z(2, 3, 12, dt=BF16), z(5, 12, dt=BF16), None, tg, m), lambda: ops.linear_lm_loss(x, w, z(4), tg, m), lambda: ops.linear_lm_loss(x, w, b, tg.int(), m),
        lambda: ops.linear_lm_loss(x, w, b, tg[:, :2], m), lambda: ops.linear_lm_loss(x, w, b, tg, m.double()), lambda: ops.linear_lm_loss(x, w, b, tg[:1], m),
        lambda: ops.linear_lm_loss(x, w, b, tg, m, denom=z(2)), lambda: ops.linear_lm_loss(x, z(0, 16), None, tg, m), lambda: ops.linear_lm_loss(x, w, b, tg, m.cpu()),
    ]
    for i, f in enumerate(bad):
        with pytest.raises(EkaidError):
            f()
            raise AssertionError('call %d was taken' % i)


def test_c_entry_refuses_bad_descriptors():
    from ekaid_amd import hip
    L = hip.load()

    def desc(**kw):
        d = hip.LinearLoss()
        for n in ('x', 'weight', 'target', 'mask', 'loss', 'state', 'dloss', 'dx', 'dweight'):
            setattr(d, n, 1 << 20)
        d.dtype, d.B, d.T, d.D, d.V, d.ldx, d.ld_target, d.ld_mask = 1, 2, 3, 64, 100, 64, 3, 3
        for n, x in kw.items():
            setattr(d, n, x)
        return d
    for kw in (dict(dtype=5), dict(B=-1), dict(D=0), dict(V=0), dict(D=60), dict(ldx=68), dict(ldx=32), dict(x=(1 << 20) + 2), dict(weight=(1 << 20) + 8), dict(T=1 << 30),
               dict(dx=(1 << 20) + 4)):
        d = desc(**kw)
        for entry in (L.ekaid_linear_loss_fwd, L.ekaid_linear_loss_bwd):
            assert entry(ctypes.byref(d), 1 << 20, 1 << 40, None) < 0 and hip.last_error(), kw
        assert L.ekaid_linear_loss_workspace_bytes(ctypes.byref(d), 1) == 0 and L.ekaid_linear_loss_state_bytes(ctypes.byref(d)) == 0
    for n in ('x', 'weight', 'target', 'mask', 'state'):
        d = desc(**{n: None})
        assert L.ekaid_linear_loss_fwd(ctypes.byref(d), 1 << 20, 1 << 40, None) < 0
        assert L.ekaid_linear_loss_bwd(ctypes.byref(d), 1 << 20, 1 << 40, None) < 0
    assert L.ekaid_linear_loss_fwd(ctypes.byref(desc()), None, 0, None) < 0 and 'workspace' in hip.last_error()
    assert L.ekaid_linear_loss_bwd(ctypes.byref(desc()), 1 << 20, 16, None) < 0
    assert L.ekaid_linear_loss_bwd(ctypes.byref(desc(B=0)), 1 << 20, 1 << 40, None) < 0
    assert L.ekaid_linear_loss_fwd(None, None, 0, None) < 0 and L.ekaid_linear_loss_bwd(None, None, 0, None) < 0


def test_few_words_state_and_alignment():
    """The logits kept for the backward are a matter of sizes, not of addresses; what the kernels write whole vectors to must be aligned."""
    from ekaid_amd import hip
    L = hip.load()

    def desc(**kw):
        d = hip.LinearLoss()
        for n in ('x', 'weight', 'target', 'mask', 'loss', 'state', 'dloss', 'dx', 'dweight'):
            setattr(d, n, 1 << 20)
        d.dtype, d.B, d.T, d.D, d.V, d.ldx, d.ld_target, d.ld_mask = 0, 2, 3, 64, 50, 64, 3, 3
        for n, x in kw.items():
            setattr(d, n, x)
        return d

    def state(**kw):
        return L.ekaid_linear_loss_state_bytes(ctypes.byref(desc(**kw)))
    wide = state(V=65)
    assert state() == state(x=(1 << 20) + 4, weight=0) == wide + 6 * 64 * 4
    assert state(V=64) == state() and state(V=16) == wide + 6 * 16 * 4 and state(V=256, D=256, ldx=256) == wide + 6 * 256 * 4
    for kw in (dict(V=257, D=512, ldx=512), dict(D=62, V=20, ldx=62), dict(dtype=1), dict(B=1 << 14, T=1 << 7, D=1024, ldx=1024, V=1),
               dict(B=1 << 13, T=1 << 7, D=1028, ldx=1028, V=1)):
        n = max(kw.get('B', 2) * kw.get('T', 3), 6)
        assert state(**kw) <= 512 + 20 * n, kw
    assert L.ekaid_linear_loss_workspace_bytes(ctypes.byref(desc()), 0) == 0
    for kw in (dict(state=(1 << 20) + 8), dict(dx=(1 << 20) + 4)):
        assert L.ekaid_linear_loss_bwd(ctypes.byref(desc(**kw)), 1 << 20, 1 << 40, None) < 0 and 'aligned' in hip.last_error(), kw
    assert L.ekaid_linear_loss_fwd(ctypes.byref(desc(state=(1 << 20) + 8)), 1 << 20, 1 << 40, None) < 0


@gpu
@pytest.mark.parametrize('offset', [0.0, 40.0, -3000.0])
@pytest.mark.parametrize('V', [6001, 10007], ids=['128-tiles', '256-tiles'])
def test_f32_rows_decided_by_their_own_target(V, offset):
    """Well predicted words, target logits of 20 to 90 above a common offset: what is left of 1 - p is the rounding of the logits, and
    every gradient keeps its bound.  (N V D above 2^31: the route of two f16 terms.)"""
    B, T, D = 8, 128, 512
    t = make(F32, B, T, D, V)
    height = torch.linspace(20, 90, B * T, device=DEV).view(B, T, 1)
    t['mask'][:] = 1
    t['mask'][3, 50:] = 0.25
    w = t['weight'][t['target']]
    t['x'] = w * (height / (w * w).sum(2, keepdim=True))
    t['bias'] = t['bias'] * 0.1 + offset
    assert B * T * V * D >= 1 << 31
    want = reference(t)
    compare(run(t), want)
    t['x'][0, 5:9] *= -1                                          # some of them predicted as badly
    compare(run(t), reference(t), 'mixed')


@gpu
def test_f32_rows_decided_against_large_cancelling_bias():
    """Logits that are the small difference of a large bias and a large product: their error is that of the large parts, no gradient overflows."""
    B, T, D, V = 8, 128, 512, 6001
    t = make(F32, B, T, D, V)
    t['mask'][:] = 1
    w = t['weight'][t['target']]
    t['x'] = w * (60.0 / (w * w).sum(2, keepdim=True))
    t['x'][..., 0], t['weight'][:, 0] = 64.0, -64.0                # -4096 in every logit
    t['bias'] = t['bias'] * 0.1 + 4096.0
    compare(run(t), reference(t))


@gpu
def test_f32_terms_of_the_largest_magnitudes():
    """A row of x near the end of f32's range: its logits are finite, and so is everything else (N V D above 2^31)."""
    t = make(F32, 4, 256, 256, 8200)
    t['mask'][:] = 1
    t['mask'][1, :100] = 0
    t['x'][2, 7] *= 2.0 ** 120
    compare(run(t), reference(t))


@gpu
def test_f32_words_of_a_hundred_powers_of_ten():
    """Words of 2^90 and 2^-100 of the usual size beside the others: their gradients come out as every other word's (N V D above 2^31)."""
    t = make(F32, 4, 256, 256, 8200)
    t['mask'][:] = 1
    t['weight'][5] *= 2.0 ** 90
    t['weight'][9] *= 2.0 ** -100
    t['target'][t['target'] == 5] = 6
    got, want = run(t), reference(t)
    compare(got, want)
    # the largest word's bound hides the others': for the tiny word, where the largest takes no part (its logit far below), by hand
    x, w, u = t['x'].double().view(-1, 256), t['weight'].double(), 2.0 ** -24
    z = x @ w.t() + t['bias'].double()
    p = torch.softmax(z, 1)[:, 9:10]
    S = float((x.abs() @ torch.cat((w[:5], w[6:])).abs().t()).max())
    rel = 2 * ((256 + 8) * u + 2.0 ** -21) * S + (300 + 8200 / 64) * u + 8 * u * (1 + S) + (1024 + 8) * u + 2.0 ** -21
    assert bool(((got[2][9].double() - want[0][2][9]).abs() <= rel * (p * x.abs()).sum(0) / 1024 + 2.0 ** -23 * want[0][2][9].abs()).all())


@gpu
@pytest.mark.parametrize('shape', [(2, 21, 37, 203), (3, 50, 64, 300), (8, 256, 516, 6001)], ids=str)
@pytest.mark.parametrize('first,then', [(0, 1), (1, 0), (2, 0), (1, 2)])
def test_f32_arithmetic_is_the_forwards(first, then, shape):
    """The mode is changed between the forward and its backward: the backward stays with the arithmetic its denominators came from."""
    from ekaid_amd import ops
    t = make(F32, *shape)
    leaves = [t[n].detach().requires_grad_(True) for n in ('x', 'weight', 'bias')]
    old, res = ops.get_gemm_mode(), []
    try:
        for later in (first, then):
            ops.set_gemm_mode(first)
            loss = ops.linear_lm_loss(*leaves, t['target'], t['mask'])
            ops.set_gemm_mode(later)
            res.append([loss.detach()] + list(torch.autograd.grad(loss, leaves)))
            assert ops.get_gemm_mode() == later
    finally:
        ops.set_gemm_mode(old)
    assert all(torch.equal(a, b) for a, b in zip(*res))


def test_c_entry_refuses_unknown_arithmetics():
    from ekaid_amd import hip
    L = hip.load()
    d = hip.LinearLoss()
    for n in ('x', 'weight', 'target', 'mask', 'loss', 'state', 'dloss', 'dx', 'dweight'):
        setattr(d, n, 1 << 20)
    d.dtype, d.B, d.T, d.D, d.V, d.ldx, d.ld_target, d.ld_mask = 0, 2, 3, 64, 500, 64, 3, 3
    for arith in (-1, 3, 7):
        d.arith = arith
        for entry in (L.ekaid_linear_loss_fwd, L.ekaid_linear_loss_bwd):
            assert entry(ctypes.byref(d), 1 << 20, 1 << 40, None) < 0 and 'arithmetic' in hip.last_error()
        assert L.ekaid_linear_loss_workspace_bytes(ctypes.byref(d), 1) == 0


@gpu
def test_operands_are_copied_only_where_it_helps():
    """A width of no whole vectors has no aligned rows to copy to: x is kept as it is.  Rows that a copy aligns are copied."""
    from ekaid_amd import ops
    t = make(F32, 2, 9, 37, 300)
    for x, kept in ((t['x'], True), (make(F32, 2, 9, 40, 300)['x'], True), (torch.randn(2 * 9 * 37 + 1, device=DEV)[1:].view(2, 9, 37), True), (torch.randn(2, 9, 41, device=DEV)[..., :40], False),
                    (torch.randn(2 * 9 * 40 + 1, device=DEV)[1:].view(2, 9, 40), False)):
        w = torch.randn(300, x.shape[2], device=DEV, requires_grad=True)
        loss = ops.linear_lm_loss(x, w, None, t['target'], t['mask'])
        assert (loss.grad_fn.saved_tensors[0].data_ptr() == x.data_ptr()) == kept
        assert torch.equal(loss.detach(), ops.linear_lm_loss(x.clone(memory_format=torch.contiguous_format), w, None, t['target'], t['mask']).detach())


def test_c_entry_refuses_more_threads_than_a_launch_counts():
    from ekaid_amd import hip
    L = hip.load()

    def desc(dtype, n, V, D=64, arith=2):
        d = hip.LinearLoss()
        for name in ('x', 'weight', 'target', 'mask', 'loss', 'state', 'dloss', 'dx', 'dweight'):
            setattr(d, name, 1 << 20)
        d.dtype, d.B, d.T, d.D, d.V, d.ldx, d.ld_target, d.ld_mask, d.arith = dtype, 1, n, D, V, D, n, n, arith
        return d
    for case in ((0, 1 << 26, 1), (0, 1 << 25, 1 << 25), (0, 1 << 20, 1 << 19), (1, 1 << 20, 1 << 19), (2, 1 << 28, 1)):
        d = desc(*case)
        for entry in (L.ekaid_linear_loss_fwd, L.ekaid_linear_loss_bwd):
            assert entry(ctypes.byref(d), 1 << 20, 1 << 60, None) < 0 and 'too many' in hip.last_error(), case
        assert L.ekaid_linear_loss_state_bytes(ctypes.byref(d)) == 0
    for case in ((0, 1 << 25, 1), (0, 1 << 20, 1 << 19, 64, 0), (0, 1 << 19, 1 << 19), (1, 1 << 19, 1 << 19), (2, 1 << 27, 1)):
        assert L.ekaid_linear_loss_state_bytes(ctypes.byref(desc(*case))) > 0, case
