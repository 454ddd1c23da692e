"""relative_attention, cross_attention and linear_lm_loss together, as a decoder over regions uses them: words attend to earlier words with a
learned distance bias, then to the regions, and the loss of the next word is taken without its logits; words one at a time against the
sequence at once.

Bounds, relative in the 2-norm of a tensor.  float32: 16 u for every term of the longest sums in turn (widths 64, 48, 45 keys, 40 regions,
203 words; u = 2^-24; 16 for the growth through six stages), plus 2^-21 of each of the six split-arithmetic products, times 4 for the
same growth.  16 bits: half a step for each of the twelve tensors that are rounded along the longest path."""
import ctypes
import math
import os
import shutil
import subprocess

import pytest
import torch

F32, BF16 = torch.float32, torch.bfloat16
DEV = 'cuda'
gpu = pytest.mark.gpu
ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
BOUND = {F32: 16 * (64 + 48 + 45 + 40 + 203) * 2.0 ** -24 + 4 * 6 * 2.0 ** -21, BF16: 12 * 2.0 ** -8}


def test_descriptors_have_the_layout_of_the_c_structs(tmp_path):
    """Size and every field's offset of the two descriptors, as gcc lays the header out, against their ctypes mirrors."""
    from ekaid_amd import hip
    if shutil.which('gcc') is None:
        pytest.skip('no C compiler')
    src = ['#include <stdio.h>', '#include <stddef.h>', '#include "%s"' % os.path.join(ROOT, 'include', 'ekaid_hip.h'), 'int main(void) {']
    want = []
    for cname, mirror in (('ekaid_attn_t', hip.Attn), ('ekaid_linear_loss_t', hip.LinearLoss)):
        src.append('  printf("%%zu\\n", sizeof(%s));' % cname)
        want.append(ctypes.sizeof(mirror))
        for f in mirror._fields_:
            src.append('  printf("%%zu\\n", offsetof(%s, %s));' % (cname, f[0]))
            want.append(getattr(mirror, f[0]).offset)
    c, exe = tmp_path / 'layout.c', tmp_path / 'layout'
    c.write_text('\n'.join(src + ['  return 0;', '}']))
    subprocess.run(['gcc', str(c), '-o', str(exe)], check=True)
    assert [int(x) for x in subprocess.run([str(exe)], check=True, capture_output=True, text=True).stdout.split()] == want


B, T, R, E, H, KV, V, NB, MD = 3, 45, 40, 48, 6, 2, 203, 16, 24
DH = E // H
NAMES = ('wq', 'wk', 'wv', 'table', 'cq', 'ck', 'cv', 'words', 'bias')


def tensors(dtype):
    g = torch.Generator().manual_seed(5)
    r = lambda *s: torch.randn(*s, generator=g)                        # noqa: E731
    t = dict(x=r(B, T, E), regions=r(B, R, 64), wq=r(E, E) / E ** 0.5, wk=r(E, E) / E ** 0.5, wv=r(E, E) / E ** 0.5, table=r(NB, H) * 0.5, cq=r(E, E) / E ** 0.5,
             ck=r(KV * DH, 64) / 8, cv=r(KV * DH, 64) / 8, words=r(V, E) / E ** 0.5, bias=r(V) * 0.3)
    t = {n: (v if n == 'table' else v.to(dtype)) for n, v in t.items()}
    t['target'] = torch.randint(0, V, (B, T), generator=g)
    t['mask'] = (torch.arange(T)[None] < torch.tensor([[T], [1], [17]])).float()
    t['seen'] = torch.arange(R)[None] < torch.tensor([[R], [7], [0]])               # one sample sees no region
    return t


def linear(x, w):
    from ekaid_amd import ops
    return ops.linear(x, w, None) if x.dtype == F32 else torch.nn.functional.linear(x, w)


def decoder(t):
    from ekaid_amd import ops
    y = t['x'] + ops.relative_attention(linear(t['x'], t['wq']), linear(t['x'], t['wk']), linear(t['x'], t['wv']), t['table'], H, causal=True, max_distance=MD)
    y = y + ops.cross_attention(linear(y, t['cq']), linear(t['regions'], t['ck']), linear(t['regions'], t['cv']), H, kv_heads=KV, key_mask=t['seen'])
    return y, ops.linear_lm_loss(y, t['words'], t['bias'], t['target'], t['mask'])


def bucket(d):
    """One-sided: distance d back."""
    e = NB // 2
    return d if d < e else e + min(NB - e - 1, int(math.floor(math.log(d / e) / math.log(MD / e) * (NB - e) + 1e-9)))


def plain(t):
    """The same in float64, on the CPU."""
    def heads(x, n):
        return x.reshape(B, -1, n, DH).transpose(1, 2)

    def attend(q, k, v, n, s_bias, ok):
        k, v = (heads(x, n).repeat_interleave(H // n, 1) for x in (k, v))
        s = (heads(q, H) @ k.transpose(2, 3) / DH ** 0.5 + s_bias).masked_fill(~ok, -1e300)
        p = torch.softmax(s, 3) * ok
        return (p @ v).transpose(1, 2).reshape(B, T, E)
    back = torch.arange(T)[:, None] - torch.arange(T)[None]
    which = torch.tensor([[bucket(max(int(d), 0)) for d in row] for row in back])
    y = t['x'] + attend(t['x'] @ t['wq'].t(), t['x'] @ t['wk'].t(), t['x'] @ t['wv'].t(), H, t['table'][which].permute(2, 0, 1)[None], (back >= 0)[None, None])
    y = y + attend(y @ t['cq'].t(), t['regions'] @ t['ck'].t(), t['regions'] @ t['cv'].t(), KV, 0.0, t['seen'][:, None, None])
    nll = -torch.log_softmax(y @ t['words'].t() + t['bias'], 2).gather(2, t['target'][:, :, None])[:, :, 0]
    return y, (nll * t['mask']).sum() / t['mask'].sum()


def off(got, want):
    return float((got.double().cpu() - want).norm() / want.norm())


@gpu
@pytest.mark.parametrize('dtype', [F32, BF16], ids=['f32', 'bf16'])
def test_decoder_and_its_gradients(dtype):
    t = tensors(dtype)
    ref = {n: (v.double() if v.is_floating_point() else v) for n, v in t.items()}
    leaves = ('x', 'regions') + NAMES
    for n in leaves:
        ref[n].requires_grad_(True)
    y0, l0 = plain(ref)
    want = torch.autograd.grad(l0, [ref[n] for n in leaves])
    d = {n: v.to(DEV) for n, v in t.items()}
    for n in leaves:
        d[n].requires_grad_(True)
    y, loss = decoder(d)
    got = torch.autograd.grad(loss, [d[n] for n in leaves])
    for n, a, w in (('states', y.detach(), y0.detach()), ('loss', loss.detach(), l0.detach()), *zip(leaves, got, want)):
        assert off(a, w) <= BOUND[dtype], (n, off(a, w), BOUND[dtype])
    assert float(got[leaves.index('regions')][2].abs().max()) == 0          # (the sample that sees none)


@gpu
def test_words_one_at_a_time():
    """The states of a sequence at once, and word by word: keys and values of earlier words from a cache longer than the sequence, whose free
    places hold NaN, samples at different positions."""
    from ekaid_amd import ops
    d = {n: v.to(DEV) for n, v in tensors(F32).items()}
    whole = decoder(d)[0]
    start = torch.tensor([0, 3, 9], device=DEV)                              # words each sample has already read
    room = T + 20
    ck, cv = (torch.full((B, room, E), float('nan'), device=DEV) for _ in range(2))
    k, v = linear(d['x'], d['wk']), linear(d['x'], d['wv'])
    rk, rv = linear(d['regions'], d['ck']), linear(d['regions'], d['cv'])
    for b in range(B):
        n = int(start[b])
        ck[b, :n], cv[b, :n] = k[b, :n], v[b, :n]
    one = torch.arange(B, device=DEV)
    for step in range(30):
        at = start + step
        x = d['x'][one, at][:, None].contiguous()
        ck[one, at], cv[one, at] = linear(x, d['wk'])[:, 0], linear(x, d['wv'])[:, 0]
        y = x + ops.relative_attention(linear(x, d['wq']), ck, cv, d['table'], H, k_len=(at + 1).int(), q_pos=at.int(), causal=True, max_distance=MD)
        y = y + ops.cross_attention(linear(y, d['cq']), rk, rv, H, kv_heads=KV, key_mask=d['seen'])
        want = whole[one, at][:, None].double().cpu()
        assert off(y, want) <= BOUND[F32], (step, off(y, want))


@gpu
def test_decoder_replayed_from_a_graph():
    """Loss and gradients captured once, replayed with other inputs, eager work and a synchronization between the replays."""
    d = {n: v.to(DEV) for n, v in tensors(F32).items()}
    leaves = [d[n].requires_grad_(True) for n in NAMES]

    def run():
        y, loss = decoder(d)
        return [loss.detach()] + list(torch.autograd.grad(loss, leaves))
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        run()
    torch.cuda.current_stream().wait_stream(s)
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        kept = run()
    for k in range(4):
        with torch.no_grad():
            d['x'].normal_()
            d['target'].copy_((d['target'] * 7 + k) % V)
            d['mask'].copy_((torch.rand_like(d['mask']) < 0.3).float())
        d['mask'][0, 0] = 1.0
        torch.cuda.synchronize()
        eager = run()
        torch.cuda.synchronize()
        g.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(kept, eager)), k
