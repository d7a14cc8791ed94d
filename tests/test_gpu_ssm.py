"""The state-space layer's operators on the GPU against the plain float64 forms of ref_ssm.py.

Tolerances, in roundings of float32 (2^-24) at the largest value of a tensor:
  conv   K + 8 for an output (K products, the bias, SiLU's exponential, reciprocal and product, a few roundings each); a gradient
         adds another such chain: 4 (K + 8); dw / dbias are sums of M = B T terms added in runs of at most 32 and then of
         partial sums: at most M + 4 (K + 8) roundings of a running sum that is at most sum|terms| <= 4 sqrt(M) max|sum| for
         the random signs used here, in total far below M + 64.
  scan   8 roundings a frame at most enter the state (exponent argument 2, exponential 2, two products, one addition, delta's
         own) and |a| <= 1 carries them on: 8 T + 2 N + 32; a gradient runs such a chain twice and sums over N: 4 times as
         much, over frames and rows for parameters: + B T.
  norm   n / 64 + 16 roundings in a row's sum (64 lanes add at most n / 64 values each, then six joins): forward and backward.
  clip   the norm is summed in double: one rounding of the norm, two of the multiplier, one of the product: 8.
"""
import numpy as np
import pytest
import torch

import ref_ssm as R

pytestmark = pytest.mark.gpu
TY = {'f32': torch.float32, 'bf16': torch.bfloat16, 'f16': torch.float16}


def gen(seed):
    return torch.Generator(device='cpu').manual_seed(seed)


def rn(g, *shape, dtype=torch.float32, scale=1.0):
    return (torch.randn(*shape, generator=g) * scale).to(dtype).cuda()


def strided(g, T, B, D, dtype, kind):
    """'c': contiguous; 'half': the right half of twice the channels; 'bt': a (B, T, D) batch seen time-major; 'odd': rows one
    value longer than the channels (no 16-byte access)"""
    if kind == 'c':
        return rn(g, T, B, D, dtype=dtype)
    if kind == 'half':
        return rn(g, T, B, 2 * D, dtype=dtype)[:, :, D:]
    if kind == 'bt':
        return rn(g, B, T, D, dtype=dtype).transpose(0, 1)
    return rn(g, T, B, D + 1, dtype=dtype)[:, :, 1:]


def spoil(t, lens):
    """NaN and infinities in the padding: nothing of it may be used"""
    if lens is None:
        return t
    for b, n in enumerate(lens.tolist()):
        t[max(0, min(t.shape[0], n)):, b] = float('nan') if b % 2 else float('inf')
    return t


def clean(t, lens):
    v = R.leaf(t, False)
    if lens is not None and v is not None:
        for b, n in enumerate(lens.tolist()):
            v[max(0, min(v.shape[0], n)):, b] = 0
    return v


# ---------------------------------------------------------------------------------------------- convolution
CONV = [  # T, B, D, K, type, layout, lens, reverse, state, bias, act
    (1, 1, 1, 2, 'f32', 'c', None, False, False, True, 'silu'),
    (1, 3, 8, 4, 'bf16', 'c', None, False, True, True, 'silu'),
    (2, 2, 64, 4, 'f32', 'c', None, False, True, False, 'silu'),
    (7, 3, 5, 8, 'f32', 'c', [7, 0, 3], False, True, True, 'silu'),
    (33, 2, 100, 4, 'f32', 'half', [33, 17], False, False, True, 'silu'),
    (65, 3, 256, 4, 'bf16', 'half', [65, 64, 1], True, True, True, 'silu'),
    (130, 2, 72, 3, 'f16', 'bt', [130, 9], True, False, True, None),
    (129, 1, 24, 5, 'bf16', 'odd', None, True, True, False, 'silu'),
    (40, 4, 16, 7, 'f32', 'odd', [0, 0, 0, 0], False, True, True, 'silu'),
    (300, 2, 520, 4, 'f32', 'c', [300, 299], False, True, True, 'silu'),
    (64, 2, 40, 6, 'f16', 'c', [2, 64], False, True, True, 'silu'),
    (0, 2, 8, 4, 'f32', 'c', None, False, True, True, 'silu'),
    # a last thread whose channels are moved back to end with D, at either width of either pass
    (150, 2, 203, 4, 'bf16', 'odd', [150, 31], True, True, True, 'silu'),
    (70, 3, 131, 8, 'f16', 'half', [70, 0, 1], False, True, True, 'silu'),
    (90, 2, 130, 6, 'f32', 'odd', [90, 6], False, True, True, 'silu'),
    (40, 2, 67, 2, 'f32', 'c', None, True, True, True, None),
    (50, 2, 515, 3, 'f16', 'bt', [50, 50], True, True, False, 'silu'),
]


@pytest.mark.parametrize('case', CONV, ids=lambda c: '-'.join(str(v) for v in c).replace(' ', ''))
def test_conv(case):
    from asr_amd import ops
    T, B, D, K, ty, lay, lens, rev, st, bi, act = case
    ty = TY[ty]
    g = gen(T * 31 + D)
    x = strided(g, T, B, D, ty, lay)
    do = strided(g, T, B, D, ty, 'c')
    w = rn(g, D, K, scale=K ** -0.5)
    bias = rn(g, D, scale=0.3) if bi else None
    state = rn(g, K - 1, B, D, dtype=ty) if st else None
    dst = rn(g, K - 1, B, D, dtype=ty) if st else None
    ln = torch.tensor(lens, dtype=torch.int32).cuda() if lens else None
    x, do = spoil(x, ln), spoil(do, ln)
    out, new = ops.causal_conv_fwd(x, w, bias=bias, state=state, lens=ln, act=act, reverse=rev, want_state=True)
    gr = ops.causal_conv_bwd(do, x, w, bias=bias, state=state, lens=ln, act=act, reverse=rev, dstate_out=dst)
    torch.cuda.synchronize()
    rx, rw, rb, rs = clean(x, ln).requires_grad_(), R.leaf(w), R.leaf(bias), R.leaf(state)
    ro, rnew = R.conv(rx, rw, rb, rs, lens, act, rev)
    R.close(out, ro, K + 8, 'out')
    R.close(new, rnew, 0, 'state')
    loss = (ro * clean(do, ln)).sum()
    if st:
        loss = loss + (rnew * R.leaf(dst, False)).sum()
    ins = [('x', rx), ('w', rw)] + ([('bias', rb)] if bi else []) + ([('state', rs)] if st else [])
    ref = torch.autograd.grad(loss, [v for _, v in ins], allow_unused=True) if loss.requires_grad else [None] * len(ins)
    for (name, v), r in zip(ins, ref):
        r = torch.zeros_like(v) if r is None else r
        R.close(gr[name], r, 4 * (K + 8) + (B * T + 64 if name in ('w', 'bias') else 1), 'd' + name)
    assert (gr['bias'] is None) == (not bi) and (gr['state'] is None) == (not st)


@pytest.mark.parametrize('ty', ['f32', 'bf16', 'f16'])
@pytest.mark.parametrize('D,K', [(64, 4), (37, 3), (8, 8), (1, 2)])
def test_conv_steps_are_the_sequence(ty, D, K):
    """frame after frame through the state = the sequence at once, bit for bit (the same products in the same order), and a
    sequence in two calls = one"""
    from asr_amd import ops
    ty = TY[ty]
    g = gen(D)
    T, B = 11, 3
    x, w, bias = rn(g, T, B, D, dtype=ty), rn(g, D, K), rn(g, D)
    s0 = rn(g, K - 1, B, D, dtype=ty)
    out, end = ops.causal_conv_fwd(x, w, bias=bias, state=s0, want_state=True)
    st = s0.clone()
    steps = torch.stack([ops.causal_conv_step(x[t], st, w, bias=bias) for t in range(T)])
    assert torch.equal(steps, out) and torch.equal(st, end)
    a, mid = ops.causal_conv_fwd(x[:4], w, bias=bias, state=s0, want_state=True)
    b, end2 = ops.causal_conv_fwd(x[4:], w, bias=bias, state=mid, want_state=True)
    assert torch.equal(torch.cat([a, b]), out) and torch.equal(end2, end)


# ---------------------------------------------------------------------------------------------- scan
def scan_inputs(g, T, B, D, N, G, ty, lay='c', dt_scale=0.5):
    A = -(torch.arange(1, N + 1).float().repeat(D, 1) * (0.5 + torch.rand(D, N, generator=g))).cuda()
    a = dict(x=strided(g, T, B, D, ty, lay), dt=strided(g, T, B, D, ty, lay if lay != 'half' else 'c'), A=A)
    if dt_scale != 0.5:
        a['dt'] = a['dt'] * (2 * dt_scale)
    a['Bm'] = rn(g, T, B, G, N, dtype=ty)
    a['Cm'] = rn(g, T, B, G, 2 * N, dtype=ty)[..., N:] if lay == 'half' else rn(g, T, B, G, N, dtype=ty)
    step = torch.exp(torch.rand(D, generator=g) * 4.6 - 6.9)
    opt = dict(D=rn(g, D), z=strided(g, T, B, D, ty, lay), dt_bias=(step + torch.log(-torch.expm1(-step))).cuda(),
               h0=rn(g, B, D, N))
    return a, opt


SCAN = [  # T, B, D, N, G, type, layout, lens, reverse, options kept
    (1, 1, 1, 1, 1, 'f32', 'c', None, False, 'D z dt_bias h0'),
    (1, 2, 64, 16, 1, 'bf16', 'c', None, False, 'D z dt_bias h0'),
    (15, 2, 65, 16, 1, 'f32', 'c', None, False, ''),
    (16, 2, 63, 16, 1, 'f32', 'c', [16, 0], False, 'z'),
    (17, 3, 128, 16, 2, 'f32', 'half', [17, 16, 1], True, 'D z dt_bias h0'),
    (33, 2, 40, 8, 4, 'f32', 'bt', [33, 5], False, 'D dt_bias'),
    (37, 3, 200, 8, 2, 'bf16', 'half', [37, 0, 20], True, 'D z dt_bias h0'),
    (50, 2, 30, 5, 3, 'f16', 'odd', None, True, 'D z dt_bias h0'),
    (70, 2, 96, 20, 1, 'f32', 'c', [70, 33], False, 'D z dt_bias h0'),
    (66, 1, 130, 64, 1, 'f32', 'c', None, True, 'z h0'),
    (40, 2, 24, 33, 2, 'bf16', 'c', [1, 40], False, 'D z dt_bias h0'),
    (90, 1, 10, 3, 1, 'f32', 'c', None, False, 'D z dt_bias h0'),
    (40, 3, 16, 16, 1, 'f32', 'c', [0, 0, 0], False, 'D z dt_bias h0'),
    # long enough, and few enough rows, that time is cut into chunks
    (300, 1, 70, 16, 1, 'f32', 'c', None, False, 'D z dt_bias h0'),
    (300, 2, 48, 16, 3, 'f32', 'half', [300, 130], True, 'D z dt_bias h0'),
    (260, 2, 20, 4, 1, 'bf16', 'c', [64, 0], False, 'D z dt_bias h0'),
    (200, 1, 16, 40, 1, 'f32', 'c', [199], False, 'z dt_bias'),
]


def run_scan(case, softplus=True, seed=0):
    from asr_amd import ops
    T, B, D, N, G, ty, lay, lens, rev, keep = case
    g = gen(T * 7 + D + seed)
    a, opt = scan_inputs(g, T, B, D, N, G, TY[ty], lay)
    if not softplus:                                   # delta = dt + bias: keep it positive
        a['dt'] = a['dt'].abs() * 0.2
        opt['dt_bias'] = opt['dt_bias'].abs() * 0.01
    opt = {k: (v if k in keep.split() else None) for k, v in opt.items()}
    ln = torch.tensor(lens, dtype=torch.int32).cuda() if lens else None
    do, dh = rn(g, T, B, D, dtype=TY[ty]), rn(g, B, D, N)
    for k in ('x', 'dt', 'Bm', 'Cm'):
        a[k] = spoil(a[k], ln)
    if opt['z'] is not None:
        opt['z'] = spoil(opt['z'], ln)
    do = spoil(do, ln)
    kw = dict(lens=ln, reverse=rev, softplus=softplus, **opt)
    out, h, saved = ops.selective_scan_fwd(*a.values(), train=True, **kw)
    gr = ops.selective_scan_bwd(do, *a.values(), saved, dh_last=dh, **kw)
    torch.cuda.synchronize()
    ra = {k: (R.leaf(v) if k == 'A' else clean(v, ln).requires_grad_()) for k, v in a.items()}
    rop = {k: None if v is None else (clean(v, ln).requires_grad_() if k == 'z' else R.leaf(v)) for k, v in opt.items()}
    ro, rh = R.scan(*ra.values(), lens=lens, reverse=rev, softplus=softplus, **rop)
    return a, opt, kw, (out, h, gr), (ra, rop, ro, rh), (do, dh, ln)


@pytest.mark.parametrize('softplus', [True, False])
@pytest.mark.parametrize('case', SCAN, ids=lambda c: '-'.join(str(v) for v in c).replace(' ', ''))
def test_scan(case, softplus):
    T, B, D, N, G, ty, lay, lens, rev, keep = case
    a, opt, kw, (out, h, gr), (ra, rop, ro, rh), (do, dh, ln) = run_scan(case, softplus)
    steps = 8 * T + 2 * N + 32
    R.close(out, ro, steps, 'out')
    R.close(h, rh, steps, 'h')
    ((ro * clean(do, ln)).sum() + (rh * R.leaf(dh, False)).sum()).backward()
    names = dict(x=ra['x'], dt=ra['dt'], A=ra['A'], B=ra['Bm'], C=ra['Cm'], D=rop['D'], z=rop['z'], dt_bias=rop['dt_bias'],
                 h0=rop['h0'])
    for k, v in names.items():
        if v is None:
            assert gr[k] is None, k
            continue
        ref = v.grad if v.grad is not None else torch.zeros_like(v)
        R.close(gr[k], ref, 4 * steps + (B * T if k in ('A', 'D', 'dt_bias') else D if k in ('B', 'C') else 0), 'd' + k)


@pytest.mark.parametrize('case', [SCAN[4], SCAN[13], SCAN[14]], ids=['short', 'chunks', 'chunks-reverse'])
def test_scan_gradient_against_differences(case):
    """Along a random direction of every input, (L(+e) - L(-e)) / 2e of the kernel's own forward pass against <gradient,
    direction>, L = <out, dout> + <h, dh> in float64.  Rounding of out and h gives at most (8 T + 2 N + 32) 2^-24 of the sum of
    |out dout| / e, the third derivative e^2 of the second's size: e = 2^-6 leaves both below 2e-2 of the root of the sum
    of squares used as the scale."""
    from asr_amd import ops
    a, opt, kw, (out, h, gr), _, (do, dh, ln) = run_scan(case)
    T, B, D, N, G = case[:5]
    a = {k: (torch.nan_to_num(v, 0, 0, 0) if k != 'A' else v) for k, v in a.items()}
    opt = {k: None if v is None else torch.nan_to_num(v, 0, 0, 0) for k, v in opt.items()}
    do = torch.nan_to_num(do, 0, 0, 0)
    base = dict(lens=ln, reverse=case[8])

    def loss(a, opt):
        o, hh, _ = ops.selective_scan_fwd(*a.values(), **base, **opt)
        return float((o.double() * do.double()).sum() + (hh.double() * dh.double()).sum())
    e = 2.0 ** -6
    g = gen(5)
    for k, gk in [('x', 'x'), ('dt', 'dt'), ('A', 'A'), ('Bm', 'B'), ('Cm', 'C'), ('D', 'D'), ('z', 'z'),
                  ('dt_bias', 'dt_bias'), ('h0', 'h0')]:
        src = a if k in a else opt
        if src[k] is None:
            continue
        v = torch.randn(src[k].shape, generator=g).cuda()
        if k == 'A':
            v = v * 0.2
        up, dn = dict(src), dict(src)
        up[k], dn[k] = src[k] + e * v, src[k] - e * v
        lu = loss(up, opt) if src is a else loss(a, up)
        ld = loss(dn, opt) if src is a else loss(a, dn)
        want = float((gr[k if k not in ('Bm', 'Cm') else gk].double() * v.double()).sum())
        scale = float(gr[gk].double().norm()) + 1e-3
        assert abs((lu - ld) / (2 * e) - want) < 2e-2 * scale, (k, (lu - ld) / (2 * e), want, scale)


@pytest.mark.parametrize('ty', ['f32', 'bf16', 'f16'])
@pytest.mark.parametrize('D,N,G', [(64, 16, 1), (70, 16, 2), (30, 5, 3), (8, 1, 1), (40, 64, 1), (9, 20, 1)])
def test_scan_steps_are_the_sequence(ty, D, N, G):
    """frame after frame through the state against the sequence at once (which may join the sum over states in another
    order), a sequence in two calls, and the float64 form"""
    from asr_amd import ops
    ty = TY[ty]
    T, B = 13, 3
    a, opt = scan_inputs(gen(D + N), T, B, D, N, G, ty)
    out, h, none = ops.selective_scan_fwd(*a.values(), **opt)
    assert none is None
    ro, rh = R.scan(*[R.leaf(v, False) for v in a.values()], **{k: R.leaf(v, False) for k, v in opt.items()})
    st = opt['h0'].clone()
    seq = {k: v for k, v in a.items() if k != 'A'}
    steps = [ops.selective_scan_step(st, seq['x'][t], seq['dt'][t], a['A'], seq['Bm'][t], seq['Cm'][t], D=opt['D'],
                                     z=opt['z'][t], dt_bias=opt['dt_bias']) for t in range(T)]
    k = 8 * T + 2 * N + 32
    R.close(torch.stack(steps), ro, k, 'steps')
    R.close(st, rh, k, 'h after steps')
    R.close(out, ro, k, 'out')
    half = {n: (v[:6], v[6:]) if n != 'A' else (v, v) for n, v in a.items()}
    o1, h1, _ = ops.selective_scan_fwd(*[v[0] for v in half.values()], D=opt['D'], z=opt['z'][:6], dt_bias=opt['dt_bias'], h0=opt['h0'])
    o2, h2, _ = ops.selective_scan_fwd(*[v[1] for v in half.values()], D=opt['D'], z=opt['z'][6:], dt_bias=opt['dt_bias'], h0=h1)
    R.close(torch.cat([o1, o2]), ro, k, 'two calls')
    R.close(h2, rh, k, 'h after two calls')


def test_scan_extreme_steps():
    """softplus far in both tails: a state that is forgotten at once (delta = 60 and beyond) and one that never moves"""
    from asr_amd import ops
    T, B, D, N = 20, 2, 64, 16
    a, opt = scan_inputs(gen(3), T, B, D, N, 1, torch.float32)
    a['dt'][:10] = 60.0
    a['dt'][10:, :, 32:] = -200.0
    opt['dt_bias'] = None
    out, h, _ = ops.selective_scan_fwd(*a.values(), **opt)
    ro, rh = R.scan(*[R.leaf(v, False) for v in a.values()], **{k: R.leaf(v, False) for k, v in opt.items()})
    # the exponent's argument reaches 60 * 24 * log2(e) and is rounded twice, but then the exponential is zero; above
    # exp(-100) its relative error is below 100 * 2 * 2^-24, of a state that is itself below 1e-40 of the rest
    R.close(out, ro, 8 * T + 2 * N + 32, 'out')
    R.close(h, rh, 8 * T + 2 * N + 32, 'h')


def test_scan_growing_states_over_chunks():
    """Rates above zero over a time that is walked in chunks: a state that is still zero stays zero (a chunk's whole growth,
    e^128 at 64 frames of delta = 2, is infinite in float32), and what enters near the end grows by e^2 a frame.  The roundings
    of 20 growing frames are relative to what has grown: 8 a frame, as for a state that decays."""
    from asr_amd import ops
    T, B, D, N = 2048, 1, 64, 4
    g = gen(11)
    x = torch.zeros(T, B, D).cuda()
    x[-20:] = rn(g, 20, B, D)
    dt = torch.full((T, B, D), 2.0).cuda()
    A = torch.tensor([1.0, 0.5, -0.5, -1.0]).repeat(D, 1).cuda()
    Bm, Cm = rn(g, T, B, 1, N), rn(g, T, B, 1, N)
    a = (x, dt, A, Bm, Cm)
    out, h, saved = ops.selective_scan_fwd(*a, softplus=False, train=True)
    ro, rh = R.scan(*[R.leaf(v, False) for v in a], softplus=False)
    R.close(out, ro, 8 * 20 + 2 * N + 32, 'out')
    R.close(h, rh, 8 * 20 + 2 * N + 32, 'h')
    # the adjoint of the first 20 frames, with nothing behind them: dx = delta sum_n B dh
    x.zero_()
    out, h, saved = ops.selective_scan_fwd(*a, softplus=False, train=True)
    assert not out.any() and not h.any()
    do = torch.zeros(T, B, D).cuda()
    do[:20] = rn(g, 20, B, D)
    gr = ops.selective_scan_bwd(do, *a, saved, softplus=False)
    lx = R.leaf(x)
    ro, _ = R.scan(lx, *[R.leaf(v, False) for v in a[1:]], softplus=False)
    ref, = torch.autograd.grad((ro * R.leaf(do, False)).sum(), lx)
    R.close(gr['x'], ref, 4 * (8 * 20 + 2 * N + 32), 'dx')
    for k in ('dt', 'A', 'C'):
        assert not gr[k].any(), k                      # the state is zero all along


def test_scan_infinite_decay():
    """a rate of -inf (and one whose product with log2(e) overflows) forgets everything behind its own frame, exactly, in ragged
    rows too; its state's share of dA is zero"""
    from asr_amd import ops
    T, B, D, N = 150, 3, 64, 8
    lens = torch.tensor([150, 37, 0], dtype=torch.int32).cuda()
    a, opt = scan_inputs(gen(21), T, B, D, N, 1, torch.float32)
    a['A'][:, 0], a['A'][:, 1] = float('-inf'), -3e38
    opt['h0'] = None
    out, h, saved = ops.selective_scan_fwd(*a.values(), lens=lens, train=True, **opt)
    ro, rh = R.scan(*[R.leaf(v, False) for v in a.values()], lens=lens.cpu(), **{k: R.leaf(v, False) for k, v in opt.items()})
    R.close(out, ro, 8 * T + 2 * N + 32, 'out')
    R.close(h, rh, 8 * T + 2 * N + 32, 'h')
    gr = ops.selective_scan_bwd(rn(gen(2), T, B, D), *a.values(), saved, lens=lens, **opt)
    assert all(v is None or torch.isfinite(v).all() for v in gr.values()) and not gr['A'][:, :2].any()


def test_scan_shared_projections_by_expand():
    """B and C handed in with stride 0 over the rows: values shared, gradients per row"""
    from asr_amd import ops
    T, B, D, N = 30, 3, 64, 16
    a, opt = scan_inputs(gen(9), T, B, D, N, 1, torch.float32)
    one_b, one_c = a['Bm'][:, :1].contiguous(), a['Cm'][:, :1].contiguous()
    wide = dict(a, Bm=one_b.expand(T, B, 1, N), Cm=one_c.expand(T, B, 1, N))
    full = dict(a, Bm=one_b.repeat(1, B, 1, 1), Cm=one_c.repeat(1, B, 1, 1))
    do = rn(gen(1), T, B, D)
    res = []
    for q in (wide, full):
        out, h, saved = ops.selective_scan_fwd(*q.values(), train=True, **opt)
        res.append([out, h] + [v for v in ops.selective_scan_bwd(do, *q.values(), saved, **opt).values()])
    for u, v in zip(*res):
        assert torch.equal(u, v)


# ---------------------------------------------------------------------------------------------- norm
@pytest.mark.parametrize('ty', ['f32', 'bf16', 'f16'])
@pytest.mark.parametrize('rows,n,res,lay', [(1, 1, False, 'c'), (3, 64, True, 'c'), (5, 100, True, 'c'), (7, 512, True, 'half'),
                                            (9, 1000, True, 'odd'), (2, 1024, True, 'c'), (3, 1032, True, 'c'), (2, 2047, True, 'c'),
                                            (4, 4096, False, 'c'), (3, 8192, True, 'c'), (2, 5001, True, 'c'),
                                            (2, 9000, True, 'c'), (2500, 40, True, 'c'), (2100, 1040, True, 'c'), (0, 16, True, 'c'),
                                            (6, 7, True, 'odd'), (6, 9, True, 'half'), (2100, 333, True, 'odd'), (1100, 1025, True, 'odd'),
                                            (5, 8191, True, 'odd'), (5, 8193, True, 'odd'), (3, 20003, True, 'c')])
def test_rms_norm(ty, rows, n, res, lay):
    from asr_amd import ops
    ty = TY[ty]
    g = gen(rows + n)
    x = strided(g, 1, rows, n, ty, lay)[0]
    r = rn(g, rows, n, dtype=ty, scale=2.0) if res else None
    w, dy, dres = 1 + rn(g, n, scale=0.2), rn(g, rows, n, dtype=ty), rn(g, rows, n, dtype=ty)
    y, s, rstd = ops.add_rms_norm_fwd(x, w, residual=r, eps=1e-5)
    steps = n // 64 + 16
    rx, rw = R.leaf(x), R.leaf(w)
    ry, rs = R.rms(rx, rw, R.leaf(r, False), 1e-5)
    R.close(y, ry, steps, 'y')
    R.close(s, rs, 2, 'r')
    R.close(rstd, 1 / torch.sqrt((rs * rs).mean(-1) + 1e-5), steps, 'rstd')
    for d in (None, dres):
        dx, dw = ops.add_rms_norm_bwd(dy, x, w, rstd, residual=r, dres=d)
        gx, gw = torch.autograd.grad(ry, (rx, rw), R.leaf(dy, False), retain_graph=True)
        if d is not None:
            gx = gx + R.leaf(d, False)
        # dx = (g - xhat m) rstd: the roundings act on g and xhat m, both up to max|g| (|xhat m| <= |xhat| rms(g) rms(xhat)),
        # before they cancel (one column: xhat^2 is 1 - eps / r^2 and next to nothing is left)
        size = float((R.leaf(dy, False) * R.leaf(w, False)).abs().max() * R.leaf(rstd, False).max()) if rows else None
        size = max(size, float(gx.abs().max())) if rows else None
        R.close(dx, gx, 4 * steps, 'dx', size)
        R.close(dw, gw, 4 * steps + rows, 'dw')


def test_rms_norm_of_zeros_and_huge_rows():
    from asr_amd import ops
    x = torch.zeros(3, 64, device='cuda')
    x[1] = 1e15
    y, s, rstd = ops.add_rms_norm_fwd(x, torch.ones(64, device='cuda'), residual=torch.zeros_like(x), eps=1e-6)
    assert (y[0] == 0).all() and (y[2] == 0).all() and torch.allclose(y[1], torch.ones(64, device='cuda'), atol=1e-6)
    dx, dw = ops.add_rms_norm_bwd(torch.ones_like(x), x, torch.ones(64, device='cuda'), rstd, residual=torch.zeros_like(x))
    assert torch.isfinite(dx).all() and torch.isfinite(dw).all()


# ---------------------------------------------------------------------------------------------- clip
def make_list(g, sizes):
    kinds = [torch.float32, torch.bfloat16, torch.float16]
    return [rn(g, *(s if isinstance(s, tuple) else (s,)), dtype=kinds[i % 3]) for i, s in enumerate(sizes)]


@pytest.mark.parametrize('sizes', [[1], [0, 5], [8192], [8193, 7, 100000], [(33, 65), (3, 5, 7), 64, 0, 1],
                                   list(range(1, 131)), [70000] * 65], ids=lambda s: '%dx' % len(s))
@pytest.mark.parametrize('max_norm', [0.0, 0.5, 1e9])
def test_clip_list(sizes, max_norm):
    from asr_amd import updates
    ts = make_list(gen(len(sizes)), sizes)
    if len(ts) > 2:
        ts[2] = ts[2].reshape(-1)[1:]                               # not aligned to 16 bytes
        if ts[0].dim() == 2:
            ts[0] = ts[0].t()                                       # not contiguous
    keep = [t.clone() for t in ts]
    got, norm = updates.total_norm_constraint(ts, max_norm, 1e-7, return_norm=True)
    ref, rnorm = R.clip([R.leaf(t, False) for t in ts], max_norm, 1e-7)
    R.close(norm, rnorm.reshape(1), 2, 'norm')
    for i, (u, v) in enumerate(zip(got, ref)):
        R.close(u, v, 8, 'tensor %d' % i)
    for u, v in zip(keep, ts):
        assert torch.equal(u, v)                                    # the inputs stay
    again = updates.total_norm_constraint(tuple(ts), max_norm)
    assert all(torch.equal(u, v) for u, v in zip(again, got))


def test_clip_list_large_and_not_finite():
    from asr_amd import ops
    big = torch.full((3,), 1e30, device='cuda')
    out, norm = ops.clip_list([big], 1.0)
    assert abs(float(norm) / (3 ** 0.5 * 1e30) - 1) < 1e-6 and torch.allclose(out[0], torch.full_like(big, 3 ** -0.5))
    bad = [torch.tensor([1.0, float('nan')], device='cuda'), torch.ones(4, device='cuda')]
    out, norm = ops.clip_list(bad, 1.0)
    assert torch.isnan(norm).all() and all(torch.isnan(t).all() for t in out)
    inf = [torch.tensor([1.0, float('inf')], device='cuda')]
    out, norm = ops.clip_list(inf, 1.0)
    assert torch.isinf(norm).all() and float(out[0][0]) == 0.0 and torch.isnan(out[0][1])


def test_clip_in_place_through_the_c_entry():
    import ctypes as C
    from asr_amd import _lib
    L = _lib.lib()
    t = torch.arange(1, 20001, dtype=torch.float32, device='cuda')
    want, norm = R.clip([R.leaf(t, False)], 2.0, 1e-7)
    p = (C.c_void_p * 1)(t.data_ptr())
    n = (C.c_longlong * 1)(t.numel())
    nt = torch.empty(1, device='cuda')
    ws = torch.empty(L.asr_clip_list_ws_bytes(1, n), dtype=torch.uint8, device='cuda')
    assert L.asr_clip_list(1, (C.c_int * 1)(0), p, p, n, 2.0, 1e-7, nt.data_ptr(), ws.data_ptr(), ws.numel(),
                           torch.cuda.current_stream().cuda_stream) == 0
    R.close(t, want[0], 8, 't')
    R.close(nt, norm.reshape(1), 2, 'norm')
