"""Measured cases of the operators of a selective state-space layer and of its training.

Four operators:
  conv  the short causal depthwise convolution over time with SiLU
  scan  the selective state-space scan
  norm  the root-mean-square norm with the residual's addition
  clip  the global norm over a list of gradients and their scaling

`run` computes them from elementary torch operations in float32 (rounded once at the end), or, where `own` is true, with
asr_amd's calls.  Sequences are time-major (T, B, channels).  Frames at and behind lens[b] are padding: outputs and
gradients there are zero, the state stays what the last valid frame left.
"""
import math

import torch
import torch.nn.functional as F

own = False

TYPES = {'f32': torch.float32, 'bf16': torch.bfloat16, 'f16': torch.float16}

# ---------------------------------------------------------------------------------------------- cases
# Widths 512 / 1024 are the stacks of this repository (4x512, both directions: 1024), T = 1207 / 2262 its batches of one /
# two concatenated utterances, 16 its batch rows; an inner width of twice the model width, 16 states and 4 taps are the
# usual form of the layer.
LISTED = [
    # one training step's convolution over a ragged batch of two-utterance rows at the stack's width
    dict(name='conv_train_f32', op='conv', mode='train', T=2262, B=16, D=1024, K=4, type='f32', ragged=True, reverse=False),
    # the same for a wide layer in bf16
    dict(name='conv_train_bf16_wide', op='conv', mode='train', T=4096, B=16, D=2048, K=4, type='bf16', ragged=False,
         reverse=False),
    # one frame of sixteen streams
    dict(name='conv_step_f32', op='conv', mode='step', T=1, B=16, D=1024, K=4, type='f32', ragged=False, reverse=False),
    # one frame of sixteen streams
    dict(name='scan_step_f32', op='scan', mode='step', T=1, B=16, D=1024, N=16, G=1, type='f32', ragged=False, reverse=False),
    # one token of many streams: the state's traffic counts
    dict(name='scan_step_bf16_wide', op='scan', mode='step', T=1, B=256, D=4096, N=16, G=1, type='bf16', ragged=False,
         reverse=False),
    # a short odd window of the backward-running direction, few channels, shared projections in two groups
    dict(name='scan_train_odd', op='scan', mode='train', T=37, B=3, D=200, N=8, G=2, type='f32', ragged=True, reverse=True),
    # one training step's scan over a ragged batch at the stack's width
    dict(name='scan_train_f32', op='scan', mode='train', T=1207, B=16, D=1024, N=16, G=1, type='f32', ragged=True,
         reverse=False),
    # the same for a wide layer in bf16
    dict(name='scan_train_bf16_wide', op='scan', mode='train', T=2048, B=16, D=2048, N=16, G=1, type='bf16', ragged=False,
         reverse=False),
    # one long recording read at once, state kept for what follows
    dict(name='scan_prompt_bf16', op='scan', mode='prompt', T=16384, B=1, D=2048, N=16, G=1, type='bf16', ragged=False,
         reverse=False),
    # the norm in front of one frame of sixteen streams
    dict(name='norm_step_f32', op='norm', mode='infer', rows=16, n=512, type='f32'),
    # the norm of a training step over all frames of a batch, forward and backward
    dict(name='norm_train_bf16', op='norm', mode='train', rows=2262 * 16, n=1024, type='bf16'),
    # the gradients of a stack of such layers, matrices and small vectors, clipped before the optimiser's step
    dict(name='clip_stack', op='clip', count=56, big=4 << 20, type='mixed'),
]


def listed():
    return [dict(c) for c in LISTED]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(['conv', 'conv', 'scan', 'scan', 'scan', 'norm', 'clip'])
    type_ = rng.choice(['f32', 'bf16', 'f16'])
    if op == 'norm':
        n = _log(rng, 64, 8192)
        rows = _log(rng, 1, max(1, min(40000, (2262 * 16 * 1024) // n)))
        return dict(op=op, mode=rng.choice(['infer', 'train']), rows=rows, n=n, type=type_)
    if op == 'clip':
        return dict(op=op, count=rng.randint(1, 56), big=_log(rng, 1 << 10, 4 << 20),
                    type=rng.choice(['f32', 'bf16', 'mixed']))
    D = _log(rng, 48, 2048)
    c = dict(op=op, mode='', T=0, B=0, D=D, type=type_, ragged=rng.random() < 0.5, reverse=rng.random() < 0.3)
    if op == 'conv':
        c['K'] = rng.randint(2, 8)
        c['mode'] = rng.choice(['train', 'train', 'step'])
        if c['mode'] == 'step':
            c.update(T=1, B=_log(rng, 1, 256), ragged=False, reverse=False)
        else:
            c['B'] = _log(rng, 1, 16)
            c['T'] = _log(rng, 2, 4096)
        return c
    c['N'] = rng.choice([4, 8, 16, 16, 16, 24, 32, 64])
    c['G'] = rng.choice([1, 1, 2, 4])
    c['D'] = max(c['G'], D // c['G'] * c['G'])
    c['mode'] = rng.choice(['train', 'train', 'prompt', 'step'])
    if c['mode'] == 'step':
        c.update(T=1, B=_log(rng, 1, 256), ragged=False, reverse=False)
    else:
        c['B'] = _log(rng, 1, 16)
        most = (2048 * 16 * 2048 * 16) // (c['B'] * c['D'] * max(16, c['N']))
        c['T'] = min(most, _log(rng, 2, 2048 if c['mode'] == 'train' else 16384))
    return c


# ---------------------------------------------------------------------------------------------- inputs
def _clip_sizes(case):
    """Sizes like a stack's: a few matrices, as many vectors, some of them odd."""
    big = case['big']
    kinds = [big, 512, big // 2 + 1, 1024, big // 16, 64, big // 4, 33, 1024 * 16, 7]
    return [max(1, kinds[i % len(kinds)]) for i in range(case['count'])]


def prepare(case, seed):
    g = torch.Generator(device='cuda').manual_seed(seed)

    def rn(*shape, dtype=torch.float32, scale=1.0):
        return (torch.randn(*shape, generator=g, device='cuda') * scale).to(dtype)

    def ru(*shape):
        return torch.rand(*shape, generator=g, device='cuda')

    s = dict(case)
    if case['op'] == 'clip':
        both = [torch.float32, torch.bfloat16]
        s['grads'] = []
        for i, n in enumerate(_clip_sizes(case)):
            dt = both[(i // 3) % 2] if case['type'] == 'mixed' else TYPES[case['type']]
            s['grads'].append(rn(n, dtype=dt, scale=0.02))
        s['max_norm'] = 1.0
        return s
    ty = TYPES[case['type']]
    if case['op'] == 'norm':
        r, n = case['rows'], case['n']
        s['x'], s['res'] = rn(r, n, dtype=ty), rn(r, n, dtype=ty, scale=2.0)
        s['w'] = 1.0 + rn(n, scale=0.1)
        if case['mode'] == 'train':
            s['dy'], s['dres'] = rn(r, n, dtype=ty), rn(r, n, dtype=ty, scale=0.5)
        return s
    T, B, D = case['T'], case['B'], case['D']
    s['lens'] = None
    if case['ragged']:                    # one row of full length, the others down to a quarter of it
        le = (T * (0.25 + 0.75 * ru(B))).ceil().clamp(1, T).to(torch.int32)
        le[0] = T
        s['lens'] = le
    if case['op'] == 'conv':
        K = case['K']
        s['w'], s['bias'] = rn(D, K, scale=K ** -0.5), rn(D, scale=0.1)
        if case['mode'] == 'step':
            s['x'], s['state'] = rn(B, D, dtype=ty), rn(K - 1, B, D, dtype=ty)
        else:                             # x is the left half of the input projection's output, as the layer has it
            s['x'] = rn(T, B, 2 * D, dtype=ty)[:, :, :D]
            s['dout'] = rn(T, B, D, dtype=ty)
        return s
    N, G = case['N'], case['G']
    # the usual start of such a layer: decay rates 1..N, step sizes between 1e-3 and 1e-1
    s['A'] = -(torch.arange(1, N + 1, device='cuda', dtype=torch.float32).repeat(D, 1) * (0.5 + ru(D, N)))
    step = torch.exp(ru(D) * (math.log(0.1) - math.log(1e-3)) + math.log(1e-3))
    s['dt_bias'] = step + torch.log(-torch.expm1(-step))
    s['Dskip'] = 1.0 + rn(D, scale=0.1)
    if case['mode'] == 'step':
        s['x'], s['dt'], s['z'] = rn(B, D, dtype=ty), rn(B, D, dtype=ty, scale=0.5), rn(B, D, dtype=ty)
        s['Bm'], s['Cm'] = rn(B, G, N, dtype=ty), rn(B, G, N, dtype=ty)
        s['h'] = rn(B, D, N)
        return s
    s['x'], s['dt'] = rn(T, B, D, dtype=ty), rn(T, B, D, dtype=ty, scale=0.5)
    s['z'] = rn(T, B, 2 * D, dtype=ty)[:, :, D:]      # the right half of the input projection's output
    s['Bm'], s['Cm'] = rn(T, B, G, N, dtype=ty), rn(T, B, G, N, dtype=ty)
    s['h0'] = rn(B, D, N) if case['mode'] == 'prompt' else None
    if case['mode'] == 'train':
        s['dout'] = rn(T, B, D, dtype=ty)
    return s


# ---------------------------------------------------------------------------------------------- plain forms
def _valid(s, T, B):
    """(T, B, 1) truth values: frames in front of lens[b]."""
    t = torch.arange(T, device='cuda')[:, None]
    n = torch.full((B,), T, device='cuda') if s['lens'] is None else s['lens']
    return (t < n[None, :])[:, :, None]


def _in_order(v, s):
    return v.flip(0) if s['reverse'] else v


def _silu(v):
    return v / (1 + torch.exp(-v))


def _dsilu(v):
    e = 1 / (1 + torch.exp(-v))
    return e * (1 + v * (1 - e))


def _softplus(v):
    return torch.where(v > 20, v, torch.log1p(torch.exp(v.clamp(max=20))))


def _plain_conv(s):
    x, w, b, ty = s['x'], s['w'], s['bias'], s['x'].dtype
    K = s['K']
    if s['mode'] == 'step':
        win = torch.cat([s['state'].float(), x.float()[None]])                 # (K, B, D)
        out = _silu((win * w.t()[:, None, :]).sum(0) + b)
        state = s['state']
        state.copy_(win[1:])                                                   # the streams' own buffer moves on
        return [out.to(ty), state]
    T, B, D = x.shape
    ok = _in_order(_valid(s, T, B), s)
    xs = torch.where(ok, _in_order(x.float(), s), 0.0)
    win = F.pad(xs, (0, 0, 0, 0, K - 1, 0)).unfold(0, K, 1)                     # (T, B, D, K)
    pre = (win * w).sum(-1) + b
    out = torch.where(ok, _silu(pre), 0.0)
    dpre = torch.where(ok, _in_order(s['dout'].float(), s) * _dsilu(pre), 0.0)
    dwin = F.pad(dpre, (0, 0, 0, 0, 0, K - 1)).unfold(0, K, 1)
    dx = torch.where(ok, (dwin * w.flip(1)).sum(-1), 0.0)
    dw = (win * dpre[..., None]).sum((0, 1))
    return [_in_order(out, s).to(ty), _in_order(dx, s).to(ty), dw, dpre.sum((0, 1))]


def _recur(a, b):
    """h[t] = a[t] h[t-1] + b[t] over the first axis, h[-1] = 0: spans of doubling length are joined."""
    T, span = a.shape[0], 1
    while span < T:
        b = torch.cat([b[:span], torch.addcmul(b[span:], a[span:], b[:-span])])
        if 2 * span < T:
            a = torch.cat([a[:span], a[span:] * a[:-span]])
        span *= 2
    return b


def _plain_scan(s):
    ty, A, Dk = s['x'].dtype, s['A'], s['Dskip']
    rep = s['D'] // s['G']
    if s['mode'] == 'step':
        x, z = s['x'].float(), s['z'].float()
        d = _softplus(s['dt'].float() + s['dt_bias'])
        Bm = s['Bm'].float().repeat_interleave(rep, 1)
        Cm = s['Cm'].float().repeat_interleave(rep, 1)
        h = s['h']
        h.mul_(torch.exp(d[..., None] * A)).add_((d * x)[..., None] * Bm)      # the streams' own buffer moves on
        y = (h * Cm).sum(-1) + Dk * x
        return [(y * _silu(z)).to(ty), h]
    T, B, D = s['x'].shape
    ok = _in_order(_valid(s, T, B), s)
    x = torch.where(ok, _in_order(s['x'].float(), s), 0.0)
    z = torch.where(ok, _in_order(s['z'].float(), s), 0.0)
    raw = _in_order(s['dt'].float(), s) + s['dt_bias']
    d = torch.where(ok, _softplus(raw), 0.0)
    Bm = torch.where(ok[..., None], _in_order(s['Bm'].float(), s), 0.0).repeat_interleave(rep, 2)
    Cm = torch.where(ok[..., None], _in_order(s['Cm'].float(), s), 0.0).repeat_interleave(rep, 2)
    a = torch.exp(d[..., None] * A)                                             # (T, B, D, N)
    u = (d * x)[..., None] * Bm
    if s['h0'] is not None:
        u[0] += a[0] * s['h0']
    h = _recur(a, u)
    del u
    y = (h * Cm).sum(-1) + Dk * x
    gate = _silu(z)
    out = [_in_order(torch.where(ok, y * gate, 0.0), s).to(ty), h[-1].clone()]
    if s['mode'] != 'train':
        return out
    do = torch.where(ok, _in_order(s['dout'].float(), s), 0.0)
    dz, dy = do * y * _dsilu(z), do * gate
    later = torch.cat([a[1:], torch.zeros_like(a[:1])]).flip(0)                 # dh[t] = C dy + a[t+1] dh[t+1]
    dh = _recur(later, (dy[..., None] * Cm).flip(0)).flip(0)
    del later, Cm
    dC = (dy[..., None] * h).unflatten(2, (s['G'], rep)).sum(3)
    before = torch.cat([torch.zeros_like(h[:1]), h[:-1]])
    del h
    q = dh * a * before                                                        # d(delta A)
    del a, before
    dA = (q * d[..., None]).sum((0, 1))
    dd = (q * A).sum(-1)
    del q
    su = (dh * Bm).sum(-1)
    del Bm
    dB = (dh * (d * x)[..., None]).unflatten(2, (s['G'], rep)).sum(3)
    dd = dd + su * x
    dx = su * d + Dk * dy
    ddt = torch.where(ok, dd / (1 + torch.exp(-raw)), 0.0)
    back = lambda v: _in_order(v, s).to(ty)  # noqa: E731
    return out + [back(dx), back(ddt), dA, back(dB), back(dC), (dy * x).sum((0, 1)), back(dz), ddt.sum((0, 1))]


EPS = 1e-6


def _plain_norm(s):
    ty, w = s['x'].dtype, s['w']
    r = s['x'].float() + s['res'].float()
    rstd = torch.rsqrt(r.square().mean(-1, keepdim=True) + EPS)
    xhat = r * rstd
    out = [(xhat * w).to(ty), r.to(ty)]
    if s['mode'] != 'train':
        return out
    dy = s['dy'].float()
    gw = dy * w
    dx = (gw - xhat * (gw * xhat).mean(-1, keepdim=True)) * rstd + s['dres'].float()
    return out + [dx.to(ty), (dy * xhat).sum(0)]


def _plain_clip(s):
    sq = torch.stack([g.float().square().sum() for g in s['grads']])
    norm = sq.sum().sqrt()
    mult = norm.clamp(0.0, s['max_norm']) / (1e-7 + norm)
    return [(g.float() * mult).to(g.dtype) for g in s['grads']] + [norm.reshape(1)]


# ---------------------------------------------------------------------------------------------- the framework's calls
def _own_conv(s):
    from asr_amd import ops
    if s['mode'] == 'step':
        return [ops.causal_conv_step(s['x'], s['state'], s['w'], bias=s['bias']), s['state']]
    kw = dict(bias=s['bias'], lens=s['lens'], reverse=s['reverse'])
    out, _ = ops.causal_conv_fwd(s['x'], s['w'], **kw)
    g = ops.causal_conv_bwd(s['dout'], s['x'], s['w'], **kw)
    return [out, g['x'], g['w'], g['bias']]


def _own_scan(s):
    from asr_amd import ops
    args = (s['x'], s['dt'], s['A'], s['Bm'], s['Cm'])
    if s['mode'] == 'step':
        return [ops.selective_scan_step(s['h'], *args, D=s['Dskip'], z=s['z'], dt_bias=s['dt_bias']), s['h']]
    kw = dict(D=s['Dskip'], z=s['z'], dt_bias=s['dt_bias'], h0=s['h0'], lens=s['lens'], reverse=s['reverse'])
    if s['mode'] == 'prompt':
        out, h, _ = ops.selective_scan_fwd(*args, **kw)
        return [out, h]
    out, h, saved = ops.selective_scan_fwd(*args, train=True, **kw)
    g = ops.selective_scan_bwd(s['dout'], *args, saved, **kw)
    return [out, h] + [g[k] for k in ('x', 'dt', 'A', 'B', 'C', 'D', 'z', 'dt_bias')]


def _own_norm(s):
    from asr_amd import ops
    y, r, rstd = ops.add_rms_norm_fwd(s['x'], s['w'], residual=s['res'], eps=EPS)
    if s['mode'] != 'train':
        return [y, r]
    dx, dw = ops.add_rms_norm_bwd(s['dy'], s['x'], s['w'], rstd, residual=s['res'], dres=s['dres'])
    return [y, r, dx, dw]


def _own_clip(s):
    from asr_amd import updates
    scaled, norm = updates.total_norm_constraint(s['grads'], s['max_norm'], return_norm=True)
    return list(scaled) + [norm]


def run(state):
    if own:
        return {'conv': _own_conv, 'scan': _own_scan, 'norm': _own_norm, 'clip': _own_clip}[state['op']](state)
    return {'conv': _plain_conv, 'scan': _plain_scan, 'norm': _plain_norm, 'clip': _plain_clip}[state['op']](state)


# ---------------------------------------------------------------------------------------------- what a pass cannot do without
def work(case):
    e = 4 if case.get('type') in ('f32', 'mixed') else 2
    if case['op'] == 'clip':
        n = _clip_sizes(case)
        size = [(4 if case['type'] == 'f32' or (case['type'] == 'mixed' and (i // 3) % 2 == 0) else 2) * v
                for i, v in enumerate(n)]
        return dict(bytes=2 * sum(size), flops=3 * sum(n))
    if case['op'] == 'norm':
        m = case['rows'] * case['n']
        if case['mode'] == 'train':       # x, residual, dy, dres in; y, sum, dx out
            return dict(bytes=7 * m * e, flops=14 * m)
        return dict(bytes=4 * m * e, flops=5 * m)
    T, B, D = case['T'], case['B'], case['D']
    m = T * B * D
    if case['op'] == 'conv':
        K = case['K']
        if case['mode'] == 'step':        # x, state in; out, state out
            return dict(bytes=2 * (m + (K - 1) * B * D) * e, flops=(2 * K + 5) * m)
        return dict(bytes=4 * m * e, flops=(8 * K + 12) * m)      # x, dout in; out, dx out
    N, G = case['N'], case['G']
    bc, st = 2 * T * B * G * N * e, B * D * N * 4
    if case['mode'] == 'train':           # x, dt, z, B, C, dout in; out, dx, ddt, dz, dB, dC, state out
        return dict(bytes=8 * m * e + 2 * bc + st, flops=(23 * N + 40) * m)
    return dict(bytes=4 * m * e + bc + 2 * st, flops=(7 * N + 20) * m)


# ---------------------------------------------------------------------------------------------- 64-bit values
def _exact_conv(s):
    x, w, b = s['x'].double(), s['w'].double(), s['bias'].double()
    K = s['K']
    if s['mode'] == 'step':
        past = s['state'].double()
        pre = b + x * w[:, K - 1]
        for k in range(K - 1):
            pre = pre + past[k] * w[:, k]
        return [pre * torch.sigmoid(pre), torch.cat([past[1:], x[None]])]
    T, B, D = x.shape
    ok = _valid(s, T, B)
    x = torch.where(ok, x, torch.zeros_like(x)).requires_grad_()
    w.requires_grad_(), b.requires_grad_()
    pre = b.expand(T, B, D)
    for k in range(K):                    # tap K-1 meets the frame itself, tap k the frame K-1-k before it
        back = min(K - 1 - k, T)
        gone = torch.zeros(back, B, D, device='cuda', dtype=torch.float64)
        moved = torch.cat([x[back:], gone]) if s['reverse'] else torch.cat([gone, x[:T - back]])
        pre = pre + moved * w[:, k]
    out = torch.where(ok, pre * torch.sigmoid(pre), torch.zeros((), device='cuda', dtype=torch.float64))
    dx, dw, db = torch.autograd.grad(out, (x, w, b), s['dout'].double())
    return [out.detach(), torch.where(ok, dx, torch.zeros_like(dx)), dw, db]


def _exact_scan(s):
    f = torch.float64
    A, Dk, bias = s['A'].to(f), s['Dskip'].to(f), s['dt_bias'].to(f)
    G, D, N = s['G'], s['D'], s['N']
    x, dt, z, Bm, Cm = (s[k].to(f) for k in ('x', 'dt', 'z', 'Bm', 'Cm'))

    def frame(h, x, dt, z, Bm, Cm, A, Dk, bias):
        B = x.shape[0]
        step = F.softplus(dt + bias, threshold=40)
        hg = h * torch.exp(step[:, :, None] * A) + ((step * x).view(B, G, -1, 1) * Bm[:, :, None, :]).reshape(B, D, N)
        y = torch.einsum('bgdn,bgn->bgd', hg.view(B, G, -1, N), Cm).reshape(B, D) + Dk * x
        return hg, y * z * torch.sigmoid(z)

    if s['mode'] == 'step':
        h, y = frame(s['h'].to(f), x, dt, z, Bm, Cm, A, Dk, bias)
        return [y, h]
    T, B, _ = x.shape
    train = s['mode'] == 'train'
    if train and T * B * D * N > 1 << 30:
        return None
    ins = [x, dt, A, Bm, Cm, Dk, z, bias]
    if train:
        ins = [v.clone().requires_grad_() for v in ins]
    x, dt, A, Bm, Cm, Dk, z, bias = ins
    h = torch.zeros(B, D, N, device='cuda', dtype=f) if s['h0'] is None else s['h0'].to(f)
    rows = torch.full((B,), T, device='cuda') if s['lens'] is None else s['lens']
    xs, dts, zs, Bs, Cs = (v.unbind(0) for v in (x, dt, z, Bm, Cm))
    out = [None] * T
    zero = torch.zeros((), device='cuda', dtype=f)
    for t in (range(T - 1, -1, -1) if s['reverse'] else range(T)):
        new, y = frame(h, xs[t], dts[t], zs[t], Bs[t], Cs[t], A, Dk, bias)
        if s['lens'] is None:
            h, out[t] = new, y
        else:
            live = (rows > t)[:, None]
            h, out[t] = torch.where(live[..., None], new, h), torch.where(live, y, zero)
    out = torch.stack(out)
    if not train:
        return [out, h]
    g = torch.autograd.grad(out, ins, s['dout'].to(f))
    return [out.detach(), h.detach()] + list(g)


def _exact_norm(s):
    r = (s['x'].double() + s['res'].double()).requires_grad_()
    w = s['w'].double().requires_grad_()
    y = r / torch.sqrt(r.pow(2).sum(-1, keepdim=True) / s['n'] + EPS) * w
    if s['mode'] != 'train':
        return [y.detach(), r.detach()]
    dr, dw = torch.autograd.grad(y, (r, w), s['dy'].double())
    return [y.detach(), r.detach(), dr + s['dres'].double(), dw]


def _exact_clip(s):
    every = torch.cat([g.double() for g in s['grads']])
    norm = torch.linalg.vector_norm(every)
    mult = torch.minimum(norm, torch.full_like(norm, s['max_norm'])) / (norm + 1e-7)
    return [g.double() * mult for g in s['grads']] + [norm.reshape(1)]


def exact(case, seed):
    s = prepare(case, seed)
    return {'conv': _exact_conv, 'scan': _exact_scan, 'norm': _exact_norm, 'clip': _exact_clip}[case['op']](s)
