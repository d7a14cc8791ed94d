"""The state-space layer's operators as they are used: a residual block of them with the library's products, its loss, gradients,
clipping and an optimiser step; the same block streamed window by window and frame by frame; captured graphs, several streams,
views far apart in memory, empty calls."""
import pytest
import torch

import ref_ssm as R
from test_gpu_ssm import gen, rn, scan_inputs, clean, spoil

pytestmark = pytest.mark.gpu
F64 = torch.float64

# ---------------------------------------------------------------------------------------------- a block of the layer
T, B, W, D, N, RK, K, C = 37, 3, 48, 96, 16, 8, 4, 11          # frames, rows, model width, inner width, states, dt rank, taps, classes


def block_params(g):
    def m(i, o):
        return rn(g, i, o, scale=i ** -0.5)
    step = torch.exp(torch.rand(D, generator=g) * 4.6 - 6.9)
    return dict(norm=1 + rn(g, W, scale=0.1), w_in=m(W, 2 * D), conv_w=rn(g, D, K, scale=0.5), conv_b=rn(g, D, scale=0.1),
                w_x=m(D, RK + 2 * N), w_dt=m(RK, D), dt_bias=(step + torch.log(-torch.expm1(-step))).cuda(),
                A=-(torch.arange(1, N + 1).float().repeat(D, 1)).cuda(), Dk=1 + rn(g, D, scale=0.1), w_out=m(D, W),
                norm_f=1 + rn(g, W, scale=0.1), w_c=m(W, C), b_c=rn(g, C, scale=0.1))


def product(a, b):
    from asr_amd import ops
    out = torch.empty(a.shape[0], b.shape[1], device='cuda')
    ops.gemm(a, b, out)
    return out


def product_grads(a, b, dc):
    from asr_amd import ops
    da, db = torch.empty(a.shape, device='cuda'), torch.empty(b.shape, device='cuda')
    ops.gemm(dc, b, da, tb=True)
    ops.gemm(a, dc, db, ta=True)
    return da, db


def block_fwd(p, res, h, lens=None, conv_state=None, ssm_state=None, reverse=False, train=False):
    """res, h (T*B, W): the residual stream and what is to be added to it -> block output, new residual, states, saved"""
    from asr_amd import ops
    t = h.shape[0] // B
    y, r, rstd = ops.add_rms_norm_fwd(h, p['norm'], residual=res)
    xz = product(y, p['w_in']).view(t, B, 2 * D)
    x, z = xz[:, :, :D], xz[:, :, D:]
    u, cs = ops.causal_conv_fwd(x, p['conv_w'], bias=p['conv_b'], state=conv_state, lens=lens, reverse=reverse, want_state=True)
    dbc = product(u.view(t * B, D), p['w_x'])
    dt = product(dbc[:, :RK], p['w_dt']).view(t, B, D)
    bm = dbc.view(t, B, 1, RK + 2 * N)[..., RK:RK + N]
    cm = dbc.view(t, B, 1, RK + 2 * N)[..., RK + N:]
    args = (u, dt, p['A'], bm, cm)
    kw = dict(D=p['Dk'], z=z, dt_bias=p['dt_bias'], h0=ssm_state, lens=lens, reverse=reverse)
    o, hs, saved = ops.selective_scan_fwd(*args, train=train, **kw)
    out = product(o.view(t * B, D), p['w_out'])
    return out, r, cs, hs, dict(h=h, res=res, rstd=rstd, y=y, x=x, u=u, dbc=dbc, args=args, kw=kw, saved=saved, o=o,
                                conv=dict(bias=p['conv_b'], state=conv_state, lens=lens, reverse=reverse))


def block_bwd(p, s, dout, dres):
    from asr_amd import ops
    g = {}
    t = s['h'].shape[0] // B
    do, g['w_out'] = product_grads(s['o'].view(t * B, D), p['w_out'], dout)
    sg = ops.selective_scan_bwd(do.view(t, B, D), *s['args'], s['saved'], **s['kw'])
    g['A'], g['Dk'], g['dt_bias'] = sg['A'], sg['D'], sg['dt_bias']
    ddt_low, g['w_dt'] = product_grads(s['dbc'][:, :RK], p['w_dt'], sg['dt'].view(t * B, D))
    ddbc = torch.cat([ddt_low, sg['B'].view(t * B, N), sg['C'].view(t * B, N)], 1)
    du, g['w_x'] = product_grads(s['u'].view(t * B, D), p['w_x'], ddbc)
    cg = ops.causal_conv_bwd(sg['x'] + du.view(t, B, D), s['x'], p['conv_w'], **s['conv'])
    g['conv_w'], g['conv_b'] = cg['w'], cg['bias']
    dxz = torch.cat([cg['x'], sg['z']], 2).view(t * B, 2 * D)
    dy, g['w_in'] = product_grads(s['y'], p['w_in'], dxz)
    dh, g['norm'] = ops.add_rms_norm_bwd(dy, s['h'], p['norm'], s['rstd'], residual=s['res'], dres=dres)
    return dh, g


def ref_loss(p, x, res, y, mask, lens, reverse):
    """the same in float64, by autograd"""
    n, r = R.rms(x, p['norm'], res)
    xz = (n @ p['w_in']).view(T, B, 2 * D)
    u, _ = R.conv(xz[:, :, :D], p['conv_w'], p['conv_b'], None, lens, 'silu', reverse)
    dbc = u.reshape(T * B, D) @ p['w_x']
    dt = (dbc[:, :RK] @ p['w_dt']).view(T, B, D)
    o, _ = R.scan(u, dt, p['A'], dbc.view(T, B, 1, -1)[..., RK:RK + N], dbc.view(T, B, 1, -1)[..., RK + N:], p['Dk'],
                  xz[:, :, D:], p['dt_bias'], None, lens, True, reverse)
    out = o.reshape(T * B, D) @ p['w_out']
    f, _ = R.rms(out, p['norm_f'], r)
    logp = torch.log_softmax(f @ p['w_c'] + p['b_c'], 1)
    return -(logp[torch.arange(T * B), y.t().reshape(-1).long()] * mask.t().reshape(-1)).sum()


@pytest.mark.parametrize('reverse', [False, True])
def test_training_step_of_a_block(reverse):
    """Residual block, final norm, framewise cross-entropy, all gradients, clipping by their global norm, one step of descent.
    Tolerance: the chain has 5 products over at most 96 terms, the scan over 37 frames and two norms, forward and backward:
    below 2 * (8 T + 2 N + 32 + 5 * 96 + T B) < 2000 roundings of float32 (1.2e-4 of a tensor's largest value); the loss's
    sum of 111 terms stays within the same."""
    from asr_amd import ops, updates
    g = gen(4)
    p = block_params(g)
    x, res = rn(g, T * B, W), rn(g, T * B, W)
    lens_l = [37, 20, 1]
    lens = torch.tensor(lens_l, dtype=torch.int32).cuda()
    y = torch.randint(0, C, (B, T), generator=g, dtype=torch.int32).cuda()
    mask = (torch.arange(T)[None] < torch.tensor(lens_l)[:, None]).float().cuda()
    out, r, _, _, s = block_fwd(p, res, x, lens, reverse=reverse, train=True)
    f, r2, rstd2 = ops.add_rms_norm_fwd(out, p['norm_f'], residual=r)
    logits = torch.empty(T * B, C, device='cuda')
    ops.gemm(f, p['w_c'], logits, bias=p['b_c'])
    dlog, ce = torch.empty_like(logits), torch.empty(T * B, device='cuda')
    ops.softmax_ce(logits, C, B, T, target=y, tmask=mask, scale=1.0, dlogits=dlog, row_ce=ce)
    loss = ce.sum()
    df, g_wc = product_grads(f, p['w_c'], dlog)
    g_bc = torch.empty(C, device='cuda')
    ops.colreduce(dlog, g_bc, T * B, C)
    dsum, g_nf = ops.add_rms_norm_bwd(df, out, p['norm_f'], rstd2, residual=r)
    dx, grads = block_bwd(p, s, dsum, dsum)
    grads.update(w_c=g_wc, b_c=g_bc, norm_f=g_nf)

    rp = {k: R.leaf(v) for k, v in p.items()}
    rx = R.leaf(x)
    rl = ref_loss(rp, rx, R.leaf(res, False), y.cpu(), mask.cpu().double(), lens_l, reverse)
    rl.backward()
    assert abs(float(loss) - rl.item()) < 2000 * R.U * abs(rl.item())
    R.close(dx, rx.grad, 2000, 'dx')
    assert sorted(grads) == sorted(p)
    for k in p:
        R.close(grads[k], rp[k].grad, 2000, 'd' + k)

    names = sorted(grads)
    scaled, norm = updates.total_norm_constraint([grads[k] for k in names], 0.5, return_norm=True)
    rnorm = torch.sqrt(sum((v.grad ** 2).sum() for v in rp.values()))
    assert float(rnorm) > 0.5 and abs(float(norm) / float(rnorm) - 1) < 2000 * R.U
    assert abs(float(torch.sqrt(sum((v.double() ** 2).sum() for v in scaled))) - 0.5) < 1e-5
    # a small step against the clipped gradient lowers the loss by lr * 0.5 * norm, to first order
    lr = 1e-3
    for k, v in zip(names, scaled):
        rp[k].data -= lr * v.cpu().double()
    new = ref_loss(rp, rx, R.leaf(res, False), y.cpu(), mask.cpu().double(), lens_l, reverse)
    want = lr * 0.5 * float(rnorm)
    assert 0.9 * want < rl.item() - new.item() < 1.1 * want


def test_streaming_of_a_block():
    """window by window and frame by frame through the carried states = the utterance at once"""
    from asr_amd import ops
    g = gen(6)
    p = block_params(g)
    x, res = rn(g, T * B, W), rn(g, T * B, W)
    whole, r, cs, hs, _ = block_fwd(p, res, x)
    outs, c, h = [], None, None
    for a, b in ((0, 10), (10, 11), (11, 30), (30, T)):
        o, _, c, h, _ = block_fwd(p, res[a * B:b * B], x[a * B:b * B], conv_state=c, ssm_state=h)
        outs.append(o)
    steps = 8 * T + 2 * N + 32 + 3 * 96                       # the roundings of the scan and three products
    R.close(torch.cat(outs), R.leaf(whole, False), steps, 'windows')
    R.close(h, R.leaf(hs, False), steps, 'h')
    R.close(c, R.leaf(cs, False), steps, 'conv state')
    c, h = torch.zeros(K - 1, B, D, device='cuda'), torch.zeros(B, D, N, device='cuda')
    outs = []
    for t in range(T):
        y, _, _ = ops.add_rms_norm_fwd(x[t * B:(t + 1) * B], p['norm'], residual=res[t * B:(t + 1) * B])
        xz = product(y, p['w_in'])
        u = ops.causal_conv_step(xz[:, :D], c, p['conv_w'], bias=p['conv_b'])
        dbc = product(u, p['w_x'])
        dt = product(dbc[:, :RK], p['w_dt'])
        o = ops.selective_scan_step(h, u, dt, p['A'], dbc.view(B, 1, -1)[..., RK:RK + N], dbc.view(B, 1, -1)[..., RK + N:],
                                    D=p['Dk'], z=xz[:, D:], dt_bias=p['dt_bias'])
        outs.append(product(o, p['w_out']))
    R.close(torch.cat(outs), R.leaf(whole, False), steps, 'frames')
    R.close(h, R.leaf(hs, False), steps, 'h after frames')


# ---------------------------------------------------------------------------------------------- graphs, streams
def training_pass(s):
    from asr_amd import ops
    kw = dict(D=s['D'], z=s['z'], dt_bias=s['dt_bias'], h0=s['h0'], lens=s['lens'])
    u, cs = ops.causal_conv_fwd(s['x'], s['w'], lens=s['lens'], want_state=True)
    args = (u, s['dt'], s['A'], s['Bm'], s['Cm'])
    out, h, saved = ops.selective_scan_fwd(*args, train=True, **kw)
    sg = ops.selective_scan_bwd(s['do'], *args, saved, **kw)
    cg = ops.causal_conv_bwd(sg['x'], s['x'], s['w'], lens=s['lens'])
    t, b, d = s['x'].shape
    y, r, rstd = ops.add_rms_norm_fwd(out.view(t * b, d), s['nw'], residual=u.view(t * b, d))
    dx, dw = ops.add_rms_norm_bwd(s['do'].view(t * b, d), out.view(t * b, d), s['nw'], rstd, residual=u.view(t * b, d))
    clipped, norm = ops.clip_list([sg['A'], cg['w'], dw, sg['x']], 0.1)
    return [u, cs, out, h, *[v for v in sg.values() if v is not None], cg['x'], cg['w'], y, r, dx, dw, *clipped, norm]


def training_state(seed, t=150, b=2, d=80, n=16, ty=torch.float32):
    g = gen(seed)
    a, opt = scan_inputs(g, t, b, d, n, 1, ty)
    return dict(a, **opt, w=rn(g, d, 4), nw=1 + rn(g, d, scale=0.1), do=rn(g, t, b, d, dtype=ty),
                lens=torch.tensor([t, t // 3], dtype=torch.int32).cuda()[:b].contiguous())


def copy_in(dst, src):
    for k, v in src.items():
        if v is not None:
            dst[k].copy_(v)


@pytest.mark.parametrize('ty', [torch.float32, torch.bfloat16])
def test_captured_pass_replays_like_the_eager_one(ty):
    states = [training_state(s, ty=ty) for s in (1, 2, 3, 4)]
    eager = [[v.clone() for v in training_pass(s)] for s in states]
    inp = {k: v.clone() for k, v in states[0].items()}
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        training_pass(inp)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = training_pass(inp)
    for i in (1, 0, 2, 3, 3, 0):
        copy_in(inp, states[i])
        graph.replay()
        torch.cuda.synchronize()
        for k, (u, v) in enumerate(zip(out, eager[i])):
            assert torch.equal(u, v), (i, k)
        again = training_pass(states[i])                       # eager work between the replays
        for u, v in zip(again, eager[i]):
            assert torch.equal(u, v)
        torch.cuda.synchronize()


def test_two_captured_graphs_share_nothing():
    """both replayed at once on two streams, each into its own outputs"""
    states = [training_state(s, t=300, b=2, d=130) for s in (5, 6)]
    eager = [[v.clone() for v in training_pass(s)] for s in states]
    graphs, outs = [], []
    for s in states:
        gr = torch.cuda.CUDAGraph()
        with torch.cuda.graph(gr):
            outs.append(training_pass(s))
        graphs.append(gr)
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    for _ in range(5):
        for st, gr in zip(streams, graphs):
            st.wait_stream(torch.cuda.current_stream())
            with torch.cuda.stream(st):
                gr.replay()
        for st in streams:
            torch.cuda.current_stream().wait_stream(st)
        torch.cuda.synchronize()
        for o, e in zip(outs, eager):
            assert all(torch.equal(u, v) for u, v in zip(o, e))


def test_two_streams_at_once_and_repeated_calls_agree():
    states = [training_state(s, t=200, b=2, d=100) for s in (7, 8)]
    eager = [[v.clone() for v in training_pass(s)] for s in states]
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    got = [[], []]
    for _ in range(4):
        for i, st in enumerate(streams):
            st.wait_stream(torch.cuda.current_stream())
            with torch.cuda.stream(st):
                got[i].append(training_pass(states[i]))
    torch.cuda.synchronize()
    for i in range(2):
        for o in got[i]:
            assert all(torch.equal(u, v) for u, v in zip(o, eager[i]))


# ---------------------------------------------------------------------------------------------- extents
def test_lens_out_of_range_are_clamped():
    from asr_amd import ops
    a, opt = scan_inputs(gen(2), 20, 4, 64, 16, 1, torch.float32)
    w = rn(gen(3), 64, 4)
    odd = torch.tensor([-5, 0, 20, 99], dtype=torch.int32).cuda()
    fine = torch.tensor([0, 0, 20, 20], dtype=torch.int32).cuda()
    res = []
    for ln in (odd, fine):
        out, h, sv = ops.selective_scan_fwd(*a.values(), lens=ln, train=True, **opt)
        g = ops.selective_scan_bwd(a['x'], *a.values(), sv, lens=ln, **opt)
        c, cs = ops.causal_conv_fwd(a['x'], w, lens=ln, want_state=True)
        cg = ops.causal_conv_bwd(a['x'], a['x'], w, lens=ln)
        res.append([out, h, *g.values(), c, cs, cg['x'], cg['w']])
    assert all(torch.equal(u, v) for u, v in zip(*res))
    assert (res[0][0][:, :2] == 0).all() and torch.equal(res[0][1][:2], opt['h0'][:2])


@pytest.mark.parametrize('t,b', [(0, 2), (4, 0), (0, 0)])
def test_empty_calls(t, b):
    from asr_amd import ops
    a, opt = scan_inputs(gen(2), t, b, 24, 16, 1, torch.float32)
    dh = rn(gen(1), b, 24, 16)
    out, h, sv = ops.selective_scan_fwd(*a.values(), train=True, **opt)
    g = ops.selective_scan_bwd(torch.empty(t, b, 24, device='cuda'), *a.values(), sv, dh_last=dh, **opt)
    assert out.shape == (t, b, 24) and torch.equal(h, opt['h0']) and torch.equal(g['h0'], dh)
    for k in ('A', 'D', 'dt_bias'):
        assert (g[k] == 0).all()
    w = rn(gen(3), 24, 4)
    s0 = rn(gen(4), 3, b, 24)
    c, cs = ops.causal_conv_fwd(a['x'], w, state=s0, want_state=True)
    cg = ops.causal_conv_bwd(a['x'], a['x'], w, bias=opt['D'], state=s0, dstate_out=s0)
    assert c.shape == (t, b, 24) and (cg['w'] == 0).all() and (cg['bias'] == 0).all()
    if t == 0:
        assert torch.equal(cs, s0) and torch.equal(cg['state'], s0)
    if b == 0:
        z = torch.empty(0, 24, device='cuda')
        assert ops.causal_conv_step(z, s0, w).shape == (0, 24)
        e = torch.empty(0, 1, 16, device='cuda')
        assert ops.selective_scan_step(opt['h0'], z, z, a['A'], e, e).shape == (0, 24)


def test_one_frame_of_many_kinds_of_rows():
    """single frames: states and parameters off the 16-byte grid, strided inputs, every option left out once"""
    from asr_amd import ops
    for B_, D_, N_, G_ in ((5, 33, 16, 3), (2, 64, 4, 1), (300, 8, 12, 2), (1, 1, 64, 1)):
        g = gen(B_ + D_)
        a, opt = scan_inputs(g, 1, B_, D_, N_, G_, torch.float32)
        flat = torch.empty(B_ * D_ * N_ + 1, device='cuda')
        A = torch.empty(D_ * N_ + 1, device='cuda')[1:].view(D_, N_)
        A.copy_(a['A'])
        for leave in ('D', 'z', 'dt_bias', None):
            o = {k: v for k, v in opt.items() if k != leave and k != 'h0'}
            h = flat[1:].view(B_, D_, N_)
            h.copy_(opt['h0'])
            wide = rn(g, B_, 2 * D_)
            x = wide[:, D_:]
            got = ops.selective_scan_step(h, x, a['dt'][0], A, a['Bm'][0], a['Cm'][0], **{k: (v[0] if k == 'z' else v) for k, v in o.items()})
            ro, rh = R.scan(R.leaf(x, False)[None], R.leaf(a['dt'], False), R.leaf(a['A'], False), R.leaf(a['Bm'], False),
                            R.leaf(a['Cm'], False), h0=R.leaf(opt['h0'], False), **{k: R.leaf(v, False) for k, v in o.items()})
            R.close(got, ro[0], 8 + 2 * N_ + 32, 'out')
            R.close(h, rh, 8 + 2 * N_ + 32, 'h')


def test_frames_far_apart_in_memory():
    """strides that pass 32 bits: frames 1.3e9 values apart, forward and back, in bfloat16"""
    from asr_amd import ops
    t, d, far = 3, 64, 1_300_000_000
    buf = torch.empty((t - 1) * far + 4 * d, dtype=torch.bfloat16, device='cuda')
    a, opt = scan_inputs(gen(12), t, 1, d, 16, 1, torch.bfloat16)
    w = rn(gen(13), d, 4)
    do = rn(gen(14), t, 1, d, dtype=torch.bfloat16)

    def apart(v, at):
        o = buf.as_strided((t, 1, d), (far, d, 1), at)
        o.copy_(v)
        return o
    x, z, df = apart(a['x'], 0), apart(opt['z'], d), apart(do, 2 * d)
    res = []
    for xx, zz, dd in ((a['x'], opt['z'], do), (x, z, df)):
        q = dict(a, x=xx)
        kw = dict(opt, z=zz)
        for rev in (False, True):
            out, h, sv = ops.selective_scan_fwd(*q.values(), train=True, reverse=rev, **kw)
            g = ops.selective_scan_bwd(dd, *q.values(), sv, reverse=rev, **kw)
            c, _ = ops.causal_conv_fwd(xx, w, reverse=rev)
            cg = ops.causal_conv_bwd(dd, xx, w, reverse=rev)
            y, r, rstd = ops.add_rms_norm_fwd(xx[:, 0], opt['D'], residual=zz[:, 0])
            dx, dw = ops.add_rms_norm_bwd(dd[:, 0], xx[:, 0], opt['D'], rstd, residual=zz[:, 0])
            res.append([out, h, *g.values(), c, cg['x'], cg['w'], y, r, dx, dw])
    assert all(torch.equal(u, v) for u, v in zip(res[0] + res[1], res[2] + res[3]))


def test_list_of_scalars_views_and_repeats():
    from asr_amd import updates
    t = rn(gen(1), 4, 6)
    ts = [torch.tensor(3.0, device='cuda'), t, t, t[:, 1], t.expand(2, 4, 6), torch.empty(0, 5, device='cuda')]
    got, norm = updates.total_norm_constraint(ts, 1.0, return_norm=True)
    ref, rnorm = R.clip([R.leaf(v, False) for v in ts], 1.0, 1e-7)
    R.close(norm, rnorm.reshape(1), 2, 'norm')
    for u, v in zip(got, ref):
        R.close(u, v, 8, 'scaled')
