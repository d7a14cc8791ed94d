"""Values at the ends of float32's range in the selective scan: rates of -1e38 and below, gradients of large states, in front of
the padding that fills a row's last tile; the tolerances are test_gpu_ssm's."""
import pytest
import torch

import ref_ssm as R
from test_gpu_ssm import gen, rn, scan_inputs

pytestmark = pytest.mark.gpu


def gradients(a, opt, lens, do, dh, names, sizes={}):
    """the kernel's gradients against autograd of the float64 form; `names` of the inputs that are given; sizes: of the terms of a
    gradient that cancel in its sum"""
    from asr_amd import ops
    ln = torch.tensor(lens, dtype=torch.int32).cuda()
    out, h, saved = ops.selective_scan_fwd(*a.values(), lens=ln, train=True, **opt)
    gr = ops.selective_scan_bwd(do, *a.values(), saved, lens=ln, dh_last=dh, **opt)
    # a rate of -inf is what it is the limit of: all but -3e38 and below leave exp(delta A) zero for every delta above 1e-36
    ra = {k: R.leaf(v.clamp(min=-3e38) if k == 'A' else v) for k, v in a.items()}
    rop = {k: R.leaf(v) for k, v in opt.items()}
    ro, rh = R.scan(*ra.values(), lens=lens, **rop)
    (T, B, D), N = a['x'].shape, a['A'].shape[1]
    steps = 8 * T + 2 * N + 32
    R.close(out, ro, steps, 'out')
    R.close(h, rh, steps, 'h')
    ((ro * R.leaf(do, False)).sum() + (rh * R.leaf(dh, False)).sum()).backward()
    leafs = dict(x=ra['x'], dt=ra['dt'], A=ra['A'], B=ra['Bm'], C=ra['Cm'], **rop)
    for k in names:
        ref = leafs[k].grad
        R.close(gr[k], ref, 4 * steps + (B * T if k in ('A', 'D', 'dt_bias') else D if k in ('B', 'C') else 0), 'd' + k,
                max(sizes.get(k, 0.0), float(ref.abs().max())))


@pytest.mark.parametrize('T,lens', [(37, [37, 21]), (330, [330, 200])])
@pytest.mark.parametrize('D,N', [(64, 16), (70, 16), (64, 20)])
def test_gradient_of_infinite_decay_with_a_gradient_of_the_state(T, lens, D, N):
    """dh_last reaches the last valid frame through padding whose delta is zero; a rate that overflows against it there must
    leave nothing in the gradient of dt_bias"""
    a, opt = scan_inputs(gen(31), T, 2, D, N, 1, torch.float32)
    a['A'][:, 0], a['A'][:, 1] = -1e38, float('-inf')
    opt['dt_bias'].zero_()
    opt['h0'][..., :2] = 0
    dh = rn(gen(32), 2, D, N)
    dh[..., :2] *= 100.0
    gradients(a, opt, lens, rn(gen(33), T, 2, D), dh, ('x', 'dt', 'A', 'B', 'C', 'D', 'z', 'dt_bias', 'h0'))


@pytest.mark.parametrize('D,N', [(64, 16), (70, 4), (64, 33)])
def test_gradient_of_a_large_state_in_front_of_padding(D, N):
    """The product of the last state (5e19) and its gradient (2e19) is above float32; no valid frame has it, since a state is
    gone after a frame (delta 50, rate -100), and none of the gradients is: x dh B = 2e37 in dt, 1e30 in x and B, zero in A.
    dB is a sum of D terms of +-1e30, which may cancel to nothing: four roundings in a term and one in each of the seven levels that
    add them (64 lanes, then workgroups) leave at most 11 D of them at 1e30, fewer than 4 steps + D for D <= 70 (770 of 1414)."""
    T, B = 37, 2
    g = gen(41)

    def sign(*s):
        return (torch.randint(0, 2, s, generator=g) * 2.0 - 1.0).cuda()
    Bm = rn(g, T, B, 1, N)
    Bm[..., 0] = 1e9 * sign(T, B, 1)
    a = dict(x=1e9 * sign(T, B, D), dt=torch.full((T, B, D), 50.0).cuda(), A=torch.full((D, N), -100.0).cuda(), Bm=Bm,
             Cm=rn(g, T, B, 1, N))
    dh = rn(g, B, D, N)
    dh[..., 0] = 2e19 * sign(B, D)
    gradients(a, dict(dt_bias=torch.zeros(D).cuda()), [37, 21], rn(g, T, B, D), dh, ('x', 'dt', 'A', 'B', 'C', 'dt_bias'),
              dict(B=1e30))


@pytest.mark.parametrize('softplus', [True, False])
@pytest.mark.parametrize('rate', [float('-inf'), -3e38])
@pytest.mark.parametrize('N', [16, 5])
def test_a_frame_without_delta_leaves_the_state_alone_at_any_rate(N, rate, softplus):
    """single frames and the sequence: delta is exactly zero in every third frame (softplus(-200), or dt = 0), where a decay of
    any rate has no time to act"""
    from asr_amd import ops
    T, B, D = 12, 3, 64
    a, opt = scan_inputs(gen(51), T, B, D, N, 1, torch.float32)
    opt['dt_bias'] = None
    a['dt'] = a['dt'].abs() + 0.1
    a['dt'][::3] = -200.0 if softplus else 0.0
    a['A'][:, 0] = rate
    kw = dict(softplus=softplus)
    out, h, _ = ops.selective_scan_fwd(*a.values(), **opt, **kw)
    st = opt['h0'].clone()
    steps = torch.stack([ops.selective_scan_step(st, a['x'][t], a['dt'][t], a['A'], a['Bm'][t], a['Cm'][t], D=opt['D'],
                                                 z=opt['z'][t], **kw) for t in range(T)])
    ra = {k: R.leaf(v.clamp(min=-3e38) if k == 'A' else v, False) for k, v in a.items()}
    ro, rh = R.scan(*ra.values(), **{k: R.leaf(v, False) for k, v in opt.items()}, **kw)
    k = 8 * T + 2 * N + 32
    for name, got, ref in (('out', out, ro), ('h', h, rh), ('steps', steps, ro), ('h after steps', st, rh)):
        R.close(got, ref, k, name)


@pytest.mark.parametrize('T', [20, 150])
def test_a_growing_rate_above_the_range_of_its_product_with_log2_e(T):
    """a rate of 3e38 over frames whose delta is exactly zero: nothing grows, in single frames, in the sequence, in its chunks of
    time, in the padding and in the gradients"""
    from asr_amd import ops
    B, D, N = 2, 64, 8
    lens = [T, T - 7]
    a, opt = scan_inputs(gen(61), T, B, D, N, 1, torch.float32)
    opt.update(z=None, dt_bias=torch.zeros(D).cuda())
    a['dt'].fill_(-200.0)
    a['A'][:, 0] = 3e38
    do, dh = rn(gen(62), T, B, D), rn(gen(63), B, D, N) * 0.1
    gradients(a, {k: v for k, v in opt.items() if v is not None}, lens, do, dh, ('x', 'C', 'D', 'h0'))
    st = opt['h0'].clone()
    got = ops.selective_scan_step(st, a['x'][0], a['dt'][0], a['A'], a['Bm'][0], a['Cm'][0], D=opt['D'])
    assert torch.equal(st, opt['h0'])
    ref, _ = R.scan(*[R.leaf(v[:1] if k != 'A' else v, False) for k, v in a.items()], D=R.leaf(opt['D'], False),
                    h0=R.leaf(opt['h0'], False))
    R.close(got, ref[0], 8 + 2 * N + 32, 'out')
