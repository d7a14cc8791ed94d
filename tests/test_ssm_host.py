"""Host side of the state-space layer's operators (no GPU): the refusals of the wrappers and of the C entries, the layout of the
descriptor, workspace sizes, and the plain float64 forms against differences."""
import ctypes as C
import os
import subprocess

import numpy as np
import pytest
import torch

import ref_ssm as R

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def test_descriptor_layout_matches_ctypes(tmp_path):
    from asr_amd import _lib
    names = [f[0] for f in _lib.SscanDesc._fields_]
    prog = tmp_path / 'layout.c'
    prog.write_text('#include <stdio.h>\n#include <stddef.h>\n#include "asr_amd.h"\nint main(void) {\n'
                    + ''.join('printf("%%zu ", offsetof(asr_sscan_desc, %s));\n' % n for n in names)
                    + 'printf("%zu", sizeof(asr_sscan_desc));\nreturn 0;\n}\n')
    exe = tmp_path / 'layout'
    subprocess.check_call(['gcc', '-std=c99', '-Wall', '-Werror', '-I', os.path.join(ROOT, 'include'), str(prog), '-o', str(exe)])
    got = [int(v) for v in subprocess.check_output([str(exe)]).decode().split()]
    assert got == [getattr(_lib.SscanDesc, n).offset for n in names] + [C.sizeof(_lib.SscanDesc)]
    # the wrapper packs the members as eight ints and 8-byte words
    from asr_amd import ops_ssm
    words = list(range(1, len(names) + 1))
    d = _lib.SscanDesc.from_buffer_copy(ops_ssm._MEMBERS.pack(*words))
    assert [getattr(d, n) for n in names] == words and ops_ssm._MEMBERS.size == C.sizeof(_lib.SscanDesc)
    assert names.index('ckpt') + 1 + len(ops_ssm._FORWARD_ONLY) == len(names)


def conv_args(**kw):
    a = dict(x=torch.zeros(5, 2, 8), w=torch.zeros(8, 4), bias=torch.zeros(8), state=torch.zeros(3, 2, 8),
             lens=torch.tensor([5, 2], dtype=torch.int32))
    a.update(kw)
    return a


@pytest.mark.parametrize('kw,msg', [
    (dict(x=torch.zeros(5, 8)), 'axes'), (dict(x=torch.zeros(5, 2, 8, dtype=torch.float64)), 'float64'),
    (dict(x=torch.zeros(5, 2, 16)[..., ::2]), 'stride 1'), (dict(w=torch.zeros(8, 1)), 'K <= 8'), (dict(w=torch.zeros(8, 9)), 'K <= 8'),
    (dict(w=torch.zeros(7, 4)), 'shape'), (dict(w=torch.zeros(4, 8).t()), 'contiguous'), (dict(w=torch.zeros(8, 4).half()), 'float32'),
    (dict(bias=torch.zeros(9)), 'shape'), (dict(state=torch.zeros(4, 2, 8)), 'shape'), (dict(state=torch.zeros(3, 2, 8).half()), 'like'),
    (dict(lens=torch.tensor([5, 2])), 'int32'), (dict(lens=torch.zeros(3, dtype=torch.int32)), 'int32'), (dict(act='relu'), 'silu'),
    (dict(), 'GPU'), (dict(x=torch.zeros(5, 2, 0), w=torch.zeros(0, 4)), 'channels')])
def test_conv_refusals(kw, msg):
    from asr_amd import ops
    with pytest.raises(ValueError, match=msg):
        ops.causal_conv_fwd(**conv_args(**kw))
    with pytest.raises(ValueError, match=msg):
        ops.causal_conv_bwd(torch.zeros(5, 2, 8), **conv_args(**kw))


def test_conv_step_and_gradient_refusals():
    from asr_amd import ops
    x, st, w = torch.zeros(2, 8), torch.zeros(3, 2, 8), torch.zeros(8, 4)
    for args, msg in [((torch.zeros(1, 2, 8), st, w), 'axes'), ((x, torch.zeros(2, 2, 8), w), 'shape'), ((x, st.half(), w), 'like'),
                      ((x, torch.zeros(3, 8, 2).transpose(1, 2), w), 'stride'), ((x, torch.zeros(2, 3, 8).transpose(0, 1), w), 'contiguous'),
                      ((x, st, torch.zeros(8, 9)), 'K <= 8'), ((x[:, :0], st[..., :0], w[:0]), 'channels'), ((x.double(), st, w), 'float64'),
                      ((x, st, w[:4]), 'shape'), ((x, st, w, torch.zeros(7)), 'bias'), ((x, st, w, None, 'relu'), 'silu'), ((x, st, w), 'GPU')]:
        with pytest.raises(ValueError, match=msg):
            ops.causal_conv_step(*args)
    with pytest.raises(ValueError, match='dout'):
        ops.causal_conv_bwd(torch.zeros(4, 2, 8), **conv_args())
    with pytest.raises(ValueError, match='dstate_out'):
        ops.causal_conv_bwd(torch.zeros(5, 2, 8), dstate_out=torch.zeros(2, 2, 8), **conv_args())


def scan_args(**kw):
    a = dict(x=torch.zeros(5, 2, 8), dt=torch.zeros(5, 2, 8), A=torch.zeros(8, 4), Bm=torch.zeros(5, 2, 2, 4), Cm=torch.zeros(5, 2, 2, 4),
             D=torch.zeros(8), z=torch.zeros(5, 2, 8), dt_bias=torch.zeros(8), h0=torch.zeros(2, 8, 4),
             lens=torch.tensor([5, 2], dtype=torch.int32))
    a.update(kw)
    return a


SCAN_BAD = [
    (dict(x=torch.zeros(5, 8)), 'axes'), (dict(x=torch.zeros(5, 2, 8).double()), 'float64'), (dict(dt=torch.zeros(5, 2, 7)), 'dt'),
    (dict(dt=torch.zeros(5, 2, 8).bfloat16()), 'like'), (dict(A=torch.zeros(8, 65)), 'N <= 64'), (dict(A=torch.zeros(8, 0)), 'N <= 64'),
    (dict(A=torch.zeros(8, 4).half()), 'float32'), (dict(A=torch.zeros(4, 8).t()), 'contiguous'), (dict(Bm=torch.zeros(5, 2, 4)), 'axes'),
    (dict(Bm=torch.zeros(5, 2, 3, 4)), 'divide'), (dict(Cm=torch.zeros(5, 2, 1, 4)), 'Cm'), (dict(Cm=torch.zeros(5, 2, 2, 8)[..., ::2]), 'stride 1'),
    (dict(D=torch.zeros(4)), 'D'), (dict(z=torch.zeros(5, 2, 4)), 'z'), (dict(z=torch.zeros(5, 2)), 'z'), (dict(dt=torch.zeros(5)), 'dt'),
    (dict(x=torch.zeros(5, 2, 0), dt=torch.zeros(5, 2, 0), A=torch.zeros(0, 4)), 'divide'), (dict(Bm=torch.zeros(5, 2, 0, 4)), 'divide'), (dict(dt_bias=torch.zeros(8).half()), 'float32'),
    (dict(h0=torch.zeros(2, 4, 8)), 'h0'), (dict(lens=torch.zeros(2)), 'int32'), (dict(), 'GPU')]


@pytest.mark.parametrize('kw,msg', SCAN_BAD)
def test_scan_refusals(kw, msg):
    from asr_amd import ops, _lib
    with pytest.raises(ValueError, match=msg):
        ops.selective_scan_fwd(**scan_args(**kw))
    saved = torch.zeros(_lib.lib().asr_sscan_ckpt_floats(5, 2, 8, 4))
    with pytest.raises(ValueError, match=msg):
        ops.selective_scan_bwd(torch.zeros(5, 2, 8), saved=saved, **scan_args(**kw))


def test_scan_gradient_and_step_refusals():
    from asr_amd import ops, _lib
    saved = torch.zeros(_lib.lib().asr_sscan_ckpt_floats(5, 2, 8, 4))
    for do, sv, kw, msg in [(torch.zeros(5, 2, 7), saved, {}, 'dout'), (torch.zeros(5, 2, 8), None, {}, 'saved'),
                            (torch.zeros(5, 2, 8), saved[1:], {}, 'saved'), (torch.zeros(5, 2, 8), saved, dict(dh_last=torch.zeros(2, 8)), 'dh_last')]:
        with pytest.raises(ValueError, match=msg):
            ops.selective_scan_bwd(do, saved=sv, **scan_args(), **kw)
    h, x, A, b = torch.zeros(2, 8, 4), torch.zeros(2, 8), torch.zeros(8, 4), torch.zeros(2, 2, 4)
    for args, kw, msg in [((h, torch.zeros(1, 2, 8), x, A, b, b), {}, 'axes'), ((h.half(), x, x, A, b, b), {}, 'float32'),
                          ((h[:1], x, x, A, b, b), {}, 'h:'), ((h, x, x, A, torch.zeros(2, 3, 4), b), {}, 'divide'), ((h, x, x, A, b, b[:, :1]), {}, 'Cm'),
                          ((h, x, x, A, b, b), dict(z=x.half()), 'like'), ((h, x, x, A, b, b), {}, 'GPU'),
                          ((torch.zeros(2, 4, 8).transpose(1, 2), x, x, A, b, b), {}, 'contiguous'),
                          ((h, x, x, A, b[:, :0], b[:, :0]), {}, 'divide'), ((h[:, :0], x[:, :0], x[:, :0], A[:0], b, b), {}, 'divide'),
                          ((h, x.double(), x, A, b, b), {}, 'float64'), ((h, x, x[:1], A, b, b), {}, 'dt'), ((h, x, x, A[:4], b, b), {}, 'A:'),
                          ((h, x, x, A, b, b), dict(D=x[0, :4]), 'D:'), ((h, x, x, A, b, b), dict(dt_bias=x[0].half()), 'dt_bias'),
                          ((h, torch.zeros(2, 16)[:, ::2], x, A, b, b), {}, 'stride 1'), ((h, x, x, torch.zeros(8, 65), b, b), {}, 'N <= 64'),
                          ((h, x, x, A, b[0], b), {}, 'axes'), ((h, x, x, A, b, b), dict(z=x[0]), 'z:')]:
        with pytest.raises(ValueError, match=msg):
            ops.selective_scan_step(*args, **kw)


def test_norm_and_list_refusals():
    from asr_amd import ops, updates
    x, w = torch.zeros(3, 8), torch.zeros(8)
    for args, kw, msg in [((torch.zeros(8), w), {}, 'axes'), ((torch.zeros(3, 0), torch.zeros(0)), {}, 'columns'), ((x.double(), w), {}, 'float64'),
                          ((x, torch.zeros(7)), {}, 'w'), ((x, w), dict(residual=torch.zeros(2, 8)), 'residual'), ((x, w), dict(eps=-1.0), 'negative'),
                          ((x, w), dict(eps=float('nan')), 'negative'), ((torch.zeros(3, 16)[:, ::2], w), {}, 'stride 1'), ((x, w), {}, 'GPU')]:
        with pytest.raises(ValueError, match=msg):
            ops.add_rms_norm_fwd(*args, **kw)
    for args, kw, msg in [((torch.zeros(3, 7), x, w, torch.zeros(3)), {}, 'dy'), ((x, x, w, torch.zeros(2)), {}, 'rstd'),
                          ((x, x, w, torch.zeros(3)), dict(dres=x.half()), 'like'),
                          ((x, x, w, torch.zeros(3)), dict(residual=x[:2]), 'residual'), ((x, x, w, torch.zeros(3)), {}, 'GPU')]:
        with pytest.raises(ValueError, match=msg):
            ops.add_rms_norm_bwd(*args, **kw)
    for args, msg in [(([torch.zeros(3).long()], 1.0), 'int64'), (([torch.zeros(3)], -1.0), 'negative'), (([torch.zeros(3)], 1.0, -1.0), 'negative'),
                      (([torch.zeros(3)], 1.0), 'GPU')]:
        with pytest.raises(ValueError, match=msg):
            ops.clip_list(*args)
    with pytest.raises(ValueError, match='none'):
        ops.clip_list([], 1.0)
    # a network's own gradients go on as before
    for own in (None, [], [np.zeros(3)], [torch.zeros(3)]):
        cg = updates.total_norm_constraint(own, 1.0)
        assert type(cg) is updates.ClippedGrads and cg.max_norm == 1.0


def test_updater_behind_a_clipped_list_still_clips(monkeypatch):
    """adam(total_norm_constraint([tensors], 5)) clips the network's own gradients, as it does behind any other tensor_vars."""
    from asr_amd import ops, updates

    class OnGpu(torch.Tensor):
        is_cuda = True
    ts = [torch.zeros(3).as_subclass(OnGpu), torch.zeros(2).as_subclass(OnGpu)]
    monkeypatch.setattr(ops, 'clip_list', lambda tensors, max_norm, eps: ([t + 1 for t in tensors], torch.ones(1)))
    scaled, norm = updates.total_norm_constraint(ts, 5.0, 1e-6, return_norm=True)
    assert isinstance(scaled, list) and len(scaled) == 2 and float(norm) == 1.0
    for updater in (updates.adam, updates.sgd):
        step, _ = updater(scaled)
        assert step.clip.max_norm == 5.0 and step.clip.epsilon == 1e-6


def test_c_entries_refuse_before_they_launch():
    from asr_amd import _lib
    L = _lib.lib()
    ARG, WS, LIMIT = -1, -3, -5
    p = 1 << 20                                            # never dereferenced: the calls below return first
    assert L.asr_conv_fwd(3, 4, 2, 8, 4, p, 16, 8, p, None, None, None, 1, 0, p, 16, 8, None, None) == ARG
    assert L.asr_conv_fwd(0, 4, 2, 8, 9, p, 16, 8, p, None, None, None, 1, 0, p, 16, 8, None, None) == LIMIT
    assert L.asr_conv_fwd(0, 4, 2, 8, 1, p, 16, 8, p, None, None, None, 1, 0, p, 16, 8, None, None) == ARG
    assert L.asr_conv_fwd(0, 4, 2, 8, 4, None, 16, 8, p, None, None, None, 1, 0, p, 16, 8, None, None) == ARG
    assert L.asr_conv_fwd(0, 4, 2, 8, 4, p, 16, 8, p, None, p, None, 1, 0, p, 16, 8, p, None) == ARG       # state_out is state
    assert L.asr_conv_fwd(0, 4, 0, 8, 4, None, 16, 8, p, None, None, None, 1, 0, None, 16, 8, None, None) == 0
    assert L.asr_conv_fwd(0, 4, 1 << 17, 8, 4, p, 16, 8, p, None, None, None, 1, 0, p, 16, 8, None, None) == LIMIT
    need = L.asr_conv_bwd_ws_bytes(300, 2, 8, 4)
    assert need > 0
    assert L.asr_conv_bwd(0, 300, 2, 8, 4, p, 16, 8, p, 16, 8, p, None, None, None, 1, 0, None, p, p, None, p, need - 1, None) == WS
    assert L.asr_conv_bwd(0, 300, 2, 8, 4, p, 16, 8, p, 16, 8, p, None, None, None, 1, 0, None, p, p, None, None, need, None) == WS
    assert L.asr_conv_step(0, 2, 8, 4, p, 8, None, p, None, 1, p, 8, None) == ARG

    def desc(**kw):
        d = _lib.SscanDesc()
        d.T, d.B, d.D, d.N, d.G = 300, 1, 64, 16, 1
        for n in ('x', 'dt', 'Bm', 'Cm', 'A', 'out', 'dout', 'ckpt', 'dx', 'ddt', 'dB', 'dC', 'dA'):
            setattr(d, n, p)
        for k, v in kw.items():
            setattr(d, k, v)
        return C.byref(d)
    assert L.asr_sscan_ws_bytes(300, 1, 64, 16, 1, 0) > 0
    assert L.asr_sscan_fwd(desc(), None, 0, None) == WS
    assert L.asr_sscan_fwd(desc(), p, L.asr_sscan_ws_bytes(300, 1, 64, 16, 1, 0) - 1, None) == WS
    assert L.asr_sscan_bwd(desc(), p, L.asr_sscan_ws_bytes(300, 1, 64, 16, 1, 1) - 1, None) == WS
    for fn in (L.asr_sscan_fwd, L.asr_sscan_bwd):
        assert fn(None, p, 1 << 40, None) == ARG
        assert fn(desc(N=65), p, 1 << 40, None) == LIMIT
        assert fn(desc(G=3), p, 1 << 40, None) == ARG
        assert fn(desc(dtype=7), p, 1 << 40, None) == ARG
        assert fn(desc(A=None), p, 1 << 40, None) == ARG
        assert fn(desc(x=None), p, 1 << 40, None) == ARG
        assert fn(desc(B=1 << 17), p, 1 << 40, None) == LIMIT
    assert L.asr_sscan_fwd(desc(h0=p, h_last=p), p, 1 << 40, None) == ARG
    assert L.asr_sscan_fwd(desc(out=None), p, 1 << 40, None) == ARG
    assert L.asr_sscan_bwd(desc(z=p), p, 1 << 40, None) == ARG                     # z without dz
    assert L.asr_sscan_bwd(desc(ckpt=None), p, 1 << 40, None) == ARG
    assert L.asr_sscan_fwd(desc(B=0), None, 0, None) == 0
    assert L.asr_sscan_step(0, 2, 8, 70, 1, p, p, 8, p, 8, p, p, 70, 70, p, 70, 70, None, None, 0, None, 1, p, 8, None) == LIMIT
    assert L.asr_sscan_step(0, 2, 8, 16, 3, p, p, 8, p, 8, p, p, 16, 16, p, 16, 16, None, None, 0, None, 1, p, 8, None) == ARG
    assert L.asr_sscan_step(0, 2, 8, 16, 1, None, p, 8, p, 8, p, p, 16, 16, p, 16, 16, None, None, 0, None, 1, p, 8, None) == ARG
    assert L.asr_rms_norm_fwd(0, p, 8, None, 0, p, 3, 0, 1e-6, p, None, None, None) == ARG
    assert L.asr_rms_norm_fwd(0, p, 8, None, 0, p, 3, 8, -1.0, p, None, None, None) == ARG
    assert L.asr_rms_norm_fwd(0, p, 8, None, 0, p, 0, 8, 1e-6, None, None, None, None) == 0
    assert L.asr_rms_norm_bwd(0, p, 8, p, 8, None, 0, p, p, None, 0, 3, 8, p, p, p, L.asr_rms_norm_bwd_ws_bytes(3, 8) - 1, None) == WS
    one, kind, ptr = (C.c_longlong * 1)(100), (C.c_int * 1)(0), (C.c_void_p * 1)(p)
    need = L.asr_clip_list_ws_bytes(1, one)
    assert L.asr_clip_list(1, kind, ptr, ptr, one, 1.0, 1e-7, p, p, need - 1, None) == WS
    assert L.asr_clip_list(1, kind, ptr, ptr, one, -1.0, 1e-7, p, p, need, None) == ARG
    assert L.asr_clip_list(1, (C.c_int * 1)(4), ptr, ptr, one, 1.0, 1e-7, p, p, need, None) == ARG
    assert L.asr_clip_list(1, kind, ptr, ptr, (C.c_longlong * 1)(-1), 1.0, 1e-7, p, p, need, None) == ARG
    assert L.asr_clip_list(1, kind, (C.c_void_p * 1)(None), ptr, one, 1.0, 1e-7, p, p, need, None) == ARG
    assert L.asr_clip_list(1, kind, ptr, ptr, one, 1.0, 1e-7, p, p + 4, need, None) == ARG
    # beyond a launch's work items, and workspaces off the 16-byte grid
    assert L.asr_sscan_bwd(desc(T=1 << 23, B=64), p, 1 << 60, None) == LIMIT
    assert L.asr_sscan_step(0, 1 << 13, 1 << 15, 16, 1, p, p, 8, p, 8, p, p, 16, 16, p, 16, 16, None, None, 0, None, 1, p, 8, None) == LIMIT
    assert L.asr_rms_norm_fwd(0, p, 8, None, 0, p, 1 << 24, 8, 1e-6, p, None, None, None) == LIMIT
    assert L.asr_clip_list(1, kind, ptr, ptr, (C.c_longlong * 1)(1 << 38), 1.0, 1e-7, p, p, 1 << 60, None) == LIMIT
    assert L.asr_conv_fwd(0, 1 << 22, 2, 8, 4, p, 16, 8, p, None, None, None, 1, 0, p, 16, 8, None, None) == LIMIT
    assert L.asr_conv_fwd(0, 4, 2, 1 << 21, 4, p, 16, 8, p, None, None, None, 1, 0, p, 16, 8, None, None) == LIMIT
    assert L.asr_sscan_fwd(desc(), p + 8, 1 << 40, None) == ARG and L.asr_sscan_bwd(desc(), p + 8, 1 << 40, None) == ARG
    assert L.asr_conv_bwd(0, 30, 2, 8, 4, p, 16, 8, p, 16, 8, p, None, None, None, 1, 0, None, p, p, None, p + 4, 1 << 30, None) == ARG
    assert L.asr_rms_norm_bwd(0, p, 8, p, 8, None, 0, p, p, None, 0, 3, 8, p, p, p + 4, 1 << 30, None) == ARG


def test_plain_forms_against_differences():
    """the float64 forms the kernels are held to: directional derivatives by central differences, error e^2 and 2^-53 / e"""
    g = torch.Generator().manual_seed(1)

    def rn(*s):
        return torch.randn(*s, generator=g, dtype=torch.float64)
    T, B, D, N, G, K = 6, 2, 4, 3, 2, 4
    lens = [6, 3]
    a = dict(x=rn(T, B, D), dt=rn(T, B, D), A=-rn(D, N).exp(), Bm=rn(T, B, G, N), Cm=rn(T, B, G, N), D=rn(D), z=rn(T, B, D),
             dt_bias=rn(D), h0=rn(B, D, N))
    do, dh = rn(T, B, D), rn(B, D, N)
    c = dict(x=rn(T, B, D), w=rn(D, K), bias=rn(D), state=rn(K - 1, B, D))
    ds = rn(K - 1, B, D)

    def l_scan(a):
        o, h = R.scan(**a, lens=lens, reverse=True)
        return (o * do).sum() + (h * dh).sum()

    def l_conv(a):
        o, s = R.conv(**a, lens=lens, reverse=True)
        return (o * do).sum() + (s * ds).sum()
    for loss, args in ((l_scan, a), (l_conv, c)):
        leafs = {k: v.clone().requires_grad_() for k, v in args.items()}
        grads = dict(zip(leafs, torch.autograd.grad(loss(leafs), list(leafs.values()))))
        for k in args:
            v, e = rn(*args[k].shape), 1e-5
            up, dn = dict(args), dict(args)
            up[k], dn[k] = args[k] + e * v, args[k] - e * v
            diff = float(loss(up) - loss(dn)) / (2 * e)
            want = float((grads[k] * v).sum())
            assert abs(diff - want) < 1e-7 * (1 + abs(want)), (k, diff, want)
