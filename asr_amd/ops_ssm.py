"""The operators of a selective state-space layer: short causal convolution over time, selective scan, root-mean-square norm
with the residual's addition, and the global norm over a list of gradients.  Wrappers over the C-ABI (include/asr_amd.h)
like asr_amd.ops, which re-exports them; the reference has no such layer (its recurrences are LSTMs), so no file of it is cited.

Shapes.  Sequences are time-major (T, B, channels) with unit channel stride and any (t, b) strides, in float32, bfloat16 or
float16, all activations of a call in one type.  Parameters, scan states and parameter gradients are float32.  `lens` (B,)
int32: frames at and behind lens[b] are padding, whose values are never used (they may be NaN); outputs and gradients there
are zero and the state is what the last valid frame left.  reverse=True walks every row from its last valid frame to the first.

Every call is enqueued on the current stream of the tensors' device and allocates its outputs and its workspace through
torch, so calls on several streams and calls captured into graphs share nothing.  Results do not vary from run to run.
A wrong argument raises ValueError before anything is launched.
"""
import ctypes as C

import torch

from . import _lib
from ._lib import check

_DTYPES = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}
MAX_STATES = 64
MAX_TAPS = 8


def _fail(msg):
    raise ValueError(msg)


def _p(t):
    return None if t is None else t.data_ptr()


def _act(name, t, shape, dtype):
    """an activation: the shape, the call's type, unit stride of the last axis"""
    if t.shape != shape:
        _fail('%s: shape %s, expected %s' % (name, tuple(t.shape), tuple(shape)))
    if t.dtype != dtype:
        _fail('%s: %s, expected %s like the other activations' % (name, t.dtype, dtype))
    if t.stride(-1) != 1 and t.shape[-1] > 1:
        _fail('%s: the last axis must have stride 1' % name)


def _par(name, t, shape):
    """a parameter or a state: float32, contiguous"""
    if t.shape != shape:
        _fail('%s: shape %s, expected %s' % (name, tuple(t.shape), tuple(shape)))
    if t.dtype != torch.float32:
        _fail('%s: %s, expected torch.float32' % (name, t.dtype))
    if not t.is_contiguous():
        _fail('%s: must be contiguous' % name)


def _type(name, t):
    if t.dtype not in _DTYPES:
        _fail('%s: %s, expected float32, bfloat16 or float16' % (name, t.dtype))
    return _DTYPES[t.dtype]


def _lens(lens, B):
    if lens is not None and (lens.shape != (B,) or lens.dtype != torch.int32 or not lens.is_contiguous()):
        _fail('lens: expected %d contiguous int32 values' % B)


def _device(first, *others):
    """all tensors on one GPU; its index"""
    dev = first.device
    if dev.type != 'cuda':
        _fail('tensors must be on the GPU (there is no CPU path)')
    for t in others:
        if t is not None and t.device != dev:
            _fail('tensors on different devices: %s and %s' % (dev, t.device))
    return dev.index


class _On(object):
    """Makes the tensors' device current for the launches of a call, if it is not."""
    __slots__ = ('index', 'before')

    def __init__(self, index):
        self.index = index

    def __enter__(self):
        self.before = torch.cuda.current_device()
        if self.before != self.index:
            torch.cuda.set_device(self.index)
        return torch.cuda.current_stream().cuda_stream

    def __exit__(self, *a):
        if self.before != self.index:
            torch.cuda.set_device(self.before)


# ---------------------------------------------------------------------------------------------- convolution
def _act_kind(act):
    if act not in ('silu', None):
        _fail("act: 'silu' or None, got %r" % (act,))
    return 1 if act else 0


def _conv_args(x, w, bias, state, lens):
    if x.dim() != 3:
        _fail('x: expected (T, B, D), got %d axes' % x.dim())
    T, B, D = x.shape
    if w.dim() != 2 or not 2 <= w.shape[1] <= MAX_TAPS:
        _fail('w: expected (D, K) with 2 <= K <= %d, got %s' % (MAX_TAPS, tuple(w.shape)))
    K = w.shape[1]
    dt = _type('x', x)
    if D < 1:
        _fail('x: no channels')
    _act('x', x, (T, B, D), x.dtype)
    _par('w', w, (D, K))
    if bias is not None:
        _par('bias', bias, (D,))
    if state is not None:
        _act('state', state, (K - 1, B, D), x.dtype)
        if not state.is_contiguous():
            _fail('state: must be contiguous')
    _lens(lens, B)
    return dt, T, B, D, K


def causal_conv_fwd(x, w, bias=None, state=None, lens=None, act='silu', reverse=False, want_state=False):
    """out[s] = act(bias + sum_k w[:, k] x[s - (K-1) + k]) over the valid frames s of every row; x (T, B, D), w (D, K).
    state (K-1, B, D): the frames in front of the first one (None: zeros).  -> (out, the state behind the last valid frame
    if want_state, else None)."""
    dt, T, B, D, K = _conv_args(x, w, bias, state, lens)
    kind = _act_kind(act)
    dev = _device(x, w, bias, state, lens)
    out = torch.empty((T, B, D), dtype=x.dtype, device=x.device)
    new = torch.empty((K - 1, B, D), dtype=x.dtype, device=x.device) if want_state else None
    with _On(dev) as st:
        check(_lib.lib().asr_conv_fwd(dt, T, B, D, K, _p(x), x.stride(0), x.stride(1), _p(w), _p(bias), _p(state), _p(lens),
                                      kind, int(reverse), _p(out), B * D, D, _p(new), st), 'asr_conv_fwd')
    return out, new


def causal_conv_bwd(dout, x, w, bias=None, state=None, lens=None, act='silu', reverse=False, dstate_out=None):
    """Gradients of causal_conv_fwd for the gradient dout of its output (and dstate_out of the state it returned):
    {'x', 'w', 'bias', 'state'}; 'bias' / 'state' are None when there was none."""
    dt, T, B, D, K = _conv_args(x, w, bias, state, lens)
    kind = _act_kind(act)
    _act('dout', dout, (T, B, D), x.dtype)
    if dstate_out is not None:
        _act('dstate_out', dstate_out, (K - 1, B, D), x.dtype)
        if not dstate_out.is_contiguous():
            _fail('dstate_out: must be contiguous')
    dev = _device(x, dout, w, bias, state, lens, dstate_out)
    dx = torch.empty((T, B, D), dtype=x.dtype, device=x.device)
    dwb = torch.empty(D * (K + 1), dtype=torch.float32, device=x.device)
    ds = torch.empty((K - 1, B, D), dtype=x.dtype, device=x.device) if state is not None else None
    L = _lib.lib()
    with _On(dev) as st:
        ws = torch.empty(L.asr_conv_bwd_ws_bytes(T, B, D, K), dtype=torch.uint8, device=x.device)
        check(L.asr_conv_bwd(dt, T, B, D, K, _p(dout), dout.stride(0), dout.stride(1), _p(x), x.stride(0), x.stride(1),
                             _p(w), _p(bias), _p(state), _p(lens), kind, int(reverse), _p(dstate_out), _p(dx), _p(dwb),
                             _p(ds), _p(ws), ws.numel(), st), 'asr_conv_bwd')
    return {'x': dx, 'w': dwb[:D * K].view(D, K), 'bias': dwb[D * K:] if bias is not None else None, 'state': ds}


def causal_conv_step(x, state, w, bias=None, act='silu'):
    """One frame: x (B, D), state (K-1, B, D), which moves on in place.  -> out (B, D).  Equal to causal_conv_fwd over one
    frame."""
    if x.dim() != 2:
        _fail('x: expected (B, D), got %d axes' % x.dim())
    B, D = x.shape
    if w.dim() != 2 or not 2 <= w.shape[1] <= MAX_TAPS:
        _fail('w: expected (D, K) with 2 <= K <= %d, got %s' % (MAX_TAPS, tuple(w.shape)))
    K = w.shape[1]
    dt = _type('x', x)
    if D < 1:
        _fail('x: no channels')
    _act('x', x, (B, D), x.dtype)
    _par('w', w, (D, K))
    if bias is not None:
        _par('bias', bias, (D,))
    _act('state', state, (K - 1, B, D), x.dtype)
    if not state.is_contiguous():
        _fail('state: must be contiguous')
    kind = _act_kind(act)
    dev = _device(x, state, w, bias)
    out = torch.empty((B, D), dtype=x.dtype, device=x.device)
    with _On(dev) as st:
        check(_lib.lib().asr_conv_step(dt, B, D, K, x.data_ptr(), x.stride(0), state.data_ptr(), w.data_ptr(), _p(bias),
                                       kind, out.data_ptr(), D, st), 'asr_conv_step')
    return out


# ---------------------------------------------------------------------------------------------- selective scan
def _scan_args(x, dt, A, Bm, Cm, D, z, dt_bias, h0, lens):
    if x.dim() != 3:
        _fail('x: expected (T, B, D), got %d axes' % x.dim())
    T, B, Dn = x.shape
    if A.dim() != 2 or not 1 <= A.shape[1] <= MAX_STATES:
        _fail('A: expected (D, N) with 1 <= N <= %d, got %s' % (MAX_STATES, tuple(A.shape)))
    N = A.shape[1]
    if Bm.dim() != 4:
        _fail('Bm: expected (T, B, G, N), got %d axes' % Bm.dim())
    G = Bm.shape[2]
    if Dn < 1 or G < 1 or Dn % G:
        _fail('Bm: %d groups do not divide %d channels' % (G, Dn))
    kind = _type('x', x)
    ty = x.dtype
    _act('x', x, (T, B, Dn), ty)
    _act('dt', dt, (T, B, Dn), ty)
    _par('A', A, (Dn, N))
    _act('Bm', Bm, (T, B, G, N), ty)
    _act('Cm', Cm, (T, B, G, N), ty)
    if z is not None:
        _act('z', z, (T, B, Dn), ty)
    if D is not None:
        _par('D', D, (Dn,))
    if dt_bias is not None:
        _par('dt_bias', dt_bias, (Dn,))
    if h0 is not None:
        _par('h0', h0, (B, Dn, N))
    _lens(lens, B)
    return kind, T, B, Dn, N, G


def _scan_desc(kind, T, B, Dn, N, G, x, dt, A, Bm, Cm, D, z, dt_bias, h0, lens, softplus, reverse):
    return (T, B, Dn, N, G, kind, int(reverse), int(softplus), _p(lens),
            x.data_ptr(), x.stride(0), x.stride(1), dt.data_ptr(), dt.stride(0), dt.stride(1),
            _p(z), z.stride(0) if z is not None else 0, z.stride(1) if z is not None else 0,
            Bm.data_ptr(), Bm.stride(0), Bm.stride(1), Bm.stride(2), Cm.data_ptr(), Cm.stride(0), Cm.stride(1), Cm.stride(2),
            A.data_ptr(), _p(D), _p(dt_bias), _p(h0))


def selective_scan_fwd(x, dt, A, Bm, Cm, D=None, z=None, dt_bias=None, h0=None, lens=None, softplus=True, reverse=False,
                       train=False):
    """h[s] = exp(delta A) h[s-1] + delta x B[s],  y = C[s] h[s] + D x,  out = y silu(z)  (y without z), with
    delta = softplus(dt + dt_bias)  (dt + dt_bias with softplus=False).

    x, dt, z (T, B, D); A (D, N), N <= 64; Bm, Cm (T, B, G, N), shared by the D / G channels of a group; D, dt_bias (D,);
    h0 (B, D, N) (None: zeros).  -> (out (T, B, D), the state behind the last valid frame (B, D, N), what
    selective_scan_bwd needs if train, else None)."""
    a = _scan_args(x, dt, A, Bm, Cm, D, z, dt_bias, h0, lens)
    kind, T, B, Dn, N, G = a
    dev = _device(x, dt, A, Bm, Cm, D, z, dt_bias, h0, lens)
    L = _lib.lib()
    out = torch.empty((T, B, Dn), dtype=x.dtype, device=x.device)
    h = torch.empty((B, Dn, N), dtype=torch.float32, device=x.device)
    saved = torch.empty(L.asr_sscan_ckpt_floats(T, B, Dn, N), dtype=torch.float32, device=x.device) if train else None
    desc = _lib.SscanDesc(*_scan_desc(*a, x, dt, A, Bm, Cm, D, z, dt_bias, h0, lens, softplus, reverse),
                          out.data_ptr(), B * Dn, Dn, h.data_ptr(), _p(saved))
    with _On(dev) as st:
        need = L.asr_sscan_ws_bytes(T, B, Dn, N, G, 0)
        ws = torch.empty(need, dtype=torch.uint8, device=x.device) if need else None
        check(L.asr_sscan_fwd(C.byref(desc), _p(ws), need, st), 'asr_sscan_fwd')
    return out, h, saved


def selective_scan_bwd(dout, x, dt, A, Bm, Cm, saved, D=None, z=None, dt_bias=None, h0=None, lens=None, softplus=True,
                       reverse=False, dh_last=None):
    """Gradients of selective_scan_fwd(..., train=True) called with the same arguments, for the gradient dout of its output
    (and dh_last of the state it returned): {'x', 'dt', 'A', 'B', 'C', 'D', 'z', 'dt_bias', 'h0'}, None where the argument
    was.  `saved` is what the forward call returned."""
    a = _scan_args(x, dt, A, Bm, Cm, D, z, dt_bias, h0, lens)
    kind, T, B, Dn, N, G = a
    _act('dout', dout, (T, B, Dn), x.dtype)
    L = _lib.lib()
    if saved is None or saved.dtype != torch.float32 or saved.numel() != L.asr_sscan_ckpt_floats(T, B, Dn, N) or \
            not saved.is_contiguous():
        _fail('saved: not what selective_scan_fwd(..., train=True) returned for these shapes')
    if dh_last is not None:
        _par('dh_last', dh_last, (B, Dn, N))
    dev = _device(x, dout, dt, A, Bm, Cm, saved, D, z, dt_bias, h0, lens, dh_last)

    def new(shape, dtype):
        return torch.empty(shape, dtype=dtype, device=x.device)
    ty, f32 = x.dtype, torch.float32
    g = {'x': new((T, B, Dn), ty), 'dt': new((T, B, Dn), ty), 'A': new((Dn, N), f32), 'B': new((T, B, G, N), ty),
         'C': new((T, B, G, N), ty), 'D': new((Dn,), f32) if D is not None else None,
         'z': new((T, B, Dn), ty) if z is not None else None,
         'dt_bias': new((Dn,), f32) if dt_bias is not None else None,
         'h0': new((B, Dn, N), f32) if h0 is not None else None}
    desc = _lib.SscanDesc(*_scan_desc(*a, x, dt, A, Bm, Cm, D, z, dt_bias, h0, lens, softplus, reverse),
                          None, 0, 0, None, saved.data_ptr(), dout.data_ptr(), dout.stride(0), dout.stride(1), _p(dh_last),
                          _p(g['x']), _p(g['dt']), _p(g['z']), _p(g['B']), _p(g['C']), _p(g['A']), _p(g['D']),
                          _p(g['dt_bias']), _p(g['h0']))
    with _On(dev) as st:
        need = L.asr_sscan_ws_bytes(T, B, Dn, N, G, 1)
        ws = torch.empty(need, dtype=torch.uint8, device=x.device)
        check(L.asr_sscan_bwd(C.byref(desc), _p(ws), need, st), 'asr_sscan_bwd')
    return g


def selective_scan_step(h, x, dt, A, Bm, Cm, D=None, z=None, dt_bias=None, softplus=True):
    """One frame of selective_scan_fwd: h (B, D, N) moves on in place; x, dt, z (B, D); Bm, Cm (B, G, N).  -> out (B, D)."""
    if x.dim() != 2:
        _fail('x: expected (B, D), got %d axes' % x.dim())
    B, Dn = x.shape
    if A.dim() != 2 or not 1 <= A.shape[1] <= MAX_STATES:
        _fail('A: expected (D, N) with 1 <= N <= %d, got %s' % (MAX_STATES, tuple(A.shape)))
    N = A.shape[1]
    if Bm.dim() != 3:
        _fail('Bm: expected (B, G, N), got %d axes' % Bm.dim())
    G = Bm.shape[1]
    if Dn < 1 or G < 1 or Dn % G:
        _fail('Bm: %d groups do not divide %d channels' % (G, Dn))
    kind = _type('x', x)
    ty = x.dtype
    _act('x', x, (B, Dn), ty)
    _act('dt', dt, (B, Dn), ty)
    _par('A', A, (Dn, N))
    _act('Bm', Bm, (B, G, N), ty)
    _act('Cm', Cm, (B, G, N), ty)
    if z is not None:
        _act('z', z, (B, Dn), ty)
    if D is not None:
        _par('D', D, (Dn,))
    if dt_bias is not None:
        _par('dt_bias', dt_bias, (Dn,))
    _par('h', h, (B, Dn, N))
    dev = _device(x, h, dt, A, Bm, Cm, D, z, dt_bias)
    out = torch.empty((B, Dn), dtype=ty, device=x.device)
    with _On(dev) as st:
        check(_lib.lib().asr_sscan_step(kind, B, Dn, N, G, h.data_ptr(), x.data_ptr(), x.stride(0), dt.data_ptr(),
                                        dt.stride(0), A.data_ptr(), Bm.data_ptr(), Bm.stride(0), Bm.stride(1),
                                        Cm.data_ptr(), Cm.stride(0), Cm.stride(1), _p(D), _p(z),
                                        z.stride(0) if z is not None else 0, _p(dt_bias), int(softplus), out.data_ptr(),
                                        Dn, st), 'asr_sscan_step')
    return out


# ---------------------------------------------------------------------------------------------- norm
def add_rms_norm_fwd(x, w, residual=None, eps=1e-6):
    """r = x + residual,  y = r / sqrt(mean(r^2) + eps) * w over rows; x, residual (rows, n) with unit column stride, w (n,).
    -> (y, r in the type of x (x itself without a residual), 1 / sqrt(...) of every row for the backward pass)."""
    if x.dim() != 2:
        _fail('x: expected (rows, n), got %d axes' % x.dim())
    rows, n = x.shape
    if n < 1:
        _fail('x: no columns')
    kind = _type('x', x)
    _act('x', x, (rows, n), x.dtype)
    _par('w', w, (n,))
    if residual is not None:
        _act('residual', residual, (rows, n), x.dtype)
    if not eps >= 0:
        _fail('eps: %r is negative' % (eps,))
    dev = _device(x, w, residual)
    y = torch.empty((rows, n), dtype=x.dtype, device=x.device)
    r = torch.empty((rows, n), dtype=x.dtype, device=x.device) if residual is not None else None
    rstd = torch.empty((rows,), dtype=torch.float32, device=x.device)
    with _On(dev) as st:
        check(_lib.lib().asr_rms_norm_fwd(kind, x.data_ptr(), x.stride(0), _p(residual),
                                          residual.stride(0) if residual is not None else 0, w.data_ptr(), rows, n, eps,
                                          y.data_ptr(), _p(r), rstd.data_ptr(), st), 'asr_rms_norm_fwd')
    return y, (x if r is None else r), rstd


def add_rms_norm_bwd(dy, x, w, rstd, residual=None, dres=None):
    """Gradients of add_rms_norm_fwd(x, w, residual): dy (rows, n) of y, dres (rows, n) of r (None: r went nowhere else),
    rstd as the forward call returned it.  -> (dr, dw); dr is the gradient of x and of the residual alike."""
    if x.dim() != 2:
        _fail('x: expected (rows, n), got %d axes' % x.dim())
    rows, n = x.shape
    if n < 1:
        _fail('x: no columns')
    kind = _type('x', x)
    _act('x', x, (rows, n), x.dtype)
    _act('dy', dy, (rows, n), x.dtype)
    _par('w', w, (n,))
    _par('rstd', rstd, (rows,))
    if residual is not None:
        _act('residual', residual, (rows, n), x.dtype)
    if dres is not None:
        _act('dres', dres, (rows, n), x.dtype)
    dev = _device(x, dy, w, rstd, residual, dres)
    dx = torch.empty((rows, n), dtype=x.dtype, device=x.device)
    dw = torch.empty((n,), dtype=torch.float32, device=x.device)
    L = _lib.lib()
    with _On(dev) as st:
        ws = torch.empty(L.asr_rms_norm_bwd_ws_bytes(rows, n), dtype=torch.uint8, device=x.device)
        check(L.asr_rms_norm_bwd(kind, dy.data_ptr(), dy.stride(0), x.data_ptr(), x.stride(0), _p(residual),
                                 residual.stride(0) if residual is not None else 0, w.data_ptr(), rstd.data_ptr(),
                                 _p(dres), dres.stride(0) if dres is not None else 0, rows, n, dx.data_ptr(), dw.data_ptr(),
                                 _p(ws), ws.numel(), st), 'asr_rms_norm_bwd')
    return dx, dw


# ---------------------------------------------------------------------------------------------- gradients in a list
def clip_list(tensors, max_norm, eps=1e-7):
    """-> ([t * clip(norm, 0, max_norm) / (eps + norm) for t in tensors], norm (1,)), norm the root of the sum of all squares:
    libs/lasagne_libs/updates.py:845-855 for gradients that do not lie in one buffer.  float32, bfloat16 and float16 tensors of
    any shape may be mixed; the multiplier stays on the device."""
    tensors = list(tensors)
    if not tensors:
        _fail('tensors: none given')
    if not max_norm >= 0 or not eps >= 0:
        _fail('max_norm %r and eps %r must not be negative' % (max_norm, eps))
    kinds = [_type('tensors[%d]' % i, t) for i, t in enumerate(tensors)]
    dev = _device(*tensors)
    n = len(tensors)
    src = [t if t.is_contiguous() else t.contiguous() for t in tensors]
    out = [torch.empty(t.shape, dtype=t.dtype, device=t.device) for t in src]
    norm = torch.empty((1,), dtype=torch.float32, device=tensors[0].device)
    sizes = (C.c_longlong * n)(*[t.numel() for t in src])
    L = _lib.lib()
    with _On(dev) as st:
        ws = torch.empty(L.asr_clip_list_ws_bytes(n, sizes), dtype=torch.uint8, device=norm.device)
        check(L.asr_clip_list(n, (C.c_int * n)(*kinds), (C.c_void_p * n)(*[t.data_ptr() for t in src]),
                              (C.c_void_p * n)(*[t.data_ptr() for t in out]), sizes, max_norm, eps, norm.data_ptr(),
                              ws.data_ptr(), ws.numel(), st), 'asr_clip_list')
    return out, norm
