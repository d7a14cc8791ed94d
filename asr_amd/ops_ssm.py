"""The operators of a selective state-space layer: short causal convolution over time, selective scan, root-mean-square norm
with the residual's addition, and the global norm over a list of gradients.  Wrappers over the C-ABI (include/asr_amd.h)
like asr_amd.ops, which re-exports them; the reference has no such layer (its recurrences are LSTMs), so no file of it is cited.

Shapes.  Sequences are time-major (T, B, channels) with unit channel stride and any (t, b) strides, in float32, bfloat16 or
float16, all activations of a call in one type.  Parameters, scan states and parameter gradients are float32.  `lens` (B,)
int32: frames at and behind lens[b] are padding, whose values are never used (they may be NaN); outputs and gradients there
are zero and the state is what the last valid frame left.  reverse=True walks every row from its last valid frame to the first.

Every call is enqueued on the current stream of the tensors' device and allocates its outputs and its workspace through
torch, so calls on several streams and calls captured into graphs share nothing.  Results do not vary from run to run.
A wrong argument raises ValueError before anything is launched, a size beyond the C entry's limits (include/asr_amd.h) AsrError.
"""
import ctypes as C
import struct

import torch

from . import _lib
from ._lib import check

_DTYPES = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}
MAX_STATES = 64
MAX_TAPS = 8


def _fail(msg):
    raise ValueError(msg)


# the handle and the index alone: torch.cuda.current_stream() makes an object, torch.cuda.current_device() looks for a first use
_stream = getattr(torch._C, '_cuda_getCurrentRawStream', None) or (lambda dev: torch.cuda.current_stream(dev).cuda_stream)
_current = getattr(torch._C, '_cuda_getDevice', None) or torch.cuda.current_device


def _p(t):
    return None if t is None else t.data_ptr()


def _new(t, _row_major=torch.contiguous_format):
    """a contiguous tensor of t's shape and type (None for None)"""
    return None if t is None else torch.empty_like(t, memory_format=_row_major)


def _act(name, t, shape, dtype, dev):
    """an activation: the shape, the call's type, the call's device, unit stride of the last axis; -> its strides"""
    st = t.stride()
    if t.shape != shape or t.dtype is not dtype or t.get_device() != dev or (st[-1] != 1 and shape[-1] > 1):
        if t.shape != shape:
            _fail('%s: shape %s, expected %s' % (name, tuple(t.shape), tuple(shape)))
        if t.dtype is not dtype:
            _fail('%s: %s, expected %s like the other activations' % (name, t.dtype, dtype))
        if t.get_device() == dev:
            _fail('%s: the last axis must have stride 1' % name)
        _fail('%s: on %s, unlike the other tensors' % (name, t.device))
    return st


def _par(name, t, shape, dev, like=None):
    """a parameter or a state: float32 (or the activations' type), contiguous, on the call's device; -> its address"""
    dtype = like or torch.float32
    if t.shape != shape or t.dtype is not dtype or not t.is_contiguous() or t.get_device() != dev:
        if t.shape != shape:
            _fail('%s: shape %s, expected %s' % (name, tuple(t.shape), tuple(shape)))
        if t.dtype is not dtype:
            _fail('%s: %s, expected %s%s' % (name, t.dtype, dtype, ' like x' if like else ''))
        if t.get_device() == dev:
            _fail('%s: must be contiguous, has strides %s' % (name, t.stride()))
        _fail('%s: on %s, unlike the other tensors' % (name, t.device))
    return t.data_ptr()


def _vec(t, n, dev):
    return t.shape == (n,) and t.dtype is torch.float32 and t.is_contiguous() and t.get_device() == dev


def _type(name, t):
    k = _DTYPES.get(t.dtype)
    if k is None:
        _fail('%s: %s, expected float32, bfloat16 or float16' % (name, t.dtype))
    return k


def _gpu(dev):
    """behind all other checks, which need no GPU"""
    if dev < 0:
        _fail('tensors must be on the GPU (there is no CPU path)')


def _call(what, dev, fn, *args):
    """fn(*args, the current stream of device dev), with that device current"""
    if _current() == dev:
        rc = fn(*args, _stream(dev))
    else:
        with torch.cuda.device(dev):
            rc = fn(*args, _stream(dev))
    if rc:
        check(rc, what)


# ---------------------------------------------------------------------------------------------- convolution
def _act_kind(act):
    if act != 'silu' and act is not None:
        _fail("act: 'silu' or None, got %r" % (act,))
    return 1 if act else 0


def _taps(w):
    if w.dim() != 2 or not 2 <= w.shape[1] <= MAX_TAPS:
        _fail('w: expected (D, K) with 2 <= K <= %d, got %s' % (MAX_TAPS, tuple(w.shape)))
    return w.shape[1]


def _lens(lens, B, dev):
    if lens is None:
        return None
    if lens.shape != (B,) or lens.dtype is not torch.int32 or not lens.is_contiguous():
        _fail('lens: expected %d contiguous int32 values' % B)
    if lens.get_device() != dev:
        _fail('lens: on %s, unlike the other tensors' % lens.device)
    return lens.data_ptr()


def _conv_args(x, w, bias, state, lens, act):
    if x.dim() != 3:
        _fail('x: expected (T, B, D), got %d axes' % x.dim())
    T, B, D = x.shape
    K = _taps(w)
    kind = _type('x', x)
    if D < 1:
        _fail('x: no channels')
    dev = x.get_device()
    st = _act('x', x, (T, B, D), x.dtype, dev)
    pw = _par('w', w, (D, K), dev)
    pb = _par('bias', bias, (D,), dev) if bias is not None else None
    ps = _par('state', state, (K - 1, B, D), dev, x.dtype) if state is not None else None
    return kind, T, B, D, K, dev, st, pw, pb, ps, _lens(lens, B, dev), _act_kind(act)


def causal_conv_fwd(x, w, bias=None, state=None, lens=None, act='silu', reverse=False, want_state=False):
    """out[s] = act(bias + sum_k w[:, k] x[s - (K-1) + k]) over the valid frames s of every row; x (T, B, D), w (D, K).
    state (K-1, B, D): the frames in front of the first one (None: zeros).  -> (out, the state behind the last valid frame
    if want_state, else None)."""
    kind, T, B, D, K, dev, st, pw, pb, ps, pl, silu = _conv_args(x, w, bias, state, lens, act)
    _gpu(dev)
    out = _new(x)
    new = torch.empty(K - 1, B, D, dtype=x.dtype, device=x.device) if want_state else None
    _call('asr_conv_fwd', dev, _lib.lib().asr_conv_fwd, kind, T, B, D, K, x.data_ptr(), st[0], st[1], pw, pb, ps, pl, silu,
          int(reverse), out.data_ptr(), B * D, D, _p(new))
    return out, new


def causal_conv_bwd(dout, x, w, bias=None, state=None, lens=None, act='silu', reverse=False, dstate_out=None):
    """Gradients of causal_conv_fwd for the gradient dout of its output (and dstate_out of the state it returned):
    {'x', 'w', 'bias', 'state'}; 'bias' / 'state' are None when there was none."""
    kind, T, B, D, K, dev, st, pw, pb, ps, pl, silu = _conv_args(x, w, bias, state, lens, act)
    so = _act('dout', dout, (T, B, D), x.dtype, dev)
    pd = _par('dstate_out', dstate_out, (K - 1, B, D), dev, x.dtype) if dstate_out is not None else None
    _gpu(dev)
    L = _lib.lib()
    dx = _new(x)
    dwb = torch.empty(D * (K + 1), dtype=torch.float32, device=x.device)
    ds = _new(state)
    need = L.asr_conv_bwd_ws_bytes(T, B, D, K)
    ws = torch.empty(need, dtype=torch.uint8, device=x.device)
    _call('asr_conv_bwd', dev, L.asr_conv_bwd, kind, T, B, D, K, dout.data_ptr(), so[0], so[1], x.data_ptr(), st[0], st[1], pw,
          pb, ps, pl, silu, int(reverse), pd, dx.data_ptr(), dwb.data_ptr(), _p(ds), ws.data_ptr(), need)
    return {'x': dx, 'w': dwb[:D * K].view(D, K), 'bias': dwb[D * K:] if bias is not None else None, 'state': ds}


def causal_conv_step(x, state, w, bias=None, act='silu'):
    """One frame: x (B, D), state (K-1, B, D), which moves on in place.  -> out (B, D).  Equal to causal_conv_fwd over one
    frame."""
    sh, ty, dev, sx, sw = x.shape, x.dtype, x.get_device(), x.stride(), w.shape
    kind = _DTYPES.get(ty)
    # everything in one expression, and name by name where that fails, as in selective_scan_step
    if kind is None or dev < 0 or len(sh) != 2 or len(sw) != 2 or (act != 'silu' and act is not None) or not (
            sw[0] == sh[1] > 0 and 2 <= sw[1] <= MAX_TAPS and state.shape == (sw[1] - 1, sh[0], sh[1]) and state.dtype is ty
            and w.dtype is torch.float32 and sx[1] == 1 and state.is_contiguous() and w.is_contiguous()
            and dev == state.get_device() == w.get_device() and (bias is None or _vec(bias, sh[1], dev))):
        _conv_step_refusal(x, state, w, bias, act)
    out = _new(x)
    _call('asr_conv_step', dev, _lib.lib().asr_conv_step, kind, sh[0], sh[1], sw[1], x.data_ptr(), sx[0], state.data_ptr(),
          w.data_ptr(), _p(bias), 1 if act else 0, out.data_ptr(), sh[1])
    return out


def _conv_step_refusal(x, state, w, bias, act):
    """says what is wrong with a single frame's arguments (and accepts axes of one value with any stride)"""
    if x.dim() != 2:
        _fail('x: expected (B, D), got %d axes' % x.dim())
    B, D = x.shape
    K = _taps(w)
    _type('x', x)
    if D < 1:
        _fail('x: no channels')
    ty, dev = x.dtype, x.get_device()
    _act('x', x, (B, D), ty, dev)
    _par('w', w, (D, K), dev)
    if bias is not None:
        _par('bias', bias, (D,), dev)
    _par('state', state, (K - 1, B, D), dev, ty)
    _act_kind(act)
    _gpu(dev)


# ---------------------------------------------------------------------------------------------- selective scan
def _states(A, Bm, Dn, axes):
    """N, G"""
    if A.dim() != 2 or not 1 <= A.shape[1] <= MAX_STATES:
        _fail('A: expected (D, N) with 1 <= N <= %d, got %s' % (MAX_STATES, tuple(A.shape)))
    if Bm.dim() != axes:
        _fail('Bm: expected %s, got %d axes' % ('(T, B, G, N)' if axes == 4 else '(B, G, N)', Bm.dim()))
    G = Bm.shape[-2]
    if Dn < 1 or G < 1 or Dn % G:
        _fail('Bm: %d groups do not divide %d channels' % (G, Dn))
    return A.shape[1], G


# the descriptor's members in their order: eight ints, then pointers (0 for NULL) and strides
_MEMBERS = struct.Struct('8i%dq' % (len(_lib.SscanDesc._fields_) - 8))


def _desc(*members):
    return C.byref(_lib.SscanDesc.from_buffer_copy(_MEMBERS.pack(*members)))


_FORWARD_ONLY = (0,) * (len(_lib.SscanDesc._fields_) - 35)      # the members behind ckpt


def _a(t):
    return 0 if t is None else t.data_ptr()


def _scan_args(x, dt, A, Bm, Cm, D, z, dt_bias, h0, lens, softplus, reverse):
    """the sizes, the device, and the descriptor's members up to h0"""
    sh, ty, dev = x.shape, x.dtype, x.get_device()
    kind = _DTYPES.get(ty)
    sx, sd, sB, sC = x.stride(), dt.stride(), Bm.stride(), Cm.stride()
    sz = z.stride() if z is not None else sx
    sb, sA = Bm.shape, A.shape
    if kind is None or len(sh) != 3 or len(sb) != 4 or len(sA) != 2 or not (
            sh[2] > 0 and sb[2] > 0 and sh[2] % sb[2] == 0 and dt.shape == sh and Cm.shape == sb and sb[:2] == sh[:2]
            and (z is None or (z.shape == sh and z.dtype is ty and z.get_device() == dev))
            and sA[0] == sh[2] and sA[1] == sb[3] and 1 <= sA[1] <= MAX_STATES
            and dt.dtype is ty and Bm.dtype is ty and Cm.dtype is ty and A.dtype is torch.float32
            and sx[2] == sd[2] == sz[2] == sB[3] == sC[3] == 1 and A.is_contiguous()
            and dev == dt.get_device() == Bm.get_device() == Cm.get_device() == A.get_device()
            and (D is None or _vec(D, sh[2], dev)) and (dt_bias is None or _vec(dt_bias, sh[2], dev))):
        _scan_refusal(x, dt, A, Bm, Cm, D, z, dt_bias)
    T, B, Dn = sh
    N, G = sA[1], sb[2]
    if h0 is not None:
        _par('h0', h0, (B, Dn, N), dev)
    return (T, B, Dn, N, G), dev, (T, B, Dn, N, G, kind, 1 if reverse else 0, 1 if softplus else 0, _lens(lens, B, dev) or 0,
                                   x.data_ptr(), sx[0], sx[1], dt.data_ptr(), sd[0], sd[1], _a(z), sz[0], sz[1], Bm.data_ptr(),
                                   sB[0], sB[1], sB[2], Cm.data_ptr(), sC[0], sC[1], sC[2], A.data_ptr(), _a(D), _a(dt_bias),
                                   _a(h0))


def _scan_refusal(x, dt, A, Bm, Cm, D, z, dt_bias):
    """says what is wrong with a sequence's arguments (and accepts axes of one value with any stride)"""
    if x.dim() != 3:
        _fail('x: expected (T, B, D), got %d axes' % x.dim())
    sh = T, B, Dn = x.shape
    N, G = _states(A, Bm, Dn, 4)
    _type('x', x)
    ty, dev = x.dtype, x.get_device()
    for name, t, shape in (('x', x, sh), ('dt', dt, sh), ('Bm', Bm, (T, B, G, N)), ('Cm', Cm, (T, B, G, N)), ('z', z, sh)):
        if t is not None:
            _act(name, t, shape, ty, dev)
    for name, t, shape in (('A', A, (Dn, N)), ('D', D, (Dn,)), ('dt_bias', dt_bias, (Dn,))):
        if t is not None:
            _par(name, t, shape, dev)


def selective_scan_fwd(x, dt, A, Bm, Cm, D=None, z=None, dt_bias=None, h0=None, lens=None, softplus=True, reverse=False,
                       train=False):
    """h[s] = exp(delta A) h[s-1] + delta x B[s],  y = C[s] h[s] + D x,  out = y silu(z)  (y without z), with
    delta = softplus(dt + dt_bias)  (dt + dt_bias with softplus=False).

    x, dt, z (T, B, D); A (D, N), N <= 64; Bm, Cm (T, B, G, N), shared by the D / G channels of a group; D, dt_bias (D,);
    h0 (B, D, N) (None: zeros).  -> (out (T, B, D), the state behind the last valid frame (B, D, N), what
    selective_scan_bwd needs if train, else None)."""
    (T, B, Dn, N, G), dev, members = _scan_args(x, dt, A, Bm, Cm, D, z, dt_bias, h0, lens, softplus, reverse)
    _gpu(dev)
    L = _lib.lib()
    f32, on = torch.float32, x.device
    out = _new(x)
    h = torch.empty(B, Dn, N, dtype=f32, device=on)
    saved = torch.empty(L.asr_sscan_ckpt_floats(T, B, Dn, N), dtype=f32, device=on) if train else None
    need = L.asr_sscan_ws_bytes(T, B, Dn, N, G, 0)
    ws = torch.empty(need, dtype=torch.uint8, device=on) if need else None
    desc = _desc(*members, out.data_ptr(), B * Dn, Dn, h.data_ptr(), _a(saved), *_FORWARD_ONLY)
    _call('asr_sscan_fwd', dev, L.asr_sscan_fwd, desc, _p(ws), need)
    return out, h, saved


def selective_scan_bwd(dout, x, dt, A, Bm, Cm, saved, D=None, z=None, dt_bias=None, h0=None, lens=None, softplus=True,
                       reverse=False, dh_last=None):
    """Gradients of selective_scan_fwd(..., train=True) called with the same arguments, for the gradient dout of its output
    (and dh_last of the state it returned): {'x', 'dt', 'A', 'B', 'C', 'D', 'z', 'dt_bias', 'h0'}, None where the argument
    was.  `saved` is what the forward call returned."""
    (T, B, Dn, N, G), dev, members = _scan_args(x, dt, A, Bm, Cm, D, z, dt_bias, h0, lens, softplus, reverse)
    so = _act('dout', dout, (T, B, Dn), x.dtype, dev)
    L = _lib.lib()
    if saved is None or saved.shape != (L.asr_sscan_ckpt_floats(T, B, Dn, N),):
        _fail('saved: not what selective_scan_fwd(..., train=True) returned for these shapes')
    ps = _par('saved', saved, saved.shape, dev)
    ph = _par('dh_last', dh_last, (B, Dn, N), dev) if dh_last is not None else 0
    _gpu(dev)
    on = x.device
    g = {'x': _new(x), 'dt': _new(dt), 'A': _new(A), 'B': _new(Bm), 'C': _new(Cm), 'D': _new(D), 'z': _new(z),
         'dt_bias': _new(dt_bias), 'h0': _new(h0)}
    need = L.asr_sscan_ws_bytes(T, B, Dn, N, G, 1)
    ws = torch.empty(need, dtype=torch.uint8, device=on)
    desc = _desc(*members, 0, 0, 0, 0, ps, dout.data_ptr(), so[0], so[1], ph, g['x'].data_ptr(), g['dt'].data_ptr(), _a(g['z']),
                 g['B'].data_ptr(), g['C'].data_ptr(), g['A'].data_ptr(), _a(g['D']), _a(g['dt_bias']), _a(g['h0']))
    _call('asr_sscan_bwd', dev, L.asr_sscan_bwd, desc, ws.data_ptr(), need)
    return g


def selective_scan_step(h, x, dt, A, Bm, Cm, D=None, z=None, dt_bias=None, softplus=True):
    """One frame of selective_scan_fwd: h (B, D, N) moves on in place; x, dt, z (B, D); Bm, Cm (B, G, N).  -> out (B, D)."""
    sh, ty, dev = x.shape, x.dtype, x.get_device()
    kind = _DTYPES.get(ty)
    sx, sd, sB, sC = x.stride(), dt.stride(), Bm.stride(), Cm.stride()
    sz = z.stride() if z is not None else sx
    sb, sA = Bm.shape, A.shape
    # a stream's frame is a few microseconds of work: everything is looked at in one expression, and name by name where that fails
    if kind is None or dev < 0 or len(sh) != 2 or len(sb) != 3 or len(sA) != 2 or not (
            sh[1] > 0 and sb[1] > 0 and sh[1] % sb[1] == 0 and dt.shape == sh and Cm.shape == sb and sb[0] == sh[0]
            and (z is None or (z.shape == sh and z.dtype is ty and z.get_device() == dev))
            and sA[0] == sh[1] and sA[1] == sb[2] and 1 <= sA[1] <= MAX_STATES and h.shape == (sh[0], sh[1], sA[1])
            and dt.dtype is ty and Bm.dtype is ty and Cm.dtype is ty and A.dtype is h.dtype is torch.float32
            and sx[1] == sd[1] == sz[1] == sB[2] == sC[2] == 1 and A.is_contiguous() and h.is_contiguous()
            and dev == dt.get_device() == Bm.get_device() == Cm.get_device() == A.get_device() == h.get_device()
            and (D is None or _vec(D, sh[1], dev)) and (dt_bias is None or _vec(dt_bias, sh[1], dev))):
        _step_refusal(h, x, dt, A, Bm, Cm, D, z, dt_bias)
    out = _new(x)
    _call('asr_sscan_step', dev, _lib.lib().asr_sscan_step, kind, sh[0], sh[1], sA[1], sb[1], h.data_ptr(), x.data_ptr(), sx[0],
          dt.data_ptr(), sd[0], A.data_ptr(), Bm.data_ptr(), sB[0], sB[1], Cm.data_ptr(), sC[0], sC[1], _p(D), _p(z), sz[0],
          _p(dt_bias), 1 if softplus else 0, out.data_ptr(), sh[1])
    return out


def _step_refusal(h, x, dt, A, Bm, Cm, D, z, dt_bias):
    """says what is wrong with a single frame's arguments (and accepts axes of one value with any stride)"""
    if x.dim() != 2:
        _fail('x: expected (B, D), got %d axes' % x.dim())
    sh = B, Dn = x.shape
    N, G = _states(A, Bm, Dn, 3)
    _type('x', x)
    ty, dev = x.dtype, x.get_device()
    for name, t, shape in (('x', x, sh), ('dt', dt, sh), ('Bm', Bm, (B, G, N)), ('Cm', Cm, (B, G, N)), ('z', z, sh)):
        if t is not None:
            _act(name, t, shape, ty, dev)
    for name, t, shape in (('A', A, (Dn, N)), ('D', D, (Dn,)), ('dt_bias', dt_bias, (Dn,)), ('h', h, (B, Dn, N))):
        if t is not None:
            _par(name, t, shape, dev)
    _gpu(dev)


# ---------------------------------------------------------------------------------------------- norm
def _rows(x):
    if x.dim() != 2:
        _fail('x: expected (rows, n), got %d axes' % x.dim())
    if x.shape[1] < 1:
        _fail('x: no columns')
    return x.shape, _type('x', x), x.dtype, x.get_device()


def add_rms_norm_fwd(x, w, residual=None, eps=1e-6):
    """r = x + residual,  y = r / sqrt(mean(r^2) + eps) * w over rows; x, residual (rows, n) with unit column stride, w (n,).
    -> (y, r in the type of x (x itself without a residual), 1 / sqrt(...) of every row for the backward pass)."""
    sh, kind, ty, dev = _rows(x)
    rows, n = sh
    sx = _act('x', x, sh, ty, dev)
    pw = _par('w', w, (n,), dev)
    pr, sr = (residual.data_ptr(), _act('residual', residual, sh, ty, dev)[0]) if residual is not None else (None, 0)
    if not eps >= 0:
        _fail('eps: %r is negative' % (eps,))
    _gpu(dev)
    y = _new(x)
    r = _new(residual)
    rstd = torch.empty(rows, dtype=torch.float32, device=x.device)
    _call('asr_rms_norm_fwd', dev, _lib.lib().asr_rms_norm_fwd, kind, x.data_ptr(), sx[0], pr, sr, pw, rows, n, eps,
          y.data_ptr(), _p(r), rstd.data_ptr())
    return y, (x if r is None else r), rstd


def add_rms_norm_bwd(dy, x, w, rstd, residual=None, dres=None):
    """Gradients of add_rms_norm_fwd(x, w, residual): dy (rows, n) of y, dres (rows, n) of r (None: r went nowhere else),
    rstd as the forward call returned it.  -> (dr, dw); dr is the gradient of x and of the residual alike."""
    sh, kind, ty, dev = _rows(x)
    rows, n = sh
    sx = _act('x', x, sh, ty, dev)
    sy = _act('dy', dy, sh, ty, dev)
    pw = _par('w', w, (n,), dev)
    ps = _par('rstd', rstd, (rows,), dev)
    pr, sr = (residual.data_ptr(), _act('residual', residual, sh, ty, dev)[0]) if residual is not None else (None, 0)
    pd, sd = (dres.data_ptr(), _act('dres', dres, sh, ty, dev)[0]) if dres is not None else (None, 0)
    _gpu(dev)
    L = _lib.lib()
    dx, dw = _new(x), _new(w)
    need = L.asr_rms_norm_bwd_ws_bytes(rows, n)
    ws = torch.empty(need, dtype=torch.uint8, device=x.device)
    _call('asr_rms_norm_bwd', dev, L.asr_rms_norm_bwd, kind, dy.data_ptr(), sy[0], x.data_ptr(), sx[0], pr, sr, pw, ps, pd, sd,
          rows, n, dx.data_ptr(), dw.data_ptr(), ws.data_ptr(), need)
    return dx, dw


# ---------------------------------------------------------------------------------------------- gradients in a list
def clip_list(tensors, max_norm, eps=1e-7):
    """-> ([t * clip(norm, 0, max_norm) / (eps + norm) for t in tensors], norm (1,)), norm the root of the sum of all squares:
    libs/lasagne_libs/updates.py:845-855 for gradients that do not lie in one buffer.  float32, bfloat16 and float16 tensors of
    any shape may be mixed; the multiplier stays on the device.  The results of one type share one buffer."""
    tensors = list(tensors)
    if not tensors:
        _fail('tensors: none given')
    if not max_norm >= 0 or not eps >= 0:
        _fail('max_norm %r and eps %r must not be negative' % (max_norm, eps))
    kinds = [_DTYPES.get(t.dtype) for t in tensors]
    dev = tensors[0].get_device()
    if None in kinds or [t.get_device() for t in tensors].count(dev) < len(tensors):
        for i, t in enumerate(tensors):
            _type('tensors[%d]' % i, t)
            if t.get_device() != dev:
                _fail('tensors[%d]: on %s, unlike the others' % (i, t.device))
    try:
        whole = [t.is_contiguous() for t in tensors]
    except RuntimeError:                               # compressed sparse layouts have no answer
        whole = [False]
    if not all(whole):
        for i, t in enumerate(tensors):
            if t.layout is not torch.strided:
                _fail('tensors[%d]: %s, expected a strided tensor' % (i, t.layout))
    _gpu(dev)
    n, on = len(tensors), tensors[0].device
    src = tensors if all(whole) else [t if c else t.contiguous() for t, c in zip(tensors, whole)]
    sizes = [t.numel() for t in src]
    out, dst = [None] * n, [0] * n
    for dtype, kind in _DTYPES.items():
        mine = [i for i in range(n) if kinds[i] == kind]
        if not mine:
            continue
        parts = [sizes[i] for i in mine]
        flat = torch.empty(sum(parts), dtype=dtype, device=on)
        at, e = flat.data_ptr(), flat.element_size()
        for i, view in zip(mine, flat.split(parts)):
            out[i], dst[i] = (view if src[i].dim() == 1 else view.view(src[i].shape)), at
            at += sizes[i] * e
    L = _lib.lib()
    csizes = (C.c_longlong * n)(*sizes)
    need = L.asr_clip_list_ws_bytes(n, csizes)
    norm = torch.empty(1, dtype=torch.float32, device=on)
    ws = torch.empty(need, dtype=torch.uint8, device=on)
    _call('asr_clip_list', dev, L.asr_clip_list, n, (C.c_int * n)(*kinds), (C.c_void_p * n)(*[t.data_ptr() for t in src]),
          (C.c_void_p * n)(*dst), csizes, max_norm, eps, norm.data_ptr(), ws.data_ptr(), need)
    return out, norm
