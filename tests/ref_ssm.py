"""Plain float64 forms of the state-space layer's operators on the CPU, frame by frame and differentiable by autograd, and the
tolerances their float32 kernels are held to."""
import torch

F64 = torch.float64
U = 2.0 ** -24                       # half a step of float32
HALF = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}


def frames(T, n, reverse):
    """valid frames of a row in walking order"""
    n = max(0, min(T, n))
    return list(range(n - 1, -1, -1)) if reverse else list(range(n))


def conv(x, w, bias=None, state=None, lens=None, act='silu', reverse=False):
    """-> out (T,B,D), state (K-1,B,D)"""
    T, B, D = x.shape
    K = w.shape[1]
    rows, ends = [], []
    for b in range(B):
        fs = frames(T, T if lens is None else int(lens[b]), reverse)
        past = [state[k, b] if state is not None else torch.zeros(D, dtype=F64) for k in range(K - 1)]
        seq = past + [x[f, b] for f in fs]
        out = [torch.zeros(D, dtype=F64)] * T
        for i, f in enumerate(fs):
            pre = sum(w[:, k] * seq[i + k] for k in range(K))
            if bias is not None:
                pre = pre + bias
            out[f] = pre * torch.sigmoid(pre) if act == 'silu' else pre
        rows.append(torch.stack(out) if T else torch.zeros(0, D, dtype=F64))
        ends.append(torch.stack(seq[len(seq) - (K - 1):]))
    return torch.stack(rows, 1), torch.stack(ends, 1)


def scan(x, dt, A, Bm, Cm, D=None, z=None, dt_bias=None, h0=None, lens=None, softplus=True, reverse=False):
    """-> out (T,B,D), h (B,D,N)"""
    T, B, Dn = x.shape
    N, G = A.shape[1], Bm.shape[2]
    rep = Dn // G
    rows, ends = [], []
    for b in range(B):
        h = h0[b] if h0 is not None else torch.zeros(Dn, N, dtype=F64)
        out = [torch.zeros(Dn, dtype=F64)] * T
        for f in frames(T, T if lens is None else int(lens[b]), reverse):
            v = dt[f, b] + dt_bias if dt_bias is not None else dt[f, b]
            de = torch.logaddexp(v, torch.zeros_like(v)) if softplus else v
            Bf = Bm[f, b].repeat_interleave(rep, 0)
            Cf = Cm[f, b].repeat_interleave(rep, 0)
            h = torch.exp(de[:, None] * A) * h + (de * x[f, b])[:, None] * Bf
            y = (h * Cf).sum(1)
            if D is not None:
                y = y + D * x[f, b]
            if z is not None:
                y = y * z[f, b] * torch.sigmoid(z[f, b])
            out[f] = y
        rows.append(torch.stack(out) if T else torch.zeros(0, Dn, dtype=F64))
        ends.append(h)
    return torch.stack(rows, 1), torch.stack(ends)


def rms(x, w, residual=None, eps=1e-6):
    r = x + residual if residual is not None else x
    return r / torch.sqrt((r * r).mean(-1, keepdim=True) + eps) * w, r


def clip(ts, max_norm, eps):
    norm = torch.sqrt(sum((t * t).sum() for t in ts))
    m = torch.clamp(norm, 0.0, max_norm) / (eps + norm)
    return [t * m for t in ts], norm


def leaf(t, grad=True):
    """the float64 copy of a GPU tensor; padding that holds no number becomes zero (it is never used)"""
    if t is None:
        return None
    v = t.detach().cpu().to(F64)
    return v.requires_grad_() if grad else v


def close(got, ref, steps, name, scale=None):
    """got against the float64 value ref: `steps` roundings of float32 at the tensor's largest value, and the one rounding of
    the stored type at each value (below float16's normal range its spacing, 2^-24, halved).  scale: the size of the terms
    that the roundings act on where they cancel in the result."""
    assert got is not None and tuple(got.shape) == tuple(ref.shape), (name, None if got is None else got.shape, ref.shape)
    if got.numel() == 0:
        return
    g, r = got.detach().cpu().to(F64), ref.detach()
    assert torch.isfinite(g).all(), '%s: not finite' % name
    scale = float(r.abs().max()) if scale is None else scale
    tol = steps * U * scale + r.abs() * HALF[got.dtype] * (1.0 + 2 * steps * U)
    if got.dtype == torch.float16:
        tol = tol + 2.0 ** -25
    worst = float(((g - r).abs() - tol).max())
    assert worst <= 0, '%s: %.3g beyond the tolerance (scale %.3g, max error %.3g)' % (
        name, worst, scale, float((g - r).abs().max()))
