"""The kernels that ordinary sizes of the state-space layer's operators run on, against the float64 forms: the scan where a
group's channels are a multiple of 64 and rows are long enough for tiles of valid frames alone, the convolution at its full width
with an odd or a large number of taps, lists whose results go past the caches.  Tolerances as in test_gpu_ssm."""
import pytest
import torch

import ref_ssm as R
from test_gpu_ssm import CONV, SCAN, clean, gen, rn, run_scan, test_conv as check_conv

pytestmark = pytest.mark.gpu

WIDE_SCAN = [  # T, B, D, N, G, type, layout, lens, reverse, options kept
    # one pass over a row of full tiles and a last one that is not (fewer than eight tiles are not cut into chunks)
    (100, 2, 64, 16, 1, 'f32', 'c', [100, 61], False, 'D z dt_bias h0'),
    (112, 2, 128, 16, 1, 'bf16', 'half', [112, 96], True, 'D z dt_bias h0'),
    (121, 1, 128, 16, 2, 'f16', 'bt', None, False, 'D z dt_bias h0'),
    (100, 2, 128, 8, 1, 'f32', 'c', [100, 64], True, 'D z dt_bias h0'),
    (90, 1, 64, 4, 1, 'bf16', 'c', None, False, 'z dt_bias'),
    (90, 2, 64, 24, 1, 'f32', 'half', [90, 33], False, 'D z dt_bias h0'),
    (75, 1, 128, 32, 2, 'bf16', 'c', None, True, 'D z dt_bias h0'),
    (80, 2, 64, 64, 1, 'f32', 'c', [80, 77], False, 'D z dt_bias h0'),
    (70, 1, 64, 40, 1, 'f16', 'c', None, True, 'D dt_bias h0'),
    # time in chunks
    (330, 2, 64, 16, 1, 'f32', 'c', [330, 305], False, 'D z dt_bias h0'),
    (330, 2, 128, 16, 1, 'bf16', 'half', [330, 129], True, 'D z dt_bias h0'),
    (320, 1, 64, 16, 1, 'f16', 'c', None, False, 'D z dt_bias h0'),
    (300, 2, 128, 8, 2, 'bf16', 'c', [300, 14], False, 'D z dt_bias h0'),
    (300, 1, 64, 24, 1, 'f32', 'bt', None, True, 'D z dt_bias h0'),
    (260, 2, 64, 32, 1, 'f16', 'c', [260, 177], False, 'D z dt_bias h0'),
    (260, 1, 64, 64, 1, 'f32', 'c', [259], True, 'D z dt_bias h0'),
    (300, 1, 70, 24, 1, 'f32', 'c', None, False, 'D z dt_bias h0'),
]
assert not set(map(str, WIDE_SCAN)) & set(map(str, SCAN))


@pytest.mark.parametrize('case', WIDE_SCAN, ids=lambda c: '-'.join(str(v) for v in c).replace(' ', ''))
def test_scan_of_whole_tiles(case):
    T, B, D, N, G, ty, lay, lens, rev, keep = case
    a, opt, kw, (out, h, gr), (ra, rop, ro, rh), (do, dh, ln) = run_scan(case)
    steps = 8 * T + 2 * N + 32
    R.close(out, ro, steps, 'out')
    R.close(h, rh, steps, 'h')
    ((ro * clean(do, ln)).sum() + (rh * R.leaf(dh, False)).sum()).backward()
    names = dict(x=ra['x'], dt=ra['dt'], A=ra['A'], B=ra['Bm'], C=ra['Cm'], D=rop['D'], z=rop['z'], dt_bias=rop['dt_bias'],
                 h0=rop['h0'])
    for k, v in names.items():
        assert (gr[k] is None) == (v is None), k
        if v is not None:
            R.close(gr[k], v.grad, 4 * steps + (B * T if k in ('A', 'D', 'dt_bias') else D if k in ('B', 'C') else 0), 'd' + k)


WIDE_CONV = [  # T, B, D, K, type, layout, lens, reverse, state, bias, act
    (90, 2, 264, 5, 'bf16', 'half', [90, 31], False, True, True, 'silu'),
    (70, 2, 200, 5, 'f32', 'c', [70, 4], True, True, True, 'silu'),
    (77, 2, 256, 7, 'bf16', 'c', [77, 50], True, True, True, 'silu'),
    (100, 1, 201, 7, 'f32', 'odd', None, False, True, True, None),
    (85, 2, 320, 6, 'bf16', 'half', [85, 6], False, True, True, 'silu'),
    (85, 1, 133, 6, 'f16', 'c', None, True, True, True, 'silu'),
    (99, 2, 259, 7, 'f16', 'bt', [99, 7], False, True, True, 'silu'),
    (130, 2, 256, 8, 'bf16', 'c', [130, 64], False, True, True, 'silu'),
]
assert not set(map(str, WIDE_CONV)) & set(map(str, CONV))


@pytest.mark.parametrize('case', WIDE_CONV, ids=lambda c: '-'.join(str(v) for v in c).replace(' ', ''))
def test_conv_at_full_width(case):
    check_conv(case)


def test_list_whose_results_go_past_the_caches():
    """76 MB in three types, sizes off the 16-byte grid; new tensors, and in place through the C entry"""
    import ctypes as C
    from asr_amd import _lib, ops
    g = gen(71)
    sizes = [(12_000_001, torch.float32), (7, torch.float32), (8_000_003, torch.bfloat16), (33, torch.bfloat16),
             (6_000_001, torch.float16), (1, torch.float16)]
    ts = [rn(g, n, dtype=t, scale=0.05) for n, t in sizes]
    assert sum(t.numel() * t.element_size() for t in ts) >= 64 << 20
    ref, rnorm = R.clip([R.leaf(t, False) for t in ts], 1.0, 1e-7)
    keep = [t.clone() for t in ts]
    got, norm = ops.clip_list(ts, 1.0)
    R.close(norm, rnorm.reshape(1), 2, 'norm')
    for i, (u, v) in enumerate(zip(got, ref)):
        R.close(u, v, 8, 'tensor %d' % i)
    for u, v in zip(keep, ts):
        assert torch.equal(u, v)
    n = len(ts)
    p = (C.c_void_p * n)(*[t.data_ptr() for t in ts])
    c = (C.c_longlong * n)(*[t.numel() for t in ts])
    L = _lib.lib()
    nt = torch.empty(1, device='cuda')
    ws = torch.empty(L.asr_clip_list_ws_bytes(n, c), dtype=torch.uint8, device='cuda')
    kinds = (C.c_int * n)(*[{torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}[t.dtype] for t in ts])
    assert L.asr_clip_list(n, kinds, p, p, c, 1.0, 1e-7, nt.data_ptr(), ws.data_ptr(), ws.numel(),
                           torch.cuda.current_stream().cuda_stream) == 0
    assert torch.equal(nt, norm) and all(torch.equal(u, v) for u, v in zip(ts, got))
