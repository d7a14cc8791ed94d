"""Builds the C-ABI shared library asr_amd/libasr_amd.so from the HIP sources for gfx950.
hipcc cross-compiles without a GPU.  Run:  python -m asr_amd.build"""
import os
import subprocess
import sys

HERE = os.path.dirname(os.path.abspath(__file__))
CSRC = os.path.join(HERE, 'csrc')
LIB = os.path.join(HERE, 'libasr_amd.so')
HEADER = os.path.join(os.path.dirname(HERE), 'include', 'asr_amd.h')


# Per-file compiler flags.  gemm.hip: hipcc's SLP vectoriser turns the operand split's residual subtractions and the
# K-tile joins into v_pk_add_f32 / v_pk_fma_f32, which cost more issue time beside MFMAs than the scalar forms they
# replace (MI355X_MICROARCH.md, 'price of one filler beside MFMAs'): without it the split GEMMs run 4-6 % faster with
# bit-identical results (profiles/r03_gemm_no_slp.txt).
# The state-space layer's files are built without packed fp32 instructions: builds with some of their forms have shown differing
# bits, for a reason that is not established (tests/test_isa_guard.py); the host pass warns that it does not know the feature,
# which is harmless.
_NO_PACKED_FP32 = ['-Xclang', '-target-feature', '-Xclang', '-packed-fp32-ops']
FILE_FLAGS = {'gemm.hip': ['-fno-slp-vectorize']}
FILE_FLAGS.update({f: _NO_PACKED_FP32 for f in ('conv.hip', 'sscan_fwd.hip', 'sscan_bwd.hip', 'rmsnorm.hip',
                                                'gradclip.hip')})
# sscan_bwd.hip: with more than 16 states a lane's adjoints and rates of all groups of states are indexed arrays that belong in
# scratch; promoted to registers they push a tile's states out (64 states: 210 spilled registers, T 512, B 16, D 2048, bf16 1314 us
# instead of 1145).
FILE_FLAGS['sscan_bwd.hip'] = _NO_PACKED_FP32 + ['-mllvm', '-disable-promote-alloca-to-vector=1']


def file_flags(src):
    return FILE_FLAGS.get(os.path.basename(src), [])


def sources():
    return sorted(os.path.join(CSRC, f) for f in os.listdir(CSRC) if f.endswith('.hip'))


def build(force=False, verbose=True, stamps=False):
    """stamps=True builds the diagnostic libasr_amd_stamps.so (in-kernel phase stamps; select it with
    ASR_AMD_LIB=...); never used by tests or bench numbers."""
    global LIB
    srcs = sources()
    if stamps:
        return _build_stamps(srcs)
    # the kernels take descriptors from the public header, and the flags of this file
    deps = srcs + [os.path.join(CSRC, f) for f in os.listdir(CSRC) if f.endswith('.h')] + [HEADER, os.path.abspath(__file__)]
    if not force and os.path.exists(LIB) and all(os.path.getmtime(LIB) >= os.path.getmtime(s) for s in deps):
        return LIB
    objs = []
    procs = []
    for s in srcs:
        o = s[:-4] + '.o'
        objs.append(o)
        cmd = ['hipcc', '--offload-arch=gfx950', '-O3', '-fPIC', '-std=c++17', '-Wno-unused-value'] + file_flags(s) + \
              ['-c', s, '-o', o]
        procs.append((cmd, subprocess.Popen(cmd, stdout=subprocess.PIPE, stderr=subprocess.STDOUT)))
    for cmd, p in procs:
        out, _ = p.communicate()
        if p.returncode != 0:
            sys.stderr.write(out.decode())
            raise RuntimeError('hipcc failed: ' + ' '.join(cmd))
        if verbose and out.strip():
            sys.stderr.write(out.decode())
    cmd = ['hipcc', '--offload-arch=gfx950', '-shared', '-fPIC', '-o', LIB] + objs
    subprocess.check_call(cmd)
    return LIB


def _build_stamps(srcs):
    lib = os.path.join(HERE, 'libasr_amd_stamps.so')
    cmd = ['hipcc', '--offload-arch=gfx950', '-O3', '-fPIC', '-std=c++17', '-Wno-unused-value',
           '-DSCAN_STAMPS', '-shared', '-o', lib] + srcs
    subprocess.check_call(cmd)
    return lib


if __name__ == '__main__':
    if '--stamps' in sys.argv:
        print(build(stamps=True))
        sys.exit(0)
    print(build(force='--force' in sys.argv))
