"""When asr_amd.build compiles again: the library must not stay behind what it was made from."""
import os

import pytest

from asr_amd import build

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


class Compiles(Exception):
    pass


@pytest.mark.parametrize('path', ['asr_amd/csrc/sscan_bwd.hip', 'asr_amd/csrc/sscan.h', 'include/asr_amd.h', 'asr_amd/build.py', None])
def test_a_newer_source_header_or_flag_compiles_again(path, tmp_path, monkeypatch):
    """nothing is compiled: the first compiler call raises"""
    newer = os.path.join(ROOT, path) if path else None
    assert newer is None or os.path.exists(newer)
    lib = tmp_path / 'lib.so'
    lib.write_bytes(b'')

    def compiler(*args, **kw):
        raise Compiles()
    monkeypatch.setattr(build, 'LIB', str(lib))
    monkeypatch.setattr(build.subprocess, 'Popen', compiler)
    monkeypatch.setattr(build.os.path, 'getmtime', lambda p: 2.0 if newer and os.path.realpath(p) == os.path.realpath(newer) else 1.0)
    if newer:
        with pytest.raises(Compiles):
            build.build()
    else:
        assert build.build() == str(lib)
