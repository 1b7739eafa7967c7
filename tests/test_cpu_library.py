"""The library as it was built, disassembled (its gfx950 code, built here from csrc/): no packed f32
instruction in any file's kernels, whatever the compiler made of their arithmetic."""
import glob
import os
import re
import shutil
import subprocess

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
OBJDUMP = '/opt/rocm/llvm/bin/llvm-objdump'


def test_no_packed_f32_in_the_library(tmp_path):
    from gluonnlp_amd import _lib
    if not os.path.exists(OBJDUMP):
        pytest.skip('llvm-objdump not available')
    _lib.load()
    shutil.copy(_lib.LIB_PATH, str(tmp_path / 'lib.so'))
    subprocess.run([OBJDUMP, '--offloading', 'lib.so'], cwd=str(tmp_path), check=True,
                   capture_output=True)
    objects = glob.glob(str(tmp_path / '*gfx950'))
    sources = glob.glob(os.path.join(ROOT, 'gluon-nlp_amd', 'csrc', '*.hip'))
    assert len(objects) == len(sources)
    kernels = 0
    for f in objects:
        text = subprocess.run([OBJDUMP, '-d', '--mcpu=gfx950', f], check=True, capture_output=True,
                              text=True).stdout
        kernels += text.count('s_endpgm')
        assert not re.search(r'v_pk_(add|mul|fma)_f32', text), f
    assert kernels > 100
