"""What the build's own flags make of the kernels (hipcc cross-compiles, no GPU): no packed f32
instruction anywhere, and nothing of the hand-scheduled GEMM spilled -- its waits count every
vector-memory instruction in flight, scratch traffic included."""
import os
import re
import subprocess

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
CSRC = os.path.join(ROOT, 'gluon-nlp_amd', 'csrc')
HIPCC = '/opt/rocm/bin/hipcc'
FLAGS = ['-Xclang', '-target-feature', '-Xclang', '-packed-fp32-ops']


def _assembly(name, to):
    if not os.path.exists(HIPCC):
        pytest.skip('hipcc not available')
    subprocess.run([HIPCC, '--offload-arch=gfx950', '-O3', '-std=c++17', '-fPIC'] + FLAGS +
                   ['-S', '--cuda-device-only', '-o', str(to), os.path.join(CSRC, name)],
                   check=True, capture_output=True)
    return open(str(to)).read()


def test_makefile_has_the_flags():
    text = open(os.path.join(ROOT, 'gluon-nlp_amd', 'Makefile')).read()
    assert ' '.join(FLAGS) in text


def test_sources_write_no_packed_f32():
    for f in os.listdir(CSRC):
        code = re.sub(r'//.*', '', open(os.path.join(CSRC, f)).read())
        assert not re.search(r'v_pk_(add|mul|fma)_f32', code), f


def test_gemm_with_the_build_flags(tmp_path):
    text = _assembly('gemm_bf16_w4.hip', tmp_path / 'w4.s')
    assert not re.search(r'v_pk_(add|mul|fma)_f32', text)
    for key in ('vgpr_spill_count', 'private_segment_fixed_size'):
        vals = [int(v) for v in re.findall(r'\.%s:\s+(\d+)' % key, text)]
        assert len(vals) == 24 and not any(vals), (key, vals)


@pytest.mark.parametrize('name', ['kv4.hip', 'kv4_attn.hip', 'beam.hip'])
def test_decoding_kernels_with_the_build_flags(tmp_path, name):
    """Registers are cut to the waves that a SIMD is to hold: nothing may be spilled for it."""
    text = _assembly(name, tmp_path / 'k.s')
    assert not re.search(r'v_pk_(add|mul|fma)_f32', text)
    vals = [int(v) for v in re.findall(r'\.vgpr_spill_count:\s+(\d+)', text)]
    assert vals and not any(vals), vals
