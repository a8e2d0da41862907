"""What code the run-time compiler makes."""
import os
import subprocess

import pytest

from mxnet_amd import rtc

OBJDUMP = '/opt/rocm/llvm/bin/llvm-objdump'


@pytest.mark.skipif(not os.path.exists(OBJDUMP), reason='no disassembler')
def test_no_packed_float32_instructions(tmp_path):
    """Four independent float products next to each other, which the compiler
    likes to pack."""
    mod = rtc.HipModule('''
        extern "C" __global__ void k(const float4 *x, float4 *y) {
            float4 a = x[threadIdx.x], b = y[threadIdx.x];
            a.x = a.x * b.x + 1.f;
            a.y = a.y * b.y + 1.f;
            a.z = a.z * b.z * a.w;
            a.w = a.w + b.w;
            y[threadIdx.x] = a;
        }''')
    path = tmp_path / 'k.co'
    path.write_bytes(bytes(mod._code))
    code = subprocess.run([OBJDUMP, '-d', str(path)], capture_output=True,
                          text=True, check=True).stdout
    assert 's_endpgm' in code
    for name in ('add', 'mul', 'fma'):
        assert f'v_pk_{name}_f32' not in code
