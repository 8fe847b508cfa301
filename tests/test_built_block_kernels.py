"""The 8-bit products and the weight gradients place their tiles in LDS by the
same hand-counted loads as the attention kernels: they spill no vector register
and leave the register that places the loads to them."""
from __future__ import annotations

import re
import subprocess

import pytest

from test_built_kernels import LIBRARY, code_objects, tool

KERNELS = ('product_kernel', 'weight_grad_kernel')


@pytest.fixture(scope='module')
def objects(pkg, tmp_path_factory):
    paths = []
    for i, code in enumerate(code_objects(LIBRARY.read_bytes())):
        if any(k.encode() in code for k in KERNELS):
            paths.append(tmp_path_factory.mktemp('code') / f'{i}.o')
            paths[-1].write_bytes(code)
    assert len(paths) >= 2
    return paths


def test_no_vector_register_is_spilled(objects):
    seen = dict.fromkeys(KERNELS, 0)
    for path in objects:
        notes = subprocess.run([tool('llvm-readelf'), '--notes', str(path)], check=True,
                               capture_output=True, text=True).stdout
        for kernel in notes.split('- .agpr_count')[1:]:
            name = re.search(r'\.symbol:\s+(\S+)', kernel).group(1)
            for k in KERNELS:
                if k in name:
                    seen[k] += 1
                    assert re.search(r'\.vgpr_spill_count:\s+(\d+)', kernel).group(1) == '0', name
    assert all(seen.values()), seen


def test_nothing_else_uses_the_register_of_the_loads(objects):
    for path in objects:
        text = subprocess.run([tool('llvm-objdump'), '-d', '--no-show-raw-insn',
                               '--no-leading-addr', str(path)], check=True, capture_output=True,
                              text=True).stdout
        lines = [line.split('//')[0].split() for line in text.splitlines()]
        lines = [line for line in lines if line]
        loads = 0
        for i, line in enumerate(lines):
            if any(part.rstrip(',') == 'm0' for part in line[1:]):
                assert line[:2] == ['s_mov_b32', 'm0,'], line
                assert lines[i + 1] == ['s_nop', '3']
                assert lines[i + 2][0].startswith('global_load_lds_dword'), lines[i + 2]
                loads += 1
        assert loads == sum(line[0].startswith('global_load_lds') for line in lines) > 0
