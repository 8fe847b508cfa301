"""What the attention kernels' hand-written waits rely on, in the built library:
they spill no vector register (a reload counts among the loads that they wait
for), and the register that places their loads in LDS, which the compiler takes
as its own and does not see written, is used by nothing else."""
from __future__ import annotations

import re
import shutil
import struct
import subprocess
from pathlib import Path

import pytest

from conftest import ROOT

LIBRARY = ROOT / 'bevfusion-triton_amd' / 'libbevpool_amd.so'
KERNELS = ('packed_forward_kernel', 'query_grad_kernel', 'key_grad_kernel', 'parts_kernel')


def tool(name):
    path = shutil.which(name) or f'/opt/rocm/llvm/bin/{name}'
    if not Path(path).exists():
        pytest.skip(f'no {name}')
    return path


def code_objects(data):
    """The gfx950 code objects of a library: entries (offset, size, length of
    the target's name, name) behind the magic and the count of every bundle."""
    magic = b'__CLANG_OFFLOAD_BUNDLE__'
    at = data.find(magic)
    while at >= 0:
        n, = struct.unpack_from('<Q', data, at + len(magic))
        entry = at + len(magic) + 8
        for _ in range(n):
            offset, size, length = struct.unpack_from('<QQQ', data, entry)
            target = data[entry + 24:entry + 24 + length]
            entry += 24 + length
            if b'gfx950' in target and size:
                yield data[at + offset:at + offset + size]
        at = data.find(magic, at + 1)


@pytest.fixture(scope='module')
def attention_objects(pkg, tmp_path_factory):
    paths = []
    for i, code in enumerate(code_objects(LIBRARY.read_bytes())):
        if any(k.encode() in code for k in KERNELS):
            paths.append(tmp_path_factory.mktemp('code') / f'{i}.o')
            paths[-1].write_bytes(code)
    assert len(paths) >= 3
    return paths


def test_no_vector_register_is_spilled(attention_objects):
    seen = dict.fromkeys(KERNELS, 0)
    for path in attention_objects:
        notes = subprocess.run([tool('llvm-readelf'), '--notes', str(path)], check=True,
                               capture_output=True, text=True).stdout
        for kernel in notes.split('- .agpr_count')[1:]:
            name = re.search(r'\.symbol:\s+(\S+)', kernel).group(1)
            for k in KERNELS:
                if k in name:
                    seen[k] += 1
                    spilled = re.search(r'\.vgpr_spill_count:\s+(\d+)', kernel).group(1)
                    assert spilled == '0', name
    assert all(seen.values()), seen


def test_nothing_else_uses_the_register_of_the_loads(attention_objects):
    for path in attention_objects:
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
