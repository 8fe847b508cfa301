"""How the native parts are built: for the interpreter that runs the build, and
the C ABI without one."""
from __future__ import annotations

import subprocess
import sys

import __graft_entry__ as entry

CSRC = entry.PKG_DIR / 'csrc'


def planned(*args):
    """What make would do, with every output out of date."""
    return subprocess.run(['make', '-B', '-n', '-C', str(CSRC), *args], capture_output=True, text=True)


def test_the_build_is_for_its_own_interpreter(pkg, monkeypatch):
    commands = []
    monkeypatch.setattr(entry, '_run', commands.append)
    entry.build()
    calls, = (c for c in commands if str(CSRC) in c)
    assert f'PYTHON={sys.executable}' in calls


def test_an_interpreter_without_torch(tmp_path):
    """It says so, and the library alone needs none."""
    bare = tmp_path / 'bare'
    bare.write_text(f'#!/bin/sh\nexec {sys.executable} -S -E "$@"\n')  # (no installed packages)
    bare.chmod(0o755)
    plan = planned(f'PYTHON={bare}')
    assert plan.returncode != 0 and f'{bare} has no torch' in plan.stderr, plan.stderr
    plan = planned('library', f'PYTHON={bare}')
    assert plan.returncode == 0 and 'libbevpool_amd.so' in plan.stdout
    assert '_block_calls' not in plan.stdout and str(bare) not in plan.stdout
    plan = planned(f'PYTHON={sys.executable}')
    assert plan.returncode == 0 and '_block_calls.so' in plan.stdout, plan.stderr
