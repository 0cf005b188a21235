"""The build: what is compiled again, and when."""
import os
import subprocess

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
CSRC = os.path.join(ROOT, 'dp_cgans_amd', 'csrc')


@pytest.mark.parametrize('changed', ['../../include/dpcgan_hip.h', 'dpc_common.h', 'Makefile'])
def test_every_object_follows_what_all_share(changed):
    """Objects that hold different layouts of one struct, or were compiled with other flags, must not meet in one library."""
    out = subprocess.run(['make', '-C', CSRC, '-n', '-W', changed], capture_output=True, text=True, check=True).stdout
    sources = sorted(f for f in os.listdir(CSRC) if f.endswith('.hip'))
    assert sources and [f for f in sources if ' -c %s ' % f not in out] == []


def test_build_compiles_what_is_there_again(monkeypatch):
    """A library that is newer than its sources says nothing about whether they compile."""
    import __graft_entry__ as entry
    ran = []
    monkeypatch.setattr(entry.subprocess, 'check_call', lambda cmd, **kw: ran.append(cmd))
    entry.build()
    plan = subprocess.run(list(ran[0]) + ['-n'], capture_output=True, text=True, check=True).stdout
    assert len(ran) == 1 and plan.count(' -c ') == len([f for f in os.listdir(CSRC) if f.endswith('.hip')])
