"""What a caller that mirrors the header's structs goes by: the version, and the sizes."""
import ctypes
import os
import re
import shutil
import subprocess

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
HEADER = os.path.join(ROOT, 'include', 'dpcgan_hip.h')


def test_the_version_grew_with_the_descriptor():
    """100 was the version of a shorter dpc_gemm_desc, which the library would read past."""
    from dp_cgans_amd import _lib
    declared = int(re.search(r'^#define DPC_VERSION (\d+)$', open(HEADER).read(), flags=re.M).group(1))
    assert _lib.lib().cdll.dpc_version() == declared > 100


def test_a_library_of_another_version_is_refused(monkeypatch, tmp_path):
    from dp_cgans_amd import _lib
    other = tmp_path / 'dpcgan_hip.h'
    other.write_text(re.sub(r'(#define DPC_VERSION) \d+', r'\1 99', open(HEADER).read()))
    monkeypatch.setattr(_lib, 'HEADER_PATH', str(other))
    with pytest.raises(ImportError, match='99'):
        _lib._Lib()


@pytest.mark.skipif(not shutil.which('gcc'), reason='no C compiler')
def test_the_mirrored_structs_have_the_headers_layout(tmp_path):
    from dp_cgans_amd import ops
    mirrors = {'dpc_gemm_desc': ops.GemmDesc, 'dpc_multi_tensor': ops.MultiTensor, 'dpc_multi_info': ops.MultiInfo}
    lines = ['printf("%%zu ", sizeof(%s));' % s for s in mirrors]
    for s, m in mirrors.items():
        lines += ['printf("%%zu ", offsetof(%s, %s));' % (s, name) for name, _ in m._fields_]
    src = tmp_path / 'sizes.c'
    src.write_text('#include <stdio.h>\n#include <stddef.h>\n#include "%s"\nint main(void) {%s return 0;}' % (HEADER, '\n'.join(lines)))
    subprocess.run(['gcc', str(src), '-o', str(tmp_path / 'sizes')], check=True)
    got = [int(x) for x in subprocess.run([str(tmp_path / 'sizes')], capture_output=True, text=True, check=True).stdout.split()]
    want = [ctypes.sizeof(m) for m in mirrors.values()] + [getattr(m, n).offset for m in mirrors.values() for n, _ in m._fields_]
    assert got == want
