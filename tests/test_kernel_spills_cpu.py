"""No kernel of sampling or of the plain 4-bit linears spills registers: a spill
puts scratch traffic into loops that live on their loads in flight."""
import os
import re
import shutil
import subprocess

import pytest

from ornith_g256 import _build


@pytest.mark.skipif(not (shutil.which(_build.HIPCC) or os.path.exists(_build.HIPCC)), reason='no hipcc')
@pytest.mark.parametrize('source', ['w4.hip', 'sample.hip'])
def test_no_spills(tmp_path, source):
    cmd = [_build.HIPCC, *_build.FLAGS, '-DORNITH_ROUTED_TILE=32', '--offload-device-only',
           '-Rpass-analysis=kernel-resource-usage', '-c', str(_build.CSRC / source), '-o', str(tmp_path / 'k.o')]
    res = subprocess.run(cmd, capture_output=True, text=True)
    assert res.returncode == 0, res.stderr
    names = re.findall(r'Function Name: (\S+)', res.stderr)
    for what in (r'VGPRs Spill: (\d+)', r'ScratchSize \[bytes/lane\]: (\d+)'):
        counts = [int(c) for c in re.findall(what, res.stderr)]
        assert len(counts) == len(names) > 10
        assert not any(counts), [(n, c) for n, c in zip(names, counts) if c]
