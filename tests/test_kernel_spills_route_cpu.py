"""No kernel of expert routing or of the adapters spills registers."""
import os
import shutil

import pytest

import test_kernel_spills_cpu as S
from ornith_g256 import _build


@pytest.mark.skipif(not (shutil.which(_build.HIPCC) or os.path.exists(_build.HIPCC)), reason='no hipcc')
@pytest.mark.parametrize('source', ['route.hip', 'adapter.hip'])
def test_no_spills(tmp_path, source):
    S.test_no_spills(tmp_path, source)
