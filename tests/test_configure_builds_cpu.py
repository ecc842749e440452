"""configure loads the builds that its roles name, and no other."""
import pytest

from ornith_g256 import native


@pytest.mark.parametrize('tile', [16])
def test_one_build_serves_every_role(monkeypatch, tile):
    monkeypatch.setattr(native, '_handles', {})
    real = native.library_path
    monkeypatch.setattr(native, 'library_path', lambda t=32: real(t) if t == tile else real(t).with_name('absent.so'))
    native.reset_binding()
    try:
        path = str(real(tile))
        size = native.configure(dict(dense_library=path, routed_library=path, head_library=path), 64, ((512, 2048),))
        assert size >= native.logits_sample_bytes(native.HEAD_MAX_ROWS, native.HEAD_VOCAB, tile=tile) > 0
        assert set(native._handles) == {tile}
    finally:
        native.reset_binding()
