"""The Python extension of the 4-bit cache's calls beside another torch than its own."""
import pytest
import torch

from llamamps_b200 import _lib
from llamamps_b200 import kernels as K


@pytest.fixture
def fresh(monkeypatch):
    monkeypatch.setattr(_lib, "_BIND", None)
    return monkeypatch


def _refused():
    """A call goes all the way to the checks behind the extension."""
    q, one = torch.zeros(1, 1536, dtype=torch.float16), torch.ones(1, dtype=torch.int32)
    pool, bt = torch.zeros(2, 2, 64 * 72, dtype=torch.uint8), torch.zeros(1, 2, dtype=torch.int32)
    with pytest.raises(RuntimeError, match="CUDA"):
        K.gqa_decode_attention_q4(q, pool, pool, bt, one, q.clone(), None, 64, 12, 2, 128, 128, 1)


def test_the_extension_is_built_for_this_torch(fresh):
    assert _lib.binding().torch_version == torch.__version__
    _refused()


def test_another_torch_is_not_read(fresh):
    fresh.setattr(torch, "__version__", "0.0.0")
    with pytest.warns(RuntimeWarning, match="built against"):
        assert _lib.binding().append() is None
    _refused()


def test_an_extension_that_does_not_load(fresh, tmp_path):
    (tmp_path / "bind_q4.so").write_bytes(b"not a library")
    fresh.setattr(_lib, "BIND_PATH", str(tmp_path / "bind_q4.so"))
    with pytest.warns(RuntimeWarning, match="left out"):
        assert _lib.binding() is _lib._Unbound
    _refused()
    fresh.setattr(_lib, "_BIND", None)
    fresh.setattr(_lib, "BIND_PATH", str(tmp_path / "none.so"))
    with pytest.raises(RuntimeError, match="missing"):
        _lib.binding()
