"""The module of direct entries: which build of it is used, and calls without
it (no GPU)."""
import subprocess
from types import SimpleNamespace

import pytest
import torch

from cdq_lrr_b200 import _lib as L
from cdq_lrr_b200 import build


@pytest.mark.parametrize("what", ["torch", "abi", "python"])
def test_another_torch_or_python_gets_a_module_of_its_own(monkeypatch, what):
    """The module is bound to the C++ ABI of the torch and the Python that it was compiled against."""
    build.build_torch()
    here = L.direct_path()
    assert here.exists()
    if what == "torch":
        monkeypatch.setattr(torch, "__version__", "0.0.1+test")
    elif what == "abi":
        monkeypatch.setattr(torch._C, "_GLIBCXX_USE_CXX11_ABI", not torch._C._GLIBCXX_USE_CXX11_ABI)
    else:
        import sys
        monkeypatch.setattr(sys, "implementation", SimpleNamespace(cache_tag="cpython-00"))
    other = L.direct_path()
    assert other != here and not other.exists()
    commands = []

    def compile_(cmd, **kw):
        commands.append(cmd)
        open(cmd[cmd.index("-o") + 1], "w").close()
        return SimpleNamespace(returncode=0)

    monkeypatch.setattr(subprocess, "run", compile_)
    try:
        assert build.build_torch() == other and len(commands) == 1
        assert build.build_torch() == other and len(commands) == 1    # and is kept
    finally:
        other.unlink(missing_ok=True)
    assert here.exists()


def test_calls_without_the_module(monkeypatch, tmp_path):
    """Without a module for this torch every call takes the general path, which says what it wants; one warning."""
    from cdq_lrr_b200 import sampling
    from cdq_lrr_b200.kvcache import QuantKVCache
    monkeypatch.setattr(L, "_direct", None)
    monkeypatch.setattr(L, "direct_path", lambda: tmp_path / "_cdq_torch.none.so")
    c = QuantKVCache(1, 2, 8, 64, device="cpu")
    x = torch.zeros(1, 1, 2, 64, dtype=torch.bfloat16)
    p, u = torch.zeros(1, dtype=torch.int32), torch.zeros(1)
    with pytest.warns(RuntimeWarning, match="cdq_lrr_b200.build"):
        with pytest.raises(RuntimeError, match="no CPU path"):
            c.append(x, x, p)
    for call in (lambda: c.attend(x, p), lambda: c.read(p, 1), lambda: sampling.sample_tokens(x[0, 0], u),
                 lambda: sampling.verify_drafts(x[:, 0], p.long()[:, None], None, u[:, None], u)):
        with pytest.raises(RuntimeError, match="no CPU path"):
            call()


def test_cpu_tensors_are_refused_by_name():
    """The refusal of CPU tensors is the call's own, with the module as without."""
    from cdq_lrr_b200.kvcache import QuantKVCache
    build.build_torch()
    assert hasattr(L.direct(), "kv_append")
    c = QuantKVCache(1, 2, 8, 64, device="cpu")
    x = torch.zeros(1, 1, 2, 64, dtype=torch.bfloat16)
    p = torch.zeros(1, dtype=torch.int32)
    for call in (lambda: c.append(x, x, p), lambda: c.attend(x, p), lambda: c.read(p, 1)):
        with pytest.raises(RuntimeError, match="no CPU path"):
            call()


def test_build_without_torch(monkeypatch):
    """The C library needs nvcc alone: without torch there is no module to build, and that is no error."""
    import sys
    monkeypatch.setitem(sys.modules, "torch", None)
    assert build.build_torch() is None
    assert build.build() == build.LIB


def test_numbers_that_no_integer_type_holds():
    """An n beyond 64 bits goes to the general path and its message, not to an interpreter error."""
    from cdq_lrr_b200.kvcache import QuantKVCache
    c = QuantKVCache(1, 2, 8, 64, device="cpu")
    for n in (2 ** 63, 2 ** 70, -2 ** 70):
        assert L.direct().kv_read(c._address, c._index, None, n) is None
        with pytest.raises(RuntimeError, match="no CPU path"):
            c.read(None, n)


@pytest.mark.gpu
def test_out_of_memory_is_torchs_own_error():
    """A result that no device can hold (1.1 TB, refused by the allocator): callers catch torch's error by its type;
    the cache and the device go on."""
    from cdq_lrr_b200.kvcache import QuantKVCache
    c = QuantKVCache(1, 1024, 1, 128)
    with pytest.raises(torch.OutOfMemoryError):
        c.read(None, 1 << 22)
    k, v = c.read(None, 1)
    assert k.shape == (1, 1, 1024, 128) and not k.any() and not v.any()
