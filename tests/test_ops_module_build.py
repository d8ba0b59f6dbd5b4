"""CPU: a _g2v_torch.so of another build is told apart, when it is built and
when it is loaded."""
import importlib
import os
import subprocess

import pytest
import torch

from gene2vec_amd import _g2v_torch as X
from gene2vec_amd import _native as N
from gene2vec_amd import build as B
from gene2vec_amd import ops


def test_module_states_what_it_was_compiled_against():
    assert X.abi_version() == N.ABI_VERSION
    assert X.torch_version() == torch.__version__.split("+")[0]
    # its own constant: nothing of libg2v answers in its place
    r = subprocess.run(["nm", "-D", "--undefined-only", B.TORCH_LIB], capture_output=True, text=True,
                       check=True)
    assert "g2v_embed_lookup" in r.stdout and "g2v_abi_version" not in r.stdout


@pytest.mark.parametrize("name,value", [("abi_version", N.ABI_VERSION - 1),
                                        ("torch_version", "1.0.0")])
def test_another_build_is_refused(monkeypatch, name, value):
    with monkeypatch.context() as m:
        m.setattr(X, name, lambda: value)
        with pytest.raises(N.NativeLibraryError, match="built for"):
            importlib.reload(ops)
    importlib.reload(ops)


def test_module_is_rebuilt_for_another_torch(monkeypatch, tmp_path):
    lib, stamp = tmp_path / "x.so", tmp_path / "build" / "torch.stamp"
    ran = []

    def run(cmd, **kw):
        ran.append(cmd)
        (tmp_path / "x.so.tmp").write_text("built")
        return subprocess.CompletedProcess(cmd, 0, "", "")

    monkeypatch.setattr(B, "TORCH_LIB", str(lib))
    monkeypatch.setattr(B, "TORCH_STAMP", str(stamp))
    monkeypatch.setattr(B.subprocess, "run", run)
    B.build_torch()
    B.build_torch()
    assert len(ran) == 1 and lib.read_text() == "built"
    with monkeypatch.context() as m:
        m.setattr(torch, "__version__", "9.9.9")
        B.build_torch()
        B.build_torch()
    assert len(ran) == 2
    B.build_torch(force=True)
    assert len(ran) == 3
    stamp.unlink()
    B.build_torch()
    assert len(ran) == 4
    source = tmp_path / "s.cpp"
    source.write_text("another")
    monkeypatch.setattr(B, "TORCH_SOURCE", str(source))
    B.build_torch()
    assert len(ran) == 5 and os.path.exists(stamp)
