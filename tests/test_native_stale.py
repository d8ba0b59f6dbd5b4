"""CPU: a libg2v.so of an older tree is refused by name, not by an
AttributeError from the middle of the binding."""
import subprocess

import pytest

from gene2vec_amd import _native as N


@pytest.mark.parametrize("version,symbols,match", [
    (N.ABI_VERSION - 1, [], "version mismatch"),
    (None, [], "version mismatch"),
    (N.ABI_VERSION, [], "without .*g2v_create"),
    (N.ABI_VERSION, sorted(set(N.SIGNATURES) - {"g2v_embed_lookup", "g2v_abi_version"}),
     "without g2v_embed_lookup;")])
def test_stale_library_is_refused(tmp_path, monkeypatch, version, symbols, match):
    lib = tmp_path / "libg2v.so"
    source = "".join(f"int {s}(void) {{ return 0; }}\n" for s in symbols)
    if version is not None:
        source += f"int g2v_abi_version(void) {{ return {version}; }}\n"
    subprocess.run(["gcc", "-shared", "-fPIC", "-x", "c", "-", "-o", str(lib)],
                   input=source, text=True, check=True)
    monkeypatch.setattr(N, "_lib", None)
    monkeypatch.setattr(N, "LIB_PATH", str(lib))
    with pytest.raises(N.NativeLibraryError, match=match) as e:
        N.lib()
    assert "gene2vec_amd.build" in str(e.value)
