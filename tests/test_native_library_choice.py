"""A library chosen by path or by LDMSEG_HIP_LIB: tuning hooks may be missing from it, entries of operators may not."""
import subprocess

import pytest

from ldmseg.ops import native as K


def _library(tmp_path, without):
    src, so = tmp_path / "entries.c", tmp_path / f"lib_{without}.so"
    src.write_text("".join(f"int {name}(void) {{ return 0; }}\n" for name in K.EXPORTS if name != without))
    subprocess.run(["gcc", "-shared", "-fPIC", "-o", str(so), str(src)], check=True)
    return str(so)


@pytest.mark.parametrize("by_env", [False, True])
@pytest.mark.parametrize("entry", ["ldm_conv2d", "ldm_attention", "ldm_label_log_probs", "ldm_grad_norm"])
def test_a_library_without_an_operator_does_not_load(tmp_path, monkeypatch, entry, by_env):
    assert entry in K.EXPORTS
    monkeypatch.setattr(K, "_lib", None)
    path = _library(tmp_path, entry)
    if by_env:
        monkeypatch.setenv("LDMSEG_HIP_LIB", path)
        path = None
    with pytest.raises(AttributeError, match=entry):
        K.load_library(path)
    assert K._lib is None


def test_a_library_without_a_tuning_hook_loads(tmp_path, monkeypatch):
    hook = "ldm_conv2d_set_halo"
    assert hook in K.EXPORTS
    monkeypatch.setattr(K, "_lib", None)
    lib = K.load_library(_library(tmp_path, hook))
    assert lib.ldm_abi_version() == 0 and not hasattr(lib, hook)
