"""The block-scaled entry points' host side, further: what each call refuses or asks for."""

from __future__ import annotations

import ctypes
import importlib.machinery
import subprocess

import pytest
import torch

from marathon_amd import _lib, scaled_cache, shift_kernels
from tests.test_scaled_plain import attend_desc

#: The ABI's last version without the block-scaled cache.
EARLIER = (3 << 16) | 5


@pytest.mark.parametrize("token,head", [(128, 128), (256, 128), (128, 256), (0, 128), (512, 0),
                                        (512, 64), (64, 512)])
def test_attend_refuses_outputs_that_overlap(token, head):
    """Three tokens of four heads of 128."""
    desc = attend_desc(out_token_stride=token, out_head_stride=head)
    assert _lib.lib().mkv_attend_scaled(ctypes.byref(desc), None) == _lib.MKV_ERR_ARG
    assert b"overlap" in _lib.lib().mkv_last_error()


def test_a_library_of_an_earlier_version_is_named_as_one(monkeypatch, tmp_path):
    """It lacks entry points; the refusal speaks of its version, not of the first of them."""
    src, out = tmp_path / "old.c", tmp_path / "libold.so"
    src.write_text(f"int mkv_abi_version(void) {{ return {EARLIER}; }}\n")
    subprocess.run(["gcc", "-shared", "-fPIC", str(src), "-o", str(out)], check=True)
    monkeypatch.setattr(_lib, "LIB_PATH", str(out))
    monkeypatch.setattr(_lib, "_LIB", None)
    with pytest.raises(RuntimeError, match="version"):
        _lib.lib()
    monkeypatch.undo()
    assert _lib.lib().mkv_abi_version() == _lib.MKV_ABI_VERSION


def test_without_its_module_of_this_version_scatter_goes_the_general_way(monkeypatch):
    """A module from before the block-scaled cache has no bind_scaled."""
    class Loader(importlib.machinery.ExtensionFileLoader):
        def create_module(self, spec):
            return None

        def exec_module(self, module):
            module.abi, module.torch, module.bind = EARLIER, torch.__version__, lambda at: None

    _lib.lib()
    monkeypatch.setattr(importlib.machinery, "ExtensionFileLoader", Loader)
    monkeypatch.setattr(_lib, "_BINDING", None)
    monkeypatch.setattr(shift_kernels, "_usual_call", None)
    with pytest.raises(RuntimeError, match="rebuild"):
        _lib.binding()
    with pytest.warns(RuntimeWarning, match="general path"):
        with pytest.raises(RuntimeError, match="not on a HIP device"):
            shift_kernels.scatter_shifted(torch.zeros(2, 8, 128), torch.zeros(4, 8, 16, 128),
                                          torch.zeros(2, dtype=torch.int64), 16, True, None)
    t = torch.zeros((1, 2), dtype=torch.int32)
    with pytest.warns(RuntimeWarning, match="general path"):
        assert scaled_cache._Usual().slots(t) is None
