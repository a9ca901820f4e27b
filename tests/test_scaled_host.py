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


@pytest.mark.parametrize("d", [64, 128, 256])
@pytest.mark.parametrize("tokens,requests,group", [(8192, 1, 4), (8192, 1, 64), (60000, 2, 1),
                                                   (2048, 32, 16), (20000, 4096, 8)])
def test_a_small_hint_for_a_large_array_asks_for_a_bounded_workspace(tokens, requests, group, d):
    """A row of D sums and its two statistics, 32 bits each; 8 * 4,096 parts of 32 rows, or
    8 * 1,536 of 128, at most, for each of two launches."""
    heads = 8
    desc = attend_desc(heads=heads, head_size=d, num_blocks=1 << 20, tokens=tokens,
                       requests=requests, q_heads=heads * group, table_width=1 << 16, max_new=1)
    most = 2 * 8 * max(4096 * 32, 1536 * 128) * (d + 2) * 4
    size = _lib.lib().mkv_attend_workspace_size(ctypes.byref(desc))
    assert 0 <= size <= most


@pytest.mark.parametrize("d,tokens,parts", [
    (256, 2048, 1), (256, 1024, 1),  # 512 and 256 tiles, 256 at once
    (256, 512, 2),    # 128
    (256, 704, 5),    # 176: one or two parts each would leave a third of the slots empty
    (128, 4096, 1), (128, 2048, 1),  # 1,024 and 512 tiles, 512 at once
    (128, 1024, 2),
    (128, 2560, 3),   # 640
])
def test_the_parts_of_a_chunk_fill_the_chip(d, tokens, parts):
    """One request, 8 heads of 4 query heads, 8,192 tokens held: tiles of 128 rows, of which as
    many run at once as the kernel's registers and LDS let."""
    desc = attend_desc(heads=8, head_size=d, num_blocks=4096, tokens=tokens, requests=1, q_heads=32,
                       table_width=1024, max_new=tokens, max_len=8192 + tokens)
    rows = tokens * 4 // 128 + 1  # and a tile to spare
    want = rows * 8 * parts * 128 * (d + 2) * 4 if parts > 1 else 0
    assert _lib.lib().mkv_attend_workspace_size(ctypes.byref(desc)) == want
