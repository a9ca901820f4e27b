"""The step's operators without a GPU: the descriptors' layout, every refusal that needs no device
memory, and the workspace that attention over shared tokens asks for."""

from __future__ import annotations

import ctypes
import os
import subprocess

import pytest
import torch

from marathon_amd import _lib, norm_rotate
from tests.test_scaled_plain import BAD_CACHES, ROOT, attend_desc, cache_desc

STRUCTS = {"mkv_turn_t": _lib.Turn, "mkv_head_rows_t": _lib.HeadRows,
           "mkv_norm_rotate_desc_t": _lib.NormRotateDesc,
           "mkv_store_rotated_desc_t": _lib.StoreRotatedDesc,
           "mkv_attend_shared_desc_t": _lib.AttendSharedDesc}


def test_descriptors_match_the_header(tmp_path):
    lines = [f'  printf("{n} %zu\\n", sizeof({n}));' for n in STRUCTS]
    lines += [f'  printf("{n}.{f[0]} %zu\\n", offsetof({n}, {f[0]}));'
              for n, s in STRUCTS.items() for f in s._fields_]
    src, exe = tmp_path / "probe.c", tmp_path / "probe"
    src.write_text('#include <stddef.h>\n#include <stdio.h>\n#include "marathon_kvstep.h"\n'
                   "int main(void) {\n" + "\n".join(lines) + "\n  return 0;\n}\n")
    subprocess.run(["gcc", "-std=c99", f"-I{os.path.join(ROOT, 'include')}", str(src), "-o", str(exe)],
                   check=True)
    out = subprocess.run([str(exe)], check=True, capture_output=True, text=True).stdout
    for name, at in (line.split() for line in out.splitlines()):
        name, _, field = name.partition(".")
        s = STRUCTS[name]
        assert (getattr(s, field).offset if field else ctypes.sizeof(s)) == int(at), (name, field)


def set_fields(d, **kw):
    for path, value in kw.items():
        *parents, last = path.split("__")
        at = d
        for p in parents:
            at = getattr(at, p)
        setattr(at, last, value)
    return d


def rows(d, heads, head_size=128):
    return set_fields(d, x=1 << 20, out=1 << 21, token_stride=heads * head_size, head_stride=head_size,
                      out_token_stride=heads * head_size, out_head_stride=head_size, heads=heads)


def turn(d):
    return set_fields(d, inv_freq=1 << 20, q_weight=1 << 20, k_weight=1 << 20, rotary=128,
                      weight_dtype=_lib.MKV_BF16, eps=1e-6, norm=1)


TURNS = [
    (dict(turn__rotary=48), _lib.MKV_ERR_ARG), (dict(turn__rotary=160), _lib.MKV_ERR_ARG),
    (dict(turn__rotary=-32), _lib.MKV_ERR_ARG), (dict(turn__inv_freq=None), _lib.MKV_ERR_ARG),
    (dict(turn__inv_freq=(1 << 20) + 2), _lib.MKV_ERR_ALIGN), (dict(turn__eps=-1.0), _lib.MKV_ERR_ARG),
    (dict(turn__eps=float("nan")), _lib.MKV_ERR_ARG), (dict(turn__eps=float("inf")), _lib.MKV_ERR_ARG),
    (dict(turn__norm=0), _lib.MKV_ERR_ARG), (dict(turn__weight_dtype=_lib.MKV_FP8_E4M3), _lib.MKV_ERR_DTYPE),
    (dict(turn__k_weight=(1 << 20) + 2), _lib.MKV_ERR_ALIGN),
    (dict(q__heads=-1), _lib.MKV_ERR_ARG), (dict(q__heads=1 << 20), _lib.MKV_ERR_ARG),
    (dict(q__token_stride=-512), _lib.MKV_ERR_ARG), (dict(q__head_stride=1 << 61), _lib.MKV_ERR_ARG),
    (dict(q__x=None), _lib.MKV_ERR_ARG), (dict(q__out=None), _lib.MKV_ERR_ARG),
    (dict(q__x=(1 << 20) + 8), _lib.MKV_ERR_ALIGN), (dict(q__out_head_stride=132), _lib.MKV_ERR_ALIGN),
    (dict(q__out_head_stride=64), _lib.MKV_ERR_ARG), (dict(q__out_token_stride=0), _lib.MKV_ERR_ARG),
    (dict(dtype=_lib.MKV_FP8_E4M3), _lib.MKV_ERR_DTYPE), (dict(tokens=-1), _lib.MKV_ERR_ARG),
    (dict(tokens=1 << 31), _lib.MKV_ERR_ARG),
]


def rotate_desc(**kw):
    d = _lib.NormRotateDesc()
    rows(d.q, 4), rows(d.k, 2), turn(d.turn)
    d.positions, d.position_bytes, d.tokens, d.head_size, d.dtype = 1 << 20, 4, 3, 128, _lib.MKV_BF16
    return set_fields(d, **kw)


@pytest.mark.parametrize("change,code", TURNS + [
    (dict(head_size=96), _lib.MKV_ERR_UNSUPPORTED), (dict(positions=None), _lib.MKV_ERR_ARG),
    (dict(position_bytes=2), _lib.MKV_ERR_ARG), (dict(positions=(1 << 20) + 2), _lib.MKV_ERR_ALIGN),
    (dict(position_bytes=8, positions=(1 << 20) + 4), _lib.MKV_ERR_ALIGN),
    (dict(k__x=None), _lib.MKV_ERR_ARG), (dict(k__out_token_stride=128), _lib.MKV_ERR_ARG),
    (dict(tokens=(1 << 31) - 1, q__heads=600, q__token_stride=600 * 128, q__out_token_stride=600 * 128),
     _lib.MKV_ERR_UNSUPPORTED),
    (dict(tokens=0), _lib.MKV_OK), (dict(q__heads=0, k__heads=0), _lib.MKV_OK)])
def test_norm_rotate_refuses(change, code):
    assert _lib.lib().mkv_norm_rotate(ctypes.byref(rotate_desc(**change)), None) == code
    if code:
        assert _lib.lib().mkv_last_error()


def put_desc(**kw):
    d = _lib.StoreRotatedDesc()
    d.cache = cache_desc(**{k: kw.pop(k) for k in list(kw) if hasattr(_lib.ScaledCacheDesc, k)})
    rows(d.q, 4), turn(d.turn)
    d.k = d.v = d.block_tables = d.starts = d.lens = 1 << 20
    d.k_token_stride, d.k_head_stride, d.v_token_stride, d.v_head_stride = 256, 128, 256, 128
    d.table_stride = d.table_width = 8
    d.tokens, d.requests, d.dtype = 3, 2, _lib.MKV_BF16
    return set_fields(d, **kw)


@pytest.mark.parametrize("change,code", BAD_CACHES + TURNS + [
    (dict(k=None), _lib.MKV_ERR_ARG), (dict(v=(1 << 20) + 4), _lib.MKV_ERR_ALIGN),
    (dict(k_token_stride=252), _lib.MKV_ERR_ALIGN), (dict(v_head_stride=-128), _lib.MKV_ERR_ARG),
    (dict(k_head_stride=1 << 61), _lib.MKV_ERR_ARG), (dict(lens=None), _lib.MKV_ERR_ARG),
    (dict(requests=4097), _lib.MKV_ERR_ARG), (dict(table_width=-1), _lib.MKV_ERR_ARG),
    (dict(tokens=0), _lib.MKV_OK), (dict(requests=0), _lib.MKV_OK)])
def test_store_rotated_refuses(change, code):
    assert _lib.lib().mkv_store_rotated(ctypes.byref(put_desc(**change)), None) == code


def shared_desc(n_groups=2, groups=1 << 20, shared=1 << 20, max_shared=0, **kw):
    d = _lib.AttendSharedDesc()
    d.attend = attend_desc(**kw)
    d.n_groups, d.groups, d.shared, d.max_shared = n_groups, groups, shared, max_shared
    return d


@pytest.mark.parametrize("change,code", BAD_CACHES + [
    (dict(n_groups=-1), _lib.MKV_ERR_ARG), (dict(n_groups=4097), _lib.MKV_ERR_ARG),
    (dict(groups=None), _lib.MKV_ERR_ARG), (dict(shared=None), _lib.MKV_ERR_ARG),
    (dict(max_shared=-1), _lib.MKV_ERR_ARG), (dict(dtype=_lib.MKV_F32), _lib.MKV_ERR_DTYPE),
    (dict(q_heads=3), _lib.MKV_ERR_ARG), (dict(softmax_scale=0.0), _lib.MKV_ERR_ARG),
    (dict(q=None), _lib.MKV_ERR_ARG), (dict(out=(1 << 20) + 2), _lib.MKV_ERR_ALIGN),
    (dict(out_head_stride=64), _lib.MKV_ERR_ARG), (dict(requests=5000), _lib.MKV_ERR_ARG),
    (dict(), _lib.MKV_ERR_ARG),  # no workspace
    (dict(tokens=1 << 28, q_heads=2, cache_heads=1), _lib.MKV_ERR_UNSUPPORTED)])
def test_attend_shared_refuses(change, code):
    change = dict(change)
    if "cache_heads" in change:
        change["heads"] = change.pop("cache_heads")
    desc = shared_desc(**change)
    assert _lib.lib().mkv_attend_shared(ctypes.byref(desc), None) == code
    assert _lib.lib().mkv_last_error()


def test_attend_shared_of_nothing_and_its_workspace():
    L = _lib.lib()

    def size(**kw):
        return L.mkv_attend_shared_workspace_size(ctypes.byref(shared_desc(**kw)))

    assert L.mkv_attend_shared(ctypes.byref(shared_desc(tokens=0)), None) == _lib.MKV_OK
    assert L.mkv_attend_shared(ctypes.byref(shared_desc(requests=0)), None) == _lib.MKV_OK
    assert L.mkv_attend_shared(None, None) == _lib.MKV_ERR_ARG
    assert L.mkv_attend_shared_workspace_size(None) == -1
    assert size(head_size=96) == -1 and size(tokens=0) == 0
    assert 0 < size() and size(n_groups=0, groups=None, shared=None) > 0


@pytest.mark.parametrize("d", [64, 128, 256])
@pytest.mark.parametrize("tokens,requests,group,groups", [
    (8192, 1, 4, 1), (8192, 1, 64, 1), (60000, 2, 1, 2), (2048, 32, 16, 4), (20000, 4096, 8, 4096)])
def test_a_small_hint_for_a_large_array_asks_for_a_bounded_workspace(tokens, requests, group, groups, d):
    """A row of D sums and its two statistics, 32 bits each: 8 * 4,096 parts of 32 rows, or 8 * 1,536
    of 128, or a part for each tile where there are more, for both ranges; and 16 bytes a row."""
    heads = 8
    desc = shared_desc(n_groups=groups, heads=heads, head_size=d, num_blocks=1 << 20, tokens=tokens,
                       requests=requests, q_heads=heads * group, table_width=1 << 16, max_new=1)
    tiles = (tokens * group / 16 + requests) * 16 * heads
    most = max(8 * max(4096 * 32, 1536 * 128), 2 * tiles)
    size = _lib.lib().mkv_attend_shared_workspace_size(ctypes.byref(desc))
    assert 0 < size <= 3 * most * (d + 2) * 4 + tokens * group * 16 + 64


def test_there_is_no_cpu_path():
    x = torch.zeros((2, 3, 64))
    with pytest.raises(RuntimeError, match="no CPU path"):
        norm_rotate(x, x, torch.zeros(2, dtype=torch.int32), torch.ones(32))
