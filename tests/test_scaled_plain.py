"""The block-scaled cache's host side without a GPU: the oracle that the GPU tests compare
with, the descriptors' layout, and every refusal that needs no device memory."""

from __future__ import annotations

import ctypes
import os
import subprocess

import numpy as np
import pytest
import torch

from marathon_amd import ScaledCache, _lib, step_slots
from tests import scaled_plain as plain

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def test_the_oracles_codec_is_e4m3fn():
    codes = torch.arange(256, dtype=torch.uint8)
    want = codes.view(torch.float8_e4m3fn).double().numpy()
    assert np.array_equal(plain.VALUES, want, equal_nan=True)
    x = np.concatenate((np.linspace(-448, 448, 40001), np.ldexp(np.linspace(-3, 3, 20001), -8)))
    x = x.astype(np.float32)
    got = torch.from_numpy(x).to(torch.float8_e4m3fn).view(torch.uint8).numpy()
    assert np.array_equal(plain.encode(x.astype(np.float64)), got)
    assert plain.encode(np.array([np.nan, np.inf, -1e9]))[:].tolist() == [0x7F, 0x7E, 0xFE]


def test_the_oracles_scale_is_the_least_that_fits():
    rng = np.random.default_rng(0)
    for top in [448.0, 448.0001, 447.0, 1.75, 1.7500001, 3e-38, 5e35, *np.exp2(rng.uniform(-60, 60, 200))]:
        e = plain.exponent_for(np.array([top, -top / 3, np.nan, np.inf]))
        if plain.LOW < e < plain.HIGH:
            assert top <= 448 * 2.0 ** e and top > 448 * 2.0 ** (e - 1)
    assert plain.exponent_for(np.zeros(3)) == plain.LOW
    assert plain.exponent_for(np.array([3e38])) == plain.HIGH


PROBE = r"""
#include <stddef.h>
#include <stdio.h>
#include "marathon_kvscaled.h"
#define O(T, f) printf(#T "." #f " %zu\n", offsetof(T, f))
int main(void) {
  printf("%zu %zu %zu\n", sizeof(mkv_scaled_cache_t), sizeof(mkv_attend_desc_t),
         sizeof(mkv_scaled_shift_desc_t));
@
  printf("limits %d %d %d\n", MKV_SCALE_MIN_EXP, MKV_SCALE_MAX_EXP, MKV_MAX_REQUESTS);
  for (int s = 16; s <= 128; s *= 2)
    for (int d = 16; d <= 128; d *= 2) printf("%d ", MKV_UNIT_WORDS(s, d));
  printf("\n");
  return 0;
}
"""
STRUCTS = {"mkv_scaled_cache_t": _lib.ScaledCacheDesc, "mkv_attend_desc_t": _lib.AttendDesc,
           "mkv_scaled_shift_desc_t": _lib.ScaledShiftDesc}


def test_descriptors_match_the_header(tmp_path):
    lines = "\n".join(f"  O({name}, {f[0]});" for name, s in STRUCTS.items() for f in s._fields_)
    src = tmp_path / "probe.c"
    src.write_text(PROBE.replace("@", lines))
    exe = tmp_path / "probe"
    subprocess.run(["gcc", "-std=c99", f"-I{os.path.join(ROOT, 'include')}", str(src), "-o",
                    str(exe)], check=True)
    out = subprocess.run([str(exe)], check=True, capture_output=True, text=True).stdout.split("\n")
    assert [int(x) for x in out[0].split()] == [ctypes.sizeof(s) for s in STRUCTS.values()]
    for line in out[1:]:
        if "." in line:
            field, at = line.split()
            name, f = field.split(".")
            assert getattr(STRUCTS[name], f).offset == int(at), field
    assert out[-3] == (f"limits {_lib.MKV_SCALE_MIN_EXP} {_lib.MKV_SCALE_MAX_EXP} "
                       f"{_lib.MKV_MAX_REQUESTS}")
    sizes = (16, 32, 64, 128)
    assert out[-2].split() == [str(_lib.unit_words(s, d)) for s in sizes for d in sizes]


def cache_desc(**kw):
    d = _lib.ScaledCacheDesc()
    d.k_base, d.v_base, d.scales = 1 << 20, (1 << 20) + 128, 1 << 24
    d.num_blocks, d.block_stride, d.head_stride, d.token_stride = 10, 16 * 2 * 256, 16 * 256, 256
    d.block_size, d.heads, d.head_size = 16, 2, 128
    for k, v in kw.items():
        setattr(d, k, v)
    return d


BAD_CACHES = [
    (dict(head_size=96), _lib.MKV_ERR_UNSUPPORTED), (dict(block_size=8), _lib.MKV_ERR_UNSUPPORTED),
    (dict(block_size=24), _lib.MKV_ERR_UNSUPPORTED), (dict(heads=0), _lib.MKV_ERR_ARG),
    (dict(num_blocks=-1), _lib.MKV_ERR_ARG), (dict(token_stride=250), _lib.MKV_ERR_ALIGN),
    (dict(head_stride=-16), _lib.MKV_ERR_ARG), (dict(k_base=None), _lib.MKV_ERR_ARG),
    (dict(v_base=(1 << 20) + 8), _lib.MKV_ERR_ALIGN), (dict(scales=(1 << 24) + 1), _lib.MKV_ERR_ALIGN),
    (dict(token_stride=1 << 32), _lib.MKV_ERR_UNSUPPORTED),
    (dict(head_stride=1 << 62), _lib.MKV_ERR_UNSUPPORTED),
    (dict(block_stride=1 << 62), _lib.MKV_ERR_UNSUPPORTED),
]


def attend_desc(**kw):
    d = _lib.AttendDesc()
    d.cache = cache_desc(**{k: kw.pop(k) for k in list(kw) if hasattr(_lib.ScaledCacheDesc, k)})
    d.q = d.out = d.starts = d.lens = d.block_tables = 1 << 20
    d.q_token_stride = d.out_token_stride = 512
    d.q_head_stride = d.out_head_stride = 128
    d.table_stride = d.table_width = 8
    d.tokens, d.requests, d.q_heads, d.dtype, d.softmax_scale = 3, 2, 4, _lib.MKV_BF16, 0.1
    for k, v in kw.items():
        setattr(d, k, v)
    return d


@pytest.mark.parametrize("change,code", BAD_CACHES + [
    (dict(dtype=_lib.MKV_F32), _lib.MKV_ERR_DTYPE), (dict(q_heads=3), _lib.MKV_ERR_ARG),
    (dict(q_heads=0), _lib.MKV_ERR_ARG), (dict(tokens=-1), _lib.MKV_ERR_ARG),
    (dict(tokens=1 << 31), _lib.MKV_ERR_ARG), (dict(requests=5000), _lib.MKV_ERR_ARG),
    (dict(requests=-1), _lib.MKV_ERR_ARG), (dict(starts=None), _lib.MKV_ERR_ARG),
    (dict(block_tables=None), _lib.MKV_ERR_ARG), (dict(table_width=-1), _lib.MKV_ERR_ARG),
    (dict(softmax_scale=0.0), _lib.MKV_ERR_ARG), (dict(softmax_scale=float("nan")), _lib.MKV_ERR_ARG),
    (dict(softmax_scale=1e6), _lib.MKV_ERR_ARG), (dict(max_new=-1), _lib.MKV_ERR_ARG),
    (dict(q=None), _lib.MKV_ERR_ARG), (dict(q=(1 << 20) + 2), _lib.MKV_ERR_ALIGN),
    (dict(out_head_stride=60), _lib.MKV_ERR_ALIGN), (dict(q_token_stride=-8), _lib.MKV_ERR_ARG),
    (dict(q_token_stride=1 << 60), _lib.MKV_ERR_ARG),
    (dict(max_len=100000, table_width=100000), _lib.MKV_ERR_ARG),  # no workspace
    (dict(table_width=1 << 27), _lib.MKV_ERR_UNSUPPORTED),
    (dict(tokens=1 << 23, q_heads=4), _lib.MKV_ERR_UNSUPPORTED),  # more tiles than a grid has
])
def test_attend_refuses(change, code):
    desc = attend_desc(**change)
    assert _lib.lib().mkv_attend_scaled(ctypes.byref(desc), None) == code
    assert _lib.lib().mkv_last_error()


def test_attend_of_nothing_and_its_workspace():
    L = _lib.lib()
    assert L.mkv_attend_scaled(ctypes.byref(attend_desc(tokens=0)), None) == _lib.MKV_OK
    assert L.mkv_attend_scaled(ctypes.byref(attend_desc(requests=0)), None) == _lib.MKV_OK
    assert L.mkv_attend_scaled(None, None) == _lib.MKV_ERR_ARG
    assert L.mkv_attend_workspace_size(None) == -1
    assert L.mkv_attend_workspace_size(ctypes.byref(attend_desc(head_size=96))) == -1
    assert L.mkv_attend_workspace_size(ctypes.byref(attend_desc(max_len=10))) == 0
    assert L.mkv_attend_workspace_size(
        ctypes.byref(attend_desc(max_len=100000, table_width=100000))) > 0


def store_args(cache=None, **kw):
    a = dict(cache=cache or cache_desc(), k=1 << 20, kt=256, kh=128, v=1 << 20, vt=256, vh=128,
             tokens=3, dtype=_lib.MKV_BF16, tables=1 << 20, stride=8, width=8, starts=1 << 20,
             lens=1 << 20, requests=2)
    a.update(kw)
    return [ctypes.byref(a.pop("cache")), *a.values(), None, None]


@pytest.mark.parametrize("change,code", BAD_CACHES)
def test_store_refuses_caches(change, code):
    assert _lib.lib().mkv_store_scaled(*store_args(cache_desc(**change))) == code


@pytest.mark.parametrize("change,code", [
    (dict(dtype=_lib.MKV_FP8_E4M3), _lib.MKV_ERR_DTYPE), (dict(tokens=-1), _lib.MKV_ERR_ARG),
    (dict(k=None), _lib.MKV_ERR_ARG), (dict(v=(1 << 20) + 4), _lib.MKV_ERR_ALIGN),
    (dict(kt=252), _lib.MKV_ERR_ALIGN), (dict(vh=-128), _lib.MKV_ERR_ARG),
    (dict(lens=None), _lib.MKV_ERR_ARG), (dict(requests=4097), _lib.MKV_ERR_ARG),
    (dict(tokens=0), _lib.MKV_OK), (dict(requests=0), _lib.MKV_OK)])
def test_store_refuses(change, code):
    assert _lib.lib().mkv_store_scaled(*store_args(**change)) == code


@pytest.mark.parametrize("change,code", [
    (dict(requests=4097), _lib.MKV_ERR_ARG), (dict(requests=-1), _lib.MKV_ERR_ARG),
    (dict(bs=0), _lib.MKV_ERR_ARG), (dict(width=-1), _lib.MKV_ERR_ARG),
    (dict(max_tokens=1 << 31), _lib.MKV_ERR_ARG), (dict(held=None), _lib.MKV_ERR_ARG),
    (dict(slots=None), _lib.MKV_ERR_ARG), (dict(out=1 << 20), _lib.MKV_ERR_ARG)])
def test_slots_refuse(change, code):
    p = 1 << 20
    a = dict(held=p, fresh=p, requests=2, tables=p, stride=4, width=4, free=p, free_len=9, at=p,
             bs=16, starts=p, lens=p, slots=p, positions=p, max_tokens=5, out=p + 64)
    a.update(change)
    assert _lib.lib().mkv_step_slots(*a.values(), None, None) == code


def shift_desc(src=None, dst=None, **kw):
    d = _lib.ScaledShiftDesc()
    d.src, d.dst = cache_desc(**(src or {})), cache_desc(**(dst or {}))
    for f in ("src_layers", "dst_layers", "units", "tables"):
        setattr(d, f, 1 << 20)
    d.n_units, d.n_spans, d.layers, d.rotary = 4, 2, 3, 128
    for k, v in kw.items():
        setattr(d, k, v)
    return d


@pytest.mark.parametrize("change,code", [
    (dict(src=dict(head_size=64)), _lib.MKV_ERR_ARG), (dict(dst=dict(heads=1)), _lib.MKV_ERR_ARG),
    (dict(src=dict(block_size=20)), _lib.MKV_ERR_UNSUPPORTED),
    (dict(rotary=16), _lib.MKV_ERR_UNSUPPORTED), (dict(rotary=160), _lib.MKV_ERR_UNSUPPORTED),
    (dict(rotary=-32), _lib.MKV_ERR_UNSUPPORTED), (dict(n_spans=5000), _lib.MKV_ERR_ARG),
    (dict(layers=70000), _lib.MKV_ERR_ARG), (dict(n_units=1 << 31), _lib.MKV_ERR_ARG),
    (dict(units=None), _lib.MKV_ERR_ARG), (dict(tables=None), _lib.MKV_ERR_ARG),
    (dict(tables=(1 << 20) + 4), _lib.MKV_ERR_ALIGN), (dict(units=(1 << 20) + 8), _lib.MKV_ERR_ALIGN),
    (dict(on_host=1, units=None), _lib.MKV_ERR_ARG),
    (dict(n_units=0), _lib.MKV_OK), (dict(layers=0), _lib.MKV_OK)])
def test_shift_refuses(change, code):
    assert _lib.lib().mkv_shift_scaled(ctypes.byref(shift_desc(**change)), None) == code


@pytest.mark.parametrize("span", [-2, 2, 1 << 30])
def test_shift_refuses_units_of_no_span(span):
    units, tables = np.zeros((3, 8), np.int32), np.zeros((2, 2, 128), np.float32)
    units[2, 2] = span
    desc = shift_desc(on_host=1, n_units=3, units=units.ctypes.data, tables=tables.ctypes.data)
    assert _lib.lib().mkv_shift_scaled(ctypes.byref(desc), None) == _lib.MKV_ERR_ARG


def units_of(rows, src_table, dst_table, sbs=16, dbs=16, blocks=(50, 60), room=None):
    """(status, units as int32 [n, words], flags)."""
    spans = np.zeros(len(rows), _lib.SPAN_DTYPE)
    for i, r in enumerate(rows):
        spans[i] = r
    st, dt = np.asarray(src_table, np.int32), np.asarray(dst_table, np.int32)
    room = sum(-(-max(r[4], 0) // dbs) for r in rows) if room is None else room
    words = _lib.unit_words(sbs, dbs)
    out, got = np.full((room + 1, words), 77, np.int32), np.zeros(2, np.int64)
    a, b = (cache_desc(block_size=s, num_blocks=n) for s, n in zip((sbs, dbs), blocks))
    rc = _lib.lib().mkv_scaled_units(
        spans.ctypes.data, len(rows), st.ctypes.data, st.size, dt.ctypes.data, dt.size,
        ctypes.byref(a), ctypes.byref(b), out.ctypes.data, room, got.ctypes.data, got.ctypes.data + 8)
    assert (out[room] == 77).all()
    return rc, out[:int(got[0])], int(got[1])


@pytest.mark.parametrize("sbs", [16, 32, 128])
@pytest.mark.parametrize("dbs", [16, 64, 128])
def test_units_name_every_rows_blocks(sbs, dbs):
    rng = np.random.default_rng(sbs + dbs)
    st, dt = rng.permutation(50), rng.permutation(60)
    rows = [(5, 2 * dbs, 3, 1, 2 * dbs + 7, 11, 0, 0), (sbs * 2, 8 * dbs, 0, 0, 1, 0, 0, 0),
            (0, 0, 0, 0, 0, 4, 0, 0)]
    rc, units, flags = units_of(rows, st, dt, sbs, dbs)
    assert rc == _lib.MKV_OK and flags == 0 and len(units) == 4
    k = 0
    for i, (sp, dp, si, di, n, delta, _, _) in enumerate(rows):
        for at in range(0, n, dbs):
            u = units[k]
            k += 1
            assert u[0] == dt[di + (dp + at) // dbs] and u[1] == min(dbs, n - at)
            assert u[2] == (i if delta else -1)
            for row in range(u[1]):
                p = sp + at + row
                assert u[4 + (u[3] + row) // sbs] == st[si + p // sbs]
                assert (u[3] + row) % sbs == p % sbs


def test_units_of_bad_spans_and_ids():
    table = np.arange(10)
    bad = [(0, 8, 0, 0, 4, 0, 0, 0), (-1, 0, 0, 0, 4, 0, 0, 0), (0, 0, 0, 0, -4, 0, 0, 0),
           (0, -16, 0, 0, 4, 0, 0, 0)]
    rc, units, flags = units_of(bad, table, table)
    assert rc == _lib.MKV_OK and len(units) == 0 and flags == _lib.MKV_FLAG_SPAN
    rc, units, flags = units_of([(0, 0, 0, 0, 40, 0, 0, 0)], table, [1, 60, -1])
    assert flags == _lib.MKV_FLAG_DST_RANGE and units[:, 0].tolist() == [1]
    rc, units, flags = units_of([(8, 0, 0, 0, 32, 0, 0, 0)], [3, 50], table)
    assert flags == _lib.MKV_FLAG_SRC_RANGE
    assert units[:, 4:6].tolist() == [[3, -1], [-1, -1]]
    rc, units, flags = units_of([(2**62, 0, 2**62, 2**62, 20, 0, 0, 0)], table, table)
    assert flags == _lib.MKV_FLAG_DST_RANGE and len(units) == 0
    rc, units, flags = units_of([(2**63 - 5, 0, 2**63 - 1, 0, 20, 0, 0, 0)], table, table)
    assert flags == _lib.MKV_FLAG_SPAN and len(units) == 0
    assert units_of([(0, 0, 0, 0, 40, 0, 0, 0)], table, table, room=2)[0] == _lib.MKV_ERR_ARG
    assert units_of([], [], [])[0] == _lib.MKV_OK


def test_units_refuse_a_block_twice():
    table = np.arange(10)
    rows = [(0, 0, 0, 0, 40, 0, 0, 0), (50, 64, 0, 0, 16, 0, 0, 0)]
    assert units_of(rows, table, [9, 8, 7, 5, 6])[0] == _lib.MKV_OK
    assert units_of(rows, table, [9, 8, 7, 5, 8])[0] == _lib.MKV_ERR_ARG
    assert units_of([rows[0], rows[0]], table, table)[0] == _lib.MKV_ERR_ARG


def test_units_of_one_cache_refuse_a_source_that_is_written():
    cache, out = cache_desc(num_blocks=12), np.zeros((8, 8), np.int32)
    spans, got = np.zeros(1, _lib.SPAN_DTYPE), np.zeros(2, np.int64)
    spans[0] = (9, 0, 0, 0, 31, 5, 0, 0)  # of blocks 0, 1 and 2 of its table

    def rc(dst, src_desc):
        st, dt = np.asarray([3, 4, 5, 6], np.int32), np.asarray(dst, np.int32)
        return _lib.lib().mkv_scaled_units(
            spans.ctypes.data, 1, st.ctypes.data, 4, dt.ctypes.data, 2, ctypes.byref(src_desc),
            ctypes.byref(cache), out.ctypes.data, 8, got.ctypes.data, got.ctypes.data + 8)

    for dst, code in (([0, 11], _lib.MKV_OK), ([6, 2], _lib.MKV_OK), ([0, 3], _lib.MKV_ERR_ARG),
                      ([5, 11], _lib.MKV_ERR_ARG), ([4, 0], _lib.MKV_ERR_ARG)):
        assert rc(dst, cache) == code
        assert rc(dst, cache_desc(num_blocks=12)) == _lib.MKV_OK


def test_there_is_no_cpu_path():
    kv = torch.zeros((4, 2, 16, 256), dtype=torch.uint8).view(torch.float8_e4m3fn)
    scales = torch.zeros((4, 2, 2), dtype=torch.uint8).view(torch.float8_e8m0fnu)
    with pytest.raises(RuntimeError, match="no CPU path"):
        ScaledCache(kv, scales, "hnd")
    t = torch.zeros((1, 2), dtype=torch.int32)
    with pytest.raises(RuntimeError, match="no CPU path"):
        step_slots(t[:, 0], t[:, 0], t, t[0], t[0, :1], 16, 4)
