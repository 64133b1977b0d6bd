"""The int8 key/value cache's entry points refuse what they cannot do, before
they touch the device (none is needed here), and the Python mirror of the
cache's struct agrees with the header."""

import ctypes
import subprocess

import pytest
import torch

from accelep_b200 import kernels as K
from accelep_b200._lib import Q8CacheStruct
from tests.conftest import ROOT

P = 1 << 20  # an aligned address that is never read


def cache(**change):
    d = {"k": P, "v": 2 * P, "k_scale": 3 * P, "v_scale": 4 * P, "seq_stride": 2 * 100 * 64, "head_stride": 100 * 64,
         "scale_seq_stride": 4, "scale_head_stride": 2, "slots": 3, "kv_heads": 2, "head_dim": 64, "context": 100,
         "block": 64}
    d.update(change)
    return ctypes.byref(Q8CacheStruct(*[d[name] for name, _ in Q8CacheStruct._fields_]))


BAD_CACHES = [{"k": None}, {"v_scale": None}, {"head_dim": 96}, {"head_dim": 32}, {"block": 16}, {"block": 0},
              {"block": 48}, {"slots": 0}, {"kv_heads": 0}, {"context": 0}, {"k": P + 8}, {"v_scale": P + 2}, {"v": P}, {"v_scale": 3 * P},
              {"head_stride": 99 * 64}, {"seq_stride": 100 * 64}, {"seq_stride": 2 * 100 * 64 + 8},
              {"scale_head_stride": 1}, {"scale_seq_stride": 3}, {"head_stride": -100 * 64},
              {"seq_stride": 64 << 56}, {"head_stride": 64 << 56, "seq_stride": 64 << 57},
              {"seq_stride": 64 << 30}, {"seq_stride": 64 << 55, "slots": 1 << 10},
              {"v": P + 99 * 64}, {"v": P - 64}, {"v": P + 5 * 100 * 64}, {"v": P + 2 * 2 * 100 * 64 + 16},
              {"v_scale": 3 * P + 4}, {"v_scale": 3 * P - 4 * 11}]


def append(lib, c, **change):
    d = {"qkv": P, "ld": 8 * 64, "rows": 5, "first": P, "count": P, "pos0": P, "batch": 3, "max_rows": 4, "heads": 4,
         "cos": P, "sin": P, "q": 5 * P, "q_ld": 4 * 64}
    d.update(change)
    return lib.accel_b200_rope_append_q8(d["qkv"], d["ld"], d["rows"], c, d["first"], d["count"], d["pos0"],
                                         d["batch"], d["max_rows"], d["heads"], d["cos"], d["sin"], d["q"], d["q_ld"],
                                         None, None)


def read(lib, c, **change):
    d = {"first": P, "count": P, "pos0": P, "batch": 3, "max_rows": 4, "k": P, "v": 2 * P, "ld": 128, "rows": 5}
    d.update(change)
    return lib.accel_b200_cache_rows_q8(c, d["first"], d["count"], d["pos0"], d["batch"], d["max_rows"], d["k"],
                                        d["v"], d["ld"], d["rows"], None, None)


def decode(lib, c, **change):
    d = {"q": P, "ld": 256, "seq": None, "pos": P, "rows": 3, "heads": 4, "window": 0, "sinks": 0, "out": 2 * P,
         "out_ld": 256}
    d.update(change)
    return lib.accel_b200_attention_decode_q8(d["q"], d["ld"], c, d["seq"], d["pos"], d["rows"], d["heads"],
                                              d["window"], d["sinks"], d["out"], d["out_ld"], None, 0, None, None)


def prefill(lib, c, **change):
    d = {"q": P, "ld": 256, "first": P, "count": P, "pos0": P, "batch": 3, "max_rows": 4, "rows": 5, "heads": 4,
         "window": 0, "sinks": 0, "out": 2 * P, "out_ld": 256}
    d.update(change)
    return lib.accel_b200_attention_prefill_q8(d["q"], d["ld"], c, d["first"], d["count"], d["pos0"], d["batch"],
                                               d["max_rows"], d["rows"], d["heads"], d["window"], d["sinks"],
                                               d["out"], d["out_ld"], None, 0, None, None)


@pytest.mark.parametrize("change", BAD_CACHES, ids=str)
@pytest.mark.parametrize("call", [append, read, decode, prefill])
def test_bad_caches_are_refused(lib, call, change):
    assert call(lib, cache(**change)) == 1
    assert lib.accel_b200_last_error()
    assert call(lib, None) == 1


@pytest.mark.parametrize("call,change", [
    (append, {"qkv": None}), (append, {"q": None}), (append, {"pos0": None}), (append, {"cos": None}),
    (append, {"rows": -1}), (append, {"batch": -1}), (append, {"batch": 4}), (append, {"heads": 3}),
    (append, {"heads": 0}), (append, {"ld": 7 * 64}), (append, {"q_ld": 4 * 64 - 4}), (append, {"ld": 8 * 64 + 2}),
    (append, {"qkv": P + 4}), (append, {"q": P + 8}), (append, {"max_rows": -1}),
    (append, {"q": P}), (append, {"q": P + 16, "q_ld": 8 * 64}), (append, {"q": P + 4 * 512, "q_ld": 512}),
    (append, {"q": P - 4 * 128, "q_ld": 512}), (read, {"v": P}), (read, {"v": P + 64}), (read, {"v": P + 4 * 128}),
    (decode, {"out": P + 64}), (decode, {"out": P, "out_ld": 512}), (prefill, {"out": P + 4 * 256}),
    (read, {"first": None}), (read, {"batch": 4}), (read, {"ld": 124}), (read, {"ld": 130}), (read, {"k": P + 4}),
    (read, {"rows": -2}),
    (decode, {"q": None}), (decode, {"pos": None}), (decode, {"rows": 4}), (decode, {"rows": -1}),
    (decode, {"rows": 65536, "seq": P}), (decode, {"heads": 5}), (decode, {"window": -1}), (decode, {"sinks": -1}),
    (decode, {"ld": 252}), (decode, {"out_ld": 258}), (decode, {"out": P + 4}),
    (prefill, {"count": None}), (prefill, {"batch": 4}), (prefill, {"heads": 6 + 1}), (prefill, {"window": -5}),
    (prefill, {"out": None}), (prefill, {"rows": -1}), (prefill, {"out_ld": 128}),
], ids=str)
def test_bad_arguments_are_refused(lib, call, change):
    assert call(lib, cache(), **change) == 1
    assert lib.accel_b200_last_error()


def test_overlaps_that_are_taken(lib):
    """In place, and other columns of the same rows (no rows: nothing runs)."""
    assert append(lib, cache(), q=P, q_ld=512, max_rows=0) == 0
    assert append(lib, cache(), ld=1024, q=P + 4 * 512, q_ld=1024, max_rows=0) == 0
    assert append(lib, cache(), qkv=P + 4 * 256, ld=1024, q=P, q_ld=1024, max_rows=0) == 0
    assert read(lib, cache(), ld=256, v=P + 4 * 128, max_rows=0) == 0
    assert prefill(lib, cache(), out=P, max_rows=0) == 0


def test_empty_calls_queue_nothing(lib):
    before = lib.accel_b200_launch_count()
    for empty in ({"batch": 0}, {"max_rows": 0}, {"rows": 0}):
        assert append(lib, cache(), **empty) == 0
        assert read(lib, cache(), **empty) == 0
        assert prefill(lib, cache(), **empty) == 0
    assert read(lib, cache(), k=None, v=None) == 0
    assert decode(lib, cache(), rows=0) == 0
    assert lib.accel_b200_launch_count() == before


@pytest.mark.parametrize("order", [
    {"seq_stride": 100 * 64, "head_stride": 3 * 100 * 64, "scale_seq_stride": 2, "scale_head_stride": 6},  # heads outside
    {"slots": 1, "seq_stride": 0, "scale_seq_stride": 0},       # one slot: its stride is never used
    {"kv_heads": 1, "head_stride": 0, "scale_head_stride": 0},  # one head: the same
    # Keys and values by turns: of each (slot, head), of each slot, of all.
    {"v": P + 100 * 64, "head_stride": 2 * 100 * 64, "seq_stride": 4 * 100 * 64, "v_scale": 3 * P + 8,
     "scale_head_stride": 4, "scale_seq_stride": 8},
    {"v": P - 2 * 100 * 64, "seq_stride": 4 * 100 * 64, "v_scale": 3 * P + 16, "scale_seq_stride": 8},
    {"v": P + 6 * 100 * 64, "v_scale": 3 * P - 48},
    {"v": P + 64 * 100, "seq_stride": 64 << 29, "slots": 4, "head_stride": 64 << 27},
])
def test_other_orders_of_the_cache_are_taken(lib, order):
    batch = {"batch": min(3, order.get("slots", 3)), "max_rows": 0}
    assert append(lib, cache(**order), **batch) == 0
    assert prefill(lib, cache(**order), **batch) == 0


def test_struct_layout_matches_the_header(tmp_path):
    lines = ['#include <stddef.h>', '#include <stdio.h>', '#include "accel_b200.h"', "int main(void) {",
             '  printf("size %zu\\n", sizeof(accel_b200_q8_cache));']
    lines += [f'  printf("{f} %zu\\n", offsetof(accel_b200_q8_cache, {f}));' for f, _ in Q8CacheStruct._fields_]
    src, exe = tmp_path / "layout.c", tmp_path / "layout"
    src.write_text("\n".join(lines + ["  return 0;", "}"]) + "\n")
    subprocess.run(["gcc", "-std=c11", f"-I{ROOT / 'include'}", "-I/usr/local/cuda/include", str(src), "-o", str(exe)],
                   check=True, capture_output=True, text=True)
    for line in subprocess.run([str(exe)], check=True, capture_output=True, text=True).stdout.splitlines():
        name, value = line.split()
        want = ctypes.sizeof(Q8CacheStruct) if name == "size" else getattr(Q8CacheStruct, name).offset
        assert int(value) == want, name


def test_python_cache_refuses_host_tensors():
    k = torch.zeros(1, 1, 8, 64, dtype=torch.int8)
    s = torch.zeros(1, 1, 1)
    with pytest.raises(ValueError):
        K.Q8Cache(k, k.clone(), s, s.clone())


@pytest.mark.parametrize("block", [0, -64, 16, 65])
def test_python_cache_refuses_other_blocks(block):
    k, s = torch.zeros(1, 1, 8, 64, dtype=torch.int8), torch.zeros(1, 1, 1)
    with pytest.raises(ValueError, match="block"):
        K.Q8Cache(k, k.clone(), s, s.clone(), block)
    with pytest.raises(ValueError, match="block"):
        K.Q8Cache.zeros(1, 1, 8, 64, block, device="cpu")


def test_python_rows_of_one_have_no_stride():
    """One row of a wider tensor, whatever its stride there."""
    wide = torch.zeros(3, 131)
    assert K._rows("x", wide[1:2, :128], -1, 128) == (1, 128)
    assert K._rows("x", wide[:1, :128], -1, 128) == K._rows("x", torch.zeros(1, 128), -1, 128)
    assert K._rows("x", torch.zeros(1, 128).expand(1, 128), -1, 128) == (1, 128)
    assert K._rows("x", wide[:0, :128], -1, 128) == (0, 128)
    assert K._rows("x", torch.zeros(3, 136)[:, :128], -1, 128) == (3, 136)


def test_prefill_without_a_device_says_so(lib):
    """The tile kernel's registers cannot be asked for without a device: the
    call gives CUDA's error, not one about the registers."""
    if torch.cuda.is_available():
        pytest.skip("there is a device")
    big = cache(k=1 << 30, v=1 << 31, k_scale=1 << 32, v_scale=1 << 33, context=512, seq_stride=2 * 512 * 64,
                head_stride=512 * 64, scale_seq_stride=16, scale_head_stride=8)
    for _ in range(2):
        assert prefill(lib, big, heads=16, ld=1024, out=1 << 34, out_ld=1024, max_rows=512) == 3
        assert b"CUDA" in lib.accel_b200_last_error() and b"registers" not in lib.accel_b200_last_error()


def test_which_kernel_a_prefill_takes(lib):
    """By sizes alone; bad sizes: 0."""
    def tiles(c, batch, rows, heads, window=0, sinks=0):
        return lib.accel_b200_attention_prefill_q8_tiles(c, batch, rows, heads, window, sinks)

    c = cache()
    assert tiles(c, 3, 100, 4) == 0  # 3 x 2 x 25 groups
    assert tiles(c, 3, 100, 64) == 1  # 3 x 2 x 400
    assert tiles(c, 3, 1 << 30, 64) == tiles(c, 3, 100, 64)  # a run is no longer than the context
    long = cache(context=1 << 16, seq_stride=2 << 22, head_stride=1 << 22, scale_seq_stride=2048, scale_head_stride=1024,
                 k=1 << 30, v=1 << 31, k_scale=1 << 32, v_scale=1 << 33)
    assert tiles(long, 1, 4000, 8) == 1 and tiles(long, 1, 1, 8) == 0
    for bad in ((0, 5, 4), (1, 0, 4), (1, 5, 3), (1, 5, 0), (1, 5, 4, -1), (1, 5, 4, 0, -1)):
        assert tiles(c, *bad) == 0
    assert tiles(None, 1, 5, 4) == 0 and tiles(cache(block=16), 3, 100, 64) == 0
