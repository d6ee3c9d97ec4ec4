"""The paged int8 KV cache without a GPU: its index rules (csrc/paged.hpp)
compiled for the host, the 64-bit restatement that the GPU tests compare with,
and the refusals of its entry points."""
import ctypes as C
import functools
import os
import subprocess
import tempfile

import numpy as np
import pytest

import paged_ref as R
from gpu_util import ROOT, nnhip

I32 = 2 ** 31 - 1


@functools.lru_cache(None)
def rules():
    with tempfile.TemporaryDirectory() as d:
        lib = os.path.join(d, "paged_rules.so")
        subprocess.check_call(
            ["g++", "-std=c++17", "-Wall", "-Werror", "-shared", "-fPIC",
             "-I", os.path.join(ROOT, "neural-network_amd", "csrc"),
             os.path.join(ROOT, "tests", "cpp", "paged_rules.cpp"), "-o", lib])
        L = C.CDLL(lib)
    L.block_scale.restype, L.block_scale.argtypes = C.c_double, [C.c_double]
    L.head_offset.restype = C.c_longlong
    L.request_len.restype = C.c_longlong
    L.tables_status.argtypes = [C.c_int, C.c_void_p, C.c_void_p, C.c_void_p, C.c_int, C.c_int,
                                C.c_longlong, C.c_longlong, C.c_int]
    return L


def test_block_sizes():
    assert [rules().log2_block(b) for b in (16, 32, 64, 128)] == [4, 5, 6, 7]
    assert all(rules().log2_block(b) < 0 for b in (0, 1, 8, 24, 48, 256, -16))


@pytest.mark.parametrize("x", [1e-45, 2.0 ** -126, 127 * 2.0 ** -126, 1e-30, 0.5, 1.0, 126.9,
                               127.0, 127.0000001, 127.5, 128.0, 254.0, 254.1, 3.4e38, 4.8e38])
def test_scale_of_a_block(x):
    s = rules().block_scale(x)
    assert s == R.block_scale(x)
    assert x <= 127 * s and s >= 2.0 ** -126
    assert s == 2.0 ** -126 or x > 127 * s / 2
    assert np.isfinite(np.float32(s)) and float(np.float32(s)) == s


def test_scale_of_zeros():
    assert rules().block_scale(0.0) == 0.0 == R.block_scale(0.0)


@pytest.mark.parametrize("slot,ok", [(-1, 0), (0, 1), (159, 1), (160, 0), (I32, 0), (-I32 - 1, 0)])
def test_slots_outside_the_pool(slot, ok):
    assert rules().slot_ok(10, 16, slot) == ok


@pytest.mark.parametrize("block,ok", [(-1, 0), (0, 1), (9, 1), (10, 0), (I32, 0), (-I32 - 1, 0)])
def test_blocks_outside_the_pool(block, ok):
    assert rules().block_ok(block, 10) == ok


def test_every_code_lies_in_its_pool():
    for bs in (16, 32, 64, 128):
        for D in (32, 64, 128):
            seen = [rules().head_offset(5, bs, 3, D, b, kv, h)
                    for b in range(5) for kv in range(2) for h in range(3)]
            assert seen == [i * bs * D for i in range(30)]


def test_offsets_pass_32_bits():
    # the last block of a pool of 2^31 - 64 slots
    assert rules().head_offset(I32 // 64, 64, 8, 128, I32 // 64 - 1, 1, 7) == \
        ((I32 // 64 - 1) * 16 + 15) * 64 * 128


@pytest.mark.parametrize("a,z,want", [(0, 3, (0, 3)), (2, 9, (2, 5)), (-4, 2, (0, 2)),
                                      (4, 1, (4, 4)), (7, 9, (5, 5)), (3, -8, (3, 3)),
                                      (-9, -2, (0, 0)), (I32, -I32, (5, 5))])
def test_rows_are_cut_to_the_call(a, z, want):
    out = (C.c_int * 2)()
    rules().request_rows((C.c_int * 2)(a, z), 0, 5, out)
    assert tuple(out) == want


@pytest.mark.parametrize("n,want", [(-3, 0), (0, 0), (47, 47), (48, 48), (49, 48), (I32, 48)])
def test_lengths_are_cut_to_the_table(n, want):
    assert rules().request_len(n, 3, 4) == want


def _status(cached, added, held, room, free, blocks, bs=16, mb=4):
    a = [np.asarray(x, np.int32) for x in (cached, added, held)]
    return rules().tables_status(len(cached), *(x.ctypes.data_as(C.c_void_p) for x in a), bs, mb,
                                 room, free, blocks)


@pytest.mark.parametrize("want,cached,added,held,room,free,blocks", [
    (0, [5, 0], [1, 20], [1, 0], 21, 2, 4),
    (1, [-1, 0], [1, 1], [0, 0], 9, 4, 4),
    (1, [70, 0], [1, -1], [0, 0], 9, 4, 4),       # before 2
    (2, [60, 0], [5, 1], [4, 0], 9, 4, 8),
    (2, [I32, 0], [I32, 1], [4, 0], 9, 4, 8),
    (3, [0, 0], [20, 20], [0, 0], 39, 1, 4),      # before 4
    (4, [0, 0], [20, 20], [0, 0], 40, 3, 4),
    (0, [0, 0], [20, 20], [0, 0], 40, 4, 4),
    (0, [0, 0], [20, 40], [2, 1], 60, 2, 5),      # what is held counts
    (0, [0, 0], [64, 0], [0, 4], 64, 0, 4),       # what is returned is taken again
    (5, [0], [1], [-1], 1, 1, 4), (5, [0], [1], [5], 1, 1, 8), (5, [0], [1], [0], 1, -1, 4),
    (5, [0], [0], [2], 0, 3, 4)])
def test_status_of_a_step(want, cached, added, held, room, free, blocks):
    assert _status(cached, added, held, room, free, blocks) == want
    t = R.Tables(len(cached), 4, blocks, 16)
    t.held[:], t.count = held, free
    assert t.status(np.array(cached), np.array(added), room) == want


def test_a_step_taken_back_restores_the_stack():
    rng = np.random.default_rng(3)
    t = R.Tables(5, 9, 40, 16, rng)
    t.step(np.zeros(5, np.int32), np.array([3, 0, 60, 16, 17], np.int32), 96)
    free, count, held = t.free.copy(), t.count, t.held.copy()
    lens = np.array([3, 0, 60, 16, 17], np.int32)
    assert t.step(lens, np.array([20, 40, 5, 1, 0], np.int32), 66)[0] == 0
    assert t.count < count
    t.step(lens, np.zeros(5, np.int32), 0)
    assert t.count == count and (t.free[:count] == free[:count]).all() and (t.held == held).all()


# -------------------------------------------------------------- refusals ----
# Every check comes before the context is used, so no pointer here is followed.
P = C.c_void_p(4096)
ODD = C.c_void_p(4100)

TABLES = dict(ctx=None, B=2, cached=P, added=P, block_size=16, max_blocks=4, tables=P, held=P,
              num_blocks=8, free_list=P, free_count=P, T=3, row_start=P, lens=P, pos=P, slots=P,
              status=P)
APPEND = dict(ctx=None, qkv=P, T=3, H=4, Hkv=2, D=64, pos=P, slots=P, cos=P, sin=P, n_pos=10,
              q_out=P, codes=P, scales=P, block_size=16, num_blocks=8)
ATTENTION = dict(ctx=None, q=P, T=3, codes=P, scales=P, block_size=16, num_blocks=8, tables=P,
                 max_blocks=4, row_start=P, lens=P, B=2, H=4, Hkv=2, D=64, out=P)
READ = dict(ctx=None, codes=P, scales=P, block_size=16, num_blocks=8, slots=P, T=3, Hkv=2, D=64,
            k=P, v=P)
OPS = {"nnhip_block_tables": TABLES, "nnhip_rope_kv_append_paged_q8": APPEND,
       "nnhip_attention_paged_q8": ATTENTION, "nnhip_kv_read_paged_q8": READ}

SIZES = [("block_size", 0, "block_size"), ("block_size", 24, "block_size"),
         ("block_size", 256, "block_size"), ("num_blocks", 0, "num_blocks"),
         ("num_blocks", -1, "num_blocks"), ("num_blocks", 2 ** 27, "num_blocks"),
         ("T", -1, "negative"), ("B", 0, "B must be"), ("B", 4097, "B must be"),
         ("max_blocks", 0, "max_blocks"), ("max_blocks", 2 ** 27, "max_blocks"),
         ("H", 3, "H must be"), ("H", 0, "H must be"), ("Hkv", 0, "Hkv"), ("Hkv", -2, "Hkv"),
         ("D", 0, "head dim"), ("D", 48, "head dim"), ("D", 256, "head dim"),
         ("n_pos", 0, "n_pos"), ("cos", None, "cos and sin"), ("sin", None, "cos and sin"),
         ("qkv", ODD, "aligned"), ("q_out", ODD, "aligned"), ("codes", ODD, "aligned"),
         ("q", ODD, "aligned"), ("out", ODD, "aligned"), ("k", ODD, "aligned"),
         ("v", ODD, "aligned"), ("cos", ODD, "aligned"), ("scales", C.c_void_p(4097), "aligned")]


@pytest.mark.skipif(not os.path.exists(nnhip.LIB_PATH), reason="libnnhip.so not built")
@pytest.mark.parametrize("op", OPS)
def test_refusals(op):
    good = OPS[op]
    tried = 0
    for name, value, text in SIZES:
        if name not in good:
            continue
        if name == "cos" and value is ODD:
            value = C.c_void_p(4098)
        with pytest.raises(nnhip.NNHipError, match=text) as e:
            nnhip.call(op, *dict(good, **{name: value}).values())
        assert e.value.code == (nnhip.EUNSUPPORTED if name == "D" else nnhip.EARG), name
        tried += 1
    # each pointer missing, and the context
    for name, value in good.items():
        if value is P and name not in ("cos", "sin"):
            with pytest.raises(nnhip.NNHipError, match="NULL") as e:
                nnhip.call(op, *dict(good, **{name: None}).values())
            assert e.value.code == nnhip.EARG
            tried += 1
    with pytest.raises(nnhip.NNHipError, match="NULL"):
        nnhip.call(op, *good.values())
    assert tried >= 9
