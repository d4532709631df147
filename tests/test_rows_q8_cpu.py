"""The 8-bit kept rows' host-side checks: every call that must not reach the GPU is refused before anything is
launched, and the workspace sizes add up."""
import ctypes as C

import pytest


@pytest.fixture(scope="module")
def world():
    from tessera_b200 import _lib
    raw = (C.c_char * 4096)()
    p = (C.addressof(raw) + 255) // 256 * 256
    good = _lib.TsRowsQ8(p, p, p, p, p, 16, 8)
    paged = _lib.TsKept(2, 64, 2, p, 4, 128)
    return _lib, raw, p, good, paged


def refused(_lib, rc, text):
    assert rc == _lib.TS_ERR_BAD_INPUT and text.encode() in _lib.lib.ts_last_error(), _lib.lib.ts_last_error()


def calls(world, kv, kept, width=64, kv_heads=2, p=None):
    _lib, _, base, _, _ = world
    p = base if p is None else p
    lib = _lib.lib
    return [
        lib.ts_qk_norm_rope_append_q8(p, None, None, p, p, p, p, kv, kept, 1, 4, kv_heads, width, 1e-6, None),
        lib.ts_rows_unpack_q8(kv, p, p, p, p, kept, 1, kv_heads, width, None),
        lib.ts_attend_rows_q8(p, kv, p, p, p, kept, 1, 64, 4, kv_heads, width, 0xFFFFFFFF, 1.0, None, 0, None),
        lib.ts_select_blocks_q8(p, kv, p, p, p, kept, 1, 64, 4, kv_heads, width, 1, 0, 0, None, 0, None),
        lib.ts_attend_blocks_q8(p, kv, p, p, p, p, kept, 1, 64, 4, kv_heads, width, 1, 1.0, None, 0, None),
    ]


def test_records_that_describe_no_rows_are_refused(world):
    _lib, raw, p, good, paged = world
    R, K = _lib.TsRowsQ8, _lib.TsKept
    cases = [
        (R(None, p, p, p, p, 16, 8), paged, 64, 2, "NULL"),
        (R(p, p, None, p, p, 16, 8), paged, 64, 2, "NULL"),
        (R(p + 8, p, p, p, p, 16, 8), paged, 64, 2, "16-byte aligned"),
        (R(p, p, p, p, p + 8, 16, 8), paged, 64, 2, "16-byte aligned"),
        (R(p, p, p + 2, p, p, 16, 8), paged, 64, 2, "4-byte aligned"),
        (R(p, p, p, p, p, 8, 8), paged, 64, 2, "16, 32 or 64"),
        (R(p, p, p, p, p, 128, 8), paged, 64, 2, "16, 32 or 64"),
        (R(p, p, p, p, p, 0, 8), paged, 64, 2, "16, 32 or 64"),
        (R(p, p, p, p, p, 16, 0), paged, 64, 2, "block count"),
        (good, paged, 96, 2, "64, 128 or 256"),
        (good, paged, 64, 0, "kv heads"),
        (good, K(1, 64, 2, p, 4, 128), 64, 2, "dense or a paged"),
        (good, K(9, 64, 2, p, 4, 128), 64, 2, "dense or a paged"),
        (good, K(0, 1, 40, None, 0, 128), 64, 2, "multiple of the block"),
        (good, K(0, 1, 0, None, 0, 128), 64, 2, "multiple of the block"),
        (good, K(2, 8, 2, p, 4, 128), 64, 2, "whole blocks"),
        (good, K(2, 48, 2, p, 4, 128), 64, 2, "whole blocks"),
        (good, K(2, 64, 2, None, 4, 128), 64, 2, "page table"),
        (good, K(2, 64, 2, p, 0, 128), 64, 2, "page table"),
        (good, K(2, 64, 0, p, 4, 128), 64, 2, "page table"),
    ]
    for kv, kept, width, kv_heads, text in cases:
        for i in range(5):
            rc = calls(world, kv, kept, width, kv_heads)[i]
            assert rc == _lib.TS_ERR_BAD_INPUT
        refused(_lib, _lib.lib.ts_rows_unpack_q8(kv, p, p, p, p, kept, 1, kv_heads, width, None), text)
    for rc in calls(world, None, paged):
        assert rc == _lib.TS_ERR_BAD_INPUT
    for rc in calls(world, good, None):
        assert rc == _lib.TS_ERR_BAD_INPUT


def test_buffers_and_counts_are_checked(world):
    _lib, raw, p, good, paged = world
    lib = _lib.lib
    refused(_lib, lib.ts_qk_norm_rope_append_q8(None, None, None, p, p, p, p, good, paged, 1, 4, 2, 64, 1e-6, None), "NULL")
    refused(_lib, lib.ts_qk_norm_rope_append_q8(p, None, None, None, p, p, p, good, paged, 1, 4, 2, 64, 1e-6, None), "NULL")
    refused(_lib, lib.ts_qk_norm_rope_append_q8(p + 2, None, None, p, p, p, p, good, paged, 1, 4, 2, 64, 1e-6, None), "aligned")
    refused(_lib, lib.ts_qk_norm_rope_append_q8(p, None, None, p, p, p, p, good, paged, 1, 0, 2, 64, 1e-6, None), "heads")
    refused(_lib, lib.ts_rows_unpack_q8(good, p, p, None, p, paged, 1, 2, 64, None), "NULL")
    refused(_lib, lib.ts_attend_rows_q8(p, good, None, p, p, paged, 1, 64, 4, 2, 64, 0, 1.0, None, 0, None), "NULL")
    refused(_lib, lib.ts_attend_rows_q8(p, good, p, p, p, paged, 1, 64, 5, 2, 64, 0, 1.0, None, 0, None), "split over")
    refused(_lib, lib.ts_attend_rows_q8(p, good, p, p, p, paged, 1, 64, 0, 2, 64, 0, 1.0, None, 0, None), "split over")
    long = _lib.TsKept(2, 64, 2000, p, 4, 128)
    refused(_lib, lib.ts_attend_rows_q8(p, good, p, p, p, long, 1, 100000, 4, 2, 64, 0xFFFFFFFF, 1.0, None, 0, None), "workspace")
    refused(_lib, lib.ts_attend_blocks_q8(p, good, None, p, p, p, paged, 1, 64, 4, 2, 64, 1, 1.0, None, 0, None), "ids")
    refused(_lib, lib.ts_attend_blocks_q8(p, good, p, p, p, p, paged, 1, 64, 4, 2, 64, 0, 1.0, None, 0, None), "1 to")
    bare = _lib.TsRowsQ8(p, p, p, p, None, 16, 8)
    refused(_lib, lib.ts_select_blocks_q8(p, bare, p, p, p, paged, 1, 64, 4, 2, 64, 1, 0, 0, None, 0, None), "bounds")
    for count, first, recent in ((0, 0, 0), (4097, 0, 0), (2, 2, 1), (2, 0, 3), (2, 3, 0), (2, 0xFFFFFFFF, 3)):
        refused(_lib, lib.ts_select_blocks_q8(p, good, p, p, p, paged, 1, 64, 4, 2, 64, count, first, recent, None, 0, None), "blocks (1 to 4096)")
    refused(_lib, lib.ts_select_blocks_q8(p, good, p, p, p, paged, 1, 64, 514, 2, 64, 1, 0, 0, None, 0, None), "at most 256")
    refused(_lib, lib.ts_select_blocks_q8(p, good, p, p, p, long, 1, 100000, 4, 2, 64, 2, 0, 0, None, 0, None), "workspace")
    for i in range(5):  # gains, frequencies, slots, positions, ids, page table
        o = [p + 2 if k == i else p for k in range(5)]
        refused(_lib, lib.ts_qk_norm_rope_append_q8(p, *o, p + 2048, good, paged, 1, 4, 2, 64, 1e-6, None), "4-byte")
    for i in range(2):
        o = [p + 2 if k == i else p for k in range(2)]
        refused(_lib, lib.ts_rows_unpack_q8(good, *o, p, p, paged, 1, 2, 64, None), "4-byte")
        refused(_lib, lib.ts_attend_rows_q8(p, good, p, *o, paged, 1, 64, 4, 2, 64, 0, 1.0, None, 0, None), "4-byte")
        refused(_lib, lib.ts_attend_blocks_q8(p, good, p, p, *o, paged, 1, 64, 4, 2, 64, 1, 1.0, None, 0, None), "4-byte")
    refused(_lib, lib.ts_attend_blocks_q8(p, good, p + 2, p, p, p, paged, 1, 64, 4, 2, 64, 1, 1.0, None, 0, None), "4-byte")
    for i in range(3):
        o = [p + 2 if k == i else p for k in range(3)]
        refused(_lib, lib.ts_select_blocks_q8(p, good, *o, paged, 1, 64, 4, 2, 64, 1, 0, 0, None, 0, None), "4-byte")
    odd = _lib.TsKept(2, 64, 2, p + 2, 4, 128)
    refused(_lib, lib.ts_rows_unpack_q8(good, p, p, p, p, odd, 1, 2, 64, None), "4-byte")
    # results over inputs that other blocks still read
    refused(_lib, lib.ts_qk_norm_rope_append_q8(p, None, None, p, p, p, p, good, paged, 1, 4, 2, 64, 1e-6, None), "where qkv lies")
    refused(_lib, lib.ts_attend_rows_q8(p, good, p, p, p, paged, 1, 64, 4, 2, 64, 0, 1.0, None, 0, None), "where q lies")
    refused(_lib, lib.ts_attend_blocks_q8(p, good, p, p, p, p, paged, 1, 64, 4, 2, 64, 1, 1.0, None, 0, None), "where q lies")
    # no rows: nothing to do, and nothing of the GPU is touched
    assert lib.ts_attend_rows_q8(p, good, p, p, p, paged, 0, 64, 4, 2, 64, 0, 1.0, None, 0, None) == 0
    assert lib.ts_rows_unpack_q8(good, p, p, p, p, paged, 0, 2, 64, None) == 0


def test_workspace_sizes(world):
    _lib = world[0]
    lib = _lib.lib
    assert lib.ts_attend_rows_q8_workspace_bytes(0, 4096, 16, 8, 128, 0xFFFFFFFF) == 0
    assert lib.ts_attend_rows_q8_workspace_bytes(1, 0, 16, 8, 128, 0xFFFFFFFF) == 0
    assert lib.ts_attend_rows_q8_workspace_bytes(1, 16, 16, 8, 128, 0xFFFFFFFF) == 0       # one piece
    assert lib.ts_attend_rows_q8_workspace_bytes(1, 100000, 16, 8, 128, 0xFFFFFFFF) > 0
    # a window bounds what a row reads, and with it the pieces
    assert lib.ts_attend_rows_q8_workspace_bytes(1, 100000, 16, 8, 128, 10) <= lib.ts_attend_rows_q8_workspace_bytes(1, 100000, 16, 8, 128, 50000)
    assert lib.ts_select_blocks_q8_workspace_bytes(3, 1000, 2, 16, 62) == 0                # scored and picked in one kernel
    assert lib.ts_select_blocks_q8_workspace_bytes(3, 40000, 2, 16, 2500) == 0             # every block is taken
    assert lib.ts_select_blocks_q8_workspace_bytes(3, 40000, 2, 16, 2499) >= 3 * 2 * 2500 * 4
    assert lib.ts_attend_blocks_q8_workspace_bytes(2, 0, 16, 8, 128, 64) == 0


def test_python_face_refuses_what_is_not_on_a_device():
    import torch
    from tessera_b200 import TesseraError, ops
    kv = ops.RowsQ8.empty(64, 2, 64, 16, device="cpu")
    at = torch.zeros(1, dtype=torch.int32)
    q = torch.zeros((1, 4, 64), dtype=torch.bfloat16)
    kept = ops.Kept("dense", 64, None, 64)
    for call in (lambda: ops.attend_rows_q8(q, kv, at, at, kept, 64, scale=1.0),
                 lambda: ops.select_blocks_q8(q, kv, at, at, kept, 64, 1, first=0, recent=0),
                 lambda: ops.rows_unpack_q8(kv, at, at, kept)):
        with pytest.raises(TesseraError) as e:
            call()
        assert e.value.code == 3
