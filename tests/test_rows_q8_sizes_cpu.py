"""Workspace sizes of the calls over 8-bit kept rows: every argument has an answer, and a longer context never a smaller one."""
import subprocess
import sys

import pytest

# In a process of their own: a size query must not end the one that asks.
ASK = "from tessera_b200._lib import lib; print(lib.{})"


@pytest.mark.parametrize("query", [
    "ts_attend_blocks_q8_workspace_bytes(2, 8, 16, 8, 128, 0)",           # blocks of no, of odd and of unsupported sizes
    "ts_attend_blocks_q8_workspace_bytes(2, 8, 16, 8, 128, 48)",
    "ts_attend_blocks_q8_workspace_bytes(2, 8, 16, 8, 128, 128)",
    "ts_attend_blocks_q8_workspace_bytes(1, 1 << 31, 1 << 31, 1 << 31, 256, 64)",  # products of 2^64
    "ts_attend_blocks_q8_workspace_bytes(1, (1 << 24) + 1, 16, 8, 128, 64)",
    "ts_attend_rows_q8_workspace_bytes(1, 100000, 65536, 65536, 128, 0xFFFFFFFF)",
    "ts_attend_rows_q8_workspace_bytes(1, 100000, 16, 0, 128, 0xFFFFFFFF)",
    "ts_select_blocks_q8_workspace_bytes(2, 100000, 8, 0, 4)",
])
def test_sizes_that_a_call_refuses_need_no_workspace(query):
    run = subprocess.run([sys.executable, "-c", ASK.format(query)], capture_output=True, text=True, timeout=120)
    assert run.returncode == 0 and run.stdout.strip() == "0", (run.returncode, run.stdout, run.stderr[-500:])


@pytest.mark.parametrize("rows", [1, 2, 9, 64, 5000])
@pytest.mark.parametrize("heads,kv_heads,width", [(16, 8, 128), (4, 4, 64), (64, 64, 128), (40, 1, 256)])
@pytest.mark.parametrize("back", [0, 1000, 0xFFFFFFFF])
def test_a_longer_context_never_needs_less_workspace(rows, heads, kv_heads, width, back):
    """A call reads at most its slots' room, and its plan for that must fit what the size query gave for `keys`, up to the
    2^32 - 1 that says `no limit`.  (Once there are few steps enough for one launch without partial results, none.)"""
    from tessera_b200._lib import lib
    sizes = [lib.ts_attend_rows_q8_workspace_bytes(rows, min(1 << p, 0xFFFFFFFF), heads, kv_heads, width, back) for p in range(33)]
    assert sizes == sorted(sizes), sizes
    sizes = [lib.ts_select_blocks_q8_workspace_bytes(rows, min(1 << p, 0xFFFFFFFF), kv_heads, 16, 32) for p in range(33)]
    assert sizes == sorted(sizes), sizes
