"""Operators over 8-bit kept rows against plain statements of them in 64 bits (tests/q8_model.py).

Tolerances, fixed before the first run.  Values that a kernel computes in 32 bits are off by a few roundings of
2^-24: norm, rotation and scale together stay within 2^-19 of the row's largest, which is 127 * 2^-19 < 1e-3 in units of
a code, so a code may differ from the 64-bit one by one step where the value before rounding lies within 1e-3 of a
border, and nowhere else.  bf16 outputs: half a step, 2^-8.  Attention: as q8_model.attend derives it.  Chosen blocks,
read-back values given the codes, and everything a call must leave alone: equal bits."""
import ctypes as C
from zlib import crc32

import numpy as np
import pytest
import torch

from tests import q8_model as M
from tests.util import dev_u32

pytestmark = pytest.mark.gpu
FAR = 0xFFFFFFFF


def make(rng, kv_heads, width, block, pages, page, *, scales=(0.005, 0.05), bounds=True):
    from tessera_b200 import ops
    blocks = pages * page // block
    codes = lambda: torch.from_numpy(np.clip(np.rint(rng.standard_normal((blocks, kv_heads, block, width)) * 36), -127, 127).astype(np.int8)).cuda()  # noqa: E731
    scale = lambda: torch.from_numpy(np.exp(rng.uniform(np.log(scales[0]), np.log(scales[1]), (blocks, kv_heads))).astype(np.float32)).cuda()  # noqa: E731
    k = codes()
    b = torch.stack([k.amin(2), k.amax(2)], 2).contiguous() if bounds else None
    return ops.RowsQ8(k, codes(), scale(), scale(), b)


def paged(rng, slots, per_slot, pages, page):
    """(Kept, host table): every slot's pages anywhere in the pool, no page twice."""
    from tessera_b200 import ops
    table = rng.permutation(pages)[:slots * per_slot].astype(np.uint32)
    return ops.Kept("paged", per_slot, dev_u32(table), pages * page, page=page), table


def bf16(rng, *shape, std=1.0):
    return torch.from_numpy((rng.standard_normal(shape) * std).astype(np.float32)).cuda().bfloat16()


def np64(t):
    return t.detach().float().cpu().numpy().astype(np.float64)


def gains(rng, width):
    return torch.from_numpy((1 + 0.2 * rng.standard_normal(width)).astype(np.float32)).cuda()


def inv_freq(width, theta=1e6):
    return torch.from_numpy((theta ** (-np.arange(0, width, 2, dtype=np.float64) / width)).astype(np.float32)).cuda()


def check_append(kv, before, store, raw, want_q, got_q):
    q = np64(got_q)
    row = np.abs(want_q).max(-1, keepdims=True)
    assert np.all(np.abs(q - want_q) <= 2.0 ** -8 * np.abs(want_q) + 2.0 ** -19 * row)
    for n, codes, scale in (("k", kv.k, kv.k_scale), ("v", kv.v, kv.v_scale)):
        got, s = codes.cpu().numpy().astype(np.float64), scale.cpu().numpy().astype(np.float64)
        assert np.all(np.abs(s - store.scale[n]) <= 2.0 ** -19 * store.scale[n]), n
        off = got != store.codes[n]
        assert np.all(np.abs(got - store.codes[n]) <= 1), n
        frac = np.abs(raw[n] - np.floor(raw[n]) - 0.5)
        assert np.all(frac[off] < 1e-3), (n, frac[off].max())
    if kv.k_bounds is not None:
        assert np.all(np.abs(kv.k_bounds.cpu().numpy().astype(np.float64) - store.bounds) <= 1)


APPENDS = [
    # block, width, heads, kv_heads, page, layout, norm
    (16, 128, 16, 8, 64, "paged", True),
    (64, 128, 16, 8, 64, "paged", True),
    (32, 128, 4, 4, 128, "paged", False),
    (16, 64, 6, 2, 16, "paged", True),
    (64, 64, 2, 1, 64, "dense", True),
    (32, 256, 8, 1, 32, "paged", True),
    (64, 256, 2, 2, 64, "dense", False),
    (16, 256, 3, 3, 64, "dense", True),
]


@pytest.mark.parametrize("case", APPENDS, ids=lambda c: "-".join(map(str, c)))
@pytest.mark.parametrize("kind", ["steps", "prompts", "mixed", "many"])
def test_append_follows_its_definition(case, kind):
    from tessera_b200 import ops
    block, width, heads, kv_heads, page, layout, norm = case
    rng = np.random.default_rng(crc32(repr((case[:5], kind)).encode()))
    slots, per_slot = (5, 6) if kind != "many" else (90, 4)
    context = per_slot * page
    pages = slots * per_slot + 3
    kv = make(rng, kv_heads, width, block, pages if layout == "paged" else slots * per_slot, page)
    if layout == "paged":
        kept, table = paged(rng, slots, per_slot, pages, page)
        store = M.Store(kv, "paged", per_slot, page, table)
    else:
        kept = ops.Kept("dense", context, None, slots * context)
        store = M.Store(kv, "dense", context)
    at = {"steps": [(s, [0, 5, block - 1, block, 2 * block + 3][s % 5], 1) for s in (2, 0, 1, 4, 3)],
          # whole blocks, a part of one, a start inside one, one row
          "prompts": [(1, 0, 2 * block + 5), (0, block - 3, block + 7), (3, 7, 4), (2, 3 * block - 1, 1), (4, block, block)],
          "mixed": [(0, 0, 1), (1, 4, 3 * block), (2, 0, 0), (3, block - 1, 2), (4, 1, 1)],
          # over the number of rows at which the launch looks at rows in windows
          "many": [(s, (5 * s) % block, 1 + s % 5) for s in range(slots)]}[kind]
    row_slots = [s for s, _, n in at for _ in range(n)]
    row_pos = [b + i for _, b, n in at for i in range(n)]
    if kind == "mixed":  # a launch filled up with copies of its last row
        row_slots += [row_slots[-1]] * 5
        row_pos += [row_pos[-1]] * 5
    rows = len(row_slots)
    # some rows far larger than what is held, so that scales grow, some far smaller
    size = np.exp(rng.uniform(-3, 3, (rows, 1, 1)))
    qkv = (rng.standard_normal((rows, heads + 2 * kv_heads, width)) * size).astype(np.float32)
    qkv = torch.from_numpy(qkv).cuda().bfloat16().reshape(rows, -1)
    if kind == "mixed":
        qkv[-5:] = qkv[-6]
    qn, kn = (gains(rng, width), gains(rng, width)) if norm else (None, None)
    freq = inv_freq(width)
    f = lambda t: None if t is None else t.cpu().numpy().astype(np.float64)  # noqa: E731
    want_q, k, v = M.prepared(np64(qkv), f(qn), f(kn), freq.cpu().numpy(), row_pos, heads, kv_heads, width, 1e-6)
    raw = M.append(store, k, v, row_slots, row_pos)
    before = kv.k.clone()
    got = ops.qk_norm_rope_append_q8(qkv, qn, kn, freq, dev_u32(row_slots), dev_u32(row_pos), kv, kept, heads, eps=1e-6)
    torch.cuda.synchronize()
    check_append(kv, before, store, raw, want_q, got)


def test_append_steps_one_after_another_equal_the_definition_step_by_step():
    """A slot that fills token by token: scales grow, codes follow, blocks start afresh on a reused page."""
    from tessera_b200 import ops
    rng = np.random.default_rng(5)
    block, width, heads, kv_heads, page = 16, 128, 4, 2, 16
    kv = make(rng, kv_heads, width, block, 4, page)
    kept, table = paged(rng, 2, 2, 4, page)
    store = M.Store(kv, "paged", 2, page, table)
    freq = inv_freq(width)
    for pos in range(2 * block):
        qkv = bf16(rng, 2, (heads + 2 * kv_heads) * width, std=1 + pos / 4)
        at = [pos, (pos + 9) % (2 * block)]
        q, k, v = M.prepared(np64(qkv), None, None, freq.cpu().numpy(), at, heads, kv_heads, width, 1e-6)
        raw = M.append(store, k, v, [0, 1], at)
        got = ops.qk_norm_rope_append_q8(qkv, None, None, freq, dev_u32([0, 1]), dev_u32(at), kv, kept, heads, eps=1e-6)
        check_append(kv, None, store, raw, q, got)
        # one step at a time: where a border made the kernel's code the other one, the model goes on from that
        for n, t in (("k", kv.k), ("v", kv.v)):
            store.codes[n] = t.cpu().numpy().astype(np.float64)
        store.scale = {"k": kv.k_scale.cpu().numpy().astype(np.float64), "v": kv.v_scale.cpu().numpy().astype(np.float64)}
        store.bounds = kv.k_bounds.cpu().numpy().astype(np.float64)


def test_append_far_positions_keep_their_angles():
    from tessera_b200 import ops
    rng = np.random.default_rng(6)
    block, width, heads, kv_heads, page = 64, 128, 2, 1, 64
    per = 1 << 18
    table = np.zeros(per, np.uint32)
    kept = ops.Kept("paged", per, dev_u32(table), page, page=page)
    for pos in (0, 99999, 1 << 20, (1 << 24) - 1):
        kv = ops.RowsQ8.empty(page, kv_heads, width, block)
        store = M.Store(kv, "paged", per, page, table)
        qkv = bf16(rng, 1, (heads + 2 * kv_heads) * width)
        freq = inv_freq(width)
        q, k, v = M.prepared(np64(qkv), None, None, freq.cpu().numpy(), [pos], heads, kv_heads, width, 1e-6)
        raw = M.append(store, k, v, [0], [pos])
        got = ops.qk_norm_rope_append_q8(qkv, None, None, freq, dev_u32([0]), dev_u32([pos]), kv, kept, heads, eps=1e-6)
        check_append(kv, None, store, raw, q, got)


def test_append_of_infinities_nan_zeros_and_extremes():
    from tessera_b200 import ops
    rng = np.random.default_rng(7)
    block, width, heads, kv_heads = 16, 64, 1, 1
    kv = ops.RowsQ8.empty(6 * 16, kv_heads, width, block)
    kept = ops.Kept("dense", 16, None, 6 * 16)
    store = M.Store(kv, "dense", 16)
    x = rng.standard_normal((6, 3, width)).astype(np.float32)
    x[0, 2, 3] = np.inf
    x[1, 2, 5] = np.nan
    x[2, 2] = 0.0
    x[3, 2] = np.finfo(np.float32).max  # bf16 rounds it to infinity
    x[4, 2] *= 1e-30
    x[5, 2, 7] = -np.inf
    qkv = torch.from_numpy(x).cuda().bfloat16().reshape(6, -1)
    at = list(range(6))
    q, k, v = M.prepared(np64(qkv), None, None, inv_freq(width).cpu().numpy(), [0] * 6, heads, kv_heads, width, 1e-6)
    raw = M.append(store, k, v, at, [0] * 6)
    got = ops.qk_norm_rope_append_q8(qkv, None, None, inv_freq(width), dev_u32(at), dev_u32([0] * 6), kv, kept, heads, eps=1e-6)
    check_append(kv, None, store, raw, q, got)
    assert kv.v[0, 0, 0, 3] == 127 and kv.v[1, 0, 0, 5] == 0 and kv.v[5, 0, 0, 7] == -127
    assert torch.all(kv.v[2] == 0) and kv.v_scale[2, 0] == 2.0 ** -60 and kv.v_scale[4, 0] == 2.0 ** -60
    # and a block of infinities reads back finite, so that attention over it is
    k8, v8 = ops.rows_unpack_q8(kv, dev_u32(at), dev_u32([0] * 6), kept)
    assert torch.isfinite(v8.float()).all()


def test_append_outside_the_pool_writes_nothing_and_the_last_of_equal_rows_counts():
    from tessera_b200 import ops
    rng = np.random.default_rng(8)
    block, width, heads, kv_heads, page = 16, 128, 2, 2, 32
    kv = make(rng, kv_heads, width, block, 4, page)
    table = np.array([0, 9, 2, 1], np.uint32)  # page 9 is not in the pool
    kept = ops.Kept("paged", 2, dev_u32(table), 4 * page, page=page)
    store = M.Store(kv, "paged", 2, page, table)
    slots, pos = [0, 0, 1, 1, 1, 7, 0], [3, 40, 5, 5, 5, 0, 64]
    qkv = bf16(rng, 7, (heads + 2 * kv_heads) * width)
    freq = inv_freq(width)
    q, k, v = M.prepared(np64(qkv), None, None, freq.cpu().numpy(), pos, heads, kv_heads, width, 1e-6)
    raw = M.append(store, k, v, slots, pos)
    untouched = [b for b in range(8) if b not in (0, 4)]
    before = {n: getattr(kv, n)[untouched].clone() for n in ("k", "v", "k_scale", "v_scale", "k_bounds")}
    got = ops.qk_norm_rope_append_q8(qkv, None, None, freq, dev_u32(slots), dev_u32(pos), kv, kept, heads, eps=1e-6)
    check_append(kv, None, store, raw, q, got)
    for n, t in before.items():
        assert torch.equal(getattr(kv, n)[untouched], t), n


@pytest.mark.parametrize("width", [64, 128, 256])
@pytest.mark.parametrize("block", [16, 32, 64])
def test_rows_read_back_are_code_times_scale(width, block):
    from tessera_b200 import ops
    rng = np.random.default_rng(9)
    kv = make(rng, 3, width, block, 5, 64)
    table = np.array([4, 2, 1, 99], np.uint32)
    kept = ops.Kept("paged", 2, dev_u32(table), 5 * 64, page=64)
    slots = rng.integers(0, 3, 333)
    pos = rng.integers(0, 140, 333)
    k, v = ops.rows_unpack_q8(kv, dev_u32(slots), dev_u32(pos), kept)
    store = M.Store(kv, "paged", 2, 64, table)
    for r in range(333):
        blk = store.at(slots[r], pos[r] // block)
        for got, codes, scale in ((k, kv.k, kv.k_scale), (v, kv.v, kv.v_scale)):
            want = torch.zeros_like(got[r]) if blk is None else (codes[blk, :, pos[r] % block].float() * scale[blk][:, None]).bfloat16()
            assert torch.equal(got[r], want)


ATTENDS = [
    # heads, kv_heads, width, block, page, layout
    (16, 8, 128, 64, 64, "paged"), (16, 8, 128, 16, 64, "paged"), (8, 2, 128, 32, 32, "paged"), (3, 3, 128, 64, 128, "dense"),
    (8, 1, 64, 16, 16, "paged"), (6, 2, 64, 64, 64, "dense"), (16, 1, 128, 32, 64, "paged"), (20, 1, 64, 32, 64, "paged"),
    (34, 2, 128, 64, 64, "dense"), (4, 2, 256, 64, 64, "paged"), (12, 1, 256, 16, 32, "dense"),
]


def attend_case(rng, case, lengths, **more):
    from tessera_b200 import ops
    heads, kv_heads, width, block, page, layout = case
    slots = len(lengths)
    per = max(-(-n // page) for n in lengths)
    pages = slots * per + 2
    kv = make(rng, kv_heads, width, block, pages if layout == "paged" else slots * per, page, **more)
    if layout == "paged":
        kept, table = paged(rng, slots, per, pages, page)
        return kv, kept, M.Store(kv, "paged", per, page, table)
    return kv, ops.Kept("dense", per * page, None, slots * per * page), M.Store(kv, "dense", per * page)


def check_attend(got, want, tol):
    off = np.abs(np64(got) - want)
    assert np.isfinite(np64(got)).all()
    assert np.all(off <= tol), (off - tol).max()


@pytest.mark.parametrize("case", ATTENDS, ids=lambda c: "-".join(map(str, c)))
@pytest.mark.parametrize("lengths,each", [([1], 1), ([17, 1, 64], 1), ([65, 300, 129, 2], 1), ([700], 1), ([40, 333], 5), ([260], 19)],
                         ids=["1", "short", "ragged", "long", "drafts", "part"])
def test_attention_over_whole_slots(case, lengths, each):
    from tessera_b200 import ops
    rng = np.random.default_rng(crc32(repr((case, lengths, each)).encode()))
    heads, kv_heads, width = case[:3]
    kv, kept, store = attend_case(rng, case, lengths)
    slots = [s for s, n in enumerate(lengths) for _ in range(min(each, n))]
    pos = [n - min(each, n) + i for n in lengths for i in range(min(each, n))]
    q = bf16(rng, len(slots), heads, width)
    scale = width ** -0.5
    keys = max(lengths)
    for back in (FAR, 0, 21, 128):
        got = ops.attend_rows_q8(q, kv, dev_u32(slots), dev_u32(pos), kept, keys, scale=scale, back=back)
        want, tol = M.attend(store, np64(q), slots, pos, keys, scale, back)
        check_attend(got, want, tol)


@pytest.mark.parametrize("case", ATTENDS, ids=lambda c: "-".join(map(str, c)))
@pytest.mark.parametrize("kind", ["steps", "drafts", "long"])
def test_attention_of_many_rows_and_of_long_ones(case, kind):
    """More rows and kv heads than thread blocks fit the GPU at once, or a context of thousands: the steps of all of
    them are shared out evenly, whatever the lengths."""
    from tessera_b200 import ops
    rng = np.random.default_rng(crc32(repr((case, kind)).encode()))
    heads, kv_heads, width, block = case[:4]
    if kind == "long":
        lengths, each = [9001, 40, 6000], 1
    else:
        each = 1 if kind == "steps" else 3
        lengths = [int(n) for n in rng.integers(each, 300, (310 // kv_heads + 3) // each + 1)]
        lengths[1] = 2500  # one far longer than the others
    kv, kept, store = attend_case(rng, case, lengths)
    slots = [s for s, n in enumerate(lengths) for _ in range(each)]
    pos = [n - each + i for n in lengths for i in range(each)]
    q = bf16(rng, len(slots), heads, width)
    keys, scale = max(lengths), width ** -0.5
    for back in (FAR, 700):
        got = ops.attend_rows_q8(q, kv, dev_u32(slots), dev_u32(pos), kept, keys, scale=scale, back=back)
        want, tol = M.attend(store, np64(q), slots, pos, keys, scale, back)
        check_attend(got, want, tol)
    # the same through lists that name every block, in reversed order
    n = -(-keys // block)
    if kind == "steps":
        ids = np.broadcast_to(np.arange(n, dtype=np.uint32)[::-1], (len(slots), kv_heads, n))
        got = ops.attend_blocks_q8(q, kv, dev_u32(ids), dev_u32(slots), dev_u32(pos), kept, keys, scale=scale)
        want, tol = M.attend(store, np64(q), slots, pos, keys, scale)
        check_attend(got, want, tol)


def test_attention_of_rows_in_any_order_and_rows_that_see_nothing():
    """Rows of one slot out of order, the same row twice, positions past `keys`, slots and pages outside the pool."""
    from tessera_b200 import ops
    rng = np.random.default_rng(11)
    case = (4, 2, 128, 32, 64, "paged")
    heads, kv_heads, width, block, page, _ = case
    kv = make(rng, kv_heads, width, block, 8, page)
    table = np.array([5, 77, 1, 3, 0, 2], np.uint32)
    kept = ops.Kept("paged", 2, dev_u32(table), 8 * page, page=page)
    store = M.Store(kv, "paged", 2, page, table)
    slots = [1, 1, 1, 0, 0, 2, 1, 1, 9, 2, 2, 2, 1]
    pos = [90, 3, 91, 100, 63, 127, 5, 5, 4, 0, FAR, 130, 300]
    q = bf16(rng, len(slots), heads, width)
    for keys, back in ((128, FAR), (128, 10), (64, 10), (1, FAR), (0, FAR)):
        got = ops.attend_rows_q8(q, kv, dev_u32(slots), dev_u32(pos), kept, keys, scale=0.09, back=back)
        if keys == 0:
            assert torch.all(got == 0)
            continue
        want, tol = M.attend(store, np64(q), slots, pos, keys, 0.09, back)
        check_attend(got, want, tol)
        empty = np.all(want == 0, axis=(1, 2))
        assert np.all(np64(got)[empty] == 0)


def test_attention_with_scales_of_any_size():
    """Scales from 1e-17 to 1e17 side by side, zero ones, and NaN in blocks that no row sees."""
    from tessera_b200 import ops
    rng = np.random.default_rng(12)
    case = (4, 2, 128, 16, 16, "dense")
    heads, kv_heads, width, block, page, _ = case
    lengths = [95, 40]
    for low, high in ((1e-17, 1e17), (1e-3, 1e3), (1e12, 1e17), (1e-17, 1e-12)):
        kv, kept, store = attend_case(rng, case, lengths)
        v = np.exp(rng.uniform(np.log(low), np.log(high), kv.v_scale.shape)).astype(np.float32)
        v[1] = 0
        kv.v_scale.copy_(torch.from_numpy(v))
        kv.v[1] = 0  # a scale of zero goes with codes of zero, as append leaves them
        kv.k_scale[2] = 0
        kv.v_scale[9:] = float("nan")  # slot 1 sees blocks 6, 7, 8
        kv.k_scale[9:] = float("nan")
        store = M.Store(kv, "dense", 96)
        q = bf16(rng, 2, heads, width)
        got = ops.attend_rows_q8(q, kv, dev_u32([0, 1]), dev_u32([94, 39]), kept, 95, scale=0.09)
        want, tol = M.attend(store, np64(q), [0, 1], [94, 39], 95, 0.09)
        check_attend(got, want, tol)


def test_attention_of_queries_of_any_size():
    from tessera_b200 import ops
    rng = np.random.default_rng(13)
    case = (2, 1, 128, 64, 64, "dense")
    kv, kept, store = attend_case(rng, case, [200])
    q = bf16(rng, 4, 2, 128)
    q[0] *= 1e-30
    q[1] *= 2.0 ** 100
    q[2] = 0
    scale = [0.09, 2.0 ** -100 * 0.09, 0.09, 0.09]
    for r in range(4):
        got = ops.attend_rows_q8(q[r:r + 1], kv, dev_u32([0]), dev_u32([199]), kept, 200, scale=scale[r])
        want, tol = M.attend(store, np64(q[r:r + 1]), [0], [199], 200, scale[r])
        check_attend(got, want, tol)
    q[3, 0, 5] = float("nan")  # stays in its own head
    got = ops.attend_rows_q8(q[3:], kv, dev_u32([0]), dev_u32([199]), kept, 200, scale=0.09)
    assert torch.isnan(got[0, 0].float()).all() and torch.isfinite(got[0, 1].float()).all()


@pytest.mark.parametrize("case", [(4, 4, 128, 64, 64, "dense"), (16, 2, 128, 32, 64, "paged"), (5, 1, 64, 16, 16, "paged"), (8, 1, 256, 64, 64, "dense")],
                         ids=lambda c: "-".join(map(str, c)))
@pytest.mark.parametrize("each", [1, 3])
def test_attention_where_later_keys_score_higher(case, each):
    """Every head's query along one channel that the keys climb (or fall, or jump over), by up to 2^9 a block of positions."""
    from tessera_b200 import ops
    rng = np.random.default_rng(20)
    heads, kv_heads, width, block = case[:4]
    n = 1000
    kv, kept, store = attend_case(rng, case, [n])
    at = np.array([store.at(0, b) for b in range(n // block)])
    kv.k.zero_()
    kv.k_scale.fill_(1.0)
    q = torch.zeros((each, heads, width), dtype=torch.bfloat16, device="cuda")
    q[:, :, 7] = 1.0
    for path in (np.linspace(0, 127, len(at)), np.linspace(127, -127, len(at)), np.where(np.arange(len(at)) % 5 == 4, 100, -100) + np.arange(len(at)) // 3,
                 np.where(np.arange(len(at)) == len(at) - 2, 127, np.arange(len(at)) % 7)):
        codes = torch.from_numpy(np.rint(path).astype(np.int8)).cuda()
        kv.k[torch.from_numpy(at).cuda(), :, :, 7] = codes[:, None, None]
        store = M.Store(kv, store.layout, store.scalar, store.page, store.table)
        pos = list(range(n - each, n))
        # a score of 15 a step at most in powers of two: the products are whole numbers times the scale, exact
        for scale in (0.02, 0.1):
            got = ops.attend_rows_q8(q, kv, dev_u32([0] * each), dev_u32(pos), kept, n, scale=scale)
            want, tol = M.attend(store, np64(q), [0] * each, pos, n, scale)
            check_attend(got, want, tol)


COLD = """
import torch
from tessera_b200 import ops
kv = ops.RowsQ8.empty({pages} * 64, 2, 128, 64)
kept = ops.Kept("dense", {pages} * 64, None, {pages} * 64)
at, pos = torch.zeros(1, dtype=torch.int32, device="cuda"), torch.full((1,), {pages} * 64 - 1, dtype=torch.int32, device="cuda")
qkv, freq = torch.ones((1, 8 * 128), dtype=torch.bfloat16, device="cuda"), torch.ones(64, device="cuda")
g, side = torch.cuda.CUDAGraph(), torch.cuda.Stream()
torch.cuda.synchronize()
with torch.cuda.graph(g, stream=side):
    q = ops.qk_norm_rope_append_q8(qkv, None, None, freq, at, pos, kv, kept, 4, eps=1e-6)
    a = ops.attend_rows_q8(q, kv, at, pos, kept, {pages} * 64, scale=0.1)
    ids = ops.select_blocks_q8(q, kv, at, pos, kept, {pages} * 64, 4)
    b = ops.attend_blocks_q8(q, kv, ids, at, pos, kept, {pages} * 64, scale=0.1)
    k, v = ops.rows_unpack_q8(kv, at, pos, kept)
for _ in range(2):
    g.replay()
torch.cuda.synchronize()
assert ids[0, 0, 3].item() == {pages} - 1 and (v.float() == 1).all() and a.float().abs().max() > 0 and b.float().abs().max() > 0
print("replayed")
"""


@pytest.mark.parametrize("pages", [8, 700])
def test_the_first_calls_of_a_process_may_be_captured(pages):
    import subprocess
    import sys
    run = subprocess.run([sys.executable, "-c", COLD.format(pages=pages)], capture_output=True, text=True, timeout=300)
    assert run.returncode == 0 and "replayed" in run.stdout, run.stderr[-2000:]


def test_more_rows_than_one_launch_chooses_for():
    from tessera_b200 import ops
    rng = np.random.default_rng(21)
    case = (2, 1, 64, 16, 16, "dense")
    rows = 70001
    for length in (160, 520 * 16):  # one kernel, and two
        kv, kept, store = attend_case(rng, case, [length])
        q = bf16(rng, 3, 2, 64).repeat(-(-rows // 3), 1, 1)[:rows].contiguous()
        pos = torch.full((rows,), length - 1, dtype=torch.int32, device="cuda")
        got = ops.select_blocks_q8(q, kv, torch.zeros_like(pos), pos, kept, length, 3)
        want = M.select(store, np64(q[:3]), [0] * 3, [length - 1] * 3, length, 3, 1, 1)
        want = torch.from_numpy(want.astype(np.int32)).cuda().repeat(-(-rows // 3), 1, 1)[:rows]
        assert torch.equal(got, want)


@pytest.mark.parametrize("case", [(16, 8, 128, 16, 64, "paged"), (8, 1, 64, 32, 32, "paged"), (32, 4, 128, 64, 64, "paged"),
                                  (4, 2, 256, 64, 128, "dense"), (3, 1, 256, 16, 16, "paged")], ids=lambda c: "-".join(map(str, c)))
@pytest.mark.parametrize("count,first,recent", [(1, 0, 0), (1, 0, 1), (3, 1, 1), (7, 0, 2), (40, 2, 3), (300, 1, 1)])
def test_chosen_blocks_equal_the_definition(case, count, first, recent):
    from tessera_b200 import ops
    rng = np.random.default_rng(crc32(repr((case, count, first, recent)).encode()))
    heads, kv_heads, width, block = case[:4]
    lengths = [1, block, block + 1, 23 * block - 5, 611 if block < 64 else 2500]
    kv, kept, store = attend_case(rng, case, lengths)
    slots, pos = list(range(5)) + [4], [n - 1 for n in lengths] + [3 * block]
    q = bf16(rng, 6, heads, width)
    got = ops.select_blocks_q8(q, kv, dev_u32(slots), dev_u32(pos), kept, max(lengths), count, first=first, recent=recent)
    want = M.select(store, np64(q), slots, pos, max(lengths), count, first, recent)
    assert np.array_equal(got.cpu().numpy().view(np.uint32), want)


def test_chosen_blocks_with_ties_zero_queries_holes_and_many_blocks():
    from tessera_b200 import ops
    rng = np.random.default_rng(15)
    block, width, heads, kv_heads, page = 16, 64, 2, 1, 16
    per = 5000
    kv = make(rng, kv_heads, width, block, per, page)
    kv.k_bounds[100:4000] = kv.k_bounds[100]  # thousands of equal scores
    kv.k_scale[100:4000] = kv.k_scale[100]
    table = np.arange(per).astype(np.uint32)
    table[[50, 4500]] = 1 << 30  # pages outside the pool
    kept = ops.Kept("paged", per, dev_u32(table), per * page, page=page)
    store = M.Store(kv, "paged", per, page, table)
    q = bf16(rng, 3, heads, width)
    q[1] = 0
    keys = per * page
    pos = [keys - 1, keys - 7, FAR]
    for count, first, recent in ((64, 1, 1), (1500, 0, 0), (4096, 3, 5), (2, 2, 0), (2, 0, 2)):
        got = ops.select_blocks_q8(q, kv, dev_u32([0, 0, 0]), dev_u32(pos), kept, keys, count, first=first, recent=recent)
        want = M.select(store, np64(q), [0, 0, 0], pos, keys, count, first, recent)
        assert np.array_equal(got.cpu().numpy().view(np.uint32), want), (count, first, recent)
    none = ops.select_blocks_q8(q, kv, dev_u32([0, 0, 0]), dev_u32(pos), kept, 0, 4, first=0, recent=0)
    assert torch.all(none == -1)


@pytest.mark.parametrize("case", ATTENDS, ids=lambda c: "-".join(map(str, c)))
@pytest.mark.parametrize("count", [1, 5, 33])
def test_attention_over_listed_blocks(case, count):
    from tessera_b200 import ops
    rng = np.random.default_rng(crc32(repr((case, count)).encode()))
    heads, kv_heads, width, block = case[:4]
    lengths = [1, block, 3 * block + 1, 900]
    kv, kept, store = attend_case(rng, case, lengths)
    slots, pos = [0, 1, 2, 3, 3], [n - 1 for n in lengths] + [5]
    # any order, some twice, some past the row, spare ones
    ids = rng.integers(0, -(-900 // block) + 2, (5, kv_heads, count)).astype(np.uint32)
    ids[rng.random(ids.shape) < 0.2] = M.SPARE
    ids[0, 0] = M.SPARE
    q = bf16(rng, 5, heads, width)
    got = ops.attend_blocks_q8(q, kv, dev_u32(ids), dev_u32(slots), dev_u32(pos), kept, 900, scale=width ** -0.5)
    want, tol = M.attend(store, np64(q), slots, pos, 900, width ** -0.5, ids=ids)
    check_attend(got, want, tol)
    assert torch.all(got[0, :heads // kv_heads] == 0)


def test_a_serving_run_prompt_steps_choice_and_page_copy():
    """A prompt, steps, a fork's page copy, attention over everything and over chosen blocks, as a server calls them; the
    outputs against the definition over the rows the store holds and against attention over the unrounded rows."""
    from tessera_b200 import ops
    from tessera_b200.kv import PageCopy
    from tessera_b200._lib import lib
    rng = np.random.default_rng(16)
    heads, kv_heads, width, block, page, per, pages = 8, 2, 128, 16, 64, 8, 24
    kv = ops.RowsQ8.empty(pages * page, kv_heads, width, block)
    table = rng.permutation(pages)[:3 * per].reshape(3, per).astype(np.uint32)
    kept = ops.Kept("paged", per, dev_u32(table.reshape(-1)), pages * page, page=page)
    freq, qn, kn = inv_freq(width), gains(rng, width), gains(rng, width)
    f = lambda t: t.cpu().numpy().astype(np.float64)  # noqa: E731
    exact = {}  # (slot, position) -> (k, v) before rounding

    def feed(slots, pos):
        qkv = bf16(rng, len(slots), (heads + 2 * kv_heads) * width)
        q = ops.qk_norm_rope_append_q8(qkv, qn, kn, freq, dev_u32(slots), dev_u32(pos), kv, kept, heads, eps=1e-6)
        _, k, v = M.prepared(np64(qkv), f(qn), f(kn), freq.cpu().numpy(), pos, heads, kv_heads, width, 1e-6)
        exact.update({(s, p): (k[i], v[i]) for i, (s, p) in enumerate(zip(slots, pos))})
        return q

    feed([0] * 301 + [1] * 77, list(range(301)) + list(range(77)))
    # slot 2 forks slot 0 at row 150: two whole pages are shared, the third is copied up to row 150
    table[2, :2] = table[0, :2]
    kept = ops.Kept("paged", per, dev_u32(table.reshape(-1)), pages * page, page=page)
    share = page // block
    copy = (PageCopy * 1)(PageCopy(int(table[0, 2]), int(table[2, 2]), -(-(150 - 2 * page) // block)))
    stream = C.c_void_p(torch.cuda.current_stream().cuda_stream)
    for t, row in ((kv.k, block * kv_heads * width), (kv.v, block * kv_heads * width), (kv.k_scale, 4 * kv_heads),
                   (kv.v_scale, 4 * kv_heads), (kv.k_bounds, 2 * kv_heads * width)):
        assert lib.ts_kv_copy_pages(C.c_void_p(t.data_ptr()), copy, 1, share, row, stream) == 0
    exact.update({(2, p): exact[0, p] for p in range(150)})
    at = [301, 77, 150]
    for step in range(20):
        pos = [a + step for a in at]
        q = feed([0, 1, 2], pos)
        keys = max(pos) + 1
        got = ops.attend_rows_q8(q, kv, dev_u32([0, 1, 2]), dev_u32(pos), kept, keys, scale=width ** -0.5)
        ids = ops.select_blocks_q8(q, kv, dev_u32([0, 1, 2]), dev_u32(pos), kept, keys, 6, first=1, recent=2)
        few = ops.attend_blocks_q8(q, kv, ids, dev_u32([0, 1, 2]), dev_u32(pos), kept, keys, scale=width ** -0.5)
        every = ops.select_blocks_q8(q, kv, dev_u32([0, 1, 2]), dev_u32(pos), kept, keys, 64)
        same = ops.attend_blocks_q8(q, kv, every, dev_u32([0, 1, 2]), dev_u32(pos), kept, keys, scale=width ** -0.5)
        if step % 5:
            continue
        store = M.Store(kv, "paged", per, page, table.reshape(-1))
        q64 = np64(q)
        want, tol = M.attend(store, q64, [0, 1, 2], pos, keys, width ** -0.5)
        check_attend(got, want, tol)
        check_attend(same, want, tol)
        chosen = ids.cpu().numpy().view(np.uint32)
        assert np.array_equal(chosen, M.select(store, q64, [0, 1, 2], pos, keys, 6, 1, 2))
        want, tol = M.attend(store, q64, [0, 1, 2], pos, keys, width ** -0.5, ids=chosen)
        check_attend(few, want, tol)
        # rows as stored against rows as given: half a code of the block's largest, and as much again for each growth
        for r in range(3):
            for p in range(0, pos[r] + 1, 13):
                for h in range(kv_heads):
                    k8, v8 = store.keys_of(r, h, [p])
                    blk = store.at(r, p // block)
                    for x8, x, n in ((k8[0], exact[r, p][0][h], "k"), (v8[0], exact[r, p][1][h], "v")):
                        assert np.abs(x8 - x).max() <= 0.5 * store.scale[n][blk, h] * block


def test_a_captured_step_replays_over_new_inputs_beside_another_on_its_own_stream():
    from tessera_b200 import ops
    rng = np.random.default_rng(17)
    case = (16, 8, 128, 32, 64, "paged")
    heads, kv_heads, width, block, page, _ = case
    freq = inv_freq(width)

    def world(seed):
        r = np.random.default_rng(seed)
        kv, kept, _ = attend_case(r, case, [2000, 1500])
        return dict(kv=kv, kept=kept, qkv=bf16(r, 2, (heads + 2 * kv_heads) * width), pos=dev_u32([1999, 1400]), slots=dev_u32([0, 1]))

    def step(w):
        q = ops.qk_norm_rope_append_q8(w["qkv"], None, None, freq, w["slots"], w["pos"], w["kv"], w["kept"], heads, eps=1e-6)
        a = ops.attend_rows_q8(q, w["kv"], w["slots"], w["pos"], w["kept"], 2000, scale=0.09)
        ids = ops.select_blocks_q8(q, w["kv"], w["slots"], w["pos"], w["kept"], 2000, 9)
        return q, a, ids, ops.attend_blocks_q8(q, w["kv"], ids, w["slots"], w["pos"], w["kept"], 2000, scale=0.09)

    worlds = [world(1), world(2)]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    graphs, outs = [], []
    with torch.cuda.stream(side):
        for w in worlds:
            step(w)
        side.synchronize()
        for w in worlds:
            g = torch.cuda.CUDAGraph()
            with torch.cuda.graph(g, stream=side):
                outs.append(step(w))
            graphs.append(g)
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    for turn in range(3):
        want = []
        for i, w in enumerate(worlds):
            w["qkv"].copy_(bf16(np.random.default_rng(100 + 10 * turn + i), 2, (heads + 2 * kv_heads) * width))
            w["pos"].copy_(dev_u32([1999 - turn, 1400 + turn]))
            kv = w["kv"]
            fresh = dict(w, kv=ops.RowsQ8(*(t.clone() for t in (kv.k, kv.v, kv.k_scale, kv.v_scale, kv.k_bounds))))
            torch.cuda.synchronize()
            want.append([t.clone() for t in step(fresh)])
        torch.cuda.synchronize()
        for g, s in zip(graphs, streams):
            with torch.cuda.stream(s):
                g.replay()
        torch.cuda.synchronize()
        for out, w in zip(outs, want):
            for a, b in zip(out, w):
                assert torch.equal(a, b)


def test_dependent_launches_and_repeats_give_the_same_bits():
    from tessera_b200 import ops
    rng = np.random.default_rng(18)
    kv, kept, store = attend_case(rng, (16, 8, 128, 64, 64, "paged"), [3000, 10, 700])
    q = bf16(rng, 3, 16, 128)
    slots, pos = dev_u32([0, 1, 2]), dev_u32([2999, 9, 699])
    run = lambda: (ops.attend_rows_q8(q, kv, slots, pos, kept, 3000, scale=0.09), ops.select_blocks_q8(q, kv, slots, pos, kept, 3000, 8))  # noqa: E731
    first = run()
    ops.set_pdl(True)
    try:
        for _ in range(5):
            for a, b in zip(run(), first):
                assert torch.equal(a, b)
    finally:
        ops.set_pdl(False)
    assert ops.device_status() == 0


def test_offsets_past_32_bits():
    from tessera_b200 import ops
    rng = np.random.default_rng(19)
    kv_heads, width, block, page = 8, 128, 64, 64
    pages = (1 << 32) // (page * kv_heads * width) + 8  # codes of 2^32 bytes and more, each of K and V
    kv = ops.RowsQ8.empty(pages * page, kv_heads, width, block)
    table = np.array([pages - 1, pages - 3, 1, 0], np.uint32)
    kept = ops.Kept("paged", 2, dev_u32(table), pages * page, page=page)
    qkv = bf16(rng, 100, (16 + 16) * width)
    slots, pos = dev_u32([0] * 100), dev_u32(np.arange(100))
    q = ops.qk_norm_rope_append_q8(qkv, None, None, inv_freq(width), slots, pos, kv, kept, 16, eps=1e-6)
    small = ops.RowsQ8(*(t[[pages - 1, pages - 3]].contiguous() for t in (kv.k, kv.v, kv.k_scale, kv.v_scale, kv.k_bounds)))
    assert small.k.abs().sum() > 0
    near = ops.Kept("paged", 2, dev_u32([0, 1]), 2 * page, page=page)
    twin = ops.RowsQ8.empty(2 * page, kv_heads, width, block)
    ops.qk_norm_rope_append_q8(qkv, None, None, inv_freq(width), slots, pos, twin, near, 16, eps=1e-6)
    for n in ("k", "v", "k_scale", "v_scale", "k_bounds"):
        assert torch.equal(getattr(twin, n), getattr(small, n)), n
    a = ops.attend_rows_q8(q, kv, slots, pos, kept, 100, scale=0.09)
    assert torch.equal(a, ops.attend_rows_q8(q, twin, slots, pos, near, 100, scale=0.09))
    ids = ops.select_blocks_q8(q, kv, slots, pos, kept, 100, 1, first=0)
    assert torch.equal(ids, ops.select_blocks_q8(q, twin, slots, pos, near, 100, 1, first=0))
    assert torch.equal(ops.attend_blocks_q8(q, kv, ids, slots, pos, kept, 100, scale=0.09),
                       ops.attend_blocks_q8(q, twin, ids, slots, pos, near, 100, scale=0.09))
    for a, b in zip(ops.rows_unpack_q8(kv, slots, pos, kept), ops.rows_unpack_q8(twin, slots, pos, near)):
        assert torch.equal(a, b)


def test_no_rows():
    from tessera_b200 import ops
    kv = ops.RowsQ8.empty(64, 2, 64, 16)
    kept = ops.Kept("dense", 64, None, 64)
    none = dev_u32(np.zeros(0, np.uint32))
    q = torch.empty((0, 4, 64), dtype=torch.bfloat16, device="cuda")
    assert ops.attend_rows_q8(q, kv, none, none, kept, 64, scale=1.0).shape == (0, 4, 64)
    assert ops.select_blocks_q8(q, kv, none, none, kept, 64, 3).shape == (0, 2, 3)
    assert ops.attend_blocks_q8(q, kv, torch.empty((0, 2, 3), dtype=torch.int32, device="cuda"), none, none, kept, 64, scale=1.0).shape == (0, 4, 64)
    assert ops.rows_unpack_q8(kv, none, none, kept)[0].shape == (0, 2, 64)
    assert ops.qk_norm_rope_append_q8(torch.empty((0, 8 * 64), dtype=torch.bfloat16, device="cuda"), None, None, inv_freq(64), none,
                                      none, kv, kept, 4, eps=1e-6).shape == (0, 4, 64)


def test_python_refusals_on_the_device():
    from tessera_b200 import TesseraError, ops
    kv = ops.RowsQ8.empty(128, 2, 64, 16)
    bare = ops.RowsQ8.empty(128, 2, 64, 16, bounds=False)
    kept = ops.Kept("dense", 64, None, 128)
    q = torch.zeros((2, 4, 64), dtype=torch.bfloat16, device="cuda")
    at = dev_u32([0, 1])
    bad = [
        lambda: ops.attend_rows_q8(q.float(), kv, at, at, kept, 64, scale=1.0),
        lambda: ops.attend_rows_q8(q.transpose(0, 1), kv, at, at, kept, 64, scale=1.0),
        lambda: ops.attend_rows_q8(q, kv, at.long(), at, kept, 64, scale=1.0),
        lambda: ops.attend_rows_q8(q, kv, at, at[:1], kept, 64, scale=1.0),
        lambda: ops.attend_rows_q8(q[:, :3], kv, at, at, kept, 64, scale=1.0),
        lambda: ops.attend_rows_q8(q.cpu(), kv, at, at, kept, 64, scale=1.0),
        lambda: ops.attend_rows_q8(q, kv, at, at, ops.Kept("interleaved", 2, None, 128), 64, scale=1.0),
        lambda: ops.attend_rows_q8(q, kv, at, at, ops.Kept("dense", 40, None, 128), 64, scale=1.0),
        lambda: ops.attend_rows_q8(q, kv, at, at, ops.Kept("paged", 2, at, 128, page=8), 64, scale=1.0),
        lambda: ops.attend_rows_q8(q, kv, at, at, kept, -1, scale=1.0),
        lambda: ops.attend_rows_q8(q, kv, at, at, kept, 64, scale=1.0, out=q),
        lambda: ops.select_blocks_q8(q, bare, at, at, kept, 64, 2),
        lambda: ops.select_blocks_q8(q, kv, at, at, kept, 64, 1, first=1, recent=1),
        lambda: ops.select_blocks_q8(q, kv, at, at, kept, 64, 0, first=0, recent=0),
        lambda: ops.select_blocks_q8(q, kv, at, at, kept, 64, 5000),
        lambda: ops.attend_blocks_q8(q, kv, torch.zeros((2, 1, 3), dtype=torch.int32, device="cuda"), at, at, kept, 64, scale=1.0),
        lambda: ops.RowsQ8(kv.k, kv.v, kv.k_scale.half(), kv.v_scale),
        lambda: ops.RowsQ8(kv.k, kv.v[:1], kv.k_scale, kv.v_scale),
        lambda: ops.RowsQ8.empty(100, 2, 64, 64),
        lambda: ops.qk_norm_rope_append_q8(torch.zeros((2, 8 * 64), dtype=torch.bfloat16, device="cuda"), inv_freq(64)[:3], None,
                                           inv_freq(64), at, at, kv, kept, 4, eps=1e-6),
    ]
    for i, call in enumerate(bad):
        with pytest.raises(TesseraError) as e:
            call()
        assert e.value.code == 3, i
    torch.cuda.synchronize()
