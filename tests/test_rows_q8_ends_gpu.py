"""What calls over 8-bit kept rows hold to at the ends of their ranges: weights far below a row's largest, scales that are
no numbers, codes half-way between two, rows of a block in any order, several launches and several host threads."""
import numpy as np
import pytest
import torch

from tests import q8_model as M
from tests.test_rows_q8_gpu import attend_case, bf16, check_append, inv_freq, make, np64, paged
from tests.util import dev_u32

pytestmark = pytest.mark.gpu
FAR = 0xFFFFFFFF


@pytest.mark.parametrize("width,heads", [(64, 16), (128, 16), (128, 3), (256, 8)])
@pytest.mark.parametrize("weight", [20.5, 5.5, 1.5])
def test_many_small_weights_beside_one_large_one_that_adds_nothing(width, heads, weight):
    """The first key has nearly all of the weight and the value zero; the others, `weight` * 2^-24 of it each, make up the
    output.  Rows enough that one worker takes a whole row: a run of its own, where the others' weights stand beside the
    first one's.  Scores are 0 and one number; so what counts is the weights' rounding to f16: half a step, 2^-11, and
    2^-32 of the largest weight (2^7 in a run's own units) where that is subnormal, for each key; the sum's own error
    (8193 terms, 2^-24 each) is below 2^-11 as well.  bf16: half a step."""
    from tessera_b200 import ops
    rng = np.random.default_rng(30)
    n, rows = 8193, 1300
    kv, kept, _ = attend_case(rng, (heads, 1, width, 64, 64, "dense"), [n])
    kv.k.zero_()
    kv.k_scale.fill_(1.0)
    kv.v_scale.fill_(1.0)
    kv.k[0, 0, 0, 7] = 127
    kv.v.copy_(torch.from_numpy(rng.integers(40, 128, tuple(kv.v.shape)).astype(np.int8)))
    kv.v[0, 0, 0] = 0
    store = M.Store(kv, "dense", kept.scalar)
    q = torch.zeros((rows, heads, width), dtype=torch.bfloat16, device="cuda")
    q[:, :, 7] = 1.0
    scale = (24 - np.log2(weight)) * np.log(2.0) / 127
    at = dev_u32([0] * rows)
    # (positions that are not neighbours, so that every row is a tile)
    pos = [n - 1 if r % 2 == 0 else n - 5 for r in range(rows)]
    got = np64(ops.attend_rows_q8(q, kv, at, dev_u32(pos), kept, n, scale=scale))
    for r in (0, 1):
        want, a, top, keys = M.attend_keys(store, np64(q[0]), 0, 0, range(pos[r] + 1), np.float32(scale).astype(np.float64))
        largest = 1 / (1 + (keys - 1) * weight * 2.0 ** -24)
        tol = 2.0 ** -8 * np.abs(want) + 2.0 ** -10 * a + keys * 2.0 ** -32 * largest * top
        off = np.abs(got[r::2] - want)
        assert np.all(off <= tol), (off / np.abs(want)).max()


@pytest.mark.parametrize("which", ["k_scale", "v_scale"])
@pytest.mark.parametrize("case", [(16, 8, 128, 64, 64, "paged"), (8, 2, 128, 16, 32, "paged"), (6, 2, 64, 16, 64, "dense"), (4, 2, 256, 32, 64, "paged")],
                         ids=lambda c: "-".join(map(str, c)))
@pytest.mark.parametrize("rows", [6, 600])
def test_a_scale_that_is_no_number_shows_in_every_row_that_sees_its_block_and_in_no_other(which, case, rows):
    """One kv head of the block of positions 64 .. 64 + block has it.  Drafted rows (some see the block, some do not) and
    rows of a window behind it; the few rows take the cluster's kernel, the many the other one."""
    from tessera_b200 import ops
    rng = np.random.default_rng(31)
    heads, kv_heads, width, block = case[:4]
    kv, kept, store = attend_case(rng, case, [300, 200])
    pos = [61, 62, 63, 64, 65, 66] if rows == 6 else [61 + i % 120 for i in range(rows)]
    pos[0] = 199
    q = bf16(rng, len(pos), heads, width)
    slots, at = dev_u32([0] * len(pos)), dev_u32(pos)
    group = heads // kv_heads
    blk, h = store.at(0, 64 // block), kv_heads - 1
    for back in (FAR, 40):
        clean = ops.attend_rows_q8(q, kv, slots, at, kept, 300, scale=width ** -0.5, back=back)
        ids = dev_u32(np.broadcast_to(np.arange(6, dtype=np.uint32), (len(pos), kv_heads, 6)))
        clean_listed = ops.attend_blocks_q8(q, kv, ids, slots, at, kept, 300, scale=width ** -0.5)
        scales = getattr(kv, which)
        was = scales[blk, h].clone()
        scales[blk, h] = float("nan")
        got = ops.attend_rows_q8(q, kv, slots, at, kept, 300, scale=width ** -0.5, back=back)
        listed = ops.attend_blocks_q8(q, kv, ids, slots, at, kept, 300, scale=width ** -0.5)
        scales[blk, h] = was
        for out, want, low in ((got, clean, [max(0, p - back) for p in pos]), (listed, clean_listed, [0] * len(pos))):
            sees = torch.tensor([p >= 64 and l < 64 + block for p, l in zip(pos, low)], device="cuda")
            if out is listed:
                sees &= 64 // block < 6
            mine = out[:, h * group:(h + 1) * group]
            assert torch.isnan(mine[sees].float()).all()
            assert torch.equal(mine[~sees], want[~sees][:, h * group:(h + 1) * group])
            assert torch.equal(out[:, :h * group], want[:, :h * group])


@pytest.mark.parametrize("width,block", [(64, 16), (128, 64), (128, 16), (256, 32)])
@pytest.mark.parametrize("length", [1, 3, 64])
def test_values_half_way_between_two_codes_take_the_even_one(width, block, length):
    """Values are bf16 and kept as they come, so that x / scale is often exactly half-way.  The codes equal round(x / scale)
    with the quotient rounded to f32 and no step more; codes that follow a grown scale equal round(code * old / new) so.
    The scales are maxima / 127 in f32.  Keys at position 0 with no norm are turned by nothing: the same."""
    from tessera_b200 import ops
    rng = np.random.default_rng(32)
    heads, kv_heads, slots, page = 1, 4, 60, 64
    kv = make(rng, kv_heads, width, block, 2 * slots, page)
    kept = ops.Kept("dense", 2 * page, None, 2 * slots * page)
    old = {n: getattr(kv, n).cpu().numpy() for n in ("v", "v_scale")}
    begin = [0 if s % 2 else 3 for s in range(slots)]  # fresh blocks, and blocks that hold other rows
    row_slots = [s for s in range(slots) for _ in range(length)]
    row_pos = [begin[s] + i for s in range(slots) for i in range(length)]
    # a largest value per slot, some below what is held, some above
    size = np.exp2(rng.integers(-4, 4, (slots, 1))).repeat(length, 0)[..., None]
    qkv = torch.from_numpy((rng.standard_normal((slots * length, heads + 2 * kv_heads, width)) * size).astype(np.float32)).cuda().bfloat16()
    ops.qk_norm_rope_append_q8(qkv.reshape(len(row_pos), -1), None, None, inv_freq(width), dev_u32(row_slots), dev_u32(row_pos), kv, kept,
                               heads, eps=1e-6)
    x = qkv.float().cpu().numpy()[:, heads + kv_heads:].reshape(slots, length, kv_heads, width)
    v, scale = kv.v.cpu().numpy(), kv.v_scale.cpu().numpy()
    per = 2 * page // block
    follows = 0
    for s in range(slots):
        for b in range((begin[s] + length - 1) // block + 1):
            blk, rows = s * per + b, [i for i in range(length) if (begin[s] + i) // block == b]
            at = [(begin[s] + i) % block for i in rows]
            most = np.abs(x[s, rows]).max((0, 2))
            was = np.zeros(kv_heads, np.float32) if 0 in at else old["v_scale"][blk]
            now = np.maximum(was, most / np.float32(127))
            assert np.array_equal(scale[blk], now)
            want = np.rint(x[s, rows] / now[:, None])  # f32
            assert np.array_equal(v[blk][:, at].transpose(1, 0, 2), want)
            held = [i for i in range(block) if i not in at]
            if 0 not in at:
                moved = (old["v"][blk][:, held].astype(np.float64) * was.astype(np.float64)[:, None, None] / now.astype(np.float64)[:, None, None])
                assert np.array_equal(v[blk][:, held], np.rint(moved.astype(np.float32)))
                follows += (now > was).sum()
    assert follows > 0 or length == 64 and block < 64
    fresh = [s for s in range(slots) if begin[s] == 0]
    k, k_scale = kv.k.cpu().numpy(), kv.k_scale.cpu().numpy()
    first = qkv.float().cpu().numpy()[[s * length for s in fresh], heads:heads + kv_heads]
    for i, s in enumerate(fresh):
        assert np.array_equal(k[s * per, :, 0], np.rint(first[i] / k_scale[s * per][:, None]))
    blocks = np.array([s * per for s in fresh])
    for j, pick in ((0, "min"), (1, "max")):  # and the bounds are those of the codes
        n = min(length, block)
        assert np.array_equal(kv.k_bounds.cpu().numpy()[blocks, :, j], getattr(k[blocks][:, :, :n], pick)(2))


def test_host_threads_on_one_stream_get_their_own_results():
    """Both calls leave partial results in scratch for a second kernel, and the library runs without the interpreter's lock."""
    import threading
    from tessera_b200 import ops
    rng = np.random.default_rng(33)
    case = (16, 8, 128, 16, 64, "paged")
    jobs = []
    for lengths in ([9000, 40, 8500], [8800, 8800, 9]):
        kv, kept, _ = attend_case(rng, case, lengths)
        q, slots, pos = bf16(rng, 3, 16, 128), dev_u32([0, 1, 2]), dev_u32([n - 1 for n in lengths])
        jobs.append(lambda q=q, kv=kv, slots=slots, pos=pos, kept=kept: (
            ops.attend_rows_q8(q, kv, slots, pos, kept, 9000, scale=0.09), ops.select_blocks_q8(q, kv, slots, pos, kept, 9000, 20)))
    want = [job() for job in jobs]
    torch.cuda.synchronize()
    stream, bad, meet = torch.cuda.Stream(), [], threading.Barrier(2, timeout=60)

    def work(i):
        with torch.cuda.stream(stream):
            for _ in range(20):
                meet.wait()
                got = [jobs[i]() for _ in range(20)]
                if not all(torch.equal(a, b) for g in got for a, b in zip(g, want[i])):
                    bad.append(i)

    threads = [threading.Thread(target=work, args=(i,)) for i in range(2)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not bad


@pytest.mark.parametrize("case", [(16, 8, 128, 64, 64, "paged"), (4, 4, 64, 16, 32, "dense"), (20, 1, 256, 32, 64, "paged")], ids=lambda c: "-".join(map(str, c)))
def test_keys_without_a_limit_are_the_room_of_a_slot(case):
    from tessera_b200 import _lib, ops
    import ctypes as C
    rng = np.random.default_rng(34)
    kv, kept, _ = attend_case(rng, case, [20000, 700])
    heads, kv_heads, width, block = case[:4]
    q, slots, pos = bf16(rng, 4, heads, width), dev_u32([0, 1, 1, 0]), dev_u32([19999, 5, 6, FAR])
    room = kept.scalar * (case[4] if case[5] == "paged" else 1)
    want = ops.attend_rows_q8(q, kv, slots, pos, kept, room, scale=0.09), ops.select_blocks_q8(q, kv, slots, pos, kept, room, 9)
    for keys in (room + 1, 1 << 28, FAR):
        assert torch.equal(ops.attend_rows_q8(q, kv, slots, pos, kept, keys, scale=0.09), want[0])
        assert torch.equal(ops.select_blocks_q8(q, kv, slots, pos, kept, keys, 9), want[1])
        # and through the library's own face, with the workspace that it asks for
        nbytes = _lib.lib.ts_attend_rows_q8_workspace_bytes(4, keys, heads, kv_heads, width, FAR)
        ws, out = torch.empty(nbytes, dtype=torch.uint8, device="cuda"), torch.empty_like(q)
        p = lambda t: C.c_void_p(t.data_ptr())  # noqa: E731
        _lib.check(_lib.lib.ts_attend_rows_q8(p(q), kv._held[0], p(out), p(slots), p(pos), kept.c(), 4, keys, heads, kv_heads, width, FAR,
                                              0.09, p(ws), nbytes, torch.cuda.current_stream().cuda_stream))
        assert torch.equal(out, want[0])


@pytest.mark.parametrize("case", [(16, 128, 4, 2, 64, True), (64, 128, 4, 2, 64, False), (32, 64, 3, 1, 32, True), (16, 256, 2, 2, 32, True), (64, 64, 2, 1, 64, True)],
                         ids=lambda c: "-".join(map(str, c)))
@pytest.mark.parametrize("order", ["draft by draft", "pairs apart", "any", "1024"])
def test_rows_of_a_block_may_stand_anywhere_in_a_call(case, order):
    """Against the definition, which knows no order but that of rows of one slot and position, the last of which counts; and
    the values, which are kept as they come, equal those of the same rows slot by slot to the bit.  (Keys do not have to:
    a run of up to four rows takes its angles from the positions, a longer one turns on by a fixed angle from pass to
    pass, at most 15 times 2^-24; the tolerances of check_append hold for both.)"""
    from tessera_b200 import ops
    rng = np.random.default_rng(35)
    block, width, heads, kv_heads, page, norm = case
    slots, per = 11, 5
    kv = make(rng, kv_heads, width, block, slots * per, page)
    kept, table = paged(rng, slots, per, slots * per, page)
    store = M.Store(kv, "paged", per, page, table)
    begin = rng.integers(0, 2 * block, slots)
    each = {"draft by draft": 5, "pairs apart": 2, "any": block + 3, "1024": 93}[order]
    where = [(s, int(begin[s]) + i) for i in range(each) for s in range(slots)]
    where = [w for w in where if w[1] < per * page]
    if order in ("any", "1024"):
        where = [where[i] for i in rng.permutation(len(where))] + where[:4]  # some of them twice
        where = where[:1024]
    if order == "1024" and len(where) > 1000:
        where += [where[0]] * (1024 - len(where))
    qkv = bf16(rng, len(where), (heads + 2 * kv_heads) * width, std=1.5)
    gain = torch.ones(width, device="cuda") * 1.25 if norm else None
    twin, other = (ops.RowsQ8(*(t.clone() for t in (kv.k, kv.v, kv.k_scale, kv.v_scale, kv.k_bounds))) for _ in range(2))

    def feed(into, rows):
        at = [dev_u32([where[r][j] for r in rows]) for j in (0, 1)]
        return ops.qk_norm_rope_append_q8(qkv[torch.tensor(rows, device="cuda")].contiguous(), gain, gain, inv_freq(width), *at, into, kept, heads, eps=1e-6)

    row_slots, row_pos = [w[0] for w in where], [w[1] for w in where]
    f = None if gain is None else gain.cpu().numpy().astype(np.float64)
    want_q, k, v = M.prepared(np64(qkv), f, f, inv_freq(width).cpu().numpy(), row_pos, heads, kv_heads, width, 1e-6)
    raw = M.append(store, k, v, row_slots, row_pos)
    got = feed(kv, list(range(len(where))))
    check_append(kv, None, store, raw, want_q, got)
    feed(other, list(range(len(where))))
    last = {w: r for r, w in enumerate(where)}
    for s in range(slots):
        feed(twin, [r for w, r in sorted(last.items()) if w[0] == s])
    assert torch.equal(kv.v, twin.v) and torch.equal(kv.v_scale, twin.v_scale)
    for n in ("k", "v", "k_scale", "v_scale", "k_bounds"):  # nothing of it is left to chance
        again = getattr(other, n)
        assert torch.equal(again, getattr(kv, n)), n


@pytest.mark.parametrize("case", [(4, 2, 128, 16, 16, "dense"), (16, 1, 64, 32, 32, "paged"), (2, 1, 256, 64, 64, "dense")], ids=lambda c: "-".join(map(str, c)))
def test_attention_over_infinities_as_append_keeps_them(case):
    """An infinite value is kept as the largest finite one: outputs stay finite.  So is an infinite key, but its score leaves
    f32: where it is +infinity the head is NaN, where it is -infinity the key has no weight."""
    from tessera_b200 import ops
    rng = np.random.default_rng(36)
    heads, kv_heads, width, block = case[:4]
    n = 3 * block
    kv, kept, _ = attend_case(rng, case, [n, n])
    where = [(s, p) for s in (0, 1) for p in range(n)]
    qkv = bf16(rng, len(where), heads + 2 * kv_heads, width)
    qkv[5, heads + kv_heads:, 3] = float("inf")  # a value of slot 0
    qkv[n, heads:heads + kv_heads, 3] = float("inf")  # the key at slot 1's position 0, which rotation leaves as it is but for ...
    qkv[n, heads:heads + kv_heads, width // 2 + 3] = 0.0  # ... 0 * infinity: its pair is NaN then, which is kept as 0
    ops.qk_norm_rope_append_q8(qkv.reshape(len(where), -1), None, None, inv_freq(width), dev_u32([w[0] for w in where]),
                               dev_u32([w[1] for w in where]), kv, kept, heads, eps=1e-6)
    k8, v8 = ops.rows_unpack_q8(kv, dev_u32([0, 1]), dev_u32([5, 0]), kept)
    assert torch.isfinite(k8.float()).all() and torch.isfinite(v8.float()).all()
    assert (v8[0, :, 3].float() > 3e38).all() and (k8[1, :, 3].float() > 3e38).all()
    q = bf16(rng, 3, heads, width)
    q[1, :, 3], q[2, :, 3] = 8.0, -8.0
    for run in (lambda: ops.attend_rows_q8(q, kv, dev_u32([0, 1, 1]), dev_u32([n - 1] * 3), kept, n, scale=1.0),
                lambda: ops.attend_blocks_q8(q, kv, dev_u32(np.broadcast_to(np.arange(3, dtype=np.uint32), (3, kv_heads, 3))),
                                             dev_u32([0, 1, 1]), dev_u32([n - 1] * 3), kept, n, scale=1.0)):
        out = run()
        assert torch.isfinite(out[0].float()).all() and torch.isnan(out[1].float()).all() and torch.isfinite(out[2].float()).all()


@pytest.mark.parametrize("case", [(4, 2, 128, 64, 64, "dense"), (16, 1, 64, 16, 64, "paged"), (8, 1, 256, 32, 64, "dense")], ids=lambda c: "-".join(map(str, c)))
@pytest.mark.parametrize("ratio", [30, 300, 3000])
def test_queries_with_one_channel_far_above_the_others(case, ratio):
    """A query is rounded to steps of its head's largest magnitude / 32639: with the queries rounded so in 64 bits the
    tolerance is the usual one.  An element counted in steps is off by two roundings, 2^-23 of itself, so those nearer than
    2^-21 of themselves to a half may be rounded the other way: a score is then off by a step times those keys' magnitudes,
    d in all, and the output by (e^(2 d) - 1) sum p |v|.  Against the queries as they are, every element may be off by half
    a step.  (The keys of the large channel are zero, so that the others decide.)"""
    from tessera_b200 import ops
    rng = np.random.default_rng(37)
    heads, kv_heads, width, block = case[:4]
    n = 700
    kv, kept, store = attend_case(rng, case, [n, n])
    kv.k[..., 5] = 0
    store = M.Store(kv, store.layout, store.scalar, store.page, store.table)
    slots, pos, scale = [0, 1, 1, 0], [n - 1, 333, 334, 20], 5 * width ** -0.5
    q = bf16(rng, 4, heads, width)
    q[..., 5] = torch.tensor([1.0, -1.0], device="cuda").repeat(heads // 2) * ratio
    got = np64(ops.attend_rows_q8(q, kv, dev_u32(slots), dev_u32(pos), kept, n, scale=scale))
    x = np64(q)
    step = np.abs(x).max(-1, keepdims=True) / 32639
    units = x / step
    rounded = np.rint(units) * step
    unsure = np.abs(np.abs(units - np.floor(units)) - 0.5) < 2.0 ** -21 * np.abs(units)
    group = heads // kv_heads
    most = np.stack([np.abs(store.keys_of(s, h, range(p + 1))[0]).max(0) for s, p in zip(slots, pos) for h in range(kv_heads)])
    most = most.reshape(4, kv_heads, 1, width).repeat(group, 2).reshape(4, heads, width)
    for query, off in ((rounded, scale * (step * unsure * most).sum(-1)), (x, scale * (step * 0.51 * most).sum(-1))):
        want, tol = M.attend(store, query, slots, pos, n, scale)
        weighed = (tol - 2.0 ** -8 * np.abs(want)) * 2.0 ** 10  # at least the sum of p |v|
        assert np.all(np.abs(got - want) <= tol + np.expm1(2 * off)[..., None] * weighed)


def test_more_rows_than_one_attention_launch_counts_steps_for():
    """Steps are counted in 32 bits by a slot's room: with 2^22 positions of 8 kv heads a launch takes 2040 rows.  The rows
    of all launches, the shorter last one among them, equal those of calls of their own."""
    from tessera_b200 import ops
    rng = np.random.default_rng(38)
    heads, kv_heads, width, block, room, rows = 16, 8, 128, 64, 1 << 22, 4500
    kv = make(rng, kv_heads, width, block, 8, 64)
    kept = ops.Kept("dense", room, None, 8 * 64)  # a pool far smaller than the room: positions past it are not there
    q = bf16(rng, rows, heads, width)
    at = rng.integers(0, 500, rows).astype(np.uint32)
    at[1000:1040] = np.arange(100, 140)  # drafted rows too, and some on both sides of a launch's end
    at[2030:2060] = np.arange(200, 230)
    slots, pos = dev_u32([0] * rows), dev_u32(at)
    got = ops.attend_rows_q8(q, kv, slots, pos, kept, room, scale=0.09)
    cuts = list(range(0, rows, 300)) + [rows]
    for a, b in zip(cuts, cuts[1:]):
        want = ops.attend_rows_q8(q[a:b].contiguous(), kv, slots[a:b].contiguous(), pos[a:b].contiguous(), kept, 512, scale=0.09)
        # the two calls cut a row's keys in different places: two roundings to bf16 and the sums' own error apart
        x, y = got[a:b].float(), want.float()
        assert torch.all((x - y).abs() <= 2.0 ** -7 * y.abs() + 2.0 ** -9 * 127 * 0.05), (x - y).abs().max()
    store = M.Store(kv, "dense", room)
    sample = [0, 1, 1005, 2031, 2038, 2039, 2040, 2041, 2055, 4079, 4080, 4499]
    want, tol = M.attend(store, np64(q[torch.tensor(sample, device="cuda")]), [0] * len(sample), at[sample], room, 0.09)
    off = np.abs(np64(got[torch.tensor(sample, device="cuda")]) - want)
    assert np.all(off <= tol)


@pytest.mark.parametrize("width", [64, 128, 256])
@pytest.mark.parametrize("kv_heads,rows", [(1, 3), (1, 127), (1, 128), (8, 37), (8, 38), (2, 149)])
@pytest.mark.parametrize("blocks", [65, 256, 257, 512, 513])
def test_choices_on_both_sides_of_one_and_two_launches(width, kv_heads, rows, blocks):
    """One kernel or two launches, by rows x kv heads, blocks and width: the ids are the definition's either way."""
    from tessera_b200 import ops
    rng = np.random.default_rng(39)
    block, heads = 16, 2 * kv_heads
    kv, kept, store = attend_case(rng, (heads, kv_heads, width, block, 16, "dense"), [blocks * block])
    three = bf16(rng, 3, heads, width)
    which = torch.arange(rows, device="cuda") % 3
    q, pos = three[which].contiguous(), [blocks * block - 1, blocks * block - 5, 70 * block]
    got = ops.select_blocks_q8(q, kv, dev_u32([0] * rows), dev_u32([pos[r % 3] for r in range(rows)]), kept, blocks * block, 40, first=1, recent=2)
    want = M.select(store, np64(three), [0, 0, 0], pos, blocks * block, 40, 1, 2)
    assert torch.equal(got, torch.from_numpy(want.astype(np.int32)).cuda()[which])


def test_steps_of_dependent_launches_give_the_same_bits():
    """Append, read back, attention and choice as programmatic dependent launches: each waits for what the one before wrote."""
    from tessera_b200 import ops
    case = (16, 8, 128, 16, 64, "paged")
    heads, kv_heads, width = case[:3]

    def steps():
        rng = np.random.default_rng(40)
        kv, kept, _ = attend_case(rng, case, [1500, 900, 60])
        outs = []
        for step in range(12):
            slots = [0, 1, 2, 0, 1, 2] if step % 2 else [0, 1, 2]
            pos = [[1400, 800, 10][s] + 2 * step + i // 3 for i, s in enumerate(slots)]
            at = dev_u32(slots), dev_u32(pos)
            qkv = bf16(rng, len(slots), (heads + 2 * kv_heads) * width, std=1 + step)
            q = ops.qk_norm_rope_append_q8(qkv, None, None, inv_freq(width), *at, kv, kept, heads, eps=1e-6)
            ids = ops.select_blocks_q8(q, kv, *at, kept, 1500, 20)
            outs += [q, ops.attend_rows_q8(q, kv, *at, kept, 1500, scale=0.09), ids,
                     ops.attend_blocks_q8(q, kv, ids, *at, kept, 1500, scale=0.09), *ops.rows_unpack_q8(kv, *at, kept)]
        return outs + [kv.k.clone(), kv.v.clone(), kv.k_scale.clone(), kv.v_scale.clone(), kv.k_bounds.clone()]

    want = steps()
    ops.set_pdl(True)
    try:
        for _ in range(5):
            assert all(torch.equal(a, b) for a, b in zip(steps(), want))
    finally:
        ops.set_pdl(False)
    assert ops.device_status() == 0
