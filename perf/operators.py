"""Operators over kept rows held in 8 bits, as a decoder that serves long contexts runs them.

The kept keys and values of a slot are signed 8-bit codes in blocks of `block` positions; every block and kv head
has one f32 scale for its keys and one for its values, and (for the choice of blocks) the lowest and the highest
key code of each channel.  Layouts: codes int8 [blocks, kv_heads, block, width], scales f32 [blocks, kv_heads],
bounds int8 [blocks, kv_heads, 2, width]; the block of a slot's position goes through the page table.

  append   per-head norm and rotation of q and k, q out, k and v into their blocks (scales grow, held codes follow)
  read     kept rows of given slots and positions back as bf16
  attend   causal attention of rows over their slots' 8-bit rows
  select   the blocks that a row and kv head should read, by an upper bound of q . k from the block's bounds
  blocks   causal attention over chosen blocks only

`run` computes one of them, in plain torch operations or (own) through tessera_b200.ops.
"""
import math

import torch

own = False

FLOOR = 2.0 ** -60   # the smallest scale a block gets
SPARE = -1           # an entry of a block list that names no block (all bits set)
FAR = 0xFFFFFFFF     # no window


# ---- the cases ---------------------------------------------------------------------------------------------------

def listed():
    return [
        # one decode step's append: a token for each of 64 slots, far into their contexts, blocks partly filled
        dict(name="append step 64", op="append", slots=64, length=1, far=32000, aligned=False, heads=16, kv_heads=8, width=128, page=64, block=16, norm=True),
        # prompts: three of them, of odd lengths, one starting a block, two inside a block that holds earlier rows
        dict(name="append prompts 8165", op="append", slots=3, length=2722, far=5000, aligned=True, heads=16, kv_heads=8, width=128, page=64, block=64, norm=True),
        # a short prefix that another request shares, read back in bf16 for its prompt's attention
        dict(name="read prefix 160", op="read", slots=1, length=160, heads=32, kv_heads=8, width=64, page=16, block=16),
        # long prefixes of two requests
        dict(name="read prefix 2x16001", op="read", slots=2, length=16001, heads=16, kv_heads=8, width=128, page=64, block=64),
        # the first steps of a single conversation
        dict(name="attend 1x517", op="attend", slots=1, each=1, length=517, heads=16, kv_heads=8, width=128, page=64, block=16, back=FAR),
        # a full batch of decode rows, ragged lengths of 8192 at most
        dict(name="attend 64x8192", op="attend", slots=64, each=1, length=8192, heads=16, kv_heads=8, width=128, page=64, block=64, back=FAR),
        # a few very long documents, four query heads a kv head
        dict(name="attend 4x100003", op="attend", slots=4, each=1, length=100003, heads=32, kv_heads=8, width=128, page=64, block=32, back=FAR),
        # drafted tokens: eight rows of each slot are checked in one step, eight query heads a kv head
        dict(name="attend drafts 16x7x4099", op="attend", slots=16, each=7, length=4099, heads=32, kv_heads=4, width=128, page=64, block=64, back=FAR),
        # which blocks to read: a small batch of medium contexts, a large one of long contexts
        dict(name="select 8x4096", op="select", slots=8, each=1, length=4096, heads=16, kv_heads=8, width=128, page=64, block=16, count=32, first=1, recent=2),
        dict(name="select 64x32768", op="select", slots=64, each=1, length=32768, heads=32, kv_heads=4, width=128, page=64, block=64, count=64, first=1, recent=1),
        # and the attention over what was chosen
        dict(name="blocks 8 of 32x16", op="blocks", slots=8, each=1, length=4096, heads=16, kv_heads=8, width=128, page=64, block=16, count=32, first=1, recent=2),
        dict(name="blocks 64 of 64x64", op="blocks", slots=64, each=1, length=32768, heads=32, kv_heads=4, width=128, page=64, block=64, count=64, first=1, recent=1),
    ]


def _spread(rng, lo, hi):
    """A whole number between lo and hi, its logarithm spread evenly."""
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["append", "read", "attend", "select", "blocks"])
    kv_heads = rng.choice([1, 2, 4, 8])
    heads = kv_heads * rng.choice([1, 2, 3, 4, 8])
    width = rng.choice([64, 128, 128, 256])
    block = rng.choice([16, 32, 64])
    case = dict(op=op, heads=heads, kv_heads=kv_heads, width=width, page=max(block, rng.choice([16, 64, 128])), block=block)
    per = kv_heads * width  # values of a position: the bounds below keep a draw under the largest listed case
    if op == "append":
        length = rng.choice([1, 1, _spread(rng, 2, 4000)])
        slots = _spread(rng, 1, max(1, min(256, 8000 // length)))
        return dict(case, slots=slots, length=length, far=_spread(rng, 2 * length, 100000), aligned=rng.random() < 0.5, norm=rng.random() < 0.8)
    if op == "read":
        slots = _spread(rng, 1, 8)
        return dict(case, slots=slots, length=_spread(rng, 1, max(1, 30000000 // (per * slots))))
    slots = _spread(rng, 1, 64)
    each = rng.choice([1, 1, 1, rng.randint(2, 8)])
    longest = max(64, min(120000, 60000000 // (slots * each) * 8 // per))
    case = dict(case, slots=slots, each=each, length=_spread(rng, max(1, each), longest))
    if op == "attend":
        return dict(case, back=rng.choice([FAR, FAR, _spread(rng, 1, case["length"])]))
    first, recent = rng.randint(0, 2), rng.randint(1, 3)
    return dict(case, count=first + recent + _spread(rng, 1, 96), first=first, recent=recent)


def _starts(case):
    """Slot, first position and number of rows of each slot's part of an append, from the case alone."""
    at = []
    for s in range(case["slots"]):
        begin = case["far"] * ((s + 1) * 40503 % 65536) // 65536  # spread over the context
        if case["aligned"] and s % 3 == 0:
            begin -= begin % case["block"]
        at.append((s, begin, max(1, case["length"] - 7 * s)))
    return at


def _lengths(case):
    """How many positions each slot holds: ragged, the first one full."""
    return [max(case.get("each", 1), case["length"] - (case["length"] * ((s * 40503) % 65536) // 65536) // 2) for s in range(case["slots"])]


# ---- inputs ------------------------------------------------------------------------------------------------------

def _kept_rows(case, pages, gen):
    """Codes as quantised normal values have them, scales of some spread, and the bounds of the key codes."""
    block, kv_heads, width = case["block"], case["kv_heads"], case["width"]
    blocks = pages * (case["page"] // block)
    out = {}
    for name in ("k", "v"):
        codes = torch.empty((blocks, kv_heads, block, width), dtype=torch.int8, device="cuda")
        for at in range(0, blocks, max(1, (1 << 26) // (kv_heads * block * width))):
            part = codes[at:at + max(1, (1 << 26) // (kv_heads * block * width))]
            part.copy_((torch.randn(part.shape, device="cuda", generator=gen) * 36).round_().clamp_(-127, 127))
        out[name] = codes
        out[name + "_scale"] = 0.027 * torch.exp(0.3 * torch.randn((blocks, kv_heads), device="cuda", generator=gen))
    out["bounds"] = torch.stack([out["k"].amin(2), out["k"].amax(2)], 2).contiguous()
    return out


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    slots, page, block, width = case["slots"], case["page"], case["block"], case["width"]
    heads, kv_heads = case["heads"], case["kv_heads"]
    lists = _starts(case) if case["op"] == "append" else None
    # The page table: pages in shuffled order.  In an append only the pages that are written are in the pool (a
    # server lets go of what lies behind a window); the entries before them are never read.
    if lists:
        spans = [(b // page, (b + n - 1) // page) for _, b, n in lists]
    else:
        spans = [(0, (n - 1) // page) for n in _lengths(case)]
    kept_pages = max(last for _, last in spans) + 1
    pages = sum(last - first + 1 for first, last in spans)
    order = torch.randperm(pages, device="cuda", generator=gen).to(torch.int32)
    table = torch.zeros((slots, kept_pages), dtype=torch.int32, device="cuda")
    at = 0
    for s, (first, last) in enumerate(spans):
        table[s, first:last + 1] = order[at:at + last - first + 1]
        at += last - first + 1
    state = dict(case=case, table=table, pages=pages, kept_pages=kept_pages, **_kept_rows(case, pages, gen))
    if lists:
        slot = [s for s, _, n in lists for _ in range(n)]
        position = [b + i for _, b, n in lists for i in range(n)]
        rows = len(slot)
        scale = torch.exp(0.5 * torch.randn((1, heads + 2 * kv_heads, 1), device="cuda", generator=gen))
        state["qkv"] = (torch.randn((rows, heads + 2 * kv_heads, width), device="cuda", generator=gen) * scale).bfloat16().reshape(rows, -1)
        state["q_norm"] = 1 + 0.1 * torch.randn(width, device="cuda", generator=gen) if case["norm"] else None
        state["k_norm"] = 1 + 0.1 * torch.randn(width, device="cuda", generator=gen) if case["norm"] else None
        state["inv_freq"] = (1e6 ** (-torch.arange(0, width, 2, device="cuda", dtype=torch.float64) / width)).float()
        # every row of the pool, to be read back
        where = [(s, p) for s, (first, last) in enumerate(spans) for p in range(first * page, (last + 1) * page)]
        state["read_slots"] = torch.tensor([s for s, _ in where], dtype=torch.int32, device="cuda")
        state["read_positions"] = torch.tensor([p for _, p in where], dtype=torch.int32, device="cuda")
        state["bounds_out"] = torch.empty(state["bounds"].shape, dtype=torch.bfloat16, device="cuda")
    elif case["op"] == "read":
        slot = [s for s, n in enumerate(_lengths(case)) for _ in range(n)]
        position = [p for n in _lengths(case) for p in range(n)]
    else:
        slot = [s for s in range(slots) for _ in range(case["each"])]
        position = [n - case["each"] + i for n in _lengths(case) for i in range(case["each"])]
        rows = len(slot)
        state["q"] = torch.randn((rows, heads, width), device="cuda", generator=gen).bfloat16()
        state["keys"] = max(_lengths(case))
    state["slots"] = torch.tensor(slot, dtype=torch.int32, device="cuda")
    state["positions"] = torch.tensor(position, dtype=torch.int32, device="cuda")
    if case["op"] == "blocks":
        state["ids"] = _some_blocks(case, state, gen)
    if own:
        from tessera_b200 import ops
        state["kv"] = ops.RowsQ8(state["k"], state["v"], state["k_scale"], state["v_scale"], state["bounds"])
        state["kept"] = ops.Kept("paged", kept_pages, table.reshape(-1), pages * page, page=page)
    return state


def _some_blocks(case, state, gen):
    """Ascending lists of blocks that a row may see: the first ones, the most recent ones and others at random."""
    rows, count = len(state["positions"]), case["count"]
    have = (state["positions"].long() // case["block"] + 1)[:, None, None]  # blocks in sight
    most = int(have.max())
    want = torch.rand((rows, case["kv_heads"], most), device="cuda", generator=gen)
    at = torch.arange(most, device="cuda")
    want = torch.where((at < case["first"]) | ((at >= have - case["recent"]) & (at < have)), 2.0, want)
    want = torch.where(at < have, want, -1.0)
    take = min(count, most)
    value, index = torch.topk(want, take, dim=2)
    ids = torch.where(value >= 0, index, most).sort(dim=2).values
    ids = torch.where(ids < most, ids, SPARE)
    return torch.nn.functional.pad(ids, (0, count - take), value=SPARE).to(torch.int32)


# ---- the plain forms ---------------------------------------------------------------------------------------------

def _block_of(state, slot, block_index):
    """Which block of the pool holds block `block_index` of a slot's positions."""
    per = state["case"]["page"] // state["case"]["block"]
    page = state["table"][slot, block_index // per].long()
    return page * per + block_index % per


def _plain_append(state):
    c = state["case"]
    heads, kv_heads, width, block = c["heads"], c["kv_heads"], c["width"], c["block"]
    rows = state["qkv"].shape[0]
    x = state["qkv"].float().reshape(rows, heads + 2 * kv_heads, width)
    q, k, v = x[:, :heads], x[:, heads:heads + kv_heads], x[:, heads + kv_heads:]
    angle = state["positions"].double()[:, None] * state["inv_freq"].double()
    cos, sin = torch.cos(angle).float()[:, None], torch.sin(angle).float()[:, None]

    def turned(t, gain):
        if gain is not None:
            t = t * (1.0 / torch.sqrt(t.square().mean(-1, keepdim=True) + 1e-6)) * gain
        a, b = t[..., :width // 2], t[..., width // 2:]
        return torch.cat([a * cos - b * sin, a * sin + b * cos], -1)

    q_out, k = turned(q, state["q_norm"]).bfloat16(), turned(k, state["k_norm"])
    slot, position = state["slots"].long(), state["positions"].long()
    blk, within = _block_of(state, slot, position // block), position % block
    blocks = state["k"].shape[0]
    touched = torch.zeros(blocks, device="cuda").index_fill_(0, blk, 1.0)[:, None] > 0
    starts = torch.zeros(blocks, device="cuda").index_reduce_(0, blk, (within == 0).float(), "amax")[:, None] > 0
    for_k = None
    for name, t in (("k", k), ("v", v)):
        codes, scale = state[name], state[name + "_scale"]
        most = torch.zeros((blocks, kv_heads), device="cuda").index_reduce_(0, blk, t.abs().amax(-1), "amax")
        new = torch.maximum(torch.where(starts, 0.0, scale), (most / 127).clamp_min(FLOOR))
        new = torch.where(touched, new, scale)
        ratio = torch.where(starts, 1.0, scale / new)
        written = torch.round(t / new[blk][..., None]).clamp(-127, 127)
        codes.copy_(torch.round(codes.float() * ratio[..., None, None]))
        codes[blk, :, within] = written.to(torch.int8)
        scale.copy_(new)
        if name == "k":
            for_k = ratio, written
    ratio, written = for_k
    low = torch.where(starts[..., None], 127.0, torch.round(state["bounds"][:, :, 0].float() * ratio[..., None]))
    high = torch.where(starts[..., None], -127.0, torch.round(state["bounds"][:, :, 1].float() * ratio[..., None]))
    low.index_reduce_(0, blk, written, "amin")
    high.index_reduce_(0, blk, written, "amax")
    state["bounds"].copy_(torch.stack([low, high], 2))
    return q_out


def _plain_read(state, slots, positions):
    block = state["case"]["block"]
    position = positions.long()
    blk = _block_of(state, slots.long(), position // block)
    return [(state[n][blk, :, position % block].float() * state[n + "_scale"][blk][..., None]).bfloat16() for n in ("k", "v")]


def _plain_attention(state, blk, at, back):
    """Softmax over the keys of blocks `blk` [rows, kv_heads, n] of the pool, whose first positions are `at` (negative:
    no block)."""
    c = state["case"]
    rows, kv_heads, n = blk.shape
    block, width, group = c["block"], c["width"], c["heads"] // c["kv_heads"]
    head = torch.arange(kv_heads, device="cuda")[:, None]
    key = (at[..., None] + torch.arange(block, device="cuda")).reshape(rows, kv_heads, 1, n * block)
    position = state["positions"].long()[:, None, None, None]
    seen = (key >= 0) & (key <= position) & (key >= position - back) & (key < state["keys"])
    seen &= (at[..., None] >= 0).expand(rows, kv_heads, n, block).reshape(rows, kv_heads, 1, n * block)
    q = state["q"].float().reshape(rows, kv_heads, group, width)
    k = (state["k"][blk, head].float() * state["k_scale"][blk, head][..., None, None]).reshape(rows, kv_heads, n * block, width)
    score = torch.matmul(q, k.transpose(-1, -2)) * width ** -0.5
    del k
    score = torch.where(seen, score, -math.inf)
    most = score.amax(-1, keepdim=True)
    p = torch.exp(score - torch.where(most == -math.inf, 0.0, most))
    v = (state["v"][blk, head].float() * state["v_scale"][blk, head][..., None, None]).reshape(rows, kv_heads, n * block, width)
    total = p.sum(-1, keepdim=True)
    out = torch.matmul(p, v) / torch.where(total == 0, 1.0, total)
    return out.reshape(rows, c["heads"], width).bfloat16()


def _all_blocks(state):
    c = state["case"]
    n = -(-state["keys"] // c["block"])
    index = torch.arange(n, device="cuda")[None]
    have = state["positions"].long()[:, None] // c["block"]  # later blocks are out of sight and may have no page
    blk = _block_of(state, state["slots"].long()[:, None], torch.minimum(index, have))
    shape = (blk.shape[0], c["kv_heads"], n)
    return blk[:, None].expand(shape), (index * c["block"])[:, None].expand(shape)


def _plain_select(state):
    c = state["case"]
    rows, kv_heads, group, width, block = state["q"].shape[0], c["kv_heads"], c["heads"] // c["kv_heads"], c["width"], c["block"]
    q = state["q"].float().reshape(rows, kv_heads, group, width)
    most = q.abs().amax((-1, -2), keepdim=True)
    codes = torch.where(most > 0, torch.round(q * 127 / torch.where(most > 0, most, 1.0)), 0.0)
    up, down = codes.clamp_min(0).sum(2), codes.clamp_max(0).sum(2)  # [rows, kv_heads, width]
    blk, at = _all_blocks(state)
    head = torch.arange(kv_heads, device="cuda")[:, None]
    bounds = state["bounds"][blk, head].double()  # whole numbers, summed without rounding
    total = torch.matmul(bounds[..., 1, :], up.double()[..., None])[..., 0] + torch.matmul(bounds[..., 0, :], down.double()[..., None])[..., 0]
    score = total.float() * state["k_scale"][blk, head]
    n = score.shape[-1]
    have = torch.minimum(state["positions"].long(), torch.tensor(state["keys"] - 1, device="cuda"))[:, None, None] // block + 1
    index = torch.arange(n, device="cuda")
    score = torch.where((index < c["first"]) | (index >= have - c["recent"]), math.inf, score)
    score = torch.where(index < have, score, -math.inf)
    order = torch.sort(score, dim=-1, descending=True, stable=True).indices[..., :c["count"]]
    ids = torch.where(order < have, order, n).sort(dim=-1).values
    ids = torch.where(ids < n, ids, SPARE)
    return torch.nn.functional.pad(ids, (0, c["count"] - ids.shape[-1]), value=SPARE).to(torch.int32)


def _plain_blocks(state):
    c = state["case"]
    ids = state["ids"].long()
    here = (ids * c["block"] <= state["positions"].long()[:, None, None]) & (ids != SPARE)
    index = torch.where(here, ids, 0)
    blk = _block_of(state, state["slots"].long()[:, None, None], index)
    return _plain_attention(state, blk, torch.where(here, ids * c["block"], -1 << 40), FAR)


# ---- one pass ----------------------------------------------------------------------------------------------------

def run(state):
    c = state["case"]
    if own:
        from tessera_b200 import ops
        kv, kept, slots, positions = state["kv"], state["kept"], state["slots"], state["positions"]
        if c["op"] == "append":
            q = ops.qk_norm_rope_append_q8(state["qkv"], state["q_norm"], state["k_norm"], state["inv_freq"], slots, positions, kv, kept, c["heads"], eps=1e-6)
            k, v = ops.rows_unpack_q8(kv, state["read_slots"], state["read_positions"], kept)
        elif c["op"] == "read":
            k, v = ops.rows_unpack_q8(kv, slots, positions, kept)
        elif c["op"] == "attend":
            return ops.attend_rows_q8(state["q"], kv, slots, positions, kept, state["keys"], scale=c["width"] ** -0.5, back=c["back"])
        elif c["op"] == "select":
            return ops.select_blocks_q8(state["q"], kv, slots, positions, kept, state["keys"], c["count"], first=c["first"], recent=c["recent"])
        else:
            return ops.attend_blocks_q8(state["q"], kv, state["ids"], slots, positions, kept, state["keys"], scale=c["width"] ** -0.5)
    elif c["op"] == "append":
        q = _plain_append(state)
        k, v = _plain_read(state, state["read_slots"], state["read_positions"])
    elif c["op"] == "read":
        k, v = _plain_read(state, state["slots"], state["positions"])
    elif c["op"] == "attend":
        return _plain_attention(state, *_all_blocks(state), c["back"])
    elif c["op"] == "select":
        return _plain_select(state)
    else:
        return _plain_blocks(state)
    if c["op"] == "read":
        return {"k": k, "v": v}
    torch.mul(state["bounds"], state["k_scale"][..., None, None], out=state["bounds_out"])
    return {"q": q, "k": k, "v": v, "k_scale": state["k_scale"], "v_scale": state["v_scale"], "bounds": state["bounds_out"]}


def work(case):
    heads, kv_heads, width, block, page = case["heads"], case["kv_heads"], case["width"], case["block"], case["page"]
    row = kv_heads * (width + 4 / block)  # bytes of a position's keys, or values, with their share of the scales
    if case["op"] == "append":
        at = _starts(case)
        n = sum(n for _, _, n in at)
        held = sum(((b + n - 1) // page - b // page + 1) * page for _, b, n in at)
        moved = n * (2 * heads + 2 * kv_heads) * width * 2 + n * 2 * row      # qkv in, q and the codes out
        moved += held * (2 * row + 2 * kv_heads * width * 2)                  # the pool read back in bf16
        moved += held / block * 2 * kv_heads * width * 3                      # bounds in, their values out
        return {"bytes": moved, "flops": n * (heads + 2 * kv_heads) * width * 8}
    if case["op"] == "read":
        n = sum(_lengths(case))
        return {"bytes": n * (2 * row + 2 * kv_heads * width * 2), "flops": n * 2 * kv_heads * width}
    held, rows = _lengths(case), case["slots"] * case["each"]
    if case["op"] == "select":
        blocks = sum(-(-n // block) for n in held)
        return {"bytes": blocks * kv_heads * (2 * width + 4) + rows * (heads * width * 2 + kv_heads * case["count"] * 4),
                "flops": case["each"] * blocks * kv_heads * 4 * width}
    # keys that a row sees; the rows of a slot share what they read
    if case["op"] == "attend":
        read = sum(min(n, case["back"] + case["each"]) for n in held)
        seen = sum(min(n, case["back"] + 1) for n in held) * case["each"]
    else:
        read = seen = sum(min(n, case["count"] * block) for n in held) * case["each"]
        read = min(read, sum(held))
    return {"bytes": read * 2 * row + rows * heads * width * 4, "flops": seen * heads * width * 4}


# ---- the definitions in 64 bits ----------------------------------------------------------------------------------

def exact(case, seed):
    state = prepare(case, seed)
    op, block, page, width = case["op"], case["block"], case["page"], case["width"]
    heads, kv_heads = case["heads"], case["kv_heads"]
    group, per = heads // kv_heads, page // block
    table = state["table"].cpu().tolist()
    slots, positions = state["slots"].tolist(), state["positions"].tolist()

    def places(slot, count):
        return torch.tensor([table[slot][j // per] * per + j % per for j in range(count)], device="cuda")

    if op == "select":
        return None  # whole numbers: the plain form's sums have no rounding
    if op in ("append", "read"):
        if op == "append":
            if len(slots) > 20000:
                return None
            q, scales, codes, bounds = _exact_append(state, table, per)
            slots, positions = state["read_slots"].tolist(), state["read_positions"].tolist()
        else:
            codes, scales = {n: state[n] for n in "kv"}, {n: state[n + "_scale"].double() for n in "kv"}
        at = torch.tensor([table[s][p // page] * page + p % page for s, p in zip(slots, positions)], device="cuda")
        values = {n: codes[n].transpose(1, 2).reshape(-1, kv_heads, width)[at].double() * scales[n].repeat_interleave(block, 0)[at][..., None] for n in "kv"}
        if op == "read":
            return values
        return {"q": q, **values, "k_scale": scales["k"], "v_scale": scales["v"], "bounds": bounds * scales["k"][..., None, None]}
    out = torch.zeros((len(slots), heads, width), dtype=torch.float64, device="cuda")
    ids = state["ids"].tolist() if op == "blocks" else None
    for r, (s, p) in enumerate(zip(slots, positions)):
        in_sight = p // block + 1
        blk = places(s, in_sight)
        for h in range(kv_heads):
            if op == "attend":
                low = max(0, p - case["back"]) // block
                chosen = torch.arange(low, in_sight, device="cuda")
            else:
                chosen = torch.tensor([i for i in ids[r][h] if 0 <= i < in_sight], device="cuda", dtype=torch.int64)
            key = (chosen[:, None] * block + torch.arange(block, device="cuda")).reshape(-1)
            keep = (key <= p) & (key >= p - case.get("back", FAR))
            k = (state["k"][blk[chosen], h].double() * state["k_scale"][blk[chosen], h].double()[:, None, None]).reshape(-1, width)[keep]
            v = (state["v"][blk[chosen], h].double() * state["v_scale"][blk[chosen], h].double()[:, None, None]).reshape(-1, width)[keep]
            if len(k):
                score = state["q"][r, h * group:(h + 1) * group].double() @ k.T / math.sqrt(width)
                out[r, h * group:(h + 1) * group] = torch.softmax(score, -1) @ v
    return out


def _exact_append(state, table, per):
    c = state["case"]
    heads, kv_heads, width, block = c["heads"], c["kv_heads"], c["width"], c["block"]
    x = state["qkv"].double().reshape(-1, heads + 2 * kv_heads, width)
    half = width // 2
    turn = torch.polar(torch.ones((), dtype=torch.float64, device="cuda"), torch.outer(state["positions"].double(), state["inv_freq"].double()))[:, None]
    parts = []
    for t, gain in ((x[:, :heads], state["q_norm"]), (x[:, heads:heads + kv_heads], state["k_norm"])):
        if gain is not None:
            t = t / (t.pow(2).mean(-1, keepdim=True) + 1e-6).sqrt() * gain.double()
        z = torch.complex(t[..., :half], t[..., half:]) * turn
        parts.append(torch.cat([z.real, z.imag], -1))
    q, new = parts[0], {"k": parts[1], "v": x[:, heads + kv_heads:]}
    where = {}
    for r, (s, p) in enumerate(zip(state["slots"].tolist(), state["positions"].tolist())):
        j = p // block
        where.setdefault(table[s][j // per] * per + j % per, []).append((r, p % block))
    codes = {n: state[n].clone() for n in "kv"}
    scales = {n: state[n + "_scale"].double() for n in "kv"}
    bounds = state["bounds"].double()
    for b, rows in where.items():
        r, at = [a for a, _ in rows], [i for _, i in rows]
        starts = 0 in at
        held = [i for i in range(block) if i not in set(at)]
        for n in "kv":
            t = new[n][r]
            old = torch.zeros(kv_heads, dtype=torch.float64, device="cuda") if starts else scales[n][b]
            grown = torch.maximum(old, (t.abs().amax((0, 2)) / 127).clamp_min(FLOOR))
            if not starts:
                follow = old / grown
                codes[n][b][:, held] = torch.round(codes[n][b][:, held].double() * follow[:, None, None]).to(torch.int8)
            fresh = torch.round(t / grown[:, None]).clamp(-127, 127)
            codes[n][b][:, at] = fresh.transpose(0, 1).to(torch.int8)
            scales[n][b] = grown
            if n == "k":
                low, high = fresh.amin(0), fresh.amax(0)
                if not starts:
                    low = torch.minimum(low, torch.round(bounds[b][:, 0] * follow[:, None]))
                    high = torch.maximum(high, torch.round(bounds[b][:, 1] * follow[:, None]))
                bounds[b] = torch.stack([low, high], 1)
    return q, scales, codes, bounds
