"""Plain 64-bit statements of the operators over 8-bit kept rows, one loop at a time, for the tests."""
import numpy as np

FLOOR = 2.0 ** -60
LARGEST = 255 * 2.0 ** 120  # of the finite bf16 values
SPARE = 0xFFFFFFFF


def to_code(x):
    x = np.where(np.isnan(x), 0.0, x)
    return np.clip(np.rint(x), -127, 127)


class Store:
    """The pool in 64 bits: codes [blocks, kv_heads, block, width], scales, bounds, and the walk to a block."""

    def __init__(self, kv, layout, scalar, page=None, table=None):
        f = lambda t: t.detach().cpu().numpy().astype(np.float64)  # noqa: E731
        self.codes = {"k": f(kv.k), "v": f(kv.v)}
        self.scale = {"k": f(kv.k_scale), "v": f(kv.v_scale)}
        self.bounds = f(kv.k_bounds) if kv.k_bounds is not None else None
        self.blocks, self.kv_heads, self.block, self.width = self.codes["k"].shape
        self.layout, self.scalar, self.page, self.table = layout, scalar, page, table

    def at(self, slot, b):
        """The pool's block with block b of a slot, or None outside it."""
        if self.layout == "dense":
            per = self.scalar // self.block
            if b >= per:
                return None
            blk = slot * per + b
        else:
            per = self.page // self.block
            entry = slot * self.scalar + b // per
            if b // per >= self.scalar or entry >= len(self.table):
                return None
            blk = int(self.table[entry]) * per + b % per
        return blk if blk < self.blocks else None

    def keys_of(self, slot, head, positions):
        """(k, v) in f64 at positions of a slot; positions outside the pool are left out."""
        positions = np.asarray(list(positions), np.int64)
        where = {b: self.at(slot, int(b)) for b in np.unique(positions // self.block)}
        blk = np.array([-1 if where[b] is None else where[b] for b in positions // self.block], np.int64)
        i, blk = positions[blk >= 0] % self.block, blk[blk >= 0]
        return tuple(self.codes[n][blk, head, i].reshape(-1, self.width) * self.scale[n][blk, head].reshape(-1, 1) for n in "kv")


def prepared(qkv, q_norm, k_norm, inv_freq, positions, heads, kv_heads, width, eps):
    """(q, k, v) f64 after norm and rotation."""
    x = qkv.astype(np.float64).reshape(len(positions), heads + 2 * kv_heads, width)
    angle = np.asarray(positions, np.float64)[:, None] * inv_freq.astype(np.float64)
    cos, sin = np.cos(angle)[:, None], np.sin(angle)[:, None]

    def turned(t, gain):
        if gain is not None:
            t = t / np.sqrt((t ** 2).mean(-1, keepdims=True) + eps) * gain
        a, b = t[..., :width // 2], t[..., width // 2:]
        return np.concatenate([a * cos - b * sin, a * sin + b * cos], -1)

    return turned(x[:, :heads], q_norm), turned(x[:, heads:heads + kv_heads], k_norm), x[:, heads + kv_heads:]


def append(store, k, v, slots, positions):
    """Writes k, v [rows, kv_heads, width] f64 into the store.  Returns, like the codes, the values before rounding."""
    raw = {n: store.codes[n].copy() for n in "kv"}
    runs = {}
    for r, (s, p) in enumerate(zip(slots, positions)):
        blk = store.at(int(s), int(p) // store.block)
        if blk is not None:
            runs.setdefault(blk, {})[int(p) % store.block] = r  # the last row of a position counts
    for blk, rows in runs.items():
        at, src = list(rows), list(rows.values())
        fresh = 0 in rows
        held = [i for i in range(store.block) if i not in rows]
        for n, x in (("k", k), ("v", v)):
            for h in range(store.kv_heads):
                t = x[src, h]
                a = min(np.abs(np.where(np.isnan(t), 0.0, t)).max(), LARGEST)
                old = 0.0 if fresh else store.scale[n][blk, h]
                new = max(old, a / 127, FLOOR)
                with np.errstate(invalid="ignore"):
                    raw[n][blk, h, at] = np.clip(np.where(np.isnan(t), 0.0, t) / new, -127, 127)
                ratio = 1.0 if fresh else old / new
                if not fresh:
                    raw[n][blk, h, held] = store.codes[n][blk, h, held] * ratio
                codes = to_code(raw[n][blk, h])
                written = codes[at]
                store.codes[n][blk, h] = codes
                store.scale[n][blk, h] = new
                if n == "k" and store.bounds is not None:
                    low, high = written.min(0), written.max(0)
                    if not fresh:
                        low = np.minimum(low, to_code(store.bounds[blk, h, 0] * ratio))
                        high = np.maximum(high, to_code(store.bounds[blk, h, 1] * ratio))
                    store.bounds[blk, h] = np.stack([low, high])
    return raw


def attend_keys(store, q, slot, head, positions, scale):
    """q [group, width] over the given positions: (out, sum of p |v|, largest |v|, keys), zeros where there are none."""
    k, v = store.keys_of(slot, head, positions)
    if len(k) == 0:
        z = np.zeros((q.shape[0], store.width))
        return z, z, 0.0, 0
    s = q @ k.T * scale
    p = np.exp(s - s.max(-1, keepdims=True))
    p /= p.sum(-1, keepdims=True)
    return p @ v, p @ np.abs(v), np.abs(v).max(), len(k)


def attend(store, q, slots, positions, keys, scale, back=0xFFFFFFFF, ids=None):
    """(out, tolerance) [rows, heads, width].  The tolerance: half a step of bf16 (2^-8 of the value); probabilities in
    f16, half a step 2^-11, or 2^-25 of the largest where they are subnormal; scores in f32, 256 terms of at most 15 in
    all (in powers of two) off by 256 * 2^-24 each way, 2^-11 of every probability and of their sum together."""
    rows, heads, width = q.shape
    group = heads // store.kv_heads
    out, tol = np.zeros(q.shape), np.zeros(q.shape)
    for r in range(rows):
        pos = int(positions[r])
        last = min(pos, keys - 1)
        for h in range(store.kv_heads):
            if ids is None:
                span = range(max(0, pos - back), last + 1)
            else:
                span = [p for b in ids[r, h] for p in range(int(b) * store.block, min(int(b) * store.block + store.block, last + 1))]
            g = slice(h * group, (h + 1) * group)
            o, a, top, n = attend_keys(store, q[r, g].astype(np.float64), int(slots[r]), h, span, scale)
            out[r, g] = o
            tol[r, g] = 2.0 ** -8 * np.abs(o) + 2.0 ** -10 * a + n * 2.0 ** -25 * top
    return out, tol


def select(store, q, slots, positions, keys, count, first, recent):
    """ids u32 [rows, kv_heads, count]."""
    rows, heads, width = q.shape
    group = heads // store.kv_heads
    ids = np.full((rows, store.kv_heads, count), SPARE, np.uint32)
    for r in range(rows):
        n = min(int(positions[r]), keys - 1) // store.block + 1
        for h in range(store.kv_heads):
            if n <= count:
                ids[r, h, :n] = np.arange(n)
                continue
            x = q[r, h * group:(h + 1) * group].astype(np.float64)
            top = np.abs(x).max()
            c = np.rint(x * 127 / top) if top > 0 else np.zeros_like(x)
            up, down = np.maximum(c, 0).sum(0), np.minimum(c, 0).sum(0)
            best = []
            for b in range(n):
                if b < first or b >= n - recent:
                    best.append((-np.inf, b))
                    continue
                blk = store.at(int(slots[r]), b)
                if blk is None:
                    best.append((np.inf, b))
                    continue
                total = np.float32((up * store.bounds[blk, h, 1] + down * store.bounds[blk, h, 0]).sum())
                best.append((-float(total * np.float32(store.scale["k"][blk, h])), b))
            ids[r, h] = sorted(b for _, b in sorted(best)[:count])
    return ids
