"""Plain 64-bit restatement of the paged int8 KV cache's operators
(nnhip_block_tables, nnhip_rope_kv_append_paged_q8, nnhip_attention_paged_q8,
nnhip_kv_read_paged_q8), request by request, in numpy."""
import math

import numpy as np


class Tables:
    """Block tables over a stack of free blocks."""

    def __init__(self, batch, max_blocks, num_blocks, bs, rng=None):
        self.bs, self.max_blocks, self.num_blocks = bs, max_blocks, num_blocks
        ids = np.arange(num_blocks, dtype=np.int32)
        if rng is not None:
            rng.shuffle(ids)
        self.free = ids.copy()
        self.count = num_blocks
        self.tables = np.full((batch, max_blocks), -7, np.int32)
        self.held = np.zeros(batch, np.int32)

    def status(self, cached, added, T):
        cached, added = cached.astype(np.int64), added.astype(np.int64)
        if (cached < 0).any() or (added < 0).any():
            return 1
        if (cached + added > self.max_blocks * self.bs).any():
            return 2
        if added.sum() > T:
            return 3
        need = -(-(cached + added) // self.bs)
        back = np.maximum(self.held - need, 0).sum()
        if (self.held < 0).any() or (self.held > self.max_blocks).any() or self.count < 0 or \
                self.count + back > self.num_blocks:
            return 5
        return 4 if np.maximum(need - self.held, 0).sum() > self.count + back else 0

    def step(self, cached, added, T):
        """(status, row_start, lens, pos, slots); the state is updated."""
        B = len(cached)
        pos, slots = np.full(T, -1, np.int32), np.full(T, -1, np.int32)
        st = self.status(cached, added, T)
        if st:
            return st, np.zeros(B + 1, np.int32), np.zeros(B, np.int32), pos, slots
        need = -(-(cached.astype(np.int64) + added) // self.bs)
        stack = list(self.free[:self.count])
        # the first request's first block ends uppermost
        for b in reversed(range(B)):
            for j in reversed(range(need[b], self.held[b])):
                stack.append(self.tables[b, j])
        for b in range(B):
            for j in range(self.held[b], need[b]):
                self.tables[b, j] = stack.pop()
        self.count = len(stack)
        self.free[:self.count] = stack
        self.held[:] = need
        start = np.concatenate(([0], np.cumsum(added))).astype(np.int32)
        for b in range(B):
            p = cached[b] + np.arange(added[b])
            pos[start[b]:start[b + 1]] = p
            slots[start[b]:start[b + 1]] = self.tables[b, p // self.bs] * self.bs + p % self.bs
        return 0, start, (cached + added).astype(np.int32), pos, slots


def grids(codes, Hkv, D, bs):
    """codes [blocks][2][Hkv][bs * D] as views k, v [blocks][Hkv][bs][D]."""
    k = codes[:, 0].reshape(-1, Hkv, bs, D)
    v = codes[:, 1].reshape(-1, Hkv, D, bs).swapaxes(2, 3)
    return k, v


def block_scale(amax):
    """The smallest 2^e, e >= -126, with amax <= 127 * 2^e; 0 for 0."""
    if amax == 0:
        return 0.0
    m, x = math.frexp(amax)                       # amax = m * 2^x, m in [1/2, 1)
    return 2.0 ** max(x - 7 + (m * 128 > 127), -126)


def rope(x, cos, sin):
    """x [rows][heads][D] with cos, sin [rows][D / 2], in 64 bits."""
    e, o = x[..., 0::2], x[..., 1::2]
    c, s = cos[:, None], sin[:, None]
    return np.stack((e * c - o * s, e * s + o * c), -1).reshape(x.shape)


def append(qkv, pos, slots, cos, sin, H, codes, scales, D, bs, q_out):
    """Updates codes, scales and q_out (float64 rows) in place."""
    n_blocks, _, Hkv, _ = codes.shape
    f8 = np.float64
    x = qkv.astype(f8).reshape(len(qkv), H + 2 * Hkv, D)
    ok = (slots >= 0) & (slots < n_blocks * bs) & (pos >= 0) & (pos < len(cos))
    at = np.where(ok, pos, 0)
    with np.errstate(invalid="ignore"):
        rot = rope(x[:, :H + Hkv], cos[at].astype(f8), sin[at].astype(f8))
    q_out[ok] = rot[ok, :H].reshape(-1, H * D)
    grid = grids(codes, Hkv, D, bs)               # views of codes
    new = (rot[:, H:], x[:, H + Hkv:])
    taken = np.zeros(len(slots), bool)
    for t in range(len(slots)):
        if not ok[t] or taken[t]:
            continue
        # the block's rows: within bs rows of the first, the last one of a slot
        blk = int(slots[t]) // bs
        group = [r for r in range(t, min(t + bs, len(slots))) if ok[r] and slots[r] // bs == blk]
        taken[group] = True
        row = {int(slots[r]) % bs: r for r in group}
        toks = sorted(row)
        pick = [row[o] for o in toks]
        off = toks[0]
        for i in range(2):
            for h in range(Hkv):
                rows = new[i][pick, h]
                old = float(scales[blk, i, h]) if off else 0.0
                cells = grid[i][blk, h]
                if not np.isfinite(rows).all() or not np.isfinite(old):
                    scales[blk, i, h] = np.nan
                    cells[toks] = 0
                    continue
                now = max(old, block_scale(np.abs(rows).max()))
                if now > old:
                    cells[:off] = np.rint(cells[:off] * (old / now))
                cells[toks] = np.rint(rows / now) if now else 0
                scales[blk, i, h] = now


def read(codes, scales, slots, D, bs):
    Hkv = codes.shape[2]
    k, v = grids(codes, Hkv, D, bs)
    blk, off = slots // bs, slots % bs
    return (k[blk, :, off].astype(np.float64) * scales[blk, 0][..., None].astype(np.float64),
            v[blk, :, off].astype(np.float64) * scales[blk, 1][..., None].astype(np.float64))


def attention(q, codes, scales, tables, row_start, lens, H, D, bs, out):
    """out (float64 rows) and its allowed error are filled per request;
    returns the error bound, as large as out.

    Bound: with u = 2^-24 a score of D products of fp32-accurate factors is
    off by at most (D + 16) u sum|q k| / sqrt(D) (a q carried as two 11-bit
    halves is within 4 u of itself; 12 u more cover the scalings and the
    conversion of the exponent's argument), so a weight relative to another by
    2 max|ds| + 8 u (exponential, split into two halves, block scale), and sums
    of n terms by n u more, in the numerator and in the denominator:
    |d out| <= (2 (2 max|ds| + 8 u) + 2 (n + 8) u) sum p|v|.
    Underflow adds, for each of the n terms: a weight below 2^-126 that is lost
    (2^-126 max|v|, the denominator being at least 1), a product below 2^-126
    that is lost (2^-126), and, where weights times block scales are carried as
    two halves of at most 2^14 for the largest of them, half a step of the
    smallest half, 2^-25 / 2^14 of that largest, times a code of at most 128:
    n (2^-126 (1 + max|v|) + 2^-39 128 max(p vs))."""
    n_blocks, _, Hkv, _ = codes.shape
    T = len(q)
    u = 2.0 ** -24
    bound = np.zeros_like(out)
    k, v = grids(codes, Hkv, D, bs)
    for b in range(len(lens)):
        a, z = (int(np.clip(row_start[i], 0, T)) for i in (b, b + 1))
        n = max(z - a, 0)
        total = int(np.clip(lens[b], 0, tables.shape[1] * bs))
        see0 = total - n + 1                       # tokens the first row sees
        if n == 0:
            continue
        if total == 0:
            out[a:z] = 0
            continue
        ids = tables[b, :-(-total // bs)].astype(np.int64)
        bad = (ids < 0) | (ids >= n_blocks)
        ids = np.where(bad, 0, ids)
        bad = np.repeat(bad, bs)[:total]
        for h in range(H):
            hk = h // (H // Hkv)
            ks = np.repeat(scales[ids, 0, hk].astype(np.float64), bs)[:total]
            vs = np.repeat(scales[ids, 1, hk].astype(np.float64), bs)[:total]
            kk = k[ids, hk].reshape(-1, D)[:total].astype(np.float64) * ks[:, None]
            vv = v[ids, hk].reshape(-1, D)[:total].astype(np.float64) * vs[:, None]
            for i in range(n):
                m = see0 + i
                sl = np.s_[(a + i), h * D:(h + 1) * D]
                if m <= 0:
                    out[sl] = 0
                    continue
                if bad[:m].any() or not np.isfinite(kk[:m]).all() or not np.isfinite(vv[:m]).all():
                    out[sl] = np.nan
                    continue
                x = q[sl].astype(np.float64)
                s = kk[:m] @ x / math.sqrt(D)
                p = np.exp(s - s.max())
                p /= p.sum()
                out[sl] = p @ vv[:m]
                ds = (D + 16) * u * (np.abs(kk[:m]) @ np.abs(x)).max() / math.sqrt(D)
                bound[sl] = (2 * (2 * ds + 8 * u) + 2 * (m + 8) * u) * (p @ np.abs(vv[:m])) + \
                    m * (2.0 ** -126 * (1 + np.abs(vv[:m]).max()) +
                         2.0 ** -39 * 128 * (p * vs[:m]).max())
    return bound
