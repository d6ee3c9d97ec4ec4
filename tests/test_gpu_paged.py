"""The paged int8 KV cache on the GPU against its 64-bit restatement
(paged_ref.py).  Tables, slots, codes and scales are whole or exact and have to
be equal; q, read rows and attention go by their roundings."""
import ctypes as C

import numpy as np
import pytest

import paged_ref as R
from gpu_util import nnhip

pytestmark = pytest.mark.gpu

U = 2.0 ** -24          # half a step of fp32
I32 = 2 ** 31 - 1


def i32(x):
    return np.ascontiguousarray(x, np.int32)


# ----------------------------------------------------------- block tables ----
class Dev:
    """The device's state beside a R.Tables."""

    def __init__(self, ctx, ref, T):
        self.ctx, self.ref = ctx, ref
        B = len(ref.held)
        self.tables, self.held = ctx.array(ref.tables), ctx.array(ref.held)
        self.free, self.count = ctx.array(ref.free), ctx.array(i32([ref.count]))
        self.row_start, self.lens = (ctx.array(np.full(n, 9, np.int32)) for n in (B + 1, B))
        self.pos, self.slots = (ctx.array(np.full(max(T, 1), 9, np.int32)) for _ in range(2))
        self.status = ctx.array(i32([77]))

    def call(self, cached, added, T):
        r = self.ref
        c, a = self.ctx.array(i32(cached)), self.ctx.array(i32(added))
        nnhip.call("nnhip_block_tables", self.ctx.h, len(r.held), c.p, a.p, r.bs, r.max_blocks,
                   self.tables.p, self.held.p, r.num_blocks, self.free.p, self.count.p, T,
                   self.row_start.p, self.lens.p, self.pos.p, self.slots.p, self.status.p)
        got = (int(self.status.numpy()[0]), self.row_start.numpy(), self.lens.numpy(),
               self.pos.numpy()[:T], self.slots.numpy()[:T])
        del c, a
        return got

    def state(self):
        return (self.tables.numpy(), self.held.numpy(), self.free.numpy(),
                int(self.count.numpy()[0]))


def same_step(dev, cached, added, T):
    want = dev.ref.step(i32(cached), i32(added), T)
    got = dev.call(cached, added, T)
    for w, g, name in zip(want, got, ("status", "row_start", "lens", "pos", "slots")):
        assert np.array_equal(w, g), name
    r = dev.ref
    for w, g, name in zip((r.tables, r.held, r.free, r.count), dev.state(),
                          ("tables", "held", "free_list", "free_count")):
        assert np.array_equal(w, g), name
    return want[0]


@pytest.mark.parametrize("B,most,bs,steps", [(1, 40, 16, 12), (3, 200, 32, 12), (70, 90, 64, 8),
                                             (1025, 20, 16, 5), (4096, 9, 128, 4),
                                             (64, 700, 16, 4)])
def test_tables_over_steps(ctx, B, most, bs, steps):
    """Requests grow, are cut back, end and begin anew."""
    rng = np.random.default_rng(B)
    mb = 3 * most // bs + 2
    pool = B * mb * 2 // 3 + 2
    room = B * most + 5
    dev = Dev(ctx, R.Tables(B, mb, pool, bs, rng), room)
    lens = np.zeros(B, np.int64)
    seen = set()
    for _ in range(steps):
        cached = np.where(rng.random(B) < 0.3, rng.integers(0, lens + 1), lens)
        cached[rng.random(B) < 0.1] = 0
        added = np.where(rng.random(B) < 0.2, 0, rng.integers(0, most + 1, B))
        st = same_step(dev, cached, added, room)
        seen.add(st)
        if st == 0:
            lens = cached + added
        else:                                      # some requests end, then on
            lens[rng.random(B) < 0.5] = 0
            assert same_step(dev, lens, np.zeros(B), 0) == 0
    assert 0 in seen


@pytest.mark.parametrize("want,cached,added,held,count,T", [
    (1, [-1, 0, 3], [1, 1, 1], [0, 0, 1], 5, 8), (1, [0, 0, 0], [1, -5, 1], [0, 0, 0], 5, 8),
    (2, [60, 0, 0], [5, 1, 0], [4, 0, 0], 5, 8), (2, [I32, 0, 0], [I32, 0, 0], [4, 0, 0], 5, 8),
    (3, [0, 0, 0], [5, 4, 0], [0, 0, 0], 5, 8), (4, [0, 0, 0], [20, 20, 20], [0, 0, 0], 5, 60),
    (5, [0, 0, 0], [1, 1, 1], [-1, 0, 0], 5, 8), (5, [0, 0, 0], [1, 1, 1], [9, 0, 0], 5, 8),
    (5, [0, 0, 0], [1, 1, 1], [0, 0, 0], -2, 8), (5, [0, 0, 0], [0, 0, 0], [4, 0, 0], 7, 8)])
def test_a_step_that_cannot_be_leaves_all_as_it_was(ctx, want, cached, added, held, count, T):
    ref = R.Tables(3, 4, 10, 16, np.random.default_rng(1))
    ref.held[:], ref.count = held, count
    dev = Dev(ctx, ref, T)
    assert same_step(dev, cached, added, T) == want
    # and the next good step runs
    fine = Dev(ctx, R.Tables(3, 4, 10, 16), 8)
    assert same_step(fine, [0, 0, 0], [3, 0, 5], 8) == 0


def test_a_free_list_with_a_block_outside_the_pool_gives_no_slot(ctx):
    ref = R.Tables(2, 4, 6, 16)
    ref.free[:] = [0, 1, 2, 3, 99, -4]
    dev = Dev(ctx, ref, 40)
    st, _, _, pos, slots = dev.call([0, 0], [20, 3], 40)
    assert st == 0
    # -4 and 99 go to request 0, block 3 to request 1
    assert (slots[:20] == -1).all() and (slots[20:23] == 48 + np.arange(3)).all()
    assert (slots[23:] == -1).all() and (pos[23:] == -1).all()


def test_two_contexts_take_turns(ctx):
    with nnhip.Context(0) as other:
        devs = [Dev(c, R.Tables(5, 6, 30, 16, np.random.default_rng(i)), 400)
                for i, c in enumerate((ctx, other))]
        for n in (3, 17, 40, 2):
            for d in devs:
                assert same_step(d, [0] * 5, [n, 0, n + 1, 2 * n, 1], 400) == 0


# ------------------------------------------------------------------ append ----
def angles(n, D):
    w = np.arange(n)[:, None] * 10000.0 ** (-np.arange(0, D, 2) / D)
    return np.cos(w).astype(np.float32), np.sin(w).astype(np.float32)


class Cache:
    """A pool with its host twin."""

    def __init__(self, ctx, blocks, Hkv, D, bs, rng, empty=False):
        self.ctx, self.blocks, self.Hkv, self.D, self.bs = ctx, blocks, Hkv, D, bs
        self.codes = rng.integers(-127, 128, (blocks, 2, Hkv, bs * D)).astype(np.int8)
        self.scales = np.float32(2.0) ** rng.integers(-9, -3, (blocks, 2, Hkv)).astype(np.float32)
        if empty:
            self.codes[:], self.scales[:] = 0, 0
        self.dc, self.ds = ctx.array(self.codes), ctx.array(self.scales)

    def append(self, qkv, pos, slots, H, cos, sin, tables=True):
        """Both sides append; (device's q, the twin's q)."""
        T = len(pos)
        q = np.full((T, H * self.D), 7.0)
        want = q.copy()
        R.append(qkv, pos, slots, cos, sin, H, self.codes, self.scales, self.D, self.bs, want)
        a = [self.ctx.array(x) for x in (qkv, i32(pos), i32(slots), q.astype(np.float32))]
        t = [self.ctx.array(x) for x in (cos, sin)] if tables else [None, None]
        nnhip.call("nnhip_rope_kv_append_paged_q8", self.ctx.h, a[0].p, T, H, self.Hkv, self.D,
                   a[1].p, a[2].p, t[0] and t[0].p, t[1] and t[1].p, len(cos), a[3].p, self.dc.p,
                   self.ds.p, self.bs, self.blocks)
        return a[3].numpy(), want

    def assert_same(self):
        assert np.array_equal(self.ds.numpy(), self.scales, equal_nan=True), "scales"
        assert np.array_equal(self.dc.numpy(), self.codes), "codes"


def q_close(got, want):
    """One rounding of a value formed in 64 bits."""
    assert np.array_equal(np.isnan(got), np.isnan(want))
    ok = ~np.isnan(want)
    assert (np.abs(got[ok] - want[ok]) <= U * np.abs(want[ok]) + 2.0 ** -149).all()


def rows_of(lists, bs):
    """(pos, slots) of [(blocks, start, count)] requests."""
    pos, slots = [], []
    for ids, start, n in lists:
        p = start + np.arange(n)
        pos.append(p)
        slots.append(np.asarray(ids, np.int64)[p // bs] * bs + p % bs)
    return np.concatenate(pos), np.concatenate(slots)


@pytest.mark.parametrize("D", [32, 64, 128])
@pytest.mark.parametrize("bs", [16, 32, 64, 128])
@pytest.mark.parametrize("H,Hkv", [(1, 1), (6, 2), (5, 5), (16, 1)])
def test_append(ctx, D, bs, H, Hkv):
    rng = np.random.default_rng(D + bs + H)
    c = Cache(ctx, 30, Hkv, D, bs, rng)
    ids = rng.permutation(30)
    # a prompt over several blocks, one that ends with a block, one token at
    # the start of a block, within and at its end, a chunk that goes on
    pos, slots = rows_of([(ids[:4], 0, 3 * bs + 5), (ids[4:6], 0, 2 * bs), (ids[6:7], 0, 1),
                          (ids[7:8], 5, 1), (ids[8:9], bs - 1, 1), (ids[9:12], bs - 3, bs + 7),
                          (ids[12:14], 7, 6)], bs)
    qkv = rng.standard_normal((len(pos), (H + 2 * Hkv) * D)).astype(np.float32)
    qkv *= np.exp2(rng.integers(-3, 4, (len(pos), 1))).astype(np.float32)
    cos, sin = angles(4 * bs + 1, D)
    q_close(*c.append(qkv, pos, slots, H, cos, sin))
    c.assert_same()


def test_append_many_rows(ctx):
    """More rows than one at a time are dealt out: runs of every length."""
    rng = np.random.default_rng(9)
    D, bs, H, Hkv = 64, 16, 4, 2
    n = rng.integers(1, 90, 300)
    blocks = -(-n // bs)
    ids = rng.permutation(int(blocks.sum()))
    lists, at = [], 0
    for k, m in zip(blocks, n):
        start = int(rng.integers(0, m))
        lists.append((ids[at:at + k], start, int(m - start)))
        at += k
    pos, slots = rows_of(lists, bs)
    slots[rng.random(len(slots)) < 0.02] = -1
    c = Cache(ctx, len(ids), Hkv, D, bs, rng)
    qkv = rng.standard_normal((len(pos), (H + 2 * Hkv) * D)).astype(np.float32)
    cos, sin = angles(100, D)
    q_close(*c.append(qkv, pos, slots, H, cos, sin))
    c.assert_same()


@pytest.mark.parametrize("bs,D", [(16, 64), (64, 128), (32, 32)])
def test_append_token_by_token(ctx, bs, D):
    """A block that is filled in single steps, by growing values: its scale
    grows and the older codes with it, as in the restatement."""
    rng = np.random.default_rng(bs)
    c = Cache(ctx, 3, 2, D, bs, rng)
    cos, sin = angles(2 * bs, D)
    for p in range(bs + 3):
        pos, slots = rows_of([([2, 0], p, 1)], bs)
        qkv = rng.standard_normal((1, 6 * D)).astype(np.float32) * np.float32(1.3 ** p)
        if p in (1, 5):
            qkv[:] = 0
        q_close(*c.append(qkv, pos, slots, 2, cos, sin))
        c.assert_same()


def test_append_rows_of_a_block_in_any_order(ctx):
    """Out of order, with rows between them, the same slot twice (the last row
    counts), and a first row that is not the block's first token."""
    rng = np.random.default_rng(3)
    D, bs, H, Hkv = 64, 32, 2, 2
    c = Cache(ctx, 6, Hkv, D, bs, rng)
    cos, sin = angles(70, D)
    slots = np.r_[40, 3, 41, 2, 39, 3, 100, 64 + rng.permutation(32), 45, 44, 44]
    qkv = rng.standard_normal((len(slots), (H + 2 * Hkv) * D)).astype(np.float32)
    slots[-3:] += 128
    q_close(*c.append(qkv, slots % 70, slots, H, cos, sin))
    c.assert_same()


def test_append_skips_what_is_outside(ctx):
    rng = np.random.default_rng(4)
    D, bs, H, Hkv = 64, 16, 4, 2
    c = Cache(ctx, 4, Hkv, D, bs, rng)
    cos, sin = angles(20, D)
    #       padding, outside, good run cut by a bad position, last slot, first
    slots = np.array([-1, 64, I32, -I32 - 1, 3, 4, 5, 6, 63, 16, 17, 18])
    pos = np.array([0, 0, 0, 0, 3, 20, 5, -1, 15, 0, 1, 19])
    qkv = rng.standard_normal((12, (H + 2 * Hkv) * D)).astype(np.float32)
    got, want = c.append(qkv, pos, slots, H, cos, sin)
    q_close(got, want)
    assert (got[[0, 1, 2, 3, 5, 7]] == 7).all()
    c.assert_same()


@pytest.mark.parametrize("value", [0.0, -0.0, 1e-45, -1e-40, 2.0 ** -126, 3.4e38, -3.4e38, np.nan,
                                   np.inf, -np.inf])
def test_append_extreme_values(ctx, value):
    rng = np.random.default_rng(5)
    D, bs = 64, 16
    c = Cache(ctx, 3, 1, D, bs, rng)
    cos, sin = angles(40, D)
    qkv = rng.standard_normal((7, 3 * D)).astype(np.float32)
    qkv[2, D:] = value                             # k and v of one row
    if value == 0:
        qkv[:] = value
    # a new block, and one that goes on; then both start anew
    pos, slots = rows_of([([1], 0, 4), ([0], 4, 3)], bs)
    with np.errstate(over="ignore"):
        c.append(qkv, pos, slots, 1, cos, sin)
    c.assert_same()
    qkv = rng.standard_normal((7, 3 * D)).astype(np.float32)
    pos, slots = rows_of([([1], 4, 4), ([0], 0, 3)], bs)
    c.append(qkv, pos, slots, 1, cos, sin)
    c.assert_same()


def test_append_with_the_references_angles(ctx):
    """Without tables, q is what nnhip_rope_kv_append_gqa rotates: that one
    rounds two products and their sum, so up to 2 u (|x0| + |x1|) off."""
    rng = np.random.default_rng(6)
    D, bs, H, Hkv, S = 64, 16, 4, 2, 40
    c = Cache(ctx, 4, Hkv, D, bs, rng)
    pos, slots = rows_of([([3, 1, 2], 0, S)], bs)
    qkv = rng.standard_normal((S, (H + 2 * Hkv) * D)).astype(np.float32)
    cos, sin = angles(64, D)
    got, _ = c.append(qkv, pos, slots, H, cos, sin, tables=False)
    x, z = ctx.array(qkv), ctx.array(i32([0]))
    q, k, v = (ctx.array(np.zeros(s, np.float32)) for s in
               ((S, H * D), (Hkv, 64, D), (Hkv, 64, D)))
    nnhip.call("nnhip_rope_kv_append_gqa", ctx.h, x.p, 1, S, H, Hkv, D, z.p, q.p, k.p, v.p, 64)
    pair = np.abs(qkv[:, :H * D]).reshape(S, -1, 2).sum(-1).repeat(2, -1)
    assert (np.abs(got - q.numpy()) <= 3 * U * pair).all()


def test_append_of_nothing(ctx):
    c = Cache(ctx, 4, 1, 32, 16, np.random.default_rng(1))
    nnhip.call("nnhip_rope_kv_append_paged_q8", ctx.h, None, 0, 1, 1, 32, None, None, None, None, 8,
               None, c.dc.p, c.ds.p, 16, 4)
    nnhip.call("nnhip_kv_read_paged_q8", ctx.h, c.dc.p, c.ds.p, 16, 4, None, 0, 1, 32, None, None)
    t = ctx.array(i32([[0]]))
    nnhip.call("nnhip_attention_paged_q8", ctx.h, None, 0, c.dc.p, c.ds.p, 16, 4, t.p, 1, t.p, t.p,
               1, 1, 1, 32, None)
    c.assert_same()


# -------------------------------------------------------------------- read ----
@pytest.mark.parametrize("D,bs,Hkv", [(32, 16, 3), (64, 16, 2), (64, 64, 1), (128, 32, 4),
                                      (128, 128, 2)])
def test_read(ctx, D, bs, Hkv):
    rng = np.random.default_rng(D + bs)
    c = Cache(ctx, 7, Hkv, D, bs, rng)
    c.scales *= 1.3                                # any scale, not a power of two
    c.ds.upload(c.scales)
    n = 7 * bs
    for slots in (np.arange(n), rng.permutation(n)[:n // 2], np.array([n - 1]),
                  np.arange(3, n - 2), np.r_[np.arange(5, 40) % n, 5, 5, 6, np.arange(bs)]):
        a = ctx.array(i32(slots))
        k, v = (ctx.array(np.full((len(slots), Hkv, D), 5.0, np.float32)) for _ in range(2))
        nnhip.call("nnhip_kv_read_paged_q8", ctx.h, c.dc.p, c.ds.p, bs, 7, a.p, len(slots), Hkv, D,
                   k.p, v.p)
        for got, want in zip((k, v), R.read(c.codes, c.scales, slots, D, bs)):
            assert np.array_equal(got.numpy(), want.astype(np.float32))


def test_read_leaves_rows_outside_as_they_were(ctx):
    c = Cache(ctx, 2, 1, 64, 16, np.random.default_rng(1))
    slots = np.array([-1, 0, 32, 31, I32, -I32 - 1, 16])
    a = ctx.array(i32(slots))
    k, v = (ctx.array(np.full((7, 1, 64), 5.0, np.float32)) for _ in range(2))
    nnhip.call("nnhip_kv_read_paged_q8", ctx.h, c.dc.p, c.ds.p, 16, 2, a.p, 7, 1, 64, k.p, v.p)
    ok = [1, 3, 6]
    for got, want in zip((k.numpy(), v.numpy()), R.read(c.codes, c.scales, slots[ok], 64, 16)):
        assert np.array_equal(got[ok], want.astype(np.float32))
        assert (np.delete(got, ok, 0) == 5).all()


# --------------------------------------------------------------- attention ----
def attend(ctx, c, q, tables, row_start, lens, H):
    T = len(q)
    a = [ctx.array(x) for x in (q, i32(tables), i32(row_start), i32(lens))]
    out = ctx.array(np.full((T, H * c.D), 7.0, np.float32))
    nnhip.call("nnhip_attention_paged_q8", ctx.h, a[0].p, T, c.dc.p, c.ds.p, c.bs, c.blocks, a[1].p,
               tables.shape[1], a[2].p, a[3].p, len(lens), H, c.Hkv, c.D, out.p)
    return out.numpy()


def check_attention(ctx, c, q, tables, row_start, lens, H):
    want = np.full((len(q), H * c.D), 7.0)
    bound = R.attention(q, c.codes, c.scales, tables, row_start, lens, H, c.D, c.bs, want)
    got = attend(ctx, c, q, tables, row_start, lens, H)
    assert np.array_equal(np.isnan(got), np.isnan(want))
    d = np.where(np.isnan(want), 0, np.abs(got - want) - U * np.abs(want))
    assert (d <= bound).all(), f"off by {(d / np.maximum(bound, 1e-30)).max():.3g} bounds"
    return got


def batch(rng, lens, counts, bs, extra=1, blocks=None):
    """tables and row_start; unused entries of the tables are garbage."""
    need = [-(-n // bs) for n in lens]
    mb = max(max(need), 1) + extra
    blocks = blocks or sum(need) + 2
    ids = rng.permutation(blocks)
    tables = rng.integers(-I32, I32, (len(lens), mb))
    at = 0
    for b, k in enumerate(need):
        tables[b, :k] = ids[at:at + k]
        at += k
    return tables, np.concatenate(([0], np.cumsum(counts))), blocks


def run_attention(ctx, rng, lens, counts, H, Hkv, D, bs, pad=0, std=2.0):
    tables, start, blocks = batch(rng, lens, counts, bs)
    c = Cache(ctx, blocks, Hkv, D, bs, rng)
    q = (rng.standard_normal((start[-1] + pad, H * D)) * std).astype(np.float32)
    got = check_attention(ctx, c, q, tables, start, lens, H)
    assert (got[start[-1]:] == 7).all()
    return c, q, tables, start, got


@pytest.mark.parametrize("D", [32, 64, 128])
@pytest.mark.parametrize("bs", [16, 32, 64, 128])
@pytest.mark.parametrize("H,Hkv", [(1, 1), (6, 2), (5, 5), (32, 2), (17, 1)])
def test_attention_of_single_tokens(ctx, D, bs, H, Hkv):
    rng = np.random.default_rng(D * bs + H)
    lens = [1, 2, bs - 1, bs, bs + 1, 63, 64, 65, 300, 5]
    run_attention(ctx, rng, lens, [1] * len(lens), H, Hkv, D, bs, pad=2)


@pytest.mark.parametrize("D,bs,H,Hkv", [(32, 16, 8, 8), (64, 16, 16, 16), (64, 32, 8, 2),
                                        (128, 64, 4, 1), (128, 16, 6, 2)])
def test_attention_of_few_rows(ctx, D, bs, H, Hkv):
    """Verify steps: two to nine rows a request, some without any."""
    rng = np.random.default_rng(D + H)
    counts = [6, 0, 2, 9, 1, 3, 5, 0, 8, 7]
    lens = [6, 40, 130, 9, 1, 77, 333, 0, 64, 71]
    run_attention(ctx, rng, lens, counts, H, Hkv, D, bs, pad=3)


@pytest.mark.parametrize("D,bs,H,Hkv,counts,cached", [
    (64, 16, 4, 1, [257], [0]), (64, 16, 4, 2, [100, 33, 17], [0, 0, 0]),
    (64, 32, 2, 2, [130, 64, 1], [70, 0, 500]), (128, 16, 4, 2, [65, 128, 40], [0, 33, 200]),
    (32, 64, 3, 1, [200, 3, 90], [5, 64, 0]), (128, 128, 8, 1, [47, 31], [129, 0]),
    (64, 16, 16, 16, [90, 90], [0, 10])])
def test_attention_of_prompts(ctx, D, bs, H, Hkv, counts, cached):
    rng = np.random.default_rng(D + H)
    lens = [a + b for a, b in zip(counts, cached)]
    run_attention(ctx, rng, lens, counts, H, Hkv, D, bs, pad=1)


def test_attention_of_prompts_beside_single_tokens(ctx):
    rng = np.random.default_rng(8)
    counts = [1, 1, 150, 0, 1, 70, 2, 1]
    cached = [5, 700, 0, 9, 0, 300, 31, 64]
    lens = [a + b for a, b in zip(counts, cached)]
    run_attention(ctx, rng, lens, counts, 8, 2, 64, 16, pad=2)


@pytest.mark.parametrize("n", [2000, 9001])
def test_attention_of_one_long_request(ctx, n):
    """Keys split over workgroups and joined; beside short requests."""
    rng = np.random.default_rng(n)
    run_attention(ctx, rng, [n], [1], 4, 1, 64, 16)
    run_attention(ctx, rng, [3, n, 40], [1, 2, 0], 2, 2, 128, 64)


def test_attention_of_many_requests(ctx):
    rng = np.random.default_rng(12)
    lens = rng.integers(0, 60, 1500)
    counts = np.minimum(rng.integers(0, 3, 1500), lens)
    run_attention(ctx, rng, list(lens), list(counts), 2, 1, 32, 16)


def test_attention_rows_that_see_nothing_are_zero(ctx):
    """More rows than tokens, and requests without tokens."""
    rng = np.random.default_rng(13)
    lens, counts = [3, 0, 0, 20, 40], [5, 4, 0, 30, 41]
    _, _, _, _, got = run_attention(ctx, rng, lens, counts, 4, 2, 64, 16)
    assert (got[:2] == 0).all() and (got[5:9] == 0).all() and (got[9:19] == 0).all()


@pytest.mark.parametrize("counts", [[1, 1, 1], [3, 3, 3], [40, 33, 20]])
def test_attention_does_not_see_what_is_behind_the_tokens(ctx, counts):
    """Codes behind the last token, scales of blocks that no row sees and the
    table entries behind change nothing, to the bit."""
    rng = np.random.default_rng(14)
    D, bs, H, Hkv = 64, 16, 4, 2
    lens = [50, 64, 21]
    tables, start, blocks = batch(rng, lens, counts, bs, extra=3)
    c = Cache(ctx, blocks, Hkv, D, bs, rng)
    q = rng.standard_normal((start[-1], H * D)).astype(np.float32)
    first = check_attention(ctx, c, q, tables, start, lens, H)
    used = np.zeros(blocks, bool)
    k, v = R.grids(c.codes, Hkv, D, bs)
    for b, n in enumerate(lens):
        for j in range(-(-n // bs)):
            used[tables[b, j]] = True
            k[tables[b, j], :, max(n - j * bs, 0):] = 127
            v[tables[b, j], :, max(n - j * bs, 0):] = -127
        tables[b, -(-n // bs):] = rng.integers(0, blocks, tables.shape[1] + -n // bs)
    c.scales[~used] = np.nan
    c.codes[~used] = -128
    c.dc.upload(c.codes)
    c.ds.upload(c.scales)
    assert np.array_equal(first, attend(ctx, c, q, tables, start, lens, H))


@pytest.mark.parametrize("counts", [[2, 2], [60, 40]])
def test_attention_of_a_poisoned_block(ctx, counts):
    """A scale that is NaN reaches the rows that see its block, no others."""
    rng = np.random.default_rng(15)
    D, bs, H, Hkv = 64, 16, 4, 2
    lens = [70, 70]
    for i in range(2):
        tables, start, blocks = batch(rng, lens, counts, bs)
        c = Cache(ctx, blocks, Hkv, D, bs, rng)
        c.scales[tables[0, 3], i, 1] = np.nan      # tokens 48 .. 63, kv head 1
        c.ds.upload(c.scales)
        q = rng.standard_normal((start[-1], H * D)).astype(np.float32)
        got = check_attention(ctx, c, q, tables, start, lens, H)
        assert np.isnan(got[:counts[0], 2 * D:]).any() and not np.isnan(got[:, :2 * D]).any()


@pytest.mark.parametrize("counts", [[1, 1], [5, 5], [60, 40]])
@pytest.mark.parametrize("bad", [-1, I32, -I32 - 1])
def test_attention_of_a_table_entry_outside_the_pool(ctx, counts, bad):
    rng = np.random.default_rng(16)
    D, bs, H = 64, 16, 4
    lens = [90, 61]
    tables, start, blocks = batch(rng, lens, counts, bs)
    tables[0, 4] = blocks if bad == -1 else bad
    c = Cache(ctx, blocks, 2, D, bs, rng)
    q = rng.standard_normal((start[-1], H * D)).astype(np.float32)
    got = check_attention(ctx, c, q, tables, start, lens, H)
    assert np.isnan(got[counts[0] - 1]).all() and not np.isnan(got[counts[0]:]).any()


def test_attention_cuts_lengths_and_rows_to_the_buffers(ctx):
    rng = np.random.default_rng(17)
    c = Cache(ctx, 9, 2, 64, 16, rng)
    tables = rng.integers(0, 9, (3, 2))
    q = rng.standard_normal((6, 4 * 64)).astype(np.float32)
    for lens, start in (([I32, 33, -5], [0, 2, 4, 6]), ([5, 6, 7], [-9, 2, 4, I32]),
                        ([20, 20, 20], [4, 2, 6, 1])):
        check_attention(ctx, c, q, tables, start, lens, 4)


def test_attention_of_shared_blocks(ctx):
    """Requests with a common prefix, one of them twice the same."""
    rng = np.random.default_rng(18)
    c = Cache(ctx, 12, 2, 64, 16, rng)
    tables = np.array([[0, 1, 2, 3], [0, 1, 4, 5], [0, 1, 2, 3], [7, 7, 7, 7]])
    q = rng.standard_normal((9, 4 * 64)).astype(np.float32)
    q[6:8] = q[:2]
    got = check_attention(ctx, c, q, tables, [0, 2, 6, 8, 9], [60, 50, 60, 64], 4)
    assert np.array_equal(got[:2], got[6:8])


@pytest.mark.parametrize("scale", [1e-30, 1e30])
def test_attention_of_extreme_scales(ctx, scale):
    """v's scales far apart in one context, q large and small by rows."""
    rng = np.random.default_rng(19)
    D, bs, H = 64, 16, 4
    for counts in ([1, 4], [50, 20]):
        lens = [130, 300]
        tables, start, blocks = batch(rng, lens, counts, bs)
        c = Cache(ctx, blocks, 2, D, bs, rng)
        c.scales[::2, 1] *= scale
        c.scales[::3, 1] = 0
        c.scales[:, 0] *= np.float32(2.0 ** -20)
        c.ds.upload(c.scales)
        q = rng.standard_normal((start[-1], H * D)).astype(np.float32)
        q *= np.exp2(rng.integers(10, 22, (start[-1], 1))).astype(np.float32)
        q[-1] = 0
        check_attention(ctx, c, q, tables, start, lens, H)


@pytest.mark.parametrize("value", [np.nan, np.inf])
def test_attention_of_a_row_that_is_no_number(ctx, value):
    """It is NaN itself and leaves the other rows and heads alone."""
    rng = np.random.default_rng(20)
    for counts in ([1, 3], [50, 20]):
        lens = [70, 90]
        tables, start, blocks = batch(rng, lens, counts, 16)
        c = Cache(ctx, blocks, 2, 64, 16, rng)
        q = rng.standard_normal((start[-1], 4 * 64)).astype(np.float32)
        clean = check_attention(ctx, c, q, tables, start, lens, 4)
        q[-1, 64 + 3] = value
        got = attend(ctx, c, q, tables, start, lens, 4)
        assert np.isnan(got[-1, 64:128]).all()
        got[-1, 64:128] = clean[-1, 64:128]
        assert np.array_equal(got, clean)


def test_offsets_beyond_32_bits(ctx):
    """Blocks whose codes lie past 2^32 bytes: the same rows and results as at
    the pool's start."""
    D, bs, Hkv, H = 128, 128, 8, 8
    blocks = 2 ** 32 // (2 * Hkv * bs * D) + 40
    rng = np.random.default_rng(21)
    codes = ctx.array(shape=(blocks, 2, Hkv, bs * D), dtype=np.int8)
    scales = ctx.array(shape=(blocks, 2, Hkv))
    n = 2 * bs + 9
    qkv = ctx.array(rng.standard_normal((n, (H + 2 * Hkv) * D)).astype(np.float32))
    got = []
    for ids in ([0, 2, 1], [blocks - 1, blocks - 30, blocks - 2]):
        pos, slots = rows_of([(ids, 0, n)], bs)
        p, s, t = ctx.array(i32(pos)), ctx.array(i32(slots)), ctx.array(i32([ids]))
        start, lens = ctx.array(i32([0, n])), ctx.array(i32([n]))
        one = ctx.array(i32([0, 1]))
        q, out, last, k, v = (ctx.array(np.zeros(sh, np.float32)) for sh in
                              ((n, H * D), (n, H * D), (1, H * D), (n, Hkv, D), (n, Hkv, D)))
        nnhip.call("nnhip_rope_kv_append_paged_q8", ctx.h, qkv.p, n, H, Hkv, D, p.p, s.p, None,
                   None, n, q.p, codes.p, scales.p, bs, blocks)
        nnhip.call("nnhip_attention_paged_q8", ctx.h, q.p, n, codes.p, scales.p, bs, blocks, t.p, 3,
                   start.p, lens.p, 1, H, Hkv, D, out.p)
        nnhip.call("nnhip_attention_paged_q8", ctx.h, q.p, 1, codes.p, scales.p, bs, blocks, t.p, 3,
                   one.p, lens.p, 1, H, Hkv, D, last.p)
        nnhip.call("nnhip_kv_read_paged_q8", ctx.h, codes.p, scales.p, bs, blocks, s.p, n, Hkv, D,
                   k.p, v.p)
        got.append([x.numpy() for x in (q, out, last, k, v)])
    for a, b in zip(*got):
        assert np.abs(a).max() > 0 and np.array_equal(a, b)
    codes.free()


# ---------------------------------------------------------------- together ----
@pytest.mark.parametrize("bs,H,Hkv,D", [(16, 4, 2, 64), (64, 8, 1, 128), (32, 2, 2, 32)])
def test_serving_steps(ctx, bs, H, Hkv, D):
    """Prompts are admitted, requests decode, verify steps are cut back, a
    request ends and another takes its place: two layers over one plan."""
    rng = np.random.default_rng(bs)
    B, layers = 4, 2
    pc = nnhip.PagedKVCache(ctx, B, 12, 30, bs, H, Hkv, D, layers=layers)
    ref = R.Tables(B, 12, 30, bs)
    ref.free[:] = np.arange(30)[::-1]
    ref.tables[:] = -1
    codes = [np.zeros((30, 2, Hkv, bs * D), np.int8) for _ in range(layers)]
    scales = [np.zeros((30, 2, Hkv), np.float32) for _ in range(layers)]
    cos, sin = angles(12 * bs, D)
    dcos, dsin = ctx.array(cos), ctx.array(sin)
    lens = np.zeros(B, np.int64)
    steps = [([0, 0, 0, 0], [50, 0, 33, 2]), (None, [1, 20, 1, 1]), (None, [1, 1, 1, 1]),
             ([48, 0, 0, 0], [6, 6, 6, 6]), ([-3, -5, -1, 0], [6, 6, 6, 6]),
             ([-6, 0, -6, -2], [1, 1, 1, 0]), ([-999, 0, 0, -999], [70, 1, 1, 0]),
             (None, [1, 1, 1, 0])]
    for n, (cut, added) in enumerate(steps):
        if cut is None:
            cached = lens.copy()
        else:                                      # negative: tokens taken back
            cut = np.array(cut)
            cached = np.where(cut > 0, np.minimum(cut, lens), np.maximum(lens + cut, 0))
        added = np.array(added)
        pad = n % 3
        T = int(added.sum()) + pad
        pc.step(cached, added, rows=T)
        st, start, total, pos, slots = ref.step(i32(cached), i32(added), T)
        assert st == 0
        assert np.array_equal(pc.slots.numpy()[:T], slots)
        for layer in range(layers):
            qkv = rng.standard_normal((T, (H + 2 * Hkv) * D)).astype(np.float32)
            want_q = np.full((T, H * D), 7.0)
            R.append(qkv, pos, slots, cos, sin, H, codes[layer], scales[layer], D, bs, want_q)
            x, q, out = (ctx.array(a) for a in (qkv, np.full((T, H * D), 7.0, np.float32),
                                                np.full((T, H * D), 7.0, np.float32)))
            pc.append(x, q, len(cos), dcos, dsin, layer=layer)
            pc.attention(q, out, layer=layer)
            q_close(q.numpy(), want_q)
            want = np.full((T, H * D), 7.0)
            bound = R.attention(q.numpy(), codes[layer], scales[layer], ref.tables, start, total, H,
                                D, bs, want)
            assert (np.abs(out.numpy() - want) <= bound + U * np.abs(want)).all()
            live = slots[slots >= 0]
            for got, w in zip(pc.read(live, layer=layer),
                              R.read(codes[layer], scales[layer], live, D, bs)):
                assert np.array_equal(got, w.astype(np.float32))
        lens = cached + added
    with pytest.raises(nnhip.NNHipError, match="max_blocks"):
        pc.step(lens, np.full(B, 13 * bs))
    with pytest.raises(nnhip.NNHipError, match="free"):
        pc.step(lens, np.full(B, 11 * bs) - lens)
    pc.step(lens, np.ones(B))                      # the pool is as it was
    assert ref.step(i32(lens), i32(np.ones(B)), B)[0] == 0
    assert np.array_equal(pc.slots.numpy()[:B], slots_of(ref, lens, bs))


def slots_of(ref, pos, bs):
    return ref.tables[np.arange(len(pos)), pos // bs] * bs + pos % bs


def test_attention_agrees_with_the_contiguous_cache(ctx):
    """Values that both caches hold exactly (codes times a power of two) give
    what nnhip_attention_kq gives over an fp32 cache, within both bounds."""
    rng = np.random.default_rng(30)
    B, S, H, Hkv, D, bs, cap = 3, 2, 4, 2, 64, 16, 64
    lens = np.array([40, 64, 17])
    tables, start, blocks = batch(rng, list(lens), [S] * B, bs)
    c = Cache(ctx, blocks, Hkv, D, bs, rng)
    q = rng.standard_normal((B * S, H * D)).astype(np.float32)
    kv = np.zeros((2, B, Hkv, cap, D), np.float32)
    for b in range(B):
        slots = tables[b, np.arange(lens[b]) // bs] * bs + np.arange(lens[b]) % bs
        for i, x in enumerate(R.read(c.codes, c.scales, slots, D, bs)):
            kv[i, b, :, :lens[b]] = x.swapaxes(0, 1)
    a = [ctx.array(x) for x in (q, kv[0], kv[1], i32(lens - S), np.zeros_like(q))]
    nnhip.call("nnhip_attention_kq", ctx.h, a[0].p, a[1].p, a[2].p, cap, a[3].p, B, S, H, Hkv, D,
               a[4].p)
    want = np.zeros((B * S, H * D))
    bound = R.attention(q, c.codes, c.scales, tables, start, lens, H, D, bs, want)
    got = attend(ctx, c, q, tables, start, lens, H)
    assert (np.abs(got - a[4].numpy()) <= 2 * (bound + U * np.abs(want))).all()
