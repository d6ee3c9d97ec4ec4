"""The paged cache's kernels at the sizes where each of them runs: wide and narrow
units of attention, ranges that are joined, units that wait in queues, appends of
many rows, large steps of tables, against the 64-bit restatement (paged_ref.py)."""
import numpy as np
import pytest

import paged_ref as R
from gpu_util import dispatch_rules, nnhip
from test_gpu_paged import (Cache, Dev, U, angles, attend, batch, i32, q_close, rows_of, same_step)

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def rules():
    return dispatch_rules()


def kernel(rules, T, B, H, Hkv):
    G = H // Hkv
    return "tall" if rules.attention_paged_tall(T, B, G, Hkv) else \
        "solo" if rules.attention_paged_solo(T, B, G, Hkv) else "short"


def problem(ctx, seed, lens, counts, H, Hkv, D, bs, pad=0):
    rng = np.random.default_rng(seed)
    tables, start, blocks = batch(rng, lens, counts, bs)
    c = Cache(ctx, blocks, Hkv, D, bs, rng)
    q = (rng.standard_normal((start[-1] + pad, H * D)) * 2).astype(np.float32)
    return c, q, tables, start


def check_rows(got, c, q, tables, start, lens, H, rows):
    """Rows of attention: each as the last token of a request of its own."""
    for b in range(len(lens)):
        n = start[b + 1] - start[b]
        for t in [t for t in rows if start[b] <= t < start[b + 1]]:
            seen = lens[b] - n + (t - start[b]) + 1
            want = np.full((1, H * c.D), 7.0)
            bound = R.attention(q[t:t + 1], c.codes, c.scales, tables[b:b + 1], [0, 1], [max(seen, 0)],
                                H, c.D, c.bs, want)
            assert np.array_equal(np.isnan(got[t]), np.isnan(want[0])), f"row {t} of request {b}"
            ok = ~np.isnan(want[0])
            d = (np.abs(got[t] - want[0]) - U * np.abs(want[0]) - bound[0])[ok]
            assert (d <= 0).all(), f"row {t} of request {b}: {d.max():.3g}"


def sample(rng, start, each):
    """The first and last rows of every request, and some between."""
    rows = set()
    for a, z in zip(start[:-1], start[1:]):
        if z > a:
            rows |= {a, z - 1} | set(rng.integers(a, z, each).tolist())
    return sorted(rows)


WIDE = [(32, 16, 32, 4, [400, 368, 1, 0], [0, 77, 30, 0]),
        (64, 64, 32, 4, [768, 130], [33, 0]),
        (64, 16, 16, 16, [900, 700, 40], [0, 100, 9]),
        (128, 32, 16, 4, [1500, 63], [0, 64]),
        (128, 128, 6, 1, [2100, 2100], [1, 0]),
        (32, 128, 17, 1, [1500], [40])]


@pytest.mark.parametrize("D,bs,H,Hkv,counts,cached", WIDE)
def test_wide_units(ctx, rules, D, bs, H, Hkv, counts, cached):
    lens = [a + b for a, b in zip(counts, cached)]
    c, q, tables, start = problem(ctx, D + bs, lens, counts, H, Hkv, D, bs, pad=3)
    assert kernel(rules, len(q), len(lens), H, Hkv) == "tall"
    got = attend(ctx, c, q, tables, start, lens, H)
    assert (got[start[-1]:] == 7).all()
    check_rows(got, c, q, tables, start, lens, H, sample(np.random.default_rng(1), start, 12))


@pytest.mark.parametrize("D", [32, 64, 128])
def test_wide_units_of_several_ranges(ctx, rules, D):
    """Chunks of prompts behind long contexts, one behind none; more units than
    workgroups run at once."""
    H, Hkv, counts, cached = 96, 2, [250, 140, 300], [5000, 0, 3000]
    lens = [a + b for a, b in zip(counts, cached)]
    c, q, tables, start = problem(ctx, D, lens, counts, H, Hkv, D, 32)
    assert kernel(rules, len(q), 3, H, Hkv) == "tall"
    got = attend(ctx, c, q, tables, start, lens, H)
    check_rows(got, c, q, tables, start, lens, H, sample(np.random.default_rng(2), start, 2))


def test_long_requests_without_rows_beside_prompts(ctx, rules):
    """They have no ranges to count, however long they are."""
    counts, lens = [900, 0, 0, 700, 0], [930, 2 ** 30, 2 ** 30, 700, 5000]
    rng = np.random.default_rng(28)
    mb = 2 ** 30 // 128
    tables = np.zeros((5, 64), np.int64)
    tables[0, :8], tables[3, :6] = rng.permutation(20)[:8], rng.permutation(20)[:6]
    c = Cache(ctx, 20, 2, 64, 128, rng)
    start = np.concatenate(([0], np.cumsum(counts)))
    q = rng.standard_normal((1600, 16 * 64)).astype(np.float32)
    assert kernel(rules, 1600, 5, 16, 2) == "tall"
    wide = ctx.array(shape=(5, mb), dtype=np.int32)     # rows of 2^23 entries
    flat = np.zeros((5, mb), np.int32)
    flat[:, :64] = tables
    wide.upload(flat)
    a = [ctx.array(x) for x in (q, i32(start), i32(lens))]
    out = ctx.array(np.full((1600, 16 * 64), 7.0, np.float32))
    nnhip.call("nnhip_attention_paged_q8", ctx.h, a[0].p, 1600, c.dc.p, c.ds.p, 128, 20, wide.p, mb,
               a[1].p, a[2].p, 5, 16, 2, 64, out.p)
    check_rows(out.numpy(), c, q, tables, start, lens, 16, sample(rng, start, 3))


def test_wide_units_that_see_nothing(ctx, rules):
    """More rows than tokens: the first of them are zero."""
    counts, lens = [800, 700, 400], [30, 700, 0]
    c, q, tables, start = problem(ctx, 3, lens, counts, 16, 2, 64, 16)
    assert kernel(rules, len(q), 3, 16, 2) == "tall"
    got = attend(ctx, c, q, tables, start, lens, 16)
    assert (got[:770] == 0).all() and (got[1500:] == 0).all()
    check_rows(got, c, q, tables, start, lens, 16, [769, 770, 771, 799, 800, 801, 1100, 1499])


@pytest.mark.parametrize("D", [32, 64, 128])
@pytest.mark.parametrize("H,Hkv", [(16, 16), (48, 16)])
def test_units_of_a_wave_each(ctx, rules, D, H, Hkv):
    """Many short requests, and one whose keys are split and joined."""
    rng = np.random.default_rng(D + H)
    lens = rng.integers(1, 200, 110)
    lens[[3, 50, 109]] = 2500, 0, 1100
    counts = (lens > 0).astype(int)
    c, q, tables, start = problem(ctx, D, list(lens), list(counts), H, Hkv, D, 16, pad=1)
    assert kernel(rules, len(q), 110, H, Hkv) == "solo"
    got = attend(ctx, c, q, tables, start, list(lens), H)
    assert (got[start[-1]:] == 7).all()
    rows = [start[b] for b in (0, 1, 3, 49, 51, 70, 108, 109)]
    check_rows(got, c, q, tables, start, list(lens), H, rows)


def test_as_many_requests_as_there_may_be(ctx, rules):
    rng = np.random.default_rng(5)
    lens = rng.integers(0, 40, 4096)
    counts = np.minimum(rng.integers(0, 3, 4096), lens)
    for H, Hkv, want in ((2, 1, "solo"), (1, 1, "solo")):
        c, q, tables, start = problem(ctx, 6, list(lens), list(counts), H, Hkv, 32, 16)
        assert kernel(rules, len(q), 4096, H, Hkv) == want
        got = attend(ctx, c, q, tables, start, list(lens), H)
        check_rows(got, c, q, tables, start, list(lens), H, range(0, len(q), 7))
    # most of them without rows
    counts[np.arange(4096) % 100 != 7] = 0
    c, q, tables, start = problem(ctx, 7, list(lens), list(counts), 4, 2, 64, 16)
    assert kernel(rules, len(q), 4096, 4, 2) == "short"
    got = attend(ctx, c, q, tables, start, list(lens), 4)
    check_rows(got, c, q, tables, start, list(lens), 4, range(len(q)))


@pytest.mark.parametrize("D", [32, 64, 128])
def test_narrow_units_in_queues(ctx, rules, D):
    """More units than workgroups, some of many ranges and some of few."""
    rng = np.random.default_rng(D)
    lens = rng.integers(1, 150, 90)
    lens[[0, 20, 89]] = 4000, 900, 14000
    counts = np.minimum(rng.integers(1, 4, 90), lens)
    c, q, tables, start = problem(ctx, D, list(lens), list(counts), 16, 8, D, 64)
    assert kernel(rules, len(q), 90, 16, 8) == "short"
    got = attend(ctx, c, q, tables, start, list(lens), 16)
    rows = sorted({start[b] + i for b in (0, 1, 20, 47, 88, 89) for i in range(counts[b])})
    check_rows(got, c, q, tables, start, list(lens), 16, rows)


@pytest.mark.parametrize("B", [63, 64, 65])
@pytest.mark.parametrize("D", [64, 128])
def test_as_many_requests_as_a_wave_has_lanes(ctx, rules, B, D):
    """And one more: the plan is a wave's or the workgroup's.  Units in queues, some
    requests without rows or tokens, the last with several ranges."""
    rng = np.random.default_rng(B)
    lens = rng.integers(0, 100, B)
    lens[[1, B - 1]] = 3000, 1300
    counts = np.minimum(1 + (np.arange(B) % 5 != 2), lens)
    counts[[7, 30]] = 0
    c, q, tables, start = problem(ctx, D, list(lens), list(counts), 16, 16, D, 32, pad=2)
    assert kernel(rules, len(q), B, 16, 16) == "short" and B * 16 > 512
    got = attend(ctx, c, q, tables, start, list(lens), 16)
    assert (got[start[-1]:] == 7).all()
    check_rows(got, c, q, tables, start, list(lens), 16, range(0, start[-1], 3))


@pytest.mark.parametrize("B", [64, 70])
def test_wide_units_of_many_requests(ctx, rules, B):
    rng = np.random.default_rng(B)
    counts = rng.integers(0, 60, B)
    lens = counts + rng.integers(0, 90, B)
    lens[5] += 2500
    c, q, tables, start = problem(ctx, 1, list(lens), list(counts), 32, 4, 64, 16, pad=1)
    assert kernel(rules, len(q), B, 32, 4) == "tall"
    got = attend(ctx, c, q, tables, start, list(lens), 32)
    check_rows(got, c, q, tables, start, list(lens), 32, sample(rng, start, 1))


def test_calls_of_all_kinds_follow_one_another(ctx, rules):
    """Counters and scratch that a context keeps are left as the next call needs
    them: the same bits again, whatever ran before, also by turns with a context of
    its own stream."""
    rng = np.random.default_rng(9)
    many = list(rng.integers(1, 120, 110))
    many[7] = 1500
    kinds = [("tall", [5000, 400], [300, 400], 64, 2, 64), ("solo", many, [1] * 110, 16, 16, 64),
             ("short", [9000, 40, 2000], [1, 3, 2], 8, 2, 128), ("short", many, [1] * 110, 16, 8, 32)]
    with nnhip.Context(0) as other:
        runs = []
        for want, lens, counts, H, Hkv, D in kinds:
            for o in (ctx, other):
                c, q, tables, start = problem(o, 11, lens, counts, H, Hkv, D, 32)
                assert kernel(rules, len(q), len(lens), H, Hkv) == want
                runs.append((o, c, q, tables, start, lens, H))
        first = [attend(*r) for r in runs]
        for a, b in zip(first[::2], first[1::2]):
            assert np.array_equal(a, b)
        for _ in range(3):
            for i in rng.permutation(len(runs)):
                assert np.array_equal(attend(*runs[i]), first[i])
        for r in runs:
            r[1].dc = r[1].ds = None               # the other context's before it ends


def test_calls_without_a_wait_between_them(ctx):
    """Attention of different sizes one after the other on a stream."""
    rng = np.random.default_rng(10)
    lens = [7000, 30, 1]
    c, q, tables, start = problem(ctx, 12, lens, [2, 3, 1], 8, 2, 64, 16)
    want = attend(ctx, c, q, tables, start, lens, 8)
    a = [ctx.array(x) for x in (q, i32(tables), i32(start), i32(lens))]
    outs = [ctx.array(np.zeros_like(q)) for _ in range(20)]
    for o in outs:
        nnhip.call("nnhip_attention_paged_q8", ctx.h, a[0].p, len(q), c.dc.p, c.ds.p, 16, c.blocks,
                   a[1].p, tables.shape[1], a[2].p, a[3].p, 3, 8, 2, 64, o.p)
    for o in outs:
        assert np.array_equal(o.numpy(), want)


# What the narrow kernel's tests in test_gpu_paged.py hold it to, for the others.
def kinds(ctx, rules, kind, seed):
    """(cache, q, tables, start, lens, H, rows to look at)"""
    if kind == "tall":
        lens, counts, H, Hkv, rows = [1100, 61], [820, 10], 32, 2, [0, 300, 819, 820, 829]
    else:
        lens = [100 + i % 9 for i in range(110)]
        lens[0] = 1100
        counts, H, Hkv, rows = [1] * 110, 16, 16, [0, 1, 2, 108, 109]
    c, q, tables, start = problem(ctx, seed, lens, counts, H, Hkv, 64, 16)
    assert kernel(rules, len(q), len(lens), H, Hkv) == kind
    return c, q, tables, start, lens, H, rows


@pytest.mark.parametrize("kind", ["tall", "solo"])
def test_nothing_behind_the_tokens_is_seen(ctx, rules, kind):
    c, q, tables, start, lens, H, rows = kinds(ctx, rules, kind, 21)
    rng = np.random.default_rng(22)
    first = attend(ctx, c, q, tables, start, lens, H)
    check_rows(first, c, q, tables, start, lens, H, rows)
    used = np.zeros(c.blocks, bool)
    k, v = R.grids(c.codes, c.Hkv, 64, 16)
    for b, n in enumerate(lens):
        for j in range(-(-n // 16)):
            used[tables[b, j]] = True
            k[tables[b, j], :, max(n - j * 16, 0):] = 127
            v[tables[b, j], :, max(n - j * 16, 0):] = -127
        tables[b, -(-n // 16):] = rng.integers(0, c.blocks, tables.shape[1] + -n // 16)
    c.scales[~used] = np.nan
    c.codes[~used] = -128
    c.dc.upload(c.codes)
    c.ds.upload(c.scales)
    assert np.array_equal(first, attend(ctx, c, q, tables, start, lens, H))


@pytest.mark.parametrize("kind,T,B,H,Hkv", [("short", 100, 50, 4, 2), ("tall", 800, 6, 32, 2),
                                            ("solo", 400, 4096, 8, 8), ("tall", 4096, 200, 64, 2)])
def test_requests_that_have_the_same_rows_have_none(ctx, rules, kind, T, B, H, Hkv):
    """Bounds that go up and down: half the requests have all of the rows."""
    D, bs = 32, 16
    assert kernel(rules, T, B, H, Hkv) == kind
    c = Cache(ctx, 8, Hkv, D, bs, np.random.default_rng(1))
    start = np.where(np.arange(B + 1) % 2, T, 0)
    a = [ctx.array(i32(x)) for x in (np.arange(B * 2).reshape(B, 2) % 8, start, np.full(B, 30))]
    q, out = (ctx.array(np.full((T, H * D), x, np.float32)) for x in (1, 7))
    nnhip.call("nnhip_attention_paged_q8", ctx.h, q.p, T, c.dc.p, c.ds.p, bs, c.blocks, a[0].p, 2,
               a[1].p, a[2].p, B, H, Hkv, D, out.p)
    assert (out.numpy() == 7).all()


@pytest.mark.parametrize("kind", ["tall", "solo"])
@pytest.mark.parametrize("kv", [0, 1])
def test_a_block_whose_scale_is_no_number(ctx, rules, kind, kv):
    c, q, tables, start, lens, H, rows = kinds(ctx, rules, kind, 23)
    c.scales[tables[0, 60], kv, 1] = np.nan        # tokens 960 on, one head
    c.ds.upload(c.scales)
    got = attend(ctx, c, q, tables, start, lens, H)
    rows += [679, 680, 681] if kind == "tall" else []  # see 960 tokens, 961, 962
    check_rows(got, c, q, tables, start, lens, H, rows)
    assert np.isnan(got[start[1] - 1]).any() and not np.isnan(got[start[1]:]).any()


@pytest.mark.parametrize("kind", ["tall", "solo"])
@pytest.mark.parametrize("bad", [-1, 10 ** 6, 2 ** 31 - 1, -2 ** 31])
def test_a_table_entry_outside_the_pool(ctx, rules, kind, bad):
    c, q, tables, start, lens, H, rows = kinds(ctx, rules, kind, 24)
    tables[0, 50], tables[1, 0] = bad, bad
    got = attend(ctx, c, q, tables, start, lens, H)
    check_rows(got, c, q, tables, start, lens, H, rows)


@pytest.mark.parametrize("kind", ["tall", "solo"])
@pytest.mark.parametrize("scale", [1e-37, 1e-20, 1e20])
def test_scales_far_apart(ctx, rules, kind, scale):
    c, q, tables, start, lens, H, rows = kinds(ctx, rules, kind, 25)
    c.scales[::3, 1] *= np.float32(scale)
    c.scales[::5, 0] *= np.float32(min(scale, 1e-3))
    c.scales[::7] = 0
    c.ds.upload(c.scales)
    q[::2] *= np.float32(1e-15)
    got = attend(ctx, c, q, tables, start, lens, H)
    check_rows(got, c, q, tables, start, lens, H, rows)


@pytest.mark.parametrize("kind", ["tall", "solo"])
@pytest.mark.parametrize("value", [np.nan, np.inf, -np.inf])
def test_a_row_that_is_no_number(ctx, rules, kind, value):
    c, q, tables, start, lens, H, rows = kinds(ctx, rules, kind, 26)
    first = attend(ctx, c, q, tables, start, lens, H)
    bad = [0, len(q) // 2, len(q) - 1]
    q[bad, 64 * 3 + 5] = value
    got = attend(ctx, c, q, tables, start, lens, H)
    head = np.zeros(got.shape, bool)
    head[bad, 64 * 3:64 * 4] = True
    assert np.isnan(got[head]).all() and np.array_equal(got[~head], first[~head])


@pytest.mark.parametrize("kind,H,B", [("tall", 128, 1), ("solo", 8, 200)])
def test_codes_beyond_32_bits(ctx, rules, kind, H, B):
    """Blocks past 2^32 bytes of codes: what the same blocks give at the start."""
    D, bs, Hkv, T = 128, 128, 8, 265 if kind == "tall" else B
    blocks = 2 ** 32 // (2 * Hkv * bs * D) + 40
    assert kernel(rules, T, B, H, Hkv) == kind
    rng = np.random.default_rng(27)
    codes = ctx.array(shape=(blocks, 2, Hkv, bs * D), dtype=np.int8)
    scales = ctx.array(shape=(blocks, 2, Hkv))
    n = 1100
    qkv = ctx.array(rng.standard_normal((n, 3 * Hkv * D)).astype(np.float32))
    q = ctx.array(rng.standard_normal((T, H * D)).astype(np.float32))
    start = ctx.array(i32([0, T] if kind == "tall" else range(B + 1)))
    lens = ctx.array(i32([n] * B))
    got = []
    for ids in (np.arange(9), blocks - 1 - 3 * np.arange(9)):
        pos, slots = rows_of([(ids, 0, n)], bs)
        p, s = ctx.array(i32(pos)), ctx.array(i32(slots))
        t = ctx.array(i32(np.tile(ids, (B, 1))))
        turned, out = (ctx.array(np.zeros(sh, np.float32)) for sh in ((n, Hkv * D), (T, H * D)))
        nnhip.call("nnhip_rope_kv_append_paged_q8", ctx.h, qkv.p, n, Hkv, Hkv, D, p.p, s.p, None,
                   None, n, turned.p, codes.p, scales.p, bs, blocks)
        nnhip.call("nnhip_attention_paged_q8", ctx.h, q.p, T, codes.p, scales.p, bs, blocks, t.p, 9,
                   start.p, lens.p, B, H, Hkv, D, out.p)
        got.append((turned.numpy(), out.numpy()))
    for a, b in zip(*got):
        assert np.abs(a).max() > 0 and np.array_equal(a, b)
    codes.free()


# ------------------------------------------------------------------ append ----
@pytest.mark.parametrize("D,bs,Hkv,n", [(64, 16, 16, 520), (128, 64, 8, 1000), (32, 128, 16, 700)])
def test_append_of_many_single_tokens(ctx, D, bs, Hkv, n):
    """A decode step of many requests: every row leads a block."""
    rng = np.random.default_rng(n)
    c = Cache(ctx, n, Hkv, D, bs, rng)
    pos = rng.integers(0, bs, n)
    slots = rng.permutation(n) * bs + pos
    slots[rng.random(n) < 0.03] = -1
    qkv = rng.standard_normal((n, (2 * Hkv) * D + Hkv * D)).astype(np.float32)
    qkv *= np.exp2(rng.integers(-6, 7, (n, 1))).astype(np.float32)
    cos, sin = angles(bs, D)
    q_close(*c.append(qkv, pos, slots, Hkv, cos, sin))
    c.assert_same()


@pytest.mark.parametrize("D", [32, 64, 128])
@pytest.mark.parametrize("bs", [16, 32, 64, 128])
def test_append_of_long_prompts(ctx, D, bs):
    """Blocks that a workgroup shares, some begun before the call, rows skipped."""
    Hkv, n = 8, [517, 3, 460, 90, 1]
    rng = np.random.default_rng(D * bs)
    lists, at = [], 0
    for i, m in enumerate(n):
        begun = [0, 5, bs - 1, 0, 9][i]
        k = -(-(m + begun) // bs)
        lists.append((np.arange(at, at + k), begun, m))
        at += k
    pos, slots = rows_of(lists, bs)
    c = Cache(ctx, at + 3, Hkv, D, bs, rng)
    slots[rng.random(len(slots)) < 0.02] = -1
    qkv = rng.standard_normal((len(pos), 3 * Hkv * D)).astype(np.float32)
    qkv *= np.exp2(rng.integers(-3, 8, (len(pos), 1))).astype(np.float32)
    cos, sin = angles(520 + bs, D)
    q_close(*c.append(qkv, pos, slots, Hkv, cos, sin))
    c.assert_same()


@pytest.mark.parametrize("H,Hkv", [(1, 1), (3, 3), (128, 1), (40, 5)])
def test_append_of_other_numbers_of_heads(ctx, H, Hkv):
    rng = np.random.default_rng(H)
    c = Cache(ctx, 9, Hkv, 128, 16, rng)
    pos = np.arange(130)
    qkv = rng.standard_normal((130, (H + 2 * Hkv) * 128)).astype(np.float32)
    cos, sin = angles(130, 128)
    q_close(*c.append(qkv, pos, pos, H, cos, sin))
    c.assert_same()


@pytest.mark.parametrize("bs", [16, 32])
@pytest.mark.parametrize("lead", [0, 1, 3, 14, 15, 17])
def test_append_of_blocks_that_share_rows_on_end(ctx, bs, lead):
    """Two blocks by turns over bs rows, wherever these begin; among many others."""
    rng = np.random.default_rng(lead)
    for n, Hkv in ((70, 2), (1600, 8)):
        blocks = n // bs + 4
        c = Cache(ctx, blocks, Hkv, 64, bs, rng)
        ids = rng.permutation(blocks)
        slots = np.full(n, -1)
        for i, at in enumerate(range(lead, n - bs + 1, bs)):
            pair = ids[2 * (i // 2):2 * (i // 2) + 2] if i % 2 == 0 else None
            if pair is None:
                continue
            off = rng.permutation(bs)
            slots[at:at + bs] = pair[np.arange(bs) % 2] * bs + off
        pos = rng.integers(0, 60, n)
        qkv = rng.standard_normal((n, 3 * Hkv * 64)).astype(np.float32)
        cos, sin = angles(60, 64)
        q_close(*c.append(qkv, pos, slots, Hkv, cos, sin))
        c.assert_same()


@pytest.mark.parametrize("n", [1, 9])
def test_append_behind_any_scale(ctx, n):
    """Blocks whose scale is no power of two, or below the smallest that a call
    sets: it is kept while the new values fit."""
    rng = np.random.default_rng(n)
    bs, Hkv, D = 16, 4, 64
    c = Cache(ctx, 40, Hkv, D, bs, rng)
    c.scales[:] = rng.uniform(0.05, 0.3, c.scales.shape).astype(np.float32)
    c.scales[5:9] = 2.0 ** -140
    c.scales[9:12] = 0
    c.ds.upload(c.scales)
    pos, slots = rows_of([([b], 3, n) for b in range(40)], bs)
    qkv = rng.standard_normal((len(pos), 3 * Hkv * D)).astype(np.float32)
    qkv[(slots // bs == 5) | (slots // bs == 9)] = 0
    cos, sin = angles(20, D)
    q_close(*c.append(qkv, pos, slots, Hkv, cos, sin))
    c.assert_same()


@pytest.mark.parametrize("where", [0, 7, 15])
@pytest.mark.parametrize("value", [np.nan, np.inf, -np.inf, 3e38])
def test_append_of_one_value_among_many(ctx, where, value):
    """A value that is no number spoils its own head's block and no other."""
    rng = np.random.default_rng(1)
    D, bs, Hkv = 64, 16, 8
    c = Cache(ctx, 70, Hkv, D, bs, rng)
    pos = np.arange(1000)
    qkv = rng.standard_normal((1000, 3 * Hkv * D)).astype(np.float32)
    qkv[320 + where, (Hkv + 2) * D + 63] = value   # k of head 2, last dim
    qkv[656 + where, (2 * Hkv + 5) * D] = value    # v of head 5, first dim
    cos, sin = angles(1000, D)
    with np.errstate(invalid="ignore"):
        q_close(*c.append(qkv, pos, pos, Hkv, cos, sin))
    c.assert_same()


# ------------------------------------------------------------------ tables ----
@pytest.mark.parametrize("B,bs,most", [(256, 16, 60), (257, 32, 60), (777, 64, 130), (1024, 16, 30),
                                       (1500, 16, 40), (2, 16, 90000), (3, 128, 300000)])
def test_tables_of_every_number_of_requests(ctx, B, bs, most):
    """Taken, given back without rows of its own, taken again in another order."""
    rng = np.random.default_rng(B)
    added = rng.integers(0, most + 1, B)
    mb = -(-2 * most // bs) + 1
    ref = R.Tables(B, mb, int((-(-added // bs)).sum() * 3 // 2) + 9, bs, rng)
    T = int(added.sum()) + 3
    dev = Dev(ctx, ref, T)
    assert same_step(dev, [0] * B, added, T) == 0
    kept = rng.integers(0, added + 1)
    assert same_step(dev, kept, [0] * B, 0) == 0
    again = np.minimum(rng.integers(0, most + 1, B), added - kept)
    assert same_step(dev, kept, again, T) == 0
    assert same_step(dev, [0] * B, [0] * B, 2) == 0


# -------------------------------------------------------------------- read ----
@pytest.mark.parametrize("D,bs", [(32, 16), (64, 32), (128, 128)])
def test_read_of_runs_that_begin_and_end_anywhere(ctx, D, bs):
    rng = np.random.default_rng(D)
    Hkv = 5
    c = Cache(ctx, 40, Hkv, D, bs, rng)
    parts = [np.arange(a, min(a + n, 40 * bs)) for a, n in
             zip(rng.integers(0, 40 * bs, 60), rng.integers(1, 70, 60))]
    parts += [np.arange(50, 20, -1), np.full(33, 17), np.array([15, 16, 31, 32, 47])]
    slots = np.concatenate([parts[i] for i in rng.permutation(len(parts))])
    slots[rng.random(len(slots)) < 0.05] = -1
    a = ctx.array(i32(slots))
    k, v = (ctx.array(np.full((len(slots), Hkv, D), 5.0, np.float32)) for _ in range(2))
    nnhip.call("nnhip_kv_read_paged_q8", ctx.h, c.dc.p, c.ds.p, bs, 40, a.p, len(slots), Hkv, D,
               k.p, v.p)
    ok = slots >= 0
    for got, want in zip((k.numpy(), v.numpy()), R.read(c.codes, c.scales, slots[ok], D, bs)):
        assert np.array_equal(got[ok], want.astype(np.float32)) and (got[~ok] == 5).all()
