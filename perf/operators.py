"""The paged int8 KV cache of libnnhip as cases that can be timed and checked:
one dict of plain values per case.

  listed()             the fixed cases
  draw(rng)            one more case of the same ranges
  prepare(case, seed)  inputs and buffers a serving program holds beforehand
  run(state)           one pass: the library's entry points where `own`, else
                       the same operators in elementary torch operations
  work(case)           bytes and operations a pass cannot do without
  exact(case, seed)    the outputs in 64 bits, from the definitions

Kinds of case:

  tables     block tables and slot maps of a step built from request lengths,
             then the step's rollback (a verify step whose drafts are
             rejected, prompts that are taken back): blocks are taken from the
             pool and returned to it
  append     RoPE, then the k / v rows into their slots: int8 codes, one
             power-of-two scale a block, head and k or v; returned as the
             values that the requests' cached rows then stand for
  attention  causal attention of ragged rows over the cache
  read       cached rows as fp32

Cache layout: codes [blocks][k, v][Hkv][bs * D], k as [bs][D], v as [D][bs];
scales [blocks][k, v][Hkv].
"""
import ctypes
import math
import os
import random
import sys

import torch

own = False

DEV = "cuda"
F64 = torch.float64


def listed():
    return [
        # a decode step of a large batch: one token a request, few blocks move
        dict(name="tables_decode", kind="tables", B=256, S=1, cached=700, back=0, bs=16),
        # prompts admitted at once, and taken back
        dict(name="tables_prompts", kind="tables", B=64, S=2000, cached=0, back=0, bs=16),
        # a decode step's append: blocks that are continued
        dict(name="append_decode", kind="append", B=32, S=1, cached=100, H=16, Hkv=16, D=64,
             bs=16),
        # prompts with grouped heads
        dict(name="append_prompts", kind="append", B=9, S=1000, cached=0, H=16, Hkv=4, D=64,
             bs=32),
        # one request's first tokens: latency
        dict(name="attention_one", kind="attention", B=1, S=1, prompts=0, chunk=0, cached=99,
             H=16, Hkv=16, D=64, bs=16, pad=0),
        # a decode step with grouped heads, lengths of all sizes
        dict(name="attention_decode", kind="attention", B=32, S=1, prompts=0, chunk=0, cached=1023,
             H=16, Hkv=4, D=64, bs=16, pad=3),
        # a verify step: k + 1 = 6 rows a request
        dict(name="attention_verify", kind="attention", B=32, S=6, prompts=0, chunk=0, cached=320,
             H=16, Hkv=16, D=64, bs=32, pad=0),
        # a few requests with long contexts
        dict(name="attention_long", kind="attention", B=4, S=1, prompts=0, chunk=0, cached=131071,
             H=32, Hkv=8, D=128, bs=64, pad=0),
        # prompts
        dict(name="attention_prompts", kind="attention", B=4, S=1, prompts=4, chunk=1000, cached=0,
             H=16, Hkv=4, D=64, bs=16, pad=0),
        # chunks of two long prompts beside requests that decode
        dict(name="attention_mixed", kind="attention", B=33, S=3, prompts=2, chunk=500,
             cached=1500, H=16, Hkv=4, D=128, bs=32, pad=5),
        # a request's rows read back
        dict(name="read_one", kind="read", B=1, S=130, cached=0, Hkv=8, D=64, bs=16),
        # a batch's contexts read back
        dict(name="read_batch", kind="read", B=24, S=1000, cached=0, Hkv=8, D=128, bs=64),
    ]


def _log(rng, lo, hi):
    """An integer spread over the logarithm of [lo, hi]."""
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    kind = rng.choice(["tables", "append", "append", "attention", "attention", "attention",
                       "attention", "read"])
    bs = rng.choice([16, 16, 32, 64])
    if kind == "tables":
        S = _log(rng, 1, 2000)
        cached = rng.choice([0, _log(rng, 1, 2000)])
        return dict(kind=kind, B=_log(rng, 1, min(2048, 128000 // S)), S=S, cached=cached,
                    back=rng.randint(0, S), bs=bs)
    D = rng.choice([32, 64, 64, 64, 128, 128])
    Hkv = rng.choice([1, 2, 4, 8, 16] if D < 128 else [1, 2, 4, 8])
    if kind == "read":
        S = _log(rng, 1, 2000)
        return dict(kind=kind, B=_log(rng, 1, max(1, 16000 // S)), S=S, cached=0, Hkv=Hkv, D=D,
                    bs=bs)
    H = Hkv * rng.choice([1, 1, 2, 3, 4, 8])
    if kind == "append":
        S = rng.choice([1, rng.randint(2, 9), _log(rng, 10, 1000)])
        return dict(kind=kind, B=_log(rng, 1, max(1, min(128, 8000 // S))), S=S,
                    cached=rng.choice([0, _log(rng, 1, 200)]), H=H, Hkv=Hkv, D=D, bs=bs)
    form = rng.choice(["decode", "verify", "prompt", "mixed"])
    pad = rng.choice([0, 0, rng.randint(1, 9)])
    if form == "prompt":
        S, B, cached = _log(rng, 10, 1000), rng.randint(1, 6), rng.choice([0, _log(rng, 1, 2000)])
        return dict(kind=kind, B=B, S=1, prompts=B, chunk=S, cached=cached, H=min(H, 4 * Hkv),
                    Hkv=Hkv, D=D, bs=bs, pad=pad)
    if form == "mixed":
        return dict(kind=kind, B=rng.randint(4, 40), S=rng.randint(1, 4), prompts=rng.randint(1, 3),
                    chunk=_log(rng, 20, 500), cached=_log(rng, 1, 1500), H=min(H, 4 * Hkv),
                    Hkv=Hkv, D=D, bs=bs, pad=pad)
    B = _log(rng, 1, 128)
    return dict(kind=kind, B=B, S=1 if form == "decode" else rng.randint(2, 9), prompts=0, chunk=0,
                cached=_log(rng, 1, min(100000 if form == "decode" else 30000, 200000 // B)), H=H,
                Hkv=Hkv, D=D, bs=bs, pad=pad)


# ---------------------------------------------------------------- requests ----
def _lengths(case):
    """(cached, added) of every request.  In a batch one request in seven adds
    nothing, contexts are up to a quarter shorter than the longest, and one in
    five is much shorter."""
    B, S = case["B"], case["S"]
    cached, added = [], []
    for b in range(B):
        n = case["cached"] - (b * 37) % (case["cached"] // 4 + 1)
        cached.append(n // 16 if b % 5 == 2 else n)
        if b < case.get("prompts", 0):
            added.append(case["chunk"] - (b * 29) % (case["chunk"] // 4 + 1))
        else:
            added.append(0 if b % 7 == 3 else S - (b * 5) % (S // 2 + 1))
    return cached, added


def _gen(seed):
    return torch.Generator(device=DEV).manual_seed(int(seed))


def _randn(g, *shape, std=1.0):
    return torch.randn(*shape, generator=g, device=DEV) * std


def _ints(v):
    return torch.tensor(v, dtype=torch.int32, device=DEV)


def _blocks(n, bs):
    return -(-n // bs)


def _tables_for(lens, bs, max_blocks, num_blocks, seed):
    """Tables [B][max_blocks] that give the requests blocks of a shuffled pool;
    entries behind a request's blocks are -1.  Also the blocks left over."""
    ids = list(range(num_blocks))
    random.Random(seed).shuffle(ids)
    rows, at = [], 0
    for n in lens:
        k = _blocks(n, bs)
        rows.append(ids[at:at + k] + [-1] * (max_blocks - k))
        at += k
    return _ints(rows), ids[at:]


def _slots_of(tables, starts, counts, bs):
    """Slots of positions [start, start + count) of every request, in order."""
    n = sum(counts)
    b = torch.repeat_interleave(torch.arange(len(counts), device=DEV),
                                torch.tensor(counts, device=DEV), output_size=n)
    first = torch.tensor(counts, device=DEV).cumsum(0) - torch.tensor(counts, device=DEV)
    pos = torch.arange(n, device=DEV) - first[b] + torch.tensor(starts, device=DEV)[b]
    slots = tables[b, pos // bs].long() * bs + pos % bs
    return pos.int(), slots.int()


def _random_cache(g, nb, Hkv, D, bs):
    """Codes of normal values (the largest of a block near 127) and scales."""
    codes = torch.empty(nb, 2, Hkv, bs * D, device=DEV, dtype=torch.int8)
    step = max(1, (1 << 26) // (2 * Hkv * bs * D))
    for at in range(0, nb, step):
        part = codes[at:at + step]
        part.copy_(_randn(g, *part.shape, std=28.0).round_().clamp_(-127, 127))
    scales = torch.randint(-6, -3, (nb, 2, Hkv), generator=g, device=DEV).float().exp2()
    return codes, scales


def _rope_tables(n, D):
    """cos and sin [n][D / 2] of the usual angles, as fp32 inputs."""
    theta = 10000.0 ** (-torch.arange(0, D, 2, device=DEV, dtype=F64) / D)
    w = torch.arange(n, device=DEV, dtype=F64)[:, None] * theta
    return w.cos().float(), w.sin().float()


_CTX = None


def _nnhip():
    """The binding and the program's one context."""
    global _CTX
    path = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))),
                        "neural-network_amd", "python")
    if path not in sys.path:
        sys.path.insert(0, path)
    import nnhip
    if _CTX is None:
        torch.cuda.init()
        _CTX = nnhip.Context(0)
    return nnhip, _CTX.h


def _p(t):
    return ctypes.c_void_p(t.data_ptr())


def prepare(case, seed):
    s = _PREPARE[case["kind"]](case, seed)
    s["case"] = case
    return s


def run(state):
    return _RUN[state["case"]["kind"]](state)


def work(case):
    return _WORK[case["kind"]](case)


def exact(case, seed):
    return _EXACT[case["kind"]](case, seed)


# ------------------------------------------------------------------ tables ----
def _prep_tables(case, seed):
    B, bs = case["B"], case["bs"]
    cached, added = _lengths(case)
    mb = _blocks(case["cached"] + case["S"], bs) + 1
    nb = sum(_blocks(c + a, bs) for c, a in zip(cached, added)) + 8
    T = sum(added) + B % 5
    tables, rest = _tables_for(cached, bs, mb, nb, seed)
    free = _ints(rest + [-1] * (nb - len(rest)))
    # what is kept of the rows once the step is over
    kept = [c + min(a, case["back"]) for c, a in zip(cached, added)]
    s = dict(cached=_ints(cached), added=_ints(added), kept=_ints(kept), none=_ints([0] * B),
             tables=tables, held=_ints([_blocks(c, bs) for c in cached]), free=free,
             count=_ints([len(rest)]), mb=mb, nb=nb, T=T)
    for n in ("step", "back"):
        rows = T if n == "step" else 1
        s[n] = dict(row_start=_ints([0] * (B + 1)), lens=_ints([0] * B), pos=_ints([0] * rows),
                    slots=_ints([0] * rows), status=_ints([7]))
    return s


def _step_plain(s, cached, added, out, T):
    """One call of the block-table operator in torch."""
    bs, mb, nb = s["case"]["bs"], s["mb"], s["nb"]
    lens = (cached + added).long()
    need = torch.div(lens + bs - 1, bs, rounding_mode="floor")
    held, count = s["held"].long(), s["count"].long()
    back, take = (held - need).clamp(min=0), (need - held).clamp(min=0)
    j = torch.arange(mb, device=DEV)[None]
    R, K = back.sum(), take.sum()
    # returned blocks go on top of the stack, the first of them uppermost
    stack = torch.cat((s["free"], s["free"].new_zeros(1)))
    gone = (j >= need[:, None]) & (j < held[:, None])
    at = count + R - 1 - ((back.cumsum(0) - back)[:, None] + j - need[:, None])
    stack = stack.index_put((torch.where(gone, at, nb).flatten(),), s["tables"].flatten())
    new = (j >= held[:, None]) & (j < need[:, None])
    at = count + R - 1 - ((take.cumsum(0) - take)[:, None] + j - held[:, None])
    s["tables"].copy_(torch.where(new, stack[torch.where(new, at, nb)], s["tables"]))
    left = count + R - K
    s["free"].copy_(torch.where(torch.arange(nb, device=DEV) < left, stack[:nb], s["free"]))
    s["count"].copy_(left)
    s["held"].copy_(need)
    ends = added.long().cumsum(0)
    start = torch.cat((ends.new_zeros(1), ends))
    t = torch.arange(T, device=DEV)
    b = torch.searchsorted(ends, t, right=True).clamp(max=len(ends) - 1)
    pos = cached.long()[b] + t - start[b]
    ok = t < ends[-1]
    slot = s["tables"][b, torch.where(ok, pos // bs, 0)].long() * bs + pos % bs
    out["row_start"].copy_(start)
    out["lens"].copy_(lens)
    out["pos"].copy_(torch.where(ok, pos, -1))
    out["slots"].copy_(torch.where(ok, slot, -1))
    out["status"].zero_()


def _step_own(s, cached, added, out, T):
    nnhip, h = _nnhip()
    nnhip.call("nnhip_block_tables", h, s["case"]["B"], _p(cached), _p(added), s["case"]["bs"],
               s["mb"], _p(s["tables"]), _p(s["held"]), s["nb"], _p(s["free"]), _p(s["count"]), T,
               _p(out["row_start"]), _p(out["lens"]), _p(out["pos"]), _p(out["slots"]),
               _p(out["status"]))


def _run_tables(s):
    step = _step_own if own else _step_plain
    step(s, s["cached"], s["added"], s["step"], s["T"])
    step(s, s["kept"], s["none"], s["back"], 1)
    return [s["tables"], s["held"], s["free"], s["count"], s["step"], s["back"]]


def _work_tables(case):
    cached, added = _lengths(case)
    bs, B = case["bs"], case["B"]
    moved = sum(_blocks(c + a, bs) - _blocks(c + min(a, case["back"]), bs)
                for c, a in zip(cached, added))
    # 3 lengths in, 3 out a request and call; 2 integers a row; a block that is
    # taken, and one that is returned, is read once and written once
    return dict(bytes=2 * 24 * B + 8 * (sum(added) + B % 5) + 4 * moved * 4, flops=0)


# ------------------------------------------------------------------ append ----
def _prep_append(case, seed):
    g = _gen(seed)
    bs, H, Hkv, D = (case[n] for n in ("bs", "H", "Hkv", "D"))
    cached, added = _lengths(case)
    lens = [c + a for c, a in zip(cached, added)]
    mb = max(1, _blocks(max(lens), bs))
    nb = sum(_blocks(n, bs) for n in lens) + 2
    tables, _ = _tables_for(lens, bs, mb, nb, seed)
    pos, slots = _slots_of(tables, cached, added, bs)
    _, rows = _slots_of(tables, [0] * len(lens), lens, bs)
    codes, scales = _random_cache(g, nb, Hkv, D, bs)
    T = len(pos)
    qkv = _randn(g, T, H + 2 * Hkv, D)
    qkv[:, H:, : D // 16] *= 4.0                     # a few strong channels
    cos, sin = _rope_tables(max(1, max(lens)), D)
    e = torch.zeros
    return dict(qkv=qkv.flatten(1), pos=pos, slots=slots, rows=rows, codes=codes, scales=scales,
                cos=cos, sin=sin, nb=nb, q=e(T, H * D, device=DEV),
                k=e(len(rows), Hkv, D, device=DEV), v=e(len(rows), Hkv, D, device=DEV))


def _step_of(amax):
    """The smallest power of two 2^e, e >= -126, with amax <= 127 * 2^e; 0 for 0."""
    m, x = torch.frexp(amax)
    e = (x - 7 + (m * 128 > 127).int()).clamp(min=-126)
    step = (e.long() + 1023 << 52).view(F64)         # by its bits: ldexp's power is not exact
    return torch.where(amax > 0, step, 0.0)


def _read_plain(codes, scales, rows, bs, D):
    """k and v [rows][Hkv][D] that the cache holds in slots `rows`."""
    nb, _, Hkv, _ = codes.shape
    blk, off = (rows // bs).long(), (rows % bs).long()
    k = codes[:, 0].view(nb, Hkv, bs, D)[blk, :, off]
    v = codes[:, 1].view(nb, Hkv, D, bs)[blk, :, :, off]
    return (k.float() * scales[blk, 0][..., None], v.float() * scales[blk, 1][..., None])


def _run_append(s):
    c = s["case"]
    bs, H, Hkv, D = (c[n] for n in ("bs", "H", "Hkv", "D"))
    if own:
        nnhip, h = _nnhip()
        nnhip.call("nnhip_rope_kv_append_paged_q8", h, _p(s["qkv"]), len(s["pos"]), H, Hkv, D,
                   _p(s["pos"]), _p(s["slots"]), _p(s["cos"]), _p(s["sin"]), len(s["cos"]),
                   _p(s["q"]), _p(s["codes"]), _p(s["scales"]), bs, s["nb"])
        nnhip.call("nnhip_kv_read_paged_q8", h, _p(s["codes"]), _p(s["scales"]), bs, s["nb"],
                   _p(s["rows"]), len(s["rows"]), Hkv, D, _p(s["k"]), _p(s["v"]))
        return s["q"], s["k"], s["v"], s["scales"]
    # 64 bits: a code next to a rounding border has to fall on the right side
    x = s["qkv"].to(F64).view(-1, H + 2 * Hkv, D)
    at = s["pos"].long()
    cs, sn = s["cos"][at].to(F64)[:, None], s["sin"][at].to(F64)[:, None]
    a, b = x[:, :H + Hkv, 0::2], x[:, :H + Hkv, 1::2]
    rot = torch.stack((a * cs - b * sn, a * sn + b * cs), -1).flatten(-2)
    kv = torch.stack((rot[:, H:], x[:, H + Hkv:]), 1)          # [T][k, v][Hkv][D]
    codes, scales = s["codes"], s["scales"]
    nb = s["nb"]
    blk, off = (s["slots"] // bs).long(), (s["slots"] % bs).long()
    need = torch.zeros(nb, 2, Hkv, device=DEV, dtype=F64).scatter_reduce_(
        0, blk[:, None, None].expand(-1, 2, Hkv), kv.abs().amax(-1), "amax")
    first = torch.full((nb,), bs, device=DEV).scatter_reduce_(0, blk, off, "amin")
    old = torch.where((first == 0)[:, None, None], 0.0, scales.to(F64))
    new = torch.maximum(old, _step_of(need))
    # the codes of the block's older rows in the grown scale
    keep = torch.arange(bs, device=DEV) < torch.where(first < bs, first, 0)[:, None]
    ratio = torch.where(new > 0, old / new, 0.0)
    kc, vc = codes[:, 0].view(nb, Hkv, bs, D), codes[:, 1].view(nb, Hkv, D, bs)
    kc.copy_(torch.where(keep[:, None, :, None], (kc * ratio[:, 0, :, None, None]).round(), kc))
    vc.copy_(torch.where(keep[:, None, None, :], (vc * ratio[:, 1, :, None, None]).round(), vc))
    q8 = torch.where(new[blk][..., None] > 0, kv / new[blk][..., None], 0.0).round()
    kc[blk, :, off] = q8[:, 0].to(torch.int8)
    vc[blk, :, :, off] = q8[:, 1].to(torch.int8)
    scales.copy_(torch.where((first < bs)[:, None, None], new, scales.to(F64)))
    return (rot[:, :H].flatten(1).float(), *_read_plain(codes, scales, s["rows"], bs, D), scales)


def _exact_append(case, seed):
    s = _prep_append(case, seed)
    bs, H, Hkv, D = (case[n] for n in ("bs", "H", "Hkv", "D"))
    cached, added = _lengths(case)
    codes, scales = s["codes"], s["scales"].to(F64)
    x = s["qkv"].to(F64).view(-1, H + 2 * Hkv, D)
    z = torch.complex(x[:, :H + Hkv, 0::2], x[:, :H + Hkv, 1::2])
    turn = torch.complex(s["cos"].to(F64), s["sin"].to(F64))[s["pos"].long()]
    z = torch.view_as_real(z * turn[:, None]).flatten(-2)
    q, k, v = z[:, :H].flatten(1), z[:, H:], x[:, H + Hkv:]
    # block by block of every request: its rows of this call, and older ones
    vals, t, r = [], 0, 0
    rows = s["rows"].long()
    for c, a in zip(cached, added):
        n = c + a
        for lo in range(0, n, bs):
            hi = min(n, lo + bs)
            blk = int(rows[r + lo]) // bs
            first = max(lo, c)                      # first new position
            for i, fresh in enumerate((k, v)):
                grid = codes[blk, i].view(Hkv, bs, D) if i == 0 else \
                    codes[blk, i].view(Hkv, D, bs).transpose(1, 2)
                w = grid[:, :hi - lo].to(F64)
                sc = scales[blk, i].clone()
                if first < hi:
                    new = fresh[t + first - c:t + hi - c].transpose(0, 1)
                    top = new.abs().amax((1, 2)) / 127.0
                    want = torch.where(top > 0, top.log2().ceil().exp2(), 0.0)
                    # log2 may round across a power of two
                    want = torch.where(want >= 2 * top, want / 2, want)
                    want = torch.where(want < top, want * 2, want)
                    if first > lo:
                        to = torch.maximum(sc, want)
                        w[:, :first - lo] = (w[:, :first - lo] * (sc / to)[:, None, None]).round()
                        sc = to
                    else:
                        sc = want
                    w[:, first - lo:] = torch.where(sc[:, None, None] > 0,
                                                    new / sc[:, None, None], 0.0).round()
                    scales[blk, i] = sc
                vals.append((w * sc[:, None, None]).transpose(0, 1))
        t, r = t + a, r + n
    return q, torch.cat(vals[0::2]), torch.cat(vals[1::2]), scales


def _work_append(case):
    cached, added = _lengths(case)
    H, Hkv, D = case["H"], case["Hkv"], case["D"]
    T, rows = sum(added), sum(cached) + sum(added)
    # fp32 rows in, q out, codes out, cos / sin in; then the read of every row
    return dict(bytes=T * (4 * (H + 2 * Hkv) * D + 4 * H * D + 2 * Hkv * D + 4 * D + 8)
                + rows * (10 * Hkv * D + 4), flops=3 * T * (H + Hkv) * D)


# -------------------------------------------------------------------- read ----
def _prep_read(case, seed):
    g = _gen(seed)
    bs, Hkv, D = (case[n] for n in ("bs", "Hkv", "D"))
    _, lens = _lengths(case)
    nb = sum(_blocks(n, bs) for n in lens) + 2
    tables, _ = _tables_for(lens, bs, max(1, _blocks(max(lens), bs)), nb, seed)
    _, rows = _slots_of(tables, [0] * len(lens), lens, bs)
    codes, scales = _random_cache(g, nb, Hkv, D, bs)
    e = torch.zeros
    return dict(codes=codes, scales=scales, rows=rows, nb=nb,
                k=e(len(rows), Hkv, D, device=DEV), v=e(len(rows), Hkv, D, device=DEV))


def _run_read(s):
    c = s["case"]
    if own:
        nnhip, h = _nnhip()
        nnhip.call("nnhip_kv_read_paged_q8", h, _p(s["codes"]), _p(s["scales"]), c["bs"], s["nb"],
                   _p(s["rows"]), len(s["rows"]), c["Hkv"], c["D"], _p(s["k"]), _p(s["v"]))
        return s["k"], s["v"]
    return _read_plain(s["codes"], s["scales"], s["rows"], c["bs"], c["D"])


def _exact_read(case, seed):
    s = _prep_read(case, seed)
    bs, Hkv, D = (case[n] for n in ("bs", "Hkv", "D"))
    rows = s["rows"].long()
    val = s["codes"].to(F64) * s["scales"].to(F64)[..., None]
    k = val[:, 0].view(-1, Hkv, bs, D).transpose(1, 2).reshape(-1, Hkv, D)
    v = val[:, 1].view(-1, Hkv, D, bs).permute(0, 3, 1, 2).reshape(-1, Hkv, D)
    return k[rows], v[rows]


def _work_read(case):
    return dict(bytes=sum(_lengths(case)[1]) * (10 * case["Hkv"] * case["D"] + 4), flops=0)


# --------------------------------------------------------------- attention ----
def _prep_attention(case, seed):
    g = _gen(seed)
    bs, H, Hkv, D = (case[n] for n in ("bs", "H", "Hkv", "D"))
    cached, added = _lengths(case)
    lens = [c + a for c, a in zip(cached, added)]
    mb = max(1, _blocks(max(lens), bs) + case["B"] % 3)
    nb = sum(_blocks(n, bs) for n in lens) + 2
    tables, _ = _tables_for(lens, bs, mb, nb, seed)
    codes, scales = _random_cache(g, nb, Hkv, D, bs)
    starts = [0]
    for a in added:
        starts.append(starts[-1] + a)
    T = starts[-1] + case["pad"]
    # scores of a few units: some keys stand out
    q = _randn(g, T, H * D, std=1.7)
    return dict(q=q, codes=codes, scales=scales, tables=tables, lens=_ints(lens), nb=nb, mb=mb,
                row_start=_ints(starts), out=torch.zeros(T, H * D, device=DEV),
                most=max(added), longest=max(lens))


def _run_attention(s):
    c = s["case"]
    B, bs, H, Hkv, D = (c[n] for n in ("B", "bs", "H", "Hkv", "D"))
    if own:
        nnhip, h = _nnhip()
        nnhip.call("nnhip_attention_paged_q8", h, _p(s["q"]), len(s["q"]), _p(s["codes"]),
                   _p(s["scales"]), bs, s["nb"], _p(s["tables"]), s["mb"], _p(s["row_start"]),
                   _p(s["lens"]), B, H, Hkv, D, _p(s["out"]))
        return s["out"]
    # the requests padded to the longest: keys and values as fp32, then
    # products, a masked softmax and products
    most, n = s["most"], _blocks(s["longest"], bs) * bs
    tab = s["tables"][:, :n // bs].clamp(min=0).long()
    k = (s["codes"][:, 0][tab].float() * s["scales"][:, 0][tab][..., None]).view(B, -1, Hkv, bs, D)
    k = k.transpose(1, 2).reshape(B, Hkv, n, D)
    v = (s["codes"][:, 1][tab].float() * s["scales"][:, 1][tab][..., None]).view(B, -1, Hkv, D, bs)
    v = v.permute(0, 2, 1, 4, 3).reshape(B, Hkv, n, D)
    first, rows = s["row_start"][:-1].long(), s["row_start"].long().diff()
    i = torch.arange(most, device=DEV)
    live = i < rows[:, None]
    t = torch.where(live, first[:, None] + i, len(s["q"]))     # [B][most], pad: behind all rows
    q = torch.cat((s["q"], s["q"].new_zeros(1, H * D)))[t].view(B, most, Hkv, H // Hkv, D)
    q = q.permute(0, 2, 3, 1, 4).reshape(B, Hkv, H // Hkv * most, D)
    sc = torch.matmul(q, k.transpose(2, 3).contiguous()).mul_(1 / math.sqrt(D))
    sc = sc.view(B, Hkv, H // Hkv, most, n)
    last = s["lens"].long()[:, None] - rows[:, None] + i       # the row's own position
    hide = torch.arange(n, device=DEV) > last[:, :, None]
    sc.masked_fill_(hide[:, None, None], -math.inf)
    p = sc.sub_(sc.amax(-1, keepdim=True)).exp_()
    p = (p / p.sum(-1, keepdim=True)).view(B, Hkv, -1, n)
    o = torch.matmul(p, v).view(B, H, most, D).transpose(1, 2).reshape(B, most, H * D)
    out = torch.cat((s["out"], s["out"].new_zeros(1, H * D)))
    out = out.index_put((t,), torch.where(live[..., None], o, 0.0))
    return out[:-1]


def _exact_attention(case, seed):
    s = _prep_attention(case, seed)
    bs, H, Hkv, D = (case[n] for n in ("bs", "H", "Hkv", "D"))
    cached, added = _lengths(case)
    out = torch.zeros(len(s["q"]), H, D, device=DEV, dtype=F64)
    at = 0
    for b, (c, a) in enumerate(zip(cached, added)):
        if a == 0:
            continue
        own_blocks = s["tables"][b, :_blocks(c + a, bs)].long()
        q = s["q"][at:at + a].to(F64).view(a, H, D)
        see = torch.arange(c + a, device=DEV)[None] <= c + torch.arange(a, device=DEV)[:, None]
        for h in range(Hkv):
            x = s["codes"][own_blocks, :, h].to(F64) * s["scales"][own_blocks, :, h].to(F64)[..., None]
            k = x[:, 0].reshape(-1, D)[:c + a]
            v = x[:, 1].view(-1, D, bs).transpose(1, 2).reshape(-1, D)[:c + a]
            for i in range(h * (H // Hkv), (h + 1) * (H // Hkv)):
                w = torch.where(see, q[:, i] @ k.T / math.sqrt(D), -math.inf)
                out[at:at + a, i] = torch.softmax(w, -1) @ v
        at += a
    return out.flatten(1)


def _work_attention(case):
    cached, added = _lengths(case)
    H, Hkv, D, bs = (case[n] for n in ("H", "Hkv", "D", "bs"))
    live = [(c, a) for c, a in zip(cached, added) if a]
    keys = sum(c + a for c, a in live)
    blocks = sum(_blocks(c + a, bs) for c, a in live)
    pairs = sum(a * c + a * (a + 1) // 2 for c, a in live)     # (row, visible key)
    return dict(bytes=8 * sum(added) * H * D + 2 * keys * Hkv * D + blocks * (8 * Hkv + 4),
                flops=4 * H * D * pairs)


_PREPARE = dict(tables=_prep_tables, append=_prep_append, read=_prep_read,
                attention=_prep_attention)
_RUN = dict(tables=_run_tables, append=_run_append, read=_run_read, attention=_run_attention)
_WORK = dict(tables=_work_tables, append=_work_append, read=_work_read, attention=_work_attention)
_EXACT = dict(tables=lambda case, seed: None, append=_exact_append, read=_exact_read,
              attention=_exact_attention)
