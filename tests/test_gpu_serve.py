"""The serving operators (include/b200serve.h) on the device against the plain implementations of tests/serve_oracle.py."""
import math

import numpy as np
import pytest
import torch

import serve_oracle as so
from gpu_util import dev, empty, host, ops, pkg, sync

pytestmark = pytest.mark.gpu


def i32(x):
    return torch.tensor(np.asarray(x), dtype=torch.int32, device="cuda")


def workspace(query, *sizes, fill=0xff):
    size = np.zeros(1, np.uint64)
    query(*sizes, size.ctypes.data)
    return torch.full((int(size[0]),), fill, dtype=torch.uint8, device="cuda")


# ---- plan ----------------------------------------------------------------------------------
def run_plan(ctx, new, held, table, page, pool, ring, at, max_rows, in_place):
    B = len(ctx)
    c, n, h, t, rg = i32(ctx), i32(new), i32(held), dev(np.asarray(table, np.int32)), dev(np.asarray(ring, np.int32))
    a = torch.tensor(at, dtype=torch.int64, device="cuda")
    lens, ho, ao = (c, h, a) if in_place else (empty(B, torch.int32), empty(B, torch.int32), torch.zeros(2, dtype=torch.int64, device="cuda"))
    off, pos, slots, counts = empty(B + 1, torch.int32), empty(max_rows, torch.int32), empty(max_rows, torch.int32), empty(4, torch.int32)
    ops.paged_plan(c, n, h, B, t, t.shape[1] if B else 1, page, pool, rg, len(ring), a, ao, lens, ho, off, pos, slots, max_rows, counts)
    return dict(seq_lens=host(lens), held=host(ho), offsets=host(off), positions=host(pos), slots=host(slots), at=host(ao), counts=host(counts),
                table=host(t), ring=host(rg))


PLANS = [(1, 64, 9, 3, 40), (3, 1, 30, 4, 60), (5, 16, 12, 5, 4000), (64, 17, 9, 30, 300), (65, 8, 20, 3, 100), (700, 16, 40, 200, 60000),
         (2048, 4, 6, 9, 9000), (2047, 3, 8, 2, 1500)]


@pytest.mark.parametrize("in_place", [False, True])
@pytest.mark.parametrize("batch,page,cap,most,max_rows", PLANS)
def test_plan(batch, page, cap, most, max_rows, in_place):
    r = np.random.default_rng(batch * 7 + page)
    for tight in (False, True):
        ctx = r.integers(0, cap * page + 1, batch)
        held = np.minimum(-(-ctx // page) + r.integers(0, 2, batch), cap)
        new = np.where(r.random(batch) < 0.15, -1, r.integers(0, most + 1, batch))
        used = int(held.sum())
        free = int(r.integers(1, 8)) if tight else batch * (most // page + 2)
        pool = used + free
        order = r.permutation(pool)
        table = np.full((batch, cap), -5)
        table[np.arange(cap)[None] < held[:, None]] = order[:used]
        head = int(r.integers(0, 10)) * pool + int(r.integers(0, pool))
        ring = np.full(pool + 3, -9)
        ring[(np.arange(free) + head) % len(ring)] = order[used:]
        want_table, want_ring = table.copy(), ring.copy()
        want = so.plan(ctx, new, held, want_table, cap, page, pool, want_ring, [head, head + free], max_rows)
        got = run_plan(ctx, new, held, table, page, pool, ring, [head, head + free], max_rows, in_place)
        for k in want:
            assert np.array_equal(got[k], want[k]), (k, tight)
        assert np.array_equal(got["table"], want_table) and np.array_equal(got["ring"], want_ring)


def test_plan_of_nothing_and_of_bad_numbers():
    got = run_plan([], [], [], np.zeros((0, 1)), 16, 4, [0, 1, 2, 3], [0, 4], 5, False)
    assert got["offsets"].tolist() == [0] and got["positions"].tolist() == [-1] * 5 and got["counts"].tolist() == [0] * 4
    # held beyond the table, a negative context, sums beyond 32 bits, page ids that are none, a ring out of order
    big = 2 ** 31 - 1
    ctx, new, held = [5, -3, big, 0, 7, 0], [big, 4, 2, 3, 1, 2], [1, 0, 0, 99, 1, 0]
    for at in ([0, 4], [3, 1], [-1, 2], [0, 9]):
        table, ring = np.full((6, 4), 77), np.array([2, -1, 50, 3])
        wt, wr = table.copy(), ring.copy()
        want = so.plan(ctx, new, held, wt, 4, 4, 4, wr, at, 8)
        got = run_plan(ctx, new, held, table, 4, 4, ring, at, 8, False)
        for k in want:
            assert np.array_equal(got[k], want[k]), (k, at)
        assert np.array_equal(got["table"], wt) and np.array_equal(got["ring"], wr)


# ---- rope ------------------------------------------------------------------------------------
# cos and sin are rounded to fp32 (2^-24 of 1 at most each, the argument's first-order rest included 2^-23), then two products and
# a sum: at most 2^-22 of |a| + |b| times the factor.
ROPE_TOL = 2.0 ** -22


@pytest.mark.parametrize("scaling", range(5))
@pytest.mark.parametrize("rot", [2, 6, 64, 128])
def test_rope_frequencies(rot, scaling):
    f = torch.zeros(rot // 2 + 1, dtype=torch.float64, device="cuda")
    factor = np.zeros(1)
    low, high = (1.0, 32.0) if scaling == 3 else (1.0, 4.0)
    ops.rope_frequencies(f, rot, 1e4, scaling, 8.0, 4096, low, high, factor.ctypes.data)
    want = so.frequencies(rot, 1e4, scaling, 8.0, 4096, low, high)
    np.testing.assert_allclose(host(f)[:-1], want, rtol=1e-13)
    assert host(f)[-1] == 0 and abs(factor[0] - (1 + 0.1 * math.log(8) if scaling == 3 else 1)) < 1e-15


@pytest.mark.parametrize("rope_type", [0, 1])
@pytest.mark.parametrize("n,H,KV,hd,rot,pad", [(1, 4, 2, 64, 64, 0), (3, 12, 4, 128, 96, 0), (300, 3, 1, 64, 24, 4), (5, 2, 2, 80, 6, 0), (7, 5, 1, 128, 64, 3),
                                               (700, 32, 8, 128, 64, 0), (2, 1, 1, 1024, 1024, 0), (9, 4, 4, 34, 34, 1), (4, 2, 1, 64, 4, 0)])
def test_rope(rope_type, n, H, KV, hd, rot, pad):
    r = np.random.default_rng(n + hd)
    freq = so.frequencies(rot, 1e4, 3, 8.0, 4096, 1.0, 32.0)
    pos = r.integers(0, 1 << 20, n)
    pos[0] = 2 ** 26                                   # where a 64-bit angle is still good to 2^-27
    if n > 1:
        pos[n // 2] = -1
    # queries and keys inside one projection's rows, as split by views
    row = (H + 2 * KV) * hd + pad
    x = r.standard_normal((n, row)).astype(np.float32)
    q, k = x[:, :H * hd].reshape(n, H, hd), x[:, H * hd:(H + KV) * hd].reshape(n, KV, hd)
    live = pos >= 0
    want = [so.rope(t, np.maximum(pos, 0), freq, rot, rope_type, 1.2) for t in (q, k)]
    f, p, src = torch.tensor(freq, device="cuda"), i32(pos), dev(x)
    qo, ko = empty((n, H * hd + pad)), empty((n, KV * hd))
    ops.rope_forward_scaled(src, src[:, H * hd:], qo, ko, p, f, n, H, KV, hd, rot, rope_type, row, row, H * hd + pad, KV * hd, 1.2)
    for got, w, t in ((qo[:, :H * hd].reshape(n, H, hd), want[0], q), (ko.reshape(n, KV, hd), want[1], k)):
        got = host(got)
        assert np.isnan(got[~live]).all()                              # rows without a position are left as they were
        pair = 1.2 * np.sqrt(2) * np.abs(t).max()
        assert np.abs(got[live] - w[live]).max() <= 2 * ROPE_TOL * pair
        assert np.array_equal(got[live][..., rot:], t[live][..., rot:])
    assert pad == 0 or torch.isnan(qo[:, H * hd:]).all()
    # in place, and one of the two alone
    both = dev(x)
    ops.rope_forward_scaled(both, both[:, H * hd:], both, both[:, H * hd:], p, f, n, H, KV, hd, rot, rope_type, row, row, row, row, 1.2)
    assert torch.equal(both[live][:, :H * hd], qo[live][:, :H * hd]) and torch.equal(both[live][:, H * hd:(H + KV) * hd], ko[live])
    assert torch.equal(both[:, (H + KV) * hd:], src[:, (H + KV) * hd:]) and torch.equal(both[~live], src[~live])
    alone = empty((n, KV, hd))
    ops.rope_forward_scaled(None, src[:, H * hd:], None, alone, p, f, n, 0, KV, hd, rot, rope_type, 0, row, 0, KV * hd, 1.2)
    assert torch.equal(alone[live].reshape(-1, KV * hd), ko[live])


def test_rope_into_other_columns_of_the_same_rows():
    r = np.random.default_rng(6)
    x = r.standard_normal((5, 400)).astype(np.float32)
    buf, f, p = dev(x), torch.tensor(so.frequencies(16, 1e4, 0, 1.0, 1, 1.0, 2.0), device="cuda"), i32([3, 1, 4, 1, 5])
    ops.rope_forward_scaled(buf, None, buf[:, 130:], None, p, f, 5, 2, 0, 64, 16, 1, 400, 0, 400, 0, 1.0)
    got = host(buf)
    want = so.rope(x[:, :128].reshape(5, 2, 64), [3, 1, 4, 1, 5], host(f), 16, 1, 1.0).reshape(5, 128)
    assert np.abs(got[:, 130:258] - want).max() <= 4 * ROPE_TOL * np.abs(x).max()
    assert np.array_equal(got[:, :130], x[:, :130]) and np.array_equal(got[:, 258:], x[:, 258:])


def test_rope_agrees_with_the_cached_form():
    """Unscaled, whole head: the framework's own rotation up to its fp32 angle (2^-24 of the angle, here at most 500)."""
    r = np.random.default_rng(5)
    q, k = r.standard_normal((6, 4, 64)).astype(np.float32), r.standard_normal((6, 2, 64)).astype(np.float32)
    f32 = (1e4 ** (-np.arange(32) / 32.0)).astype(np.float32)
    p = i32(r.integers(0, 500, 6))
    for t in (0, 1):
        a, b = dev(q), dev(k)
        ops.rope_forward_cached(a, b, p, dev(f32), 6, 4, 2, 64, t)
        c, d = empty((6, 4, 64)), empty((6, 2, 64))
        ops.rope_forward_scaled(dev(q), dev(k), c, d, p, torch.tensor(f32.astype(np.float64), device="cuda"), 6, 4, 2, 64, 64, t, 256, 128, 256, 128, 1.0)
        for x, y in ((a, c), (b, d)):
            assert float((x - y).abs().max()) <= (500 * 2.0 ** -24 + 4 * ROPE_TOL) * 2 * float(np.abs(q).max())


# ---- the cache ---------------------------------------------------------------------------------
def tricky_rows(r, n, KV, hd):
    x = (r.standard_normal((n, KV, hd)) * np.exp(r.standard_normal((n, KV, 1)))).astype(np.float32)
    x[0, 0, :32] = 0
    x[n // 2, 0, 3] = np.nan
    x[n // 3, KV - 1, hd - 1] = -np.inf
    x[-1, 0, 32:64] = 3.0
    x[-1, -1, 5] = 3e38
    x[-1, -1, 6] = -3e38
    x[n // 4, 0, 0] = 1e-42
    return x


@pytest.mark.parametrize("kind", [0, 1])
@pytest.mark.parametrize("n,page,KV,hd,pad", [(1, 1, 1, 64, 0), (5, 16, 4, 64, 0), (64, 64, 4, 128, 8), (37, 33, 3, 128, 3), (300, 7, 8, 128, 0), (3, 256, 33, 64, 0)])
def test_store_and_fetch(kind, n, page, KV, hd, pad):
    r = np.random.default_rng(n + page)
    num_pages = n // page + 3
    k, v = tricky_rows(r, n, KV, hd), tricky_rows(r, n, KV, hd)[::-1].copy()
    slots = r.permutation(num_pages * page)[:n]
    if n > 4:
        slots[1], slots[2] = -1, num_pages * page              # in no page
    cache = so.Cache(num_pages, page, KV, hd, kind, fill=0xA5)
    pages = dev(cache.bytes)
    cache.store(k, v, slots)
    row = KV * hd + pad
    src = [torch.full((n, row), 7.0, device="cuda") for _ in range(2)]
    for s, x in zip(src, (k, v)):
        s[:, :KV * hd] = dev(x.reshape(n, -1))
    ops.kv4_store(src[0], src[1], row, row, i32(slots), n, pages, num_pages, page, KV, hd, kind)
    assert np.array_equal(host(pages), cache.bytes)            # other tokens, padding and all
    live = (slots >= 0) & (slots < num_pages * page)
    wk, wv = cache.rows(slots[live])
    for stride, both in ((row, True), (KV * hd + 1, True), (row, False)):
        gk, gv = empty((n, stride)), empty((n, stride))
        ops.kv4_fetch(pages, num_pages, page, i32(slots), n, gk if both else None, gv, stride, stride, KV, hd, kind)
        # d * code + m: one rounding of the sum, the product is exact
        for got, want in ((gk, wk), (gv, wv)) if both else ((gv, wv),):
            got = host(got)
            assert np.array_equal(got[live][:, :KV * hd].reshape(-1, KV, hd), want.astype(np.float32))
            assert np.isnan(got[~live]).all() and np.isnan(got[:, KV * hd:]).all()
        assert both or torch.isnan(gk).all()


@pytest.mark.parametrize("kind", [0, 1])
@pytest.mark.parametrize("n,page,KV,hd,pad", [(4801, 16, 1, 64, 0), (1603, 64, 3, 64, 1), (811, 32, 5, 128, 4), (2051, 128, 2, 128, 3)])
def test_store_of_many_rows(kind, n, page, KV, hd, pad):
    """Enough rows that a thread has K and V of one; half of them have values halfway between codes."""
    r = np.random.default_rng(n)
    num_pages = n // page + 2
    k, v = tricky_rows(r, n, KV, hd), tricky_rows(r, n, KV, hd)[::-1].copy()
    k[1::2] = r.integers(-16, 17, k[1::2].shape) / 2.0 * 2.0 ** r.integers(-20, 20, (len(k[1::2]), KV, 1))
    v[1::2] = r.integers(0, 31, v[1::2].shape) / 2.0
    slots = r.permutation(num_pages * page)[:n]
    slots[n // 2], slots[n - 2] = -7, num_pages * page + 5
    cache = so.Cache(num_pages, page, KV, hd, kind, fill=0x5A)
    pages = dev(cache.bytes)
    cache.store(k, v, slots)
    row = KV * hd + pad
    src = [torch.full((n, row), 7.0, device="cuda") for _ in range(2)]
    for s, x in zip(src, (k, v)):
        s[:, :KV * hd] = dev(x.reshape(n, -1))
    ops.kv4_store(src[0], src[1], row, row, i32(slots), n, pages, num_pages, page, KV, hd, kind)
    assert np.array_equal(host(pages), cache.bytes)


# ---- attention -----------------------------------------------------------------------------------
def make_cache(r, lens, page, KV, hd, kind, scale=1.0):
    """A cache in host memory with rows of about unit size in the pages of len(lens) sequences, junk everywhere else."""
    need = [-(-n // page) for n in lens]
    pool = sum(need) + 3
    cache = so.Cache(pool, page, KV, hd, kind, fill=0xff)                     # an fp16 0xffff is a NaN
    order = r.permutation(pool)
    table = np.full((len(lens), max(max(need), 1) + 1), -1)
    at = 0
    for b, p in enumerate(need):
        table[b, :p] = order[at:at + p]
        at += p
    kv = []
    nb, w = hd // 32, 2 if kind == 1 else 1
    for b, n in enumerate(lens):
        slots = table[b, np.arange(n) // page] * page + np.arange(n) % page
        p, off = np.divmod(slots, page)
        for c, s in ((cache.parts[0], cache.parts[1]), (cache.parts[2], cache.parts[3])):
            codes = r.integers(0, 256, (n, KV, hd // 2)).astype(np.uint8)
            d = 0.2 * np.exp(0.5 * r.standard_normal((n, KV, nb, 1))) * scale
            sc = np.concatenate([d, -7.5 * d + 0.2 * scale * r.standard_normal(d.shape)], -1) if kind == 1 else d
            sc = np.clip(sc, -65504, 65504).astype(np.float16)      # as everything that has been stored
            for h in range(KV):
                row = h * page + off
                cache.bytes[p[:, None], c + row[:, None] * hd // 2 + np.arange(hd // 2)] = codes[:, h]
                cache.bytes[p[:, None], s + row[:, None] * nb * 2 * w + np.arange(nb * 2 * w)] = np.ascontiguousarray(sc[:, h]).view(np.uint8).reshape(n, nb * 2 * w)
        kv.append(cache.rows(slots) if n else (np.zeros((0, KV, hd)), np.zeros((0, KV, hd))))
    return cache, table, kv


def call_attention(q, qs, offsets, pages, num_pages, table, lens, out, os_, max_rows, page, H, KV, hd, kind, scale, window, work=None):
    work = workspace(ops.attention_paged_kv4_workspace, H, KV, hd, max_rows) if work is None else work
    ops.attention_paged_kv4(q, qs, offsets, pages, num_pages, table, lens, out, os_, len(lens), max_rows, table.shape[1], page, H, KV, hd,
                            kind, scale, window, work, work.numel())
    return work


def attention_bound(q, kv, scale):
    """How far an element may be off.  A score is a sum of hd products of a query (two fp16 parts: 2^-23) with d * code + m, formed as
    d * (sum of q code) + m * (sum of q), added in pieces of 32 on the tensor cores (which may cut, 2^-23 each, two in a row) and fp32 (five in a
    row): 2^-20 of the sum of |q| (|d| code + |m|), at most twice |q| (15 |d| + |m|) <= 3 |q| max|k|.  A weight is off by
    that and 2^-21 of exp; the average moves by at most twice the weights' error times max|v|, and the sums over
    the keys (three roundings of tiles, 64 a row per lane at most, 2^-24 of each in the worst case) add 2^-18 max|v|."""
    A = max([scale * np.abs(q).sum(-1).max() * np.abs(k).max() * 3 for k, _ in kv if len(k)] or [0])
    V = max([np.abs(v).max() for _, v in kv if len(v)] or [0])
    return (2 * (2.0 ** -20 * A + 2.0 ** -21) + 2.0 ** -18) * V


CASES = [  # H, KV, hd, page, lens, rows
    (4, 4, 64, 16, [1], [1]),
    (12, 4, 64, 64, [0, 5, 17, 1], [1, 1, 1, 1]),
    (12, 4, 128, 64, [33, 64, 65, 129, 200], [1, 1, 1, 1, 1]),
    (32, 8, 128, 16, [1000, 3, 511], [1, 1, 1]),
    (8, 1, 128, 5, [77, 300], [1, 1]),
    (5, 1, 64, 1, [40, 129], [1, 2]),
    (12, 4, 64, 48, [130, 700], [5, 3]),
    (32, 8, 128, 64, [600, 65, 128, 9], [5, 6, 1, 9]),
    (16, 2, 128, 33, [100, 2, 300], [13, 5, 0]),
    (12, 4, 128, 64, [4097], [1]),
    (4, 1, 128, 128, [5000], [4]),
    (12, 4, 64, 64, [300, 150, 70], [170, 150, 33]),
    (32, 8, 128, 16, [180, 260], [100, 70]),
    (3, 3, 128, 16, [90, 31, 32], [1, 2, 31]),
    (64, 1, 64, 16, [333], [2]),
    (24, 1, 128, 100, [333, 1], [3, 1]),
]


@pytest.mark.parametrize("kind", [0, 1])
@pytest.mark.parametrize("window", [0, 1, 100])
@pytest.mark.parametrize("case", range(len(CASES)))
def test_attention(case, kind, window):
    H, KV, hd, page, lens, rows = CASES[case]
    r = np.random.default_rng(case)
    cache, table, kv = make_cache(r, lens, page, KV, hd, kind)
    n, scale = sum(rows), 1 / math.sqrt(hd)
    offsets = np.concatenate([[0], np.cumsum(rows)])
    q = r.standard_normal((n + 2, H, hd)).astype(np.float32) * np.exp(r.standard_normal((n + 2, H, 1))).astype(np.float32)
    row, orow = (H + KV) * hd, H * hd + 4                        # queries inside a wider projection
    src = torch.full((n + 2, row), float("nan"), device="cuda")
    src[:, :H * hd] = dev(q.reshape(n + 2, -1))
    out = empty((n + 2, orow))
    call_attention(src, row, i32(offsets), dev(cache.bytes), cache.num_pages, i32(table), i32(lens), out, orow, max(rows), page, H, KV, hd, kind,
                   scale, window)
    got = host(out)
    assert np.isnan(got[n:]).all() and np.isnan(got[:, H * hd:]).all()       # rows of no sequence, and between the rows
    got = got[:n, :H * hd].reshape(n, H, hd).astype(np.float64)
    want = np.concatenate([so.attention(q, offsets[b], rows[b], lens[b], *kv[b], scale, window) for b in range(len(lens))])
    assert np.abs(got - want).max() <= attention_bound(q, kv, scale)
    # errors of either sign over many terms: of the whole, eight roundings' worth of the 23 bits that q and p have
    assert np.linalg.norm(got - want) <= 8 * 2.0 ** -23 * max(np.linalg.norm(want), 1e-30) * max(1.0, np.abs(q).max() / 3)
    if not any(rows[b] > lens[b] for b in range(len(lens))):
        return
    early = [offsets[b] + i for b in range(len(lens)) for i in range(rows[b]) if lens[b] - rows[b] + i < 0]
    assert (got[early] == 0).all()


def test_attention_of_one_row_each_needs_no_offsets():
    r = np.random.default_rng(50)
    lens = [10, 0, 300]
    cache, table, kv = make_cache(r, lens, 16, 2, 128, 1)
    q = r.standard_normal((3, 8, 128)).astype(np.float32)
    a, b = empty((3, 8, 128)), empty((3, 8, 128))
    args = (dev(cache.bytes), cache.num_pages, i32(table), i32(lens))
    call_attention(dev(q), 1024, None, *args, a, 1024, 1, 16, 8, 2, 128, 1, 0.1, 0)
    call_attention(dev(q), 1024, i32([0, 1, 2, 3]), *args, b, 1024, 1, 16, 8, 2, 128, 1, 0.1, 0)
    assert torch.equal(a, b) and (a[1] == 0).all()


@pytest.mark.parametrize("kind", [0, 1])
def test_attention_of_sharp_flat_and_scaled_scores(kind):
    """Scores of hundreds (one key takes all), of zero (the plain average), values of 1e-4 and of 1e4."""
    r = np.random.default_rng(51)
    H, KV, hd, page, lens = 8, 2, 128, 16, [700, 65]
    for qscale, cscale in ((60.0, 1.0), (0.0, 1.0), (1.0, 1e-4), (1e-4, 1e4), (1e5, 1e-4)):
        cache, table, kv = make_cache(r, lens, page, KV, hd, kind, cscale)
        q = (r.standard_normal((2, H, hd)) * qscale).astype(np.float32)
        out = empty((2, H, hd))
        call_attention(dev(q), H * hd, None, dev(cache.bytes), cache.num_pages, i32(table), i32(lens), out, H * hd, 1, page, H, KV, hd, kind, 0.088, 0)
        want = np.concatenate([so.attention(q, b, 1, lens[b], *kv[b], np.float32(0.088), 0) for b in range(2)])
        assert np.abs(host(out) - want).max() <= attention_bound(q, kv, 0.088), (qscale, cscale)


def test_attention_with_scales_far_apart():
    """One block of 32 dims, and one token in each page, with scales 2^12 times the others'."""
    r = np.random.default_rng(52)
    H, KV, hd, page, lens, kind = 4, 1, 64, 16, [200], 1
    cache, table, _ = make_cache(r, lens, page, KV, hd, kind)
    nb = hd // 32
    view = cache.bytes[:, cache.parts[3]:cache.parts[3] + page * nb * 4]
    s = np.ascontiguousarray(view).view(np.float16).reshape(-1, page, nb, 2).copy()
    s[:, 3] *= 64
    s[:, :, 1] *= 64
    s[~np.isfinite(s)] = 0
    cache.bytes[:, cache.parts[3]:cache.parts[3] + page * nb * 4] = s.reshape(len(s), -1).view(np.uint8)
    slots = table[0, np.arange(200) // page] * page + np.arange(200) % page
    k, v = cache.rows(slots)
    q = r.standard_normal((1, H, hd)).astype(np.float32)
    out = empty((1, H, hd))
    call_attention(dev(q), H * hd, None, dev(cache.bytes), cache.num_pages, i32(table), i32(lens), out, H * hd, 1, page, H, KV, hd, kind, 0.125, 0)
    want = so.attention(q, 0, 1, 200, k, v, 0.125, 0)
    for blk in range(nb):                                       # each block of dims to its own size
        part = np.s_[..., 32 * blk:32 * blk + 32]
        assert np.abs(host(out)[part] - want[part]).max() <= attention_bound(q, [(k, v[part])], 0.125)


def test_attention_keeps_a_bad_row_to_itself():
    """NaN and infinite queries spoil their own row and head; tokens after a row may hold anything finite, pages of no one NaNs."""
    r = np.random.default_rng(53)
    H, KV, hd, page, lens, rows = 8, 2, 64, 16, [90, 40], [6, 3]
    cache, table, kv = make_cache(r, lens, page, KV, hd, 1)
    q = r.standard_normal((9, H, hd)).astype(np.float32)
    q[2, 3, 5], q[4, 0, 1], q[7, 7, 63] = np.nan, np.inf, -np.inf
    offs = np.array([0, 6, 9])
    out = empty((9, H, hd))
    call_attention(dev(q), H * hd, i32(offs), dev(cache.bytes), cache.num_pages, i32(table), i32(lens), out, H * hd, 6, page, H, KV, hd, 1, 0.125, 0)
    got = host(out)
    clean = np.where(np.isfinite(q), q, 0).astype(np.float32)
    want = np.concatenate([so.attention(clean, offs[b], rows[b], lens[b], *kv[b], 0.125, 0) for b in range(2)])
    for i in range(9):
        for h in range(H):
            if np.isfinite(q[i, h]).all():
                assert np.abs(got[i, h] - want[i, h]).max() <= attention_bound(clean, kv, 0.125)
            else:
                assert not np.isfinite(got[i, h]).any() or not np.isfinite(q[i, h]).all()
    assert np.isnan(got[2, 3]).all()


def test_attention_reads_pages_of_no_one_as_zeros_and_cuts_long_lengths():
    r = np.random.default_rng(54)
    H, KV, hd, page, lens = 4, 2, 64, 16, [64, 100]
    cache, table, kv = make_cache(r, lens, page, KV, hd, 0)
    table = table[:, :6]                                        # the second holds 96 of its 100 tokens
    table[0, 1] = cache.num_pages
    table[0, 2] = -2 ** 31
    k, v = (x.copy() for x in kv[0])
    k[16:48], v[16:48] = 0, 0
    q = r.standard_normal((2, H, hd)).astype(np.float32)
    out = empty((2, H, hd))
    call_attention(dev(q), H * hd, None, dev(cache.bytes), cache.num_pages, i32(table), i32([64, 100]), out, H * hd, 1, page, H, KV, hd, 0, 0.125, 0)
    want = np.concatenate([so.attention(q, 0, 1, 64, k, v, 0.125, 0), so.attention(q, 1, 1, 96, kv[1][0][:96], kv[1][1][:96], 0.125, 0)])
    assert np.abs(host(out) - want).max() <= attention_bound(q, [(k, v), kv[1]], 0.125)


def test_attention_far_into_a_large_pool():
    """Pages beyond 4 GB from the pool's start."""
    r = np.random.default_rng(55)
    H, KV, hd, page, lens = 32, 8, 128, 64, [150, 90]
    cache, table, kv = make_cache(r, lens, page, KV, hd, 1)
    far = 60000
    pages = torch.zeros((far + cache.num_pages, cache.bytes.shape[1]), dtype=torch.uint8, device="cuda")
    assert pages.numel() > 2 ** 32
    pages[far:] = dev(cache.bytes)
    table = np.where(table >= 0, table + far, -1)
    q = r.standard_normal((2, H, hd)).astype(np.float32)
    out = empty((2, H, hd))
    call_attention(dev(q), H * hd, None, pages, len(pages), i32(table), i32(lens), out, H * hd, 1, page, H, KV, hd, 1, 0.1, 0)
    want = np.concatenate([so.attention(q, b, 1, lens[b], *kv[b], np.float32(0.1), 0) for b in range(2)])
    assert np.abs(host(out) - want).max() <= attention_bound(q, kv, 0.1)
    # stored and fetched there too
    x = r.standard_normal((2, KV, hd)).astype(np.float32)
    slots = [(far + 1) * page + 3, (far + cache.num_pages) * page - 1]
    a, b = empty((2, KV, hd)), empty((2, KV, hd))
    ops.kv4_store(dev(x), dev(-x), KV * hd, KV * hd, i32(slots), 2, pages, len(pages), page, KV, hd, 1)
    ops.kv4_fetch(pages, len(pages), page, i32(slots), 2, a, b, KV * hd, KV * hd, KV, hd, 1)
    assert np.array_equal(host(a), so.values(*so.quantize(x, 1), 1).astype(np.float32))
    assert np.array_equal(host(b), so.values(*so.quantize(-x, 1), 1).astype(np.float32))


@pytest.mark.parametrize("kind", [0, 1])
def test_attention_of_a_long_context(kind):
    """70 001 tokens of one sequence beside short ones: hundreds of pieces of one item."""
    r = np.random.default_rng(62)
    H, KV, hd, page, lens, rows = 4, 1, 128, 64, [70001, 3, 500], [2, 1, 1]
    cache, table, kv = make_cache(r, lens, page, KV, hd, kind)
    q, offs = r.standard_normal((4, H, hd)).astype(np.float32), np.array([0, 2, 3, 4])
    out = empty((4, H, hd))
    call_attention(dev(q), H * hd, i32(offs), dev(cache.bytes), cache.num_pages, i32(table), i32(lens), out, H * hd, 2, page, H, KV, hd, kind, 0.088, 0)
    want = np.concatenate([so.attention(q, offs[b], rows[b], lens[b], *kv[b], np.float32(0.088), 0) for b in range(3)])
    got = host(out).astype(np.float64)
    assert np.abs(got - want).max() <= attention_bound(q, kv, 0.088)
    # the long one alone, whose values average out to a hundredth: in its own size.  A weight is off by 2^-21 at most, with either sign
    assert np.linalg.norm(got[:2] - want[:2]) <= 2.0 ** -19 * np.linalg.norm(want[:2])


def test_attention_with_a_window_beyond_every_length():
    r = np.random.default_rng(59)
    lens, rows = [70, 5], [3, 9]                               # more rows than tokens, too
    cache, table, kv = make_cache(r, lens, 16, 2, 64, 1)
    q, offs = dev(r.standard_normal((12, 4, 64)).astype(np.float32)), i32([0, 3, 12])
    got = []
    for window in (0, 2 ** 31 - 1, 96, -5):
        out = empty((12, 4, 64))
        call_attention(q, 256, offs, dev(cache.bytes), cache.num_pages, i32(table), i32(lens), out, 256, 9, 16, 4, 2, 64, 1, 0.125, window)
        got.append(out)
    assert all(torch.equal(got[0], o) for o in got[1:]) and (got[0][3:7] == 0).all()


def test_attention_of_many_sequences():
    """More sequences than a block has threads, many of them without rows or tokens."""
    r = np.random.default_rng(61)
    B, H, KV, hd, page = 700, 4, 2, 64, 16
    lens = [int(x) for x in r.integers(0, 90, B)]
    rows = [int(x) for x in r.choice([0, 0, 1, 2], B)]
    rows[-3:] = [0, 0, 0]
    cache, table, kv = make_cache(r, lens, page, KV, hd, 0)
    offs = np.concatenate([[0], np.cumsum(rows)])
    q = r.standard_normal((int(offs[-1]), H, hd)).astype(np.float32)
    out = empty(q.shape)
    call_attention(dev(q), H * hd, i32(offs), dev(cache.bytes), cache.num_pages, i32(table), i32(lens), out, H * hd, 2, page, H, KV, hd, 0, 0.125, 0)
    want = np.concatenate([so.attention(q, offs[b], rows[b], lens[b], *kv[b], 0.125, 0) for b in range(B)])
    assert np.abs(host(out) - want).max() <= attention_bound(q, kv, 0.125)


def test_attention_is_the_same_every_time():
    """Whatever the workspace held, and whatever else is in the batch's order of blocks: the same bits twice."""
    r = np.random.default_rng(56)
    lens, rows = [3000, 40, 900, 1], [2, 2, 2, 1]
    cache, table, _ = make_cache(r, lens, 64, 4, 128, 1)
    q, offs = dev(r.standard_normal((7, 12, 128)).astype(np.float32)), i32([0, 2, 4, 6, 7])
    got = []
    for fill in (0, 0xff, 0x3c):
        out = empty((7, 12, 128))
        work = workspace(ops.attention_paged_kv4_workspace, 12, 4, 128, 2, fill=fill)
        call_attention(q, 1536, offs, dev(cache.bytes), cache.num_pages, i32(table), i32(lens), out, 1536, 2, 64, 12, 4, 128, 1, 0.088, 0, work)
        call_attention(q, 1536, offs, dev(cache.bytes), cache.num_pages, i32(table), i32(lens), out, 1536, 2, 64, 12, 4, 128, 1, 0.088, 0, work)
        got.append(out)
    assert torch.equal(got[0], got[1]) and torch.equal(got[0], got[2])


def test_attention_with_more_rows_than_it_was_told():
    r = np.random.default_rng(57)
    lens, rows = [200, 50], [40, 3]
    cache, table, kv = make_cache(r, lens, 16, 2, 64, 0)
    q, offs = r.standard_normal((43, 6, 64)).astype(np.float32), np.array([0, 40, 43])
    out = empty((43, 6, 64))
    call_attention(dev(q), 384, i32(offs), dev(cache.bytes), cache.num_pages, i32(table), i32(lens), out, 384, 1, 16, 6, 2, 64, 0, 0.125, 0)
    want = np.concatenate([so.attention(q, offs[b], rows[b], lens[b], *kv[b], 0.125, 0) for b in range(2)])
    assert np.abs(host(out) - want).max() <= attention_bound(q, kv, 0.125)


def test_attention_captured_with_lengths_that_change():
    """A graph of the call follows lengths, pages and offsets that are written between its replays; two graphs have a workspace each
    and run on two streams at once."""
    r = np.random.default_rng(58)
    H, KV, hd, page, kind = 12, 4, 64, 16, 1
    cache, table, _ = make_cache(r, [900, 700, 64], page, KV, hd, kind)
    pages, q = dev(cache.bytes), r.standard_normal((6, H, hd)).astype(np.float32)
    slots = [table[b, np.arange(n) // page] * page + np.arange(n) % page for b, n in enumerate([900, 700, 64])]
    kv = [cache.rows(s) for s in slots]
    made = []
    for _ in range(2):
        s = dict(q=dev(q), offs=i32([0, 1, 2, 3]), lens=i32([900, 700, 64]), out=empty((6, H, hd)), table=i32(table),
                 work=workspace(ops.attention_paged_kv4_workspace, H, KV, hd, 4), stream=torch.cuda.Stream(), graph=torch.cuda.CUDAGraph())
        torch.cuda.synchronize()
        pkg.lib().b200_set_stream(s["stream"].cuda_stream)
        try:
            with torch.cuda.graph(s["graph"], stream=s["stream"]):
                call_attention(s["q"], H * hd, s["offs"], pages, cache.num_pages, s["table"], s["lens"], s["out"], H * hd, 4, page, H, KV, hd, kind, 0.125, 0,
                               s["work"])
        finally:
            pkg.lib().b200_set_stream(None)
        made.append(s)
    for lens, rows in (([900, 700, 64], [1, 1, 1]), ([5, 0, 33], [4, 0, 2]), ([640, 699, 1], [2, 3, 1])):
        offs = np.concatenate([[0], np.cumsum(rows)])
        for s in made:
            s["lens"].copy_(i32(lens))
            s["offs"].copy_(i32(offs))
            s["out"].fill_(float("nan"))
        sync()
        for _ in range(3):
            for s in made:
                with torch.cuda.stream(s["stream"]):
                    s["graph"].replay()
        sync()
        want = np.concatenate([so.attention(q, offs[b], rows[b], lens[b], kv[b][0][:lens[b]], kv[b][1][:lens[b]], 0.125, 0) for b in range(3)])
        for s in made:
            assert np.abs(host(s["out"])[:offs[-1]] - want).max() <= attention_bound(q, kv, 0.125)
            assert torch.isnan(s["out"][int(offs[-1]):]).all()


# ---- drafted tokens ------------------------------------------------------------------------------
def run_verify(logits, draft, ids, offsets, T, u, K, rows=None, stride=0, dstride=0):
    B, V = len(offsets) - 1, logits.shape[1]
    def wide(x, s):
        t = torch.full((len(x), V + s), float("inf"), device="cuda")
        t[:, :V] = dev(x)
        return t
    l, d = wide(logits, stride), wide(draft, dstride) if draft is not None else None
    acc, tok = empty(B, torch.int32), empty((B, K + 1), torch.int32)
    rows = len(logits) if rows is None else rows
    work = workspace(ops.verify_drafts_workspace, rows, V)
    ops.verify_drafts(l, V + stride, d, V + dstride, i32(ids), i32(offsets), B, rows, V, T, dev(np.asarray(u, np.float32)), K, acc, tok, work, work.numel())
    return host(acc), host(tok)


def check_verify(logits, draft, ids, offsets, T, u, K, got):
    want = so.verify(logits, draft, ids, offsets, T, np.asarray(u, np.float32).astype(np.float64), K)
    for b, (n, cut, margin) in enumerate(want):
        # a weight is off by 2^-21 of itself at most, Z by as much
        assert margin > 2.0 ** -19, "the case checks a draft on the border"
        assert got[0][b] == n
        toks = got[1][b]
        assert list(toks[:n]) == list(ids[offsets[b] + 1:offsets[b] + 1 + n]) and (toks[n + 1:] == -1).all()
        if not isinstance(cut, tuple):
            assert toks[n] == cut
            continue
        masses, mark = cut
        sums, x = np.cumsum(masses), int(toks[n])
        assert 0 <= x < len(masses) and masses[x] > 0
        # cumulated masses: 2^-21 of all of p at most, were every weight off the same way
        slack = 2.0 ** -21
        assert sums[x] - masses[x] - slack <= mark <= sums[x] + slack


@pytest.mark.parametrize("T", [0.0, -1.0, 0.3, 1.0, 1.7])
@pytest.mark.parametrize("drafter", [False, True])
@pytest.mark.parametrize("V,counts,K,strides", [(1, [1, 2], 1, (0, 0)), (7, [3, 0, 1, 4], 3, (0, 1)), (1000, [5] * 9, 4, (0, 0)), (32768, [6, 1, 3, 2], 5, (4, 8)),
                                                (100352, [4, 5], 4, (0, 0)), (8193, [2, 3, 1], 2, (1, 0)), (50257, [9], 8, (3, 3)), (128, [1] * 40, 0, (0, 0))])
def test_verify(V, counts, K, strides, drafter, T):
    r = np.random.default_rng(V + len(counts))
    offsets = np.concatenate([[0], np.cumsum(counts)])
    n = int(offsets[-1])
    logits = (2 * r.standard_normal((n, V))).astype(np.float32)
    near = logits + 0.7 * r.standard_normal((n, V))
    q = np.exp((near - near.max(1, keepdims=True)) / max(T, 0.5))
    q = (q / q.sum(1, keepdims=True)).astype(np.float32)
    picks = np.array([int(r.choice(V, p=p.astype(np.float64) / p.astype(np.float64).sum())) for p in q]) if drafter and T > 0 else near.argmax(1)
    ids = np.concatenate([[0], picks[:-1]])
    u = r.random(n)
    draft = q if drafter else None
    check_verify(logits, draft, ids, offsets, T, u, K, run_verify(logits, draft, ids, offsets, T, u, K, stride=strides[0], dstride=strides[1]))


def test_verify_is_exact_on_flat_rows():
    """100 000 equal logits: the token drawn is floor(u V) to the border's 1e-9."""
    V, n = 100000, 64
    logits = np.full((n, V), 1.25, np.float32)
    u = (np.random.default_rng(7).integers(0, 2 ** 24, n) / 2.0 ** 24)
    u[0], u[1] = 0.0, 1 - 2.0 ** -24
    acc, tok = run_verify(logits, None, [0] * n, np.arange(n + 1), 0.7, u, 0)
    assert (acc == 0).all()
    assert np.array_equal(tok[:, 0], np.floor(u * V).astype(int))


@pytest.mark.parametrize("T", [0.0, 1.0])
def test_verify_of_banned_infinite_and_missing_logits(T):
    V = 300
    r = np.random.default_rng(8)
    base = r.standard_normal((1, V)).astype(np.float32)
    rows = np.repeat(base, 9, 0)
    rows[0, :] = -np.inf                               # nothing allowed
    rows[1, 5:] = -np.inf
    rows[2, ::2] = np.nan
    rows[3, [7, 250]] = np.inf                         # share the mass
    rows[4, :] = np.nan
    rows[5, 17] = np.inf
    rows[6, :] = -3e38
    rows[7, :200] = -np.inf
    rows[8, :] = -np.finfo(np.float32).max             # the type's lowest, and one beside it that is not
    rows[8, 123] = 0
    offsets = np.arange(10)
    u = np.array([0.3, 0.99, 0.5, 0.7, 0.1, 0.2, 0.6, 0.0, 0.9])
    got = run_verify(rows, None, [0] * 9, offsets, T, u, 0)
    check_verify(rows, None, [0] * 9, offsets, T, u, 0, got)
    assert got[1][0, 0] == -1 and got[1][4, 0] == -1
    if T > 0:
        assert got[1][3, 0] == 250 and got[1][5, 0] == 17
    # drafts: one that is banned, ids that are none, a row without logits in the middle
    ids = [0, 9, -1, V, 17, 17, 3, 3, 123]
    offs = [0, 2, 4, 9]
    check_verify(rows, None, ids, offs, T, u, 4, run_verify(rows, None, ids, offs, T, u, 4))


@pytest.mark.parametrize("scale,T", [(1e4, 0.01), (3e37, 1e30), (1e-3, 1e-4), (1.0, 1e-20), (1e5, 1.0)])
def test_verify_of_logits_of_all_sizes(scale, T):
    """Exponents of thousands and of 1e20, above and below zero: what a weight is taken relative to."""
    r = np.random.default_rng(11)
    n, V = 12, 700
    logits = ((r.standard_normal((n, V)) + np.where(np.arange(n) % 3 == 0, 6, -6)[:, None]) * scale).astype(np.float32)
    logits[:, 5] = logits.max(1)                       # two that share the mass, and some near them
    logits[:, 6:9] = (logits[:, 5:6].astype(np.float64) - T * np.array([0.1, 1.0, 3.0])).astype(np.float32)
    u = (np.arange(n) + 0.37) / n
    got = run_verify(logits, None, [0] * n, np.arange(n + 1), T, u, 0)
    check_verify(logits, None, [0] * n, np.arange(n + 1), np.float64(np.float32(T)), u, 0, got)


def test_verify_falls_back_where_the_rest_has_no_mass():
    """p = q and u = 1: refused (u is to be below 1, but nothing may break), and nothing is left of max(p - q, 0) but rounding."""
    V = 64
    logits = np.zeros((2, V), np.float32)
    q = np.full((2, V), 1 / V, np.float32)
    acc, tok = run_verify(logits, q, [0, 5], [0, 2], 1.0, [1.0, 0.5], 1)
    assert acc[0] == 0 and tok[0].tolist() == [32, -1]


def test_verify_where_p_and_q_nearly_agree():
    """What is left of p - q is rounding on most of the vocabulary and a little on a few tokens, all in one segment of a warp."""
    r = np.random.default_rng(12)
    V, n = 20000, 16
    logits = r.standard_normal((2 * n, V)).astype(np.float32)
    p = np.exp(logits.astype(np.float64))
    p /= p.sum(1, keepdims=True)
    q = p.copy()
    q[:, 7000:7004] *= 0.5                             # the rest's mass: half of these
    q[:, 3] += (p - q).sum(1)
    ids = np.tile([0, 3], n)
    u = np.tile([1 - 2.0 ** -24, 0.0], n)
    u[1::2] = (np.arange(n) + 0.5) / n
    got = run_verify(logits, q.astype(np.float32), ids, np.arange(0, 2 * n + 1, 2), 1.0, u, 1)
    assert (got[0] == 0).all()
    # of 4 tokens' mass; what q's rounding to fp32 leaves elsewhere is 2^-25 of p, together 2^-26 of 1 at most
    for b in range(n):
        part = (p - q)[2 * b, 7000:7004]
        slack = 2.0 ** -24 / part.sum()
        x = got[1][b, 0]
        if 7000 <= x < 7004:
            c = np.cumsum(part) / part.sum()
            assert c[x - 7000] - part[x - 7000] / part.sum() - slack <= u[2 * b + 1] <= c[x - 7000] + slack
        else:
            assert slack > 0.01 and 0 <= x < V


def test_verify_greedy_ties_go_to_the_lowest():
    logits = np.zeros((3, 9000), np.float32)
    logits[0, [8500, 40, 8191]] = 2.0
    acc, tok = run_verify(logits, None, [0, 40, 1], [0, 3], 0.0, [0, 0, 0], 2)
    assert acc[0] == 1 and tok[0].tolist() == [40, 0, -1]


def test_verify_looks_at_max_drafts_and_at_the_rows_there_are():
    r = np.random.default_rng(9)
    logits = r.standard_normal((8, 500)).astype(np.float32)
    best = logits.argmax(1)
    ids = np.concatenate([[0], best[:-1]])
    acc, tok = run_verify(logits, None, ids, [0, 8], 0.0, [0] * 8, 3)
    assert acc[0] == 3 and tok[0].tolist() == best[:4].tolist()
    # offsets that end before the arrays do: the rows behind hold nothing
    logits[5:] = np.nan
    acc, tok = run_verify(logits, None, ids, [0, 2, 5], 0.0, [0] * 8, 3)
    assert acc.tolist() == [1, 2]
    assert tok[0].tolist() == [best[0], best[1], -1, -1]


def test_verify_captured():
    r = np.random.default_rng(10)
    V, K, n = 5000, 4, 10
    logits, u = r.standard_normal((n, V)).astype(np.float32), r.random(n).astype(np.float32)
    ids, offs = np.concatenate([[0], (logits + 0.3 * r.standard_normal((n, V))).argmax(1)[:-1]]), np.array([0, 5, 10])
    s = dict(l=dev(logits), ids=i32(ids), offs=i32(offs), u=dev(u), acc=empty(2, torch.int32), tok=empty((2, K + 1), torch.int32),
             work=workspace(ops.verify_drafts_workspace, n, V))
    stream, graph = torch.cuda.Stream(), torch.cuda.CUDAGraph()
    sync()
    pkg.lib().b200_set_stream(stream.cuda_stream)
    try:
        with torch.cuda.graph(graph, stream=stream):
            ops.verify_drafts(s["l"], V, None, V, s["ids"], s["offs"], 2, n, V, 0.9, s["u"], K, s["acc"], s["tok"], s["work"], s["work"].numel())
    finally:
        pkg.lib().b200_set_stream(None)
    for i in range(4):
        x = (logits * (1 + 0.2 * i)).astype(np.float32)
        s["l"].copy_(dev(x))
        graph.replay()
        sync()
        check_verify(x, None, ids, offs, 0.9, u, K, (host(s["acc"]), host(s["tok"])))


# ---- a run of them together ----------------------------------------------------------------------
@pytest.mark.parametrize("kind,hd,page", [(1, 64, 16), (0, 128, 5)])
def test_a_server_that_checks_drafts(kind, hd, page):
    """Requests of different lengths through steps of plan, rotation, store, attention and verification; one finishes on the way and another
    takes its pages.  Every step's outputs are checked against a server kept in numpy."""
    r = np.random.default_rng(60 + hd)
    H, KV, V, B, cap, pool, K, max_rows = 4, 2, 600, 4, 14, 30, 3, 64
    rot, freq = hd // 2, so.frequencies(hd // 2, 1e4, 4, 8.0, 64, 1.0, 4.0)
    pages = torch.zeros((pool, so.page_parts(KV, hd, page, kind)[4]), dtype=torch.uint8, device="cuda")
    cache = so.Cache(pool, page, KV, hd, kind)
    f = torch.tensor(freq, device="cuda")
    ctx, held, at = np.zeros(B, int), np.zeros(B, int), [0, pool]
    table, ring = np.full((B, cap), -1), r.permutation(pool)
    d = dict(ctx=i32(ctx), held=i32(held), at=torch.tensor(at, dtype=torch.int64, device="cuda"), table=i32(table), ring=i32(ring), offs=empty(B + 1, torch.int32),
             pos=empty(max_rows, torch.int32), slots=empty(max_rows, torch.int32), counts=empty(4, torch.int32))
    mix = r.standard_normal((H * hd, V)).astype(np.float32) / math.sqrt(H * hd) * 4
    work = workspace(ops.attention_paged_kv4_workspace, H, KV, hd, max_rows)
    check = workspace(ops.verify_drafts_workspace, max_rows, V)
    steps = [[20, 7, 0, 30], [4, 4, 11, 4], [4, 3, 4, -1], [4, 4, 1, 0], [2, 4, 4, 25], [4, -1, 4, 4], [4, 9, 4, 4]]
    for new in steps:
        ops.paged_plan(d["ctx"], i32(new), d["held"], B, d["table"], cap, page, pool, d["ring"], pool, d["at"], d["at"], d["ctx"], d["held"], d["offs"],
                       d["pos"], d["slots"], max_rows, d["counts"])
        before = ctx.copy()
        p = so.plan(ctx, new, held, table, cap, page, pool, ring, at, max_rows)
        for name, t in (("seq_lens", "ctx"), ("held", "held"), ("offsets", "offs"), ("positions", "pos"), ("slots", "slots"), ("at", "at"), ("counts", "counts")):
            assert np.array_equal(host(d[t]), p[name]), name
        assert np.array_equal(host(d["table"]), table) and np.array_equal(host(d["ring"]), ring)
        lens, held, at, offs, n = np.array(p["seq_lens"]), np.array(p["held"]), p["at"], p["offsets"], p["counts"][0]
        # the step's projections: one matrix of q, k, v for all rows that there is room for
        x = r.standard_normal((max_rows, (H + 2 * KV) * hd)).astype(np.float32)
        qkv, row = dev(x), (H + 2 * KV) * hd
        kk, vv = qkv[:, H * hd:], qkv[:, (H + KV) * hd:]
        ops.rope_forward_scaled(qkv, kk, qkv, kk, d["pos"], f, max_rows, H, KV, hd, rot, 1, row, row, row, row, 1.0)
        ops.kv4_store(kk, vv, row, row, d["slots"], max_rows, pages, pool, page, KV, hd, kind)
        out = torch.zeros((max_rows, H, hd), device="cuda")
        call_attention(qkv, row, d["offs"], pages, pool, d["table"], d["ctx"], out, H * hd, max_rows, page, H, KV, hd, kind, 0.1, 0, work)
        # numpy's server takes the device's rotated rows, so that both store the same codes
        rotated = host(qkv)
        q = x[:, :H * hd].reshape(-1, H, hd)
        want_q = so.rope(q[:n], p["positions"][:n], freq, rot, 1, 1.0)
        got_q = rotated[:n, :H * hd].reshape(n, H, hd)
        assert np.abs(got_q - want_q).max() <= 4 * ROPE_TOL * np.abs(q).max()
        assert np.array_equal(rotated[n:], x[n:])
        cache.store(rotated[:n, H * hd:(H + KV) * hd].reshape(n, KV, hd), x[:n, (H + KV) * hd:].reshape(n, KV, hd), p["slots"][:n])
        assert np.array_equal(host(pages), cache.bytes)
        for b in range(B):
            if offs[b + 1] > offs[b]:
                slots = table[b, np.arange(lens[b]) // page] * page + np.arange(lens[b]) % page
                k, v = cache.rows(slots)
                want = so.attention(rotated[:, :H * hd].reshape(-1, H, hd), offs[b], offs[b + 1] - offs[b], lens[b], k, v, np.float32(0.1), 0)
                assert np.abs(host(out)[offs[b]:offs[b + 1]] - want).max() <= attention_bound(rotated[:, :H * hd].reshape(-1, H, hd), [(k, v)], 0.1)
        assert (host(out)[n:] == 0).all()
        logits = (out.reshape(max_rows, -1) @ dev(mix)).contiguous()
        ids = r.integers(0, V, max_rows)
        best = host(logits).argmax(1)
        keep = r.random(max_rows) < 0.7
        ids[1:] = np.where(keep[1:], best[:-1], ids[1:])
        u, acc, tok = r.random(max_rows).astype(np.float32), empty(B, torch.int32), empty((B, K + 1), torch.int32)
        ops.verify_drafts(logits, V, None, V, i32(ids), d["offs"], B, max_rows, V, 0.5, dev(u), K, acc, tok, check, check.numel())
        check_verify(host(logits), None, ids, offs, 0.5, u, K, (host(acc), host(tok)))
        # a decode request keeps its fed token and the drafts that were kept; a prompt all of its rows
        kept = host(acc)
        ctx = np.array([lens[b] if new[b] < 0 or new[b] > K + 1 or new[b] == 0 else before[b] + (1 + kept[b] if offs[b + 1] > offs[b] else 0) for b in range(B)])
        d["ctx"].copy_(i32(ctx))
