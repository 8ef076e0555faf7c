"""The plain implementations of the serving operators agree with things known in another way (no GPU)."""
import numpy as np
import pytest

import serve_oracle as so


@pytest.mark.parametrize("hd", [64, 128])
def test_codes_survive_packing(hd):
    c = np.random.default_rng(0).integers(0, 16, (3, 5, hd)).astype(np.uint8)
    assert np.array_equal(so.unpack_codes(so.pack_codes(c)), c)


@pytest.mark.parametrize("kind", [0, 1])
def test_codes_and_scales_are_those_of_the_quantiser(oracle, kind):
    r = np.random.default_rng(kind)
    x = (r.standard_normal((40, 32)) * np.exp(r.standard_normal((40, 1)))).astype(np.float32)
    x[3] = 0
    x[4, 7] = np.inf
    x[5] = 2.5
    blocks = np.asarray(oracle.quantize(x.reshape(-1), kind)).view(np.uint8).reshape(40, 18 if kind == 0 else 20)
    codes, scales = so.quantize(x, kind)
    head = 2 if kind == 0 else 4
    want = blocks[:, :head].copy().view(np.float16).reshape(40, -1)
    got = np.concatenate([blocks[:, head:] & 15, blocks[:, head:] >> 4], 1)
    if kind == 0:
        assert np.array_equal(want, scales.reshape(40, -1)) and np.array_equal(got, codes)
    else:       # a product with fp32(1/15) for the division: two roundings of 2^-24 more, so one step of fp16 and a code on a border
        np.testing.assert_allclose(scales.reshape(40, -1).astype(float), want.astype(float), rtol=2.0 ** -10)
        assert np.abs(got.astype(int) - codes).max() <= 1 and np.mean(got != codes) < 0.01


def test_stored_rows_come_back():
    r = np.random.default_rng(1)
    for kind in (0, 1):
        c = so.Cache(3, 5, 2, 64, kind)
        k, v = (r.standard_normal((6, 2, 64)).astype(np.float32) for _ in range(2))
        slots = np.array([14, 0, 7, 3, -1, 15])
        c.store(k, v, slots)
        gk, gv = c.rows(slots[:4])
        # a code is off by at most half a step, and the fp16 scale moves it by 2^-11 of itself
        for got, want in ((gk, k[:4]), (gv, v[:4])):
            assert np.abs(got - want).max() <= np.abs(want).max() / 8 * (0.5 if kind == 1 else 1.0) * 1.01 + 1e-3


def test_plan_gives_every_page_to_one_request():
    r = np.random.default_rng(2)
    page, cap, pool = 4, 9, 40
    table, ring, at = np.full((5, cap), -1), np.arange(pool), [0, pool]
    ctx, held = [0] * 5, [0] * 5
    for step in range(40):
        new = [int(x) for x in r.integers(-1, 7, 5)]
        got = so.plan(ctx, new, held, table, cap, page, pool, ring, at, 20)
        ctx, held, at = got["seq_lens"], got["held"], got["at"]
        live = [int(table[b, j]) for b in range(5) for j in range(held[b])]
        free = [int(ring[i % pool]) for i in range(at[0], at[1])]
        assert sorted(live + free) == list(range(pool))
        slots = [s for s in got["slots"] if s >= 0]
        assert len(set(slots)) == len(slots)


def test_verified_tokens_follow_the_target():
    """The rule's point: whatever the drafter's distribution, the first token out is distributed as the target's."""
    r = np.random.default_rng(3)
    V, n = 5, 40000
    logits = r.standard_normal((2, V)).astype(np.float32)
    q = np.exp(r.standard_normal(V))
    q = (q / q.sum()).astype(np.float32)
    count = np.zeros(V)
    u = r.random((n, 2))
    x = np.searchsorted(np.cumsum(q), r.random(n) * q.sum())
    for i in range(n):
        got = so.verify(logits, np.stack([q, q]), [0, int(x[i])], [0, 2], 1.0, u[i], 1)[0]
        if got[0] == 1:
            count[x[i]] += 1
        else:
            masses, mark = got[1]
            count[int((np.cumsum(masses) <= mark).sum())] += 1
    p = np.exp(logits[0].astype(np.float64))
    p /= p.sum()
    # five standard deviations of a binomial share
    assert np.all(np.abs(count / n - p) <= 5 * np.sqrt(p * (1 - p) / n))
