"""What the serving operators refuse, before any device work: observable without a GPU (no pointer is touched)."""
import ctypes as C
import importlib

import numpy as np
import pytest

pkg = importlib.import_module("jdm-ghassan_v1_flach_b200")
P = 1 << 20                                            # a 16-byte aligned address that nothing reads


def refused(name, args, **change):
    names = list(args)
    for k, v in change.items():
        assert k in names
    rc = pkg.lib().raw(name, *[change.get(k, args[k]) for k in names])
    assert rc == -1, (change, rc)
    assert name[5:].split("_")[0].encode().decode() in pkg.lib().last_error()


PLAN = dict(ctx=P, new=P, held=P, batch=4, table=P, max_pages=8, page=16, num_pages=64, ring=P, ring_size=64, at=P, at_out=P, lens=P,
            held_out=P, offsets=P, positions=P, slots=P, max_rows=32, counts=P)


@pytest.mark.parametrize("change", [dict(batch=-1), dict(batch=2049), dict(page=0), dict(max_pages=0), dict(num_pages=0), dict(ring_size=63),
                                    dict(max_rows=-1), dict(ctx=None), dict(table=None), dict(ring=None), dict(at=None), dict(counts=None),
                                    dict(positions=None), dict(offsets=None), dict(page=1 << 26, ring_size=64), dict(max_pages=1 << 28)])
def test_plan(change):
    refused("b200_paged_plan", PLAN, **change)


FREQ = dict(out=P, rot=64, theta=1e4, scaling=3, factor=8.0, ctx=4096, low=1.0, high=32.0, host=None)


@pytest.mark.parametrize("change", [dict(out=None), dict(rot=63), dict(rot=0), dict(rot=1026), dict(theta=1.0), dict(theta=float("nan")),
                                    dict(scaling=5), dict(scaling=-1), dict(factor=0.5), dict(factor=float("inf")), dict(ctx=0),
                                    dict(low=0.0), dict(low=32.0), dict(high=float("inf"))])
def test_frequencies(change):
    refused("b200_rope_frequencies", FREQ, **change)


ROPE = dict(q=P, k=2 * P, q_out=P, k_out=2 * P, pos=P, freq=P, n=4, H=4, KV=2, hd=64, rot=32, type=1, qs=256, ks=128, qos=256, kos=128,
            factor=1.0)


@pytest.mark.parametrize("change", [dict(pos=None), dict(freq=None), dict(q=None), dict(k_out=None), dict(rot=0), dict(rot=31), dict(rot=66),
                                    dict(hd=1026), dict(type=2), dict(H=0), dict(KV=0), dict(qs=255), dict(kos=127), dict(qos=512), dict(q_out=P + 4 * 200), dict(qs=400, qos=400, q_out=P + 4 * 200),
                                    dict(q_out=P + 64), dict(k_out=2 * P + 4, k=2 * P), dict(q=None, q_out=None, k=None, k_out=None),
                                    dict(type=0, hd=63, qs=256, rot=32)])
def test_rope(change):
    refused("b200_rope_forward_scaled", ROPE, **change)


STORE = dict(k=P, v=P, ks=256, vs=256, slots=P, n=3, pages=P, num_pages=10, page=16, KV=2, hd=128, kind=1)
FETCH = dict(pages=P, num_pages=10, page=16, slots=P, n=3, k=P, v=P, ks=256, vs=256, KV=2, hd=128, kind=1)
CACHE = [dict(hd=96), dict(hd=32), dict(hd=256), dict(kind=2), dict(kind=-1), dict(KV=0), dict(page=0), dict(num_pages=0), dict(pages=None),
         dict(pages=P + 8), dict(slots=None), dict(ks=255), dict(vs=255), dict(num_pages=1 << 20, page=1 << 12), dict(num_pages=1, page=(1 << 22) + 1)]


@pytest.mark.parametrize("change", CACHE + [dict(k=None), dict(v=None)])
def test_store(change):
    refused("b200_kv4_store", STORE, **change)


@pytest.mark.parametrize("change", CACHE + [dict(k=None, v=None)])
def test_fetch(change):
    refused("b200_kv4_fetch", FETCH, **change)


ATTN = dict(q=P, qs=1024, offsets=P, pages=P, num_pages=10, table=P, lens=P, out=P, os=1024, batch=2, rows=1, max_pages=4, page=16, H=8, KV=2,
            hd=128, kind=1, scale=0.1, window=0, work=P, size=1 << 40)


@pytest.mark.parametrize("change", [dict(hd=96), dict(kind=3), dict(H=7), dict(H=0), dict(KV=0), dict(rows=0), dict(max_pages=0), dict(page=0),
                                    dict(q=None), dict(out=None), dict(pages=None), dict(table=None), dict(lens=None), dict(work=None),
                                    dict(q=P + 4), dict(out=P + 8), dict(pages=P + 4), dict(work=P + 8), dict(qs=1022), dict(qs=1025), dict(os=1020),
                                    dict(size=0), dict(batch=(1 << 24) + 1), dict(num_pages=1 << 28), dict(max_pages=1 << 28)])
def test_attention(change):
    refused("b200_attention_paged_kv4", ATTN, **change)


VERIFY = dict(logits=P, ls=100, draft=P, ds=100, ids=P, offsets=P, batch=2, rows=6, V=100, T=1.0, u=P, k=4, accepted=P, tokens=P, work=P, size=1 << 30)


@pytest.mark.parametrize("change", [dict(logits=None), dict(ids=None), dict(offsets=None), dict(u=None), dict(accepted=None), dict(tokens=None),
                                    dict(work=None), dict(work=P + 8), dict(size=8), dict(V=0), dict(rows=-1), dict(ls=99), dict(ds=99), dict(k=-1),
                                    dict(k=256), dict(T=float("nan")), dict(T=float("inf")), dict(T=2e30), dict(T=1e-42)])
def test_verify(change):
    refused("b200_verify_drafts", VERIFY, **change)


def test_sizes():
    L = pkg.lib()
    size = np.zeros(1, np.uint64)
    for page, KV, hd, kind in [(16, 2, 64, 0), (64, 8, 128, 1), (1, 1, 64, 0), (33, 3, 128, 0)]:
        from serve_oracle import page_parts
        L.b200_kv4_page_bytes(page, KV, hd, kind, size.ctypes.data)
        assert int(size[0]) == page_parts(KV, hd, page, kind)[4]
    for bad in [(16, 2, 96, 0), (16, 2, 64, 2), (0, 2, 64, 0)]:
        assert L.raw("b200_kv4_page_bytes", *bad, size.ctypes.data) == -1
    assert L.raw("b200_kv4_page_bytes", 16, 2, 64, 0, None) == -1
    L.b200_attention_paged_kv4_workspace(12, 4, 128, 1, size.ctypes.data)
    assert int(size[0]) > 0
    assert L.raw("b200_attention_paged_kv4_workspace", 12, 5, 128, 1, size.ctypes.data) == -1
    assert L.raw("b200_attention_paged_kv4_workspace", 12, 4, 128, 0, size.ctypes.data) == -1
    L.b200_verify_drafts_workspace(0, 10, size.ctypes.data)
    assert int(size[0]) >= 16
    assert L.raw("b200_verify_drafts_workspace", 3, 0, size.ctypes.data) == -1


def test_nothing_to_do_is_not_an_error():
    L = pkg.lib()
    L.b200_rope_forward_scaled(*[None] * 6, 0, 4, 2, 64, 32, 1, 256, 128, 256, 128, 1.0)
    L.b200_kv4_store(None, None, 0, 0, None, 0, None, 1, 1, 1, 64, 0)
    L.b200_kv4_fetch(None, 1, 1, None, 0, None, None, 0, 0, 1, 64, 0)
    L.b200_attention_paged_kv4(None, 0, None, None, 1, None, None, None, 0, 0, 1, 1, 1, 1, 1, 64, 0, 1.0, 0, None, 0)
    L.b200_verify_drafts(None, 0, None, 0, None, None, 0, 0, 1, 1.0, None, 0, None, None, None, C.c_size_t(0).value)
