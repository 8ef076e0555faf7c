"""The serving operators around a paged 4-bit KV cache, measured as a server that checks drafted tokens uses them.

kind "plan"       the step's block tables, row offsets, positions and slots from the requests' lengths (b200_paged_plan)
kind "rope"       rotary positions of queries and keys, either layout, part of a head, scaled (b200_rope_forward_scaled)
kind "cache"      new keys and values into the 4-bit cache and read back from it (b200_kv4_store, b200_kv4_fetch)
kind "attention"  ragged rows of queries against the 4-bit pages (b200_attention_paged_kv4)
kind "verify"     drafted tokens against the target's probabilities, from given uniforms (b200_verify_drafts)

`run` computes the plain form with elementary torch operations; where `own` is true it calls the framework.

The 4-bit page.  A page of the pool holds `page` tokens: K codes, K scales, V codes, V scales, each part [KV, page, ...] and
starting on a multiple of 128 bytes.  A token's row of hd elements is cut in blocks of 32; element 32 b + 4 g + i of a row is
nibble i of its 16-bit word g * (hd / 32) + b.  Kind 0 keeps one fp16 scale d per block, value d (code - 8); kind 1 keeps (d, m),
value d code + m.
"""
import importlib
import math

import numpy as np
import torch

own = False

PKG = "jdm-ghassan_v1_flach_b200"

# Head shapes and vocabularies of the benchmark's models (the H-Small-shaped one at the op level).
HEADS = {"small": (12, 4, 64), "htiny": (12, 4, 128), "hsmall": (32, 8, 128)}
VOCAB = {"small": 32768, "htiny": 100352}
ROPE_HALF, ROPE_PAIRS = 1, 0                             # rope_type of include/b200ops.h
SCALINGS = {"none": 0, "linear": 1, "ntk": 2, "yarn": 3, "bands": 4}


def listed():
    return [
        # a handful of chats with four drafted tokens each: latency
        dict(name="plan_chats", kind="plan", batch=5, page=64, lo=100, hi=2000, new_lo=5, new_hi=5, done=0, tight=False),
        # a full server: decode rows beside pieces of prompts, some requests finished
        dict(name="plan_server", kind="plan", batch=700, page=16, lo=1, hi=8000, new_lo=1, new_hi=900, done=31, tight=False),
        # the rows of one user's step
        dict(name="rope_step", kind="rope", shape="small", rows=5, rot=64, layout=ROPE_HALF, scaling="none", reach=4000),
        # a prompt of a long-context model: half of each head rotated, frequencies scaled, positions far out
        dict(name="rope_prompt", kind="rope", shape="hsmall", rows=8191, rot=64, layout=ROPE_PAIRS, scaling="yarn", reach=131072),
        # a decode batch's new keys and values
        dict(name="cache_step", kind="cache", shape="htiny", rows=64, page=64, quant=1),
        # prompts of 16384 tokens together
        dict(name="cache_prompt", kind="cache", shape="hsmall", rows=16384, page=64, quant=0),
        # one user, a long conversation
        dict(name="attend_chat", kind="attention", shape="htiny", batch=1, lo=4097, hi=4097, q_lo=1, q_hi=1, page=64, quant=1,
             window=0),
        # a decode batch of ragged conversations
        dict(name="attend_serve", kind="attention", shape="hsmall", batch=64, lo=256, hi=8192, q_lo=1, q_hi=1, page=64, quant=1,
             window=0),
        # the same kind of batch while each request has three to five drafted tokens checked
        dict(name="attend_drafts", kind="attention", shape="hsmall", batch=32, lo=300, hi=8000, q_lo=4, q_hi=6, page=16, quant=0,
             window=0),
        # pieces of prompts behind cached prefixes
        dict(name="attend_pieces", kind="attention", shape="small", batch=6, lo=700, hi=4100, q_lo=100, q_hi=300, page=64, quant=1,
             window=0),
        # one user's drafts, greedy drafter
        dict(name="verify_chat", kind="verify", vocab="small", batch=1, k_lo=4, k_hi=4, temperature=0.8, drafter=False),
        # a batch of them with the drafter's probabilities
        dict(name="verify_server", kind="verify", vocab="htiny", batch=64, k_lo=2, k_hi=5, temperature=1.0, drafter=True),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["plan", "rope", "cache", "attention", "attention", "verify"])
    if kind == "plan":
        batch = _log(rng, 1, 700)
        lo = _log(rng, 1, 500)
        return dict(kind=kind, batch=batch, page=rng.choice([1, 8, 16, 17, 64, 100]), lo=lo, hi=lo + _log(rng, 1, 5000),
                    new_lo=rng.choice([1, 1, 2, 5]), new_hi=5 + _log(rng, 1, 500), done=rng.randrange(0, 1 + batch // 4),
                    tight=rng.random() < 0.3)
    shape = rng.choice(sorted(HEADS))
    hd = HEADS[shape][2]
    if kind == "rope":
        layout = rng.choice([ROPE_HALF, ROPE_PAIRS])
        return dict(kind=kind, shape=shape, rows=_log(rng, 1, 8191), rot=2 * rng.randrange(1, hd // 2 + 1), layout=layout,
                    scaling=rng.choice(sorted(SCALINGS)), reach=_log(rng, 100, 1000000))
    if kind == "cache":
        return dict(kind=kind, shape=shape, rows=_log(rng, 1, 16384), page=rng.choice([1, 16, 33, 64, 128]), quant=rng.choice([0, 1]))
    if kind == "attention":
        page, quant = rng.choice([5, 16, 48, 64, 128]), rng.choice([0, 1])
        if rng.random() < 0.25:                          # pieces of prompts
            q = _log(rng, 17, 250)
            return dict(kind=kind, shape="small", batch=rng.randrange(1, 7), lo=q, hi=q + _log(rng, 1, 3500), q_lo=max(1, q // 3), q_hi=q,
                        page=page, quant=quant, window=rng.choice([0, 0, 200]))
        q = rng.choice([1, 1, 1, 2, 5, 8, 13])
        batch = _log(rng, 1, 64 // (1 + q // 4))
        lo = _log(rng, q, 2000)
        return dict(kind=kind, shape=shape, batch=batch, lo=lo, hi=lo + _log(rng, 1, 6000), q_lo=max(1, q - 3), q_hi=q, page=page,
                    quant=quant, window=rng.choice([0, 0, 0, 128, 1000]))
    k = rng.randrange(0, 9)
    return dict(kind=kind, vocab=rng.choice(sorted(VOCAB)), batch=_log(rng, 1, 360 // (k + 2)), k_lo=k // 2, k_hi=k,
                temperature=rng.choice([0.0, 0.6, 1.0, 1.3]), drafter=rng.random() < 0.6)


def _spread(n, lo, hi):
    """n lengths over [lo, hi], even over their logarithm and in no order."""
    a, b = math.log(lo), math.log(hi)
    return [int(round(math.exp(a + (b - a) * (i * 0.6180339887 % 1.0)))) for i in range(n)]


def _plan_lengths(c):
    """(context, new rows; -1: finished) of every request, in the case's own order."""
    ctx, new = _spread(c["batch"], c["lo"], c["hi"]), _spread(c["batch"], c["new_lo"], c["new_hi"])
    for i in range(c["done"]):
        new[i * c["batch"] // c["done"]] = -1
    return ctx, new


def _rows(c):
    """Rows of every sequence of an attention or verify case, no more of them than the sequence has tokens."""
    if c["kind"] == "verify":
        return [1 + x for x in _spread_counts(c["batch"], c["k_lo"], c["k_hi"])]
    return [min(a, b) for a, b in zip(_spread_counts(c["batch"], c["q_lo"], c["q_hi"]), _spread(c["batch"], c["lo"], c["hi"]))]


def _spread_counts(n, lo, hi):
    return [lo + int((hi - lo + 1) * (i * 0.7548776662 % 1.0)) for i in range(n)]


def _offsets(counts):
    return torch.tensor(np.concatenate([[0], np.cumsum(counts)]), dtype=torch.int32, device="cuda")


def _page_parts(KV, hd, page, quant):
    """(start of K codes, K scales, V codes, V scales, bytes of a page)."""
    up = lambda n: -(-n // 128) * 128                     # noqa: E731
    codes, scales = up(KV * page * hd // 2), up(KV * page * (hd // 32) * (4 if quant == 1 else 2))
    return 0, codes, codes + scales, 2 * codes + scales, 2 * (codes + scales)


def _frequencies(rot, scaling):
    """(inverse frequencies in 64 bits, factor on cos and sin): base 10000, original context 4096, scaled eightfold."""
    d = torch.arange(0, rot, 2, dtype=torch.float64, device="cuda")
    f, by, ctx = 10000.0 ** (-d / rot), 8.0, 4096.0
    if scaling == "linear":
        return f / by, 1.0
    if scaling == "ntk":
        return (10000.0 * by ** (rot / max(rot - 2.0, 1.0))) ** (-d / rot), 1.0
    if scaling == "yarn":
        at = lambda turns: rot * math.log(ctx / (turns * 2 * math.pi)) / (2 * math.log(10000.0))   # noqa: E731
        lo, hi = max(math.floor(at(32.0)), 0), min(math.ceil(at(1.0)), rot - 1)
        ramp = ((d / 2 - lo) / max(hi - lo, 1e-3)).clamp(0, 1)
        return f / by * ramp + f * (1 - ramp), 0.1 * math.log(by) + 1.0
    if scaling == "bands":
        smooth = ((ctx * f / (2 * math.pi) - 1.0) / (4.0 - 1.0)).clamp(0, 1)
        return (1 - smooth) * f / by + smooth * f, 1.0
    return f, 1.0


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed * 7919 + 17)
    normal = lambda *n: torch.randn(*n, device="cuda", generator=g)      # noqa: E731
    order = lambda n: torch.randperm(n, device="cuda", generator=g)      # noqa: E731
    i32 = lambda *n: torch.zeros(*n, dtype=torch.int32, device="cuda")   # noqa: E731
    s = dict(case=case)
    if case["kind"] == "plan":
        ctx, new = (torch.tensor(x, dtype=torch.int32, device="cuda") for x in _plan_lengths(case))
        B, page = case["batch"], case["page"]
        # what a rejected draft had taken stays with its request
        held = (ctx + page - 1) // page + (torch.arange(B, device="cuda") % 5 == 3).int()
        mix = order(B)
        ctx, new, held = ctx[mix].contiguous(), new[mix].contiguous(), held[mix].int().contiguous()
        cap = -(-(case["hi"] + case["new_hi"]) // page) + 1
        total = int(held.sum())
        want = int(((ctx + new.clamp(min=0) + page - 1) // page - held).clamp(min=0)[new > 0].sum())
        free = max(1, int(want * 0.7)) if case["tight"] else want + 10 + want // 4
        pages = order(total + free).int()
        table = i32(B, cap)
        table[torch.arange(cap, device="cuda")[None] < held[:, None]] = pages[:total]
        ring = torch.full((total + free,), -1, dtype=torch.int32, device="cuda")
        head = (total + free) * 5 + seed % (total + free)                # the ring has gone round before
        ring[(torch.arange(free, device="cuda") + head) % len(ring)] = pages[total:]
        rows = max(1, sum(x for x in _plan_lengths(case)[1] if x > 0))
        s.update(ctx=ctx, new=new, held=held, table=table, ring=ring, cap=cap, rows=rows + 3, seq_lens=i32(B), held_out=i32(B),
                 at=torch.tensor([head, head + free], dtype=torch.int64, device="cuda"),
                 at_out=torch.zeros(2, dtype=torch.int64, device="cuda"), offsets=i32(B + 1), positions=i32(rows + 3),
                 slots=i32(rows + 3), counts=i32(4))
    elif case["kind"] == "rope":
        H, KV, hd = HEADS[case["shape"]]
        n = case["rows"]
        s["q"], s["k"] = normal(n, H, hd), normal(n, KV, hd)
        s["q_out"], s["k_out"] = torch.empty_like(s["q"]), torch.empty_like(s["k"])
        s["pos"] = torch.randint(0, case["reach"], (n,), device="cuda", generator=g).int()
        s["freq"], s["factor"] = _frequencies(case["rot"], case["scaling"])
    elif case["kind"] == "cache":
        H, KV, hd = HEADS[case["shape"]]
        n, page = case["rows"], case["page"]
        s["k"], s["v"] = normal(n, KV, hd) * torch.exp(0.5 * normal(1, KV, hd)) + 0.2, normal(n, KV, hd)
        s["num_pages"] = n // page + 7
        s["slots"] = order(s["num_pages"] * page)[:n].int()
        s["pages"] = torch.zeros(s["num_pages"], _page_parts(KV, hd, page, case["quant"])[4], dtype=torch.uint8, device="cuda")
        s["k_out"], s["v_out"] = torch.empty_like(s["k"]), torch.empty_like(s["v"])
    elif case["kind"] == "attention":
        H, KV, hd = HEADS[case["shape"]]
        page, quant = case["page"], case["quant"]
        lens, rows = _spread(case["batch"], case["lo"], case["hi"]), _rows(case)
        need = [-(-n // page) for n in lens]
        s["most"], s["num_pages"], s["longest"], s["most_rows"] = max(need), sum(need) + 3, max(lens), max(rows)
        pool = order(s["num_pages"]).int()
        s["table"] = i32(len(lens), s["most"])
        s["table"][torch.arange(s["most"], device="cuda")[None] < torch.tensor(need, device="cuda")[:, None]] = pool[:sum(need)]
        s["lens"], s["offsets"] = torch.tensor(lens, dtype=torch.int32, device="cuda"), _offsets(rows)
        s["q"] = normal(sum(rows), H, hd)
        s["out"] = torch.empty_like(s["q"])
        k0, k1, v0, v1, size = _page_parts(KV, hd, page, quant)
        s["pages"] = torch.randint(0, 256, (s["num_pages"], size), dtype=torch.uint8, device="cuda", generator=g)
        for at in (k1, v1):
            d = 0.2 * torch.exp(0.3 * normal(s["num_pages"], KV, page, hd // 32, 1))
            if quant == 1:
                d = torch.cat([d, -7.5 * d + 0.1 * normal(*d.shape)], -1)
            raw = d.half().reshape(s["num_pages"], -1).view(torch.uint8)
            s["pages"][:, at:at + raw.shape[1]] = raw
    else:
        V, B = VOCAB[case["vocab"]], case["batch"]
        rows = _rows(case)
        n = sum(rows)
        s["offsets"], s["most"], s["V"], s["rows"] = _offsets(rows), max(rows) - 1, V, n
        s["logits"] = 2.5 * normal(n, V)
        near = s["logits"] + 0.6 * normal(n, V)
        T = case["temperature"] if case["temperature"] > 0 else 1.0
        s["draft"] = torch.softmax(near / T, -1) if case["drafter"] else None
        picks = torch.multinomial(s["draft"], 1, generator=g)[:, 0] if case["drafter"] else near.argmax(-1)
        s["ids"] = torch.cat([picks[:1], picks[:-1]]).int()              # row j + 1 is fed what was drafted after row j
        s["uniforms"] = torch.rand(n, device="cuda", generator=g)
        s["accepted"], s["tokens"] = i32(B), i32(B, s["most"] + 1)
    return s


def _ops():
    return importlib.import_module(PKG + ".ops")


def _workspace(s, query, *sizes):
    """The buffer that a program allocates once for calls of these sizes."""
    if "work" not in s:
        size = np.zeros(1, np.uint64)
        query(*sizes, size.ctypes.data)
        s["work"] = torch.empty(int(size[0]), dtype=torch.uint8, device="cuda")
    return s["work"]


def run(s):
    c = s["case"]
    return {"plan": _plan, "rope": _rope, "cache": _cache, "attention": _attention, "verify": _verify}[c["kind"]](s, c)


def _plan(s, c):
    if own:
        _ops().paged_plan(s["ctx"], s["new"], s["held"], c["batch"], s["table"], s["cap"], c["page"], len(s["ring"]), s["ring"],
                            len(s["ring"]), s["at"], s["at_out"], s["seq_lens"], s["held_out"], s["offsets"], s["positions"],
                            s["slots"], s["rows"], s["counts"])
        return {n: s[n] for n in ("table", "ring", "at_out", "seq_lens", "held_out", "offsets", "positions", "slots", "counts")}
    ctx, new, held, page, cap, ring = s["ctx"].long(), s["new"].long(), s["held"].long(), c["page"], s["cap"], s["ring"]
    head, tail = s["at"][0], s["at"][1]
    fits = (new > 0) & (ctx + new <= cap * page)
    take = torch.where(fits, ((ctx + new + page - 1) // page - held).clamp(min=0), 0)
    rows = torch.where(fits, new, 0)
    good = fits & (rows.cumsum(0) <= s["rows"]) & (take.cumsum(0) <= tail - head)
    take, rows = take * good, rows * good
    done = new < 0
    back = torch.where(done, held, 0)
    offsets = torch.cat([rows.new_zeros(1), rows.cumsum(0)])
    column = torch.arange(cap, device="cuda")[None]
    from_ring = head + (take.cumsum(0) - take - held)[:, None] + column
    fresh = (column >= held[:, None]) & (column < (held + take)[:, None])
    to_ring = tail + (back.cumsum(0) - back)[:, None] + column
    size = len(ring)
    where = torch.where(column < back[:, None], to_ring % size, size).flatten()
    s["table"].copy_(torch.where(fresh, ring[from_ring % size], s["table"]))
    ring.copy_(torch.cat([ring, ring[:1]]).scatter(0, where, s["table"].flatten())[:size])
    row = torch.arange(s["rows"], device="cuda")
    live = row < offsets[-1]
    seq = torch.searchsorted(offsets[1:].contiguous(), row, right=True).clamp(max=c["batch"] - 1)
    pos = torch.where(live, ctx[seq] + row - offsets[seq], -1)
    slot = torch.where(live, s["table"][seq, pos.clamp(min=0) // page] * page + pos % page, -1)
    s["counts"].copy_(torch.stack([offsets[-1], take.sum(), back.sum(), ((new > 0) & ~good).sum()]))
    return {"table": s["table"], "ring": ring, "at_out": torch.stack([head + take.sum(), tail + back.sum()]),
            "seq_lens": torch.where(done, 0, ctx + rows).int(), "held_out": torch.where(done, 0, held + take).int(),
            "offsets": offsets.int(), "positions": pos.int(), "slots": slot.int(), "counts": s["counts"]}


def _rope(s, c):
    H, KV, hd = HEADS[c["shape"]]
    rot, n = c["rot"], c["rows"]
    if own:
        _ops().rope_forward_scaled(s["q"], s["k"], s["q_out"], s["k_out"], s["pos"], s["freq"], n, H, KV, hd, rot, c["layout"],
                                     H * hd, KV * hd, H * hd, KV * hd, s["factor"])
        return {"q": s["q_out"], "k": s["k_out"]}
    angle = s["pos"].double()[:, None] * s["freq"]
    cos, sin = ((f(angle) * s["factor"]).float()[:, None] for f in (torch.cos, torch.sin))
    x = torch.cat([s["q"], s["k"]], 1)
    if c["layout"] == ROPE_HALF:
        a, b = x[..., :rot // 2], x[..., rot // 2:rot]
        turned = torch.cat([a * cos - b * sin, a * sin + b * cos], -1)
    else:
        a, b = x[..., 0:rot:2], x[..., 1:rot:2]
        turned = torch.stack([a * cos - b * sin, a * sin + b * cos], -1).flatten(-2)
    x = torch.cat([turned, x[..., rot:]], -1)
    return {"q": x[:, :H], "k": x[:, H:]}


def _nearest(x):
    """The nearest whole number, halves away from zero."""
    t = torch.trunc(x)
    return t + torch.sign(x) * ((x - t).abs() >= 0.5)


def _in_four_bits(x, quant):
    """What the cache holds of rows [.., hd]: blocks of 32 by the rule of b200_quantize kinds 0 and 1."""
    b = x.unflatten(-1, (-1, 32))
    if quant == 1:
        low = b.amin(-1, keepdim=True)
        d = (b.amax(-1, keepdim=True) - low) / 15.0
        code = _nearest((b - low) * torch.where(d > 0, 1.0 / d, 0.0)).clamp(0, 15)
        return (d.half().to(x.dtype) * code + low.half().to(x.dtype)).flatten(-2)
    d = b.abs().amax(-1, keepdim=True) / 8.0
    code = _nearest(b * torch.where(d > 0, 1.0 / d, 0.0)).clamp(-8, 7)
    return (d.half().to(x.dtype) * code).flatten(-2)


def _cache(s, c):
    H, KV, hd = HEADS[c["shape"]]
    if own:
        _ops().kv4_store(s["k"], s["v"], KV * hd, KV * hd, s["slots"], c["rows"], s["pages"], s["num_pages"], c["page"], KV, hd,
                           c["quant"])
        _ops().kv4_fetch(s["pages"], s["num_pages"], c["page"], s["slots"], c["rows"], s["k_out"], s["v_out"], KV * hd, KV * hd,
                           KV, hd, c["quant"])
        return {"k": s["k_out"], "v": s["v_out"]}
    return {"k": _in_four_bits(s["k"], c["quant"]), "v": _in_four_bits(s["v"], c["quant"])}


def _values(raw, codes_at, scales_at, KV, hd, page, quant, dtype):
    """[.., pages, bytes] -> the values of one part, [.., pages * page, KV, hd]."""
    nb = hd // 32
    code = raw[..., codes_at:codes_at + KV * page * hd // 2].unflatten(-1, (KV, page, 8, nb, 2))
    code = torch.stack([code & 15, code >> 4], -1).flatten(-2)                          # [.., KV, page, g, b, i]
    width = 2 if quant == 1 else 1
    scale = raw[..., scales_at:scales_at + KV * page * nb * 2 * width].contiguous().view(torch.float16).unflatten(-1, (KV, page, nb, width))
    code = code.transpose(-3, -2).flatten(-2).to(dtype)                                 # [.., KV, page, b, 32]
    scale = scale.to(dtype)
    x = code * scale[..., :1] + scale[..., 1:] if quant == 1 else (code - 8.0) * scale
    return x.flatten(-2).transpose(-3, -2).flatten(-4, -3)


def _attention(s, c):
    H, KV, hd = HEADS[c["shape"]]
    B, page, quant, Q = c["batch"], c["page"], c["quant"], s["most_rows"]
    if own:
        work = _workspace(s, _ops().attention_paged_kv4_workspace, H, KV, hd, Q)
        _ops().attention_paged_kv4(s["q"], H * hd, s["offsets"], s["pages"], s["num_pages"], s["table"], s["lens"], s["out"], H * hd,
                                     B, Q, s["most"], page, H, KV, hd, quant, 1.0 / math.sqrt(hd), c["window"], work,
                                     work.numel())
        return {"out": s["out"]}
    k0, k1, v0, v1, _ = _page_parts(KV, hd, page, quant)
    raw = s["pages"][s["table"].long()]
    k = _values(raw, k0, k1, KV, hd, page, quant, torch.float32)
    v = _values(raw, v0, v1, KV, hd, page, quant, torch.float32)
    off = s["offsets"].long()
    count = off[1:] - off[:-1]
    i = torch.arange(Q, device="cuda")
    q = s["q"][(off[:-1, None] + i).clamp(max=len(s["q"]) - 1)].unflatten(2, (KV, H // KV)) * (1.0 / math.sqrt(hd))
    at = (s["lens"] - count)[:, None, None] + i[:, None]                                # [B, Q, 1]
    key = torch.arange(k.shape[1], device="cuda")
    seen = key <= at
    if c["window"] > 0:
        seen = seen & (key > at - c["window"])
    x = torch.matmul(q.permute(0, 2, 3, 1, 4).flatten(2, 3), k.permute(0, 2, 3, 1)).unflatten(2, (H // KV, Q))
    x = torch.where(seen[:, None, None], x, -math.inf)
    p = torch.exp(x - x.amax(-1, keepdim=True))
    o = torch.matmul(p.flatten(2, 3), v.permute(0, 2, 1, 3)).unflatten(2, (H // KV, Q)) / p.sum(-1, keepdim=True)
    row = torch.arange(len(s["q"]), device="cuda")
    seq = torch.searchsorted(off[1:].contiguous(), row, right=True)
    return {"out": o.permute(0, 3, 1, 2, 4).flatten(2, 3)[seq, row - off[seq]]}


def _verify(s, c):
    B, V, K, T = c["batch"], s["V"], s["most"], c["temperature"]
    if own:
        work = _workspace(s, _ops().verify_drafts_workspace, s["rows"], V)
        _ops().verify_drafts(s["logits"], V, s["draft"], V, s["ids"], s["offsets"], B, s["rows"], V, T, s["uniforms"], K,
                               s["accepted"], s["tokens"], work, work.numel())
        return {"accepted": s["accepted"], "tokens": s["tokens"]}
    off = s["offsets"].long()
    count = off[1:] - off[:-1]
    step = torch.arange(K + 1, device="cuda")
    row = (off[:-1, None] + step).clamp(max=s["rows"] - 1)                              # [B, K + 1]
    drafted = s["ids"].long()[(row + 1).clamp(max=s["rows"] - 1)]
    is_draft = step < (count - 1)[:, None]
    u = s["uniforms"].double()
    if T <= 0:
        best = s["logits"].argmax(-1)[row]
        passed = is_draft & (best == drafted)
    else:
        x = s["logits"].double()                                                        # borders of the draw: 64 bits
        p = torch.exp((x - x.amax(-1, keepdim=True)) / T)
        p = p / p.sum(-1, keepdim=True)
        chance = p[row, drafted]
        if s["draft"] is None:
            passed = is_draft & (u[row] < chance)
        else:
            passed = is_draft & (u[row] * s["draft"].double()[row, drafted] < chance)
    n = passed.long().cumprod(-1).sum(-1)
    if T <= 0:
        last = best.gather(1, n[:, None])[:, 0]
    else:
        at = row.gather(1, n[:, None])[:, 0]
        x = drafted.gather(1, n[:, None])
        refused = n < count - 1
        if s["draft"] is None:
            rest = p[at].scatter(1, x, 0.0)
        else:
            rest = (p[at] - s["draft"].double()[at]).clamp(min=0.0)
        rest = torch.where(refused[:, None], rest, p[at])
        sums = rest.cumsum(-1)
        mark = u[off[1:] - 1][:, None] * sums[:, -1:]                                   # its last row's uniform draws
        last = (sums <= mark).sum(-1).clamp(max=V - 1)
    tokens = torch.where(step < n[:, None], drafted, -1)
    tokens = torch.where(step == n[:, None], last[:, None], tokens)
    return {"accepted": n.int(), "tokens": tokens.int()}


def work(case):
    """Each input read once, each output written once; a draft's check reads the rows of logits up to the first one refused at the
    least, and is counted with all of them."""
    if case["kind"] == "plan":
        new = _plan_lengths(case)[1]
        rows, page = sum(x for x in new if x > 0), case["page"]
        return {"bytes": 24.0 * case["batch"] + 8.0 * rows + 8.0 * (rows / page + case["done"] * case["hi"] / page / 4), "flops": 0.0}
    if case["kind"] == "verify":
        V, rows = VOCAB[case["vocab"]], sum(_rows(case))
        more = case["batch"] * V * 4.0 if case["drafter"] and case["temperature"] > 0 else 0.0
        return {"bytes": 4.0 * rows * V + more, "flops": 4.0 * rows * V}
    H, KV, hd = HEADS[case["shape"]]
    if case["kind"] == "rope":
        return {"bytes": 8.0 * case["rows"] * (H + KV) * hd, "flops": 3.0 * case["rows"] * (H + KV) * case["rot"]}
    row = 2 * KV * (hd // 2 + hd // 32 * (4 if case["quant"] == 1 else 2))              # K and V of a token
    if case["kind"] == "cache":
        return {"bytes": case["rows"] * (2.0 * row + 16.0 * KV * hd), "flops": 12.0 * case["rows"] * KV * hd}
    lens, rows, w = _spread(case["batch"], case["lo"], case["hi"]), _rows(case), case["window"]
    reach = lambda n, r: n if w <= 0 else min(n, w + r - 1)                             # noqa: E731
    met = sum(min(n - r + i + 1, w if w > 0 else n) for n, r in zip(lens, rows) for i in range(r))
    return {"bytes": float(row) * sum(reach(n, r) for n, r in zip(lens, rows)) + 8.0 * sum(rows) * H * hd, "flops": 4.0 * met * H * hd}


# ---- what the definitions give in 64 bits ------------------------------------------------------------------------------


def exact(case, seed):
    s = prepare(case, seed)
    kind = case["kind"]
    if kind == "plan":
        return _exact_plan(s, case)
    if kind == "rope":
        return _exact_rope(s, case)
    if kind == "cache":
        return {n: _exact_four_bits(s[n].cpu().numpy(), case["quant"]) for n in ("k", "v")}
    return _exact_attention(s, case) if kind == "attention" else _exact_verify(s, case)


def _exact_plan(s, c):
    page, cap, size = c["page"], s["cap"], len(s["ring"])
    table, ring = s["table"].cpu().numpy().copy(), s["ring"].cpu().numpy().copy()
    head, tail = (int(x) for x in s["at"].cpu())
    offsets, positions, slots, seq_lens, held_out = [0], [], [], [], []
    want_rows = want_pages = taken = back = refused = 0
    for b, (ctx, new, held) in enumerate(zip(s["ctx"].tolist(), s["new"].tolist(), s["held"].tolist())):
        if new < 0:
            for j in range(held):
                ring[(tail + back + j) % size] = table[b, j]
            back, ctx, held = back + held, 0, 0
        elif new > 0:
            more = max(0, -(-(ctx + new) // page) - held)
            ok = ctx + new <= cap * page
            want_rows, want_pages = want_rows + new * ok, want_pages + more * ok
            if ok and want_rows <= s["rows"] and want_pages <= tail - head:
                for j in range(more):
                    table[b, held + j] = ring[(head + taken + j) % size]
                for p in range(ctx, ctx + new):
                    positions.append(p)
                    slots.append(int(table[b, p // page]) * page + p % page)
                taken, ctx, held = taken + more, ctx + new, held + more
            else:
                refused += 1
        offsets.append(len(positions))
        seq_lens.append(ctx)
        held_out.append(held)
    counts = [len(positions), taken, back, refused]
    positions += [-1] * (s["rows"] - len(positions))
    slots += [-1] * (s["rows"] - len(slots))
    t = lambda x, d=torch.int32: torch.tensor(np.asarray(x), dtype=d, device="cuda")    # noqa: E731
    return {"table": t(table), "ring": t(ring), "at_out": t([head + taken, tail + back], torch.int64), "seq_lens": t(seq_lens),
            "held_out": t(held_out), "offsets": t(offsets), "positions": t(positions), "slots": t(slots), "counts": t(counts)}


def _exact_rope(s, c):
    rot = c["rot"]
    turn = torch.polar(torch.full_like(s["freq"], s["factor"]).expand(c["rows"], -1), s["pos"].double()[:, None] * s["freq"])[:, None]
    got = {}
    for n in ("q", "k"):
        y = s[n].double()
        pair = (slice(0, rot // 2), slice(rot // 2, rot)) if c["layout"] == ROPE_HALF else (slice(0, rot, 2), slice(1, rot, 2))
        z = torch.complex(y[..., pair[0]], y[..., pair[1]]) * turn
        y[..., pair[0]], y[..., pair[1]] = z.real, z.imag
        got[n] = y
    return got


def _exact_four_bits(x, quant):
    """The codes are defined by single fp32 operations, as those of b200_quantize are; what they stand for is taken in 64 bits."""
    f, rows = np.float32, x.reshape(-1, 32)
    low = rows.min(1, keepdims=True) if quant == 1 else f(0)
    d = (rows.max(1, keepdims=True) - low) / f(15) if quant == 1 else np.abs(rows).max(1, keepdims=True) / f(8)
    inverse = np.divide(f(1), d, out=np.zeros_like(d), where=d > 0)
    steps = ((rows - low) * inverse).astype(np.float64)
    code = np.clip(np.copysign(np.floor(np.abs(steps) + 0.5), steps), 0 if quant == 1 else -8, 15 if quant == 1 else 7)
    value = d.astype(np.float16).astype(np.float64) * code + np.asarray(low, np.float16).astype(np.float64)
    return torch.from_numpy(value.reshape(x.shape)).cuda()


def _exact_attention(s, c):
    H, KV, hd = HEADS[c["shape"]]
    page, quant = c["page"], c["quant"]
    k0, k1, v0, v1, _ = _page_parts(KV, hd, page, quant)
    off, lens = s["offsets"].tolist(), s["lens"].tolist()
    out = torch.empty(off[-1], H, hd, dtype=torch.float64, device="cuda")
    for b, n in enumerate(lens):
        raw = s["pages"][s["table"][b, :-(-n // page)].long()]
        k = _values(raw, k0, k1, KV, hd, page, quant, torch.float64)[:n].repeat_interleave(H // KV, 1)
        v = _values(raw, v0, v1, KV, hd, page, quant, torch.float64)[:n].repeat_interleave(H // KV, 1)
        m = off[b + 1] - off[b]
        at = torch.arange(n - m, n, device="cuda")[:, None]
        key = torch.arange(n, device="cuda")
        hidden = (key > at) | ((key <= at - c["window"]) if c["window"] > 0 else False)
        x = torch.einsum("qhd,lhd->hql", s["q"][off[b]:off[b + 1]].double(), k) / math.sqrt(hd)
        out[off[b]:off[b + 1]] = torch.einsum("hql,lhd->qhd", torch.softmax(x.masked_fill(hidden, -math.inf), -1), v)
    return {"out": out}


def _exact_verify(s, c):
    T, off, u, ids = c["temperature"], s["offsets"].tolist(), s["uniforms"].tolist(), s["ids"].tolist()
    accepted, tokens = [], []
    for b in range(c["batch"]):
        first, end = off[b], off[b + 1]
        got, r = [], first
        while True:
            x = s["logits"][r].double()
            q = s["draft"][r].double() if s["draft"] is not None else None
            p = torch.softmax(x / T, 0) if T > 0 else None
            if r + 1 < end:
                y = ids[r + 1]
                if T <= 0:
                    good = int(x.argmax()) == y
                else:
                    good = u[r] * (1.0 if q is None else float(q[y])) < float(p[y])
                if good:
                    got.append(y)
                    r += 1
                    continue
                if T > 0:
                    p = torch.clamp(p - q, min=0.0) if q is not None else p.index_fill(0, torch.tensor([y], device="cuda"), 0.0)
            if T <= 0:
                pick = int(x.argmax())
            else:
                sums = p.cumsum(0)
                pick = int((sums <= u[end - 1] * sums[-1]).sum())
            accepted.append(len(got))
            tokens.append(got + [pick] + [-1] * (s["most"] - len(got)))
            break
    t = lambda x: torch.tensor(x, dtype=torch.int32, device="cuda")                     # noqa: E731
    return {"accepted": t(accepted), "tokens": t(tokens)}
