"""The serving operators of include/b200serve.h in numpy, 64 bits and loops: the plain implementations that
tests/test_serve_oracle.py, tests/test_serve_refusals.py and tests/test_gpu_serve.py compare with."""
import math

import numpy as np


# ---- the 4-bit pages -----------------------------------------------------------------------
def page_parts(KV, hd, page, kind):
    """(K codes, K scales, V codes, V scales, bytes of a page), offsets in bytes."""
    def up(n):
        return -(-n // 128) * 128
    codes, scales = up(KV * page * hd // 2), up(KV * page * (hd // 32) * (4 if kind == 1 else 2))
    return 0, codes, codes + scales, 2 * codes + scales, 2 * (codes + scales)


def quantize(x, kind):
    """Rows [.., hd] fp32 -> (codes uint8 [.., hd], scales fp16 [.., hd/32, 1 or 2]): single fp32 operations."""
    f = np.float32
    b = np.asarray(x, f).reshape(x.shape[:-1] + (-1, 32))
    bad = ~np.isfinite(b).all(-1, keepdims=True)
    b = np.where(bad, f(0), b)
    with np.errstate(over="ignore", divide="ignore", invalid="ignore"):
        low = b.min(-1, keepdims=True) if kind == 1 else f(0)
        d = (b.max(-1, keepdims=True) - low) * (f(1) / f(15)) if kind == 1 else np.abs(b).max(-1, keepdims=True) / f(8)
        inv = np.where(d > 0, f(1) / d, f(0))
        t = ((b - low) * inv).astype(np.float64)
        r = np.copysign(np.floor(np.abs(t) + 0.5), t)
        r = np.where(np.isnan(r), 0, r)
    code = np.clip(r, 0, 15) if kind == 1 else np.clip(r, -8, 7) + 8
    def half(v):
        return np.clip(v, f(-65504), f(65504)).astype(np.float16)
    scales = np.concatenate([half(d), half(low)], -1) if kind == 1 else half(d)
    return code.astype(np.uint8).reshape(x.shape), scales


def values(codes, scales, kind):
    """float64 values of quantize()'s answer."""
    c = codes.reshape(codes.shape[:-1] + (-1, 32)).astype(np.float64)
    s = scales.astype(np.float64)
    v = c * s[..., :1] + s[..., 1:] if kind == 1 else (c - 8.0) * s
    return v.reshape(codes.shape)


def pack_codes(codes):
    """[.., hd] codes -> [.., hd/2] bytes of a row: element 32 b + 4 g + i is nibble i of word g * nb + b."""
    hd = codes.shape[-1]
    c = codes.reshape(codes.shape[:-1] + (hd // 32, 8, 4)).astype(np.uint16)
    w = c[..., 0] | c[..., 1] << 4 | c[..., 2] << 8 | c[..., 3] << 12
    return np.ascontiguousarray(np.swapaxes(w, -1, -2)).view(np.uint8).reshape(codes.shape[:-1] + (hd // 2,))


def unpack_codes(rows):
    nb = rows.shape[-1] // 16
    w = np.ascontiguousarray(rows).view(np.uint16).reshape(rows.shape[:-1] + (8, nb))
    c = np.stack([w >> (4 * i) & 15 for i in range(4)], -1)                   # [.., g, b, i]
    return np.swapaxes(c, -3, -2).reshape(rows.shape[:-1] + (nb * 32,)).astype(np.uint8)


class Cache:
    """A pool of pages in host memory."""

    def __init__(self, num_pages, page, KV, hd, kind, fill=0):
        self.num_pages, self.page, self.KV, self.hd, self.kind = num_pages, page, KV, hd, kind
        self.parts = page_parts(KV, hd, page, kind)
        self.bytes = np.full((num_pages, self.parts[4]), fill, np.uint8)

    def _views(self):
        KV, page, hd, nb, w = self.KV, self.page, self.hd, self.hd // 32, 2 if self.kind == 1 else 1
        for c, s in ((self.parts[0], self.parts[1]), (self.parts[2], self.parts[3])):
            codes = self.bytes[:, c:c + KV * page * hd // 2].reshape(-1, KV, page, hd // 2)
            scales = self.bytes[:, s:s + KV * page * nb * 2 * w]
            yield c, s, codes, scales

    def store(self, k, v, slots):
        nb, w = self.hd // 32, 2 if self.kind == 1 else 1
        for x, (c, s, _, _) in zip((k, v), list(self._views())):
            codes, scales = quantize(x, self.kind)
            packed = pack_codes(codes)
            for i, slot in enumerate(slots):
                if not 0 <= slot < self.num_pages * self.page:
                    continue
                p, off = divmod(int(slot), self.page)
                for h in range(self.KV):
                    row = h * self.page + off
                    at = c + row * self.hd // 2
                    self.bytes[p, at:at + self.hd // 2] = packed[i, h]
                    at = s + row * nb * 2 * w
                    self.bytes[p, at:at + nb * 2 * w] = scales[i, h].reshape(-1).view(np.uint8)

    def rows(self, slots):
        """float64 (k, v, size of k, size of v) at the slots; size: |d| code + |m| (kind 0: |d| 8), what sums are made of."""
        got, nb, w = [], self.hd // 32, 2 if self.kind == 1 else 1
        p, off = np.divmod(np.asarray(slots, np.int64), self.page)
        for c, s, codes, _ in self._views():
            code = unpack_codes(codes[p, :, off])
            raw = np.stack([self.bytes[p, s + (h * self.page + off) * nb * 2 * w + j] for h in range(self.KV) for j in range(nb * 2 * w)], -1)
            scales = np.ascontiguousarray(raw).view(np.float16).reshape(len(p), self.KV, nb, w)
            got.append((values(code, scales, self.kind), scales.astype(np.float64), code))
        return got[0][0], got[1][0]


# ---- the plan --------------------------------------------------------------------------------
def plan(ctx, new, held, table, max_pages, page, num_pages, ring, at, max_rows):
    """table and ring are changed in place; -> dict of the outputs."""
    size, (head, tail) = len(ring), at
    sound = 0 <= head <= tail <= head + size
    avail = tail - head if sound else 0
    before = ring.copy()
    offsets, pos, slots, seq_lens, held_out, pushes = [0], [], [], [], [], []
    want_rows = want_pages = taken = refused = 0
    for b, (c, n, h) in enumerate(zip(ctx, new, held)):
        c, n, h = int(c), int(n), int(h)
        if n < 0:
            pushes += [int(table[b, j]) for j in range(min(max(h, 0), max_pages))]
            c = h = 0
        elif n > 0:
            ok = c >= 0 and 0 <= h <= max_pages and c + n <= max_pages * page
            more = max(0, -(-(c + n) // page) - h)
            want_rows, want_pages = want_rows + n * ok, want_pages + more * ok
            if ok and want_rows <= max_rows and want_pages <= avail:
                for j in range(more):
                    table[b, h + j] = before[(head + taken + j) % size]
                for p in range(c, c + n):
                    i = int(table[b, p // page])
                    pos.append(p)
                    slots.append(i * page + p % page if 0 <= i < num_pages else -1)
                taken, c, h = taken + more, c + n, h + more
            else:
                refused += 1
        offsets.append(len(pos))
        seq_lens.append(c)
        held_out.append(h)
    if not sound or len(pushes) > size - avail:
        pushes = []
    for j, i in enumerate(pushes):
        ring[(tail + j) % size] = i
    pad = [-1] * (max_rows - len(pos))
    return dict(seq_lens=seq_lens, held=held_out, offsets=offsets, positions=pos + pad, slots=slots + pad,
                at=[head + taken, tail + len(pushes)], counts=[len(pos), taken, len(pushes), refused])


# ---- rotary positions ------------------------------------------------------------------------
def frequencies(rot, theta, scaling, factor, ctx, low, high):
    i = np.arange(rot // 2)
    if scaling == 2 and rot > 2:
        theta = theta * factor ** (rot / (rot - 2.0))
    f = theta ** (-2.0 * i / rot)
    if scaling == 1:
        return f / factor
    if scaling == 3:
        def dim(turns):
            return rot * math.log(ctx / (turns * 2 * math.pi)) / (2 * math.log(theta))
        lo, hi = max(math.floor(dim(high)), 0.0), min(math.ceil(dim(low)), rot - 1.0)
        ramp = np.clip((i - lo) / max(hi - lo, 1e-3), 0, 1)
        return f / factor * ramp + f * (1 - ramp)
    if scaling == 4:
        s = np.clip((ctx * f / (2 * math.pi) - low) / (high - low), 0, 1)
        return (1 - s) * f / factor + s * f
    return f


def rope(x, pos, freq, rot, rope_type, factor):
    """x [n, heads, hd] -> float64."""
    y = np.array(x, np.float64)
    angle = np.asarray(pos, np.float64)[:, None] * freq
    c, s = (factor * np.cos(angle))[:, None], (factor * np.sin(angle))[:, None]
    a, b = (slice(0, rot // 2), slice(rot // 2, rot)) if rope_type == 1 else (slice(0, rot, 2), slice(1, rot, 2))
    u, v = y[..., a].copy(), y[..., b].copy()
    y[..., a], y[..., b] = u * c - v * s, u * s + v * c
    return y


# ---- attention -------------------------------------------------------------------------------
def attention(q, first, rows, length, k, v, scale, window):
    """Rows first .. of q [n, H, hd] against k, v [length, KV, hd]; -> float64 [rows, H, hd]."""
    H, hd = q.shape[1:]
    KV = k.shape[1]
    out = np.zeros((rows, H, hd))
    for i in range(rows):
        pos = length - rows + i
        lo = max(0, pos - window + 1) if window > 0 else 0
        if pos < 0:
            continue
        for h in range(H):
            g = h // (H // KV)
            s = (k[lo:pos + 1, g] @ q[first + i, h].astype(np.float64)) * scale
            p = np.exp(s - s.max())
            out[i, h] = p @ v[lo:pos + 1, g] / p.sum()
    return out


# ---- drafted tokens --------------------------------------------------------------------------
def verify(logits, draft, ids, offsets, temperature, uniforms, max_drafts):
    """-> per sequence (drafts kept, the drawn token's (masses, mark) or the token itself, smallest margin of the checks).
    masses: float64 [V]; mark = u * their sum.  margin: |u q / p - 1|, how near a check was to the other answer."""
    got = []
    for b in range(len(offsets) - 1):
        first, end = offsets[b], offsets[b + 1]
        drafts = min(end - first - 1, max_drafts)
        if end <= first:
            got.append((0, -1, math.inf))
            continue
        margin, n, cut = math.inf, 0, None
        for n in range(drafts + 1):
            l = logits[first + n].astype(np.float64)
            l = np.where(np.isnan(l), -np.inf, l)
            top = l.max()
            if top == -np.inf:
                cut = -1
                break
            if temperature <= 0:
                cut = int(l.argmax())
                if n < drafts and cut == ids[first + n + 1]:
                    continue
                break
            with np.errstate(invalid="ignore"):
                e = np.where(l == top, 1.0, np.exp((l - top) / temperature))
            p = e / e.sum()
            if n == drafts:
                cut = (p, uniforms[end - 1] * p.sum())
                break
            x = ids[first + n + 1]
            q = draft[first + n].astype(np.float64) if draft is not None else np.eye(1, len(p), x)[0] if 0 <= x < len(p) else 0 * p
            if 0 <= x < len(p):
                test = float(uniforms[first + n]) * q[x]
                if p[x] > 0:
                    margin = min(margin, abs(test / p[x] - 1))
                if test < p[x]:
                    continue
            rest = np.maximum(p - q, 0)
            rest = rest if rest.sum() > 0 else p
            cut = (rest, uniforms[end - 1] * rest.sum())
            break
        got.append((n, cut, margin))
    return got
