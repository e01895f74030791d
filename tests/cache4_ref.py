"""The 4-bit cache in plain numpy, in 64 bits: its format from the definition
(include/pktito_b200.h, pkb_cache4), the attention over what it holds, and
its page operations on lists. Test infrastructure only."""
import numpy as np

UNIT, BLOCK = 16, 32


def quantize(x):
    """(codes -7..7, scales) of rows of whole blocks of 32 floats, from the definition."""
    b = np.asarray(x, np.float64).reshape(*x.shape[:-1], -1, BLOCK)
    amax = np.abs(b).max(-1)
    good = np.isfinite(b).all(-1) & (np.where(np.isnan(amax), 0, amax) >= 2.0 ** -121)
    seventh = np.where(good, amax, 1.0).astype(np.float32) * (np.float32(1) / np.float32(7))  # rounded to float
    m, e = np.frexp(seventh.astype(np.float64))
    s = np.where(good, np.ldexp(np.floor(m * 32) / 32, e), 0.0)
    c = np.rint(np.where(good[..., None], b, 0.0) / np.where(good, s, 1.0)[..., None])
    assert np.abs(c).max(initial=0) <= 7
    return c.astype(np.int64).reshape(x.shape), s


def held(x):
    c, s = quantize(x)
    return (c.reshape(*s.shape, BLOCK) * s[..., None]).reshape(x.shape)


def nibble_places(dk):
    """The nibble of K's and V's value (token r, dimension d) in a unit's codes: two arrays [16, dk]."""
    r, d = np.arange(UNIT)[:, None], np.arange(dk)[None]
    w = d % 32
    k = r * dk + ((w // 8) * (dk // 32) + d // 32) * 8 + w % 8 // 2 + 4 * (d % 2)
    v = ((((d // 32) * 8 + d % 8) * 4 + r % 8 // 2) * 2 + w // 16) * 8 + 4 * (r % 2) + 2 * (r // 8) + w % 16 // 8
    return k, v


def bf16_bits(s):
    """The bits of floats that a bf16 holds exactly."""
    b = np.asarray(s, np.float32).view(np.uint32)
    assert not (b & 0xFFFF).any()
    return (b >> 16).astype(np.uint16)


class Pages:
    """The bytes of [pages, heads, page_tokens / 16 units], read and written a token at a time."""

    def __init__(self, raw, page_tokens, heads, dk):
        self.raw = raw.reshape(-1, heads, page_tokens // UNIT, 18 * dk)
        self.P, self.H, self.dk = page_tokens, heads, dk
        self.places = nibble_places(dk)

    def _nibbles(self, which):
        """Byte and shift of each value of a token, [16, dk] each."""
        at = self.places[which]
        return which * 8 * self.dk + at // 2, 4 * (at % 2)

    def write(self, page, token, which, codes, scales):
        """codes [heads, dk], scales [heads, dk / 32] of one token; which 0 K, 1 V."""
        u = self.raw[page, :, token // UNIT]
        byte, shift = self._nibbles(which)
        r = token % UNIT
        for d in range(self.dk):
            old = u[:, byte[r, d]]
            u[:, byte[r, d]] = (old & (0xF0 if shift[r, d] == 0 else 0x0F)) | ((codes[:, d] + 8) << shift[r, d]).astype(np.uint8)
        nb = self.dk // BLOCK
        for b in range(nb):
            at = (16 + which) * self.dk + 2 * (r * nb + b if which == 0 else b * UNIT + r)
            u[:, at:at + 2] = bf16_bits(scales[:, b])[:, None].view(np.uint8)

    def read(self, pages, n):
        """K and V float64 [heads, n, dk] of a sequence's first n tokens in these pages."""
        j = np.arange(n)
        u = self.raw[np.asarray(pages, np.int64)[j // self.P], :, j % self.P // UNIT]  # [n, heads, bytes]
        r, nb = j % UNIT, self.dk // BLOCK
        out = []
        for which in (0, 1):
            byte, shift = self._nibbles(which)
            code = (np.take_along_axis(u, np.broadcast_to(byte[r][:, None], (n, self.H, self.dk)), -1) >> shift[r][:, None]) & 15
            b = np.arange(nb)
            at = (16 + which) * self.dk + 2 * (r[:, None] * nb + b if which == 0 else b * UNIT + r[:, None])
            lo = np.take_along_axis(u, np.broadcast_to(at[:, None], (n, self.H, nb)), -1).astype(np.uint32)
            hi = np.take_along_axis(u, np.broadcast_to(at[:, None] + 1, (n, self.H, nb)), -1).astype(np.uint32)
            s = (lo << 16 | hi << 24).view(np.float32).astype(np.float64)
            val = (code.astype(np.float64) - 8) * np.repeat(s, BLOCK, -1)
            out.append(val.transpose(1, 0, 2))
        return out


def attention(q, k, v, n_tokens, scale, causal, window):
    """(o, A, S) of q [R, H, dk] over k, v [heads, n, dk] in 64 bits: the result [R, H, dk], sum_j p_j |v_j| and
    the largest sum_d |q_d k_jd| * |scale| of the row over the keys it sees (what rounding errors are relative to)."""
    R, H, dk = q.shape
    G = H // k.shape[0]
    k, v = np.repeat(k, G, 0), np.repeat(v, G, 0)
    s = np.einsum("rhd,hjd->rhj", q, k) * scale
    size = np.einsum("rhd,hjd->rhj", np.abs(q), np.abs(k)) * abs(scale)
    j, pos = np.arange(n_tokens)[None], (n_tokens - R + np.arange(R))[:, None]
    seen = np.ones((R, n_tokens), bool)
    if causal:
        seen &= j <= pos
    if window:
        seen &= j > pos - window
    s = np.where(seen[:, None], s, -np.inf)
    top = s.max(-1, initial=-np.inf, keepdims=True)
    p = np.exp(s - np.where(np.isfinite(top), top, 0))
    total = p.sum(-1, keepdims=True)
    p = np.where(total > 0, p / np.where(total > 0, total, 1), 0)
    return (np.einsum("rhj,hjd->rhd", p, v), np.einsum("rhj,hjd->rhd", p, np.abs(v)),
            np.where(seen[:, None], size, 0).max(-1, initial=0))


class Books:
    """table, lens, refs as lists, and the page operations as the header words them."""

    DONE, FULL, LONG, BAD = 0, 1, 2, 3

    def __init__(self, n_pages, max_seqs, max_pages, P):
        self.P, self.n_pages, self.max_pages = P, n_pages, max_pages
        self.rows = [[] for _ in range(max_seqs)]
        self.lens = [0] * max_seqs
        self.refs = [0] * n_pages

    def arrays(self):
        table = np.full((len(self.rows), self.max_pages), -1, np.int32)
        for i, r in enumerate(self.rows):
            table[i, :len(r)] = r
        return table, np.array(self.lens, np.int32), np.array(self.refs, np.int32)

    def _need(self, n):
        return -(-n // self.P)

    def _checked(self, changed, wanted):
        """The status for entries that change these sequences; wanted: (status, new pages) an entry."""
        worst, total = 0, 0
        for s, (status, pages) in zip(changed, wanted):
            worst, total = max(worst, status), total + (pages if not status else 0)
        if len(set(changed)) != len(changed) or any(not 0 <= s < len(self.rows) for s in changed):
            worst = self.BAD
        if not worst and total > self.refs.count(0):
            worst = self.FULL
        return worst

    def _take(self):
        p = self.refs.index(0)
        self.refs[p] = 1
        return p

    def grow(self, seqs, add):
        def want(s, a):
            if not 0 <= s < len(self.rows) or a < 0:
                return self.BAD, 0
            after = self.lens[s] + a
            return (self.LONG, 0) if after > self.max_pages * self.P else (0, self._need(after) - self._need(self.lens[s]))
        status = self._checked(seqs, [want(s, a) for s, a in zip(seqs, add)])
        if not status:
            for s, a in zip(seqs, add):
                while len(self.rows[s]) < self._need(self.lens[s] + a):
                    self.rows[s].append(self._take())
                self.lens[s] += a
        return status

    def take_over(self, src, dst, lens, share, other=None):
        """fork (share) and copy (into `other` or itself): (status, pages copied as (from, to))."""
        to = other or self

        def want(a, b, n):
            if not (0 <= b < len(to.rows) and 0 <= a < len(self.rows)) or to.lens[b] or not 0 <= n <= self.lens[a]:
                return self.BAD, 0
            if n > to.max_pages * self.P:
                return self.LONG, 0
            return 0, (int(n % self.P > 0) if share else self._need(n))
        status = to._checked(dst, [want(*e) for e in zip(src, dst, lens)])
        copies = []
        if not status:
            # new pages first, in the order listed: pages shared below were in use already
            for a, b, n in zip(src, dst, lens):
                whole = n // self.P if share else 0
                row = self.rows[a][:whole]
                for j in range(whole, self._need(n)):
                    p = to._take()
                    copies.append((self.rows[a][j], p))
                    row.append(p)
                for p in row[:whole]:
                    self.refs[p] += 1
                to.rows[b], to.lens[b] = row, n
        return status, copies

    def free(self, seqs):
        status = self._checked(seqs, [(0, 0)] * len(seqs))
        if not status:
            for s in seqs:
                for p in self.rows[s]:
                    self.refs[p] -= 1
                self.rows[s], self.lens[s] = [], 0
        return status

    def compact(self):
        used = sum(r != 0 for r in self.refs)
        holes = [p for p in range(used) if not self.refs[p]]
        above = [p for p in range(used, self.n_pages) if self.refs[p]]
        to = dict(zip(above, holes))
        for a, b in to.items():
            self.refs[b], self.refs[a] = self.refs[a], 0
        self.rows = [[to.get(p, p) for p in r] for r in self.rows]
        return used, list(to.items())
