"""Plain 64-bit forms of the rotary, attention and page operations, and the error bounds that
their tests use. numpy only; bf16 arrays travel as uint16."""
import math

import numpy as np

HALF_STEP = {"f32": 2.0 ** -24, "f16": 2.0 ** -11, "bf16": 2.0 ** -8}
U = 2.0 ** -24  # half a step of a float


def to_type(x, t):
    """float64 values rounded to type t (nearest, ties to even) as the array that is uploaded."""
    f = np.asarray(x, np.float32)
    if t == "f32":
        return f
    if t == "f16":
        return f.astype(np.float16)
    b = f.view(np.uint32).astype(np.uint64)
    r = ((b + 0x7FFF + ((b >> 16) & 1)) >> 16).astype(np.uint16)
    return np.where(np.isnan(f), np.uint16(0x7FC0), r)


def from_type(a, t):
    """The float64 values of an array of type t."""
    if t == "bf16":
        return (a.astype(np.uint32) << 16).view(np.float32).astype(np.float64)
    return a.astype(np.float64)


NP = {"f32": np.float32, "f16": np.float16, "bf16": np.uint16}


def download(buf, t, shape):
    return from_type(buf.download(NP[t], int(np.prod(shape))).reshape(shape), t)


# ---------------------------------------------------------------------- rotary
def frequencies(rotary, theta, scaling="none", factor=1.0, original=4096, fast=32.0, slow=1.0):
    f = []
    for i in range(rotary // 2):
        base = theta * factor ** (rotary / (rotary - 2)) if scaling == "ntk" and rotary > 2 else theta
        w = base ** (-2.0 * i / rotary)
        if scaling == "linear":
            w /= factor
        if scaling == "yarn":
            def index(turns):
                return rotary * math.log(original / (turns * 2 * math.pi)) / (2 * math.log(theta))
            low, high = max(math.floor(index(fast)), 0), min(math.ceil(index(slow)), rotary - 1)
            ramp = min(max((i - low) / max(high - low, 0.001), 0.0), 1.0)
            w = w / factor * ramp + w * (1 - ramp)
        f.append(w)
    return np.array(f)


def rotate(x, pos, freq, layout, amplitude=1.0):
    """x [tokens][heads][dim] in float64; the angle reduced exactly where that matters."""
    y = x.copy()
    n = len(freq)
    a = np.fmod(pos.astype(np.longdouble)[:, None] * freq.astype(np.longdouble), 2 * np.pi * np.longdouble(1))
    turns = pos.astype(np.longdouble)[:, None] * (freq.astype(np.longdouble) / (2 * np.longdouble("3.14159265358979323846264338327950288")))
    a = (turns - np.floor(turns)) * 2 * np.longdouble("3.14159265358979323846264338327950288")
    c, s = np.cos(a).astype(np.float64)[:, None] * amplitude, np.sin(a).astype(np.float64)[:, None] * amplitude
    if layout == "half":
        u, v = x[..., :n], x[..., n:2 * n]
        y[..., :n], y[..., n:2 * n] = u * c - v * s, u * s + v * c
    else:
        u, v = x[..., 0:2 * n:2], x[..., 1:2 * n:2]
        y[..., 0:2 * n:2], y[..., 1:2 * n:2] = u * c - v * s, u * s + v * c
    return y


def rotate_bound(x, rotary, layout, out_type, amplitude, y):
    """Sine and cosine are within 5.4 half steps of a float (three roundings of an angle of at
    most pi / 4, the last steps of the polynomials, the amplitude); two products and a sum add
    two: 8 half steps of (|x| + |y|) amplitude, and the output's rounding."""
    n = rotary // 2
    b = np.zeros_like(x)
    if layout == "half":
        m = np.abs(x[..., :n]) + np.abs(x[..., n:rotary])
        b[..., :n] = b[..., n:rotary] = m
    else:
        m = np.abs(x[..., 0:rotary:2]) + np.abs(x[..., 1:rotary:2])
        b[..., 0:rotary:2] = b[..., 1:rotary:2] = m
    half = 0.0 if out_type == "f32" else HALF_STEP[out_type]
    return 8 * U * b * amplitude + half * np.abs(y) * (1 + 1e-3) + (2.0 ** -25 if out_type == "f16" else 1e-37)


# ------------------------------------------------------------------- attention
def attend(q, k, v, seen, scale, p_type, out_type):
    """One head: q [rows][dim], k, v [keys][dim] float64, seen [rows][keys]. Returns out, lse and
    the bound of out's error:
      scores: dim + 8 float roundings of scale sum |q k|, log2 and exp2 a few of the score;
      probabilities of 16-bit types: half a step each (f16: 2^-32 of the largest below its
      normal range);
      sums over the keys: one rounding a key of sum p |v|;
      the output's own rounding."""
    with np.errstate(all="ignore"):
        s = np.where(seen, scale * (np.where(np.isfinite(q), q, 0) @ np.where(np.isfinite(k), k, 0).T), -np.inf)
    rows, dim = q.shape
    out, lse, bound = np.zeros((rows, v.shape[1])), np.full(rows, -np.inf), np.zeros((rows, v.shape[1]))
    for i in range(rows):
        keys = np.nonzero(seen[i])[0]
        if not keys.size:
            continue
        si, vi = s[i, keys], v[keys]
        top = si.max()
        p = np.exp(si - top)
        l = p.sum()
        out[i] = p @ vi / l
        lse[i] = top + math.log(l)
        a = p @ np.abs(vi) / l
        mag = scale * (np.abs(q[i]) @ np.abs(k[keys]).T).max()
        rel = U * ((dim + 8) * mag + 4 * np.abs(si).max() + keys.size + 16)
        half_p = 0.0 if p_type == "f32" else HALF_STEP[p_type]
        bound[i] = a * (half_p + 2 * rel) + HALF_STEP[out_type] * np.abs(out[i]) * (1 + 1e-3)
        if p_type == "f16":
            bound[i] += 2.0 ** -32 * np.abs(vi).sum(0) / l
        if out_type == "f16":
            bound[i] += 2.0 ** -25
    return out, lse, bound


def lse_bound(lse, dim, mag):
    """The same roundings of the scores and the sum, absolute; one of the result."""
    return U * ((dim + 8) * mag + 64) + 4 * U * np.abs(lse)


# ----------------------------------------------------------------------- pages
class Pages:
    """The cache's bookkeeping on lists: tables, lengths and counts, entry by entry."""

    def __init__(self, n_seqs, max_pages, n_pages, page):
        self.tables = [[] for _ in range(n_seqs)]
        self.lens, self.refs = [0] * n_seqs, [0] * n_pages
        self.max_pages, self.page = max_pages, page
        self.error = 0

    def ok(self, s):
        return 0 <= s < len(self.tables)

    def cut(self, s, n):
        keep = -(-n // self.page)
        for p in self.tables[s][keep:]:
            self.refs[p] -= 1
        self.tables[s], self.lens[s] = self.tables[s][:keep], n

    def extend(self, seqs, counts):
        """Returns the copies (sequence, old page, new page, rows)."""
        free = [i for i, r in enumerate(self.refs) if r == 0]
        copies, full, seen = [], False, set()
        for s, n in zip(seqs, counts):
            first = s not in seen
            seen.add(s)
            if not self.ok(s) or not first or n < 0 or self.lens[s] + n > self.max_pages * self.page:
                self.error |= 4
                continue
            part = self.lens[s] % self.page and n > 0
            copy = part and self.refs[self.tables[s][-1]] > 1
            need = -(-(self.lens[s] + n) // self.page) - len(self.tables[s]) + (1 if copy else 0)
            if full or need > len(free):
                full = True
                self.error |= 8
                continue
            new, free = free[:need], free[need:]
            if copy:
                old = self.tables[s][-1]
                self.refs[old] -= 1
                self.tables[s][-1] = new[0]
                copies.append((s, old, new[0], self.lens[s] % self.page))
            self.tables[s] += new[1:] if copy else new
            for p in new:
                self.refs[p] = 1
            self.lens[s] += n
        return copies

    def fork(self, src, dst):
        old = [list(t) for t in self.tables]
        lens = list(self.lens)
        seen = set()
        for a, b in zip(src, dst):
            first = b not in seen
            seen.add(b)
            if not self.ok(a) or not self.ok(b) or not first:
                self.error |= 4
                continue
            for p in old[a]:
                self.refs[p] += 1
            for p in old[b]:
                self.refs[p] -= 1
            self.tables[b], self.lens[b] = list(old[a]), lens[a]

    def free(self, seqs):
        seen = set()
        for s in seqs:
            if not self.ok(s) or s in seen:
                self.error |= 4
            else:
                self.cut(s, 0)
            seen.add(s)

    def compact(self, seqs, drafts, keep, kept):
        """Returns the moves (sequence, from slot, to slot, its table at the time)."""
        moves, todo, seen = [], [], set()
        for s, nd, row, nk in zip(seqs, drafts, keep, kept):
            first = s not in seen
            seen.add(s)
            fine = self.ok(s) and first and 0 <= nd <= self.lens[s] and 0 <= nk <= nd and nk <= len(row)
            if fine:
                idx, base = row[:nk], self.lens[s] - nd
                fine = all(0 <= x < nd for x in idx) and all(a < b for a, b in zip(idx, idx[1:]))
                fine = fine and all(x == j or self.refs[self.tables[s][(base + j) // self.page]] == 1
                                    for j, x in enumerate(idx))
            if not fine:
                self.error |= 4
                continue
            moves += [(s, base + x, base + j, list(self.tables[s])) for j, x in enumerate(idx)]
            todo.append((s, base + nk))
        for s, n in todo:
            self.cut(s, n)
        return moves

    def arrays(self):
        t = np.full((len(self.tables), self.max_pages), -1, np.int32)
        for i, row in enumerate(self.tables):
            t[i, :len(row)] = row
        return t, np.array(self.lens, np.int32), np.array(self.refs, np.int32)
