"""The paged cache of many sequences restated on the host with plain loops — TEST INFRASTRUCTURE
ONLY: tables, lengths and reference counts as lists, pools as numpy arrays of stored bits, and
decode attention in 64 bits."""
import numpy as np

NO_PAGE = 0xFFFFFFFF
FULL, LONG, TAKEN = 1, 2, 4
F32, F16, BF16 = 0, 1, 30
EPS = 2.0 ** -24


def store(x, kv):
    """f32 values as the cache's bits (round to nearest even)."""
    x = np.ascontiguousarray(x, np.float32)
    if kv == F32:
        return x.view(np.uint32).copy()
    if kv == F16:
        return x.astype(np.float16).view(np.uint16)
    b = x.view(np.uint32).astype(np.uint64)
    return ((b + 0x7FFF + ((b >> 16) & 1)) >> 16).astype(np.uint16)


def load(bits, kv):
    if kv == F32:
        return bits.view(np.float32).astype(np.float64)
    if kv == F16:
        return bits.view(np.float16).astype(np.float64)
    return (bits.astype(np.uint32) << 16).view(np.float32).astype(np.float64)


class Paged:
    def __init__(self, layers, pages, pt, kvh, D, kv, rows, max_pages, seed=0):
        self.pages, self.pt, self.rows, self.max_pages, self.kv, self.kvh, self.D = pages, pt, rows, max_pages, kv, kvh, D
        rng = np.random.default_rng(seed)
        shape = (layers, pages, pt, kvh, D)
        self.k, self.v = (store(rng.standard_normal(shape, np.float32), kv) for _ in range(2))
        self.tables = [[NO_PAGE] * max_pages for _ in range(rows)]
        self.n_kv, self.refs, self.status = [0] * rows, [0] * pages, 0

    def up(self, n):
        return -(-n // self.pt)

    def _take(self, want):
        """The `want` free pages of lowest id, or None."""
        free = [p for p in range(self.pages) if self.refs[p] == 0]
        if want > len(free):
            self.status |= FULL
            return None
        return free[:want]

    def _copy(self, a, b):
        self.k[:, b], self.v[:, b] = self.k[:, a], self.v[:, a]

    def grow(self, seqs, add):
        asks = []
        for s, a in zip(seqs, add):
            n = self.n_kv[s]
            if n + a > self.max_pages * self.pt:
                self.status |= LONG
                return
            last = self.tables[s][n // self.pt] if n % self.pt else NO_PAGE
            cow = a > 0 and last < self.pages and self.refs[last] > 1
            asks.append((s, n, a, cow, self.up(n + a) - self.up(n) if a else 0))
        ids = self._take(sum(c + f for _, _, _, c, f in asks))
        if ids is None:
            return
        copies = []
        for s, n, a, cow, fresh in asks:
            if cow:
                old, new = self.tables[s][n // self.pt], ids.pop(0)
                copies.append((old, new))
                self.tables[s][n // self.pt] = new
                self.refs[new] = 1
            for j in range(self.up(n), self.up(n) + fresh):
                self.tables[s][j] = ids.pop(0)
                self.refs[self.tables[s][j]] = 1
            self.n_kv[s] = n + a
        for old, new in copies:
            self.refs[old] -= 1
            self._copy(old, new)

    def fork(self, src, dst, deep=False):
        if any(self.n_kv[d] for d in dst):
            self.status |= TAKEN
            return
        asks = []
        for a in src:
            n = self.n_kv[a]
            if deep:
                asks.append(list(range(self.up(n))))
            else:
                asks.append([n // self.pt] if n % self.pt and self.tables[a][n // self.pt] < self.pages else [])
        ids = self._take(sum(map(len, asks)))
        if ids is None:
            return
        for a, d, own in zip(src, dst, asks):
            self.n_kv[d] = self.n_kv[a]
            for j in range(self.up(self.n_kv[a])):
                p = self.tables[a][j]
                if j in own:
                    new = ids.pop(0)
                    if p < self.pages:
                        self._copy(p, new)
                        self.refs[new] = 1
                        p = new
                elif p < self.pages:
                    self.refs[p] += 1
                self.tables[d][j] = p

    def free(self, seqs, keep=None):
        for i, s in enumerate(seqs):
            n = min(self.n_kv[s], keep[i] if keep is not None else 0)
            for j in range(self.up(n), self.up(self.n_kv[s])):
                if self.tables[s][j] < self.pages:
                    self.refs[self.tables[s][j]] -= 1
                self.tables[s][j] = NO_PAGE
            self.n_kv[s] = n

    def compact(self):
        live = [p for p in range(self.pages) if self.refs[p]]
        n = len(live)
        to = {}
        for hole, p in zip([h for h in range(n) if not self.refs[h]], [p for p in live if p >= n]):
            self._copy(p, hole)
            self.refs[hole], self.refs[p] = self.refs[p], 0
            to[p] = hole
        self.tables = [[to.get(p, p) for p in row] for row in self.tables]
        return n

    def check(self):
        """Counts are what the tables say, and nothing lies past a row's end."""
        held = [0] * self.pages
        for s in range(self.rows):
            for j, p in enumerate(self.tables[s]):
                if j >= self.up(self.n_kv[s]):
                    assert p == NO_PAGE
                elif p < self.pages:
                    held[p] += 1
        assert held == self.refs

    def row_bits(self, s):
        """The stored K and V bits of a row's tokens, page by page (None in a hole)."""
        got = []
        for j in range(self.n_kv[s]):
            p = self.tables[s][j // self.pt]
            got.append(None if p >= self.pages else (self.k[:, p, j % self.pt].tobytes(), self.v[:, p, j % self.pt].tobytes()))
        return got


def attend(m, layer, q, scale, rows=None, begin=None, sinks=None, k_new=None, v_new=None):
    """Decode attention of the batch in 64 bits; stores the new tokens in the model. Returns (out,
    the largest |value| and largest sum of |q k| scale met, for tolerances)."""
    n_seq, H, D = q.shape
    group = H // m.kvh
    out = np.zeros((n_seq, H, D))
    vmax = amax = 0.0
    for i in range(n_seq):
        s = i if rows is None else rows[i]
        lo, hi = (0 if begin is None else begin[i]), min(m.n_kv[s], m.max_pages * m.pt)
        at = [(m.tables[s][j // m.pt], j % m.pt) for j in range(lo, hi)]
        if k_new is not None and at and hi == m.n_kv[s] and at[-1][0] < m.pages:
            m.k[layer][at[-1]] = store(k_new[i], m.kv)
            m.v[layer][at[-1]] = store(v_new[i], m.kv)
        at = [a for a in at if a[0] < m.pages]
        if not at:
            continue
        pg, sl = np.array(at).T
        ks, vs = load(m.k[layer][pg, sl], m.kv), load(m.v[layer][pg, sl], m.kv)
        vmax = max(vmax, float(np.abs(vs).max()))
        for h in range(H):
            qh = q[i, h].astype(np.float64)
            amax = max(amax, float((np.abs(ks[:, h // group]) @ np.abs(qh)).max()) * abs(scale))
            x = ks[:, h // group] @ qh * scale
            if sinks is not None:
                x = np.append(x, float(sinks[h]))
            e = np.exp(x - x.max())
            e /= e.sum()
            out[i, h] = e[: len(at)] @ vs[:, h // group]
    return out, vmax, amax


def attend_tolerance(vmax, amax, D, n):
    """Bound on |f32 result - exact| with scores of magnitude amax over n keys. Every score is off by
    (D + 8) roundings of sums of at most amax, by 2^-22 of amax in the split of q into 16-bit terms,
    and the truncations of the tensor core's sums count twice; a weight takes that error twice (its
    own and the maximum's), the exponential's 2^-21 and the 2^-22 of its own split; the sums over
    the keys take a rounding and a rescaling for each tile of 8, twice, and a join of 600 parts at
    most. A convex combination of values up to vmax errs by the weights' relative errors twice
    (numerator and denominator)."""
    score = amax * (2 * (D + 8) * EPS + 2.0 ** -22)
    weight = 2 * score * 1.5 + 2.0 ** -20 + 2.0 ** -21
    sums = (2 * (n / 8) + 64) * EPS
    return 2 * vmax * (weight + sums)
