"""The 4-bit paged cache in 64 bits, position by position: what a group is held as, where a code lies, attention over the
values, and the page tables as Python lists. Independent of the library; CPU tensors in, CPU tensors out."""
import torch

PAGE = 64


def minus(a, b):
    """a - b as d + e exactly."""
    d = a - b
    bb = d - a
    return d, (a - (d - bb)) + (-b - bb)


def held(x):
    """(codes, scales, zeros, values) of x [..., hd] in 64 bits; a group with a NaN or an infinity is NaN. Differences are
    taken exactly: 2^-60 beside 1 is lost in 64 bits, and decides where what is left lies on a border."""
    g = x.double().unflatten(-1, (-1, 32))
    z, top = g.amin(-1), g.amax(-1)
    d, e = minus(top, z)
    low = ((d / 15).float().view(torch.int32) & -65536).view(torch.float32)  # a bf16 at or below, or the next one
    up = (low.view(torch.int32) + 65536).view(torch.float32).double()
    low = low.double()
    s = torch.where((15 * low > d) | ((15 * low == d) & (e <= 0)), low, up)
    d, e = minus(g, z[..., None])
    sc = torch.where(s > 0, s, 1.0)[..., None]
    n = torch.floor(d / sc)
    r = d - (n + 0.5) * sc
    n = n + ((r > 0) | ((r == 0) & ((e > 0) | ((e == 0) & (n % 2 == 1)))))
    v = n * s[..., None] + z[..., None]
    bad = ~torch.isfinite(g).all(-1)
    v = torch.where(bad[..., None], torch.nan, v)
    return n.flatten(-2), s, z, v.flatten(-2)


def page_bytes(nk, hd):
    return nk * 2 * PAGE * (hd // 2 + hd // 8)


def where(hd, kind, p, c):
    """Byte in a (page, head) unit and shift of the code of position p, channel c; bytes of its scale and its zero."""
    W = hd // 32
    half = (p // 32) * (32 * hd + 256 * W)
    w, r = c // 32, p % 8
    if kind == "k":
        lane, bit = 4 * r + (c % 32) // 8, 16 * (c % 2) + 4 * ((c % 8) // 2)
    else:
        lane, bit = 4 * ((c % 32) // 4) + r // 2, 16 * (r % 2) + 4 * (c % 4)
    at = half + (0 if kind == "k" else 16 * hd) + (p % 32) // 8 * 4 * hd + (lane * W + w) * 4 + bit // 8
    meta = half + 32 * hd + (0 if kind == "k" else 128 * W) + (p % 32) * 4 * W
    return at, bit % 8, meta + 2 * w, meta + 2 * W + 2 * w


_maps = {}


def _map(hd, kind):
    if (hd, kind) not in _maps:
        m = torch.tensor([[where(hd, kind, p, c) for c in range(hd)] for p in range(PAGE)])
        _maps[hd, kind] = m.reshape(-1, 4).unbind(1)
    return _maps[hd, kind]


def pool_values(pool, nk, hd):
    """K and V [npages][nk][64][hd] in 64 bits, and their scales, of a pool's bytes (CPU uint8)."""
    u = pool.view(pool.shape[0], nk, -1).long()
    out = []
    for kind in "kv":
        at, sh, ms, mz = _map(hd, kind)
        code = (u[..., at] >> sh) & 15

        def bf(m):
            return (u[..., m] | u[..., m + 1] << 8).to(torch.int32).__lshift__(16).view(torch.float32).double()

        s = bf(ms)
        out += [(code * s + bf(mz)).unflatten(-1, (PAGE, hd)), s.unflatten(-1, (PAGE, hd))]
    return out  # k, k scales, v, v scales


def take_values(pool, row, n, nk, hd):
    """K, V and V's scales [nk][n][hd] of a take with table row `row` (a list)."""
    pages = torch.tensor(row[:-(-n // PAGE)], dtype=torch.long)
    k, _, v, vs = pool_values(pool[pages], nk, hd)
    return [x.transpose(0, 1).flatten(1, 2)[:, :n] for x in (k, v, vs)]


def attend(q, k, v, scale):
    """q [nq][hd], k and v [nk][n][hd] in 64 bits -> [nq][hd]."""
    G = q.shape[0] // k.shape[0]
    w = torch.softmax(torch.einsum("hgd,hnd->hgn", q.double().view(k.shape[0], G, -1), k) * scale, -1)
    return torch.einsum("hgn,hnd->hgd", w, v).flatten(0, 1)


class Pages:
    """Tables, counts and lengths; `moved` collects page copies (from, to) in order."""

    def __init__(self, B, npages, maxpages):
        self.B, self.npages, self.maxpages = B, npages, maxpages
        self.table = [[-1] * maxpages for _ in range(B)]
        self.ref, self.lens, self.moved = [0] * npages, [0] * B, []

    def lowest(self):
        return next((i for i, r in enumerate(self.ref) if r == 0), None)

    def release(self, s):
        for k, p in enumerate(self.table[s]):
            if p >= 0:
                self.ref[p] -= 1
                self.table[s][k] = -1
        self.lens[s] = 0

    def extend(self, extra):
        missing = 0
        for s in range(self.B):
            for k in range(-(-(self.lens[s] + extra) // PAGE) if self.lens[s] > 0 else 0):
                if self.table[s][k] < 0:
                    p = self.lowest()
                    if p is None:
                        missing += 1
                    else:
                        self.table[s][k], self.ref[p] = p, 1
        return missing

    def fork(self, src, dst):
        ok = [0 <= a < self.B and 0 <= b < self.B and a != b and b not in dst[:i] and a not in dst
              for i, (a, b) in enumerate(zip(src, dst))]
        for a, b, k in zip(src, dst, ok):
            if k:
                self.release(b)
        for a, b, k in zip(src, dst, ok):
            if k:
                self.lens[b] = self.lens[a]
                for i in range(self.lens[a] // PAGE):
                    self.table[b][i] = self.table[a][i]
                    self.ref[self.table[a][i]] += 1
        need = [(a, b) for a, b, k in zip(src, dst, ok) if k and self.lens[a] % PAGE]
        short = []
        for a, b in need:
            p, i = self.lowest(), self.lens[a] // PAGE
            if p is None:
                short.append(b)
            else:
                self.table[b][i], self.ref[p] = p, 1
                self.moved.append((self.table[a][i], p))
        for b in short:
            self.release(b)
        return len(short), all(ok)

    def compact(self):
        live = sum(r > 0 for r in self.ref)
        holes = [i for i in range(live) if self.ref[i] == 0]
        movers = [i for i in range(live, self.npages) if self.ref[i] > 0]
        to = dict(zip(movers, holes))
        for a, b in to.items():
            self.ref[b], self.ref[a] = self.ref[a], 0
            self.moved.append((a, b))
        self.table = [[to.get(p, p) for p in row] for row in self.table]
        return live, len(movers)
