"""The 8-bit key/value cache in 64 bits, from its definition (test infrastructure): E4M3 numbers by a table of all codes, power-of-two
scales, causal attention, eviction.  Everything on the CPU, one sequence and one head at a time."""
import torch

F64 = torch.float64


def _table():
    vals = []
    for c in range(128):
        e, m = c >> 3, c & 7
        vals.append(float("nan") if c == 127 else (m / 8 * 2.0 ** -6 if e == 0 else (1 + m / 8) * 2.0 ** (e - 7)))
    return torch.tensor(vals + [-v for v in vals], dtype=F64)


VALUES = _table()  # of the codes 0 .. 255
_POS = VALUES[:127]


def encode(x):
    """Codes of the nearest numbers to x (f64, |x| <= 448), ties to the even code; what is not finite: NaN."""
    a = x.abs()
    fine = torch.isfinite(x)
    a = torch.where(fine, a, torch.zeros_like(a))
    hi = torch.searchsorted(_POS, a.contiguous()).clamp(max=126)
    lo = (hi - 1).clamp(min=0)
    dl, dh = a - _POS[lo], _POS[hi] - a
    code = torch.where((dl < dh) | ((dl == dh) & (lo % 2 == 0)), lo, hi)
    code = torch.where(fine, code, torch.full_like(code, 127))
    return (code + 128 * torch.signbit(x)).to(torch.uint8)


def scale_of(x):
    """Scale of a block with the numbers x."""
    x = x[torch.isfinite(x)].abs()
    k, top = -126, float(x.max()) if x.numel() else 0.0
    while 448 * 2.0 ** k < top:
        k += 1
    return 2.0 ** k


class Cache:
    """codes [slots, heads, cap, dim] uint8, scales [slots, heads, blocks] f64, weights [slots, heads, cap] f64 or None."""

    def __init__(self, k, v, ks, vs, block, weights=None):
        self.k, self.v, self.ks, self.vs, self.block = k.clone(), v.clone(), ks.double().clone(), vs.double().clone(), block
        self.weights = None if weights is None else weights.double().clone()

    def _store(self, codes, scales, slot, h, first, x, floor=None):
        """x [tokens, dim] at `first` ..; floor: scale that the first block keeps at least."""
        B = self.block
        for b in range(first // B, (first + len(x) - 1) // B + 1):
            lo, hi = max(first, b * B), min(first + len(x), (b + 1) * B)
            s = scale_of(x[lo - first:hi - first])
            if lo > b * B:
                was = float(scales[slot, h, b])
                s = max(s, was)
                codes[slot, h, b * B:lo] = encode(VALUES[codes[slot, h, b * B:lo].long()] * (was / s))
            codes[slot, h, lo:hi] = encode(x[lo - first:hi - first] / s)
            scales[slot, h, b] = s

    def append(self, k, v, entries):
        for slot, pos, row, n in entries:
            for h in range(self.k.shape[1]):
                if n:
                    self._store(self.k, self.ks, slot, h, pos, k[row:row + n, h].double())
                    self._store(self.v, self.vs, slot, h, pos, v[row:row + n, h].double())
                if self.weights is not None:
                    self.weights[slot, h, pos:pos + n] = 0.0

    def held(self, slot, h, n):
        of = torch.arange(n) // self.block
        return (VALUES[self.k[slot, h, :n].long()] * self.ks[slot, h][of][:, None],
                VALUES[self.v[slot, h, :n].long()] * self.vs[slot, h][of][:, None])

    def attention(self, q, scale, entries, softcap=0.0, sink=None, gate=None, decay=None):
        """-> out, lse [rows, heads], and for bounds on errors: sum p |v|, sum |q| |k| (largest over the keys); rows of no entry are 0."""
        rows, heads, _ = q.shape
        H, V = self.k.shape[1], self.v.shape[3]
        G = heads // H
        out, mass = torch.zeros(rows, heads, V, dtype=F64), torch.zeros(rows, heads, V, dtype=F64)
        lse, dots = torch.zeros(rows, heads, dtype=F64), torch.zeros(rows, heads, dtype=F64)
        for slot, pos, row, n in entries:
            if not n:
                continue
            for h in range(H):
                k, v = self.held(slot, h, pos + n)
                got = torch.zeros(pos + n, dtype=F64)
                for i in range(n):
                    live = pos + i + 1
                    for g in range(h * G, (h + 1) * G):
                        qi = q[row + i, g].double()
                        s = k[:live] @ qi * scale
                        if softcap:
                            s = softcap * torch.tanh(s / softcap)
                        both = s if sink is None else torch.cat([s, sink[g].double().view(1)])
                        z = torch.logsumexp(both, 0)
                        p = torch.exp(s - z)
                        got[:live] += p
                        out[row + i, g], mass[row + i, g] = p @ v[:live], p @ v[:live].abs()
                        lse[row + i, g] = z
                        dots[row + i, g] = float((k[:live].abs() @ qi.abs()).max()) * abs(scale)
                if decay is not None:
                    old = self.weights[slot, h, :pos + n]
                    self.weights[slot, h, :pos + n] = got if decay == 0 else decay * old + got
        if gate is not None:
            f = torch.sigmoid(gate.double()).view(rows, heads, V)
            out, mass = out * f, mass * f
        return out, lse, mass, dots

    def evict(self, table, keep, recent):
        kept = torch.full((len(table), self.k.shape[1], keep), -1, dtype=torch.int32)
        for e, (slot, n, _, _) in enumerate(table):
            for h in range(self.k.shape[1]):
                if n <= keep:
                    at = list(range(n))
                else:
                    w = [float("-inf") if x != x else x for x in self.weights[slot, h, :n - recent].tolist()]
                    nan = [x != x for x in self.weights[slot, h, :n - recent].tolist()]
                    best = sorted(range(n - recent), key=lambda j: (nan[j], -w[j], j))[:keep - recent]
                    at = sorted(best) + list(range(n - recent, n))
                kept[e, h, :len(at)] = torch.tensor(at, dtype=torch.int32)
                if not at:
                    continue
                k, v = self.held(slot, h, n)
                self._store(self.k, self.ks, slot, h, 0, k[at])
                self._store(self.v, self.vs, slot, h, 0, v[at])
                self.weights[slot, h, :len(at)] = self.weights[slot, h, at]
        return kept
