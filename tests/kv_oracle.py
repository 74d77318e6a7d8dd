"""Plain 64-bit forms of the operators around the paged cache, on the CPU, for their tests.

extend_exact also returns what its error bound needs. With o = sum_k p_k v_k / sum_k p_k, a kernel
that holds scores, p and sums in fp32, rounds p to the input type for the product with V and the
result to the input type is off, in each element, by at most

  half |o|                       the last rounding, half = eps / 2 of the type
  + half A                       the rounding of p, A = sum_k p_k |v_k| / sum_k p_k
  + 2 d A                        errors d of the scores (relative ones of p, in sum and product):
                                 d = (D + 8) 2^-24 S, S the largest sum_j |q_j k_j| scale of the row's
                                 keys, for the D-term sums, the scale and the exponent; and 2^-20
                                 for exp2, the sums and the divisions
  + n 2^-25 V (fp16)             p below fp16's smallest normal, n keys, V the largest |v|: the sum
                                 of p is at least 1, since the exponent reference never exceeds
                                 the maximum
"""
import math

import torch


def extend_exact(q, k, v, table, lens, cu, page, causal=True, window=0, scale=None):
    """(o, bound): float64 [T, Hq, D]; rows behind cu[-1] are NaN in o."""
    t, hq, d = q.shape
    hk = k.shape[1]
    g = hq // hk
    pool = k.shape[0]
    scale = d ** -0.5 if scale is None else scale
    half = torch.finfo(q.dtype).eps / 2
    out = torch.full((t, hq, d), math.nan, dtype=torch.float64)
    bound = torch.zeros_like(out)
    capacity = table.shape[1] * page
    for b in range(table.shape[0]):
        first, n = int(cu[b]), int(cu[b + 1]) - int(cu[b])
        length = min(max(int(lens[b]), 0), capacity)
        if n == 0:
            continue
        out[first:first + n] = 0.0
        pos = torch.arange(length)
        ids = table[b].long()[pos // page]
        rows = ids * page + pos % page
        inside = (rows >= 0) & (rows < pool)
        at = torch.arange(n) + length - n
        seen = pos[None] <= at[:, None] if causal else torch.ones(n, length, dtype=torch.bool)
        if window:
            seen &= pos[None] > at[:, None] - window
        used = inside & seen.any(0)
        safe = torch.where(used, rows, 0)
        kk = torch.where(used[:, None, None], k[safe].double(), 0.0)
        vv = torch.where(used[:, None, None], v[safe].double(), 0.0)
        for h in range(hq):
            x = q[first:first + n, h].double()
            s = x @ kk[:, h // g].T * scale
            s = s.masked_fill(~seen, -math.inf)
            top = s.amax(-1, keepdim=True) if length else torch.full((n, 1), -math.inf, dtype=s.dtype)
            p = torch.exp(s - top.clamp_min(-1e300))
            total = p.sum(-1, keepdim=True)
            p = torch.where(total > 0, p / total, 0.0)
            o = p @ vv[:, h // g]
            size = (x.abs() @ kk[:, h // g].abs().T * scale).masked_fill(~seen, 0.0)
            delta = (d + 8) * 2.0 ** -24 * (size.amax(-1, keepdim=True) if length else 0.0) + 2.0 ** -20
            a = p @ vv[:, h // g].abs()
            out[first:first + n, h] = o
            bound[first:first + n, h] = half * o.abs() + (half + 2 * delta) * a + 1e-30
            if q.dtype == torch.float16 and length:
                small = seen.sum(-1, keepdim=True) * 2.0 ** -25 * vv[:, h // g].abs().max()
                # (and results below fp16's smallest normal round to its fixed step)
                bound[first:first + n, h] += small + 2.0 ** -25
    return out, bound


def frequencies(dim, base=10000.0, scaling=None):
    """Angles a position, float64, from the formulas of the four scalings, and the factor."""
    w = torch.tensor([base ** (-2 * i / dim) for i in range(dim // 2)], dtype=torch.float64)
    if scaling is None:
        return w, 1.0
    f, kind = scaling["factor"], scaling["kind"]
    if kind == "linear":
        return w / f, 1.0
    if kind == "base":
        return (base * f ** (dim / (dim - 2))) ** (-torch.arange(0, dim, 2, dtype=torch.float64) / dim), 1.0
    turns = scaling["original"] * w / (2 * math.pi)
    if kind == "bands":
        low, high = scaling.get("low", 1.0), scaling.get("high", 4.0)
        keep = ((turns - low) / (high - low)).clamp(0, 1)
        return w * (keep + (1 - keep) / f), 1.0
    def where(n):  # pair that makes n turns: base ** (-2 i / dim) * L = 2 pi n
        return dim / 2 * math.log(scaling["original"] / (2 * math.pi * n), base)
    low = max(math.floor(where(scaling.get("beta_fast", 32.0))), 0)
    high = min(math.ceil(where(scaling.get("beta_slow", 1.0))), dim - 1)
    slow = ((torch.arange(dim // 2, dtype=torch.float64) - low) / max(high - low, 0.001)).clamp(0, 1)
    scale = scaling.get("attention") or (0.1 * math.log(f) + 1 if f > 1 else 1.0)
    return w * (1 - slow) + w / f * slow, scale


def rotate_exact(x, positions, dim, base=10000.0, interleaved=False, scaling=None, inverse=False):
    """(x', bound): float64. The bound: half a step of the type on the result, and of the fp32 parts
    |a| + |b| times s times 5 2^-24 (cosine and sine to 3 2^-24, two products and a sum)."""
    w, s = frequencies(dim, base, scaling)
    t = positions.double()[:, None] * w * (-1 if inverse else 1)
    c, n = torch.cos(t)[:, None] * s, torch.sin(t)[:, None] * s
    y = x.double()
    out, size = y.clone(), torch.zeros_like(y)
    if interleaved:
        a, b = slice(0, dim, 2), slice(1, dim, 2)
    else:
        a, b = slice(0, dim // 2), slice(dim // 2, dim)
    out[..., a] = y[..., a] * c - y[..., b] * n
    out[..., b] = y[..., b] * c + y[..., a] * n
    size[..., a] = size[..., b] = (y[..., a].abs() + y[..., b].abs()) * s
    half = torch.finfo(x.dtype).eps / 2 if x.dtype != torch.float32 else 0.0
    bound = half * out.abs() + size * 5 * 2.0 ** -24 * (1 + half)
    if x.dtype == torch.float16:
        bound[..., :dim] += 2.0 ** -25
    return out, bound


# ---- books of pages, with Python integers ---------------------------------------------------------

class Books:
    def __init__(self, refs, table, lens, page):
        self.refs, self.lens, self.page = refs.tolist(), lens.tolist(), page
        self.table = table.tolist()
        self.width = table.shape[1]

    def pages_of(self, r):
        return self.table[r][:-(-self.lens[r] // self.page)]

    def free_pages(self):
        return [i for i, n in enumerate(self.refs) if n == 0]

    def reserve(self, counts):
        free, status, asked = self.free_pages(), [0, 0], 0
        for r, add in enumerate(counts):
            if add < 0 or self.lens[r] + add > self.width * self.page:
                status[1] += 1
                continue
            have = -(-self.lens[r] // self.page)
            need = -(-(self.lens[r] + add) // self.page) - have
            asked += need
            if need and asked > len(free):
                status[0] += 1
                continue
            for j in range(need):
                page = free[asked - need + j]
                self.table[r][have + j], self.refs[page] = page, 1
            self.lens[r] += add
        return status

    def fork(self, parents, children):
        """(status, [(from, to)])"""
        free, status, moves = self.free_pages(), [0, 0], []
        rows, before = len(self.lens), [list(r) for r in self.table]
        empty, asked = [n == 0 for n in self.lens], 0
        lens = list(self.lens)
        for i, (p, c) in enumerate(zip(parents, children)):
            if not (0 <= p < rows and 0 <= c < rows and empty[c]) or c in parents or c in children[:i]:
                status[1] += 1
                continue
            whole, rest = divmod(lens[p], self.page)
            if rest:
                asked += 1
                if asked > len(free):
                    status[0] += 1
                    continue
            self.table[c] = before[p][:whole] + [-1] * (self.width - whole)
            for page in before[p][:whole]:
                self.refs[page] += 1
            if rest:
                page = free[asked - 1]
                self.table[c][whole], self.refs[page] = page, 1
                moves.append((before[p][whole], page))
            self.lens[c] = lens[p]
        return status, moves

    def free(self, rows):
        for r in rows:
            if 0 <= r < len(self.lens) and self.lens[r]:
                for page in self.pages_of(r):
                    self.refs[page] -= 1
                self.table[r], self.lens[r] = [-1] * self.width, 0

    def compact(self):
        live = sum(n > 0 for n in self.refs)
        out = [i for i in range(live, len(self.refs)) if self.refs[i] > 0]
        into = [i for i in range(live) if self.refs[i] == 0]
        moves = list(zip(out, into))
        place = dict(moves)
        for a, b in moves:
            self.refs[b], self.refs[a] = self.refs[a], 0
        for r, row in enumerate(self.table):
            n = len(self.pages_of(r))
            row[:n] = [place.get(x, x) for x in row[:n]]
        return moves
