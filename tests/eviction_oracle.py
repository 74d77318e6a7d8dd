"""Plain 64-bit forms of the attention weight of cached keys and of eviction, on the CPU, for their tests.

weights_exact also returns an error bound. A weight p = exp(s - L) of a row, L = log sum_j exp(s_j), is
off relative to itself by at most

  2 (D + 8) 2^-24 S    the scores' D-term sums and scale, in s and (log-sum-exp moves no more than its
                       scores) in L; S the largest sum_j |q_j k_j| scale of the row's keys
  (len / 32 + 16) 2^-24   the sum over the row's keys: one addition a tile of 32 to a running sum, some
                       within a tile and where waves and splits meet
  4 (S + ln len + 1) 2^-24  L, the kept score and their difference, each rounded once
  2^-20                exp2 and log2

and the sum over R rows by another (R / 8 + 32) 2^-24 (four chains a lane, parts of 1024 rows); the old
sum times the decay and the addition to it by 2^-24 each.
"""
import math

import torch


def weights_exact(scores, q, k, table, lens, cu, page, last, decay=1.0, scale=None):
    """(scores, bound): float64 [B, Hkv, S]."""
    t, hq, d = q.shape
    hk, pool = k.shape[1], k.shape[0]
    g = hq // hk
    scale = d ** -0.5 if scale is None else scale
    out = scores.double().clone()
    bound = torch.zeros_like(out)
    unit = 2.0 ** -24
    capacity = table.shape[1] * page
    for b in range(table.shape[0]):
        first, n = int(cu[b]), int(cu[b + 1]) - int(cu[b])
        length = min(max(int(lens[b]), 0), capacity)
        if n == 0 or length == 0:
            continue
        used = min(n, last)
        pos = torch.arange(length)
        ids = table[b].long()[pos // page]
        rows = ids * page + pos % page
        inside = (rows >= 0) & (rows < pool)
        at = torch.arange(n - used, n) + length - n
        seen = pos[None] <= at[:, None]
        kk = torch.where(inside[:, None, None], k[torch.where(inside, rows, 0)].double(), 0.0)
        old = max(0, length - n)
        for h in range(hk):
            total, slack = torch.zeros(length, dtype=torch.float64), torch.zeros(length, dtype=torch.float64)
            for j in range(h * g, (h + 1) * g):
                x = q[first + n - used:first + n, j].double()
                s = (x @ kk[:, h].T * scale).masked_fill(~seen, -math.inf)
                top = s.amax(-1, keepdim=True)
                p = torch.exp(s - torch.where(top > -math.inf, top, 0.0))
                p = torch.where(seen, p / p.sum(-1, keepdim=True), 0.0)
                size = (x.abs() @ kk[:, h].abs().T * scale).masked_fill(~seen, 0.0).amax(-1, keepdim=True)
                e = unit * (2 * (d + 8) * size + length / 32 + 16 + 4 * (size + math.log(length) + 1)) + 2.0 ** -20
                total += p.sum(0)
                slack += (p * e).sum(0) + 1e-30 * used
            row = out[b, h]
            before = row[:length] * decay if decay else torch.zeros(length, dtype=torch.float64)
            before[old:] = 0.0
            row[:length] = before + total
            bound[b, h, :length] = slack + unit * (g * used / 8 + 32) * total + 2 * unit * (before.abs() + total)
    return out, bound


def evict_exact(k_pools, v_pools, scores, refs, table, lens, keep, page, first=0, recent=0):
    """Books, pools and scores (all on the CPU, changed in place) after an eviction; returns the status."""
    pages, (rows, width) = refs.numel(), table.shape
    still = first // page
    free = [i for i in range(pages) if int(refs[i]) == 0]
    left, short, bad, given, todo = len(free), 0, 0, 0, []
    for r in range(rows):
        length, budget = min(max(int(lens[r]), 0), width * page), int(keep[r])
        if budget < 0 or budget >= length:
            continue
        if budget < first + recent:
            bad += 1
            continue
        need = -(-budget // page) - still
        if need and given + need > left:
            short += 1
        else:
            todo.append((r, length, budget, free[given:given + need]))
        given += need
    old = table.clone()
    for r, length, budget, fresh in todo:
        for at, pools in enumerate(zip(scores, k_pools, v_pools)):
            x, ks, vs = pools
            for h in range(x.shape[1]):
                value = [float(y) if not math.isnan(float(y)) else -math.inf for y in x[r, h, first:length - recent]]
                order = sorted(range(len(value)), key=lambda i: (-value[i], i))[:budget - first - recent]
                kept = list(range(first)) + [first + i for i in sorted(order)] + list(range(length - recent, length))
                x[r, h, :budget] = x[r, h, kept].clone()
                for d in range(still * page, budget):
                    s = kept[d]
                    src, dst = int(old[r, s // page]) * page + s % page, fresh[d // page - still] * page + d % page
                    ks[dst, h], vs[dst, h] = ks[src, h], vs[src, h]
        for j in range(still, -(-length // page)):
            refs[int(old[r, j])] -= 1
        for i in fresh:
            refs[i] = 1
        table[r, still:] = -1
        table[r, still:still + len(fresh)] = torch.tensor(fresh, dtype=torch.int32)
        lens[r] = budget
    return [short, bad]
