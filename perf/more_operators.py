"""Operators for many samples of one prompt on a bounded cache, whose time is tracked.

A case is one pass through one operator, `op` says which:
  "shared"   attention of each request's new tokens over the paged cache where groups of requests share a
             long prefix (forked samples, a common system prompt): the prefix is read once for a group;
  "weights"  the attention weight that each cached key gets from new tokens, summed over tokens and query
             heads, added to running sums for each K/V head;
  "evict"    rows shortened to a budget: each layer and K/V head keeps its first, its last and its
             heaviest keys, moved together with their sums onto fresh pages.
With `own` false, `run` computes the same in elementary torch operations.
"""
import math

import torch

own = False

_DTYPES = {"bfloat16": torch.bfloat16, "float16": torch.float16}
_MAX_FLOPS = 2.4e11  # of a drawn case: under the largest listed one
_MAX_BYTES = 3.9e8
_MAX_POOLS = 1.5e9


def _shared(name, groups, members, new, heads, kv_heads, dim, page, prefix, suffix, dtype, ragged=True):
    return dict(name=name, op="shared", groups=groups, members=members, new=new, heads=heads,
                kv_heads=kv_heads, dim=dim, page=page, prefix=prefix, suffix=suffix, dtype=dtype,
                ragged=ragged)


def _weights(name, batch, new, last, heads, kv_heads, dim, page, capacity, dtype, decay, ragged=True):
    return dict(name=name, op="weights", batch=batch, new=new, last=last, heads=heads, kv_heads=kv_heads,
                dim=dim, page=page, capacity=capacity, dtype=dtype, decay=decay, ragged=ragged)


def _evict(name, layers, rows, heads, dim, page, width, keep, first, recent, dtype, ties=False):
    return dict(name=name, op="evict", layers=layers, rows=rows, heads=heads, dim=dim, page=page,
                width=width, keep=keep, first=first, recent=recent, dtype=dtype, ties=ties)


def listed():
    bf, fp = "bfloat16", "float16"
    return [
        # Two samples of a short prompt: latency alone.
        _shared("shared_two", 1, 2, 1, 8, 2, 64, 16, 300, 40, bf),
        # A decode step of 64 samples of one long prompt, each some hundred tokens on.
        _shared("shared_samples", 1, 64, 1, 32, 8, 128, 64, 8192, 512, bf),
        # Draft tokens checked for the samples of four prompts, whose pages end within the prefix.
        _shared("shared_verify", 4, 6, 5, 32, 8, 80, 16, 3001, 200, fp),
        # Whole user prompts behind a common system prompt, the largest call.
        _shared("shared_prompts", 1, 8, 512, 32, 8, 128, 64, 4096, 512, bf),
        # One new token of one request, sums of this step alone: latency.
        _weights("weights_one", 1, 1, 1, 8, 2, 64, 16, 512, bf, 0.0),
        # A decode step of a serving batch in mid-flight adds to its sums.
        _weights("weights_decode", 32, 1, 1, 32, 8, 128, 64, 4096, bf, 1.0),
        # The last tokens of long prompts look back over all of it, with a decay.
        _weights("weights_window", 3, 4001, 32, 16, 4, 96, 48, 12288, fp, 0.5),
        # Every token of whole prompts counts.
        _weights("weights_prompt", 2, 4096, 4096, 32, 8, 128, 64, 4096, bf, 1.0, False),
        # One row of one layer past its budget: latency alone.
        _evict("evict_one", 1, 1, 8, 64, 16, 24, 200, 4, 32, fp),
        # A batch of samples cut to a quarter, four layers; equal sums among the scores.
        _evict("evict_batch", 4, 16, 8, 128, 16, 256, 1000, 20, 128, bf, True),
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, round(lo * (hi / lo) ** rng.random())))


def _draw_heads(rng):
    kv_heads = rng.choice((1, 2, 4, 8, 8))
    return kv_heads * rng.choice((1, 2, 3, 4, 4, 6, 8)), kv_heads


def _draw_shared(rng):
    heads, kv_heads = _draw_heads(rng)
    new = rng.choice((1, 1, 1, rng.randint(2, 17), _log_int(rng, 18, 600)))
    return _shared(None, rng.choice((1, 1, 2, rng.randint(3, 9))), _log_int(rng, 1, 64), new, heads, kv_heads,
                   rng.choice((64, 80, 96, 128, 128, 128, 192, 256)), rng.choice((16, 16, 32, 48, 64, 64, 128)),
                   _log_int(rng, 40, 32000), new + _log_int(rng, 1, 1024),
                   rng.choice(("bfloat16", "bfloat16", "float16")), rng.random() < 0.8)


def _draw_weights(rng):
    heads, kv_heads = _draw_heads(rng)
    page = rng.choice((16, 16, 32, 48, 64, 64, 128))
    kind = rng.choice(("decode", "decode", "verify", "window", "prompt"))
    batch = _log_int(rng, 1, 64)
    if kind == "decode":
        new = last = 1
        cap = _log_int(rng, 128, 32768)
    elif kind == "verify":
        new = last = rng.randint(2, 17)
        cap = _log_int(rng, 128, 16384)
    elif kind == "window":
        new, last = _log_int(rng, 64, 8192), rng.randint(8, 64)
        cap, batch = new + _log_int(rng, 1, 8192), _log_int(rng, 1, 8)
    else:
        new = last = _log_int(rng, 64, 4096)
        cap, batch = new + rng.choice((0, 0, _log_int(rng, 1, 2048))), _log_int(rng, 1, 4)
    return _weights(None, batch, new, last, heads, kv_heads,
                    rng.choice((64, 80, 96, 128, 128, 128, 192, 256)), page, -(-max(cap, new) // page) * page,
                    rng.choice(("bfloat16", "bfloat16", "float16")), rng.choice((0.0, 1.0, 0.9)),
                    rng.random() < 0.7)


def _draw_evict(rng):
    page, width = rng.choice((16, 16, 32, 64)), _log_int(rng, 6, 400)
    cap = page * width
    first, recent = rng.choice((0, 4, 33)), rng.choice((0, 1, 16, 64))
    return _evict(None, rng.choice((1, 2, 4, 8)), _log_int(rng, 1, 32), rng.choice((1, 2, 4, 8)),
                  rng.choice((64, 80, 128, 128, 256)), page, width,
                  max(first + recent, min(cap - 1, _log_int(rng, 8, max(16, cap // 2)))), first, recent,
                  rng.choice(("bfloat16", "float16")), rng.random() < 0.4)


def draw(rng):
    """A case of the listed ranges: odd sizes, ragged batches, every page size and type."""
    case = rng.choice((_draw_shared, _draw_weights, _draw_evict))(rng)
    del case["name"]
    while _too_large(case):
        if case["op"] == "shared":
            key = "members" if case["members"] > 2 else "new" if case["new"] > 64 else "prefix"
            if key == "new":
                case["suffix"] -= case["new"] - case["new"] // 2
            case[key] //= 2
        elif case["op"] == "weights":
            key = "batch" if case["batch"] > 1 else "last" if case["last"] > 64 else "heads"
            if key == "heads":
                case["heads"] = case["kv_heads"]
                case["capacity"] = max(case["new"], case["capacity"] // 2 // case["page"] * case["page"])
                case["capacity"] = -(-case["capacity"] // case["page"]) * case["page"]
            else:
                case[key] //= 2
        else:
            key = "layers" if case["layers"] > 1 else "rows" if case["rows"] > 1 else "heads"
            case[key] //= 2
    return case


def _too_large(case):
    w = work(case)
    if w["flops"] > _MAX_FLOPS or w["bytes"] > _MAX_BYTES:
        return True
    if case["op"] == "evict":
        return _evict_pages(case) * case["page"] * case["heads"] * case["dim"] * 4 * case["layers"] > _MAX_POOLS
    return False


# ---- sizes that follow from a case ---------------------------------------------------------------

def _spread(low, high, i, n):
    return low + (high - low) * (2 * i + 1) // (2 * n)


def _shared_sizes(case):
    """(prefix of each group, members of each group, new tokens and own keys of each request): the last
    counts the new tokens."""
    g, m = case["groups"], case["members"]
    if not case["ragged"]:
        return [case["prefix"]] * g, [m] * g, [case["new"]] * (g * m), [case["suffix"]] * (g * m)
    prefixes = [max(1, case["prefix"] - case["prefix"] * i // (2 * g)) for i in range(g)]
    members = [max(1, m - i % 3) for i in range(g)]
    n = sum(members)
    news = [max(1, case["new"] - i % 4 * (case["new"] // 9)) for i in range(n)]
    own_keys = [max(k, _spread(case["suffix"] // 4, case["suffix"], i, n)) for i, k in enumerate(news)]
    return prefixes, members, news, own_keys


def _weights_sizes(case):
    """(new tokens, cache lengths with them) of each request."""
    b, cap = case["batch"], case["capacity"]
    if not case["ragged"]:
        return [case["new"]] * b, [cap] * b
    news = [max(1, case["new"] - i % 4 * (case["new"] // 7)) for i in range(b)]
    return news, [max(n, _spread(cap // 4, cap, i, b)) for i, n in enumerate(news)]


def _evict_layout(case):
    """Lengths, budgets (-1: the row stays) and shared whole pages of each row: odd rows hold the first
    pages of the row before, as a forked sample does."""
    rows, page, cap = case["rows"], case["page"], case["width"] * case["page"]
    lens = [max(1, _spread(cap // 2, cap, r, rows) - r % 5) for r in range(rows)]
    if rows == 1:
        lens = [cap - 3]
    keep = [-1 if r % 4 == 3 else case["keep"] for r in range(rows)]
    shared = [min(lens[r], lens[r - 1]) // page // 3 if r % 2 else 0 for r in range(rows)]
    return lens, keep, shared


def _evict_fresh(case):
    lens, keep, _ = _evict_layout(case)
    page = case["page"]
    return [-(-k // page) - case["first"] // page if 0 <= k < n else 0 for n, k in zip(lens, keep)]


def _evict_pages(case):
    lens, _, shared = _evict_layout(case)
    return sum(-(-n // case["page"]) - s for n, s in zip(lens, shared)) + sum(_evict_fresh(case)) + 7


def work(case):
    """Inputs read once, outputs written once; 4 D flops for a visible pair's score and its value, 2 D for
    its score alone."""
    if case["op"] == "evict":
        lens, keep, _ = _evict_layout(case)
        page, still = case["page"], case["first"] // case["page"] * case["page"]
        moved = sum(k - still for n, k in zip(lens, keep) if 0 <= k < n)
        sums = sum(n + k for n, k in zip(lens, keep) if 0 <= k < n)
        books = 8 * (_evict_pages(case) + case["rows"] * (case["width"] + 1))
        return {"bytes": case["layers"] * case["heads"] * (8 * case["dim"] * moved + 4 * sums) + books, "flops": 0}
    h, hk, d = case["heads"], case["kv_heads"], case["dim"]
    if case["op"] == "shared":
        prefixes, members, news, own_keys = _shared_sizes(case)
        of = [p for p, m in zip(prefixes, members) for _ in range(m)]
        pairs = sum(n * (p + k - n) + n * (n + 1) // 2 for p, n, k in zip(of, news, own_keys))
        keys = sum(prefixes) + sum(own_keys)
        return {"bytes": 4 * keys * hk * d + 4 * sum(news) * h * d + 4 * keys // case["page"],
                "flops": 4 * h * d * pairs}
    news, lens = _weights_sizes(case)
    used = [min(n, case["last"]) for n in news]
    pairs = sum(u * (n - u) + u * (u + 1) // 2 for u, n in zip(used, lens))
    old = sum(n - m for n, m in zip(lens, news)) if case["decay"] else 0
    return {"bytes": 2 * sum(lens) * hk * d + 2 * sum(used) * h * d + 4 * hk * (old + sum(lens))
            + 4 * sum(lens) // case["page"], "flops": 2 * h * d * pairs}


# ---- inputs ---------------------------------------------------------------------------------------

def _offsets(counts):
    out = [0]
    for n in counts:
        out.append(out[-1] + n)
    return out


def _ints(x):
    return torch.tensor(x, dtype=torch.int32, device="cuda")


def _shared_inputs(case, seed):
    """The cache as forks leave it: the whole pages of a prefix in every row of its group, the page that
    it fills in part copied for each of them."""
    gen = torch.Generator(device="cuda").manual_seed(seed)
    dtype, page, hk, d = _DTYPES[case["dtype"]], case["page"], case["kv_heads"], case["dim"]
    prefixes, members, news, own_keys = _shared_sizes(case)
    group = [g for g, m in enumerate(members) for _ in range(m)]
    lens = [prefixes[g] + k for g, k in zip(group, own_keys)]
    width = max(-(-n // page) for n in lens) + 1
    pages = sum(p // page for p in prefixes) + sum(-(-n // page) - prefixes[g] // page for g, n in zip(group, lens)) + 3
    ids = torch.randperm(pages, generator=torch.Generator().manual_seed(seed)).tolist()
    common = [[ids.pop() for _ in range(p // page)] for p in prefixes]
    table, first = [], _offsets(members)
    for g, n in zip(group, lens):
        row = common[g] + [ids.pop() for _ in range(-(-n // page) - len(common[g]))]
        table.append(row + [-1] * (width - len(row)))
    shape = (pages * page, hk, d)
    k = torch.randn(shape, generator=gen, device="cuda", dtype=dtype)
    v = torch.randn(shape, generator=gen, device="cuda", dtype=dtype)
    for b, g in enumerate(group):
        whole, rest = divmod(prefixes[g], page)
        if rest and b != first[g]:
            src, dst = table[first[g]][whole] * page, table[b][whole] * page
            k[dst:dst + rest], v[dst:dst + rest] = k[src:src + rest], v[src:src + rest]
    cu = _offsets(news)
    q = torch.randn(cu[-1], case["heads"], d, generator=gen, device="cuda", dtype=dtype) * 2.0
    return dict(case=case, q=q, k=k, v=v, table=_ints(table), lens=lens, news=news, cu=cu, first=first,
                prefixes=prefixes, lens_dev=_ints(lens), cu_dev=_ints(cu), first_dev=_ints(first),
                prefixes_dev=_ints(prefixes))


def _weights_inputs(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    dtype, page, hk, d, b = (_DTYPES[case["dtype"]], case["page"], case["kv_heads"], case["dim"], case["batch"])
    width = case["capacity"] // page
    news, lens = _weights_sizes(case)
    order = torch.randperm(b, generator=torch.Generator().manual_seed(seed)).tolist()
    news, lens = [news[i] for i in order], [lens[i] for i in order]
    k = torch.randn(b * width * page, hk, d, generator=gen, device="cuda", dtype=dtype)
    table = torch.randperm(b * width, generator=gen, device="cuda").reshape(b, width).to(torch.int32)
    cu = _offsets(news)
    q = torch.randn(cu[-1], case["heads"], d, generator=gen, device="cuda", dtype=dtype) * 2.0
    start = torch.rand(b, hk, width * page, generator=gen, device="cuda") * 4.0
    return dict(case=case, q=q, k=k, table=table, lens=lens, news=news, cu=cu, start=start,
                scores=start.clone(), lens_dev=_ints(lens), cu_dev=_ints(cu))


def _evict_inputs(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    page, heads, rows, width = case["page"], case["heads"], case["rows"], case["width"]
    lens, keep, shared = _evict_layout(case)
    pages = _evict_pages(case)
    ids = torch.randperm(pages, generator=torch.Generator().manual_seed(seed)).tolist()
    table, refs = [], [0] * pages
    for r in range(rows):
        row = table[r - 1][:shared[r]] if shared[r] else []
        row = row + [ids.pop() for _ in range(-(-lens[r] // page) - shared[r])]
        for x in row:
            refs[x] += 1
        table.append(row + [-1] * (width - len(row)))
    shape = (pages * page, heads, case["dim"])
    pools = [torch.randn(shape, generator=gen, device="cuda", dtype=_DTYPES[case["dtype"]])
             for _ in range(2 * case["layers"])]
    sums = torch.rand(case["layers"], rows, heads, width * page, generator=gen, device="cuda")
    sums = 30.0 * sums ** 6  # few keys carry most of the weight
    if case["ties"]:
        sums = torch.round(sums * 8.0) / 8.0
    return table, lens, keep, refs, pools, sums


def prepare(case, seed):
    if case["op"] == "shared":
        s = _shared_inputs(case, seed)
        if own:
            from fgw_amd.operators.mha.shared_prefix import build_shared_kernel
            s["call"] = build_shared_kernel(case["heads"], case["kv_heads"], case["dim"], case["page"],
                                            case["dtype"], 0)
        return s
    if case["op"] == "weights":
        return _weights_inputs(case, seed)
    table, lens, keep, refs, pools, sums = _evict_inputs(case, seed)
    # One buffer for books and sums, so that a pass starts from the same ones with one copy.
    rows, width, pages, layers = case["rows"], case["width"], len(refs), case["layers"]
    parts = [sums.view(torch.int32).flatten(), _ints(refs), _ints(table).flatten(), _ints(lens)]
    start = torch.cat(parts)
    state = start.clone()
    at = _offsets([x.numel() for x in parts])
    cut = [state[a:b] for a, b in zip(at, at[1:])]
    return dict(case=case, start=start, state=state, refs=cut[1], table=cut[2].view(rows, width), lens=cut[3],
                scores=list(cut[0].view(torch.float32).view(layers, rows, case["heads"], -1).unbind(0)),
                keep=_ints(keep), k_pools=pools[0::2], v_pools=pools[1::2], lens_host=lens, keep_host=keep)


# ---- the passes -----------------------------------------------------------------------------------

def _gather(pool, table_row, lo, hi, page):
    pos = torch.arange(lo, hi, device="cuda")
    rows = table_row[pos // page].long() * page + pos % page
    return pool[rows].float().transpose(0, 1)  # [heads, keys, D]


def _part(q, k, v, hide=None):
    """Softmax numerator, its sum and its reference of some of the keys."""
    x = torch.matmul(q, k.transpose(1, 2))
    if hide is not None:
        x = x.masked_fill(hide, float("-inf"))
    top = x.amax(-1, keepdim=True)
    p = torch.exp(x - top)
    return torch.matmul(p, v), p.sum(-1, keepdim=True), top


def _plain_shared(s):
    case = s["case"]
    hk, d, page = case["kv_heads"], case["dim"], case["page"]
    g = case["heads"] // hk
    q = s["q"].float().view(-1, hk, g, d).permute(1, 0, 2, 3).reshape(hk, -1, d) * d ** -0.5
    out = torch.empty_like(q)
    for gi, prefix in enumerate(s["prefixes"]):
        b0, b1 = s["first"][gi], s["first"][gi + 1]
        r0, r1 = s["cu"][b0] * g, s["cu"][b1] * g
        kp = _gather(s["k"], s["table"][b0], 0, prefix, page)
        vp = _gather(s["v"], s["table"][b0], 0, prefix, page)
        step = max(1, (1 << 28) // (hk * prefix))
        parts = [_part(q[:, a:min(a + step, r1)], kp, vp) for a in range(r0, r1, step)]
        op, lp, mp = (torch.cat(x, 1) for x in zip(*parts))
        for b in range(b0, b1):
            a, n, keys = s["cu"][b] * g, s["news"][b], s["lens"][b] - prefix
            ks = _gather(s["k"], s["table"][b], prefix, s["lens"][b], page)
            vs = _gather(s["v"], s["table"][b], prefix, s["lens"][b], page)
            last = (torch.arange(n, device="cuda") + keys - n).repeat_interleave(g)
            hide = torch.arange(keys, device="cuda") > last[:, None]
            os, ls, ms = _part(q[:, a:a + n * g], ks, vs, hide)
            mine = slice(a - r0, a - r0 + n * g)
            top = torch.maximum(mp[:, mine], ms)
            wp, ws = torch.exp(mp[:, mine] - top), torch.exp(ms - top)
            out[:, a:a + n * g] = (op[:, mine] * wp + os * ws) / (lp[:, mine] * wp + ls * ws)
    return out.view(hk, -1, g, d).permute(1, 0, 2, 3).reshape(-1, hk * g, d).to(s["q"].dtype)


def _plain_weights(s):
    case = s["case"]
    hk, d, page = case["kv_heads"], case["dim"], case["page"]
    g = case["heads"] // hk
    for b, (n, length) in enumerate(zip(s["news"], s["lens"])):
        k = _gather(s["k"], s["table"][b], 0, length, page).transpose(1, 2).contiguous()
        used = min(n, case["last"])
        total = torch.zeros(hk, length, device="cuda")
        step = max(1, min(used, (1 << 28) // (case["heads"] * length)))
        for a in range(n - used, n, step):
            e = min(n, a + step)
            t0 = s["cu"][b]
            q = s["q"][t0 + a:t0 + e].float().view(e - a, hk, g, d).permute(1, 0, 2, 3).reshape(hk, (e - a) * g, d)
            x = torch.matmul(q * d ** -0.5, k)
            last = (torch.arange(a, e, device="cuda") + length - n).repeat_interleave(g)
            x = x.masked_fill(torch.arange(length, device="cuda") > last[:, None], float("-inf"))
            p = torch.exp(x - x.amax(-1, keepdim=True))
            total += (p / p.sum(-1, keepdim=True)).sum(1)
        row = s["scores"][b]
        old = length - n
        row[:, :old] = row[:, :old] * case["decay"] + total[:, :old] if case["decay"] else total[:, :old]
        row[:, old:length] = total[:, old:]
    return s["scores"]


def _plain_evict(s):
    case = s["case"]
    page, first, recent = case["page"], case["first"], case["recent"]
    still = first // page
    free = torch.nonzero(s["refs"] == 0)[:, 0]
    for r, (length, keep) in enumerate(zip(s["lens_host"], s["keep_host"])):
        if not 0 <= keep < length:
            continue
        fresh, free = free[:-(-keep // page) - still], free[-(-keep // page) - still:]
        old = s["table"][r].long()
        new = torch.cat([old[:still], fresh])
        dst = torch.arange(still * page, keep, device="cuda")
        dst_rows = new[dst // page] * page + dst % page
        for layer in range(case["layers"]):
            row = s["scores"][layer][r]
            order = torch.sort(row[:, first:length - recent], dim=1, descending=True, stable=True)[1]
            kept = torch.ones(case["heads"], length, dtype=torch.bool, device="cuda")
            kept[:, first:length - recent] = False
            kept.scatter_(1, order[:, :keep - first - recent] + first, True)
            at = torch.nonzero(kept)[:, 1].view(case["heads"], keep)
            row[:, :keep] = row.gather(1, at)
            src = at[:, still * page:]
            src_rows = (old[src // page] * page + src % page).T  # [tokens, heads]
            head = torch.arange(case["heads"], device="cuda")
            for pool in (s["k_pools"][layer], s["v_pools"][layer]):
                pool[dst_rows] = pool[src_rows, head]
        held = old[still:-(-length // page)]
        s["refs"][held] -= 1
        s["refs"][fresh] = 1
        s["table"][r] = -1
        s["table"][r, :new.numel()] = new.to(torch.int32)
        s["lens"][r] = keep
    return torch.zeros(2, dtype=torch.int32, device="cuda")


def run(state):
    case = state["case"]
    if case["op"] == "shared":
        if own:
            return state["call"](state["q"], state["k"], state["v"], state["table"], state["lens_dev"],
                                 state["cu_dev"], state["first_dev"], state["prefixes_dev"], max(state["news"]))
        return _plain_shared(state)
    if case["op"] == "weights":
        if case["decay"]:
            state["scores"].copy_(state["start"])
        if own:
            from fgw_amd.operators.mha.eviction import add_weights
            add_weights(state["scores"], state["q"], state["k"], state["table"], state["lens_dev"],
                        state["cu_dev"], case["page"], case["last"], decay=case["decay"])
            return state["scores"]
        return _plain_weights(state)
    state["state"].copy_(state["start"])
    if own:
        from fgw_amd.operators.mha.eviction import evict_rows
        status = evict_rows(state["k_pools"], state["v_pools"], state["scores"], state["refs"], state["table"],
                            state["lens"], state["keep"], case["page"], first=case["first"],
                            recent=case["recent"])
    else:
        status = _plain_evict(state)
    return ([state["refs"], state["table"], state["lens"], status] + state["scores"] + state["k_pools"]
            + state["v_pools"])


# ---- the definition in 64 bits ----------------------------------------------------------------------

def _where(table, b, length, page):
    return torch.cat([torch.arange(page, device="cuda") + page * int(i) for i in table[b].tolist() if i >= 0])[:length]


def _exact_shared(case, seed):
    s = _shared_inputs(case, seed)
    ratio, d = case["heads"] // case["kv_heads"], case["dim"]
    out = torch.zeros(s["q"].shape, dtype=torch.float64, device="cuda")
    for b, length in enumerate(s["lens"]):
        at = _where(s["table"], b, length, case["page"])
        a, e = s["cu"][b], s["cu"][b + 1]
        seen = torch.ones(e - a, length, device="cuda").tril(length - (e - a)).bool()
        for h in range(case["kv_heads"]):
            k, v = s["k"][at, h].double(), s["v"][at, h].double()
            for j in range(h * ratio, (h + 1) * ratio):
                x = (s["q"][a:e, j].double() / math.sqrt(d)) @ k.T
                out[a:e, j] = torch.where(seen, x, -math.inf).softmax(-1) @ v
    return out


def _exact_weights(case, seed):
    s = _weights_inputs(case, seed)
    ratio, d = case["heads"] // case["kv_heads"], case["dim"]
    out = s["start"].double()
    for b, length in enumerate(s["lens"]):
        at = _where(s["table"], b, length, case["page"])
        n = s["news"][b]
        used = min(n, case["last"])
        e = s["cu"][b + 1]
        out[b, :, :length] *= case["decay"]
        out[b, :, length - n:length] = 0
        seen = torch.ones(used, length, device="cuda").tril(length - used).bool()
        for j in range(case["heads"]):
            x = s["q"][e - used:e, j].double() @ s["k"][at, j // ratio].double().T / math.sqrt(d)
            out[b, j // ratio, :length] += torch.where(seen, x, -math.inf).softmax(-1).sum(0)
    return out


def _exact_evict(case, seed):
    table, lens, keep, refs, pools, sums = _evict_inputs(case, seed)
    page, first, recent, still = case["page"], case["first"], case["recent"], case["first"] // case["page"]
    host = sums.cpu()
    new_sums = host.clone()
    free = [i for i, n in enumerate(refs) if n == 0]
    old_table, old_lens = [list(row) for row in table], list(lens)
    moves = [([], [], []) for _ in range(case["layers"])]  # from, to, head
    for r, (length, budget) in enumerate(zip(old_lens, keep)):
        if budget < 0 or length <= budget:
            continue
        fresh = [free.pop(0) for _ in range(-(-budget // page) - still)]
        new = old_table[r][:still] + fresh
        for x in old_table[r][still:-(-length // page)]:
            refs[x] -= 1
        for x in fresh:
            refs[x] = 1
        table[r] = new + [-1] * (case["width"] - len(new))
        lens[r] = budget
        for layer in range(case["layers"]):
            for h in range(case["heads"]):
                v = host[layer, r, h, :length].tolist()
                best = sorted(range(first, length - recent), key=lambda i: (-v[i], i))[:budget - first - recent]
                kept = list(range(first)) + sorted(best) + list(range(length - recent, length))
                new_sums[layer, r, h, :budget] = host[layer, r, h, kept]
                for to, at in enumerate(kept):
                    if to >= still * page:
                        moves[layer][0].append(old_table[r][at // page] * page + at % page)
                        moves[layer][1].append(new[to // page] * page + to % page)
                        moves[layer][2].append(h)
    pools = [p.double() for p in pools]
    for layer, (src, dst, head) in enumerate(moves):
        src, dst, head = (torch.tensor(x, dtype=torch.int64, device="cuda") for x in (src, dst, head))
        for pool in pools[2 * layer:2 * layer + 2]:
            pool[dst, head] = pool[src, head]
    return ([_ints(refs), _ints(table), _ints(lens), torch.zeros(2, dtype=torch.int32, device="cuda")]
            + [x.double().cuda() for x in new_sums] + pools[0::2] + pools[1::2])


def exact(case, seed):
    """The operators' definitions in 64 bits, laid out as `run` returns them."""
    return {"shared": _exact_shared, "weights": _exact_weights, "evict": _exact_evict}[case["op"]](case, seed)
