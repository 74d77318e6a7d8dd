"""The operators around the paged cache whose time is tracked: how a serving step writes it, attends
over it with grouped heads, and moves its pages.

A case is one pass through one operator, `op` says which:
  "extend"   attention of each request's new tokens over its paged cache (they are in it already):
             packed ragged queries, grouped K/V heads, right-aligned causal, optionally a window;
  "append"   new tokens into the cache: Q and K rotated to their positions, K and V written to the
             pages that the block table names;
  "rotate"   rotary positions alone, forward, or inverse (the gradient of the forward);
  "fork"     rows of the block table forked (beams, samples): whole pages shared, the partly filled
             last page copied to a fresh one in every layer's pools;
  "compact"  finished rows freed, then the live pages moved to the low end of the pools.
With `own` false, `run` computes the same in elementary torch operations.
"""
import math

import torch

own = False

_DTYPES = {"bfloat16": torch.bfloat16, "float16": torch.float16, "float32": torch.float32}
_MAX_FLOPS = 2.6e11  # of a drawn case: under the largest listed one
_MAX_BYTES = 4.0e8


def _extend(name, batch, new, heads, kv_heads, dim, page, capacity, dtype, mix="same", ragged=False,
            causal=True, window=0):
    return dict(name=name, op="extend", batch=batch, new=new, heads=heads, kv_heads=kv_heads, dim=dim,
                page=page, capacity=capacity, dtype=dtype, mix=mix, ragged=ragged, causal=causal,
                window=window)


def _append(name, batch, new, heads, kv_heads, dim, page, capacity, dtype, mix, rot, interleaved,
            scaling="none"):
    return dict(name=name, op="append", batch=batch, new=new, heads=heads, kv_heads=kv_heads, dim=dim,
                page=page, capacity=capacity, dtype=dtype, mix=mix, ragged=True, rot=rot,
                interleaved=interleaved, scaling=scaling)


def _rotate(name, tokens, heads, dim, dtype, rot, interleaved, scaling, inverse, span):
    return dict(name=name, op="rotate", tokens=tokens, heads=heads, dim=dim, dtype=dtype, rot=rot,
                interleaved=interleaved, scaling=scaling, inverse=inverse, span=span)


def _pages(name, op, rows, active, changed, layers, heads, dim, page, width, pages, dtype):
    return dict(name=name, op=op, rows=rows, active=active, changed=changed, layers=layers, heads=heads,
                dim=dim, page=page, width=width, pages=pages, dtype=dtype)


def listed():
    bf, fp = "bfloat16", "float16"
    return [
        # One token over one short cache: latency alone.
        _extend("extend_one", 1, 1, 8, 2, 64, 16, 512, bf),
        # A decode step of a serving batch in mid-flight: ragged lengths, four query heads to a K/V head.
        _extend("extend_decode", 32, 1, 32, 8, 128, 64, 4096, bf, ragged=True),
        # A mixed step: one chunk of a prompt and a short one beside running decodes, 16-token pages.
        _extend("extend_mixed", 12, 1000, 32, 8, 128, 16, 8192, bf, mix="mixed", ragged=True),
        # Whole prompts, the largest call.
        _extend("extend_prompt", 2, 4096, 32, 8, 128, 64, 4096, fp),
        # The cache write of a decode step: one token a request, long caches.
        _append("append_decode", 32, 1, 32, 8, 128, 64, 32768, bf, "same", 128, False),
        # The cache write of prompt chunks with half of each head rotated, pairs interleaved.
        _append("append_prompt", 5, 4097, 16, 8, 128, 16, 8192, fp, "mixed", 64, True, "linear"),
        # A few rows in fp32 at far positions, scaled for a long context.
        _rotate("rotate_far", 7, 12, 80, "float32", 48, False, "yarn", False, 1000000),
        # The gradient of a training step's query rotation.
        _rotate("rotate_back", 16384, 32, 128, bf, 128, False, "none", True, 32768),
        # Two beams into four, one layer: latency alone.
        _pages("fork_beams", "fork", 8, 2, 4, 1, 8, 128, 16, 64, 256, bf),
        # Many samples of a batch's prompts, the pools of eight layers.
        _pages("fork_samples", "fork", 96, 16, 64, 8, 8, 128, 64, 64, 512, bf),
        # A small pool after one request ended.
        _pages("compact_one", "compact", 4, 4, 1, 1, 8, 64, 16, 32, 96, fp),
        # A third of a batch ended: eight layers' pools.
        _pages("compact_batch", "compact", 48, 48, 16, 8, 8, 128, 16, 32, 1024, bf),
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, round(lo * (hi / lo) ** rng.random())))


def _draw_extend(rng):
    kind = rng.choice(("decode", "decode", "verify", "mixed", "mixed", "prompt"))
    kv_heads = rng.choice((1, 2, 4, 8, 8))
    heads = kv_heads * rng.choice((1, 2, 3, 4, 4, 6, 8))
    dim = rng.choice((64, 64, 80, 96, 128, 128, 128, 128, 192, 256))
    page = rng.choice((16, 16, 32, 48, 64, 64, 128, 256))
    batch = _log_int(rng, 1, 64)
    if kind == "decode":
        new, cap = 1, _log_int(rng, 128, 32768)
    elif kind == "verify":
        new, cap = rng.randint(2, 17), _log_int(rng, 128, 16384)
    elif kind == "mixed":
        new, cap = _log_int(rng, 33, 2048), _log_int(rng, 256, 16384)
    else:
        new, batch = _log_int(rng, 512, 8192), _log_int(rng, 1, 4)
        cap = new
    cap = -(-max(cap, new) // page) * page
    causal = rng.random() < 0.85
    return _extend(None, batch, new, heads, kv_heads, dim, page, cap,
                   rng.choice(("bfloat16", "bfloat16", "float16")), "mixed" if kind == "mixed" else "same",
                   rng.random() < 0.6, causal, rng.choice((0, 0, 0, 127, 1024)) if causal else 0)


def _draw_append(rng):
    kv_heads = rng.choice((1, 2, 4, 8, 8, 16))
    dim = rng.choice((64, 80, 96, 128, 128, 128, 256))
    page = rng.choice((16, 16, 32, 48, 64, 128))
    new = rng.choice((1, 1, _log_int(rng, 2, 4097)))
    cap = -(-max(new, _log_int(rng, 128, 8192)) // page) * page
    return _append(None, _log_int(rng, 1, 64), new, kv_heads * rng.choice((1, 2, 4, 8)), kv_heads, dim,
                   page, cap, rng.choice(("bfloat16", "float16")), rng.choice(("same", "mixed")),
                   rng.choice((dim, dim, dim // 32 * 16)), rng.random() < 0.5,
                   rng.choice(("none", "linear", "base", "yarn", "bands")))


def _draw_rotate(rng):
    dim = rng.choice((64, 80, 96, 128, 128, 128, 256))
    return _rotate(None, _log_int(rng, 1, 16384), rng.choice((1, 4, 8, 12, 16, 32)), dim,
                   rng.choice(("bfloat16", "float16", "float32")), rng.choice((dim, dim, dim // 32 * 16)),
                   rng.random() < 0.5, rng.choice(("none", "linear", "base", "yarn", "bands")),
                   rng.random() < 0.5, _log_int(rng, 64, 4000000))


def _draw_pages(rng):
    op = rng.choice(("fork", "compact"))
    page, width = rng.choice((16, 16, 32, 64)), _log_int(rng, 4, 64)
    active = _log_int(rng, 2, 48)
    if op == "fork":
        changed = _log_int(rng, 1, 64)
        rows = active + changed + rng.randint(0, 5)
    else:
        changed = max(1, active * rng.randint(1, 3) // 4)
        rows = active
    return _pages(None, op, rows, active, changed, rng.choice((1, 2, 4, 8)), rng.choice((1, 2, 8)),
                  rng.choice((64, 96, 128)), page, width,
                  active * width // 2 + changed + rng.randint(8, 200), rng.choice(("bfloat16", "float16")))


def draw(rng):
    """A case of the listed ranges: odd sizes, ragged batches, every page size and type."""
    kind = rng.choice(("extend", "extend", "extend", "append", "rotate", "pages"))
    case = {"extend": _draw_extend, "append": _draw_append, "rotate": _draw_rotate,
            "pages": _draw_pages}[kind](rng)
    del case["name"]
    while work(case)["flops"] > _MAX_FLOPS or work(case)["bytes"] > _MAX_BYTES:
        if case["op"] in ("extend", "append"):
            key = "batch" if case["batch"] > 1 else ("new" if case["new"] > 64 else "heads")
            if key == "heads":
                case["heads"] = case["kv_heads"] = max(1, case["kv_heads"] // 2)
            else:
                case[key] //= 2
        elif case["op"] == "rotate":
            case["tokens"] //= 2
        else:
            case["layers"] = max(1, case["layers"] // 2)
            case["pages"] = max(case["pages"] // 2, case["active"] * case["width"] // 2 + case["changed"])
            case["heads"] = max(1, case["heads"] // 2)
    return case


# ---- sizes that follow from a case ---------------------------------------------------------------

def _news(case):
    """New tokens of each request: the same for all, or a chunk, a short chunk and single tokens."""
    b, new = case["batch"], case["new"]
    if case["mix"] == "same":
        return [new] * b
    return [new if i == 0 else new // 27 + 1 if i == 1 else 1 for i in range(b)]


def _lengths(case):
    """Cache lengths with the new tokens: full, or spread from a quarter of the capacity to all of it."""
    b, cap = case["batch"], case["capacity"]
    if not case["ragged"]:
        return [cap] * b
    low = cap // 4
    return [max(n, low + (cap - low) * (2 * i + 1) // (2 * b)) for i, n in enumerate(_news(case))]


def _pairs(case, length, new):
    """Visible (query, key) pairs of one request and one head."""
    total = 0
    for j in range(new):
        last = length - new + j + 1 if case["causal"] else length
        total += min(last, case["window"]) if case["window"] else last
    return total


def _live_keys(case, length, new):
    return min(length, case["window"] + new - 1) if case["window"] else length


def work(case):
    """Inputs read once, outputs written once; 4 D flops per visible pair, 6 per rotated pair."""
    if case["op"] == "extend":
        news, lens = _news(case), _lengths(case)
        h, hk, d = case["heads"], case["kv_heads"], case["dim"]
        live = sum(_live_keys(case, n, m) for n, m in zip(lens, news))
        meta = 4 * sum(-(-n // case["page"]) for n in lens) + 8 * case["batch"]
        return {"bytes": 4 * live * hk * d + 4 * sum(news) * h * d + meta,
                "flops": 4 * h * d * sum(_pairs(case, n, m) for n, m in zip(lens, news))}
    if case["op"] == "append":
        t, d = sum(_news(case)), case["dim"]
        qk = t * (case["heads"] + case["kv_heads"])
        return {"bytes": 4 * d * (qk + t * case["kv_heads"]) + 4 * t, "flops": 3 * qk * case["rot"]}
    if case["op"] == "rotate":
        n = case["tokens"] * case["heads"]
        return {"bytes": 2 * n * case["dim"] * _DTYPES[case["dtype"]].itemsize + 4 * case["tokens"],
                "flops": 3 * n * case["rot"]}
    moved = _moved_pages(case)
    page_bytes = case["page"] * case["heads"] * case["dim"] * 2
    meta = 8 * (case["pages"] + case["rows"] * (case["width"] + 1))
    return {"bytes": meta + 2 * moved * page_bytes * 2 * case["layers"], "flops": 0}


# ---- inputs ---------------------------------------------------------------------------------------

def _frequencies(rot, scaling):
    """Radians a position of each pair, in 64 bits, and the factor on cosine and sine."""
    i = torch.arange(0, rot, 2, dtype=torch.float64) / rot
    base, factor, original = 10000.0, 8.0, 4096
    if scaling == "base":
        base *= factor ** (rot / max(rot - 2, 1))
    w = base ** -i
    if scaling == "linear":
        return w / factor, 1.0
    if scaling == "yarn":
        def dim_of(turns):
            return rot * math.log(original / (turns * 2 * math.pi)) / (2 * math.log(base))
        low, high = max(math.floor(dim_of(32.0)), 0), min(math.ceil(dim_of(1.0)), rot - 1)
        ramp = ((torch.arange(rot // 2, dtype=torch.float64) - low) / max(high - low, 0.001)).clamp(0, 1)
        return w / factor * ramp + w * (1 - ramp), 0.1 * math.log(factor) + 1.0
    if scaling == "bands":
        turns = original * w / (2 * math.pi)  # in the original context
        mix = ((turns - 1.0) / (4.0 - 1.0)).clamp(0, 1)
        return (1 - mix) * w / factor + mix * w, 1.0
    return w, 1.0


def _rotary(case):
    """The framework's handle of the same frequencies, which a model keeps."""
    from fgw_amd.operators.mha.rotary import Rotary
    scaling = {"none": None, "linear": dict(kind="linear", factor=8.0), "base": dict(kind="base", factor=8.0),
               "yarn": dict(kind="yarn", factor=8.0, original=4096),
               "bands": dict(kind="bands", factor=8.0, original=4096, low=1.0, high=4.0)}[case["scaling"]]
    return Rotary(case["rot"], base=10000.0, interleaved=case["interleaved"], scaling=scaling, device="cuda")


def _cache_inputs(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    dtype, dev = _DTYPES[case["dtype"]], "cuda"
    b, hk, d, page = (case[k] for k in ("batch", "kv_heads", "dim", "page"))
    width = case["capacity"] // page
    order = torch.randperm(b, generator=torch.Generator().manual_seed(seed)).tolist()
    news, lens = [_news(case)[i] for i in order], [_lengths(case)[i] for i in order]
    cu = [0]
    for n in news:
        cu.append(cu[-1] + n)
    shape = (b * width * page, hk, d)
    k = torch.randn(shape, generator=gen, device=dev, dtype=dtype)
    v = torch.randn(shape, generator=gen, device=dev, dtype=dtype)
    table = torch.randperm(b * width, generator=gen, device=dev).reshape(b, width).to(torch.int32)
    return dict(gen=gen, news=news, lens=lens, cu=cu, k=k, v=v, table=table,
                lens_dev=torch.tensor(lens, dtype=torch.int32, device=dev),
                cu_dev=torch.tensor(cu, dtype=torch.int32, device=dev))


def _extend_inputs(case, seed):
    s = _cache_inputs(case, seed)
    shape = (s["cu"][-1], case["heads"], case["dim"])
    s["q"] = torch.randn(shape, generator=s.pop("gen"), device="cuda", dtype=_DTYPES[case["dtype"]]) * 2.0
    return s


def _append_inputs(case, seed):
    """Q, K and V are views of one fused projection's output, as a model has them."""
    s = _cache_inputs(case, seed)
    h, hk, d = case["heads"], case["kv_heads"], case["dim"]
    qkv = torch.randn(s["cu"][-1], h + 2 * hk, d, generator=s.pop("gen"), device="cuda",
                      dtype=_DTYPES[case["dtype"]])
    s["q"], s["new_k"], s["new_v"] = qkv[:, :h], qkv[:, h:h + hk], qkv[:, h + hk:]
    return s


def _rotate_inputs(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    x = torch.randn(case["tokens"], case["heads"], case["dim"], generator=gen, device="cuda",
                    dtype=torch.float32).to(_DTYPES[case["dtype"]])
    pos = torch.randint(0, case["span"], (case["tokens"],), generator=gen, device="cuda")
    return x, pos.to(torch.int32)


def _page_layout(case):
    """Block table of a batch on the host: active rows of ragged lengths in shuffled pages, in pairs
    that share their first pages, and each page's number of holders."""
    rows, width, page = case["rows"], case["width"], case["page"]
    free = list(range(case["pages"]))
    order = torch.randperm(case["pages"], generator=torch.Generator().manual_seed(
        case["pages"] * 131 + rows)).tolist()
    free = [free[i] for i in order]
    table = [[-1] * width for _ in range(rows)]
    lens, refs = [0] * rows, [0] * case["pages"]
    for r in range(case["active"]):
        most = max(1, width // 2) * page
        lens[r] = max(1, most * (2 * r + 1) // (2 * case["active"]) - r % 3)
        live = -(-lens[r] // page)
        for j in range(live):
            shared = r % 2 == 1 and j < min(live, lens[r - 1] // page) // 2
            table[r][j] = table[r - 1][j] if shared else free.pop()
            refs[table[r][j]] += 1
    if case["op"] == "fork":
        parents = [(7 * i) % case["active"] for i in range(case["changed"])]
        changed = [case["active"] + i for i in range(case["changed"])]
    else:
        parents = []
        changed = [(3 * i) % case["active"] if case["active"] % 3 else i for i in range(case["changed"])]
    return table, lens, refs, parents, changed


def _moved_pages(case):
    table, lens, refs, parents, changed = _page_layout(case)
    if case["op"] == "fork":
        return sum(lens[p] % case["page"] != 0 for p in parents)
    return len(_compact_host(case, table, lens, refs, changed)[3])


def _page_inputs(case, seed):
    """The layout (a fork's with its page ids permuted by the seed) and the pools."""
    gen = torch.Generator(device="cuda").manual_seed(seed)
    table, lens, refs, parents, changed = _page_layout(case)
    swap = torch.randperm(case["pages"], generator=torch.Generator().manual_seed(seed)).tolist()
    if case["op"] == "compact":  # the number of pages to move does not hang on the seed
        swap = list(range(case["pages"]))
    table = [[swap[x] if x >= 0 else -1 for x in row] for row in table]
    moved_refs = [0] * case["pages"]
    for i, n in enumerate(refs):
        moved_refs[swap[i]] = n
    shape = (case["pages"] * case["page"], case["heads"], case["dim"])
    pools = [torch.randn(shape, generator=gen, device="cuda", dtype=_DTYPES[case["dtype"]])
             for _ in range(2 * case["layers"])]
    return table, lens, moved_refs, parents, changed, pools


def prepare(case, seed):
    op = case["op"]
    if op in ("extend", "append"):
        s = _extend_inputs(case, seed) if op == "extend" else _append_inputs(case, seed)
        s["case"] = case
        if op == "extend" and own:
            from fgw_amd.operators.mha.paged_extend import build_extend_kernel
            s["call"] = build_extend_kernel(case["heads"], case["kv_heads"], case["dim"], case["page"],
                                            case["dtype"], 0, is_causal=case["causal"],
                                            window=case["window"] or None)
        if op == "append":
            s["rotary"] = _rotary(case) if own else tuple(
                x.cuda() if torch.is_tensor(x) else x for x in _frequencies(case["rot"], case["scaling"]))
        return s
    if op == "rotate":
        x, pos = _rotate_inputs(case, seed)
        rotary = _rotary(case) if own else tuple(
            x.cuda() if torch.is_tensor(x) else x for x in _frequencies(case["rot"], case["scaling"]))
        return dict(case=case, x=x, pos=pos, rotary=rotary)
    table, lens, refs, parents, changed, pools = _page_inputs(case, seed)
    def dev(x):
        return torch.tensor(x, dtype=torch.int32, device="cuda")
    # One buffer for the books, so that a pass starts from the same books with one copy.
    rows, width, pages = case["rows"], case["width"], case["pages"]
    start = torch.cat([dev(refs), dev(table).flatten(), dev(lens)])
    books = start.clone()
    return dict(case=case, start=start, books=books, refs=books[:pages],
                table=books[pages:pages + rows * width].view(rows, width), lens=books[pages + rows * width:],
                parents=dev(parents), changed=dev(changed), pools=pools,
                tails=torch.tensor([i for i, p in enumerate(parents) if lens[p] % case["page"]],
                                   dtype=torch.int64, device="cuda"))


# ---- the passes -----------------------------------------------------------------------------------

def _plain_extend(s):
    case = s["case"]
    hk, d, page = case["kv_heads"], case["dim"], case["page"]
    g = case["heads"] // hk
    out = torch.empty_like(s["q"])
    for i, (n, length) in enumerate(zip(s["news"], s["lens"])):
        lo = max(0, length - n - case["window"] + 1) if case["window"] else 0
        pos = torch.arange(lo, length, device=out.device)
        rows = s["table"][i, pos // page].long() * page + pos % page
        kk = s["k"][rows].float().transpose(0, 1)
        vv = s["v"][rows].float().transpose(0, 1)
        step = max(1, min(n, (1 << 28) // max(1, case["heads"] * len(pos))))
        for a in range(0, n, step):
            e = min(n, a + step)
            qi = s["q"][s["cu"][i] + a:s["cu"][i] + e].float().view(e - a, hk, g, d)
            qi = qi.permute(1, 0, 2, 3).reshape(hk, (e - a) * g, d)
            x = torch.matmul(qi, kk.transpose(1, 2)) * d ** -0.5
            last = torch.arange(a, e, device=out.device) + (length - n)
            if not case["causal"]:
                last = torch.full_like(last, length - 1)
            seen = pos[None] <= last[:, None]
            if case["window"]:
                seen &= pos[None] > last[:, None] - case["window"]
            seen = seen.repeat_interleave(g, 0)
            x = x.masked_fill(~seen, float("-inf"))
            top = x.amax(-1, keepdim=True).clamp_min(-1e30)
            p = torch.exp(x - top)
            o = torch.matmul(p, vv) / p.sum(-1, keepdim=True).clamp_min(1e-30)
            o = o.view(hk, e - a, g, d).permute(1, 0, 2, 3).reshape(e - a, hk * g, d)
            out[s["cu"][i] + a:s["cu"][i] + e] = o.to(out.dtype)
    return out


def _plain_rotate(x, pos, rotary, rot, interleaved, inverse=False):
    freq, scale = rotary
    angle = pos.double()[:, None] * freq  # 64 bits: far positions
    c, s = (torch.cos(angle) * scale).float()[:, None], (torch.sin(angle) * scale).float()[:, None]
    if inverse:
        s = -s
    y = x.float()
    out = y.clone()
    if interleaved:
        a, b = y[..., 0:rot:2], y[..., 1:rot:2]
        out[..., 0:rot:2], out[..., 1:rot:2] = a * c - b * s, b * c + a * s
    else:
        a, b = y[..., :rot // 2], y[..., rot // 2:rot]
        out[..., :rot // 2], out[..., rot // 2:rot] = a * c - b * s, b * c + a * s
    return out.to(x.dtype)


def _plain_append(s):
    case = s["case"]
    page, t = case["page"], s["cu"][-1]
    news = s["cu_dev"][1:] - s["cu_dev"][:-1]
    owner = torch.repeat_interleave(torch.arange(case["batch"], device="cuda"), news, output_size=t)
    pos = torch.arange(t, device="cuda") - s["cu_dev"][:-1][owner] + (s["lens_dev"] - news)[owner]
    rows = s["table"][owner, pos // page].long() * page + pos % page
    s["k"][rows] = _plain_rotate(s["new_k"], pos, s["rotary"], case["rot"], case["interleaved"])
    s["v"][rows] = s["new_v"]
    return _plain_rotate(s["q"], pos, s["rotary"], case["rot"], case["interleaved"]), s["k"], s["v"]


def _copy_plain(case, pools, src, dst):
    for pool in pools:
        pages = pool.view(case["pages"], -1)
        pages[dst] = pages[src]


def _plain_fork(s):
    case = s["case"]
    pages, page, width = case["pages"], case["page"], case["width"]
    parents, children = s["parents"].long(), s["changed"].long()
    ids = torch.arange(pages, device="cuda")
    free = s["refs"] == 0
    nth = torch.full((pages + 1,), -1, dtype=torch.int64, device="cuda")
    nth[torch.where(free, torch.cumsum(free, 0) - 1, pages)] = ids  # the n-th free page, lowest first
    lens = s["lens"][parents].long()
    whole, tail = lens // page, lens % page != 0
    fresh = nth[torch.cumsum(tail, 0) - 1]
    rows = s["table"][parents].long()
    col = torch.arange(width, device="cuda")
    shared = col < whole[:, None]
    new = torch.where(shared, rows, torch.where((col == whole[:, None]) & tail[:, None], fresh[:, None], -1))
    src = rows.gather(1, whole.clamp_max(width - 1)[:, None])[:, 0]
    count = torch.zeros(pages + 1, dtype=torch.int32, device="cuda")
    held = torch.where(new >= 0, new, pages).flatten()
    count.scatter_add_(0, held, torch.ones_like(held, dtype=torch.int32))
    s["refs"] += count[:pages]
    s["table"][children] = new.to(torch.int32)
    s["lens"][children] = lens.to(torch.int32)
    _copy_plain(case, s["pools"], src[s["tails"]], fresh[s["tails"]])
    return torch.zeros(2, dtype=torch.int32, device="cuda")


def _plain_compact(s):
    case = s["case"]
    pages, page = case["pages"], case["page"]
    gone = s["changed"].long()
    col = torch.arange(case["width"], device="cuda")
    held = s["table"][gone].long()
    held = torch.where(col < -(-s["lens"][gone].long() // page)[:, None], held, pages).flatten()
    count = torch.zeros(pages + 1, dtype=torch.int32, device="cuda")
    count.scatter_add_(0, held, torch.ones_like(held, dtype=torch.int32))
    s["refs"] -= count[:pages]
    s["table"][gone] = -1
    s["lens"][gone] = 0
    ids = torch.arange(pages, device="cuda")
    live = s["refs"] > 0
    total = live.sum()
    src, dst = torch.nonzero(live & (ids >= total))[:, 0], torch.nonzero(~live & (ids < total))[:, 0]
    _copy_plain(case, s["pools"], src, dst)
    new = ids.clone()
    new[src] = dst
    s["refs"][dst] = s["refs"][src]
    s["refs"][src] = 0
    seen = col < -(-s["lens"].long() // page)[:, None]
    s["table"][:] = torch.where(seen, new[s["table"].long().clamp_min(0)], s["table"].long()).to(torch.int32)
    return torch.full((1,), src.numel(), dtype=torch.int32, device="cuda")


def run(state):
    case = state["case"]
    op = case["op"]
    if op == "extend":
        if own:
            return state["call"](state["q"], state["k"], state["v"], state["table"], state["lens_dev"],
                                 state["cu_dev"], max(state["news"]))
        return _plain_extend(state)
    if op == "append":
        if own:
            from fgw_amd.operators.mha.paged_extend import mha_paged_append
            q = mha_paged_append(state["q"], state["new_k"], state["new_v"], state["k"], state["v"],
                                 state["table"], state["lens_dev"], state["cu_dev"], case["page"],
                                 rotary=state["rotary"])
            return q, state["k"], state["v"]
        return _plain_append(state)
    if op == "rotate":
        if own:
            from fgw_amd.operators.mha.rotary import apply_rotary
            return apply_rotary(state["x"], state["pos"], state["rotary"], inverse=case["inverse"])
        return _plain_rotate(state["x"], state["pos"], state["rotary"], case["rot"], case["interleaved"],
                             case["inverse"])
    state["books"].copy_(state["start"])
    refs, table, lens = state["refs"], state["table"], state["lens"]
    if own:
        from fgw_amd.operators.mha import cache_pages
        if op == "fork":
            status = cache_pages.fork_rows(state["pools"], refs, table, lens, state["parents"],
                                           state["changed"], case["page"])
        else:
            cache_pages.free_rows(refs, table, lens, state["changed"], case["page"])
            status = cache_pages.compact_pages(state["pools"], refs, table, lens, case["page"])
    else:
        status = _plain_fork(state) if op == "fork" else _plain_compact(state)
    return [refs, table, lens, status] + state["pools"]


# ---- the definition in 64 bits ----------------------------------------------------------------------

def _exact_extend(case, seed):
    s = _extend_inputs(case, seed)
    h, hk, d, page = (case[k] for k in ("heads", "kv_heads", "dim", "page"))
    out = torch.zeros(s["q"].shape, dtype=torch.float64, device="cuda")
    for i, (n, length) in enumerate(zip(s["news"], s["lens"])):
        keys = torch.arange(length, device="cuda")
        where = s["table"][i].long().repeat_interleave(page)[:length] * page + keys % page
        step = max(1, min(n, (1 << 26) // length))
        for head in range(h):
            k, v = s["k"][where, head // (h // hk)].double(), s["v"][where, head // (h // hk)].double()
            for a in range(0, n, step):
                e = min(n, a + step)
                first = s["cu"][i]
                x = s["q"][first + a:first + e, head].double() @ k.T / math.sqrt(d)
                at = keys.new_tensor(range(a, e)) + length - n if case["causal"] else \
                    keys.new_full((e - a,), length - 1)
                hide = keys > at[:, None]
                if case["window"]:
                    hide |= keys <= at[:, None] - case["window"]
                x[hide] = -math.inf
                out[first + a:first + e, head] = torch.nan_to_num(torch.softmax(x, -1)) @ v
    return out


def _exact_rotate(x, pos, case, inverse=False):
    freq, scale = _frequencies(case["rot"], case["scaling"])
    angle = pos.double()[:, None] * freq.cuda() * (-1 if inverse else 1)
    turn = torch.polar(torch.full_like(angle, scale), angle)[:, None]
    y = x.double().clone()
    r = case["rot"]
    if case["interleaved"]:
        z = torch.complex(y[..., 0:r:2].contiguous(), y[..., 1:r:2].contiguous()) * turn
        y[..., :r] = torch.view_as_real(z).flatten(-2)
    else:
        z = torch.complex(y[..., :r // 2].contiguous(), y[..., r // 2:r].contiguous()) * turn
        y[..., :r] = torch.cat([z.real, z.imag], -1)
    return y


def _exact_append(case, seed):
    s = _append_inputs(case, seed)
    pos = torch.cat([torch.arange(n - m, n) for n, m in zip(s["lens"], s["news"])]).cuda()
    where = torch.cat([s["table"][i, torch.arange(n - m, n, device="cuda") // case["page"]].long()
                       for i, (n, m) in enumerate(zip(s["lens"], s["news"]))]) * case["page"] \
        + pos % case["page"]
    k, v = s["k"].double(), s["v"].double()
    k[where], v[where] = _exact_rotate(s["new_k"], pos, case), s["new_v"].double()
    return _exact_rotate(s["q"], pos, case), k, v


def _compact_host(case, table, lens, refs, gone):
    """Books after freeing `gone` and compacting, and the moves (from, to)."""
    table, lens, refs = [list(r) for r in table], list(lens), list(refs)
    for r in gone:
        for j in range(-(-lens[r] // case["page"])):
            refs[table[r][j]] -= 1
        table[r], lens[r] = [-1] * case["width"], 0
    total = sum(n > 0 for n in refs)
    high = [i for i in range(total, case["pages"]) if refs[i] > 0]
    moves = list(zip(high, [i for i in range(total) if refs[i] == 0]))
    new = dict(moves)
    for a, b in moves:
        refs[b], refs[a] = refs[a], 0
    for r, row in enumerate(table):
        for j in range(-(-lens[r] // case["page"])):
            row[j] = new.get(row[j], row[j])
    return table, lens, refs, moves


def _exact_pages(case, seed):
    table, lens, refs, parents, changed, pools = _page_inputs(case, seed)
    if case["op"] == "fork":
        table, lens, refs = [list(r) for r in table], list(lens), list(refs)
        free = [i for i in range(case["pages"]) if refs[i] == 0]
        moves = []
        for p, c in zip(parents, changed):
            whole, rest = divmod(lens[p], case["page"])
            table[c], lens[c] = table[p][:whole] + [-1] * (case["width"] - whole), lens[p]
            if rest:
                table[c][whole] = free.pop(0)
                moves.append((table[p][whole], table[c][whole]))
            for j in range(whole + (rest > 0)):
                refs[table[c][j]] += 1
        status = [0, 0]
    else:
        table, lens, refs, moves = _compact_host(case, table, lens, refs, changed)
        status = [len(moves)]
    for a, b in moves:
        for pool in pools:
            p = pool.view(case["pages"], -1)
            p[b] = p[a]
    ints = [torch.tensor(x, dtype=torch.int32, device="cuda") for x in (refs, table, lens, status)]
    return ints + [pool.double() for pool in pools]


def exact(case, seed):
    """The operators' definitions in 64 bits, laid out as `run` returns them."""
    if case["op"] == "extend":
        return _exact_extend(case, seed)
    if case["op"] == "append":
        return _exact_append(case, seed)
    if case["op"] == "rotate":
        return _exact_rotate(*_rotate_inputs(case, seed), case, case["inverse"])
    return _exact_pages(case, seed)
