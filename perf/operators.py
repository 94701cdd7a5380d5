"""Measured cases of the paged key-value cache and the attention that reads it.

A decoder block that answers one token at a time keeps the keys and values of every sequence in pages of a common
pool: token p of sequence b lies in page ``block_table[b, p // page_size]`` at row ``p % page_size``.  Four operators
work on that cache:

  append     rotate the new queries and keys by their positions and write keys and values into their pages
  bounds     smallest and largest value of every key channel of the pages that the newest tokens lie in
  attention  softmax(scale * q K^T) V of one new token per sequence over all its pages (or the last `window` tokens)
  sparse     the pages whose bounds allow the largest logits are selected for every group of queries, and the
             attention runs over them only

``own`` False: the operators in elementary torch operations.  True: through the framework's entry points.
"""
import math

import torch

own = False

TYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "e4m3": torch.float8_e4m3fn}


# ---------------------------------------------------------------------------------------------------------------------
# cases
# ---------------------------------------------------------------------------------------------------------------------

def listed():
    return [
        # one token of one conversation: what every layer of a single-user answer costs; latency only
        {"name": "append_one_token", "op": "append", "batch": 1, "tokens": 1, "longest": 700, "ragged": False, "pad": 0,
         "heads": 64, "kv": 8, "dim": 128, "rotary": 128, "interleaved": False, "page": 64, "type": "bf16", "cache": "bf16"},
        # one token for each of 250 sequences of a captured batch of 256 (six padded rows), 8-bit pages
        {"name": "append_batch_e4m3", "op": "append", "batch": 250, "tokens": 1, "longest": 2000, "ragged": True, "pad": 6,
         "heads": 64, "kv": 8, "dim": 128, "rotary": 128, "interleaved": False, "page": 16, "type": "bf16", "cache": "e4m3"},
        # prompts of several sequences packed into one call, the rotation on half of an odd head size
        {"name": "append_prompts", "op": "append", "batch": 5, "tokens": 4999, "longest": 5003, "ragged": False, "pad": 0,
         "heads": 64, "kv": 8, "dim": 128, "rotary": 64, "interleaved": True, "page": 64, "type": "bf16", "cache": "bf16"},
        # the page that the newest token of 64 sequences lies in
        {"name": "bounds_decode", "op": "bounds", "batch": 64, "tokens": 1, "longest": 4096, "ragged": True,
         "heads": 64, "kv": 8, "dim": 128, "page": 64, "type": "bf16", "cache": "bf16"},
        # every page of two long prompts in 8 bits
        {"name": "bounds_prompts_e4m3", "op": "bounds", "batch": 2, "tokens": 65431, "longest": 65431, "ragged": False,
         "heads": 64, "kv": 8, "dim": 128, "page": 32, "type": "bf16", "cache": "e4m3"},
        # a short conversation with one head per query, fp16: latency only
        {"name": "attention_short", "op": "attention", "batch": 1, "longest": 37, "ragged": False, "empty": False,
         "window": 0, "heads": 16, "kv": 16, "dim": 64, "page": 16, "type": "fp16", "cache": "fp16"},
        # the ordinary serving batch: ragged lengths up to 4096, one padded sequence
        {"name": "attention_batch", "op": "attention", "batch": 64, "longest": 4096, "ragged": True, "empty": True,
         "window": 0, "heads": 64, "kv": 8, "dim": 128, "page": 64, "type": "bf16", "cache": "bf16"},
        # one long document in 8 bits: the length has to be split
        {"name": "attention_long_e4m3", "op": "attention", "batch": 1, "longest": 131071, "ragged": False, "empty": False,
         "window": 0, "heads": 64, "kv": 8, "dim": 128, "page": 64, "type": "bf16", "cache": "e4m3"},
        # a sliding window, an odd head size, small odd pages, 6 queries per key head
        {"name": "attention_window", "op": "attention", "batch": 19, "longest": 9001, "ragged": True, "empty": False,
         "window": 1000, "heads": 24, "kv": 4, "dim": 96, "page": 24, "type": "fp16", "cache": "fp16"},
        # 64 of the 2048 pages of one long document
        {"name": "sparse_long", "op": "sparse", "batch": 1, "longest": 131000, "ragged": False, "top": 64,
         "heads": 64, "kv": 8, "dim": 128, "page": 64, "type": "bf16", "cache": "bf16"},
        # a ragged batch, small 8-bit pages; the short sequences have fewer pages than may be selected
        {"name": "sparse_batch_e4m3", "op": "sparse", "batch": 24, "longest": 32768, "ragged": True, "top": 128,
         "heads": 64, "kv": 8, "dim": 128, "page": 16, "type": "bf16", "cache": "e4m3"},
        # a middling length, fp16, other head shapes
        {"name": "sparse_fp16", "op": "sparse", "batch": 7, "longest": 12345, "ragged": True, "top": 31,
         "heads": 20, "kv": 5, "dim": 64, "page": 32, "type": "fp16", "cache": "fp16"},
    ]


def _spread(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 0.49)))))))


def draw(rng):
    op = rng.choice(["append", "bounds", "attention", "attention", "sparse"])
    typ = rng.choice(["bf16", "bf16", "fp16"])
    kv = rng.randint(1, 8)
    case = {"op": op, "kv": kv, "heads": kv * rng.choice([1, 2, 3, 4, 6, 7, 8, 8, 12, 16]),
            "dim": rng.choice([64, 80, 96, 128, 128, 128, 192, 256]), "page": rng.choice([1, 8, 16, 24, 32, 64, 64, 128]),
            "type": typ, "cache": rng.choice([typ, typ, "e4m3"]), "ragged": rng.random() < 0.5}
    if op == "append":
        case["tokens"] = rng.choice([1, 1, _spread(rng, 2, 4000)])
        case["batch"] = _spread(rng, 1, max(1, min(256, 20000 // case["tokens"])))
        case["longest"] = case["tokens"] + rng.randint(0, 3000)
        case["pad"] = rng.randint(0, 5)
        case["rotary"] = rng.choice([0, 32, 64, case["dim"]])
        case["interleaved"] = rng.random() < 0.5
        return _within(case)
    most = 100_000 if op == "bounds" else 130_000
    case["batch"] = _spread(rng, 1, 64)
    case["longest"] = _spread(rng, 1, most // max(1, case["batch"] // (1 if op == "bounds" else 2)))
    if op == "bounds":
        case["tokens"] = rng.choice([1, rng.randint(1, case["longest"])])
    elif op == "attention":
        case["window"] = rng.choice([0, 0, rng.randint(1, 5000)])
        case["empty"] = rng.random() < 0.3
    else:
        case["page"] = max(8, case["page"])
        case["top"] = rng.randint(2, 128)
    return _within(case)


def _within(case):
    """The case with fewer sequences, then shorter ones, until it moves no more than 700 MB."""
    while work(case)["bytes"] > 7e8:
        if case["batch"] > 1:
            case["batch"] -= -(-case["batch"] // 4)
        else:
            case["longest"] -= case["longest"] // 4
            case["tokens"] = min(case["tokens"], case["longest"]) if "tokens" in case else 0
    return case


def _lengths(case):
    """Tokens of every sequence: all the longest, or spread from one token to the longest."""
    n, longest = case["batch"], case["longest"]
    if not case["ragged"]:
        out = [longest] * n
    else:
        out = [longest if i == 0 else 1 + int((longest - 1) * ((i * 0.6180339887498949) % 1.0) ** 2) for i in range(n)]
    if case.get("empty") and n > 1:
        out[-1] = 0
    return out


def _new(case):
    """Tokens of every sequence that the call is about: the last `tokens`, at most all."""
    return [min(case["tokens"], n) for n in _lengths(case)]


def _pages(n, page):
    return -(-n // page)


def _attended(case):
    """(tokens whose keys and values are read, pages whose bounds are read) for one key head, over the batch."""
    lens, page = _lengths(case), case["page"]
    if case["op"] == "attention":
        return sum(min(n, case["window"]) if case["window"] else n for n in lens), 0
    # all the pages selected are whole ones but the last
    return sum(min(n, (case["top"] - 1) * page + (n - 1) % page + 1) for n in lens), sum(_pages(n, page) for n in lens)


def work(case):
    e, ce = 2, 1 if case["cache"] == "e4m3" else 2
    h, kv, d, page = case["heads"], case["kv"], case["dim"], case["page"]
    if case["op"] == "append":
        rows = sum(_new(case))
        return {"bytes": rows * (2 * h * d * e + 2 * kv * d * (e + ce) + 4 * case["rotary"] + 12),
                "flops": rows * 3 * (h + kv) * case["rotary"]}
    if case["op"] == "bounds":
        pages = tokens = 0
        for n, new in zip(_lengths(case), _new(case)):
            first = (n - new) // page
            pages += _pages(n, page) - first
            tokens += n - first * page
        return {"bytes": kv * d * (tokens * ce + pages * 2 * 2) + 4 * pages, "flops": 2 * kv * d * tokens}
    tokens, pages = _attended(case)
    b = case["batch"]
    return {"bytes": 2 * tokens * kv * d * ce + pages * kv * d * 2 * 2 + 2 * b * h * d * e + 4 * tokens // page + 4 * b * h,
            "flops": 4 * tokens * h * d + 2 * pages * h * d}


# ---------------------------------------------------------------------------------------------------------------------
# inputs
# ---------------------------------------------------------------------------------------------------------------------

def prepare(case, seed):
    dev = torch.device("cuda")
    gen = torch.Generator(device=dev)
    gen.manual_seed(int(seed))
    typ, ctyp = TYPES[case["type"]], TYPES[case["cache"]]
    h, kv, d, page, b = case["heads"], case["kv"], case["dim"], case["page"], case["batch"]
    lens = _lengths(case)
    width = max(1, max(_pages(n, page) for n in lens))
    used = sum(_pages(n, page) for n in lens)
    pool = used + 3                                            # a few pages stay free
    s = {"case": dict(case), "page": page, "width": width}

    # keys have a few strong channels and drift slowly along a text, values have neither; stored 8-bit values are
    # divided by a scale per head
    def normal(*shape, dtype=torch.float32):
        return torch.randn(*shape, generator=gen, device=dev, dtype=dtype)
    strength = torch.exp(0.5 * normal(kv, d))
    s["k_scale"] = s["v_scale"] = None
    if case["cache"] == "e4m3":
        s["k_scale"] = 0.02 + 0.02 * torch.rand(kv, generator=gen, device=dev)
        s["v_scale"] = 0.01 + 0.01 * torch.rand(kv, generator=gen, device=dev)
    s["k_cache"] = torch.empty(pool, page, kv, d, dtype=ctyp, device=dev)
    s["v_cache"] = torch.empty(pool, page, kv, d, dtype=ctyp, device=dev)
    step = max(1, (64 << 20) // (page * kv * d))
    for at in range(0, pool, step):
        n = min(step, pool - at)
        k = (normal(n, page, kv, d) + 0.7 * normal(n, 1, kv, d)) * strength
        v = normal(n, page, kv, d)
        if case["cache"] == "e4m3":
            k, v = k / s["k_scale"][:, None], v / s["v_scale"][:, None]
            k, v = k.clamp(-448, 448), v.clamp(-448, 448)
        s["k_cache"][at:at + n] = k.to(ctyp)
        s["v_cache"][at:at + n] = v.to(ctyp)

    order = torch.randperm(pool, generator=gen, device=dev).to(torch.int32)
    counts = torch.tensor([_pages(n, page) for n in lens], device=dev)
    first = torch.cumsum(counts, 0) - counts
    at = torch.arange(width, device=dev)[None, :]
    spot = (first[:, None] + at).clamp(max=pool - 1)
    s["block_table"] = torch.where(at < counts[:, None], order[spot], torch.full_like(order[spot], -1)).contiguous()
    s["seq_lens"] = torch.tensor(lens, dtype=torch.int32, device=dev)

    if case["op"] == "append":
        new = _new(case)
        rows = sum(new)
        total = rows + case["pad"]
        qkv = normal(total, h + 2 * kv, d)
        qkv[:, h:h + kv] *= strength
        qkv = qkv.to(typ)                                      # the output of one fused projection
        s["q"], s["k"], s["v"] = qkv[:, :h], qkv[:, h:h + kv], qkv[:, h + kv:]
        ids = torch.repeat_interleave(torch.arange(b, device=dev), torch.tensor(new, device=dev))
        ends = torch.cumsum(torch.tensor(new, device=dev), 0)
        pos = s["seq_lens"].long()[ids] - (ends[ids] - torch.arange(rows, device=dev))
        fill = torch.full((case["pad"],), -1, device=dev)
        s["rows"] = rows
        s["seq_ids"] = torch.cat([ids, fill]).to(torch.int32)
        s["positions"] = torch.cat([pos, fill]).to(torch.int32)
        s["q_out"] = torch.zeros(total, h, d, dtype=typ, device=dev)
        s["rope"] = None
        if case["rotary"]:
            r = case["rotary"]
            freq = 10000.0 ** (-torch.arange(0, r, 2, dtype=torch.float64, device=dev) / r)
            angle = torch.arange(width * page, dtype=torch.float64, device=dev)[:, None] * freq
            s["rope"] = torch.cat([angle.cos(), angle.sin()], dim=1).to(torch.float32)
        return s
    s["q"] = normal(b, h, d).to(typ)
    s["bounds"] = torch.zeros(pool, kv, 2, d, dtype=torch.bfloat16 if case["cache"] == "e4m3" else ctyp, device=dev)
    if case["op"] == "sparse":
        for at in range(0, pool, step):
            k = s["k_cache"][at:at + step].float()
            s["bounds"][at:at + step] = torch.stack([k.amin(1), k.amax(1)], dim=2).to(s["bounds"].dtype)
    return s


# ---------------------------------------------------------------------------------------------------------------------
# the operators
# ---------------------------------------------------------------------------------------------------------------------

def run(state):
    if own:
        return _with_the_framework(state)
    return {"append": _append, "bounds": _bounds, "attention": _attention, "sparse": _sparse}[state["case"]["op"]](state)


def _with_the_framework(s):
    from wush_b200 import paged_kv
    if "cache" not in s:                                       # the handle of a layer's pages, kept as a program keeps it
        s["cache"] = paged_kv.PagedKVCache(s["k_cache"], s["v_cache"], k_scale=s["k_scale"], v_scale=s["v_scale"],
                                           bounds=s.get("bounds"))
    case, cache = s["case"], s["cache"]
    if case["op"] == "append":
        q = paged_kv.paged_kv_append(cache, s["k"], s["v"], s["block_table"], s["seq_ids"], s["positions"], q=s["q"],
                                     rope=s["rope"], interleaved=case["interleaved"], q_out=s["q_out"])
        return {"q": q, "k_cache": cache.k, "v_cache": cache.v}
    if case["op"] == "bounds":
        paged_kv.paged_kv_bounds(cache, s["block_table"], s["seq_lens"], case["tokens"])
        return {"bounds": cache.bounds}
    if case["op"] == "attention":
        out, lse = paged_kv.paged_decode_attention(s["q"], cache, s["block_table"], s["seq_lens"], window=case["window"],
                                                   return_lse=True)
        return {"out": out, "lse": lse}
    pages, counts = paged_kv.paged_select_pages(s["q"], cache, s["block_table"], s["seq_lens"], case["top"])
    out = paged_kv.paged_decode_attention(s["q"], cache, s["block_table"], s["seq_lens"], pages=pages, counts=counts)
    return {"out": out, "pages": pages, "counts": counts}


def _rotate(x, cos, sin, rotary, interleaved):
    """Pairs of the first `rotary` channels turned by their angles; pairs are (i, i + rotary/2) or (2i, 2i + 1)."""
    r, rest = x[..., :rotary], x[..., rotary:]
    a, b = (r[..., 0::2], r[..., 1::2]) if interleaved else (r[..., :rotary // 2], r[..., rotary // 2:])
    na, nb = a * cos - b * sin, b * cos + a * sin
    turned = torch.stack([na, nb], dim=-1).flatten(-2) if interleaved else torch.cat([na, nb], dim=-1)
    return torch.cat([turned, rest], dim=-1)


def _append(s):
    case, n, page = s["case"], s["rows"], s["page"]
    ids, pos = s["seq_ids"][:n].long(), s["positions"][:n].long()
    q, k, v = s["q"][:n].float(), s["k"][:n].float(), s["v"][:n].float()
    if s["rope"] is not None:
        r = case["rotary"]
        cos, sin = s["rope"][pos, None, :r // 2], s["rope"][pos, None, r // 2:]
        q = _rotate(q, cos, sin, r, case["interleaved"])
        k = _rotate(k, cos, sin, r, case["interleaved"])
    if s["k_scale"] is not None:
        k = (k / s["k_scale"][:, None]).clamp(-448, 448)
        v = (v / s["v_scale"][:, None]).clamp(-448, 448)
    where = s["block_table"][ids, pos // page].long()
    # (8-bit floats have no indexed write of their own: the bytes are written)
    bits = torch.uint8 if s["k_cache"].element_size() == 1 else s["k_cache"].dtype
    s["k_cache"].view(bits)[where, pos % page] = k.to(s["k_cache"].dtype).view(bits)
    s["v_cache"].view(bits)[where, pos % page] = v.to(s["v_cache"].dtype).view(bits)
    s["q_out"][:n] = q.to(s["q_out"].dtype)
    return {"q": s["q_out"], "k_cache": s["k_cache"], "v_cache": s["v_cache"]}


def _bounds(s):
    """Over the filled rows of every page that holds one of the last `tokens` tokens of a sequence."""
    case, page, lens = s["case"], s["page"], s["seq_lens"].long()
    most = min(s["width"], (case["tokens"] - 1) // page + 2)
    start = (lens - case["tokens"]).clamp(min=0) // page
    logical = start[:, None] + torch.arange(most, device=lens.device)
    touched = logical * page < lens[:, None]
    physical = s["block_table"].gather(1, logical.clamp(max=s["width"] - 1)).long()
    # pages past the end of a sequence stand for its first page here, whose rows are then all masked or all its own
    physical = torch.where(touched, physical, s["block_table"].gather(1, start[:, None]).long())
    logical = torch.where(touched, logical, start[:, None])
    k = s["k_cache"].view(torch.uint8 if s["k_cache"].element_size() == 1 else s["k_cache"].dtype)[physical]
    k = k.view(s["k_cache"].dtype).float()
    filled = (logical[..., None] * page + torch.arange(page, device=lens.device) < lens[:, None, None])[..., None, None]
    low = k.masked_fill(~filled, math.inf).amin(2)
    high = k.masked_fill(~filled, -math.inf).amax(2)
    s["bounds"][physical.flatten()] = torch.stack([low, high], dim=3).flatten(0, 1).to(s["bounds"].dtype)
    return {"bounds": s["bounds"]}


def _gathered(pool, physical, scale):
    """fp32 rows of pages: pool [P, page, kv, d], physical [...] -> [..., page, kv, d]."""
    bits = torch.uint8 if pool.element_size() == 1 else pool.dtype
    x = pool.view(bits)[physical].view(pool.dtype).float()
    return x if scale is None else x * scale[:, None]


def _softmax_product(q, k, v, seen):
    """q [b, kv, g, d], k and v [b, kv, n, d], seen [b, kv or 1, 1, n] -> out [b, kv * g, d], log of the sum [b, kv * g]."""
    logits = torch.matmul(q, k.transpose(-1, -2)) * (q.shape[-1] ** -0.5)
    logits = logits.masked_fill(~seen, -math.inf)
    top = logits.amax(-1, keepdim=True)
    top = torch.where(top == -math.inf, torch.zeros_like(top), top)
    e = torch.exp(logits - top)
    total = e.sum(-1, keepdim=True)
    out = torch.matmul(e / torch.where(total == 0, torch.ones_like(total), total), v)
    return out.flatten(1, 2), (torch.log(total) + top).squeeze(-1).flatten(1, 2)


def _attention(s):
    case, page, lens = s["case"], s["page"], s["seq_lens"].long()
    b, d, kv = case["batch"], case["dim"], case["kv"]
    physical = s["block_table"].clamp(min=0).long()
    k = _gathered(s["k_cache"], physical, s["k_scale"]).flatten(1, 2).transpose(1, 2)
    v = _gathered(s["v_cache"], physical, s["v_scale"]).flatten(1, 2).transpose(1, 2)
    at = torch.arange(k.shape[2], device=lens.device)
    seen = at < lens[:, None]
    if case["window"]:
        seen = seen & (at >= lens[:, None] - case["window"])
    q = s["q"].float().view(b, kv, -1, d)
    out, lse = _softmax_product(q, k, v, seen[:, None, None, :])
    return {"out": out.to(s["q"].dtype), "lse": lse}


def _sparse(s):
    """A page's score for a key head: the largest over the head's queries of sum_d max(q_d min_d, q_d max_d).  The first
    page and the last are always taken, then the best scores (the lowest page first where equal), in 64 bits because the
    last page that is taken may be only a little better than the next."""
    case, page, lens = s["case"], s["page"], s["seq_lens"].long()
    top = case["top"]
    b, d, kv, width = case["batch"], case["dim"], case["kv"], s["width"]
    dev = lens.device
    table = s["block_table"].clamp(min=0).long()
    q = s["q"].double().view(b, kv, -1, d)
    bound = s["bounds"][table].double()                         # [b, width, kv, 2, d]
    low, high = bound[:, :, :, 0].permute(0, 2, 3, 1), bound[:, :, :, 1].permute(0, 2, 3, 1)
    score = (torch.matmul(q.clamp(min=0), high) + torch.matmul(q.clamp(max=0), low)).amax(2)   # [b, kv, width]
    n = ((lens + page - 1) // page)[:, None, None]
    at = torch.arange(width, device=dev)
    score = score.masked_fill((at == 0) | (at == n - 1), math.inf).masked_fill(at >= n, -math.inf)
    best = torch.sort(score, dim=-1, descending=True, stable=True).indices[..., :min(top, width)]
    taken = torch.arange(best.shape[-1], device=dev) < n
    pages = torch.where(taken, best, torch.full_like(best, width)).sort(-1).values
    pages = torch.where(pages < width, pages, torch.full_like(pages, -1))
    pages = torch.nn.functional.pad(pages, (0, top - pages.shape[-1]), value=-1)
    counts = torch.minimum(n, torch.full_like(n, top)).expand(b, kv, 1).squeeze(-1)
    # attention over the rows of those pages
    logical = pages.clamp(min=0)
    physical = table[:, None, :].expand(b, kv, width).gather(2, logical)
    heads = torch.arange(kv, device=dev)[None, :, None]
    bits = torch.uint8 if s["k_cache"].element_size() == 1 else s["k_cache"].dtype
    k = s["k_cache"].view(bits).transpose(1, 2)[physical, heads].view(s["k_cache"].dtype).float()   # [b, kv, top, page, d]
    v = s["v_cache"].view(bits).transpose(1, 2)[physical, heads].view(s["v_cache"].dtype).float()
    if s["k_scale"] is not None:
        k, v = k * s["k_scale"][:, None, None, None], v * s["v_scale"][:, None, None, None]
    where = logical[..., None] * page + torch.arange(page, device=dev)
    seen = (pages[..., None] >= 0) & (where < lens[:, None, None, None])
    out, _ = _softmax_product(s["q"].float().view(b, kv, -1, d), k.flatten(2, 3), v.flatten(2, 3),
                              seen.flatten(2, 3)[:, :, None, :])
    return {"out": out.to(s["q"].dtype), "pages": pages.to(torch.int32), "counts": counts.to(torch.int32)}


# ---------------------------------------------------------------------------------------------------------------------
# the definitions in 64 bits, one sequence (and one head) after another
# ---------------------------------------------------------------------------------------------------------------------

def exact(case, seed):
    s = prepare(case, seed)
    page, d, kv, group = case["page"], case["dim"], case["kv"], case["heads"] // case["kv"]
    lens = _lengths(case)
    table = s["block_table"].cpu()

    if case["op"] == "append":
        q, k, v = (s[x].double() for x in "qkv")
        if case["rotary"]:
            half = case["rotary"] // 2
            i = torch.arange(half, device=q.device)
            first, second = (2 * i, 2 * i + 1) if case["interleaved"] else (i, i + half)
            turn = s["rope"][s["positions"].clamp(min=0).long()].double()
            z = torch.complex(turn[:, :half], turn[:, half:])[:, None, :]
            for x in (q, k):
                y = torch.complex(x[..., first], x[..., second]) * z
                x[..., first], x[..., second] = y.real, y.imag
        if s["k_scale"] is not None:
            k = torch.clamp(k / s["k_scale"].double()[:, None], -448, 448)
            v = torch.clamp(v / s["v_scale"].double()[:, None], -448, 448)
        out_q, out_k, out_v = s["q_out"].double(), s["k_cache"].double(), s["v_cache"].double()
        at = 0
        for b, new in enumerate(_new(case)):
            p = torch.arange(lens[b] - new, lens[b])
            pg = table[b][p // page].long().to(q.device)
            row = (p % page).to(q.device)
            out_k[pg, row], out_v[pg, row] = k[at:at + new], v[at:at + new]
            out_q[at:at + new] = q[at:at + new]
            at += new
        return {"q": out_q, "k_cache": out_k, "v_cache": out_v}

    if case["op"] == "bounds":
        out = s["bounds"].double()
        for b, new in enumerate(_new(case)):
            for lp in range((lens[b] - new) // page, _pages(lens[b], page)):
                pg = int(table[b, lp])
                keys = s["k_cache"][pg, :lens[b] - lp * page].double()
                out[pg, :, 0], out[pg, :, 1] = keys.min(0).values, keys.max(0).values
        return {"bounds": out}

    def rows(name, b, logical, upto):
        """[tokens, kv, d] of the pages `logical` of sequence b, cut at position `upto`, and the positions."""
        pg = table[b][logical].long().to(s["q"].device)
        pool = s[name + "_cache"]
        x = torch.stack([pool[int(p)].double() for p in pg]) if len(pg) < 8 else _wide(pool, pg)
        at = (logical[:, None] * page + torch.arange(page)).to(x.device)
        x, at = x.flatten(0, 1), at.flatten()
        x, at = x[at < upto], at[at < upto]
        return (x if s[name + "_scale"] is None else x * s[name + "_scale"].double()[:, None]), at

    def attend(q, k, v):
        logits = (k @ q) * d ** -0.5
        return torch.softmax(logits, 0) @ v, torch.logsumexp(logits, 0)

    dev = s["q"].device
    out = torch.zeros(case["batch"], case["heads"], d, dtype=torch.float64, device=dev)
    if case["op"] == "attention":
        lse = torch.full((case["batch"], case["heads"]), -math.inf, dtype=torch.float64, device=dev)
        for b, n in enumerate(lens):
            if n == 0:
                continue
            begin = max(0, n - case["window"]) if case["window"] else 0
            logical = torch.arange(begin // page, _pages(n, page))
            k, at = rows("k", b, logical, n)
            v, _ = rows("v", b, logical, n)
            k, v = k[at >= begin], v[at >= begin]
            for h in range(case["heads"]):
                out[b, h], lse[b, h] = attend(s["q"][b, h].double(), k[:, h // group], v[:, h // group])
        return {"out": out, "lse": lse}

    for b, n in enumerate(lens):
        count = _pages(n, page)
        bound = s["bounds"][table[b, :count].long().to(dev)].double()
        for g in range(kv):
            chosen = list(range(count))
            if count > case["top"]:
                score = torch.stack([torch.maximum(s["q"][b, h].double() * bound[:, g, 0], s["q"][b, h].double() * bound[:, g, 1])
                                     .sum(1) for h in range(g * group, (g + 1) * group)]).amax(0).tolist()
                middle = sorted(range(1, count - 1), key=lambda i: (-score[i], i))[:case["top"] - 2]
                chosen = sorted([0, count - 1] + middle)
            lp = torch.tensor(chosen)
            pg = table[b][lp].long().to(dev)
            at = (lp[:, None] * page + torch.arange(page)).flatten().to(dev)
            k = torch.cat([s["k_cache"][int(p), :, g].double() for p in pg])[at < n]
            v = torch.cat([s["v_cache"][int(p), :, g].double() for p in pg])[at < n]
            if s["k_scale"] is not None:
                k, v = k * s["k_scale"][g].double(), v * s["v_scale"][g].double()
            for h in range(g * group, (g + 1) * group):
                out[b, h], _ = attend(s["q"][b, h].double(), k, v)
    return {"out": out, "pages": None, "counts": None}


def _wide(pool, pages):
    bits = torch.uint8 if pool.element_size() == 1 else pool.dtype
    return pool.view(bits)[pages].view(pool.dtype).double()
