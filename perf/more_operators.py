"""Serving with a key-value cache held in 8 bits, for timing: the page bookkeeping of a step, made on the GPU from the
requests' lengths; appending keys and values to the cache, quantized and with the position rotation on the way; attention
of a few new tokens per sequence over it; attention of whole prompts, or chunks of them.

The cache holds numbers of 8 bits (1 sign, 4 exponent, 3 mantissa bits, up to 448) with one power of two, 2^e, for each
block of 16 tokens of a key-value head (keys and values apart): element = number * 2^e, e an int8 in -48 .. 48. A case names
the operator, the head layout (heads, kv_heads, dim), the page size, the 16-bit type of q, and a batch: `seqs` sequences,
each with `new` tokens that are being processed and `old` ones before them, drawn from the ranges given (uniform over the
logarithm) with the seed `lengths`, so that the ragged batch belongs to the case and only the values belong to prepare()'s
seed. The pages of a sequence lie scattered over the cache. Head layouts are those of the layers in
lazyweights_amd/configs.py (32 heads of 128 over 8 key-value heads, 32 of 96) and common ones beside them.

Operators, with row t = a new token of sequence s at position i (its last `new` positions), head h reading kv head
h / (heads / kv_heads), R_i the rotation of pairs (x, y) -> (x cos - y sin, y cos + x sin) by row i of the cos / sin tables:
  append   q_out[t, h] = R_i q[t, h]; keys R_i k[t] and values v[t] into the cache. A block's e is the least with
           max |x| <= 448 2^e over its new rows, or what it was where it has older rows and that is more; where it grows the
           older rows are rounded to it
  decode,  out[t, h] = sum_j p_j v[s, j], p = softmax over the positions j <= i (and j > i - window where there is a
  prompt   window) of scale q[t, h] . k[s, j]
  pages    every sequence is cut to keep[s] tokens and grown by new[s]: pages that it no longer needs go back to the pool (a
           stack), pages it needs are taken, given ones first; lengths, rows' starts, table, and each new row's position and
           slot (its row in the cache)
"""
import math
import random

import torch

own = False

TYPES = {"f16": torch.float16, "bf16": torch.bfloat16, "f32": torch.float32}
SIZE = {"f16": 2, "bf16": 2, "f32": 4}
BLOCK, LEAST, MOST = 16, -48, 48
F8 = torch.float8_e4m3fn


def _case(name, op, layout, page, kind, seqs, new, old, lengths, **more):
    heads, kv_heads, dim = layout
    case = {"name": name, "op": op, "heads": heads, "kv_heads": kv_heads, "dim": dim, "page": page, "type": kind,
            "seqs": seqs, "new_low": new[0], "new_high": new[1], "old_low": old[0], "old_high": old[1], "lengths": lengths}
    if op == "append":
        case.update({"x": "f32", "rot": dim, "pairs": "halves"})
    else:
        case.update({"out": kind, "window": 0})
    case.update(more)
    return case


def _pages_case(name, page, seqs, new, old, lengths, ended, back):
    return {"name": name, "op": "pages", "page": page, "seqs": seqs, "new_low": new[0], "new_high": new[1], "old_low": old[0],
            "old_high": old[1], "lengths": lengths, "ended": ended, "back": back}


MISTRAL, PHI, SMALL = (32, 8, 128), (32, 32, 96), (32, 32, 64)


def listed():
    return [
        # a decode step of 64 conversations with drafts of 4, some of whose tokens are taken back: the smallest call, latency
        _pages_case("pages draft step 64", 16, 64, (4, 5), (100, 8000), 1, 0.02, 4),
        # a batch in which half of the requests end and prompts take their places
        _pages_case("pages prompts 500", 32, 500, (20, 2000), (50, 3000), 2, 0.5, 0),
        # a token of one conversation: launch latency
        _case("append 1 token", "append", MISTRAL, 16, "f16", 1, (1, 1), (777, 777), 3),
        # packed prompts of odd lengths after something that ends inside a block, neighbouring elements rotated, bfloat16 in
        _case("append packed prompts", "append", SMALL, 16, "bf16", 7, (5, 900), (1, 70), 4, x="bf16", pairs="neighbours"),
        # a long prompt at once: as much as a layer's projections give
        _case("append 16383 tokens", "append", MISTRAL, 64, "f16", 1, (16383, 16383), (0, 0), 5),
        # the next token of one conversation: a short cache, launch latency
        _case("decode 1 x 778", "decode", MISTRAL, 16, "f16", 1, (1, 1), (777, 777), 6),
        # a draft of 5 tokens verified for 4 sequences, q in bfloat16, outputs in 32 bits
        _case("decode verify 4 x 5", "decode", PHI, 32, "bf16", 4, (5, 5), (301, 5003), 7, out="f32"),
        # a batch of conversations of very different lengths: bandwidth
        _case("decode batch 64", "decode", MISTRAL, 16, "f16", 64, (1, 1), (500, 16000), 8),
        # one long document: few rows, a very long axis
        _case("decode 1 x 131071", "decode", MISTRAL, 64, "f16", 1, (1, 1), (131070, 131070), 9),
        # packed prompts of different lengths, outputs in 32 bits as the prompt products of coded matrices take them
        _case("prompt packed 9", "prompt", PHI, 16, "f16", 9, (17, 2500), (0, 0), 10, out="f32"),
        # a chunk of a long prompt after what is there already, with a sliding window
        _case("prompt chunk 1000 at 9001", "prompt", MISTRAL, 64, "f16", 1, (1000, 1000), (9001, 9001), 11, window=4096),
        # a long prompt at once: the largest call
        _case("prompt 1 x 15999", "prompt", MISTRAL, 64, "bf16", 1, (15999, 15999), (0, 0), 12),
    ]


def _spread(rng, low, high):
    """A whole number in low .. high, uniform over its logarithm."""
    return min(high, max(low, int(round(math.exp(rng.uniform(math.log(max(low, 1)), math.log(max(high, 1))))))))


def _lengths(case):
    """(new, old) of every sequence."""
    rng = random.Random(case["lengths"])
    return [(_spread(rng, case["new_low"], case["new_high"]), _spread(rng, case["old_low"], case["old_high"]))
            for _ in range(case["seqs"])]


def _requests(case):
    """(new, length before, tokens kept of it) of every sequence."""
    rng = random.Random(case["lengths"] + 1)
    return [(new, old, 0 if rng.random() < case["ended"] else max(0, old - rng.randint(0, case["back"])))
            for new, old in _lengths(case)]


def draw(rng):
    op = rng.choice(("pages", "append", "decode", "decode", "prompt", "prompt"))
    page, seed = 1 << rng.randrange(4, 8), rng.randrange(1 << 20)
    if op == "pages":
        seqs = _spread(rng, 1, 1000)
        high = _spread(rng, 1, max(1, min(8000, 200000 // seqs)))
        case = _pages_case("", page, seqs, (max(1, high // 30), high), (1, _spread(rng, 20, 8000)), seed,
                           rng.choice((0.0, 0.02, 0.5)), rng.choice((0, 4, 16)))
        del case["name"]
        return case
    kv_heads = rng.choice((1, 2, 4, 8, 8, 32))
    layout = (32 if kv_heads == 32 else kv_heads * rng.choice((1, 2, 4, 7, 8)), kv_heads, rng.choice((64, 96, 128, 128)))
    kind = rng.choice(("f16", "f16", "bf16"))
    more = {}
    if op == "append":
        seqs = _spread(rng, 1, 64)
        high = max(1, 16383 // seqs)
        new = (1, 1) if rng.random() < 0.4 else (max(1, high // 20), _spread(rng, max(1, high // 20), high))
        old = (0, _spread(rng, 1, 500))
        more = {"x": rng.choice(("f32", "f32", "f16", "bf16")), "pairs": rng.choice(("halves", "halves", "neighbours")),
                "rot": layout[2] if rng.random() < 0.7 else layout[2] // 2}
    elif op == "decode":
        seqs = _spread(rng, 1, 64)
        count = 1 if rng.random() < 0.6 else rng.randrange(2, 17)
        new = (count, count) if rng.random() < 0.7 else (1, count)
        high = _spread(rng, 100, min(131000, 500000 // seqs))
        old = (max(1, high // 30), high) if seqs > 1 else (high, high)
    else:
        seqs = _spread(rng, 1, 12)
        high = _spread(rng, 17, 8000 if seqs < 3 else 2500)
        new = (max(1, high // 20), high)
        old = (0, 0) if rng.random() < 0.6 else (1, _spread(rng, 20, 4000))
    if op != "append":
        more = {"out": rng.choice((kind, kind, "f32")), "window": rng.choice((0, 0, 0, _spread(rng, 50, 4096)))}
    case = _case("", op, layout, page, kind, seqs, new, old, seed, **more)
    del case["name"]
    return case


def _exponent(most):
    """The least e in LEAST .. MOST with most <= 448 * 2^e, 448 = 0.875 * 2^9."""
    m, e = torch.frexp(most)
    return torch.where(most > 0, e - 9 + (m > 0.875), LEAST).clamp(LEAST, MOST)


def _held(x):
    """Rows x [pages, kv_heads, page, dim] as the cache holds them: numbers and exponents."""
    blocks = x.unflatten(2, (-1, BLOCK))
    e = _exponent(blocks.abs().amax((-2, -1)))
    return torch.ldexp(blocks, -e[..., None, None]).flatten(2, 3).to(F8), e.to(torch.int8)


def _inputs(case, seed):
    """The tensors of a call: cache pages [pages, kv_heads, page, dim], page table, lengths, rows of q, k and v."""
    lengths, page, dim = _lengths(case), case["page"], case["dim"]
    g = torch.Generator(device="cuda").manual_seed(seed)
    kind = TYPES[case["type"]]

    def normal(*shape):
        return torch.randn(shape, generator=g, device="cuda")

    def some(share, size, *shape):
        return 1 + (size - 1) * (torch.rand(shape, generator=g, device="cuda") < share)

    need = [-(-(n + o) // page) for n, o in lengths]
    pages = sum(need) + 3
    order = torch.randperm(pages, generator=g, device="cuda").to(torch.int32)
    table = torch.zeros((case["seqs"], max(need)), dtype=torch.int32, device="cuda")
    at = 0
    for s, n in enumerate(need):
        table[s, :n] = order[at:at + n]
        at += n
    starts = [0]
    for n, _ in lengths:
        starts.append(starts[-1] + n)
    rows, kv = starts[-1], case["kv_heads"]
    # a few channels of keys and queries are larger than the others, as trained projections have them, and a few tokens
    shape = some(0.05, 3, 1, kv, 1, dim)
    k, k_exp = _held(normal(pages, kv, page, dim) * shape * some(0.01, 2.5, pages, kv, page, 1))
    v, v_exp = _held((normal(pages, kv, page, dim) + 0.25) * some(0.01, 2.5, pages, kv, page, 1))
    s = {
        "k": k, "v": v, "k_exp": k_exp, "v_exp": v_exp, "table": table,
        "q_start": torch.tensor(starts, dtype=torch.int32, device="cuda"),
        "kv_len": torch.tensor([n + o for n, o in lengths], dtype=torch.int32, device="cuda"),
        "max_new": max(n for n, _ in lengths), "max_kv": max(n + o for n, o in lengths), "rows": rows,
    }
    if case["op"] == "append":
        x = TYPES[case["x"]]
        s["q"] = (1.5 * normal(rows, case["heads"], dim)).to(x)
        s["new_k"] = (normal(rows, kv, dim) * shape[:, :, 0] * some(0.05, 2.5, rows, kv, 1)).to(x)
        s["new_v"] = ((normal(rows, kv, dim) + 0.25) * some(0.05, 2.5, rows, kv, 1)).to(x)
        turn = torch.arange(s["max_kv"], dtype=torch.float64, device="cuda")[:, None] * 10000.0 ** (
            -torch.arange(0, case["rot"], 2, dtype=torch.float64, device="cuda") / case["rot"])
        s["cos"], s["sin"] = torch.cos(turn).float(), torch.sin(turn).float()
    else:
        s["q"] = (1.5 * normal(rows, case["heads"], dim)).to(kind)
    return s


def _page_inputs(case, seed):
    """Lengths, what is kept and added, the table and the pool before a step, and memory for what it gives."""
    requests, page = _requests(case), case["page"]
    g = torch.Generator(device="cuda").manual_seed(seed)
    had = [-(-old // page) for _, old, _ in requests]
    need = [-(-(keep + new) // page) for new, _, keep in requests]
    pool, width = sum(max(a, b) for a, b in zip(had, need)) + 5, max(had + need) + 2
    order = torch.randperm(pool, generator=g, device="cuda").to(torch.int32)
    used, at = sum(had), torch.tensor([0] + had[:-1], device="cuda").cumsum(0)[:, None] + torch.arange(width, device="cuda")
    mine = torch.arange(width, device="cuda") < torch.tensor(had, device="cuda")[:, None]
    free = torch.full((pool,), -1, dtype=torch.int32, device="cuda")
    free[:pool - used] = order[used:]

    def whole(values, kind=torch.int32):
        return torch.tensor(values, dtype=kind, device="cuda")

    rows = sum(new for new, _, _ in requests)
    return {
        "new": whole([r[0] for r in requests]), "kv_len": whole([r[1] for r in requests]), "keep": whole([r[2] for r in requests]),
        "table": torch.where(mine, order[at.clamp(max=pool - 1)], -1), "free": free, "left": whole([pool - used, 0]),
        "kv_out": whole([0] * case["seqs"]), "left_out": whole([0, 0]), "q_start": whole([0] * (case["seqs"] + 1)),
        "position": whole([0] * rows), "slot": whole([0] * rows, torch.int64), "rows": rows,
    }


def prepare(case, seed):
    if case["op"] == "pages":
        s = _page_inputs(case, seed)
        s["case"] = case
        if own:
            from lazyweights_amd import Pages
            s["pages"] = Pages(case["page"], s["kv_len"], s["table"], s["free"], s["left"])
        return s
    s = _inputs(case, seed)
    s["case"] = case
    s["out"] = torch.zeros((s["rows"], case["heads"], case["dim"]), device="cuda",
                           dtype=TYPES[case["type" if case["op"] == "append" else "out"]])
    if own:
        from lazyweights_amd import Batch, KvCache8
        s["cache"] = KvCache8(s["k"], s["v"], s["k_exp"], s["v_exp"])
        s["batch"] = Batch(s["cache"], case["heads"], s["q_start"], s["kv_len"], s["table"], s["max_new"], s["max_kv"])
    return s


def _places(s):
    """The sequence and the position of every row."""
    rows = torch.arange(s["rows"], device="cuda")
    starts, kv_len = s["q_start"].long(), s["kv_len"].long()
    seq = torch.searchsorted(starts, rows, right=True) - 1
    return seq, kv_len[seq] - starts[seq + 1] + rows


def _rotated(x, cos, sin, neighbours):
    n = cos.shape[-1]
    y = x.float().clone()
    a, b = (slice(0, 2 * n, 2), slice(1, 2 * n, 2)) if neighbours else (slice(0, n), slice(n, 2 * n))
    u, v = y[..., a].clone(), y[..., b].clone()
    y[..., a] = u * cos - v * sin
    y[..., b] = v * cos + u * sin
    return y


def _plain_quantized(s, x, codes, exps, page, off):
    """Rows x [rows, kv_heads, dim] into the cache's numbers and exponents at (page, off)."""
    pages, kv, size, dim = codes.shape
    per = size // BLOCK
    block, row = page * per + off // BLOCK, off % BLOCK
    first = torch.full((pages * per,), BLOCK, device="cuda").scatter_reduce_(0, block, row, "amin")
    most = torch.zeros((pages * per, kv), device="cuda").scatter_reduce_(0, block[:, None].expand(-1, kv), x.abs().amax(-1), "amax")
    old = exps.transpose(1, 2).reshape(pages * per, kv).int()
    e = _exponent(most)
    e = torch.where((first > 0)[:, None], torch.maximum(old, e), e)
    e = torch.where((first < BLOCK)[:, None], e, old)

    def by_head(t):  # [blocks, kv] -> [pages, kv, blocks of a page]
        return t.view(pages, per, kv).transpose(1, 2)

    # the older rows of blocks whose exponent grew
    older = (torch.arange(BLOCK, device="cuda") < first[:, None]).view(pages, 1, per, BLOCK, 1)
    less = torch.where(older, by_head(old - e)[..., None, None], 0)
    codes.copy_(torch.ldexp(codes.float().unflatten(2, (per, BLOCK)), less).flatten(2, 3).to(F8))
    exps.copy_(by_head(e))
    codes.view(torch.uint8)[page, :, off] = torch.ldexp(x, -e[block][..., None]).to(F8).view(torch.uint8)


def _plain_append(s):
    case = s["case"]
    seq, pos = _places(s)
    cos, sin, neighbours = s["cos"][pos][:, None], s["sin"][pos][:, None], case["pairs"] == "neighbours"
    page, off = s["table"][seq, pos // case["page"]].long(), pos % case["page"]
    _plain_quantized(s, _rotated(s["new_k"], cos, sin, neighbours), s["k"], s["k_exp"], page, off)
    _plain_quantized(s, s["new_v"].float(), s["v"], s["v_exp"], page, off)
    return {"q": _rotated(s["q"], cos, sin, neighbours).to(s["out"].dtype), "k": s["k"], "v": s["v"], "k_exp": s["k_exp"],
            "v_exp": s["v_exp"]}


def _plain_attention(s):
    """Every sequence padded to the batch's largest, in 32 bits."""
    case = s["case"]
    seqs, heads, kv, dim = case["seqs"], case["heads"], case["kv_heads"], case["dim"]
    group, most = heads // kv, s["max_new"]
    starts, kv_len, table = s["q_start"].long(), s["kv_len"].long(), s["table"].long()
    new = starts[1:] - starts[:-1]

    def values(codes, exps):
        x = codes.view(torch.uint8)[table].view(F8).float().unflatten(3, (-1, BLOCK))
        x = torch.ldexp(x, exps[table].int()[..., None, None])
        return x.permute(0, 2, 1, 3, 4, 5).reshape(seqs, kv, -1, dim)

    row = (starts[:-1, None] + torch.arange(most, device="cuda")).clamp(max=s["rows"] - 1)
    q = s["q"][row].float().view(seqs, most, kv, group, dim).permute(0, 2, 3, 1, 4).reshape(seqs, kv, group * most, dim)
    k = values(s["k"], s["k_exp"])
    p = (q @ k.transpose(-1, -2).contiguous()).mul_(dim ** -0.5)
    at = (kv_len - new)[:, None] + torch.arange(most, device="cuda")
    key = torch.arange(k.shape[2], device="cuda")
    hidden = key > at[..., None]
    if case["window"]:
        hidden |= key <= at[..., None] - case["window"]
    p = p.view(seqs, kv, group, most, -1).masked_fill_(hidden[:, None, None], -math.inf)
    p = p.sub_(p.amax(-1, keepdim=True).clamp(min=-3e38)).exp_()
    total = p.sum(-1)
    out = (p.view(seqs, kv, group * most, -1) @ values(s["v"], s["v_exp"])).view(seqs, kv, group, most, dim)
    out = torch.where(total[..., None] > 0, out / total[..., None], 0)
    seq, pos = _places(s)
    out = out.permute(0, 3, 1, 2, 4).reshape(seqs, most, heads, dim)
    return out[seq, pos - (kv_len - new)[seq]].to(s["out"].dtype)


def _plain_pages(s):
    """(The pool holds what the step takes.)"""
    page, table, free, before = s["case"]["page"], s["table"], s["free"], s["kv_len"].long()
    seqs, new, kept = before.shape[0], s["new"].long(), torch.minimum(s["keep"].long(), before)
    length = kept + new
    had, need = (before + page - 1) // page, (length + page - 1) // page
    take, give = (need - had).clamp(min=0), (had - need).clamp(min=0)
    takes, gives = take.cumsum(0), give.cumsum(0)
    taken, given, left = takes[-1], gives[-1], s["left"][0].long()
    i = torch.arange(free.shape[0], device="cuda")
    # the i-th page given: sequence by sequence, in the order of their positions
    giver = torch.searchsorted(gives, i, right=True).clamp(max=seqs - 1)
    back = table[giver, (need[giver] + i - (gives - give)[giver]).clamp(0, table.shape[1] - 1)]
    # the i-th page taken: a given one while there are any, then the pool's last
    page_of = torch.where(i < given, back, free[(left - 1 - (i - given)).clamp(0, free.shape[0] - 1)])
    taker = torch.searchsorted(takes, i, right=True).clamp(max=seqs - 1)
    column = had[taker] + i - (takes - take)[taker]
    mine = i < taken
    table[taker[mine], column[mine]] = page_of[mine]
    kept_back = (i >= taken) & (i < given)
    free[(left + i - taken)[kept_back]] = back[kept_back]
    s["left_out"][0] = left - (taken - given)
    s["left_out"][1] = 0
    s["kv_out"].copy_(length)
    s["q_start"][1:] = new.cumsum(0)
    starts, rows = s["q_start"].long(), torch.arange(s["rows"], device="cuda")
    seq = torch.searchsorted(starts, rows, right=True) - 1
    s["position"].copy_(kept[seq] + rows - starts[seq])
    at = s["position"].long()
    s["slot"].copy_(table[seq, at // page].long() * page + at % page)


def run(state):
    s, case = state, state["case"]
    if case["op"] == "pages":
        if not own:
            _plain_pages(s)
        else:
            s["pages"].advance(s["new"], keep=s["keep"], kv_len_out=s["kv_out"], left_out=s["left_out"], q_start=s["q_start"],
                               position=s["position"], slot=s["slot"])
        return {k: s[k] for k in ("kv_out", "left_out", "q_start", "table", "free", "position", "slot")}
    if case["op"] == "append":
        if not own:
            return _plain_append(s)
        s["cache"].append(s["batch"], s["q"], s["new_k"], s["new_v"], s["cos"], s["sin"], q_out=s["out"],
                          neighbours=case["pairs"] == "neighbours")
        return {"q": s["out"], "k": s["k"], "v": s["v"], "k_exp": s["k_exp"], "v_exp": s["v_exp"]}
    if not own:
        return _plain_attention(s)
    if case["op"] == "decode":
        return s["cache"].attend_decode(s["batch"], s["q"], out=s["out"], window=case["window"])
    return s["cache"].attend_prompt(s["batch"], s["q"], out=s["out"], window=case["window"])


def work(case):
    """pages: the sequences' lengths and starts, the new rows' positions and slots, the pages that change hands. append: rows read
    and written once, and the table rows. Attention: q and out, keys and values that some row sees once with their
    exponents, 4 dim operations for each head's pair of a row and a position it sees."""
    if case["op"] == "pages":
        requests, page = _requests(case), case["page"]
        moved = sum(abs(-(-(keep + new) // page) + -old // page) for new, old, keep in requests)
        rows = sum(new for new, _, _ in requests)
        return {"bytes": 20 * len(requests) + 12 * rows + 8 * moved, "flops": rows}
    lengths, heads, kv, dim = _lengths(case), case["heads"], case["kv_heads"], case["dim"]
    rows = sum(n for n, _ in lengths)
    if case["op"] == "append":
        queries, keys = rows * heads * dim, 2 * rows * kv * dim
        seen = max(n + o for n, o in lengths) if rows > len(lengths) else rows
        return {"bytes": queries * (SIZE[case["x"]] + 2) + keys * (SIZE[case["x"]] + 1) + 4 * case["rot"] * min(rows, seen),
                "flops": 3 * queries + 5 * keys}
    window = case["window"] or 1 << 40
    keys = sum(min(n + o, window + n - 1) for n, o in lengths)
    pairs = sum(min(i + 1, window) for n, o in lengths for i in range(o, o + n))
    return {"bytes": rows * heads * dim * (2 + SIZE[case["out"]]) + 2 * keys * kv * dim + keys * kv // 8,
            "flops": 4 * dim * heads * pairs}


def _exact_pages(case, seed):
    """The step request by request, with lists."""
    s, page = _page_inputs(case, seed), case["page"]
    table, free = s["table"].tolist(), s["free"].tolist()
    stack, back, length, starts, position, slot = free[:int(s["left"][0])], [], [], [0], [], []
    requests = _requests(case)
    for t, (new, old, keep) in enumerate(requests):
        back += table[t][-(-(keep + new) // page):-(-old // page)]
    for t, (new, old, keep) in enumerate(requests):
        for at in range(-(-old // page), -(-(keep + new) // page)):
            table[t][at] = back.pop(0) if back else stack.pop()
        length.append(keep + new)
        starts.append(starts[-1] + new)
        for i in range(keep, keep + new):
            position.append(i)
            slot.append(table[t][i // page] * page + i % page)
    stack += back
    free[:len(stack)] = stack
    made = {"kv_out": length, "left_out": [len(stack), 0], "q_start": starts, "table": table, "free": free, "position": position,
            "slot": slot}
    return {k: torch.tensor(x) for k, x in made.items()}


def _to_8_bits(x):
    """x (64 bits) rounded to 3 mantissa bits, ties to even, the least step 2^-9."""
    step = torch.exp2((torch.frexp(x)[1].double() - 1).clamp(min=-6) - 3)
    return torch.round(x / step) * step


def exact(case, seed):
    if case["op"] == "pages":
        return _exact_pages(case, seed)
    s = _inputs(case, seed)
    lengths, page, dim, heads, kv = _lengths(case), case["page"], case["dim"], case["heads"], case["kv_heads"]
    group = heads // kv
    held = {n: s[n].double() for n in ("k", "v")}
    power = {n: s[n + "_exp"].long() for n in ("k", "v")}
    out = torch.zeros((s["rows"], heads, dim), dtype=torch.float64, device="cuda")
    first = 0
    for b, (new, old) in enumerate(lengths):
        mine, position = slice(first, first + new), torch.arange(old, old + new, device="cuda")
        first += new
        where = s["table"][b].long()
        if case["op"] == "append":
            c, n = torch.complex(s["cos"].double(), s["sin"].double())[position][:, None], case["rot"] // 2

            def turned(x):
                x = x.double()
                pairs = x[..., :2 * n].unflatten(-1, (n, 2) if case["pairs"] == "neighbours" else (2, n))
                if case["pairs"] != "neighbours":
                    pairs = pairs.transpose(-1, -2)
                z = torch.view_as_real(torch.view_as_complex(pairs.contiguous()) * c)
                z = z if case["pairs"] == "neighbours" else z.transpose(-1, -2)
                return torch.cat((z.flatten(-2), x[..., 2 * n:]), -1)

            out[mine] = turned(s["q"][mine])
            # whole blocks from the first one that is touched on, old rows as they are held; [blocks, 16, kv, dim]
            begin = old // BLOCK * BLOCK
            every = torch.arange(begin, -(-(old + new) // BLOCK) * BLOCK, device="cuda")
            fresh, older = ((every >= old) & (every < old + new)).view(-1, BLOCK, 1, 1), (every < old).view(-1, BLOCK, 1, 1)
            at, row, cell = where[every // page], every % page, every[::BLOCK]
            for n_, x in (("k", turned(s["new_k"][mine])), ("v", s["new_v"][mine].double())):
                now = held[n_][at, :, row].unflatten(0, (-1, BLOCK))
                was = power[n_][where[cell // page], :, cell % page // BLOCK]
                rows = torch.zeros_like(now)
                rows.view(-1, kv, dim)[old - begin:old - begin + new] = x
                most = rows.abs().amax((1, 3))
                e = torch.ceil(torch.log2(most.clamp(min=1e-300) / 448)).long().clamp(LEAST, MOST)
                e = torch.where(older.any(1)[..., 0], torch.maximum(was, e), e)
                kept = _to_8_bits(now * torch.exp2((was - e).double())[:, None, :, None])
                put = _to_8_bits(rows * torch.exp2(-e.double())[:, None, :, None])
                held[n_][at, :, row] = torch.where(fresh, put, torch.where(older, kept, now)).flatten(0, 1)
                power[n_][where[cell // page], :, cell % page // BLOCK] = e
            continue
        every = torch.arange(old + new, device="cuda")
        for h in range(kv):
            keys, values = (held[n][where[every // page], h, every % page] *
                            torch.exp2(power[n][where[every // page], h, every % page // BLOCK].double())[:, None]
                            for n in ("k", "v"))
            for at in range(0, new, 4096):
                i = position[at:at + 4096]
                rows = s["q"][mine][at:at + 4096, h * group:(h + 1) * group].double()
                score = torch.matmul(rows.transpose(0, 1), keys.T.contiguous()) / math.sqrt(dim)
                seen = every[None] <= i[:, None]
                if case["window"]:
                    seen &= every[None] > i[:, None] - case["window"]
                weight = torch.softmax(torch.where(seen, score, -math.inf), -1)
                out[mine][at:at + 4096, h * group:(h + 1) * group] = torch.matmul(weight, values).transpose(0, 1)
    if case["op"] == "append":
        return {"q": out, "k": held["k"], "v": held["v"], "k_exp": power["k"], "v_exp": power["v"]}
    return out
