"""The attention of a decoder layer between its coded matrices, for timing: appending keys and values to a paged cache with
the position rotation applied on the way, attention of a few new tokens per sequence over that cache, and attention of
whole prompts (or chunks of them) over it.

A case names the operator, the head layout (heads, kv_heads, dim), the cache's page size and 16-bit type, and a batch:
`seqs` sequences, each with `new` tokens that are being processed and `old` ones before them, drawn from the ranges given
(uniform over the logarithm) with the seed `lengths`, so that the ragged batch belongs to the case and only the values
belong to prepare()'s seed. The pages of a sequence lie scattered over the cache. Head layouts are those of the layers in
lazyweights_amd/configs.py (32 heads of 128 over 8 key-value heads, 32 of 96) and common ones beside them.

Operators, with row t = a new token of sequence s at position i (its last `new` positions), head h reading kv head
h / (heads / kv_heads):
  append   q_out[t, h] = R_i q[t, h], cache_k[s, i] = R_i k[t], cache_v[s, i] = v[t], R_i the rotation of pairs
           (x, y) -> (x cos - y sin, y cos + x sin) with row i of the cos / sin tables
  decode,  out[t, h] = sum_j p_j v[s, j], p = softmax over the positions j <= i (and j > i - window where there is a
  prompt   window) of scale q[t, h] . k[s, j]
"""
import math
import random

import torch

own = False

TYPES = {"f16": torch.float16, "bf16": torch.bfloat16, "f32": torch.float32}
SIZE = {"f16": 2, "bf16": 2, "f32": 4}


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


MISTRAL, PHI, SMALL = (32, 8, 128), (32, 32, 96), (32, 32, 64)


def listed():
    return [
        # a token of one conversation: the smallest call, launch latency
        _case("append 1 token", "append", MISTRAL, 16, "f16", 1, (1, 1), (777, 777), 1),
        # a decode step of a batch, a cache in bfloat16, every head with keys of its own
        _case("append 48 sequences", "append", PHI, 64, "bf16", 48, (1, 1), (3, 500), 2),
        # prompts of odd lengths packed together, neighbouring elements rotated, activations in 16 bits
        _case("append packed prompts", "append", SMALL, 16, "f16", 7, (5, 900), (1, 70), 3, x="f16", pairs="neighbours"),
        # a long prompt at once: as much as a layer's projections give
        _case("append 16383 tokens", "append", MISTRAL, 64, "f16", 1, (16383, 16383), (0, 0), 4),
        # the next token of one conversation: a short cache, launch latency
        _case("decode 1 x 778", "decode", MISTRAL, 16, "f16", 1, (1, 1), (777, 777), 5),
        # a draft of 5 tokens verified for 4 sequences, outputs in 32 bits
        _case("decode verify 4 x 5", "decode", PHI, 32, "bf16", 4, (5, 5), (301, 5003), 6, out="f32"),
        # a batch of conversations of very different lengths: bandwidth
        _case("decode batch 64", "decode", MISTRAL, 16, "f16", 64, (1, 1), (500, 16000), 7),
        # one long document: few rows, a very long axis
        _case("decode 1 x 131071", "decode", MISTRAL, 64, "f16", 1, (1, 1), (131070, 131070), 8),
        # a short prompt of an odd length
        _case("prompt 1 x 33", "prompt", MISTRAL, 16, "f16", 1, (33, 33), (0, 0), 9),
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


def draw(rng):
    op = rng.choice(("append", "decode", "decode", "prompt"))
    kv_heads = rng.choice((1, 2, 4, 8, 8, 32))
    layout = (32 if kv_heads == 32 else kv_heads * rng.choice((1, 2, 4, 7, 8)), kv_heads, rng.choice((64, 96, 128, 128)))
    page, kind, seed = 1 << rng.randrange(3, 8), rng.choice(("f16", "f16", "bf16")), rng.randrange(1 << 20)
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


def _inputs(case, seed):
    """The tensors of a call: cache pages [pages, kv_heads, page, dim], page table, lengths, rows of q, k and v."""
    lengths, page, dim = _lengths(case), case["page"], case["dim"]
    g = torch.Generator(device="cuda").manual_seed(seed)
    kind = TYPES[case["type"]]

    def normal(*shape):
        return torch.randn(shape, generator=g, device="cuda")

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
    rows = starts[-1]
    # a few channels of keys and queries are larger than the others, as trained projections have them
    shape = 1 + 2 * (torch.rand((1, case["kv_heads"], 1, dim), generator=g, device="cuda") < 0.05)
    s = {
        "k_pages": (normal(pages, case["kv_heads"], page, dim) * shape).to(kind),
        "v_pages": (normal(pages, case["kv_heads"], page, dim) + 0.25).to(kind),
        "table": table,
        "q_start": torch.tensor(starts, dtype=torch.int32, device="cuda"),
        "kv_len": torch.tensor([n + o for n, o in lengths], dtype=torch.int32, device="cuda"),
        "max_new": max(n for n, _ in lengths), "max_kv": max(n + o for n, o in lengths), "rows": rows,
    }
    if case["op"] == "append":
        x = TYPES[case["x"]]
        s["q"] = (1.5 * normal(rows, case["heads"], dim)).to(x)
        s["k"] = normal(rows, case["kv_heads"], dim).to(x)
        s["v"] = normal(rows, case["kv_heads"], dim).to(x)
        turn = torch.arange(s["max_kv"], dtype=torch.float64, device="cuda")[:, None] * 10000.0 ** (
            -torch.arange(0, case["rot"], 2, dtype=torch.float64, device="cuda") / case["rot"])
        s["cos"], s["sin"] = torch.cos(turn).float(), torch.sin(turn).float()
    else:
        s["q"] = (1.5 * normal(rows, case["heads"], dim)).to(kind)
    return s


def prepare(case, seed):
    s = _inputs(case, seed)
    s["case"] = case
    s["out"] = torch.zeros((s["rows"], case["heads"], case["dim"]), device="cuda",
                           dtype=TYPES[case["type" if case["op"] == "append" else "out"]])
    if own:
        from lazyweights_amd import Batch, KvCache
        s["cache"] = KvCache(s["k_pages"], s["v_pages"])
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


def _plain_append(s):
    case = s["case"]
    seq, pos = _places(s)
    cos, sin, neighbours = s["cos"][pos][:, None], s["sin"][pos][:, None], case["pairs"] == "neighbours"
    page, off = s["table"][seq, pos // case["page"]].long(), pos % case["page"]
    s["k_pages"][page, :, off] = _rotated(s["k"], cos, sin, neighbours).to(s["k_pages"].dtype)
    s["v_pages"][page, :, off] = s["v"].float().to(s["v_pages"].dtype)
    return {"q": _rotated(s["q"], cos, sin, neighbours).to(s["out"].dtype), "k": s["k_pages"], "v": s["v_pages"]}


def _plain_attention(s):
    """Every sequence padded to the batch's largest, in 32 bits."""
    case = s["case"]
    seqs, heads, kv, dim = case["seqs"], case["heads"], case["kv_heads"], case["dim"]
    group, most = heads // kv, s["max_new"]
    starts, kv_len = s["q_start"].long(), s["kv_len"].long()
    new = starts[1:] - starts[:-1]
    row = (starts[:-1, None] + torch.arange(most, device="cuda")).clamp(max=s["rows"] - 1)
    q = s["q"][row].float().view(seqs, most, kv, group, dim).permute(0, 2, 3, 1, 4).reshape(seqs, kv, group * most, dim)
    k = s["k_pages"][s["table"].long()].float().permute(0, 2, 1, 3, 4).reshape(seqs, kv, -1, dim)
    v = s["v_pages"][s["table"].long()].float().permute(0, 2, 1, 3, 4).reshape(seqs, kv, -1, dim)
    p = (q @ k.transpose(-1, -2).contiguous()).mul_(dim ** -0.5)
    at = (kv_len - new)[:, None] + torch.arange(most, device="cuda")
    key = torch.arange(k.shape[2], device="cuda")
    hidden = key > at[..., None]
    if case["window"]:
        hidden |= key <= at[..., None] - case["window"]
    p = p.view(seqs, kv, group, most, -1).masked_fill_(hidden[:, None, None], -math.inf)
    p = p.sub_(p.amax(-1, keepdim=True).clamp(min=-3e38)).exp_()
    total = p.sum(-1)
    out = (p.view(seqs, kv, group * most, -1) @ v).view(seqs, kv, group, most, dim)
    out = torch.where(total[..., None] > 0, out / total[..., None], 0)
    seq, pos = _places(s)
    out = out.permute(0, 3, 1, 2, 4).reshape(seqs, most, heads, dim)
    return out[seq, pos - (kv_len - new)[seq]].to(s["out"].dtype)


def run(state):
    s, case = state, state["case"]
    if case["op"] == "append":
        if not own:
            return _plain_append(s)
        s["cache"].append(s["batch"], s["q"], s["k"], s["v"], s["cos"], s["sin"], q_out=s["out"],
                          neighbours=case["pairs"] == "neighbours")
        return {"q": s["out"], "k": s["k_pages"], "v": s["v_pages"]}
    if not own:
        return _plain_attention(s)
    if case["op"] == "decode":
        return s["cache"].attend_decode(s["batch"], s["q"], out=s["out"], window=case["window"])
    return s["cache"].attend_prompt(s["batch"], s["q"], out=s["out"], window=case["window"])


def work(case):
    """append: rows read and written once, and the table rows. Attention: q and out, keys and values that some row sees once,
    4 dim operations for each head's pair of a row and a position it sees."""
    lengths, heads, kv, dim = _lengths(case), case["heads"], case["kv_heads"], case["dim"]
    rows = sum(n for n, _ in lengths)
    if case["op"] == "append":
        values = rows * (heads + 2 * kv) * dim
        seen = max(n + o for n, o in lengths) if rows > len(lengths) else rows
        return {"bytes": values * (SIZE[case["x"]] + 2) + 4 * case["rot"] * min(rows, seen), "flops": 3 * values}
    window = case["window"] or 1 << 40
    keys = sum(min(n + o, window + n - 1) for n, o in lengths)
    pairs = sum(min(i + 1, window) for n, o in lengths for i in range(o, o + n))
    return {"bytes": rows * heads * dim * (2 + SIZE[case["out"]]) + keys * kv * dim * 4, "flops": 4 * dim * heads * pairs}


def exact(case, seed):
    s = _inputs(case, seed)
    lengths, page, dim, heads, kv = _lengths(case), case["page"], case["dim"], case["heads"], case["kv_heads"]
    group = heads // kv
    k64, v64 = s["k_pages"].double(), s["v_pages"].double()
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
            k64[where[position // page], :, position % page] = turned(s["k"][mine])
            v64[where[position // page], :, position % page] = s["v"][mine].double()
            continue
        every = torch.arange(old + new, device="cuda")
        for h in range(kv):
            keys = k64[where[every // page], h, every % page]
            values = v64[where[every // page], h, every % page]
            for at in range(0, new, 4096):
                i = position[at:at + 4096]
                rows = s["q"][mine][at:at + 4096, h * group:(h + 1) * group].double()
                score = torch.matmul(rows.transpose(0, 1), keys.T.contiguous()) / math.sqrt(dim)
                seen = every[None] <= i[:, None]
                if case["window"]:
                    seen &= every[None] > i[:, None] - case["window"]
                weight = torch.softmax(torch.where(seen, score, -math.inf), -1)
                out[mine][at:at + 4096, h * group:(h + 1) * group] = torch.matmul(weight, values).transpose(0, 1)
    return {"q": out, "k": k64, "v": v64} if case["op"] == "append" else out
