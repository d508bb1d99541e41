"""The operators of a decoder whose keys and values lie in pages, as cases that can be timed and compared.

Three operators, used in this order by every layer of such a decoder:

append   the rows of Q|K|V that a projection gave for the new tokens of a batch of sequences: queries and keys turned by their
         positions, keys and values stored into the pages of their sequences
attend   attention of the new tokens (one of each sequence, a chunk of some, or whole prompts) over the pages
copy     pages copied to other pages of the same cache, in all layers: what a fork, a beam search's step or a compaction asks for

A cache is [pages, kv_heads, page_size, head_dim] a layer.  Row b of `table` lists the pages of sequence b in order, `starts` says where
the rows of its new tokens begin and end, `lengths` how many keys it has, the new tokens' among them.  12 heads of 64 are those of this
repository's base model, the other head counts are generic ones.
"""
import math
import random

import torch

own = False

DTYPES = {"f16": torch.float16, "bf16": torch.bfloat16, "f32": torch.float32}


def listed():
    return [
        # one decoding step of a small service: eight sequences, a token each; nothing but latency
        {"name": "append_f16_8x1", "kind": "append", "dtype": "f16", "heads": 12, "kv_heads": 12, "head_dim": 64, "page": 16, "sequences": 8, "new_low": 1, "new_high": 1,
         "past_low": 5, "past_high": 500, "rotary": 64, "interleaved": False, "stretch": 1.0, "lengths": 1},
        # prompts in the element type a checkpoint comes in, half of each head turned, pairs side by side
        {"name": "append_f32_5_prompts", "kind": "append", "dtype": "f32", "heads": 12, "kv_heads": 12, "head_dim": 64, "page": 16, "sequences": 5, "new_low": 33, "new_high": 387,
         "past_low": 0, "past_high": 0, "rotary": 32, "interleaved": True, "stretch": 1.0, "lengths": 2},
        # chunks of long documents, shared key/value heads, positions stretched to a longer context
        {"name": "append_bf16_chunks", "kind": "append", "dtype": "bf16", "heads": 32, "kv_heads": 8, "head_dim": 128, "page": 32, "sequences": 6, "new_low": 512, "new_high": 4096,
         "past_low": 1, "past_high": 100000, "rotary": 128, "interleaved": False, "stretch": 8.0, "lengths": 3},
        # one request of the base model, one token at a time
        {"name": "decode_f16_1x387", "kind": "attend", "dtype": "f16", "heads": 12, "kv_heads": 12, "head_dim": 64, "page": 16, "sequences": 1, "chunks": 0, "new_low": 1, "new_high": 1,
         "past_low": 386, "past_high": 386, "window": 0, "lengths": 4},
        # a full batch of a service
        {"name": "decode_bf16_64", "kind": "attend", "dtype": "bf16", "heads": 32, "kv_heads": 8, "head_dim": 128, "page": 16, "sequences": 64, "chunks": 0, "new_low": 1, "new_high": 1,
         "past_low": 100, "past_high": 6000, "window": 0, "lengths": 5},
        # a few very long contexts
        {"name": "decode_f16_4_long", "kind": "attend", "dtype": "f16", "heads": 32, "kv_heads": 8, "head_dim": 128, "page": 64, "sequences": 4, "chunks": 0, "new_low": 1, "new_high": 1,
         "past_low": 60000, "past_high": 131071, "window": 0, "lengths": 6},
        # prompts without conversion to half precision
        {"name": "prompts_f32_8", "kind": "attend", "dtype": "f32", "heads": 12, "kv_heads": 12, "head_dim": 64, "page": 16, "sequences": 8, "chunks": 8, "new_low": 33, "new_high": 500,
         "past_low": 0, "past_high": 0, "window": 0, "lengths": 7},
        # decoding and prompts in one batch: 40 sequences with a token each, 3 with a chunk, the last 1000 keys only
        {"name": "mixed_f16_43_window", "kind": "attend", "dtype": "f16", "heads": 16, "kv_heads": 4, "head_dim": 64, "page": 16, "sequences": 43, "chunks": 3, "new_low": 200, "new_high": 900,
         "past_low": 50, "past_high": 5000, "window": 1000, "lengths": 8},
        # the next chunk of a few long documents
        {"name": "chunks_bf16_6", "kind": "attend", "dtype": "bf16", "heads": 32, "kv_heads": 8, "head_dim": 128, "page": 32, "sequences": 6, "chunks": 6, "new_low": 400, "new_high": 600,
         "past_low": 1500, "past_high": 9000, "window": 0, "lengths": 9},
        # one whole long prompt
        {"name": "prompt_bf16_8192", "kind": "attend", "dtype": "bf16", "heads": 32, "kv_heads": 8, "head_dim": 128, "page": 32, "sequences": 1, "chunks": 1, "new_low": 8192, "new_high": 8192,
         "past_low": 0, "past_high": 0, "window": 0, "lengths": 10},
        # a step of a beam search: the last pages of four hypotheses that share them, base model
        {"name": "copy_f16_4_forks", "kind": "copy", "dtype": "f16", "layers": 12, "kv_heads": 12, "head_dim": 64, "page": 16, "pages": 160, "count": 4},
        # a cache is compacted: the live pages of its upper part move into holes of the lower
        {"name": "copy_bf16_compaction", "kind": "copy", "dtype": "bf16", "layers": 24, "kv_heads": 8, "head_dim": 128, "page": 32, "pages": 4000, "count": 901},
    ]


def _log_int(rng, low, high):
    return min(high, max(low, int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))))


def draw(rng):
    kind = rng.choice(["append", "attend", "attend", "attend", "attend", "copy"])
    case = {"kind": kind, "dtype": rng.choice(["f16", "bf16", "f32"])}
    case["head_dim"] = rng.choice([64, 128])
    case["kv_heads"] = rng.choice([1, 2, 4, 8, 12])
    case["page"] = rng.choice([16, 32, 64, 128])
    if kind == "copy":
        case["layers"] = rng.randint(1, 24)
        page_bytes = case["kv_heads"] * case["page"] * case["head_dim"] * (4 if case["dtype"] == "f32" else 2)
        case["pages"] = min(4000, max(40, (6 << 30) // (page_bytes * case["layers"])))
        case["count"] = _log_int(rng, 1, case["pages"] // 5)
        return case
    case["heads"] = case["kv_heads"] * rng.choice([1, 2, 3, 4, 8] if case["kv_heads"] <= 4 else [1, 2, 4])
    case["lengths"] = rng.randrange(10000)
    if kind == "append":
        case["sequences"] = _log_int(rng, 1, 100)
        most = _log_int(rng, 1, 4096 if case["sequences"] <= 6 else 128)
        case["new_low"], case["new_high"] = rng.randint(1, most), most
        case["past_low"], case["past_high"] = (0, 0) if rng.random() < 0.3 else (1, _log_int(rng, 10, 20000))
        case["rotary"] = rng.choice([case["head_dim"], case["head_dim"], case["head_dim"] // 2, 0])
        case["interleaved"] = rng.random() < 0.5
        case["stretch"] = rng.choice([1.0, 4.0, 8.0])
        return case
    form = rng.choice(["decode", "decode", "chunks", "mixed", "prompts"])
    case["window"] = _log_int(rng, 16, 4000) if rng.random() < 0.25 else 0
    if form == "decode":
        case["sequences"] = _log_int(rng, 1, 100)
        longest = _log_int(rng, 8, 65536 if case["sequences"] <= 4 else 6000)
        case["past_low"], case["past_high"] = rng.randint(1, longest), longest
        case["new_low"], case["new_high"], case["chunks"] = 1, 1, 0
    elif form == "chunks":
        case["sequences"] = _log_int(rng, 1, 6)
        longest = _log_int(rng, 32, 6000)
        case["past_low"], case["past_high"] = rng.randint(1, longest), longest
        most = _log_int(rng, 2, 500)
        case["new_low"], case["new_high"], case["chunks"] = rng.randint(1, most), most, case["sequences"]
    elif form == "mixed":
        case["sequences"] = _log_int(rng, 4, 40)
        longest = _log_int(rng, 32, 2000)
        case["past_low"], case["past_high"] = rng.randint(1, longest), longest
        most = _log_int(rng, 2, 500)
        case["new_low"], case["new_high"], case["chunks"] = rng.randint(1, most), most, rng.randint(1, 3)
    else:
        case["sequences"] = _log_int(rng, 1, 8)
        most = _log_int(rng, 4, 4000 if case["sequences"] <= 2 else 1000)
        case["past_low"], case["past_high"] = 0, 0
        case["new_low"], case["new_high"], case["chunks"] = rng.randint(1, most), most, case["sequences"]
    return case


def _lengths(case):
    """New tokens and keys before them, of every sequence: given by the case."""
    rng = random.Random(case["lengths"])
    chunks = case.get("chunks", case["sequences"])
    new = [_log_int(rng, case["new_low"], case["new_high"]) if i < chunks else 1 for i in range(case["sequences"])]
    past = [_log_int(rng, case["past_low"], case["past_high"]) if case["past_high"] else 0 for _ in range(case["sequences"])]
    order = list(range(case["sequences"]))
    rng.shuffle(order)
    return [new[i] for i in order], [past[i] for i in order]


def work(case):
    size = 4 if case["dtype"] == "f32" else 2
    if case["kind"] == "copy":
        page = case["kv_heads"] * case["page"] * case["head_dim"] * size
        return {"bytes": 4 * case["layers"] * case["count"] * page, "flops": 0}
    new, past = _lengths(case)
    d, heads, kv_heads = case["head_dim"], case["heads"], case["kv_heads"]
    if case["kind"] == "append":
        return {"bytes": 2 * sum(new) * (heads + 2 * kv_heads) * d * size, "flops": 3 * sum(new) * (heads + kv_heads) * case["rotary"]}
    pairs = keys = 0
    for n, p in zip(new, past):
        reach = case["window"] or n + p
        pairs += sum(min(p + i + 1, reach) for i in range(n))
        keys += min(n + p, reach + n - 1)
    return {"bytes": (2 * sum(new) * heads * d + 2 * keys * kv_heads * d) * size, "flops": 4 * pairs * heads * d}


def prepare(case, seed):
    gen = torch.Generator("cuda").manual_seed(seed)
    dtype = DTYPES[case["dtype"]]

    def random_values(*shape):
        return torch.randn(shape, generator=gen, device="cuda").to(dtype)

    state = {"case": case}
    if case["kind"] == "copy":
        shape = (case["layers"], case["pages"], case["kv_heads"], case["page"], case["head_dim"])
        state["keys"], state["values"] = random_values(*shape), random_values(*shape)
        order = random.Random(seed).sample(range(case["pages"]), 2 * case["count"])
        state["sources"], state["destinations"] = order[: case["count"]], order[case["count"]:]
        return state
    new, past = _lengths(case)
    needed = [-(-(n + p) // case["page"]) for n, p in zip(new, past)]
    # pages of a sequence lie where the cache had room: in any order, a tenth of them unused
    pages = sum(needed) + sum(needed) // 10 + 1
    order = random.Random(seed).sample(range(pages), sum(needed))
    table = torch.zeros((len(new), max(needed)), dtype=torch.int32)
    at = 0
    for b, n in enumerate(needed):
        table[b, :n] = torch.tensor(order[at:at + n], dtype=torch.int32)
        at += n
    state["table"] = table.cuda()
    state["lengths"] = torch.tensor([n + p for n, p in zip(new, past)], dtype=torch.int32).cuda()
    state["starts"] = torch.tensor([sum(new[:b]) for b in range(len(new) + 1)], dtype=torch.int32).cuda()
    state["most_new"], state["longest"] = max(new), max(n + p for n, p in zip(new, past))
    shape = (pages, case["kv_heads"], case["page"], case["head_dim"])
    state["keys"], state["values"] = random_values(*shape), random_values(*shape)
    if case["kind"] == "append":
        state["qkv"] = random_values(sum(new), (case["heads"] + 2 * case["kv_heads"]) * case["head_dim"])
        r = case["rotary"]
        exponents = torch.arange(0, r, 2, dtype=torch.float64, device="cuda") / max(r, 1)
        state["inv_freq"] = 10000.0 ** -exponents / case["stretch"] if r else None
    else:
        state["q"] = random_values(sum(new), case["heads"], case["head_dim"])
    return state


# ------------------------------------------------------------------------------------------------ plain forms ----------
def _rows(state):
    """Of every new token: its sequence, its number among the new ones of that, its position."""
    starts = state["starts"].long()
    new = starts[1:] - starts[:-1]
    sequence = torch.repeat_interleave(torch.arange(new.numel(), device=new.device), new)
    number = torch.arange(sequence.numel(), device=new.device) - starts[sequence]
    return sequence, number, state["lengths"].long()[sequence] - new[sequence] + number


def _plain_append(state):
    case = state["case"]
    d, heads, kv_heads, r = case["head_dim"], case["heads"], case["kv_heads"], case["rotary"]
    sequence, _, position = _rows(state)
    x = state["qkv"].view(-1, heads + 2 * kv_heads, d)
    dtype = x.dtype
    q, k, v = x[:, :heads], x[:, heads:heads + kv_heads], x[:, heads + kv_heads:]
    if r:
        angle = position.double()[:, None, None] * state["inv_freq"]
        cos, sin = angle.cos().float(), angle.sin().float()
        both = x[:, :heads + kv_heads].float()
        if case["interleaved"]:
            x1, x2 = both[..., 0:r:2], both[..., 1:r:2]
            turned = torch.stack((x1 * cos - x2 * sin, x1 * sin + x2 * cos), dim=-1).flatten(-2)
        else:
            x1, x2 = both[..., : r // 2], both[..., r // 2:r]
            turned = torch.cat((x1 * cos - x2 * sin, x1 * sin + x2 * cos), dim=-1)
        both = torch.cat((turned, both[..., r:]), dim=-1).to(dtype)
        q, k = both[:, :heads], both[:, heads:]
    page = state["table"].long()[sequence, position // case["page"]]
    slot = position % case["page"]
    state["keys"][page, :, slot] = k
    state["values"][page, :, slot] = v
    return q.contiguous(), state["keys"], state["values"]


def _plain_attend(state):
    case = state["case"]
    d, heads, kv_heads = case["head_dim"], case["heads"], case["kv_heads"]
    group, longest = heads // kv_heads, state["longest"]
    sequence, number, _ = _rows(state)
    starts, lengths, table = state["starts"].long(), state["lengths"].long(), state["table"].long()
    batch, most = lengths.numel(), state["most_new"]
    # [sequences, kv_heads, keys, d]
    k = state["keys"][table].transpose(1, 2).reshape(batch, kv_heads, -1, d)[:, :, :longest].float()
    v = state["values"][table].transpose(1, 2).reshape(batch, kv_heads, -1, d)[:, :, :longest].float()
    q = torch.zeros(batch, most, heads, d, device=k.device)
    q[sequence, number] = state["q"].float()
    q = q.view(batch, most, kv_heads, group, d).transpose(1, 2).reshape(batch, kv_heads, most * group, d)
    scores = torch.matmul(q, k.transpose(2, 3).contiguous()).mul_(1.0 / math.sqrt(d))
    key = torch.arange(longest, device=k.device)
    position = (lengths - (starts[1:] - starts[:-1]))[:, None] + torch.arange(most, device=k.device)
    seen = (key <= position[..., None]) & (key < lengths[:, None, None])
    if case["window"]:
        seen &= key > position[..., None] - case["window"]
    scores = scores.view(batch, kv_heads, most, group, longest).masked_fill_(~seen[:, None, :, None], -math.inf)
    top = scores.amax(dim=-1, keepdim=True).clamp_(min=-3e38)
    p = scores.sub_(top).exp_()
    total = p.sum(dim=-1, keepdim=True)
    out = torch.matmul(p.view(batch, kv_heads, most * group, longest), v).view(batch, kv_heads, most, group, d)
    out = torch.where(total > 0, out / total, torch.zeros_like(out))
    out = out.transpose(1, 2).reshape(batch, most, heads, d)
    return out[sequence, number].to(state["q"].dtype)


def _plain_copy(state):
    keys, values = state["keys"], state["values"]
    keys[:, state["destinations"]] = keys[:, state["sources"]]
    values[:, state["destinations"]] = values[:, state["sources"]]
    return keys, values


def run(state):
    case = state["case"]
    if own:
        import turbotransformers_amd as tt
        if case["kind"] == "append":
            q = tt.rotary_append(state["qkv"], state["keys"], state["values"], state["table"], state["starts"], state["lengths"], inv_freq=state["inv_freq"],
                                 interleaved=case["interleaved"])
            return q, state["keys"], state["values"]
        if case["kind"] == "attend":
            return tt.paged_attention(state["q"], state["keys"], state["values"], state["table"], state["starts"], state["lengths"], max_tokens=state["most_new"],
                                      max_length=state["longest"], window=case["window"])
        tt.copy_pages(state["keys"], state["values"], state["sources"], state["destinations"])
        return state["keys"], state["values"]
    if case["kind"] == "append":
        return _plain_append(state)
    if case["kind"] == "attend":
        return _plain_attend(state)
    return _plain_copy(state)


# --------------------------------------------------------------------------------- from the definitions, 64 bits ----------
def exact(case, seed):
    state = prepare(case, seed)
    keys, values = state["keys"], state["values"]
    if case["kind"] == "copy":
        for src, dst in zip(state["sources"], state["destinations"]):
            keys[:, dst].copy_(keys[:, src])
            values[:, dst].copy_(values[:, src])
        return keys, values
    d, heads, kv_heads, size = case["head_dim"], case["heads"], case["kv_heads"], case["page"]
    group = heads // kv_heads
    table, starts, lengths = state["table"].tolist(), state["starts"].tolist(), state["lengths"].tolist()
    if case["kind"] == "append":
        keys, values = keys.double(), values.double()
        x = state["qkv"].double().view(-1, heads + 2 * kv_heads, d)
        r = case["rotary"]
        first, second = torch.arange(r // 2, device="cuda"), torch.arange(r // 2, r, device="cuda")
        if case["interleaved"]:
            first, second = 2 * torch.arange(r // 2, device="cuda"), 2 * torch.arange(r // 2, device="cuda") + 1
        y = x.clone()
        for b in range(len(lengths)):
            rows = slice(starts[b], starts[b + 1])
            at = torch.arange(lengths[b] - (starts[b + 1] - starts[b]), lengths[b], device="cuda")
            if r:
                turn = torch.polar(torch.ones((), dtype=torch.float64, device="cuda"), at.double()[:, None] * state["inv_freq"])
                z = torch.complex(x[rows, :heads + kv_heads][..., first], x[rows, :heads + kv_heads][..., second]) * turn[:, None]
                part = y[rows, :heads + kv_heads]
                part[..., first], part[..., second] = z.real, z.imag
            page = torch.tensor(table[b], device="cuda")[torch.div(at, size, rounding_mode="floor")]
            keys[page, :, at % size] = y[rows, heads:heads + kv_heads]
            values[page, :, at % size] = y[rows, heads + kv_heads:]
        return y[:, :heads].contiguous(), keys, values
    out = torch.zeros(state["q"].shape, dtype=torch.float64, device="cuda")
    for b, length in enumerate(lengths):
        pages = table[b][:-(-length // size)]
        n = starts[b + 1] - starts[b]
        far = torch.arange(length - n, length, device="cuda")[:, None] - torch.arange(length, device="cuda")
        hidden = far < 0
        if case["window"]:
            hidden |= far >= case["window"]
        for g in range(kv_heads):
            k = keys[pages, g].double().reshape(-1, d)[:length]
            v = values[pages, g].double().reshape(-1, d)[:length]
            for h in range(g * group, (g + 1) * group):
                s = state["q"][starts[b]:starts[b + 1], h].double() @ k.t() / math.sqrt(d)
                out[starts[b]:starts[b + 1], h] = torch.softmax(s.masked_fill(hidden, -math.inf), dim=1) @ v
    return out
