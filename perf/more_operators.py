"""More operators of a decoder whose keys and values lie in pages, as cases that can be timed and compared.

append   queries and keys of the new tokens normed head by head, turned by their positions, keys and values stored into the pages
sinks    attention that sees a window of the last tokens and the first few tokens of its sequence
shared   attention of sequences whose first tokens lie in the same pages: families of samples, of beams, of questions about one text

A cache is [pages, kv_heads, page_size, head_dim] a layer.  Row b of `table` lists the pages of sequence b in order, `starts` says where
the rows of its new tokens begin and end, `lengths` how many keys it has, the new tokens' among them.  12 heads of 64 are those of this
repository's base model, the other head counts are generic ones.
"""
import math
import random

import torch

own = False

DTYPES = {"f16": torch.float16, "bf16": torch.bfloat16, "f32": torch.float32}
EPS = 1e-6


def listed():
    base = {"heads": 12, "kv_heads": 12, "head_dim": 64, "page": 16}
    grouped = {"heads": 32, "kv_heads": 8, "head_dim": 128, "page": 16}
    return [
        # one decoding step of a small service: eight sequences, a token each; nothing but latency
        {"name": "append_f16_8x1", "kind": "append", "dtype": "f16", **base, "sequences": 8, "new_low": 1, "new_high": 1, "past_low": 5, "past_high": 500,
         "rotary": 64, "interleaved": False, "per_head": False, "weights": "f16", "lengths": 1},
        # prompts in the element type a checkpoint comes in, half of each head turned, pairs side by side, weights for each head
        {"name": "append_f32_5_prompts", "kind": "append", "dtype": "f32", **base, "sequences": 5, "new_low": 33, "new_high": 387, "past_low": 0,
         "past_high": 0, "rotary": 32, "interleaved": True, "per_head": True, "weights": "f32", "lengths": 2},
        # chunks of long documents, shared key/value heads
        {"name": "append_bf16_chunks", "kind": "append", "dtype": "bf16", **grouped, "sequences": 6, "new_low": 512, "new_high": 4096, "past_low": 1,
         "past_high": 100000, "rotary": 128, "interleaved": False, "per_head": False, "weights": "bf16", "lengths": 3},
        # a conversation that has long passed its window, one token at a time
        {"name": "sinks_f16_1x20000", "kind": "attend", "dtype": "f16", **base, "families": "1", "prefix_low": 0, "prefix_high": 0, "new_low": 1, "new_high": 1,
         "past_low": 20000, "past_high": 20000, "window": 1000, "sinks": 4, "lengths": 4},
        # a full batch of such conversations, some still within the window
        {"name": "sinks_bf16_64", "kind": "attend", "dtype": "bf16", **grouped, "families": "64x1", "prefix_low": 0, "prefix_high": 0, "new_low": 1,
         "new_high": 1, "past_low": 300, "past_high": 30000, "window": 2000, "sinks": 16, "lengths": 5},
        # prompts without conversion to half precision
        {"name": "sinks_f32_8_prompts", "kind": "attend", "dtype": "f32", **base, "families": "8x1", "prefix_low": 0, "prefix_high": 0, "new_low": 33,
         "new_high": 900, "past_low": 0, "past_high": 0, "window": 200, "sinks": 5, "lengths": 6},
        # one whole long prompt
        {"name": "sinks_bf16_8192", "kind": "attend", "dtype": "bf16", **grouped, "families": "1", "prefix_low": 0, "prefix_high": 0, "new_low": 8192,
         "new_high": 8192, "past_low": 0, "past_high": 0, "window": 1024, "sinks": 64, "lengths": 7},
        # eight samples of one short prompt, base model
        {"name": "shared_f16_8x1", "kind": "attend", "dtype": "f16", **base, "families": "8", "prefix_low": 400, "prefix_high": 400, "new_low": 1, "new_high": 1,
         "past_low": 1, "past_high": 60, "window": 0, "sinks": 0, "lengths": 8},
        # a service's full batch behind one system prompt
        {"name": "shared_bf16_64", "kind": "attend", "dtype": "bf16", **grouped, "families": "64", "prefix_low": 6000, "prefix_high": 6000, "new_low": 1,
         "new_high": 1, "past_low": 20, "past_high": 1500, "window": 0, "sinks": 0, "lengths": 9},
        # eight requests, eight samples of each, among them some that are alone
        {"name": "shared_bf16_families", "kind": "attend", "dtype": "bf16", **grouped, "families": "2x8 1 3x8 1 8 1 2x8", "prefix_low": 500,
         "prefix_high": 8000, "new_low": 1, "new_high": 1, "past_low": 10, "past_high": 300, "window": 0, "sinks": 0, "lengths": 10},
        # sixteen questions about one long document
        {"name": "shared_f16_16_questions", "kind": "attend", "dtype": "f16", **grouped, "families": "16", "prefix_low": 20000, "prefix_high": 20000,
         "new_low": 20, "new_high": 200, "past_low": 0, "past_high": 0, "window": 0, "sinks": 0, "lengths": 11},
        # four beams over a source text, without conversion to half precision
        {"name": "shared_f32_4_beams", "kind": "attend", "dtype": "f32", **base, "families": "4", "prefix_low": 1500, "prefix_high": 1500, "new_low": 1,
         "new_high": 1, "past_low": 30, "past_high": 30, "window": 0, "sinks": 0, "lengths": 12},
    ]


def _log_int(rng, low, high):
    return min(high, max(low, int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))))


def draw(rng):
    form = rng.choice(["append", "sinks", "sinks", "shared", "shared", "shared"])
    case = {"kind": "append" if form == "append" else "attend", "dtype": rng.choice(["f16", "bf16", "f32"]), "head_dim": rng.choice([64, 128]),
            "kv_heads": rng.choice([1, 2, 4, 8, 12]), "page": rng.choice([16, 32, 64, 128]), "lengths": rng.randrange(10000)}
    case["heads"] = case["kv_heads"] * rng.choice([1, 2, 3, 4, 8] if case["kv_heads"] <= 4 else [1, 2, 4])
    if form == "append":
        case["sequences"] = _log_int(rng, 1, 100)
        most = _log_int(rng, 1, 4096 if case["sequences"] <= 6 else 128)
        case["new_low"], case["new_high"] = rng.randint(1, most), most
        case["past_low"], case["past_high"] = (0, 0) if rng.random() < 0.3 else (1, _log_int(rng, 10, 20000))
        case["rotary"] = rng.choice([case["head_dim"], case["head_dim"], case["head_dim"] // 2, 0])
        case["interleaved"], case["per_head"] = rng.random() < 0.5, rng.random() < 0.3
        case["weights"] = rng.choice(["f32", case["dtype"]])
        return case
    case["window"] = case["sinks"] = case["prefix_low"] = case["prefix_high"] = 0
    if form == "sinks":
        case["window"], case["sinks"] = _log_int(rng, 16, 4000), _log_int(rng, 1, 300)
        if rng.random() < 0.5:  # decoding
            case["families"] = "%dx1" % _log_int(rng, 1, 64)
            longest = _log_int(rng, 8, 30000)
            case["past_low"], case["past_high"] = rng.randint(1, longest), longest
            case["new_low"] = case["new_high"] = 1
        else:
            count = _log_int(rng, 1, 8)
            case["families"] = "%dx1" % count
            most = _log_int(rng, 2, 3000 if count <= 2 else 500)
            longest = _log_int(rng, 8, 5000)
            case["past_low"], case["past_high"] = (0, 0) if rng.random() < 0.5 else (1, longest)
            case["new_low"], case["new_high"] = rng.randint(1, most), most
        return case
    families = [_log_int(rng, 1, 48) for _ in range(_log_int(rng, 1, 6))]
    while sum(families) > 64:
        families.pop()
    case["families"] = " ".join(map(str, families))
    case["prefix_high"] = _log_int(rng, 64, 10000)
    case["prefix_low"] = rng.randint(16, case["prefix_high"])
    longest = _log_int(rng, 1, 1500)
    case["past_low"], case["past_high"] = rng.randint(1, longest), longest
    most = _log_int(rng, 2, 100) if rng.random() < 0.3 and sum(families) <= 20 else 1
    case["new_low"], case["new_high"] = rng.randint(1, most), most
    if rng.random() < 0.2:  # a window behind a text that stays visible, the shared one or a part of it
        case["window"], case["sinks"] = _log_int(rng, 16, 4000), rng.choice([4, case["prefix_low"]])
    return case


def _families(case):
    """Sequences of every family, in order: "2x8 1" are two of eight and one that is alone."""
    if case["kind"] == "append":
        return [1] * case["sequences"]
    out = []
    for word in case["families"].split():
        count, _, members = word.rpartition("x")
        out += [int(members)] * int(count or 1)
    return out


def _lengths(case):
    """Of every sequence: new tokens, keys of its own before them; of every family: the tokens its sequences begin with."""
    rng = random.Random(case["lengths"])
    families = _families(case)
    count = sum(families)
    new = [_log_int(rng, case["new_low"], case["new_high"]) for _ in range(count)]
    past = [_log_int(rng, case["past_low"], case["past_high"]) if case["past_high"] else 0 for _ in range(count)]
    prefix = [_log_int(rng, case["prefix_low"], case["prefix_high"]) if case.get("prefix_high") else 0 for _ in families]
    return new, past, prefix


def _size(case):
    return 4 if case["dtype"] == "f32" else 2


def work(case):
    new, past, prefix = _lengths(case)
    d, heads, kv_heads, size = case["head_dim"], case["heads"], case["kv_heads"], _size(case)
    if case["kind"] == "append":
        return {"bytes": 2 * sum(new) * (heads + 2 * kv_heads) * d * size, "flops": sum(new) * (heads + kv_heads) * (4 * d + 3 * case["rotary"])}
    pairs = keys = b = 0
    for members, p in zip(_families(case), prefix):
        together = p // case["page"] * case["page"] if members > 1 else 0
        most = 0
        for n, own_past in zip(new[b:b + members], past[b:b + members]):
            before = p + own_past
            window, sinks = case["window"] or before + n, case["sinks"] if case["window"] else 0
            far = max(0, before + 1 - window)  # the first key of the first token's window
            pairs += sum(min(at + 1, window + min(sinks, max(0, at + 1 - window))) for at in range(before, before + n))
            keys += before + n - max(far, together) + max(0, min(sinks, far) - together)
            most = max(most, together - max(0, min(far, together) - sinks))
        keys += most
        b += members
    return {"bytes": (2 * sum(new) * heads * d + 2 * keys * kv_heads * d) * size, "flops": 4 * pairs * heads * d}


def prepare(case, seed):
    gen = torch.Generator("cuda").manual_seed(seed)
    dtype = DTYPES[case["dtype"]]
    d, heads, kv_heads, page = case["head_dim"], case["heads"], case["kv_heads"], case["page"]

    def random_values(*shape):
        return torch.randn(shape, generator=gen, device="cuda").to(dtype)

    state = {"case": case}
    new, past, prefix = _lengths(case)
    families = _families(case)
    # A family's full pages of common tokens are one set; the rest of a sequence lies in pages of its own.  Pages lie where the cache had room: in any order, a tenth of
    # them unused.
    shared_pages = [p // page if members > 1 else 0 for members, p in zip(families, prefix)]
    lengths, own_pages, family_of = [], [], []
    for f, members in enumerate(families):
        for _ in range(members):
            b = len(lengths)
            lengths.append(prefix[f] + past[b] + new[b])
            own_pages.append(-(-lengths[b] // page) - shared_pages[f])
            family_of.append(f)
    needed = sum(shared_pages) + sum(own_pages)
    pages = needed + needed // 10 + 1
    order = random.Random(seed).sample(range(pages), needed)
    common = [[order.pop() for _ in range(n)] for n in shared_pages]
    table = torch.zeros((len(new), max(-(-n // page) for n in lengths)), dtype=torch.int32)
    rows = []
    for b, f in enumerate(family_of):
        row = common[f] + [order.pop() for _ in range(own_pages[b])]
        table[b, :len(row)] = torch.tensor(row, dtype=torch.int32)
        first = sum(families[:f])
        rows.append([first, first + families[f], shared_pages[f] * page])
    state["table"] = table.cuda()
    state["lengths"] = torch.tensor(lengths, dtype=torch.int32).cuda()
    state["starts"] = torch.tensor([sum(new[:b]) for b in range(len(new) + 1)], dtype=torch.int32).cuda()
    state["keys"], state["values"] = random_values(pages, kv_heads, page, d), random_values(pages, kv_heads, page, d)
    if case["kind"] == "append":
        # heads of a projection differ in size, which is what they are normed for
        sizes = torch.exp(torch.randn((heads + 2 * kv_heads, 1), generator=gen, device="cuda"))
        rows = torch.randn((sum(new), heads + 2 * kv_heads, d), generator=gen, device="cuda") * sizes
        state["qkv"] = rows.flatten(1).to(dtype)
        for name, count in (("q_norm", heads), ("k_norm", kv_heads)):
            shape = (count, d) if case["per_head"] else (d,)
            state[name] = (1 + 0.3 * torch.randn(shape, generator=gen, device="cuda")).to(DTYPES[case["weights"]])
        r = case["rotary"]
        state["inv_freq"] = 10000.0 ** -(torch.arange(0, r, 2, dtype=torch.float64, device="cuda") / r) if r else None
        return state
    # the plan of a step: which sequences are a family, as a scheduler knows them
    state["families"] = torch.tensor(rows, dtype=torch.int32).cuda() if max(shared_pages) > 0 else None
    state["family_count"], state["max_shared"] = sum(n > 0 for n in shared_pages), max(shared_pages) * page
    state["max_new"], state["max_length"] = max(new), max(lengths)
    # (as numbers of the host too: the plain form goes through the batch with them)
    state["host"] = {"new": new, "lengths": lengths, "families": families, "shared": [n * page for n in shared_pages]}
    state["q"] = random_values(sum(new), heads, d)
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
    q, k, v = x[:, :heads].float(), x[:, heads:heads + kv_heads].float(), x[:, heads + kv_heads:]
    q = q * torch.rsqrt((q * q).mean(-1, keepdim=True) + EPS) * state["q_norm"].float()
    k = k * torch.rsqrt((k * k).mean(-1, keepdim=True) + EPS) * state["k_norm"].float()
    both = torch.cat((q, k), dim=1)
    if r:
        angle = position.double()[:, None, None] * state["inv_freq"]
        cos, sin = angle.cos().float(), angle.sin().float()
        if case["interleaved"]:
            x1, x2 = both[..., 0:r:2], both[..., 1:r:2]
            turned = torch.stack((x1 * cos - x2 * sin, x1 * sin + x2 * cos), dim=-1).flatten(-2)
        else:
            x1, x2 = both[..., : r // 2], both[..., r // 2:r]
            turned = torch.cat((x1 * cos - x2 * sin, x1 * sin + x2 * cos), dim=-1)
        both = torch.cat((turned, both[..., r:]), dim=-1)
    both = both.to(dtype)
    page = state["table"].long()[sequence, position // case["page"]]
    slot = position % case["page"]
    state["keys"][page, :, slot] = both[:, heads:]
    state["values"][page, :, slot] = v
    return both[:, :heads].contiguous(), state["keys"], state["values"]


def _part(scores, v):
    """Maximum, sum of exponentials and their product with v, of scores [.., rows, keys]."""
    top = scores.amax(dim=-1, keepdim=True).clamp_(min=-3e38)
    p = scores.sub_(top).exp_()
    return top, p.sum(dim=-1, keepdim=True), torch.matmul(p, v)


def _plain_attend(state):
    """Family by family: the keys that its sequences share once, for all of its rows; the others sequence by sequence, padded to the longest."""
    case, host = state["case"], state["host"]
    d, heads, kv_heads, page = case["head_dim"], case["heads"], case["kv_heads"], case["page"]
    group = heads // kv_heads
    table, dtype, device = state["table"].long(), state["q"].dtype, state["q"].device
    sequence, number, position = _rows(state)
    outs, b0, row0 = [], 0, 0
    runs = []
    for members, shared in zip(host["families"], host["shared"]):  # sequences that are alone go together
        if members == 1 and runs and runs[-1][1] == 0:
            runs[-1][0] += 1
        else:
            runs.append([members, shared])

    def seen(key, at):
        ok = key <= at
        if case["window"]:
            ok &= (key > at - case["window"]) | (key < case["sinks"])
        return ok

    for members, shared in runs:
        new = host["new"][b0:b0 + members]
        n, most, longest = sum(new), max(new), max(host["lengths"][b0:b0 + members])
        rows = slice(row0, row0 + n)
        q = state["q"][rows].float()
        at = position[rows]
        # own keys [members, kv_heads, keys, d]
        pages = table[b0:b0 + members, shared // page:-(-longest // page)]
        k = state["keys"][pages].transpose(1, 2).reshape(members, kv_heads, -1, d).float()
        v = state["values"][pages].transpose(1, 2).reshape(members, kv_heads, -1, d).float()
        local, place = sequence[rows] - b0, number[rows]
        padded = torch.zeros(members, most, heads, d, device=device)
        padded[local, place] = q
        where = torch.full((members, most), -1, dtype=torch.long, device=device)
        where[local, place] = at
        padded = padded.view(members, most, kv_heads, group, d).transpose(1, 2).reshape(members, kv_heads, most * group, d)
        scores = torch.matmul(padded, k.transpose(2, 3).contiguous()).mul_(1.0 / math.sqrt(d)).view(members, kv_heads, most, group, -1)
        ok = seen(shared + torch.arange(k.shape[2], device=device), where[..., None])
        scores = scores.masked_fill_(~ok[:, None, :, None], -math.inf).view(members, kv_heads, most * group, -1)
        parts = []
        for x in _part(scores, v):
            x = x.view(members, kv_heads, most, group, -1).transpose(1, 2).reshape(members, most, heads, -1)
            parts.append(x[local, place])
        top, total, out = parts
        if shared:
            pages = table[b0, :shared // page]
            k = state["keys"][pages].transpose(0, 1).reshape(kv_heads, -1, d).float()
            v = state["values"][pages].transpose(0, 1).reshape(kv_heads, -1, d).float()
            together = q.view(n, kv_heads, group, d).transpose(0, 1).reshape(kv_heads, n * group, d)
            scores = torch.matmul(together, k.transpose(1, 2).contiguous()).mul_(1.0 / math.sqrt(d)).view(kv_heads, n, group, -1)
            ok = seen(torch.arange(shared, device=device), at[:, None])
            scores = scores.masked_fill_(~ok[None, :, None], -math.inf).view(kv_heads, n * group, -1)
            top1, total1, out1 = (x.view(kv_heads, n, group, -1).transpose(0, 1).reshape(n, heads, -1) for x in _part(scores, v))
            both = torch.maximum(top, top1)
            w, w1 = torch.exp(top - both), torch.exp(top1 - both)
            total, out = total * w + total1 * w1, out * w + out1 * w1
        outs.append(torch.where(total > 0, out / total, torch.zeros_like(out)).to(dtype))
        b0, row0 = b0 + members, row0 + n
    return torch.cat(outs)


def run(state):
    case = state["case"]
    if own:
        import turbotransformers_amd as tt
        if case["kind"] == "append":
            q = tt.rotary_append(state["qkv"], state["keys"], state["values"], state["table"], state["starts"], state["lengths"], inv_freq=state["inv_freq"],
                                 interleaved=case["interleaved"], q_norm=state["q_norm"], k_norm=state["k_norm"], eps=EPS)
            return q, state["keys"], state["values"]
        return tt.paged_attention(state["q"], state["keys"], state["values"], state["table"], state["starts"], state["lengths"], max_tokens=state["max_new"],
                                  max_length=state["max_length"], window=case["window"], sinks=case["sinks"], families=state["families"],
                                  family_count=state["family_count"], max_shared=state["max_shared"])
    return _plain_append(state) if case["kind"] == "append" else _plain_attend(state)


# --------------------------------------------------------------------------------- from the definitions, 64 bits ----------
def exact(case, seed):
    state = prepare(case, seed)
    keys, values = state["keys"], state["values"]
    d, heads, kv_heads, size = case["head_dim"], case["heads"], case["kv_heads"], case["page"]
    group = heads // kv_heads
    table, starts, lengths = state["table"].tolist(), state["starts"].tolist(), state["lengths"].tolist()
    if case["kind"] == "append":
        keys, values = keys.double(), values.double()
        y = state["qkv"].double().view(-1, heads + 2 * kv_heads, d)
        r = case["rotary"]
        for h in range(heads + kv_heads):
            weight = (state["q_norm"] if h < heads else state["k_norm"]).double()
            if case["per_head"]:
                weight = weight[h if h < heads else h - heads]
            power = (y[:, h] ** 2).sum(-1) / d
            y[:, h] = y[:, h] / (power + EPS).sqrt()[:, None] * weight
        first, second = torch.arange(r // 2, device="cuda"), torch.arange(r // 2, r, device="cuda")
        if case["interleaved"]:
            first, second = 2 * torch.arange(r // 2, device="cuda"), 2 * torch.arange(r // 2, device="cuda") + 1
        for b in range(len(lengths)):
            rows = slice(starts[b], starts[b + 1])
            at = torch.arange(lengths[b] - (starts[b + 1] - starts[b]), lengths[b], device="cuda")
            if r:
                turn = torch.polar(torch.ones((), dtype=torch.float64, device="cuda"), at.double()[:, None] * state["inv_freq"])
                part = y[rows, :heads + kv_heads]
                z = torch.complex(part[..., first], part[..., second]) * turn[:, None]
                part[..., first], part[..., second] = z.real, z.imag
            page = torch.tensor(table[b], device="cuda")[torch.div(at, size, rounding_mode="floor")]
            keys[page, :, at % size] = y[rows, heads:heads + kv_heads]
            values[page, :, at % size] = y[rows, heads + kv_heads:]
        return y[:, :heads].contiguous(), keys, values
    out = torch.zeros(state["q"].shape, dtype=torch.float64, device="cuda")
    for b, length in enumerate(lengths):
        pages = table[b][:-(-length // size)]
        n = starts[b + 1] - starts[b]
        key = torch.arange(length, device="cuda")
        far = torch.arange(length - n, length, device="cuda")[:, None] - key
        hidden = far < 0
        if case["window"]:
            hidden |= (far >= case["window"]) & (key >= case["sinks"])
        for g in range(kv_heads):
            k = keys[pages, g].double().reshape(-1, d)[:length]
            v = values[pages, g].double().reshape(-1, d)[:length]
            for h in range(g * group, (g + 1) * group):
                s = state["q"][starts[b]:starts[b + 1], h].double() @ k.t() / math.sqrt(d)
                out[starts[b]:starts[b + 1], h] = torch.softmax(s.masked_fill(hidden, -math.inf), dim=1) @ v
    return out
