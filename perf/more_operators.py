"""Cases of a prompt's way into the cache and of a batch that shares one: their plain forms and definitions in 64 bits.

* ``rotary``: rotary positions of a step's queries and Keys (half and interleaved pairs, the whole head or a part of it,
  frequencies stretched for long contexts), at positions far from 0;
* ``prompt``: causal attention of whole prompts over their own tokens, grouped heads, sequences of different lengths packed
  behind one another or padded to one length;
* ``prefix``: attention over the 4-bit pages for sequences that share a long prefix: its pages are read once for all of them.

The geometries are those the repository measures: 28 query heads on 4 KV heads and 40 on 8, head_dim 128, 4096-token prompts,
histories of 1k to 32k tokens; head_dim 64 and fp16 stand for smaller models.
"""
import math

import torch

own = False

PAGE = 64      # tokens of a page
GROUP = 32     # channels that share a scale and a minimum
TYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}


def listed():
    big = dict(nq=28, H=4, D=128, dtype="bf16")
    wide = dict(nq=40, H=8, D=128, dtype="bf16")
    return [
        # The next token of each of 16 sequences at 8k tokens: the smallest call, where latency counts.
        dict(big, name="rotary one token", op="rotary", B=16, T=1, packed=False, first=8192, spread=127, part=128, pairs="half",
             factor=1.0),
        # Four 4096-token prompts, packed: the largest.
        dict(big, name="rotary prompts", op="rotary", B=4, T=4096, packed=True, first=0, spread=0, part=128, pairs="half", factor=1.0),
        # Ragged chunks around 128k positions, frequencies stretched four times, half of each head rotated in adjacent pairs.
        dict(name="rotary far chunks", op="rotary", B=5, T=777, nq=40, H=8, D=64, dtype="f16", packed=True, first=131000, spread=701,
             part=32, pairs="adjacent", factor=4.0),
        # A short question.
        dict(big, name="prompt short", op="prompt", B=1, T=61, spread=0, packed=True),
        # Prompts of a serving batch, of any length from a few tokens on, packed.
        dict(wide, name="prompt ragged", op="prompt", B=9, T=2305, spread=2297, packed=True),
        # The measured prompt, four at once.
        dict(big, name="prompt 4 x 4096", op="prompt", B=4, T=4096, spread=0, packed=True),
        # A long document.
        dict(big, name="prompt 8192", op="prompt", B=1, T=8192, spread=0, packed=True),
        # A padded batch of a smaller model with as many KV heads as query heads.
        dict(name="prompt padded", op="prompt", B=6, T=1500, nq=8, H=8, D=64, dtype="f16", spread=1111, packed=False),
        # Four users of one 1k system prompt, a few turns in.
        dict(big, name="prefix 4 x 1k", op="prefix", B=4, groups=1, prefix=1024, own=300, spread=280, q_len=1, alone=0),
        # A large serving batch behind a 16k system prompt with its examples.
        dict(wide, name="prefix 64 x 16k", op="prefix", B=64, groups=1, prefix=16384, own=700, spread=600, q_len=1, alone=0),
        # Three prompts shared by unequal shares of a batch, two sequences with none, three drafted tokens each, fp16.
        dict(name="prefix drafts", op="prefix", B=29, groups=3, prefix=9024, own=1500, spread=1490, q_len=3, alone=2, nq=40, H=8, D=64,
             dtype="f16"),
        # A chunk of a long prompt behind 32k tokens that are in the cache already.
        dict(big, name="prefix chunk", op="prefix", B=1, groups=1, prefix=32768, own=512, spread=0, q_len=512, alone=0),
    ]


def _spread(rng, low, high):
    return int(round(low * (high / low) ** rng.random()))


def draw(rng):
    case = dict(op=rng.choice(["rotary", "prompt", "prefix"]), D=rng.choice([64, 128, 128]), dtype=rng.choice(["bf16", "bf16", "f16"]))
    case["nq"], case["H"] = rng.choice([(28, 4), (40, 8), (8, 8), (16, 1), (14, 2), (32, 8)])
    if case["op"] == "rotary":
        case.update(dtype=rng.choice(["bf16", "bf16", "f16", "f32"]), B=_spread(rng, 1, 32), T=_spread(rng, 1, 4096),
                    packed=rng.random() < 0.5, first=_spread(rng, 1, 200000) - 1, pairs=rng.choice(["half", "half", "adjacent"]),
                    part=rng.choice([case["D"], case["D"], case["D"] // 2, case["D"] // 4]), factor=rng.choice([1.0, 1.0, 4.0, 8.0]))
        case["spread"] = rng.randrange(min(case["first"], case["T"]) + 1)
        while case["B"] * case["T"] * (case["nq"] + case["H"]) * case["D"] * (2 if case["dtype"] == "f32" else 1) > 16384 * 32 * 128:
            case["T"] = max(1, case["T"] // 2)
        case["spread"] = min(case["spread"], case["T"] - 1)
        return case
    if case["op"] == "prompt":
        case.update(B=_spread(rng, 1, 12), T=_spread(rng, 1, 6000), packed=rng.random() < 0.7)
        while case["B"] * case["nq"] * case["T"] ** 2 > 4 * 28 * 4096 ** 2:
            case["T"] = max(1, case["T"] * 2 // 3)
        case["spread"] = rng.randrange(case["T"]) if rng.random() < 0.7 else 0
        return case
    case.update(B=_spread(rng, 1, 48), q_len=rng.choice([1, 1, 1, 2, 5, 64]), prefix=PAGE * _spread(rng, 1, 400), own=_spread(rng, 64, 1200))
    while case["B"] * case["nq"] * case["q_len"] * (case["prefix"] + case["own"]) * case["D"] > 28 * 512 * 33280 * 128 or \
            case["B"] * case["H"] * (case["prefix"] + case["own"]) > 64 * 8 * 17084:
        case["B"] = max(1, case["B"] * 2 // 3)
        case["prefix"] = max(PAGE, case["prefix"] // 128 * PAGE)
    case["own"] = max(case["own"], case["q_len"])
    case["spread"] = rng.randrange(case["own"] - case["q_len"] + 1)
    case["alone"] = rng.randrange(2) if case["B"] > 2 else 0
    case["groups"] = rng.randrange(1, min(4, case["B"] - case["alone"]) + 1)
    return case


def _lengths(case, top, spread):
    """Another length for each sequence, the longest first: top, ..., at least top - spread."""
    return [top - (b * 7919) % (spread + 1) for b in range(case["B"])]


# ---------------------------------------------------------------- inputs: rotary positions

def _frequencies(case):
    """Turns per position of each pair, in 64 bits: base 10^4 ^ (-2 i / part) radians; with a factor above 1, pairs that turn
    less than once in the original 4096 positions are that much slower, those that turn 32 times are as they were, and between
    them the two are mixed in proportion.  And the factor on the rotated channels that goes with it."""
    n, part, factor = case["part"] // 2, case["part"], case["factor"]
    turns = torch.tensor([10000.0 ** (-2.0 * i / part) / (2.0 * math.pi) for i in range(n)], dtype=torch.float64)
    if factor == 1.0:
        return turns, 1.0
    where = [part * math.log(4096.0 / (beta * 2.0 * math.pi)) / (2.0 * math.log(10000.0)) for beta in (32.0, 1.0)]
    low, high = max(math.floor(where[0]), 0), min(math.ceil(where[1]), part - 1)
    ramp = ((torch.arange(n, dtype=torch.float64) - low) / max(high - low, 0.001)).clamp(0, 1)
    return turns / factor * ramp + turns * (1 - ramp), 0.1 * math.log(factor) + 1.0


def _fixed(turns):
    """Turns as whole numbers of 2^-64 turns."""
    return torch.tensor([int(round(t * 2.0 ** 64)) for t in turns.tolist()], dtype=torch.int64, device="cuda")


def _prepare_rotary(case, g):
    B, D, dt = case["B"], case["D"], TYPES[case["dtype"]]
    turns, magnitude = _frequencies(case)
    state = dict(case=case, freqs=_fixed(turns), magnitude=magnitude)
    if case["packed"]:
        counts = _lengths(case, case["T"], case["spread"])
        n = sum(counts)
        state["positions"] = torch.cat([case["first"] + 13 * b + torch.arange(c) for b, c in enumerate(counts)]).cuda()
        state["query"] = torch.randn(n, case["nq"], D, generator=g, device="cuda").to(dt)
        state["key"] = torch.randn(n, case["H"], D, generator=g, device="cuda").to(dt)
    else:
        state["start"] = torch.tensor([case["first"] - (b * 7919) % (case["spread"] + 1) for b in range(B)], dtype=torch.int32, device="cuda")
        # as the projections give them: [B, T, heads, D], seen as [B, heads, T, D]
        state["query"] = torch.randn(B, case["T"], case["nq"], D, generator=g, device="cuda").to(dt).transpose(1, 2)
        state["key"] = torch.randn(B, case["T"], case["H"], D, generator=g, device="cuda").to(dt).transpose(1, 2)
    return state


# ---------------------------------------------------------------- inputs: prompts

def _prepare_prompt(case, g):
    B, T, D, dt = case["B"], case["T"], case["D"], TYPES[case["dtype"]]
    counts = _lengths(case, T, case["spread"])
    lead = (sum(counts),) if case["packed"] else (B, T)

    def made(heads, far):
        x = torch.randn(*lead, heads, D, generator=g, device="cuda")
        if far:
            x[..., :: D // 6] *= 4.0                   # Keys have a few channels of larger values
        return x.to(dt)

    state = dict(case=case, query=made(case["nq"], False), key=made(case["H"], True), value=made(case["H"], False), scaling=D ** -0.5)
    if case["packed"]:
        ends = [sum(counts[:b]) for b in range(B + 1)]
        state["starts"] = torch.tensor(ends, dtype=torch.int32, device="cuda")
    else:
        state.update({n: state[n].transpose(1, 2) for n in ("query", "key", "value")})
        state["counts"] = torch.tensor(counts, dtype=torch.int32, device="cuda")
    return state


# ---------------------------------------------------------------- inputs: 4-bit pages

def _quantise(x):
    """Codes, scales and minima of [..., D] fp32 values, for every GROUP channels."""
    x = x.unflatten(-1, (-1, GROUP))
    lo, hi = x.amin(-1, keepdim=True), x.amax(-1, keepdim=True)
    s, z = ((hi - lo) * (1.0 / 15.0)).half(), lo.half()
    s32 = s.float()
    r = torch.where(s32 > 0, torch.ones_like(s32) / s32, torch.zeros_like(s32))
    return torch.round((x - z.float()) * r).clamp(0, 15), s, z


def _words(nibbles):
    """int32 words of the eight codes of the last axis, the first in the low bits."""
    shift = torch.arange(8, device=nibbles.device) * 4
    return (nibbles.to(torch.int64) << shift).sum(-1).to(torch.int32)


def _records(key, value):
    """The pool's records [..., pages, 20 D] of fp32 Key and Value [..., tokens, D], tokens a multiple of PAGE."""
    return torch.cat([_key_words(*_quantise(key)), _value_words(*_quantise(value))], -1)


def _params(s, z):
    n = s.shape[-3] // PAGE
    return torch.cat([s, z], -1).contiguous().view(torch.int32).reshape(*s.shape[:-3], n, -1)


def _key_words(c, s, z):
    """Channel 32 G + 8 t + n of a token is nibble n of its word (t, G)."""
    lead, n, G = c.shape[:-3], c.shape[-3] // PAGE, c.shape[-2]
    w = _words(c.reshape(*lead, n, PAGE, G, 4, 8)).transpose(-1, -2)
    return torch.cat([w.reshape(*lead, n, -1), _params(s, z)], -1)


def _value_words(c, s, z):
    """Channel 64 w + 32 u + 4 g + n of token 8 b + 2 t + o is nibble 4 u + n of the page's word (b, g, t, o, w)."""
    lead, n, G = c.shape[:-3], c.shape[-3] // PAGE, c.shape[-2]
    c = c.reshape(*lead, n, 8, 4, 2, G // 2, 2, 8, 4)
    d = len(lead) + 1
    w = _words(c.permute(*range(d), d, d + 5, d + 1, d + 2, d + 3, d + 4, d + 6).flatten(-2))
    return torch.cat([w.reshape(*lead, n, -1), _params(s, z)], -1)


def _groups(case):
    """Each sequence's group (-1: none) and each group's shared pages: all have another length."""
    B, n, pages = case["B"], case["groups"], case["prefix"] // PAGE
    return [b % n if b < B - case["alone"] else -1 for b in range(B)], [pages - (37 * g) % (pages // 2 + 1) for g in range(n)]


def _tails(case):
    """The tokens of each sequence behind its shared pages, the step's query tokens among them."""
    return _lengths(case, case["own"], case["spread"])


def _made(case, seed, what, tokens):
    """Key and Value [H, tokens, D] of a shared prefix (0, group) or a sequence's own tokens (1, sequence): normal, a few Key
    channels of each head larger, and a slow drift, so that some pages matter more than others."""
    g = torch.Generator(device="cuda")
    g.manual_seed(seed * 1009 + what[0] * 500009 + what[1] * 9176 + 11)
    H, D = case["H"], case["D"]
    k = torch.randn(H, tokens, D, generator=g, device="cuda")
    v = torch.randn(H, tokens, D, generator=g, device="cuda")
    k[:, :, :: D // 6] *= 4.0
    drift = torch.randn(H, tokens // 256 + 2, D, generator=g, device="cuda")
    k += drift.repeat_interleave(256, 1)[:, 100:100 + tokens]
    dt = TYPES[case["dtype"]]
    return k.to(dt).float(), v.to(dt).float()


def _prepare_prefix(case, seed, g):
    B, H, D = case["B"], case["H"], case["D"]
    group, shared = _groups(case)
    tails = _tails(case)
    held = [PAGE * (shared[x] if x >= 0 else 0) + t for x, t in zip(group, tails)]
    width = -(-max(held) // PAGE)
    tail_pages = [-(-t // PAGE) for t in tails]
    n = sum(shared) + sum(tail_pages)
    order = torch.randperm(n, generator=g, device="cuda")            # the pages lie in the pool in no order
    pages = torch.zeros(n, H, 20 * D, dtype=torch.int32, device="cuda")
    table = torch.full((B, width), -1, dtype=torch.int32, device="cuda")
    at = 0
    prefix_rows = []
    for x, count in enumerate(shared):
        rows = order[at:at + count]
        pages[rows] = _records(*_made(case, seed, (0, x), PAGE * count)).transpose(0, 1)
        prefix_rows.append(rows)
        at += count
    for b in range(B):
        rows = order[at:at + tail_pages[b]]
        k, v = (torch.nn.functional.pad(x, (0, 0, 0, -tails[b] % PAGE)) for x in _made(case, seed, (1, b), tails[b]))
        pages[rows] = _records(k, v).transpose(0, 1)
        at += tail_pages[b]
        first = shared[group[b]] if group[b] >= 0 else 0
        if first:
            table[b, :first] = prefix_rows[group[b]]
        table[b, first:first + tail_pages[b]] = rows
    q = torch.randn(B, case["nq"], case["q_len"], D, generator=g, device="cuda")
    return dict(case=case, pages=pages, table=table, lengths=torch.tensor(held, dtype=torch.int32, device="cuda"),
                group=torch.tensor(group, dtype=torch.int32, device="cuda"), shared=torch.tensor(shared, dtype=torch.int32, device="cuda"),
                query=q.to(TYPES[case["dtype"]]), scaling=D ** -0.5)


def prepare(case, seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed * 31 + 5)
    if case["op"] == "rotary":
        return _prepare_rotary(case, g)
    return _prepare_prompt(case, g) if case["op"] == "prompt" else _prepare_prefix(case, seed, g)


# ---------------------------------------------------------------- the plain forms

def _rotated(x, cos, sin, case):
    """x [..., D] turned by angles of cosine and sine [..., part / 2]."""
    part, n = case["part"], case["part"] // 2
    y = x.float()
    if case["pairs"] == "half":
        a, b = y[..., :n], y[..., n:part]
        turned = torch.cat([a * cos - b * sin, b * cos + a * sin], -1)
    else:
        a, b = y[..., 0:part:2], y[..., 1:part:2]
        turned = torch.stack([a * cos - b * sin, b * cos + a * sin], -1).flatten(-2)
    return torch.cat([turned, y[..., part:]], -1).to(x.dtype)


def _plain_rotary(state):
    case = state["case"]
    if case["packed"]:
        at = state["positions"].double().unsqueeze(1)                                          # [tokens, 1 head]
    else:
        at = (state["start"].view(-1, 1) + torch.arange(case["T"], device="cuda")).double().unsqueeze(1)
    turns = at.unsqueeze(-1) * (state["freqs"].double() * 2.0 ** -64)                          # in 64 bits: far positions
    angle = (turns - turns.floor()) * (2.0 * math.pi)
    cos, sin = (angle.cos() * state["magnitude"]).float(), (angle.sin() * state["magnitude"]).float()
    return _rotated(state["query"], cos, sin, case), _rotated(state["key"], cos, sin, case)


def _softmax(logits, seen):
    logits = logits.masked_fill(~seen, -float("inf"))
    most = logits.amax(-1, keepdim=True)
    p = torch.exp(logits - torch.where(most == -float("inf"), torch.zeros_like(most), most))
    total = p.sum(-1, keepdim=True)
    return p / torch.where(total == 0, torch.ones_like(total), total)


def _plain_prompt(state):
    case = state["case"]
    B, T, nq, H, D = case["B"], case["T"], case["nq"], case["H"], case["D"]
    q, k, v = state["query"], state["key"], state["value"]
    i = torch.arange(T, device="cuda")
    if case["packed"]:
        first, last = state["starts"][:-1].long(), state["starts"][1:].long()
        rows = (first.view(-1, 1) + i).clamp(max=q.shape[0] - 1)
        live = i < (last - first).view(-1, 1)                                                  # [B, T]
        q, k, v = (x[rows].transpose(1, 2) for x in (q, k, v))
    else:
        live = i < state["counts"].view(-1, 1)
    q32 = q.float().reshape(B, H, nq // H * T, D)
    seen = (i <= i.view(-1, 1)) & live.view(B, 1, 1, 1, T) & live.view(B, 1, 1, T, 1)
    logits = (q32 @ k.float().transpose(-1, -2)).view(B, H, nq // H, T, T) * state["scaling"]
    p = _softmax(logits, seen)
    out = (p.flatten(2, 3) @ v.float()).view(B, nq, T, D).to(q.dtype)
    if case["packed"]:
        return out.transpose(1, 2)[live]                                                       # [tokens, nq, D]
    return out


def _nibbles(words):
    shift = torch.arange(8, device=words.device, dtype=torch.int32) * 4
    return ((words.unsqueeze(-1) >> shift) & 15).float()


def _values(c, s, z):
    return (c * s.float() + z.float()).flatten(-2)


def _unpacked(rec):
    """fp32 Key and Value [..., PAGE, D] of records [..., 20 D]."""
    D = rec.shape[-1] // 20
    G, lead = D // GROUP, rec.shape[:-1]
    d = len(lead)
    kc, kp, vc, vp = rec.split([8 * D, 2 * D, 8 * D, 2 * D], -1)
    c = _nibbles(kc.reshape(*lead, PAGE, 4, G)).transpose(-2, -3).flatten(-2)
    p = kp.contiguous().view(torch.float16).reshape(*lead, PAGE, G, 2)
    key = _values(c, p[..., :1], p[..., 1:])
    c = _nibbles(vc.reshape(*lead, 8, 8, 4, 2, G // 2)).unflatten(-1, (2, 4))                  # b g t o w u n
    c = c.permute(*range(d), d, d + 2, d + 3, d + 4, d + 5, d + 1, d + 6)
    p = vp.contiguous().view(torch.float16).reshape(*lead, PAGE, G, 2)
    return key, _values(c.reshape(*lead, PAGE, G, GROUP), p[..., :1], p[..., 1:])


def _plain_prefix(state):
    q, case = state["query"], state["case"]
    B, nq, q_len, D = q.shape
    H = case["H"]
    rows = state["table"].long().clamp(min=0)
    k, v = (x[rows].permute(0, 2, 1, 3, 4).flatten(2, 3) for x in _unpacked(state["pages"]))   # [B, H, tokens, D]
    q32 = q.float().view(B, H, nq // H * q_len, D)
    logits = (q32 @ k.transpose(-1, -2)).view(B, H, nq // H, q_len, -1) * state["scaling"]
    sees = state["lengths"].view(-1, 1) - q_len + torch.arange(q_len, device="cuda") + 1
    seen = torch.arange(k.shape[2], device="cuda") < sees.view(B, 1, 1, q_len, 1)
    p = _softmax(logits, seen)
    return (p.flatten(2, 3) @ v).view(B, nq, q_len, D).to(q.dtype)


def run(state):
    case = state["case"]
    if not own:
        return {"rotary": _plain_rotary, "prompt": _plain_prompt, "prefix": _plain_prefix}[case["op"]](state)
    from logitfill_b200 import int4, prompt

    if case["op"] == "rotary":
        return prompt.rotary_embed(state["query"], state["key"], state["freqs"], positions=state.get("positions"), start=state.get("start"),
                                   magnitude=state["magnitude"], interleaved=case["pairs"] == "adjacent")
    if case["op"] == "prompt":
        return prompt.prompt_attention(state["query"], state["key"], state["value"], state["scaling"], starts=state.get("starts"),
                                       counts=state.get("counts"))
    return int4.int4_prefix_attention(state["query"], state["pages"], state["table"], state["lengths"], state["scaling"],
                                      state["group"], state["shared"])


# ---------------------------------------------------------------- what a pass cannot do without

def work(case):
    B, nq, H, D = case["B"], case["nq"], case["H"], case["D"]
    size = 4 if case["dtype"] == "f32" else 2
    if case["op"] == "rotary":
        n = sum(_lengths(case, case["T"], case["spread"])) if case["packed"] else B * case["T"]
        where = 8 * n if case["packed"] else 4 * B
        return {"bytes": 2 * n * (nq + H) * D * size + where + 4 * case["part"], "flops": n * (nq + H) * case["part"] * 3}
    if case["op"] == "prompt":
        counts = _lengths(case, case["T"], case["spread"])
        n = sum(counts)
        total = n * (nq + 2 * H) * D * size + (n if case["packed"] else B * case["T"]) * nq * D * size
        return {"bytes": total, "flops": sum(4 * nq * D * c * (c + 1) // 2 for c in counts)}
    group, shared = _groups(case)
    q_len, token = case["q_len"], D + D // 4                         # bytes of a token and KV head in the pages
    total = 2 * 2 * B * nq * q_len * D + H * PAGE * sum(shared) * token
    flops = 0
    for x, tail in zip(group, _tails(case)):
        length = tail + (PAGE * shared[x] if x >= 0 else 0)
        total += H * tail * token
        flops += sum(4 * nq * D * (length - i) for i in range(q_len))
    return {"bytes": total, "flops": flops}


# ---------------------------------------------------------------- the definitions in 64 bits

def _exact_rotary(case, seed):
    state = prepare(case, seed)
    n, part = case["part"] // 2, case["part"]
    turns = state["freqs"].tolist()
    at = state["positions"].tolist() if case["packed"] else [s + t for s in state["start"].tolist() for t in range(case["T"])]
    # position times frequency in whole numbers, so that whole turns drop out exactly
    distinct = sorted(set(at))
    table = torch.tensor([[(p * t) % (1 << 64) / 2.0 ** 64 for t in turns] for p in distinct], dtype=torch.float64, device="cuda")
    places = {p: i for i, p in enumerate(distinct)}
    angle = table[torch.tensor([places[p] for p in at], device="cuda")] * (2.0 * math.pi)
    turn = torch.polar(torch.full_like(angle, state["magnitude"]), angle)                      # [tokens, n] complex
    if not case["packed"]:
        turn = turn.view(case["B"], 1, case["T"], n)
    else:
        turn = turn.unsqueeze(1)
    out = []
    for x in (state["query"].double(), state["key"].double()):
        first, second = (slice(0, n), slice(n, part)) if case["pairs"] == "half" else (slice(0, part, 2), slice(1, part, 2))
        y = torch.complex(x[..., first].contiguous(), x[..., second].contiguous()) * turn
        z = x.clone()
        z[..., first], z[..., second] = y.real, y.imag
        out.append(z)
    return tuple(out)


def _exact_prompt(case, seed):
    state = prepare(case, seed)
    group = case["nq"] // case["H"]
    counts = _lengths(case, case["T"], case["spread"])
    out = torch.zeros(state["query"].shape, dtype=torch.float64, device="cuda")
    at = 0
    for b, c in enumerate(counts):
        def part(x):
            return (x[at:at + c].transpose(0, 1) if case["packed"] else x[b, :, :c]).double()   # [heads, c, D]

        q, k, v = part(state["query"]), part(state["key"]), part(state["value"])
        for h in range(case["nq"]):
            for low in range(0, c, 2048):
                high = min(c, low + 2048)
                logits = q[h, low:high] @ k[h // group, :high].T * state["scaling"]
                later = torch.arange(high, device="cuda") > torch.arange(low, high, device="cuda").view(-1, 1)
                made = torch.softmax(logits.masked_fill(later, -float("inf")), -1) @ v[h // group, :high]
                if case["packed"]:
                    out[at + low:at + high, h] = made
                else:
                    out[b, h, low:high] = made
        at += c
    return out


def _stored64(x):
    """What the cache stands for, in 64 bits, of values [..., D]: a group's scale and minimum are fp16, a code is the
    nearest whole number of steps above the minimum, found in fp32."""
    x = x.double().reshape(*x.shape[:-1], x.shape[-1] // GROUP, GROUP)
    low = x.min(-1, keepdim=True).values
    wide = (x.max(-1, keepdim=True).values - low).float().double()
    step = (wide * float(torch.tensor(1.0 / 15.0, dtype=torch.float32))).float().half().double()
    base = low.half().double()
    inverse = torch.where(step > 0, (1.0 / step).float().double(), 0.0)
    code = ((x - base).float().double() * inverse).float().round().clamp(0, 15).double()
    return (code * step + base).flatten(-2)


def _exact_prefix(case, seed):
    state = prepare(case, seed)
    q = state["query"].double()
    nq, q_len, H, D = case["nq"], case["q_len"], case["H"], case["D"]
    group, shared = _groups(case)
    tails = _tails(case)
    before = [[_stored64(x) for x in _made(case, seed, (0, x), PAGE * n)] for x, n in enumerate(shared)]
    out = torch.zeros(q.shape, dtype=torch.float64, device="cuda")
    for b in range(case["B"]):
        k, v = (_stored64(x) for x in _made(case, seed, (1, b), tails[b]))
        if group[b] >= 0:
            k, v = torch.cat([before[group[b]][0], k], 1), torch.cat([before[group[b]][1], v], 1)
        heads = q[b].reshape(H, nq // H * q_len, D)
        logits = (heads @ k.transpose(1, 2) * state["scaling"]).view(H, nq // H, q_len, -1)
        n = k.shape[1]
        later = torch.arange(n, device="cuda") > torch.arange(n - q_len, n, device="cuda").view(-1, 1)
        p = torch.softmax(logits.masked_fill(later, -float("inf")), -1)
        out[b] = (p.flatten(1, 2) @ v).reshape(nq, q_len, D)
    return out


def exact(case, seed):
    return {"rotary": _exact_rotary, "prompt": _exact_prompt, "prefix": _exact_prefix}[case["op"]](case, seed)
