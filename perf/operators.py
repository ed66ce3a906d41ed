"""Cases of the 4-bit paged cache's operators, their plain forms and their definition in 64 bits.

Three operators work on one pool of 4-bit pages (64 tokens each; scale and minimum in fp16 for every 32 channels of a
token):

* ``quantise``: new tokens are quantised into the pages and read back (and the pages' channel bounds with them);
* ``attend``: attention of new query tokens over the pages (grouped heads, causal among the new tokens);
* ``sparse``: the same over the pages that a bound on the scores selects for each query token and KV head.

The geometries are those the repository measures: 28 query heads on 4 KV heads and 40 on 8, head_dim 128, histories of
1k, 8k, 16k and 32k tokens, prompts of 4096; head_dim 64 and fp16 stand for smaller models.
"""
import torch

own = False

PAGE = 64      # tokens of a page
GROUP = 32     # channels that share a scale and a minimum
TYPES = {"bf16": torch.bfloat16, "f16": torch.float16}


def listed():
    b = dict(dtype="bf16", D=128, q_len=1)
    return [
        # One decoded token of each of 16 sequences at 8k tokens: the smallest write, where latency counts.
        dict(name="quantise one token", op="quantise", B=16, H=4, T=1, start=8192, spread=0, bounds=False, dtype="bf16", D=128),
        # A 4096-token prompt of 16 sequences: the largest write; every page completes and gets its bounds.
        dict(name="quantise prompts", op="quantise", B=16, H=4, T=4096, start=0, spread=0, bounds=True, dtype="bf16", D=128),
        # A chunk that starts inside a page and ends inside another, at another place in each sequence.
        dict(name="quantise ragged chunks", op="quantise", B=5, H=8, T=777, start=1300, spread=517, bounds=True, dtype="f16", D=64),
        # One sequence of about a thousand tokens: a short chat, one step.
        dict(b, name="attend one sequence", op="attend", B=1, nq=28, H=4, length=1061, spread=0),
        # A serving batch at 8k tokens, histories that end anywhere inside a page.
        dict(b, name="attend 16 x 8k", op="attend", B=16, nq=28, H=4, length=8319, spread=127),
        # Long context: the largest dense step.
        dict(b, name="attend 8 x 32k", op="attend", B=8, nq=28, H=4, length=32895, spread=127),
        # Five drafted tokens a sequence to verify at once, very unequal histories, small heads in fp16.
        dict(name="attend drafts", op="attend", B=6, nq=40, H=8, length=9001, spread=8990, dtype="f16", D=64, q_len=5),
        # One long conversation, 64 of its 515 pages read.
        dict(b, name="sparse one sequence", op="sparse", B=1, nq=28, H=4, length=32901, spread=0, top=61, sink=1, recent=2),
        # A large serving batch at 16k tokens, 32 of 256 pages read by each KV head.
        dict(b, name="sparse 64 x 16k", op="sparse", B=64, nq=40, H=8, length=16384, spread=0, top=29, sink=1, recent=2),
        # A document of 128k tokens asked by two users.
        dict(b, name="sparse 2 x 128k", op="sparse", B=2, nq=28, H=4, length=131072, spread=1000, top=125, sink=1, recent=2),
        # Unequal short histories (some shorter than the budget, so all is read), one head per KV head, fp16, 3 drafted tokens.
        dict(name="sparse ragged", op="sparse", B=7, nq=8, H=8, length=5003, spread=4990, dtype="f16", D=64, q_len=3, top=13,
             sink=2, recent=1),
    ]


def _spread(rng, low, high):
    return int(round(low * (high / low) ** rng.random()))


def draw(rng):
    case = dict(op=rng.choice(["quantise", "attend", "sparse"]), D=rng.choice([64, 128, 128]), dtype=rng.choice(["bf16", "bf16", "f16"]))
    if case["op"] == "quantise":
        case.update(B=_spread(rng, 1, 24), H=rng.choice([1, 2, 4, 8]), T=_spread(rng, 1, 4096), start=_spread(rng, 1, 3000) - 1,
                    bounds=rng.random() < 0.7)
        case["spread"] = rng.randrange(min(case["start"] + 1, 600))
        while case["B"] * case["H"] * (case["T"] + case["start"]) > 260000:
            case["T"] = max(1, case["T"] // 2)
            case["B"] = max(1, case["B"] * 2 // 3)
        return case
    case["nq"], case["H"] = rng.choice([(28, 4), (40, 8), (8, 8), (16, 1), (14, 2), (32, 8)])
    case.update(B=_spread(rng, 1, 32), q_len=rng.choice([1, 1, 1, 2, 3, 6]), length=_spread(rng, 1, 33000))
    while case["B"] * case["H"] * case["length"] * case["q_len"] > 1000000:
        case["B"] = max(1, case["B"] * 2 // 3)
        if case["B"] == 1:
            case["q_len"] = 1
            break
    case["spread"] = rng.randrange(case["length"] + 1) if rng.random() < 0.6 else 0
    if case["op"] == "sparse":
        case.update(top=_spread(rng, 1, 100), sink=rng.choice([0, 1, 2]), recent=rng.choice([1, 2, 4]))
    return case


def _lengths(case, top, spread):
    """Another length for each sequence, the longest first: top, ..., at least top - spread."""
    return [top - (b * 7919) % (spread + 1) for b in range(case["B"])]


def _spans(case):
    """quantise: the first position of each sequence's new tokens."""
    return _lengths(case, case["start"], case["spread"])


# ---------------------------------------------------------------- inputs

def _groups(x):
    return x.unflatten(-1, (-1, GROUP))


def _quantise(x):
    """Codes, scales and minima of [..., D] fp32 values, for every GROUP channels."""
    x = _groups(x)
    lo, hi = x.amin(-1, keepdim=True), x.amax(-1, keepdim=True)
    s, z = ((hi - lo) * (1.0 / 15.0)).half(), lo.half()
    bad = ~(torch.isfinite(s) & torch.isfinite(z))
    s32 = s.float()
    r = torch.where(s32 > 0, torch.ones_like(s32) / s32, torch.zeros_like(s32))
    c = torch.round((x - z.float()) * r).clamp(0, 15)
    nan = torch.full_like(s, float("nan"))
    return torch.where(bad, torch.zeros_like(c), c), torch.where(bad, nan, s), torch.where(bad, nan, z)


def _values(c, s, z):
    return (c * s.float() + z.float()).flatten(-2)


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


def _page_bounds(values):
    """int8 records [..., 2 D + 16] of fp32 Key values [..., PAGE, D]: upper, lower, exponent."""
    v = torch.where(torch.isfinite(values), values, torch.zeros_like(values))
    up, low = v.amax(-2), v.amin(-2)
    e = _exponent(torch.maximum(up.amax(-1, keepdim=True), -low.amin(-1, keepdim=True)))
    step = torch.ldexp(torch.ones_like(up[..., :1]), -e)
    out = torch.zeros(*up.shape[:-1], 2 * up.shape[-1] + 16, dtype=torch.int8, device=values.device)
    out[..., :up.shape[-1]] = torch.ceil(up * step).to(torch.int8)
    out[..., up.shape[-1]:2 * up.shape[-1]] = torch.floor(low * step).to(torch.int8)
    out[..., 2 * up.shape[-1]:2 * up.shape[-1] + 1] = e.to(torch.int8)
    return out


def _exponent(most):
    """The smallest e >= -40 with most <= 127 * 2^e."""
    f, x = torch.frexp(most)
    e = torch.where(f <= 127.0 / 128.0, x - 7, x - 6)
    return torch.where(most > 0, e, torch.full_like(e, -40)).clamp(min=-40).to(torch.int32)


def _made(case, seed, b, tokens):
    """Key and Value [H, tokens, D] of sequence b: normal, a few Key channels of each head ten times larger, and a slow
    drift along the sequence, so that some pages matter more than others."""
    g = torch.Generator(device="cuda")
    g.manual_seed(seed * 1009 + b * 9176 + 11)
    H, D = case["H"], case["D"]
    k = torch.randn(H, tokens, D, generator=g, device="cuda")
    v = torch.randn(H, tokens, D, generator=g, device="cuda")
    k[:, :, :: D // 6] *= 4.0
    drift = torch.randn(H, tokens // 256 + 2, D, generator=g, device="cuda")
    k += drift.repeat_interleave(256, 1)[:, 100:100 + tokens]
    dt = TYPES[case["dtype"]]
    return k.to(dt), v.to(dt)


def prepare(case, seed):
    B, H, D = case["B"], case["H"], case["D"]
    G = torch.Generator(device="cuda")
    G.manual_seed(seed * 31 + 5)
    quantise = case["op"] == "quantise"
    if quantise:
        held = _spans(case)
        most = max(held) + case["T"]
    else:
        held = _lengths(case, case["length"], case["spread"])
        most = max(held)
    width = -(-most // PAGE)
    # The pool is shared by the sequences: their pages lie in it in no order.
    table = torch.randperm(B * width, generator=G, device="cuda").to(torch.int32).view(B, width)
    pages = torch.zeros(B * width, H, 20 * D, dtype=torch.int32, device="cuda")
    bounds = torch.zeros(B * width, H, 2 * D + 16, dtype=torch.int8, device="cuda")
    state = dict(case=case, pages=pages, bounds=bounds, table=table)
    if quantise:
        state["key"] = torch.empty(B, H, case["T"], D, dtype=TYPES[case["dtype"]], device="cuda")
        state["value"] = torch.empty_like(state["key"])
        state["start"] = torch.tensor(held, dtype=torch.int32, device="cuda")
    else:
        state["lengths"] = torch.tensor(held, dtype=torch.int32, device="cuda")
        q = torch.randn(B, case["nq"], case["q_len"], D, generator=G, device="cuda")
        state["query"] = q.to(TYPES[case["dtype"]])
        state["scaling"] = D ** -0.5
    for b in range(B):
        k, v = _made(case, seed, b, most)
        if quantise:
            state["key"][b] = k[:, held[b]:held[b] + case["T"]]
            state["value"][b] = v[:, held[b]:held[b] + case["T"]]
        k, v = k.float(), v.float()
        k[:, held[b]:] = 0
        v[:, held[b]:] = 0
        pad = width * PAGE - most
        k, v = (torch.nn.functional.pad(x, (0, 0, 0, pad)) for x in (k, v))
        rows = table[b].long()
        pages[rows] = _records(k, v).transpose(0, 1)
        full = held[b] // PAGE
        if full and (case["op"] == "sparse" or case.get("bounds")):
            kv = _values(*_quantise(k[:, :full * PAGE])).view(H, full, PAGE, D)
            bounds[rows[:full]] = _page_bounds(kv).transpose(0, 1)
    return state


# ---------------------------------------------------------------- the plain forms

def _nibbles(words):
    shift = torch.arange(8, device=words.device, dtype=torch.int32) * 4
    return ((words.unsqueeze(-1) >> shift) & 15).float()


def _unpacked(rec, key_only=False):
    """fp32 Key (and Value) [..., PAGE, D] of records [..., 20 D]."""
    D = rec.shape[-1] // 20
    G, lead = D // GROUP, rec.shape[:-1]
    d = len(lead)
    kc, kp, vc, vp = rec.split([8 * D, 2 * D, 8 * D, 2 * D], -1)
    c = _nibbles(kc.reshape(*lead, PAGE, 4, G)).transpose(-2, -3).flatten(-2)
    p = kp.contiguous().view(torch.float16).reshape(*lead, PAGE, G, 2)
    key = _values(c, p[..., :1], p[..., 1:])
    if key_only:
        return key
    c = _nibbles(vc.reshape(*lead, 8, 8, 4, 2, G // 2)).unflatten(-1, (2, 4))         # b g t o w u n
    c = c.permute(*range(d), d, d + 2, d + 3, d + 4, d + 5, d + 1, d + 6)
    p = vp.contiguous().view(torch.float16).reshape(*lead, PAGE, G, 2)
    return key, _values(c.reshape(*lead, PAGE, G, GROUP), p[..., :1], p[..., 1:])


def _plain_quantise(state):
    case = state["case"]
    key, value = (_values(*_quantise(x.float())) for x in (state["key"], state["value"]))
    out = [key.to(state["key"].dtype), value.to(state["key"].dtype)]
    if case["bounds"]:
        B, H, T, D = key.shape
        rows = state["table"].long()
        known = _unpacked(state["pages"][rows], key_only=True).permute(0, 2, 1, 3, 4).flatten(2, 3)    # [B, H, tokens, D]
        at = torch.arange(known.shape[2], device="cuda") - state["start"].view(-1, 1)                  # [B, tokens]
        new = ((at >= 0) & (at < T)).view(B, 1, -1, 1)
        moved = key.gather(2, at.clamp(0, T - 1).view(B, 1, -1, 1).expand(-1, H, -1, D))
        known = torch.where(new, moved, known).unflatten(2, (-1, PAGE))
        made = _page_bounds(known).transpose(1, 2)                                                     # [B, W, H, 2 D + 16]
        full = torch.arange(rows.shape[1], device="cuda") < ((state["start"] + T) // PAGE).view(-1, 1)
        every = torch.zeros_like(state["bounds"])
        every[rows] = torch.where(full.view(B, -1, 1, 1), made, torch.zeros_like(made))
        step = torch.ldexp(torch.ones_like(every[..., :1], dtype=torch.float32), every[..., 2 * D:2 * D + 1].to(torch.int32))
        out.append(every[..., :2 * D].float().mul(step).unflatten(-1, (2, D)))
    return out


def _visible(state):
    q_len = state["query"].shape[2]
    i = torch.arange(q_len, device="cuda")
    return (state["lengths"].view(-1, 1) - q_len + i + 1).clamp(min=0)                                  # [B, q_len]


def _softmax(logits, seen):
    logits = logits.masked_fill(~seen, -float("inf"))
    most = logits.amax(-1, keepdim=True)
    p = torch.exp(logits - torch.where(most == -float("inf"), torch.zeros_like(most), most))
    total = p.sum(-1, keepdim=True)
    return p / torch.where(total == 0, torch.ones_like(total), total)


def _plain_attend(state):
    q, case = state["query"], state["case"]
    B, nq, q_len, D = q.shape
    H = case["H"]
    k, v = _unpacked(state["pages"][state["table"].long()])
    k, v = (x.permute(0, 2, 1, 3, 4).flatten(2, 3) for x in (k, v))                                     # [B, H, tokens, D]
    q32 = q.float().view(B, H, nq // H, q_len, D).flatten(2, 3)
    logits = (q32 @ k.transpose(-1, -2)).view(B, H, nq // H, q_len, -1) * state["scaling"]
    seen = torch.arange(k.shape[2], device="cuda") < _visible(state).view(B, 1, 1, q_len, 1)
    p = _softmax(logits, seen)
    return (p.flatten(2, 3) @ v).view(B, nq, q_len, D).to(q.dtype)


def _plain_sparse(state):
    q, case = state["query"], state["case"]
    B, nq, q_len, D = q.shape
    H, sink, recent, top = case["H"], case["sink"], case["recent"], case["top"]
    rows, slots = state["table"].long(), sink + recent + top
    q32 = q.float().view(B, H, nq // H, q_len, D).permute(0, 3, 1, 2, 4)                                # [B, q_len, H, heads, D]
    # Each page's score for each query token and KV head.
    safe = torch.where(torch.isfinite(q32), q32, torch.zeros_like(q32))
    eq = _exponent(safe.abs().amax((-1, -2), keepdim=True))
    qi = torch.round(torch.ldexp(safe, -eq))
    plus, minus = qi.clamp(min=0).sum(-2), qi.clamp(max=0).sum(-2)
    rec = state["bounds"][rows].transpose(1, 2)                                                         # [B, H, W, 2 D + 16]
    both = torch.cat([plus, minus], -1).to(torch.int32)                                                 # [B, q_len, H, 2 D]
    total = (both.unsqueeze(-2) * rec[..., :2 * D].unsqueeze(1).to(torch.int32)).sum(-1)                 # [B, q_len, H, W]
    score = torch.ldexp(total.float(), rec[..., 2 * D].to(torch.int32).unsqueeze(1))
    seen = _visible(state)
    n = ((seen + PAGE - 1) // PAGE).view(B, q_len, 1, 1)
    page = torch.arange(rows.shape[1], device="cuda")
    always = ((page < sink) | (page >= n - recent)) & (page < n)
    inf = torch.full_like(score, float("inf"))
    score = torch.where(always, inf, torch.where(page < n, score, -inf))
    order = score.sort(stable=True, dim=-1, descending=True).indices[..., :slots]
    # The pages chosen, in ascending order, -1 after the last.
    W = rows.shape[1]
    kept = torch.where(torch.arange(order.shape[-1], device="cuda") < n, order, torch.full_like(order, W)).sort(-1).values
    picked = torch.where(kept == W, torch.full_like(kept, -1), kept)
    picked = torch.nn.functional.pad(picked, (0, slots - picked.shape[-1]), value=-1)
    # Attention over their tokens.
    phys = rows.view(B, 1, 1, W).expand(-1, q_len, H, -1).gather(-1, picked.clamp(min=0))               # [B, q_len, H, slots]
    k, v = _unpacked(state["pages"][phys, torch.arange(H, device="cuda").view(1, 1, H, 1)])
    token = (picked.unsqueeze(-1) * PAGE + torch.arange(PAGE, device="cuda")).flatten(-2)               # [B, q_len, H, slots PAGE]
    live = (picked.unsqueeze(-1) >= 0).expand(-1, -1, -1, -1, PAGE).flatten(-2) & (token < seen.view(B, q_len, 1, 1))
    logits = (q32 @ k.flatten(-3, -2).transpose(-1, -2)) * state["scaling"]
    p = _softmax(logits, live.unsqueeze(-2))
    out = (p @ v.flatten(-3, -2)).permute(0, 2, 3, 1, 4).reshape(B, nq, q_len, D)
    return out.to(q.dtype), picked.to(torch.int32)


def run(state):
    case = state["case"]
    if not own:
        return {"quantise": _plain_quantise, "attend": _plain_attend, "sparse": _plain_sparse}[case["op"]](state)
    from logitfill_b200 import int4

    if case["op"] == "quantise":
        bounds = state["bounds"] if case["bounds"] else None
        int4.int4_write(state["key"], state["value"], state["pages"], state["table"], state["start"], bounds=bounds)
        out = list(int4.int4_read(state["pages"], state["table"], state["start"], case["T"], dtype=state["key"].dtype))
        if case["bounds"]:
            out.append(int4.int4_read_bounds(bounds))
        return out
    if case["op"] == "attend":
        return int4.int4_attention(state["query"], state["pages"], state["table"], state["lengths"], state["scaling"])
    return int4.int4_sparse_attention(state["query"], state["pages"], state["bounds"], state["table"], state["lengths"],
                                      state["scaling"], top_pages=case["top"], sink_pages=case["sink"],
                                      recent_pages=case["recent"])


# ---------------------------------------------------------------- what a pass cannot do without

def work(case):
    B, H, D = case["B"], case["H"], case["D"]
    token = D + D // 4                                   # bytes of a token and KV head in the pages
    if case["op"] == "quantise":
        n = B * H * case["T"]
        total = n * (4 * D + token + 4 * D)
        if case["bounds"]:
            done = sum((s + case["T"]) // PAGE - s // PAGE for s in _spans(case))
            held = sum((s + case["T"]) // PAGE for s in _spans(case))
            total += H * (done * (2 * D + 1) + held * 8 * D)
        return {"bytes": total, "flops": n * 2 * D * 5}
    q_len, nq = case["q_len"], case["nq"]
    total, flops = 2 * 2 * B * nq * q_len * D, 0
    for length in _lengths(case, case["length"], case["spread"]):
        if case["op"] == "attend":
            total += H * length * token
            flops += sum(4 * nq * D * max(0, length - i) for i in range(q_len))
            continue
        for i in range(q_len):
            seen = max(0, length - i)
            n = -(-seen // PAGE)
            rest = max(0, n - case["sink"] - case["recent"])
            read = min(seen, (case["sink"] + case["recent"] + case["top"]) * PAGE)
            flops += 4 * nq * D * read + 2 * H * rest * 2 * D
            if i == 0:                                   # later tokens of the sequence may read the same pages
                total += H * (rest * (2 * D + 1) + read * token)
        total += 4 * q_len * H * (case["sink"] + case["recent"] + case["top"])
    return {"bytes": total, "flops": flops}


# ---------------------------------------------------------------- the definition in 64 bits

def _power(most):
    """The smallest power of two p >= 2^-40 with most <= 127 p, for most > 0."""
    e = torch.log2(most / 127.0).round().to(torch.int32) - 2
    p = torch.ldexp(torch.ones_like(most), e)
    for _ in range(4):
        p = torch.where(most > 127.0 * p, 2 * p, p)
    return p.clamp(min=2.0 ** -40)


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


def exact(case, seed):
    B, H, D = case["B"], case["H"], case["D"]
    if case["op"] == "quantise":
        at = _spans(case)
        most = max(at) + case["T"]
        rows = prepare(dict(case, B=B), seed)["table"].long() if case["bounds"] else None
        keys, values, table = [], [], None
        if case["bounds"]:
            table = torch.zeros(rows.numel(), H, 2, D, dtype=torch.float64, device="cuda")
        for b in range(B):
            k, v = _made(case, seed, b, most)
            k, v = _stored64(k), _stored64(v)
            keys.append(k[:, at[b]:at[b] + case["T"]])
            values.append(v[:, at[b]:at[b] + case["T"]])
            for p in range((at[b] + case["T"]) // PAGE if case["bounds"] else 0):
                # the cache holds fp32(code * step + minimum)
                part = k[:, p * PAGE:(p + 1) * PAGE].float().double()
                unit = _power(part.abs().amax((1, 2)).clamp(min=1e-30)).view(H, 1)
                table[rows[b, p], :, 0] = torch.ceil(part.amax(1) / unit) * unit
                table[rows[b, p], :, 1] = torch.floor(part.amin(1) / unit) * unit
        out = [torch.stack(keys), torch.stack(values)]
        return out + [table] if case["bounds"] else out
    state = prepare(case, seed)
    q = state["query"].double()
    nq, q_len = case["nq"], case["q_len"]
    group = nq // H
    lengths = _lengths(case, case["length"], case["spread"])
    out = torch.zeros(B, nq, q_len, D, dtype=torch.float64, device="cuda")
    sparse = case["op"] == "sparse"
    slots = case["sink"] + case["recent"] + case["top"] if sparse else 0
    for b in range(B):
        k, v = _made(case, seed, b, max(lengths))
        k, v = _stored64(k), _stored64(v)
        if sparse:
            whole = lengths[b] // PAGE
            held = k[:, :whole * PAGE].float().double().reshape(H, whole, PAGE, D)
            up, low = held.amax(2), held.amin(2)
            unit = _power(torch.maximum(up.abs(), low.abs()).amax(-1, keepdim=True).clamp(min=1e-30))
            up, low = torch.ceil(up / unit) * unit, torch.floor(low / unit) * unit
        for i in range(q_len):
            seen = lengths[b] - q_len + i + 1
            if seen <= 0:
                continue
            heads = q[b, :, i].reshape(H, group, D)
            logits = (heads @ k[:, :seen].transpose(1, 2)) * state["scaling"]
            n = -(-seen // PAGE)
            if sparse and n > slots:
                whole_q = torch.round(heads / _power(heads.abs().amax((1, 2), keepdim=True)))
                first, last = case["sink"], n - case["recent"]
                bound = torch.maximum(whole_q.unsqueeze(2) * up[:, None, first:last], whole_q.unsqueeze(2) * low[:, None, first:last])
                bound = bound.sum((1, 3)).float()                                                       # [H, candidates]
                mask = torch.full((H, n), False, device="cuda")
                mask[:, :first] = True
                mask[:, last:] = True
                chosen = bound.sort(stable=True, dim=-1, descending=True).indices[:, :case["top"]] + first
                mask.scatter_(1, chosen, True)
                hide = ~mask.repeat_interleave(PAGE, 1)[:, :seen]
                logits = logits.masked_fill(hide.unsqueeze(1), -float("inf"))
            p = torch.softmax(logits, -1)
            out[b, :, i] = (p @ v[:, :seen]).reshape(nq, D)
    return (out, None) if sparse else out
