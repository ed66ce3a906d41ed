"""CPU tests of a prompt's operators and of shared prefixes: refusals before any
launch, the frequency tables, the cache's bookkeeping of shared pages."""
from __future__ import annotations

import math
import re
import struct
import time
from pathlib import Path

import numpy as np
import pytest
import torch

from logitfill_b200 import _lib, int4, prompt
from logitfill_b200.adapter import DeepSeekQwenKVAdapter
from logitfill_b200.packed import PackedKVCache
from tests.qwen_cases import tiny_qwen2
from tests.test_int4_cpu import QUERY, _query

HEADER = (Path(__file__).resolve().parents[1] / "include" / "logitfill_b200.h").read_text()
INVALID, UNSUPPORTED, OK = _lib.LF_ERR_INVALID_ARGUMENT, _lib.LF_ERR_UNSUPPORTED, _lib.LF_OK
FAKE = 1 << 20   # never dereferenced: validation fails first

ROTARY = struct.Struct("@4P12qPP2qPf10i0q")
PROMPT = struct.Struct("@4P12q3Pf6i0q")


def _fields(name):
    body = re.search(r"typedef struct %s \{(.*?)\} %s;" % (name, name), HEADER, re.S).group(1)
    body = re.sub(r"/\*.*?\*/", "", body, flags=re.S)
    out = []
    for decl in filter(None, (d.strip() for d in body.split(";"))):
        kind, names = re.match(r"(?:const )?([\w]+\s*\*?)\s*(.*)", decl, re.S).groups()
        out += [(kind.replace(" ", ""), n.strip()) for n in names.split(",")]
    return out


@pytest.mark.parametrize("name,packed", [("lf_rotary", ROTARY), ("lf_prompt", PROMPT)])
def test_packed_structs_follow_the_header(name, packed):
    code = {"void*": "P", "int32_t*": "P", "int64_t*": "P", "int64_t": "q", "int32_t": "i", "float": "f"}
    spelled = re.sub(r"(\d+)([a-zA-Z])", lambda m: int(m.group(1)) * m.group(2), packed.format.lstrip("@"))
    assert spelled == "".join(code[k] for k, _ in _fields(name))


def _rotary(**over):
    f = dict(q=FAKE, q_out=FAKE, k=FAKE, k_out=FAKE, strides=(512, 64, 1024) * 4, freqs=FAKE, positions=FAKE, ps=0, pt=1, start=0,
             magnitude=1.0, p64=1, dtype=_lib.LF_BF16, head_dim=64, part=64, interleaved=0, transposed=0, batch=1, tokens=4, n_q=8, n_kv=2)
    f.update(over)
    flat = []
    for v in f.values():
        flat += list(v) if isinstance(v, tuple) else [v]
    return ROTARY.pack(*flat)


def _prompt(**over):
    f = dict(q=FAKE, k=FAKE, v=FAKE, out=FAKE, strides=(0, 64, 512, 0, 64, 128, 0, 64, 128, 0, 64, 512), starts=FAKE, counts=0, status=0,
             scaling=0.125, head_dim=64, dtype=_lib.LF_BF16, batch=2, tokens=9, n_q=8, n_kv=2)
    f.update(over)
    flat = []
    for v in f.values():
        flat += list(v) if isinstance(v, tuple) else [v]
    return PROMPT.pack(*flat)


def test_rotary_validates_before_launch():
    f = _lib.lib().lf_rotary_embed
    assert f(None, None) == INVALID
    assert f(_rotary(tokens=0), None) == OK and f(_rotary(batch=0), None) == OK and f(_rotary(n_q=0, n_kv=0), None) == OK
    for bad in (dict(q=0), dict(q_out=0), dict(k=0), dict(freqs=0), dict(positions=0), dict(part=0), dict(part=63), dict(part=66),
                dict(tokens=-1), dict(n_q=-1), dict(dtype=5), dict(magnitude=math.nan), dict(magnitude=math.inf)):
        assert f(_rotary(**bad), None) == INVALID, bad
    for much in (dict(head_dim=258), dict(head_dim=0, part=2), dict(n_q=70000), dict(batch=1 << 30, tokens=1 << 30)):
        assert f(_rotary(**much), None) == UNSUPPORTED, much


def test_prompt_attention_validates_before_launch():
    f = _lib.lib().lf_prompt_attend
    assert f(None, None) == INVALID
    assert f(_prompt(tokens=0), None) == OK and f(_prompt(batch=0), None) == OK
    for bad in (dict(q=0), dict(out=0), dict(q=FAKE + 8), dict(n_q=7), dict(n_kv=0), dict(tokens=-1), dict(scaling=math.inf),
                dict(scaling=3.2e38), dict(strides=(0, 60, 512, 0, 64, 128, 0, 64, 128, 0, 64, 512)),
                dict(strides=(0, 64, 512, 0, 64, 0, 0, 64, 128, 0, 64, 512)), dict(strides=(0, 64, -512, 0, 64, 128, 0, 64, 128, 0, 64, 512)),
                dict(starts=0)):   # (a padded batch without a sequence stride)
        assert f(_prompt(**bad), None) == INVALID, bad
    for much in (dict(head_dim=96), dict(dtype=_lib.LF_F32), dict(n_q=258), dict(n_q=65536, n_kv=65536)):
        assert f(_prompt(**much), None) == UNSUPPORTED, much
    assert b"lf_prompt_attend" in _lib.lib().lf_last_error()


def _prefix(query=None, **over):
    f = dict(group=FAKE, shared=FAKE, ws=FAKE, ws_bytes=1 << 40, groups=2, always=1)
    f.update(over)
    return _query(**dict(dict(picked=0), **(query or {}))) + struct.pack("@PPPNii0q", *f.values())


def test_prefix_attention_validates_before_launch():
    assert QUERY.size % 8 == 0
    f = _lib.lib().lf_int4_attend_prefix
    assert f(None, None) == INVALID
    for bad in (dict(group=0), dict(shared=0), dict(groups=-1)):
        assert f(_prefix(**bad), None) in (INVALID, _lib.LF_ERR_CUDA), bad     # (without a GPU its SMs cannot be counted)
    for bad in (dict(q=0), dict(picked=FAKE), dict(n_q=9), dict(out=0), dict(lengths=0), dict(pages=FAKE + 4)):
        assert f(_prefix(bad), None) == INVALID, bad
    assert f(_prefix(dict(head_dim=96)), None) == UNSUPPORTED
    so = _lib.lib()
    assert so.lf_int4_prefix_workspace_bytes(0, 8, 40, 1, 128, 1) == 0 == so.lf_int4_prefix_workspace_bytes(1, 8, 7, 1, 128, 1)
    record = 256 * (128 + 2) * 4
    few, many = (so.lf_int4_prefix_workspace_bytes(64, 8, 40, q, 128, 1) for q in (1, 256))
    # 64 sequences' rows (5 heads on a KV head) of 255 query tokens more, in records of 256
    assert many - few == 8 * (64 * 5 * 256 // 256 - 64 * 5 // 256) * record


def _need(batch=64, kv_heads=8, n_q=40, q_len=1, head_dim=128, dtype=None, width=1000, groups=64, always=0):
    query = dict(q_len=q_len, n_q=n_q, head_dim=head_dim, dtype=_lib.LF_BF16 if dtype is None else dtype)
    pool = dict(batch=batch, kv_heads=kv_heads, table_width=width)
    return _lib.lib().lf_int4_prefix_workspace_need(_prefix(dict(query, **pool), groups=groups, always=always))


def test_prefix_attention_asks_for_no_more_workspace_than_groups_may_use():
    so = _lib.lib()
    record = 256 * (128 + 2) * 4
    any_call = so.lf_int4_prefix_workspace_bytes(1024, 8, 40, 1, 128, 1024)
    assert any_call < 0.6e9                                   # pairs of sequences, at most
    assert _need(batch=1024, groups=1024) < 0.26e9            # five sequences read a page once sooner than each for itself
    assert _need(batch=64, groups=64) < 15e6
    assert _need(batch=64, groups=64) >= (64 * 5 // 256 + 12) * 8 * record
    for none in (dict(width=3, batch=4), dict(batch=4, groups=4), dict(groups=0), dict(groups=4097), dict(q_len=0), dict(n_q=7)):
        assert _need(**none) == 0, none
    assert _need(batch=4, groups=4, always=1) > 0 and _need(batch=1, groups=1, q_len=512, n_q=28, kv_heads=4) > 0
    assert so.lf_int4_prefix_workspace_need(None) == 0


@pytest.mark.parametrize("seed", range(4))
def test_no_groups_fill_more_units_than_a_call_has_room_for(seed):
    """The plan's rule (which groups read their pages once, and how many units of 256 rows that makes), over random
    groups, lengths and shapes, against the room that a call asks for."""
    rng = np.random.default_rng(seed)
    tried = 0
    for _ in range(400):
        D, fp16, always = int(rng.choice([64, 128])), bool(rng.integers(2)), bool(rng.integers(2))
        kv_heads, heads, q_len = int(rng.choice([1, 2, 8])), int(rng.choice([1, 2, 5, 7, 16, 40])), int(rng.choice([1, 1, 2, 3, 9, 64]))
        batch = int(rng.integers(1, 200))
        groups = int(rng.integers(1, 200))
        width = int(rng.choice([1, 7, 100, 1000, 5000]))
        columns = heads * q_len
        visit = lambda pages: pages * ((columns + 15) // 16) * (20 if columns <= 8 else 29) * D // 1280  # noqa: E731
        tile = {(128, False): 16, (128, True): 23, (64, False): 11, (64, True): 16}[D, fp16]
        fewest = rng.integers(1, 12)
        count = np.bincount(rng.integers(0, max(1, min(groups, batch // fewest)), batch), minlength=groups)
        units = 0
        for c in count:
            if c == 0 or (c == 1 and columns <= 16):
                continue
            pages = width if rng.random() < 0.7 else int(rng.integers(0, width + 1))
            tiles = -(-int(c) * columns // 256) if pages else 0
            places = tiles * kv_heads * ((pages + 1) // 2 + 2)
            if pages and (always or visit(pages * int(c) * kv_heads) - places * tile > 0):
                units += tiles * kv_heads
        need = _need(batch, kv_heads, kv_heads * heads, q_len, D, _lib.LF_F16 if fp16 else _lib.LF_BF16, width, groups, int(always))
        small = visit(batch * kv_heads * width) <= (17000 if D == 128 else 12500) and not always
        if small:
            assert need == 0
            continue
        lists = (16 + 32 * groups + 12 * batch + 255) // 256 * 256
        record = 256 * (D + 2) * 4
        room = (need - lists) // record if need else 0      # (no SMs here: the records of units alone)
        assert room >= units, (D, fp16, always, kv_heads, heads, q_len, batch, groups, width)
        assert need <= _lib.lib().lf_int4_prefix_workspace_bytes(batch, kv_heads, kv_heads * heads, q_len, D, groups)
        tried += units > 0
    assert tried > 50


# ------------------------------------------------------------ frequencies

def _radians(freqs):
    return [f / 2.0 ** 64 * 2 * math.pi for f in freqs.tolist()]


@pytest.mark.parametrize("part,base", [(128, 10000.0), (64, 1e6), (2, 5e5), (34, 10000.0)])
def test_frequencies_without_scaling(part, base):
    freqs, magnitude = prompt.rotary_frequencies(part, base, device="cpu")
    assert freqs.dtype == torch.int64 and magnitude == 1.0
    for i, got in enumerate(_radians(freqs)):
        want = base ** (-2 * i / part)
        assert abs(got - want) <= 2.0 ** -50 * want + 2.0 ** -61   # fp64, then steps of 2^-64 turns
    linear, magnitude = prompt.rotary_frequencies(part, base, dict(type="linear", factor=4.0), device="cpu")
    assert magnitude == 1.0
    assert all(abs(4 * a - b) <= 2.0 ** -60 for a, b in zip(_radians(linear), _radians(freqs)))


def test_frequencies_stretched_in_part():
    """Peng et al.: pairs that turn often keep their frequency, slow ones are divided, a ramp between."""
    scaling = dict(rope_type="yarn", factor=8.0, original_max_position_embeddings=4096)
    plain = _radians(prompt.rotary_frequencies(128, device="cpu")[0])
    freqs, magnitude = prompt.rotary_frequencies(128, scaling=scaling, device="cpu")
    got = _radians(freqs)
    assert magnitude == pytest.approx(0.1 * math.log(8.0) + 1.0)
    turns = [4096 * f / (2 * math.pi) for f in plain]
    for i, (g, f, t) in enumerate(zip(got, plain, turns)):
        assert f / 8 * (1 - 1e-12) <= g <= f * (1 + 1e-12)
        if t > 40:
            assert g == pytest.approx(f, rel=1e-12), i
        if t < 0.8:
            assert g == pytest.approx(f / 8, rel=1e-12), i
    assert all(a > b for a, b in zip(got, got[1:]))
    again, m = prompt.rotary_frequencies(128, scaling=dict(scaling, attention_factor=1.5), device="cpu")
    assert m == 1.5 and torch.equal(again, freqs)


def test_frequencies_match_the_installed_transformers():
    from transformers import Qwen2Config
    from transformers.modeling_rope_utils import ROPE_INIT_FUNCTIONS

    rope = dict(rope_type="yarn", factor=4.0, original_max_position_embeddings=32768, rope_theta=1e6)
    config = Qwen2Config(hidden_size=512, num_attention_heads=4, max_position_embeddings=131072, rope_theta=1e6, rope_parameters=rope)
    want, factor = ROPE_INIT_FUNCTIONS["yarn"](config, torch.device("cpu"))
    got, magnitude = prompt.rotary_frequencies(128, 1e6, rope, device="cpu")
    assert magnitude == pytest.approx(factor)
    # its table is fp32: a power and a product, a few roundings of 2^-24
    assert np.allclose(_radians(got), want.double().numpy(), rtol=2.0 ** -20, atol=0)


def test_frequency_refusals():
    for bad in (0, 3, -2):
        with pytest.raises(ValueError):
            prompt.rotary_frequencies(bad, device="cpu")
    for bad in (0.0, -1.0, math.inf):
        with pytest.raises(ValueError):
            prompt.rotary_frequencies(64, bad, device="cpu")
    yarn = dict(rope_type="yarn", factor=2.0, original_max_position_embeddings=4096)
    for error, scaling in [(NotImplementedError, dict(rope_type="dynamic", factor=2.0)), (ValueError, dict(rope_type="linear", factor=0.5)),
                           (KeyError, dict(rope_type="linear")), (NotImplementedError, dict(yarn, mscale=1.0)),
                           (NotImplementedError, dict(yarn, truncate=False)), (ValueError, dict(yarn, original_max_position_embeddings=0))]:
        with pytest.raises(error):
            prompt.rotary_frequencies(64, scaling=scaling, device="cpu")


def test_functions_refuse_cpu_tensors():
    q, k = torch.zeros(4, 8, 64, dtype=torch.bfloat16), torch.zeros(4, 2, 64, dtype=torch.bfloat16)
    freqs, _ = prompt.rotary_frequencies(64, device="cpu")
    with pytest.raises(RuntimeError, match="CUDA"):
        prompt.rotary_embed(q, k, freqs, positions=torch.arange(4))
    with pytest.raises(RuntimeError, match="CUDA"):
        prompt.prompt_attention(q, k, k, 0.125)
    with pytest.raises(TypeError):
        prompt.prompt_attention(q, k, [1], 0.125)
    with pytest.raises(ValueError):
        prompt.prompt_attention(q, k[:3], k[:3], 0.125)
    with pytest.raises(RuntimeError, match="CUDA"):
        n = torch.zeros(1, dtype=torch.int32)
        int4.int4_prefix_attention(q[:1], torch.zeros(4, 2, 1280, dtype=torch.int32), torch.zeros(1, 2, dtype=torch.int32), n, 1.0, n, n)


def test_gradients_are_refused():
    """None of the three records a gradient, of either direction: dropping one silently would be wrong."""
    from torch.autograd import forward_ad

    q, k = torch.zeros(4, 8, 64, dtype=torch.bfloat16), torch.zeros(4, 2, 64, dtype=torch.bfloat16)
    freqs, _ = prompt.rotary_frequencies(64, device="cpu")
    n, table, pages = torch.zeros(4, dtype=torch.int32), torch.zeros(4, 2, dtype=torch.int32), torch.zeros(4, 2, 1280, dtype=torch.int32)
    calls = {
        "rotary query": lambda x: prompt.rotary_embed(x, k, freqs, positions=torch.arange(4)),
        "rotary key": lambda x: prompt.rotary_embed(k, x, freqs, positions=torch.arange(4)),
        "rotary out": lambda x: prompt.rotary_embed(q, None, freqs, positions=torch.arange(4), out=(x, None)),
        "prompt query": lambda x: prompt.prompt_attention(x, k, k, 0.125),
        "prompt key": lambda x: prompt.prompt_attention(q, x, q, 0.125),
        "prompt value": lambda x: prompt.prompt_attention(q, q, x, 0.125),
        "prompt out": lambda x: prompt.prompt_attention(q, k, k, 0.125, out=x),
        "prefix query": lambda x: int4.int4_prefix_attention(x, pages, table, n, 1.0, n, n),
        "prefix out": lambda x: int4.int4_prefix_attention(q, pages, table, n, 1.0, n, n, out=x),
    }
    for name, call in calls.items():
        with pytest.raises(NotImplementedError, match="gradient"):
            call(q.clone().requires_grad_())
        with torch.no_grad(), pytest.raises(RuntimeError, match="CUDA"):
            call(q.clone().requires_grad_())
        with forward_ad.dual_level():
            dual = forward_ad.make_dual(q.clone(), torch.ones_like(q))
            with pytest.raises(NotImplementedError, match="tangent"):
                call(dual)
            with torch.no_grad(), pytest.raises(NotImplementedError, match="tangent"):     # (no_grad does not end this mode)
                call(dual)
        with pytest.raises(RuntimeError, match="CUDA"):
            call(q.clone())


# ------------------------------------------------------------ shared pages in the cache

@pytest.fixture
def cache(monkeypatch):
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: False)
    monkeypatch.setattr(int4.Int4KVCache, "_upload", lambda self, t, host: t.copy_(torch.from_numpy(np.asarray(host).astype(np.int32))))
    return int4.Int4KVCache(1, 4, 4, 2, 64, n_pages=12, max_tokens=400, device="cpu")


def test_sharing_bookkeeping(cache):
    c = cache
    assert c.prefix_group.tolist() == [0, 1, 2, 3] and c.prefix_pages.tolist() == [0, 0, 0, 0]
    c.extend([200, 0, 0, 0])
    assert c.share(0, [2, 3]) == 192 and c.free_pages == 8
    assert c.lengths.tolist() == [200, 0, 192, 192] and c.start.tolist() == [0, 0, 192, 192] and c.counts.tolist() == [200, 0, 0, 0]
    assert torch.equal(c.page_table[2, :3], c.page_table[0, :3]) and (c.page_table[2, 3:] == -1).all()
    assert c.prefix_group.tolist() == [0, 1, 0, 0] and c.prefix_pages.tolist() == [3, 0, 0, 0]
    c.extend([1, 5, 1, 130])
    assert c.free_pages == 8 - 1 - 1 - 3
    rows = [[int(x) for x in row if x >= 0] for row in c.page_table]
    assert len(rows[0]) == 4 and len(rows[2]) == 4 and len(rows[3]) == 6 and len(rows[1]) == 1
    own = rows[0][3:] + rows[1] + rows[2][3:] + rows[3][3:]
    assert len(set(own)) == len(own) and not set(own) & set(rows[0][:3])
    with pytest.raises(ValueError, match="shares"):
        c.truncate([200, 5, 191, 300])
    with pytest.raises(ValueError, match="shares"):
        c.truncate([100, 5, 193, 300])
    c.truncate([192, 5, 192, 300])          # behind the shared pages
    c.release([0])
    assert c.prefix_group.tolist() == [0, 1, 2, 2] and c.prefix_pages.tolist() == [0, 0, 3, 0]
    c.release([2])
    assert c.prefix_group.tolist() == [0, 1, 2, 3] and c.prefix_pages.tolist() == [0, 0, 0, 0]
    c.truncate([0, 5, 0, 10])               # nobody shares these now
    c.release()
    assert c.free_pages == 12 and sorted(c._free) == list(range(12)) and not c._refs.any()


def test_sharing_a_part_and_sharing_on(cache):
    c = cache
    c.extend([300, 0, 0, 0])
    assert c.share(0, [1], tokens=130) == 128
    c.extend([0, 100, 0, 0])
    assert c.share(1, [2]) == 192            # two pages of the first, one of its own
    assert c.prefix_group.tolist() == [0, 0, 0, 3] and c.prefix_pages.tolist() == [2, 0, 0, 0]
    assert c.share(0, [3], tokens=63) == 0 and c.lengths.tolist() == [300, 228, 192, 0]
    for bad in (dict(source=0, seqs=[0]), dict(source=0, seqs=[3, 3]), dict(source=0, seqs=[1]), dict(source=0, seqs=[3], tokens=301),
                dict(source=0, seqs=[3], tokens=-1)):
        with pytest.raises(ValueError):
            c.share(**bad)
    with pytest.raises(IndexError):
        c.share(0, [4])
    c.reserve([0, 0, 0, 64])
    with pytest.raises(ValueError, match="empty"):
        c.share(0, [3])


def test_many_sequences_cost_no_more_than_before_pages_could_be_shared(cache, monkeypatch):
    """truncate() runs at every step of drafts, release() at every end of a sequence: neither walks over the batch in
    Python, and where nothing is shared the groups stay as they were, without a copy to the GPU."""
    many = int4.Int4KVCache(1, 2048, 4, 2, 64, n_pages=2 * 2048, max_tokens=640, device="cpu")
    many.extend(70)
    copied = []
    real = many._upload
    monkeypatch.setattr(many, "_upload", lambda t, host: (copied.append(t), real(t, host)), raising=False)

    def fastest(call):
        took = []
        for _ in range(20):
            since = time.perf_counter()
            call()
            took.append(time.perf_counter() - since)
        return min(took)

    # some 20 us each; truncate 6 ms and release 0.5 ms when they walked
    assert fastest(lambda: many.truncate(70)) < 1e-3
    assert fastest(lambda: many.release([5])) < 2e-4
    assert not any(t is many.prefix_group or t is many.prefix_pages for t in copied)
    many.share(0, [5])
    assert int(many.prefix_group[5]) == 0 and int(many.prefix_pages[0]) == 1
    with pytest.raises(ValueError, match="shares"):
        many.truncate(np.where(np.arange(2048) == 5, 63, many.lengths))
    assert fastest(lambda: many.truncate(many.lengths)) < 1e-3


def test_groups_follow_any_order_of_sharing_and_release(cache):
    """Against the groups counted page by page."""
    rng = np.random.default_rng(3)
    c = int4.Int4KVCache(1, 7, 4, 2, 64, n_pages=80, max_tokens=700, device="cpu")
    for step in range(300):
        b = int(rng.integers(7))
        if c.lengths[b] == 0 and rng.random() < 0.6:
            sources = [a for a in range(7) if c.lengths[a]]
            if sources:
                c.share(int(rng.choice(sources)), [b], None if rng.random() < 0.5 else 64 * int(rng.integers(0, 1 + min(c.lengths[sources]) // 64)))
        elif rng.random() < 0.4:
            c.release([b])
        else:
            n = np.zeros(7, np.int64)
            n[b] = rng.integers(1, 150)
            if (c.lengths + n).max() < 700 and c.free_pages > 3:
                c.extend(n)
        rows = [[int(p) for p in row if p >= 0] for row in c.page_table]
        held = [p for row in rows for p in row]
        groups = {}
        for a, row in enumerate(rows):
            if row and held.count(row[0]) > 1:
                groups.setdefault(row[0], []).append(a)
        want_group, want_pages = list(range(7)), [0] * 7
        for members in groups.values():
            common = 0
            while all(len(rows[a]) > common and rows[a][common] == rows[members[0]][common] for a in members):
                common += 1
            for a in members:
                want_group[a] = members[0]
            want_pages[members[0]] = common
        assert c.prefix_group.tolist() == want_group and c.prefix_pages.tolist() == want_pages
        for a, row in enumerate(rows):
            first_own = next((j for j, p in enumerate(row) if held.count(p) == 1), len(row))
            if first_own:
                with pytest.raises(ValueError, match="shares"):
                    c.truncate(np.where(np.arange(7) == a, min(64 * first_own - 1, int(c.lengths[a])), c.lengths))
            before = c.lengths
            c.truncate(before)
    assert c.free_pages + len(set(held)) == 80


def test_groups_of_a_batch_with_more_sequences_than_numbers(cache, monkeypatch):
    """A call takes MAX_GROUPS groups: those of several sequences are numbered first, what is left over is in none."""
    n = int4.MAX_GROUPS + 900
    many = int4.Int4KVCache(1, n, 1, 1, 64, n_pages=n + 50, max_tokens=64 * 3, device="cpu")
    assert many.prefix_pages.shape == (int4.MAX_GROUPS,)
    assert many.prefix_group.tolist() == [b if b < int4.MAX_GROUPS else -1 for b in range(n)]
    counts = np.zeros(n, np.int64)
    counts[[4500, 10, 3]] = 130, 64, 70
    many.extend(counts)
    many.share(4500, [4501, 7], 128)
    many.share(10, [4990])
    group, pages = many.prefix_group.tolist(), many.prefix_pages.tolist()
    assert group[7] == group[4500] == group[4501] == 0 and pages[0] == 2 and group[10] == group[4990] == 1 and pages[1] == 1
    rest = [b for b in range(n) if b not in (7, 4500, 4501, 10, 4990)]
    assert [group[b] for b in rest] == [2 + i if 2 + i < int4.MAX_GROUPS else -1 for i in range(len(rest))] and not any(pages[2:])
    many.release([4500, 7, 4990])
    assert many.prefix_group.tolist() == [b if b < int4.MAX_GROUPS else -1 for b in range(n)] and not many.prefix_pages.any()


@pytest.mark.parametrize("cls", [int4.Int4KVCache, PackedKVCache])
@pytest.mark.parametrize("inference", [False, True])
def test_status_is_raised_wherever_the_cache_was_made(cls, inference):
    """A cache that was made in inference mode (an adapter makes its at the first forward) is asked outside of it."""
    with torch.inference_mode(inference):
        holder = type("Holder", (), dict(status=torch.full((1,), _lib.LF_ERR_DEVICE_TIMEOUT, dtype=torch.int32)))()
    with pytest.raises(RuntimeError, match="timed out"):
        cls.check_status(holder)
    cls.check_status(holder)      # and is clean behind it


def test_adapter_takes_the_prompt_kernel_by_name():
    model = tiny_qwen2(n_q=4, n_kv=2, head_dim=64, layers=1, vocab=32, seed=1)
    assert DeepSeekQwenKVAdapter(model, group_size=64).prompt == "dense"
    with pytest.raises(ValueError, match="prompt"):
        DeepSeekQwenKVAdapter(model, group_size=64, prompt="fast")
    a = DeepSeekQwenKVAdapter(model, group_size=64, prompt="kernel").attach()
    a._packed = type("Empty", (), dict(seq_len=0, layer_length=lambda self, i: 0, reset=lambda self: None))()
    ids = torch.zeros(1, 5, dtype=torch.long)
    with torch.no_grad(), pytest.raises((NotImplementedError, RuntimeError)):   # fp32 on the CPU: no fallback
        model(input_ids=ids)
    masked = torch.tensor([[0, 1, 1, 1, 1]])
    with torch.no_grad(), pytest.raises(NotImplementedError, match="mask"):
        model(input_ids=ids, attention_mask=masked)
