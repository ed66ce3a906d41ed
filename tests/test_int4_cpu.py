"""CPU tests of the 4-bit cache: argument structs, validation before any launch,
page bookkeeping, and the reference's own consistency."""
from __future__ import annotations

import ctypes
import re
import struct
from pathlib import Path

import numpy as np
import pytest
import torch

from logitfill_b200 import _lib, int4
from tests import int4_reference as ref

HEADER = (Path(__file__).resolve().parents[1] / "include" / "logitfill_b200.h").read_text()
SIZES = {"void*": 8, "int32_t*": 8, "int8_t*": 8, "int64_t": 8, "size_t": 8, "int32_t": 4, "float": 4, "lf_int4_pool": 56}


# The argument structs, field by field; checked against the header below.
POOL = "PPqqqiiii"
TOKENS = struct.Struct("@" + POOL + "PP6qPPPqqPiii0q")
QUERY = struct.Struct("@" + POOL + "P3qP3qPPPqqPPNPf7i")


def _fields(name):
    """(type, name) of every field of a header struct, in order."""
    body = re.search(r"typedef struct %s \{(.*?)\} %s;" % (name, name), HEADER, re.S).group(1)
    body = re.sub(r"/\*.*?\*/", "", body, flags=re.S)
    out = []
    for decl in filter(None, (d.strip() for d in body.split(";"))):
        decl = decl.replace("const ", "")
        kind, names = re.match(r"([\w]+\s*\*?)\s*(.*)", decl, re.S).groups()
        out += [(kind.replace(" ", ""), n.strip()) for n in names.split(",")]
    return out


def _size(name):
    at = 0
    for kind, _ in _fields(name):
        n = SIZES[kind]
        align = 8 if kind == "lf_int4_pool" else n
        at = -(-at // align) * align + n
    return -(-at // 8) * 8


def test_packed_structs_follow_the_header():
    pool = POOL
    code = {"void*": "P", "int32_t*": "P", "int8_t*": "P", "int64_t": "q", "size_t": "N", "int32_t": "i", "float": "f",
            "lf_int4_pool": pool}
    assert "".join(code[k] for k, _ in _fields("lf_int4_pool")) == pool and _size("lf_int4_pool") == 56
    for name, packed in (("lf_int4_tokens", TOKENS), ("lf_int4_query", QUERY)):
        want = "".join(code[k] for k, _ in _fields(name))
        spelled = re.sub(r"(\d+)([a-zA-Z])", lambda m: int(m.group(1)) * m.group(2),
                         packed.format.lstrip("@"))
        assert spelled == want, name
        assert packed.size == _size(name)


def _tokens(**over):
    fake = 1 << 20   # never dereferenced: validation fails first
    f = dict(pages=fake, table=fake, page_stride=2560, head_stride=1280, table_stride=4, table_width=4, n_pages=8,
             kv_heads=2, batch=2, key=fake, value=fake, strides=(1024,) * 6, start=fake, counts=0, bounds=0, b0=0, b1=0,
             status=0, head_dim=64, dtype=_lib.LF_BF16, tokens=4)
    f.update(over)
    s = f.pop("strides")
    v = list(f.values())
    return TOKENS.pack(*v[:11], *s, *v[11:])


def _query(**over):
    fake = 1 << 20
    f = dict(pages=fake, table=fake, page_stride=2560, head_stride=1280, table_stride=4, table_width=4, n_pages=8,
             kv_heads=2, batch=2, q=fake, qs=(512, 64, 64), out=fake, os=(512, 64, 64), lengths=fake, counts=0, bounds=fake,
             b0=288, b1=144, picked=fake, ws=fake, ws_bytes=1 << 30, status=0, scaling=1.0, head_dim=64,
             dtype=_lib.LF_BF16, n_q=8, q_len=1, slots=6, sink=1, recent=2)
    f.update(over)
    flat = []
    for v in f.values():
        flat += list(v) if isinstance(v, tuple) else [v]
    return QUERY.pack(*flat)


def test_entry_points_validate_before_launch():
    so = _lib.lib()
    invalid, unsupported = _lib.LF_ERR_INVALID_ARGUMENT, _lib.LF_ERR_UNSUPPORTED
    for fn in (so.lf_int4_write, so.lf_int4_read):
        assert fn(None, None) == invalid
        assert fn(_tokens(tokens=0), None) == _lib.LF_OK                     # nothing to do, nothing launched
        assert fn(_tokens(pages=0), None) == invalid
        assert fn(_tokens(pages=(1 << 20) + 4), None) == invalid             # records not 16-byte aligned
        assert fn(_tokens(head_dim=96), None) == unsupported
        assert fn(_tokens(head_stride=1000), None) == invalid                # records overlap
        assert fn(_tokens(table_stride=3), None) == invalid
        assert fn(_tokens(batch=0), None) == invalid
        assert fn(_tokens(batch=70000), None) == unsupported
        assert fn(_tokens(key=0), None) == invalid
        assert fn(_tokens(key=(1 << 20) + 2), None) == invalid
        assert fn(_tokens(strides=(1024, 1024, 68, 1024, 1024, 64)), None) == invalid
        assert fn(_tokens(dtype=7), None) == invalid
        assert fn(_tokens(tokens=-1), None) == invalid
        assert fn(_tokens(bounds=1 << 20, b0=64, b1=64), None) == invalid
    for fn in (so.lf_int4_select, so.lf_int4_attend, so.lf_int4_attend_sparse):
        assert fn(None, None) == invalid
        assert fn(_query(q=0), None) == invalid
        assert fn(_query(lengths=0), None) == invalid
        assert fn(_query(dtype=_lib.LF_F32), None) == unsupported
        assert fn(_query(n_q=9), None) == invalid
        assert fn(_query(q_len=0), None) == invalid
        assert fn(_query(qs=(512, 60, 64)), None) == invalid
        assert fn(_query(head_dim=256), None) == unsupported
    for fn in (so.lf_int4_select, so.lf_int4_attend_sparse):
        assert fn(_query(bounds=0), None) == invalid
        assert fn(_query(bounds=(1 << 20) + 4), None) == invalid
        assert fn(_query(recent=0), None) == invalid
        assert fn(_query(sink=5), None) == invalid                            # more than the slots
        assert fn(_query(n_q=130), None) == unsupported                       # 65 heads per KV head
        assert fn(_query(table_width=40000, table_stride=40000), None) == unsupported
    assert so.lf_int4_attend(_query(out=0), None) == invalid
    assert so.lf_int4_attend(_query(os=(512, 62, 64)), None) == invalid
    assert so.lf_int4_attend(_query(slots=0), None) == invalid
    assert so.lf_int4_read_bounds(None, 0, 0, 1, 1, 64, None, None) == invalid
    assert b"lf_int4_read_bounds" in so.lf_last_error()


def test_functions_refuse_cpu_tensors_and_wrong_shapes():
    pages, table = torch.zeros(4, 2, 1280, dtype=torch.int32), torch.zeros(1, 2, dtype=torch.int32)
    q, n = torch.zeros(1, 4, 64, dtype=torch.bfloat16), torch.zeros(1, dtype=torch.int32)
    with pytest.raises(RuntimeError, match="CUDA"):
        int4.int4_attention(q, pages, table, n, 1.0)
    with pytest.raises(ValueError, match="pages"):
        int4.int4_attention(q, pages[0], table, n, 1.0)
    with pytest.raises(ValueError, match="page_table"):
        int4.int4_attention(q, pages, table.long(), n, 1.0)
    with pytest.raises(RuntimeError, match="CUDA"):
        int4.int4_read_bounds(torch.zeros(4, 2, 144, dtype=torch.int8))
    with pytest.raises(NotImplementedError):
        int4.Int4KVCache(1, 1, 4, 2, 80, 4, 64, device="cpu")


@pytest.fixture
def cpu_cache(monkeypatch):
    """A cache whose bookkeeping runs without a GPU."""
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: False)
    monkeypatch.setattr(int4.Int4KVCache, "_upload", lambda self, t, host: t.copy_(torch.from_numpy(host.astype(np.int32))))
    return int4.Int4KVCache(1, 3, 4, 2, 64, n_pages=8, max_tokens=300, device="cpu")


def test_cache_bookkeeping(cpu_cache):
    c = cpu_cache
    c.extend([65, 0, 64])
    assert c.lengths.tolist() == [65, 0, 64] and c.free_pages == 5
    assert c.start.tolist() == [0, 0, 0] and c.end.tolist() == [65, 0, 64] and c.counts.tolist() == [65, 0, 64]
    c.extend(1)
    assert c.start.tolist() == [65, 0, 64] and c.end.tolist() == [66, 1, 65] and c.counts.tolist() == [1, 1, 1]
    assert c.free_pages == 3
    used = [int(x) for x in c.page_table.flatten() if x >= 0]
    assert sorted(used) == sorted(set(used)) and len(used) == 5     # no page twice
    c.truncate([66, 1, 3])
    assert c.lengths.tolist() == [66, 1, 3] and c.free_pages == 3 and c.counts.tolist() == [0, 0, 0]
    with pytest.raises(RuntimeError, match="free"):
        c.extend([200, 200, 0])   # six pages more, three are free
    assert c.free_pages == 3 and c.lengths.tolist() == [66, 1, 3]
    with pytest.raises(ValueError, match="exceed"):
        c.extend([0, 400, 0])
    c.release([0])
    assert c.free_pages == 5 and c.lengths.tolist() == [0, 1, 3] and (c.page_table[0] == -1).all()
    c.reserve([300, 0, 0])
    assert c.free_pages == 0
    c.release()
    assert c.free_pages == 8 and (c.page_table == -1).all() and not c.lengths.any()


def test_reference_bounds_hold_and_record_decodes():
    rng = np.random.default_rng(0)
    x = rng.standard_normal((64, 64)).astype(np.float32) * rng.choice([1, 8], 64)
    s = ref.stored(x)
    assert np.abs(s - x).max() <= (x.reshape(64, 2, 32).max(-1) - x.reshape(64, 2, 32).min(-1)).max() / 30 * 1.01
    up, low, e = ref.page_bounds(s)
    assert (up * 2.0 ** e >= s.max(0)).all() and (low * 2.0 ** e <= s.min(0)).all() and np.abs([up, low]).max() <= 127
    q = rng.standard_normal((4, 64))
    f = ref.exponent(np.abs(q).max())
    assert np.abs(q).max() <= 127 * 2.0 ** f and np.abs(q).max() > 127 * 2.0 ** (f - 1)
    assert ref.exponent(0.0) == -40 and ref.exponent(127.0) == 0 and ref.exponent(127.0001) == 1


def test_workspace_grows_with_the_units():
    so = _lib.lib()
    small, large = (so.lf_int4_workspace_bytes(b, 8, 40, 1, 128) for b in (1, 4096))
    assert large - small == 4 * 8 * 4095 and small - so.lf_int4_workspace_clear_from() == 32
    assert so.lf_int4_workspace_bytes(0, 8, 40, 1, 128) == 0 == so.lf_int4_workspace_bytes(1, 8, 7, 1, 128)
    assert ctypes.c_size_t(so.lf_int4_workspace_clear_from()).value >= 0
