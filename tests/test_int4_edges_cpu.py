"""CPU tests of the 4-bit cache's refusals and bookkeeping at the edges."""
from __future__ import annotations

import os
import subprocess
import sys
from pathlib import Path

import pytest
import torch

from logitfill_b200 import _lib, int4
from tests.test_int4_cpu import _query, cpu_cache  # noqa: F401  (cpu_cache: a fixture)


def test_pools_without_pages_heads_or_sequences_are_refused():
    """Before anything divides by an extent: ValueError, wherever the tensors are."""
    pages, table = torch.zeros(4, 2, 1280, dtype=torch.int32), torch.zeros(1, 2, dtype=torch.int32)
    q, n = torch.zeros(1, 4, 64, dtype=torch.bfloat16), torch.zeros(1, dtype=torch.int32)
    for p, t, m, x in ((pages[:, :0], table, n, q), (pages[:0], table, n, q), (pages[..., :0], table, n, q),
                       (pages, table[:, :0], n, q), (pages, table[:0], n[:0], q[:0])):
        with pytest.raises(ValueError):
            int4.int4_attention(x, p, t, m, 1.0)
        with pytest.raises(ValueError):
            int4.int4_read(p, t, m, 3)


def test_cache_refuses_fewer_tokens_than_the_step_has(cpu_cache):  # noqa: F811
    """The lengths already count the step's tokens: a write of fewer would leave slots
    that later calls attend, and a query of fewer would be placed at the step's first
    tokens.  What has the step's tokens gets as far as the kernel."""
    c = cpu_cache
    k, q = torch.zeros(3, 2, 4, 64, dtype=torch.bfloat16), torch.zeros(3, 4, 4, 64, dtype=torch.bfloat16)

    def check(step, refused):
        c.extend(step)
        for n in range(1, 5):
            error = (ValueError, f"the step has {refused}") if n < refused else (RuntimeError, "CUDA")
            for call in (lambda: c.write(0, k[:, :, :n], k[:, :, :n]), lambda: c.attend(0, q[:, :, :n], 1.0),
                         lambda: c.attend_sparse(0, q[:, :, :n], 1.0, 4)):
                with pytest.raises(error[0], match=error[1]):
                    call()

    check([3, 0, 1], 3)
    check(2, 2)
    with pytest.raises(RuntimeError, match="CUDA"):
        c.extend(1)
        c.attend(0, q[:, :, 0], 1.0)
    c.extend(2)
    with pytest.raises(ValueError, match="the step has 2"):
        c.attend(0, q[:, :, 0], 1.0)
    c.truncate([1, 1, 1])   # no step is open: nothing of a query is attended, nothing is written
    for call in (lambda: c.write(0, k, k), lambda: c.attend(0, q, 1.0)):
        with pytest.raises(RuntimeError, match="CUDA"):
            call()


def test_release_of_a_sequence_that_is_not_there_changes_nothing(cpu_cache):  # noqa: F811
    c = cpu_cache
    c.extend([65, 10, 3])
    table, start = c.page_table.clone(), c.start.clone()
    for seqs in ([0, 3], [1, -4], [0, 1, "2"], [0, None]):
        with pytest.raises((IndexError, TypeError)):
            c.release(seqs)
        assert c.free_pages == 4 and c.lengths.tolist() == [65, 10, 3]
        assert torch.equal(c.page_table, table) and torch.equal(c.start, start)
    c.release([0, 0, -1])   # twice, and from the end
    assert c.free_pages == 7 and c.lengths.tolist() == [0, 10, 0] and c.end.tolist() == [0, 10, 0]
    assert (c.page_table[0] == -1).all() and int((c.page_table >= 0).sum()) == 1


@pytest.mark.skipif(torch.cuda.is_available(), reason="the pointers are made up: nothing may be launched")
@pytest.mark.parametrize("wrong", [dict(out=0), dict(os=(512, 62, 64)), dict(scaling=float("nan")), dict(slots=3, sink=1, recent=1, out=0)])
def test_a_sparse_call_is_checked_before_its_first_launch(wrong):
    """What only the attention refuses is refused before the choice of pages runs (whose
    launch would fail here in another way)."""
    so = _lib.lib()
    assert so.lf_int4_attend_sparse(_query(**wrong), None) == _lib.LF_ERR_INVALID_ARGUMENT
    assert b"lf_int4_attend" in so.lf_last_error()


@pytest.mark.skipif(torch.cuda.is_available(), reason="the pointers are made up: nothing may be launched")
@pytest.mark.parametrize("large", [dict(batch=65535, q_len=65535), dict(n_q=1 << 30, q_len=65535), dict(batch=65535, table_width=1 << 20, table_stride=1 << 20, picked=0),
                                   dict(slots=(1 << 31) - 1)])
def test_sizes_whose_products_pass_32_bits_are_refused(large):
    assert _lib.lib().lf_int4_attend(_query(**large), None) == _lib.LF_ERR_UNSUPPORTED


def test_a_binding_of_another_torch_is_not_loaded(monkeypatch):
    """It is compiled against torch's C++ classes: for another version there is none,
    however old the file is."""
    monkeypatch.setattr(_lib, "_BINDING", None)
    monkeypatch.setattr(torch, "__version__", "1.0.0+none")
    with pytest.raises(RuntimeError, match="binding missing"):
        _lib.int4_binding()
    monkeypatch.undo()
    assert _lib.int4_binding() is _lib.int4_binding()


def test_the_library_builds_without_torch(tmp_path):
    """A host that links the C library alone has neither torch nor its headers."""
    (tmp_path / "torch.py").write_text("raise ImportError('no torch here')\n")
    script = Path(_lib.__file__).with_name("build.py")
    env = dict(os.environ, PYTHONPATH=str(tmp_path))
    done = subprocess.run([sys.executable, str(script), "--library"], env=env, capture_output=True, text=True, timeout=900)
    assert done.returncode == 0, done.stderr
    assert done.stdout.split() == [str(_lib.LIB_PATH)]
    done = subprocess.run([sys.executable, str(script)], env=env, capture_output=True, text=True, timeout=900)
    assert done.returncode != 0 and "no torch here" in done.stderr   # the binding needs it
