"""CPU model of what the two threads of a row of scores tell one another in the tensor-core
attention kernels: every interleaving of both, over the steps that their source has; and the
order in which a CTA of theirs ends.

A row's threads exchange numbers by way of one slot each.  The order of writes, meetings,
reads and of the waits between them is read from the sources (lf_flash.cuh, lf_prompt.cu,
lf_int4_prefix.cu); a read has to find the number of its own exchange in every schedule.
"""
from __future__ import annotations

import re
from pathlib import Path

import pytest

CSRC = Path(__file__).resolve().parents[1] / "logitfill_b200" / "csrc"
FLASH = (CSRC / "lf_flash.cuh").read_text()


def _code(text: str) -> str:
    return re.sub(r"//[^\n]*", "", text)


def _function(name: str) -> str:
    """Body of a function of lf_flash.cuh."""
    at = re.search(r"__device__ __forceinline__ \w+ %s\(" % name, FLASH).start()
    at = FLASH.index("{\n", at)
    return _code(FLASH[at:FLASH.index("\n}", at)])


# What a call does, step by step.  write: this thread's slot; meet: arrive, and wait for the
# other's arrival; read: the other's slot; ready: a step's weights are handed over, or its queries.
def _steps(body: str) -> list[str]:
    out = []
    for m in re.finditer(r"pair\.(exchange|meet)\(|part == 0 \? early : (ready)", body):
        what = m.group(1) or m.group(2)
        out += {"exchange": ["write", "meet", "read"], "meet": ["meet"], "ready": ["ready"]}[what]
    return out


def _role(kernel: str) -> tuple[list[str], list[str], list[str]]:
    """(before, of a step, behind) of an item in a kernel's softmax role."""
    text = (CSRC / kernel).read_text()
    text = _code(text[text.index("- softmax, one tile a warpgroup"):])
    soften, join = _steps(_function("soften_tile")), _steps(_function("join_sums"))
    before, step, behind = [], [], []
    for m in re.finditer(r"pair\.exchange\(|wait\(&sh\.(s_full|o_done)\[t\]|(soften_tile)<|(join_sums)\(|mbar_arrive\(&sh\.(q_ready)\[t\]", text):
        token = m.group(1) or m.group(2) or m.group(3) or m.group(4) or "exchange"
        if token == "s_full":
            step.append("scores")
        elif token == "soften_tile":
            step += soften
        elif token == "q_ready":
            before.append("ready")
        elif token == "exchange" and not step:
            before += ["write", "meet", "read"]
        else:
            behind += {"o_done": ["outputs"], "join_sums": join, "exchange": ["write", "meet", "read"]}[token]
    return before, step, behind


def _stale_read(program: list[str]):
    """The first read, of any schedule of two threads that run `program`, that does not find the
    number of its own exchange (None: there is none).

    scores: the products of a step are issued behind all weights of the step before (the first
    ones of an item behind its queries, too, where the softmax makes those), the outputs'
    behind the weights of the last: both wait for as many `ready` of the other thread as this
    one has given (the kernels wait for all 8 warps')."""
    seen, todo = set(), [((0, 0), (0, 0))]   # each thread's place, and the number of the exchange in its slot
    while todo:
        state = todo.pop()
        if state in seen:
            continue
        seen.add(state)
        at, slot = state
        for me in (0, 1):
            if at[me] == len(program):
                continue
            done, other = program[:at[me]], program[:at[1 - me]]
            op, mine, place = program[at[me]], list(slot), list(at)
            if op in ("scores", "outputs") and other.count("ready") < done.count("ready"):
                continue
            if op == "write":
                mine[me] += 1
            elif op == "await" and other.count("arrive") < done.count("arrive"):
                continue
            elif op == "read" and slot[1 - me] != done.count("write"):
                return at[me], done.count("write"), slot[1 - me]
            place[me] += 1
            todo.append((tuple(place), tuple(mine)))
    return None


def _program(kernel: str, tiles: int, items: int) -> list[str]:
    before, step, behind = _role(kernel)
    flat = items * (before + tiles * step + behind)
    return [op for x in flat for op in (("arrive", "await") if x == "meet" else (x,))]


@pytest.mark.parametrize("kernel", ["lf_prompt.cu", "lf_int4_prefix.cu"])
@pytest.mark.parametrize("tiles", [1, 2, 3])
def test_no_number_is_overwritten_before_it_is_read(kernel, tiles):
    before, step, behind = _role(kernel)
    assert step[:4] == ["scores", "write", "meet", "read"] and step.count("ready") == 1 and "outputs" in behind and "write" in behind
    assert _stale_read(_program(kernel, tiles, 3)) is None


def test_the_model_finds_an_exchange_that_waits_for_nothing():
    """The sums written behind a step's weights alone: the other thread may still have to read the maximum."""
    step = ["scores", "write", "arrive", "await", "read", "ready"]
    assert _stale_read(step + ["write", "arrive", "await", "read", "outputs"]) == (4, 1, 2)
    assert _stale_read(step + ["outputs", "write", "arrive", "await", "read"]) is None


@pytest.mark.parametrize("kernel", ["lf_prompt.cu", "lf_int4_prefix.cu"])
def test_products_in_flight_end_before_the_cta(kernel):
    """Any role may give up while products run whose end only the softmax would have waited for: what decides
    whether they are waited for is read when no role can give up any more, before tensor memory goes."""
    text = _code((CSRC / kernel).read_text())
    joined = text.rindex("__syncthreads();")
    committed, gone = text.index("mma_commit(&sh.last)"), text.rindex("tmem_dealloc")
    asked = [m.start() for m in re.finditer(r"if \(sh\.[\w.]*stop != 0\)", text[:committed])][-1]
    assert text.count("mma_commit(&sh.last)") == 1
    assert joined < asked < committed < text.index("mbar_wait_bounded(&sh.last", committed) < gone
