"""The order of the output warps in enx_attn_packed (csrc/k_packed.cu), on the host: every interleaving of
threads that clean an item's V tiles (and raise the item's flag where they find what is not finite), arrive on
that item's barrier, wait for it, and look at the flag.  Each must see its own item's flag as it was left when
the barrier completed, whatever another thread does for the next items meanwhile."""

import re

import pytest

from conftest import ROOT

ITEMS, THREADS = 4, 2


def outcomes(flags, fouls):
    """All (thread, item, what it saw) over all interleavings.  fouls[t][k]: thread t finds something in
    item k.  Steps of an item: clean (and raise), arrive, pass the barrier, look."""
    seen, todo, done = set(), [((0,) * THREADS, (0,) * flags, (0,) * ITEMS)], set()
    while todo:
        state = todo.pop()
        if state in done:
            continue
        done.add(state)
        at, flag, arrived = state
        for t in range(THREADS):
            k, step = divmod(at[t], 4)
            if k == ITEMS:
                continue
            f, a = flag, arrived
            if step == 0 and fouls[t][k]:
                f = tuple(k + 1 if i == k % flags else v for i, v in enumerate(flag))
            elif step == 1:
                a = tuple(v + (i == k) for i, v in enumerate(arrived))
            elif step == 2 and arrived[k] < THREADS:
                continue  # waits
            elif step == 3:
                seen.add((t, k, flag[k % flags] == k + 1))
            todo.append((tuple(v + (i == t) for i, v in enumerate(at)), f, a))
    return seen


def wrong(flags):
    bad = 0
    for bits in range(1 << THREADS * ITEMS):
        fouls = [[bits >> (t * ITEMS + k) & 1 for k in range(ITEMS)] for t in range(THREADS)]
        bad += any(saw != any(fouls[t][k] for t in range(THREADS)) for _, k, saw in outcomes(flags, fouls))
    return bad


def test_the_kernels_flags_are_enough():
    source = (ROOT / "enargeia_b200" / "csrc" / "k_packed.cu").read_text()
    flags = re.findall(r"constexpr uint32_t kPkFoul = (\d+);", source)
    assert len(flags) == 1 and len(re.findall(r"s_foul\[k % kPkFoul\]", source)) == 2
    assert wrong(int(flags[0])) == 0


@pytest.mark.parametrize("flags", [1])
def test_one_flag_is_not(flags):
    assert wrong(flags) > 0
