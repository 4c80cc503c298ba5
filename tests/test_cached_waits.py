"""Waits of the attention over a cache for few columns, on its gfx950 assembly (CPU only).

A wave's keys arrive in LDS by loads of their own (`buffer_load_dwordx4 ... lds`), which the
compiler does not see to write what is read later: the kernel waits by hand, by the number of
loads that stand behind the keys'. That is right only while the compiled code keeps as many
behind them on every way to a read. So each kernel's body is followed along all its branches: no LDS
access may be reached while a key's load can be on its way.

Loads return in order, so a key's load is over behind a wait that lets no more loads be on their way
than were issued after it. Stores and scratch accesses are not counted: that only asks for more.
"""
import math
import re

import pytest

import test_kernel_asm as kernel_asm

asm_of = kernel_asm.asm_of

KEYS = re.compile(r"buffer_load_dwordx4 .* lds$")
LOAD = re.compile(r"(buffer|global)_load_")
WAIT = re.compile(r"s_waitcnt .*vmcnt\((\d+)\)")
LDS = re.compile(r"ds_(?!bpermute|permute|swizzle)")
BRANCH = re.compile(r"s_c?branch\w* (\S+)$")


def blocks_of(lines, prefix):
    """Basic blocks of the kernel whose symbol starts with prefix: [instructions, successors]."""
    start = next(i for i, l in enumerate(lines) if re.match(r"^\S+:", l) and l.startswith(prefix))
    end = next(i for i in range(start, len(lines)) if lines[i].startswith(".Lfunc_end"))
    blocks, labels = [[[], []]], {}
    for line in lines[start + 1:end]:
        line = line.split(";")[0].strip()
        if not line or (line.startswith(".") and not line.endswith(":")):
            continue
        if line.endswith(":"):
            blocks[-1][1].append(len(blocks))
            blocks.append([[], []])
            labels[line[:-1]] = len(blocks) - 1
            continue
        blocks[-1][0].append(line)
        assert not line.startswith(("s_setpc", "s_swappc", "s_call")), line
        if BRANCH.match(line) or line.startswith("s_endpgm"):
            if line.startswith("s_cbranch"):
                blocks[-1][1].append(len(blocks))
            if BRANCH.match(line):
                blocks[-1][1].append(BRANCH.match(line)[1])
            blocks.append([[], []])
    return [(code, [labels.get(s, s) for s in after if s != len(blocks)]) for code, after in blocks]


def too_early(blocks):
    """LDS accesses that a key's load may still be on its way at. What is known at a place: the
    fewest loads behind the last key's, inf where none is on its way."""
    known = {0: math.inf}
    todo, found = [0], set()
    while todo:
        b = todo.pop()
        n = known[b]
        for i, line in enumerate(blocks[b][0]):
            if KEYS.match(line):
                n = 0
            elif LOAD.match(line):
                n += 1
            elif WAIT.match(line):
                n = math.inf if n >= int(WAIT.match(line)[1]) else n
            elif LDS.match(line) and n < math.inf:
                found.add((b, i, line))
        n = n if n == math.inf else min(n, 64)
        for s in blocks[b][1]:
            if s not in known or n < known[s]:
                known[s] = n
                todo.append(s)
    return found


@pytest.mark.parametrize("wide", [1, 2, 3, 4])
@pytest.mark.parametrize("type", ["t", "f"])
def test_no_lds_access_before_the_keys_are_there(asm_of, type, wide):
    blocks = blocks_of(asm_of("cached_rows.hip"),
                       f"_ZN3tfd12_GLOBAL__N_118cached_rows_kernelI{type}Li{wide}E")
    keys = sum(bool(KEYS.match(line)) for code, _ in blocks for line in code)
    assert keys >= 2 * 4 * wide, "the keys no longer come by loads into LDS: update this check"
    found = too_early(blocks)
    assert not found, sorted(found)[:5]


@pytest.mark.parametrize("wide", [1, 4])
def test_the_check_sees_a_missing_wait(asm_of, wide):
    """The same body with each wait by hand left out, or for one load too many."""
    lines = asm_of("cached_rows.hip")
    prefix = f"_ZN3tfd12_GLOBAL__N_118cached_rows_kernelIfLi{wide}E"
    start = next(i for i, l in enumerate(lines) if re.match(r"^\S+:", l) and l.startswith(prefix))
    end = next(i for i in range(start, len(lines)) if lines[i].startswith(".Lfunc_end"))
    by_hand = [i for i in range(start, end)
               if lines[i].strip() == f"s_waitcnt vmcnt({4 * wide})" and "ASMSTART" in lines[i - 1]]
    assert len(by_hand) >= 2  # of the loop, and of the last block
    for other in ("", f"s_waitcnt vmcnt({4 * wide + 1})"):
        changed = [("\t" + other if i in by_hand else l) for i, l in enumerate(lines)]
        assert too_early(blocks_of(changed, prefix))
