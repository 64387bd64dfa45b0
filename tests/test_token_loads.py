"""The built code of rows_kernel (fp8_tiled.hip) waits for its tokens (CPU: compiles to assembly,
runs nothing).

A group of steps' tokens go to LDS while the group before is multiplied; behind them a wave asks
for n weights, and before the barrier that lets all waves read the tokens it waits until at most n
loads are in flight. Loads end in order, so that is enough as long as the compiler keeps at least n
of them behind the tokens': moved before them, or past the wait, they would not count."""

from __future__ import annotations

import re

from test_mma_hazards import assembly

MEMORY = ("buffer_", "global_", "scratch_", "flat_")


def functions(text, name):
    current = None
    for line in text.splitlines():
        start = re.match(r"^(_Z\w+):", line)
        if start:
            current = (start.group(1), []) if name in start.group(1) else None
        elif line.startswith(".Lfunc_end"):
            if current:
                yield current
            current = None
        elif current:
            current[1].append(line)


def blocks(lines):
    """(label, instructions) up to each branch or label."""
    out = [("", [])]
    for line in lines:
        code = line.split(";")[0].strip()
        label = re.match(r"^(\.L\w+):", code)
        if label:
            out.append((label.group(1), []))
        elif code and not code.startswith("."):
            out[-1][1].append(code)
            if code.startswith(("s_cbranch", "s_branch", "s_endpgm")):
                out.append(("", []))
    return out


def check(lines):
    """(loops over groups of steps, broken blocks). The last group's tokens are loaded for nothing:
    no barrier waits for them."""
    loops, bad, waits, starts = 0, [], set(), []
    for label, code in blocks(lines):
        loads = [i for i, c in enumerate(code) if re.search(r"\blds\b", c)]
        barriers = [i for i, c in enumerate(code) if c == "s_barrier"]
        if not loads:
            continue
        behind = sum(c.startswith(MEMORY) for c in code[loads[-1] + 1:])
        if not barriers:
            starts.append((label, behind, code[-1].endswith(" " + label) if label else False))
            continue
        wait = re.search(r"vmcnt\((\d+)\)", code[barriers[0] - 1])
        if not wait or len(barriers) > 1 or barriers[0] > loads[0]:
            bad.append((label, "no wait before the barrier"))
            continue
        waits.add(int(wait.group(1)))
        if label and code[-1].startswith("s_cbranch") and code[-1].endswith(" " + label):
            loops += 1
            if behind < int(wait.group(1)):
                bad.append((label, behind))
    # the first tokens: those whose block is repeated lane group by lane group have others behind
    firsts = [s for s in starts if not s[2]]
    if not waits or not firsts or any(behind < max(waits) for _, behind, _ in firsts):
        bad.append(("first tokens", starts, waits))
    return loops, bad


def test_tokens_are_waited_for(tmp_path):
    kernels = list(functions(assembly("fp8_tiled.hip", tmp_path), "rows_kernel"))
    assert len(kernels) == 16  # gate|up: 3 exact and 1 scaled; products: 3 heights of 4 results
    for name, lines in kernels:
        loops, bad = check(lines)
        assert loops >= 4 and not bad, (name, loops, bad)


def test_the_check_finds_a_missing_load():
    load, tokens = "\tglobal_load_dwordx4 v[0:3], v[4:5], off nt", "\tbuffer_load_dwordx4 v1, s[4:7], s2 offen lds"
    step = [".L1:", "\ts_waitcnt vmcnt(2) lgkmcnt(0)", "\ts_barrier", tokens]
    last = ["\ts_cbranch_scc1 .L1", "\ts_endpgm"]
    good = [tokens, load, load, *step, load, load, *last]
    assert check(good) == (1, [])
    for wrong in ([load, load, tokens, *step, load, load, *last],            # before the first tokens
                  [tokens, load, load, *step, load, *last],                  # one past the loop's wait
                  [tokens, load, load, *step[:1], *step[2:], load, load, *last]):  # no wait
        assert check(wrong)[1]
