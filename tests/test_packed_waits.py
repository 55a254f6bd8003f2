"""What must hold of packed attention's waits and cannot be shown by running them: that the warp which hands values on never waits for a fill of
the ring that has come and gone.  A model of the ring, over every order in which its roles can run, and what the source has them wait for."""
import os
import re

import pytest

from juliavision_b200 import build


def source():
    with open(os.path.join(build.CSRC, "attention_packed.cu")) as f:
        return re.sub(r"//[^\n]*", "", f.read())


def followed(text):
    """The sides of a block, K or V, whose landing the handing-on warp waits for."""
    role = text[text.index("} else if (warp == 11) {"):]
    role = role[:role.index("mbar_arrive(&ready[")]
    sides = []
    for at in re.findall(r"wait\(&full\[([^\]]*)\]", role):
        at = at.strip()
        if at == "st":
            at = re.search(r"const int st = ([^,;]*)", role).group(1).strip()
        sides.append({"i % STAGES": "K", "(i + 1) % STAGES": "V"}[at])
    return "".join(sides)


def stages(text):
    found = re.search(r"static constexpr int STAGES = \w+ \? (\d+) : (\d+);", text)
    return [int(n) for n in found.groups()]


def passes(done, nth):
    """mbarrier.try_wait.parity for a barrier's nth phase where `done` are over: only parities are compared."""
    return done % 2 != nth % 2


def stranded(S, follow, own_p, blocks):
    """Walks every order of: the loader, which asks for sides in turn; landings, in any order; the warp that hands values on; one issuer, which stands
    for both (each stage is released once by it).  Returns what goes wrong, or None: a wait that never ends, or one that ends early."""
    sides = 2 * blocks
    # the issuer's steps: what it waits for and what it releases
    steps = []
    for j in range(blocks):
        if own_p:
            if j == 0:
                steps.append(("K", 0))
            if j + 1 < blocks:
                steps.append(("K", j + 1))
            steps.append(("V", j))
        else:
            steps += [("K", j), ("V", j)]
    start = (0, frozenset(), (0,) * S, (0,) * S, 0, 0, 0)
    seen, todo = {start}, [start]
    while todo:
        asked, flying, full, empty, hand, at, step = todo.pop()
        nexts = []
        if asked < sides:
            st, nth = asked % S, asked // S
            if nth == 0 or passes(empty[st], nth - 1):
                if nth > empty[st]:
                    return "a stage is filled that is still read"
                nexts.append((asked + 1, flying | {asked}, full, empty, hand, at, step))
        for side in flying:
            st = side % S
            nexts.append((asked, flying - {side}, full[:st] + (full[st] + 1,) + full[st + 1:], empty, hand, at, step))
        if hand < blocks:
            side = 2 * hand + (follow[at] == "V")
            if passes(full[side % S], side // S):
                if full[side % S] <= side // S:
                    if at + 1 == len(follow):
                        return "values are handed on before they land"
                last = at + 1 == len(follow)
                nexts.append((asked, flying, full, empty, hand + last, 0 if last else at + 1, step))
        if step < len(steps):
            kind, j = steps[step]
            side = 2 * j + (kind == "V")
            st = side % S
            if passes(full[st], side // S) if kind == "K" else hand > j:
                nexts.append((asked, flying, full, empty[:st] + (empty[st] + 1,) + empty[st + 1:], hand, at, step + 1))
        if not nexts and (asked < sides or flying or hand < blocks or step < len(steps)):
            return "a wait never ends"
        for n in nexts:
            if n not in seen:
                seen.add(n)
                todo.append(n)
    return None


@pytest.mark.parametrize("own_p", [True, False])
@pytest.mark.parametrize("S", [4, 8])
def test_the_model_finds_what_is_wrong(S, own_p):
    """Following K's fills, whose release is not the warp's to give: one that is late waits for good.  Stages that K and V share, V's followed
    alone: a fill seen last two fills ago looks full."""
    assert stranded(S, "KV", own_p, S + 2) == "a wait never ends"
    assert stranded(S, "V", own_p, S + 2) is None
    assert stranded(5, "V", own_p, 8) is not None


def test_values_are_handed_on_whatever_the_order():
    text = source()
    assert re.search(r"static_assert\(STAGES % 2 == 0", text)
    for S in stages(text):
        for own_p in (True, False):
            assert stranded(S, followed(text), own_p, S + 2) is None
