"""The Julia binding of the operators around a decoder's step, read as text (no Julia here): every array whose pointer the library is given has been compared
with the sizes that it is told, before the call."""
import os
import re

import pytest

import juliavision_b200 as jv

BINDING = os.path.join(os.path.dirname(jv.__file__), "julia", "B200Backend.jl")


def body(name):
    with open(BINDING) as f:
        text = f.read()
    text = re.sub(r"#[^\n]*", "", text)
    at = text.index(f"function {name}(")
    return text[at:text.index("\nend\n", at)]


def call(text, opening):
    """What stands between the brackets after each `opening`."""
    for m in re.finditer(re.escape(opening), text):
        end, depth = m.end(), 1
        while depth:
            depth += {"(": 1, ")": -1}.get(text[end], 0)
            end += 1
        yield text[m.end():end - 1]


@pytest.mark.parametrize("name, operands", [("normrotary!", "out x weight lens news split"), ("packedsdpa!", "out q k v starts kstarts"),
                                            ("beamselect!", "best parents tokens logits scores ended"), ("cachereorder!", "caches table own parents lens")])
def test_operands_are_compared_before_the_call(name, operands):
    text = body(name)
    before, after = text[:text.index("check(ccall(")], text[text.index("check(ccall("):]
    demands = " ".join(call(before, "demand("))
    given = set(re.findall(r"(?:pointer|nullable|s3|s4)\((\w+)", after)) | ({"caches"} if "caches" in operands else set())
    assert given - {"plan"} <= set(operands.split())
    for a in operands.split():
        checked = re.findall(rf"(?:size|eltype|isdense|iscounts|length|ndims)\({a}\b|<= {a} <=|, {a}\)", demands)
        assert checked, (name, a)
    # sizes that the library is told are taken from arrays whose shape has been settled
    assert re.search(r"ndims\(\w+\) ==", demands)


def test_brackets_are_closed():
    with open(BINDING) as f:
        text = re.sub(r'"(?:[^"\\\n]|\\.)*"', '""', re.sub(r"#[^\n]*", "", f.read()))
    text = re.sub(r'"""[^"]*"""', "", text)
    for a, b in ("()", "[]", "{}"):
        assert text.count(a) == text.count(b), a
