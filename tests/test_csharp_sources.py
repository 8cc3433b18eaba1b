"""Rules of C# that the backend's sources have to keep (they are compiled where the reference is, not here)."""
import glob
import os
import re

import pytest

SOURCES = sorted(glob.glob(os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "onegpu-csharp_b200",
                                        "csharp", "RecursiveAI.OneGpu.Cuda", "*.cs")))


def code(path):
    """A file without its comments and strings."""
    text = open(path, encoding="utf-8").read()
    return re.sub(r'//[^\n]*|/\*.*?\*/|"(?:[^"\\\n]|\\.)*"', " ", text, flags=re.S)


def body(text, at):
    """The block in braces from `at` on."""
    start = text.index("{", at)
    depth = 0
    for i in range(start, len(text)):
        depth += {"{": 1, "}": -1}.get(text[i], 0)
        if depth == 0:
            return text[start:i]
    raise AssertionError("unbalanced braces")


@pytest.mark.parametrize("path", SOURCES, ids=os.path.basename)
def test_structs_with_defaults_have_a_parameterless_constructor(path):
    """Field initializers of a struct run in its declared constructors only: `new T { .. }` of one without a parameterless
    constructor is all zeros."""
    text = code(path)
    for m in re.finditer(r"\bstruct\s+(\w+)\s*\{", text):
        block = body(text, m.start())
        while re.search(r"\{[^{}]*\}", block[1:]):  # members only, not what they hold
            block = block[0] + re.sub(r"\{[^{}]*\}", ";", block[1:])
        constructors = re.findall(r"\bpublic\s+%s\s*\(([^)]*)\)" % m.group(1), block)
        assigned = [f for f in re.findall(r"\bpublic\s+[^;()=]*=(?!>)[^;]*;", block)]
        if assigned or constructors:
            assert any(not c.strip() for c in constructors), (m.group(1), assigned)


def namespace_of(path):
    return re.search(r"^namespace\s+([\w.]+);", code(path), re.M).group(1)


@pytest.mark.parametrize("path", SOURCES, ids=os.path.basename)
def test_types_of_the_other_namespace_are_imported(path):
    """A file names another namespace's types only with a using of it."""
    own, text = namespace_of(path), code(path)
    using = set(re.findall(r"^using\s+([\w.]+);", text, re.M))
    for other in SOURCES:
        space = namespace_of(other)
        if space == own or own.startswith(space + "."):
            continue
        for name in re.findall(r"\b(?:struct|class|enum)\s+(\w+)", code(other)):
            assert space in using or not re.search(r"(?<![\w.])%s\b" % name, text), (name, space)
