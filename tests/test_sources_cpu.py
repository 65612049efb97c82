"""What the kernels' sources keep to: a kernel is made resident while the kernels in front of it still run (programmatic dependent
launch), so it waits for them before it reads anything, and reads nothing through the read-only path, which is for memory that
nobody writes while the kernel lives."""
import pathlib
import re

import pytest

CSRC = pathlib.Path(__file__).parents[1] / "memorax_b200" / "csrc"
SOURCES = sorted([*CSRC.glob("*.cu"), *CSRC.glob("*.cuh")])


def code(path):
    return re.sub(r"//[^\n]*", "", path.read_text())


def closing(text, at, pair):
    """Index behind the bracket that closes the one at ``at``."""
    depth = 0
    for i in range(at, len(text)):
        depth += (text[i] == pair[0]) - (text[i] == pair[1])
        if depth == 0:
            return i + 1
    raise ValueError("unbalanced")


def kernels(text):
    """(name, parameters, body) of every kernel."""
    for start in re.finditer(r"__global__", text):
        head = re.compile(r"\s*void\s+(?:__launch_bounds__)?").match(text, start.end())
        at = head.end()
        if text[at] == "(":                                   # the bounds' brackets
            at = closing(text, at, "()")
        name = re.compile(r"\s*(\w+)\s*").match(text, at)
        ends = closing(text, name.end(), "()")
        body = text.index("{", ends)
        yield name.group(1), text[name.end():ends], text[body:closing(text, body, "{}")]


@pytest.mark.parametrize("path", SOURCES, ids=lambda p: p.name)
def test_nothing_is_read_through_the_read_only_path(path):
    text = code(path)
    assert not re.findall(r"__ldg\b|\.nc\b|ldg_|__constant__\s*const|tex\w*Fetch", text)
    # a parameter that is only read and promised not to be written by others is read that way by the compiler
    assert not re.findall(r"const\s+[\w:]+\s*\*\s*(?:const\s*)?__restrict__", text)


def test_every_kernel_waits_for_those_in_front():
    found = 0
    for path in SOURCES:
        for name, _, body in kernels(code(path)):
            found += 1
            if name == "bounded_wait_selftest_kernel":        # launched without the attribute
                continue
            waits = [m.start() for m in re.finditer(r"enter_kernel\(|griddepcontrol\.wait", body)]
            assert waits, (path.name, name)
            # nothing is read from memory before: no access through a pointer, no copy
            before = body[:waits[0]]
            assert not re.search(r"\[|ld_|load|->|copy", before), (path.name, name, before)
    assert found > 70
