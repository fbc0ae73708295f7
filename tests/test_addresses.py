"""An address handed to the library is that of a tensor which a name holds: a
temporary's memory is free again before the call is made, for another tensor of
the same call or another thread on the same stream."""

import ast
from pathlib import Path

import pytest

PACKAGE = Path(__file__).resolve().parents[1] / "wpt_amd"
CHECKS = {"_rows"}  # give back the tensor they are handed


def held(node):
    if isinstance(node, ast.Call):
        return isinstance(node.func, ast.Name) and node.func.id in CHECKS and held(node.args[0])
    if isinstance(node, ast.IfExp):
        return held(node.body) and held(node.orelse)
    if isinstance(node, ast.Subscript):
        return held(node.value)
    return isinstance(node, (ast.Name, ast.Attribute, ast.Constant))


def temporaries(source):
    for node in ast.walk(ast.parse(source)):
        if not isinstance(node, ast.Call):
            continue
        if isinstance(node.func, ast.Name) and node.func.id == "ptr" and not held(node.args[0]):
            yield node.lineno
        if isinstance(node.func, ast.Attribute) and node.func.attr == "data_ptr" and not held(node.func.value):
            yield node.lineno


def test_temporaries_are_told_from_held_tensors():
    assert list(temporaries("a = ptr(x)\nb = ptr(x[:2])\nc = ptr(None if x is None else _rows(x, 'x'))\nd = x.w.data_ptr()")) == []
    assert list(temporaries("a = ptr(x.contiguous())\nb = (x + 1).data_ptr()\nc = ptr(x if y else x.float())")) == [1, 2, 3]


@pytest.mark.parametrize("path", sorted(PACKAGE.glob("*.py")), ids=lambda p: p.name)
def test_no_address_of_a_temporary_is_handed_over(path):
    assert list(temporaries(path.read_text())) == []
