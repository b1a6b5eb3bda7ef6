"""A test whose name comes again in its file is not collected, and nothing says so."""
from __future__ import annotations

import ast
from collections import Counter
from pathlib import Path

import pytest

FILES = sorted(Path(__file__).resolve().parent.glob("*.py"))


@pytest.mark.parametrize("path", FILES, ids=[p.name for p in FILES])
def test_each_name_once(path):
    tree = ast.parse(path.read_text())
    for body in [tree.body] + [n.body for n in ast.walk(tree) if isinstance(n, ast.ClassDef)]:
        names = Counter(n.name for n in body if isinstance(n, (ast.FunctionDef, ast.AsyncFunctionDef, ast.ClassDef)))
        assert not [n for n, k in names.items() if k > 1]
