"""A second definition of a name in a test file hides the first, which is then
never run."""

import ast
import glob
import os

import pytest

HERE = os.path.dirname(os.path.abspath(__file__))


@pytest.mark.parametrize("path", sorted(glob.glob(os.path.join(HERE, "*.py"))),
                         ids=os.path.basename)
def test_no_definition_hides_another(path):
    with open(path) as f:
        tree = ast.parse(f.read())
    for scope in [tree] + [n for n in ast.walk(tree) if isinstance(n, ast.ClassDef)]:
        names = [n.name for n in scope.body
                 if isinstance(n, (ast.FunctionDef, ast.AsyncFunctionDef, ast.ClassDef))]
        assert sorted(names) == sorted(set(names)), \
            [n for n in set(names) if names.count(n) > 1]
