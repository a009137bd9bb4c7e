"""The entry file as a script: what it runs is defined before it runs it."""
import ast
import os

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def test_the_main_guard_is_the_last_statement():
    with open(os.path.join(ROOT, "__graft_entry__.py")) as f:
        body = ast.parse(f.read()).body
    guards = [i for i, s in enumerate(body) if isinstance(s, ast.If) and "__main__" in ast.unparse(s.test)]
    assert guards == [len(body) - 1], guards
