"""The entry file works as a script too: everything that its main block reaches is defined above it."""
import ast
import os

PATH = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "__graft_entry__.py")


def test_main_block_is_the_last_statement():
    with open(PATH) as f:
        body = ast.parse(f.read()).body
    mains = [i for i, node in enumerate(body) if isinstance(node, ast.If) and "__name__" in ast.unparse(node.test)]
    assert mains == [len(body) - 1]
