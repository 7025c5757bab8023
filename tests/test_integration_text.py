"""The Python programs of the integration text: that of the mixers runs as it stands,
and no call that only enqueues is given a tensor that nothing keeps."""
import ast
import os
import re

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def programs():
    with open(os.path.join(ROOT, "INTEGRATION.md")) as f:
        return re.findall(r"```python\n(.*?)```", f.read(), re.S)


def test_enqueued_calls_get_tensors_that_are_kept():
    seen = 0
    for text in programs():
        for call in ast.walk(ast.parse(text)):
            if not (isinstance(call, ast.Call) and isinstance(call.func, ast.Attribute)
                    and call.func.attr.endswith("_async")):
                continue
            seen += 1
            for arg in call.args + [k.value for k in call.keywords]:
                made = [c for c in ast.walk(arg) if isinstance(c, ast.Call)]
                assert not made, (ast.unparse(call), [ast.unparse(c) for c in made])
    assert seen >= 5


@pytest.mark.gpu
def test_the_mixers_program_runs():
    text = [t for t in programs() if "PagedKV.empty" in t]
    assert len(text) == 1
    env = {}
    exec(text[0], env)
    kv = env["kv"]
    # sequences 3 and 5 got a token, 7 became a copy of 3, which was freed
    assert kv.lens.tolist() == [1 if s in (5, 7) else 0 for s in range(64)]
    assert kv.refs.tolist() == [1, 1] + [0] * 4094
    env["ctx"].close()
