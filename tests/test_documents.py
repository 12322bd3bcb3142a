"""The Python examples of the documents: every name of the package that they use exists."""
import glob
import os
import re

import pytest

import dfattn
from dfattn import checkpoint, ops, w4

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
MODULES = {"dfattn": dfattn, "checkpoint": checkpoint, "ops": ops, "w4": w4}


def examples():
    for path in sorted(glob.glob(os.path.join(ROOT, "*.md"))):
        for block in re.findall(r"^```python\n(.*?)^```", open(path).read(), re.M | re.S):
            yield from ((os.path.basename(path), m, a) for m, a in re.findall(r"\b(dfattn|checkpoint|ops|w4)\.(\w+)", block))


@pytest.mark.parametrize("path,module,name", sorted(set(examples())))
def test_names(path, module, name):
    assert hasattr(MODULES[module], name)


def test_there_are_examples():
    assert len(set(examples())) > 10
