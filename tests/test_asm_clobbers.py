"""Inline assembly names every register that it writes outside its operands."""

import re
from pathlib import Path

import svoo_amd


def _statements():
    for path in sorted((Path(svoo_amd.__file__).parent / "csrc").iterdir()):
        text = path.read_text()
        for m in re.finditer(r"(?:__asm__|\basm)\b[^;(]*\(", text):
            depth, end = 1, m.end()
            while depth:
                depth += {"(": 1, ")": -1}.get(text[end], 0)
                end += 1
            yield f"{path.name}:{text.count(chr(10), 0, m.start()) + 1}", text[m.start():end]


def test_asm_that_writes_m0_says_so():
    writers = [(at, s) for at, s in _statements() if re.search(r"\bs_\w+ m0,", s)]
    assert len(writers) >= 5
    assert [at for at, s in writers if '"m0"' not in s] == []
