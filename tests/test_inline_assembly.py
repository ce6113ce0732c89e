"""Inline assembly names what it changes."""
import glob
import os
import re

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
FILES = sorted(f for where in ("include", "nvshmem_amd") for end in ("h", "hpp", "hip", "cpp")
               for f in glob.glob(os.path.join(ROOT, where, "**", "*." + end), recursive=True))


def statements(text):
    """Template and clobbers of every asm statement."""
    for m in re.finditer(r"\basm\s*(?:volatile)?\s*\(", text):
        depth, at, quoted = 1, m.end(), False
        while depth:
            c = text[at]
            if c == "\\" and quoted:
                at += 1
            elif c == '"':
                quoted = not quoted
            elif not quoted:
                depth += {"(": 1, ")": -1}.get(c, 0)
            at += 1
        body = text[m.end():at - 1]
        template = re.match(r'(\s*"(?:\\.|[^"\\])*")+', body)
        yield template.group(0), body[template.end():]


def changes_m0(template):
    # the first operand, of what is no wait and no store
    return any(re.match(r"\s*[sv]_\w+\s+m0\b", line) for line in re.split(r"\\n|\\t|\"", template))


def test_the_search_itself():
    found = list(statements('asm volatile("s_mov_b32 m0, %0\\n\\ts_nop 4" : : "s"(f(1)) : "memory"); asm("" : "+v"(x));'))
    assert len(found) == 2 and changes_m0(found[0][0]) and "f(1)" in found[0][1] and not changes_m0(found[1][0])
    assert not changes_m0('"s_mov_b32 %0, m0"')


@pytest.mark.parametrize("path", FILES, ids=[os.path.relpath(f, ROOT) for f in FILES])
def test_m0(path):
    for template, rest in statements(open(path).read()):
        assert not changes_m0(template) or '"m0"' in rest.split(":")[-1], template
