"""Inline assembly of the GPU sources says which of the registers that it names it writes (CPU only, reads the text)."""
import re

import pytest

from k8s_llm_monitor_amd import build


def statements(text):
    """The asm statements of a source: from `asm` to the `;` behind the closing parenthesis, strings read over."""
    for m in re.finditer(r"\basm\s*(?:volatile\s*)?\(", text):
        depth, i, quoted = 1, m.end(), False
        while depth:
            c = text[i]
            if c == "\\" and quoted:
                i += 1
            elif c == '"':
                quoted = not quoted
            elif not quoted:
                depth += (c == "(") - (c == ")")
            i += 1
        yield text[m.start():i]


SOURCES = sorted(p for pattern in ("*.hip", "*.h") for p in build.PKG.rglob(pattern))


@pytest.mark.parametrize("path", SOURCES, ids=lambda p: p.name)
def test_a_register_written_by_name_is_in_the_list_of_clobbers(path):
    for stmt in statements(path.read_text()):
        written = set(re.findall(r"\bs_mov_b(?:32|64)\s+(m0|exec|vcc)\b", stmt)) | set(re.findall(r"\bs_add_u32\s+(m0)\b", stmt))
        for reg in written:
            assert f'"{reg}"' in stmt, f"{path.name}: {reg} is written and not declared in\n{stmt}"


def test_the_reader_of_statements():
    text = 'x; asm volatile("s_mov_b32 m0, %0 ; (" : : "s"(f(1)) : "memory"); y; asm("" ::: "m0");'
    assert [s[-10:] for s in statements(text)] == [' "memory")', '"" ::: "m0")'[-10:]] and len(SOURCES) > 8
