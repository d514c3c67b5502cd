"""Inline assembly names the registers that it writes beside its outputs, so that the compiler keeps nothing in them."""

import re
from pathlib import Path

CSRC = Path(__file__).resolve().parent.parent / "cq-pretrain_amd" / "csrc"


def statements(text):
    """The asm statements of a source, with the macros of their own files in them spelled out."""
    macros = dict(re.findall(r"#define (\w+)\([^)]*\)((?:.*\\\n)*.*)", text))
    for m in re.finditer(r"\basm(?: volatile)?\(", text):
        depth, end = 1, m.end()
        while depth:
            depth += {"(": 1, ")": -1}.get(text[end], 0)
            end += 1
        body = text[m.end():end - 1]
        yield body + " ".join(macros[n] for n in macros if n + "(" in body)


def test_m0_is_named_where_it_is_written():
    found = 0
    for path in sorted(CSRC.glob("*.h*")):
        for body in statements(path.read_text()):
            if re.search(r"(s_\w+_b32|s_movk_i32) m0\b", body):
                found += 1
                assert '"m0"' in body.rsplit(":", 1)[1], (path.name, body)
    assert found >= 3
