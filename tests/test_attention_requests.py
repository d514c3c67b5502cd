"""The buffer loads of the attention over the pages (csrc/attn_attend.hip, attn_tile.hip) against the range check of
a raw buffer (lane offset >= size - scalar offset, which wraps around below 0): an entry of the block table that
names no page has a buffer of no bytes, so every scalar offset into a page has to be 0 there."""

import re

import pytest

from test_scan_requests import CSRC, _arguments

LOADS = r"\b(buf_ld\w*|__builtin_amdgcn_raw_buffer_load_b\d+|fetch)\s*(?:<[^<>()]*>)?\s*\("


def _text(name):
    return re.sub(r"//.*", "", (CSRC / name).read_text())


def _calls(text):
    """(name, arguments) of every load from a buffer, but for the definitions of the helpers."""
    out = []
    for m in re.finditer(LOADS, text):
        args = _arguments(text, m.end() - 1)
        if not any(re.match(r"(__amdgpu_buffer_rsrc_t|int|const) ", a) for a in args):
            out.append((m.group(1), args))
    return out


def _defined_by_place(text, name):
    """Every definition of the scalar is a call of place()."""
    found = [text[m.end():].split(";")[0] for m in re.finditer(rf"\b{name} = ", text)]
    found = [re.split(r",\s*\w+ = ", x)[0].strip() for x in found]
    return bool(found) and all(re.match(r"(p\.)?place\(", x) for x in found)


def test_scalar_offsets_of_the_kernel_for_few_rows():
    text = _text("attn_attend.hip")
    calls = _calls(text)
    assert len(calls) == 10, calls
    for name, args in calls:
        assert _defined_by_place(text, args[2]), (name, args)
        # page g's offset for page g's buffer
        page = re.search(r"page<D>\(([^,]+),", args[0])
        of = [m for m in re.findall(rf"\b{args[2]} = p\.place\(([^,]+),", text)]
        assert of and (page is None or page.group(1) in of), (name, args, of)
    assert re.search(r"int place\(int g, int offset\) const \{ return shown >> g & 1 \? offset : 0; \}", text)


def test_scalar_offsets_of_the_kernel_for_many_rows():
    text = _text("attn_tile.hip")
    calls = [args for name, args in _calls(text) if name == "fetch"]
    assert len(calls) == 2
    for args in calls:
        assert args[2].startswith("place(") and args[4].startswith("place("), args
    # and fetch passes its scalars on as they are
    inner = [args for name, args in _calls(text) if name != "fetch"]
    assert len(inner) == 3 and all(args[2] in ("code0", "scale0") for args in inner), inner
    assert "const auto place = [&](int offset) { return ok ? offset : 0; };" in text


@pytest.mark.parametrize("name", ["attn_attend.hip", "attn_tile.hip"])
def test_hidden_pages_have_no_bytes(name):
    assert re.search(r"buf_rsrc\([^;]*\? kv4_page_bytes\(size, D\) : 0\)", _text(name))
