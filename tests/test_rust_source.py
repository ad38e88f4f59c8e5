"""The Rust crate's sources as text (there is no Rust toolchain in this image): what any Rust
compiler refuses before it looks at a declaration."""
import os
import re

import pytest

CRATE = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "dial-8b-orin_b200", "dial-cuda")


def code_of(text):
    """The source without comments and literals (each a blank or an empty literal), lines kept."""
    out, i = [], 0
    while i < len(text):
        if text.startswith("//", i):
            j = text.find("\n", i)
            j = len(text) if j < 0 else j
        elif text.startswith("/*", i):
            depth, j = 1, i + 2
            while depth and j < len(text):
                depth += text.startswith("/*", j) - text.startswith("*/", j)
                j += 2 if text[j:j + 2] in ("/*", "*/") else 1
            out.append("\n" * text.count("\n", i, j))
        elif text[i] == '"':
            j = i + 1
            while text[j] != '"':
                j += 2 if text[j] == "\\" else 1
            j += 1
            out.append('""' + "\n" * text.count("\n", i, j))
        elif re.match(r"'(\\.[^']*|[^\\'])'", text[i:]):
            j = i + re.match(r"'(\\.[^']*|[^\\'])'", text[i:]).end()
            out.append("' '")
        else:
            out.append(text[i])
            j = i + 1
        i = j
    return "".join(out)


def faults(text):
    lines, code = text.split("\n"), code_of(text).split("\n")
    found, started = [], False
    for n, (line, bare) in enumerate(zip(lines, code), 1):
        inner = line.lstrip().startswith("//!") or bare.lstrip().startswith("#![")
        if inner and started:
            found.append((n, "an inner comment or attribute behind the first item"))
        started = started or (bool(bare.strip()) and not inner)
        found += [(n, f"{c!r} in code") for c in "`\\$" if c in bare and "macro_rules" not in text]
    for a, b in ("()", "[]", "{}"):
        if "\n".join(code).count(a) != "\n".join(code).count(b):
            found.append((0, f"unequal numbers of {a} and {b}"))
    lines = [l.strip() for l in lines]
    for n, (line, after) in enumerate(zip(lines, lines[1:] + [""]), 1):
        if line.startswith("///") and not after:
            found.append((n, "a comment on nothing"))
    return found


@pytest.mark.parametrize("file", ["src/lib.rs", "build.rs"])
def test_sources_hold_no_fault_that_text_shows(file):
    assert faults(open(os.path.join(CRATE, file)).read()) == []


def test_every_type_that_is_used_is_declared():
    code = code_of(open(os.path.join(CRATE, "src", "lib.rs")).read())
    declared = set(re.findall(r"(?:pub type|pub struct|pub enum|pub union) (\w+)", code))
    used = set(re.findall(r"(?::|->|\*const|\*mut|&)\s*(dial_\w+)", code))
    assert used and used <= declared, used - declared


def test_faults_are_found():
    good = "//! a `b`\n//! c\n\n#![allow(x)]\n\nuse a::b;\n/// d `e`\npub fn f(x: &'static str) -> char { '`'; \"`\" /* ` */ }\n"
    assert faults(good) == []
    for bad in (good.replace("//! c", "//! /// c\nstruct S;"), good.replace("//! c", "c` d"), good + "#![deny(y)]\n", good + "//! g\n",
                good + "}\n", good + "/// on nothing\n"):
        assert faults(bad), bad
