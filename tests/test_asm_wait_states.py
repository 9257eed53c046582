"""Inline assembly keeps the wait states that the compiler does not add inside an
asm string (checked in the sources; no GPU needed)."""

import os
import re

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def _asm_strings():
    for top in ("zookeeper_amd/csrc", "tools"):
        for folder, _, names in os.walk(os.path.join(ROOT, top)):
            for name in names:
                if name.endswith((".hip", ".h", ".cpp")):
                    path = os.path.join(folder, name)
                    with open(path) as f:
                        text = f.read()
                    for m in re.finditer(r"\basm\s*(?:volatile)?\s*\(((?:\s*\"(?:[^\"\\]|\\.)*\")+)",
                                         text):
                        body = "".join(re.findall(r"\"((?:[^\"\\]|\\.)*)\"", m.group(1)))
                        yield path, [i.strip() for i in re.split(r"\\n|\\t|;", body) if i.strip()]


def _unsafe(instructions):
    """Loads to LDS right behind a scalar write of M0."""
    return [b for a, b in zip(instructions, instructions[1:])
            if re.match(r"s_\w+\s+m0\b", a)
            and re.match(r"(global|buffer|scratch)_load\w*", b) and "lds" in b]


def test_the_check_itself():
    assert _unsafe(["s_mov_b32 m0, %1", "global_load_lds_dwordx4 %0, off"])
    assert not _unsafe(["s_mov_b32 m0, %1", "s_nop 0", "global_load_lds_dwordx4 %0, off"])


def test_loads_to_lds_wait_for_m0():
    """A load to LDS takes its LDS address from M0 and needs one wait state behind
    a scalar write of it; without one it may use the address before."""
    seen, bad = 0, []
    for path, instructions in _asm_strings():
        seen += any("load_lds" in i for i in instructions)
        bad += [(os.path.relpath(path, ROOT), b) for b in _unsafe(instructions)]
    assert seen >= 4 and not bad, bad
