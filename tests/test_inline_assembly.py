"""Registers that an inline assembly statement writes by name stand in its clobber list: the compiler may keep values there."""
import re
from pathlib import Path

import pytest

CSRC = Path(__file__).resolve().parent.parent / "whisperdrz_amd" / "csrc"
STATEMENT = re.compile(r"\basm\s*(?:volatile\s*)?\((.*?)\);", re.S)
WRITES = re.compile(r"\bs_\w+\s+(m0|vcc|s\d+)\b\s*,")  # the destination comes first


@pytest.mark.parametrize("path", sorted(p for p in CSRC.iterdir() if p.suffix in (".hip", ".h", ".cpp")), ids=lambda p: p.name)
def test_written_registers_are_declared(path):
    for body in STATEMENT.findall(path.read_text()):
        strings = re.findall(r'"((?:[^"\\]|\\.)*)"', body)
        for register in set(WRITES.findall(" ".join(strings[:1]))):
            assert register in strings[1:], f"{register} in {body[:80]}"
