"""Every statement of inline assembly in the kernels names what it changes besides its outputs: the registers m0, scc, vcc and exec, which
no operand can stand for, belong to its clobbers, as memory does where a load or a store is written out."""
import re
from pathlib import Path

import pytest

CSRC = Path(__file__).resolve().parent.parent / "pitch_amd" / "csrc"
FILES = sorted(p for p in CSRC.iterdir() if p.suffix in (".hip", ".h", ".cpp"))


def _statements(text):
    """(line, instructions, the rest) of each asm statement."""
    for m in re.finditer(r"\basm\b(?:\s+volatile)?\s*\(", text):
        depth, i, quoted = 1, m.end(), False
        while depth:
            c = text[i]
            if quoted:
                i += c == "\\"
                quoted = c != '"'
            elif c == '"':
                quoted = True
            else:
                depth += (c == "(") - (c == ")")
            i += 1
        body = text[m.end():i - 1]
        lead = re.match(r'\s*(?:"(?:[^"\\]|\\.)*"\s*)*', body).group()
        code = "".join(re.findall(r'"((?:[^"\\]|\\.)*)"', lead))
        yield text.count("\n", 0, m.start()) + 1, [s.strip() for s in re.split(r"\\n|\\t", code) if s.strip()], body[len(lead):]


def _changes(instruction):
    """What an instruction changes that no operand stands for."""
    name, _, operands = instruction.partition(" ")
    target = operands.split(",")[0].strip()
    found = {r for r in ("m0", "vcc", "exec") if target == r or target.startswith(r + "_")}
    if re.match(r"s_(cmp|cmpk|bitcmp|add|sub|addc|subb|min|max|and|or|xor|andn2|not|lshl|lshr|ashr|bfe|bcnt)", name):
        found.add("scc")
    if re.match(r"(buffer|global|flat|ds)_(load|store|read|write|atomic)", name):
        found.add("memory")
    return found


def _faults(text):
    return [f"line {line}: {i!r} changes {r}" for line, code, rest in _statements(text) for i in code for r in sorted(_changes(i))
            if f'"{r}"' not in rest.split(":")[-1]]


@pytest.mark.parametrize("path", FILES, ids=lambda p: p.name)
def test_statements_name_what_they_change(path):
    assert _faults(path.read_text()) == []


def test_a_statement_that_does_not_is_found():
    asm = 'asm volatile("s_mov_b32 m0, %0\\n\\ts_nop 0\\n\\tds_read_b32 %1, %2" : "=v"(x) : "s"(y), "v"(f(z)) : {});'
    assert _faults(asm.format('"memory", "m0"')) == []
    assert len(_faults(asm.format('"memory"'))) == 1 and len(_faults(asm.format('"m0"'))) == 1
    assert len(_faults('asm("s_cmp_eq_u64 %0, 0" :: "s"(go) : "memory");')) == 1
