"""Inline assembly names what it writes besides its operands: the compiler may otherwise keep a value there."""
import re
from pathlib import Path

CSRC = Path(__file__).resolve().parent.parent / "granite_amd" / "csrc"


def statements():
    for path in sorted(CSRC.glob("*.h*")):
        for m in re.finditer(r"asm\s+volatile\s*\((.*?)\);", path.read_text(), re.S):
            yield path.name, m.group(1)


def test_m0_is_named_where_it_is_written():
    writers = [(name, text) for name, text in statements() if re.search(r"s_mov_b32 m0\b", text)]
    assert {name for name, _ in writers} >= {"decode_ex_dma.hip", "prefill_dma.hip"}
    for name, text in writers:
        assert re.search(r':[^:]*"m0"[^:]*$', text), f"{name}: {text}"
