"""CPU tier: the Julia bindings of the rotation, the append and the paged attention, read as text
(their own test set, which calls them with mixed types, needs Julia): before the foreign call each
compares the element types of all its tensors, since the C descriptor holds one type for all, and
asks for 64-bit frequencies."""
import re
from pathlib import Path

import pytest

SRC = (Path(__file__).resolve().parents[1] / "lava.jl_b200" / "LavaB200" / "src" / "LavaB200.jl").read_text()


def body(name):
    """The function's text up to its foreign call."""
    text = SRC[SRC.index(f"\nfunction {name}("):]
    return text[:text.index("ccall(")]


@pytest.mark.parametrize("name,tensors", [
    ("rope!", {"Q", "Qo", "K", "Ko"}),
    ("kv_append!", {"Kc", "Vc", "K", "V", "Q", "Qo"}),
    ("attention_paged!", {"O", "Q", "Kc", "Vc"}),
])
def test_all_tensors_share_a_type(name, tensors):
    m = re.search(r'same_eltype\("%s", eltype\((\w+)\), ([\w, ]+)\)' % re.escape(name), body(name))
    assert m, "no comparison of the element types"
    assert {m[1], *m[2].split(", ")} == tensors


@pytest.mark.parametrize("name", ["rope!", "kv_append!"])
def test_frequencies_are_64_bit(name):
    assert "eltype(freqs) === Float64" in body(name)
