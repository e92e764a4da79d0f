"""The expert-layer section of the Julia extension, as text (no Julia toolchain
exists here): which value types it takes, and that a call checks the type and
size of every buffer whose address it hands to the library."""
import os
import re

import pytest

JL = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "ext", "B200Ext", "B200Ext.jl")
# the buffers of each call but the ones that give it its extents
FIT = {
    "combine!": {"y": "(N, T)", "g": "(k, T)"},
    "combine_backward!": {"dz": "(N, S)", "dg": "(k, T)", "dy": "(N, T)", "g": "(k, T)"},
    "grouped_mm!": {"y": "(N, S)", "x": "(K, T)", "rowptr": "E", "rows": "(S,)", "bias": "(N, E)",
                    "res": "(N, S)", "z": "(N, S)"},
    "grouped_mm_wgrad!": {"dz": "(N, S)", "x": "(K, T)", "rowptr": "E", "rows": "(S,)"},
    "act_backward!": {"z": "(N, S)", "dz": "(N, S)", "db": "(N, E)", "rowptr": "E"},
}


def source():
    return open(JL).read()


def test_bfloat16_is_the_only_16_bit_type():
    rule = re.search(r"^_vt\(::Type\{T\}\).*?(?=^\w|^#)", source(), re.S | re.M).group(0)
    assert "nameof(T) === :BFloat16" in rule and "sizeof" not in rule


@pytest.mark.parametrize("name", sorted(FIT))
def test_every_buffer_of_a_call_is_checked(name):
    text = re.search(r"^function " + re.escape(name) + r"\((.*?)^end$", source(), re.S | re.M).group(1)
    before = text[:text.index("ccall(")]       # sizes are looked at before the library is
    checked = dict(re.findall(r"_(?:is|maybe)\((\w+), (?:V|Int32|Float32), (\([^()]*\)), \"", before))
    checked |= dict(re.findall(r"_groups\((\w+), (E)\)", before))
    assert checked == FIT[name]
