"""The Swift wrappers of the MXFP4 and routing calls check their tensors before the
C call, which sees pointers without extents: a shape that does not fit would be a
read or a write past a buffer.  There is no Swift toolchain here, so the check is
textual: every tensor, weight and order that a function takes is asked for its
shape and type before the first C call that it makes."""
import os
import re

import pytest

HERE = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "minirun-app_amd", "swift", "Sources", "HIPBridge")
CHECKS = {"HIPTensor": r"need(Rows|Whole)\(", "HIPExpertOrder": r"needOrder\(\)", "HIPMXFP4Weights": r"(needMatrix\(|experts\b)"}


def functions(name):
    """(name, [(parameter, type)], body) of every public function of a file."""
    text = re.sub(r"//.*", "", open(os.path.join(HERE, name)).read())
    found = []
    for m in re.finditer(r"\n(?:public |private )?func (\w+)\((.*?)\)(?: throws)?(?: -> \w+)? \{\n(.*?)\n\}\n", text, flags=re.S):
        params = re.findall(r"(?:\w+ )?(\w+): (?:inout )?(\w+)\??", m.group(2))
        found.append((m.group(1), params, m.group(3)))
    return found


@pytest.mark.parametrize("name", ["Experts.swift", "MXFP4Weights.swift"])
def test_every_tensor_is_checked_before_the_call(name):
    missing, seen = [], 0
    for func, params, body in functions(name):
        call = re.search(r"\b(mr_(?!mxfp4_expert_args)\w+|hipExpertMM)\(", body)
        if not call:
            continue
        before = body[:call.start()]
        for param, kind in params:
            if kind not in CHECKS:
                continue
            seen += 1
            # the shared end of the expert products checks what it is given
            if call.group(1) == "hipExpertMM" and (param, kind) in (("y", "HIPTensor"), ("w", "HIPMXFP4Weights")):
                continue
            if func == "hipExpertMM" and kind == "HIPExpertOrder":
                continue
            name_of = "(out|all)" if func == "hipMXFP4Dequantize" and param == "out" else param
            if not re.search(rf"\b{name_of}\??\.{CHECKS[kind]}", before):
                missing.append(f"{func}: {param}")
    assert seen > 8 and not missing, missing


def test_the_weights_and_the_order_have_no_gaps():
    weights = open(os.path.join(HERE, "MXFP4Weights.swift")).read()
    for part in ("packed", "scales"):
        assert re.search(rf"try {part}\.needWhole\(", weights[:weights.index("desc = mr_mxfp4_matrix")]), part
    order = open(os.path.join(HERE, "Experts.swift")).read()
    for part in ("offsets", "pairOfRow", "rowOfPair"):
        assert re.search(rf"try {part}\.needWhole\(\"{part}\", .*dtype: MR_I32\)", order), part
