"""The Swift wrappers of the head-norm, cache and paged-attention calls check their
tensors before the C call, which sees pointers without extents.  There is no Swift
toolchain here, so the check is textual: every tensor that a function or an initialiser
takes is asked for its shape and type, and no C call comes before that."""
import os
import re

HERE = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "minirun-app_amd", "swift", "Sources", "HIPBridge")


def functions():
    """(name, [(parameter, type)], body) of every function and throwing initialiser."""
    text = re.sub(r"//.*", "", open(os.path.join(HERE, "KVAttention.swift")).read())
    found = []
    for m in re.finditer(r"\n( *)(?:public |private )?(?:func (\w+)|(init))\((.*?)\)( throws)?(?: -> \w+)? \{\n(.*?)\n\1\}\n", text,
                         flags=re.S):
        params = re.findall(r"(?:\w+ )?(\w+): (?:inout )?(\w+)\??", m.group(4))
        found.append((m.group(2) or m.group(3), params, m.group(6)))
    return found


def test_every_tensor_is_checked():
    seen, missing = 0, []
    for name, params, body in functions():
        if name == "init" and "throw" not in body:  # a plain record: its user checks it
            continue
        passed_on = re.search(r"= try (headNormArgs|attentionArgs)\(", body)  # the shared part checks them
        for param, kind in params:
            if kind != "HIPTensor":
                continue
            seen += 1
            if not passed_on and not re.search(rf"\b{param}\??\.(needHeads|needRows|needWhole|needPages)\(", body):
                missing.append((name, param))
    assert seen > 20 and not missing, missing


def test_the_records_are_checked_by_their_users():
    bodies = {name: body for name, _, body in functions()}
    for part in ("cos", "sin", "positions"):
        assert re.search(rf"\b{part}\??\.needWhole\(", bodies["needRotation"]), part
    for part, how in (("x", "needHeads"), ("out", "needHeads"), ("dOut", "needHeads"), ("weight", "needWhole"), ("dWeight", "needWhole")):
        assert re.search(rf"\b{part}\??\.{how}\(", bodies["needRows"]), part
    for name in ("headNormArgs", "hipKVAppend"):
        assert re.search(r"try rotation\.needRotation\(tokens\)", bodies[name]), name
    for rows in ("q", "k"):
        assert re.search(rf"try {rows}\.needRows\(", bodies["headNormArgs"]), rows


def test_checks_come_before_the_call():
    for name, _, body in functions():
        call = re.search(r"\bmr_(head_norm_rope\w*|kv_append|kv_attention\w*)\(", body)
        if call:
            after = body[call.end():]
            assert not re.search(r"\.need\w+\(", after), name
