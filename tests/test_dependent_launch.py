"""Kernels that start before their predecessor in the stream has ended (those that call griddep_wait) may not tell the
compiler that what they read is read-only for their lifetime: the predecessor may still be writing it."""
import glob
import os
import re

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "nvidia-x-gpu-mode-kernels_b200", "csrc")


def _block(text, at, opening, closing):
    """The text from the bracket at or after `at` up to the one that closes it, and where it ends."""
    start = text.index(opening, at)
    depth = 0
    for i in range(start, len(text)):
        depth += (text[i] == opening) - (text[i] == closing)
        if depth == 0:
            return text[start:i + 1], i + 1
    raise AssertionError("unbalanced source")


def _kernels():
    for path in sorted(glob.glob(os.path.join(CSRC, "*.cu*"))):
        text = re.sub(r"//[^\n]*", "", open(path).read())
        for m in re.finditer(r"__global__\s+void\s+(?:__launch_bounds__\s*\()?", text):
            at = m.end()
            if m.group().endswith("("):
                at = _block(text, m.end() - 1, "(", ")")[1]
            name = re.match(r"\s*(\w+)", text[at:]).group(1)
            params, at = _block(text, at, "(", ")")
            body, _ = _block(text, at, "{", "}")
            yield os.path.basename(path), name, params, body


def test_no_read_only_promises_before_the_wait():
    waiting = 0
    for path, name, params, body in _kernels():
        if "griddep_wait" not in body and "griddepcontrol.wait" not in body:
            continue
        waiting += 1
        assert "__restrict__" not in params, f"{path}: {name}"
        assert "__ldg(" not in body and "ld.global.nc" not in body, f"{path}: {name}"
    assert waiting >= 6
