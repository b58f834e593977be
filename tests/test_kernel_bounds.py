"""Bounds of kernels' loads that no run can show, by their sources: an allocation has
room behind it, so that a read past a tensor's end gives the same answers."""
import os
import re

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))),
                    "qwen2.5-jetson-inference_amd", "csrc")


def arguments(text, at):
    """Of the call whose opening bracket is at `at`."""
    found, depth, begin = [], 0, at + 1
    for i in range(at, len(text)):
        depth += (text[i] in "([{") - (text[i] in ")]}")
        if depth == 0 or (depth == 1 and text[i] == ","):
            found.append(text[begin:i].strip())
            begin = i + 1
        if depth == 0:
            return found
    raise ValueError("no closing bracket")


def test_a_rows_pieces_are_bounded_by_the_vector_offset():
    """A sampling thread asks for pieces past its row's end and counts on zeros there.  The
    bounds check of a buffer load is certain for the vector offset alone, so the piece's
    place, which may be past the end as a whole, is none of the scalar offset's."""
    text = open(os.path.join(CSRC, "sample.hip")).read()
    calls = [m.end() - 1 for m in re.finditer(r"raw_(?:ptr_)?buffer_load\w*\(", text)]
    assert calls
    for at in calls:
        _, vector, scalar, _ = arguments(text, at)
        assert scalar == "0" and "threadIdx.x" in vector and "first" in vector


def test_no_lds_address_is_made_from_a_number():
    """The bins of sampling's counts are reached from the object that they lie in, wherever
    the compiler puts that, and not as the first bytes of the workgroup's LDS."""
    text = open(os.path.join(CSRC, "sample.hip")).read()
    names = re.findall(r"address_space\(3\)\)\)[\w ]*?(\w+);", text)
    assert names
    for name in names:
        cast = rf"(\({name}\s*\*\)|reinterpret_cast<{name}\s*\*>\()\s*"
        assert not re.search(cast + r"(static_cast<uintptr_t>|\(uintptr_t\)|\d)", text)
