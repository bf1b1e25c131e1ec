"""How the token kernels order what wavefronts exchange through shared memory, read from their source: a race shows
on no machine for sure."""
import os
import re

import pytest

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "dciknn_cuda_amd", "csrc")


def body_of(source, kernel):
    """The text of a function from its name to its closing brace, without comments."""
    with open(os.path.join(CSRC, source)) as f:
        text = re.sub(r"//[^\n]*", "", f.read())
    at = text.index("{", re.search(r"\b%s\([^;]*?\) *\{" % kernel, text).start())
    depth = 0
    for end in range(at, len(text)):
        depth += {"{": 1, "}": -1}.get(text[end], 0)
        if depth == 0:
            return text[at:end + 1]
    raise AssertionError("no end of " + kernel)


def uses(part, name):
    """(reads, writes) of a shared array in a piece of source."""
    writes = re.findall(r"\b%s(?:\[[^=;]*?\])? *=(?!=)" % name, part)
    return len(re.findall(r"\b%s\b" % name, part)) - len(writes), len(writes)


def test_between_two_barriers_a_shared_array_is_read_or_written():
    """The loop over rows of distill_rows_kernel: its wavefronts are as far apart as its barriers let them be, so what
    one of them reads between two of these no other may write there."""
    body = body_of("logits.hip", "distill_rows_kernel")
    shared = re.findall(r"\b(s_\w+)", " ".join(re.findall(r"__shared__ ([^;]*);", body)))
    assert len(shared) >= 6
    head, loop = body.split("while (true) {")
    # (nothing is exchanged ahead of the loop)
    assert not any(re.search(r"\b%s\b" % name, re.sub(r"__shared__ [^;]*;", "", head)) for name in shared)
    parts = loop.split("__syncthreads();")
    assert len(parts) >= 4
    parts[0] = parts.pop() + parts[0]                   # the last part goes on into the next round's first
    for i, part in enumerate(parts):
        for name in shared:
            reads, writes = uses(part, name)
            assert not (reads and writes), "%s is read and written in part %d of the loop" % (name, i)
    for name in shared:
        assert any(uses(part, name)[0] for part in parts) and any(uses(part, name)[1] for part in parts), name


@pytest.mark.parametrize("kernel", ["chunk_kernel", "bucket_kernel", "few_kernel"])
def test_counts_that_lanes_hand_on_are_ordered(kernel):
    """One lane stores a count that other lanes of its wavefront read a round later: between the two stands a fence, which
    keeps the compiler from moving or remembering one over the other."""
    body = body_of("embed.hip", kernel)
    stores = list(re.finditer(r"lanes_below\(same\) == 0\) (?:mine|s_count\[wave\])\[[^;]*\] = [^;]*;", body))
    assert len(stores) == 1
    rest = body[stores[0].end():]
    assert re.match(r"[^;]*?(?:w\.tokens[^;]*;\s*)?\}\s*wave_fence\(\);", rest, re.S), rest[:200]
