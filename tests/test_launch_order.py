"""The order of a kernel's wait and its release of dependents, in the sources.

A kernel launched as a programmatic dependent may read early what its
predecessor did not write (hx_decode_attention under HX_KV_OVERLAP_LAUNCH does).
That is sound only if everything before the predecessor has finished by then,
i.e. if the predecessor waits (griddepcontrol.wait) before it releases its
dependents.  A race of this kind shows on a GPU now and then at best, so the
sources are read instead.
"""
import os
import re

import pytest

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "hxinfer_b200", "csrc")


def kernels():
    """(name, body without comments) of every __global__ function."""
    for name in sorted(os.listdir(CSRC)):
        if not name.endswith(".cu"):
            continue
        with open(os.path.join(CSRC, name)) as f:
            text = re.sub(r"//[^\n]*", "", f.read())
        for m in re.finditer(r"__global__\s+void\s+(?:__launch_bounds__\((?:[^()]|\([^()]*\))*\)\s*)?(\w+)\s*\(", text):
            at = text.index("{", m.end())
            depth, end = 0, at
            while True:
                depth += {"{": 1, "}": -1}.get(text[end], 0)
                end += 1
                if depth == 0:
                    break
            yield m.group(1), text[at:end]


RELEASING = {name: body for name, body in kernels() if "pdl_trigger()" in body}

# A combine kernel is itself a dependent of the attention grid, which releases it
# after its wait: what lies before that grid is complete when it starts.
COMBINES = {"decode_combine_kernel", "shared_combine_kernel"}


def test_all_kernels_are_found():
    assert len(RELEASING) >= 12 and COMBINES < set(RELEASING)


@pytest.mark.parametrize("name", sorted(set(RELEASING) - COMBINES))
def test_waits_before_it_releases(name):
    """All work is behind the wait that the release follows: the first of
    either, in the order of the text.  (decode_attention_kernel's other waits
    are its producer's and the one for empty rows, which release nothing.)"""
    body = RELEASING[name]
    assert -1 < body.find("pdl_wait()") < body.find("pdl_trigger()"), f"{name} releases dependents before its own wait"
    before = body[:body.find("pdl_trigger()")].rstrip()
    assert before.endswith("pdl_wait();"), f"{name}: the release does not follow a wait"
