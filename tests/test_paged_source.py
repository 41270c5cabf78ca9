"""Rules of the tcgen05 attention over a paged cache that no run can show to be kept, because no input makes one of its bounded waits
run out: what a block has under way when a wait gave up, and what its rows are then."""
import os
import re

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "neuralnet.cpp_b200", "csrc")


def _function(path, head):
    """The body of the function whose definition begins with `head`, without comments."""
    src = re.sub(r"//[^\n]*", "", open(os.path.join(CSRC, path)).read())
    start = src.index("{", src.index(head))
    depth, end = 1, start + 1
    while depth:
        depth += {"{": 1, "}": -1}.get(src[end], 0)
        end += 1
    return src[start:end]


def _roles():
    """The code of the loading warp, of the issuing warp, and what all threads do behind the roles."""
    body = _function("paged_attention.cu", "void attend_tc(")
    load, issue, work = (body.index(m) for m in ("if (warp == 0) {", "} else if (warp == 1) {", "const int quad = warp & 3"))
    end = body.index("tc_fence_before();\n    __syncthreads();", work)
    return body[load:issue], body[issue:work], body[end:]


def test_loads_under_way_are_waited_for_when_a_wait_gave_up():
    """A load that lands after its block has ended writes into the next block's shared memory."""
    load, _, _ = _roles()
    for place, count in (("k_full", "k_loads"), ("v_full", "v_loads")):
        issued = load.index(f"{place} + 8 * st, j * 64")
        assert issued < load.index(f"{count} = i + 1") < load.index(f"drain({place}")      # counted once they are issued
        assert re.search(rf"for \(int i = max\(0, {count} - ST\); i < {count}; \+\+i\) drain\({place}", load)
    tail = load[load.index("if (lane == 0)", load.rindex("tma_load_2d")):]
    assert "abort" not in tail and "ok" not in tail


def test_products_under_way_are_waited_for_before_their_tmem_is_freed():
    _, issue, end = _roles()
    assert re.search(r"umma_commit\((\w+)\);\s*drain\(\1, 0\);\s*\}\s*\} else \{\s*$", issue)           # whatever the loop before came to
    assert "tcgen05.dealloc" in end


def test_a_drain_does_not_end_because_another_wait_gave_up():
    body = _function("tc_ptx.cuh", "bool mbar_drain(")
    assert "abort" not in body and "clock64() - t0 >" in body


def test_rows_of_a_block_that_gave_up_are_nan():
    """What such a block has not written, or only in part, must not reach the join as numbers of an earlier call."""
    _, _, end = _roles()
    written = re.search(r"if \(\*abort_flag\)\s*for \([^{}]*k\.rows[^{}]*leave<bf16>\(a, k, dk,[^{}]*make_float4\(NAN, NAN, NAN, NAN\), -INFINITY, NAN\);", end)
    assert written and end.index("__syncthreads()") < written.start()
