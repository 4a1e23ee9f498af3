"""The barriers that the softmax warps of tree_q4_wide_kernel share have no time limit, so
no warp may reach one that another passes by.  A wait on an mbarrier has a limit and can
run out in one warp only: what hangs on its outcome must not decide over a barrier, unless
all eight warps have agreed on it (any_of).  Read from the source: a case that makes it
happen would hang a GPU."""
import os
import re

SOURCE = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))),
                      "alpacca_open_sourced_by_jt_b200", "csrc", "tree_q4_wide.cu")
BARRIER = re.compile(r"\bmeet\(\)|\bany_of\(|bar\.sync")
OWN = re.compile(r"\b(dead|alive|ok|arrived\(|wait\()")  # a warp's own outcome
LEAVE = re.compile(r"\b(break|return|continue);")


def softmax_section():
    text = open(SOURCE).read()
    text = re.sub(r"//[^\n]*", "", text)
    start = text.index("} else if (warp < 8) {")
    body = text[start + 2:text.index("tc_fence_before();\n  __syncthreads();\n  if (warp == kQWIssue)")]
    return re.sub(r"(auto (meet|any_of|wait) = .*?\n    \};|auto meet = .*?\};\n)", "", body, flags=re.S)


def statements(body):
    """(statement, headers of the blocks around it), a line at a time."""
    stack, found = [], []
    for line in body.splitlines():
        line = line.strip()
        if line.startswith("}"):
            stack.pop()
            line = line[1:].strip()
        if not line:
            continue
        found.append((line, [h for h in stack if h]))
        for ch in line:
            if ch == "{":
                stack.append(line)
            elif ch == "}":
                stack.pop()
    return found


def test_no_barrier_hangs_on_one_warps_wait():
    found = statements(softmax_section())
    barriers = [(s, heads) for s, heads in found if BARRIER.search(s)]
    assert len(barriers) >= 8
    for s, heads in barriers:
        for h in heads:
            assert not OWN.search(h), (s, h)
        assert not (s.startswith("if") and OWN.search(s) and not s.startswith("if (any_of(")), s


def test_the_loop_over_items_is_left_by_all_warps_or_none():
    exits = [(s, heads) for s, heads in statements(softmax_section())
             if LEAVE.search(s) and sum(h.startswith(("while", "for")) for h in heads) == 1
             and not any(h.startswith("auto") for h in heads)]
    assert len(exits) >= 2
    for s, heads in exits:
        assert s.startswith(("if (any_of(", "if (end)")), s
