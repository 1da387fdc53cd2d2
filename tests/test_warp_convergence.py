"""The attention kernels' source, read for instructions that a whole warp has to execute together (tcgen05.ld, .st and
.wait, named barriers, setmaxnreg: all .sync.aligned) behind a branch that lanes take apart, without a __syncwarp()
in between.  Where the lanes meet again is the compiler's choice otherwise."""
import os
import re

import pytest

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "fuse_b200", "csrc")
# what differs between the lanes of a warp, in these kernels' own names
LANE = r"\b(lane|mine|there|largest|lse|threadIdx|row)\b"
ALIGNED = r"\b(tmem_ld\w*|tmem_st\w*|tmem_wait\w*|tmem_alloc|tmem_dealloc|tmem_relinquish|named_bar_sync|setmaxnreg\w*|__syncthreads)\b"
HELPERS = ("zero_rows", "warp_arrive")


def closing(text, at):
    """The index behind the bracket that closes the one at `at`."""
    pairs, depth = {"(": ")", "{": "}"}, 0
    for i in range(at, len(text)):
        if text[i] == text[at]:
            depth += 1
        elif text[i] == pairs[text[at]]:
            depth -= 1
            if depth == 0:
                return i + 1
    raise AssertionError("unbalanced source")


def body_after(text, at):
    """(start, end) of the statement from `at` on: a block, a single statement, or a loop's or branch's own body."""
    while text[at].isspace():
        at += 1
    if text[at] == "{":
        return at, closing(text, at)
    head = re.compile(r"(for|if)\s*(constexpr\s*)?\(").match(text, at)
    if head:
        end = body_after(text, closing(text, head.end() - 1))[1]
        behind = re.compile(r"\s*else\b").match(text, end)
        return at, body_after(text, behind.end())[1] if behind and head.group(1) == "if" else end
    return at, text.index(";", at) + 1


def without_comments(text):
    text = re.sub(r"//[^\n]*", "", re.sub(r"/\*.*?\*/", "", text, flags=re.S))
    return re.sub(r"^\s*#[^\n]*", "", text, flags=re.M)


def events(text, helpers):
    """What is met in the order of execution: "apart" for a lane-dependent branch (before and behind what it holds), "together",
    the aligned instructions, and for an if with else, the tuple of its arms.  A loop's body comes twice: its end is
    followed by its beginning."""
    token = re.compile(r"\b(for|if)\s*(constexpr\s*)?\(|\b__syncwarp\(|" + ALIGNED + r"\s*(<\w+>)?\s*\(|\b(" + "|".join(HELPERS) + r")\b\s*(<\w+>)?\s*\(")
    out, at = [], 0
    while match := token.search(text, at):
        opened, at = match.end() - 1, match.end()
        if match.group(1):
            head = closing(text, opened)
            start, at = body_after(text, head)
            inner = events(text[start:at], helpers)
            if match.group(1) == "for":
                out += inner * 2
                continue
            if behind := re.compile(r"\s*else\b").match(text, at):
                start, at = body_after(text, behind.end())
                inner = [(inner, events(text[start:at], helpers))]
            condition = re.sub(r"__(any|all)_sync\([^()]*\)", "", text[opened:head])  # a vote is the same for all lanes
            out += ["apart", *inner, "apart"] if re.search(LANE, condition) else inner
        elif match.group(0).startswith("__syncwarp"):
            out.append("together")
        elif match.group(5):
            out += helpers.get(match.group(5), [])
        else:
            out.append(match.group(3))
    return out


def function_body(text, name):
    """The body of the (only) definition of `name`."""
    for match in re.finditer(r"\b" + name + r"\s*\(", text):
        end = closing(text, match.end() - 1)
        if text[end:].lstrip().startswith("{"):
            start = text.index("{", end)
            return text[start:closing(text, start)]
    return None


def walk(sequence, apart, found):
    for event in sequence:
        if isinstance(event, tuple):
            apart = any([walk(arm, apart, found) for arm in event])
        elif event in ("apart", "together"):
            apart = event == "apart"
        elif apart:
            found.append(event)
    return apart


def faults(sequence):
    found = []
    walk(sequence, False, found)
    return found


def flat(sequence):
    return [e for event in sequence for e in (sum((flat(arm) for arm in event), []) if isinstance(event, tuple) else [event])]


def source(name):
    with open(os.path.join(CSRC, name)) as file:
        return without_comments(file.read())


def helper_events():
    text = source("attention.cuh")
    found = {}
    for name in HELPERS:
        body = function_body(text, name)
        if body is not None:
            found[name] = events(body, found)
    return found


@pytest.mark.parametrize("file,kernel", [("attention.cuh", "attention_forward_kernel"),
                                         ("attention_backward.cuh", "attention_query_grad_kernel"),
                                         ("attention_backward.cuh", "attention_key_grad_kernel")])
def test_no_aligned_instruction_behind_a_divergent_branch(file, kernel):
    sequence = events(function_body(source(file), kernel), helper_events())
    names = flat(sequence)
    assert sum(e.startswith("tmem_ld") for e in names) >= 4 and "apart" in names  # the reading has found the kernel
    assert faults(sequence) == []


def test_the_reading_finds_what_it_looks_for():
    good = "for (int i = 0; i < 4; ++i) { __syncwarp(); ptx::tmem_ld_32x32b_x32(a, o); if (!mine) continue; to[i] = o; }"
    bad = good.replace("__syncwarp();", "")
    assert faults(events(good, {})) == []
    assert faults(events(bad, {})) == ["tmem_ld_32x32b_x32"]
    assert faults(events("if (lane == 0) { ptx::mbar_arrive(b); } ptx::tmem_wait_st();", {})) != []
    assert faults(events("if (lane == 0) { ptx::mbar_arrive(b); } __syncwarp(); ptx::tmem_wait_st();", {})) == []
    assert faults(events("if (mine) { ptx::tmem_wait_st(); } __syncwarp();", {})) != []
    arms = "if (warp == 0) { if (lane == 0) load(); } else if (warp == 1) { ptx::tmem_wait_st(); } else { x = 1; }"
    assert faults(events(arms, {})) == [] and faults(events(arms + "ptx::tmem_wait_ld();", {})) == ["tmem_wait_ld"]
    assert faults(events(arms + "__syncwarp(); ptx::tmem_wait_ld();", {})) == []
    assert faults(events("if (warp == 2) ptx::tmem_alloc(slot, 512);", {})) == []
    assert faults(events("zero_rows<kDim>(v, row, n); ptx::tmem_wait_st();", {"zero_rows": ["apart"]})) != []
