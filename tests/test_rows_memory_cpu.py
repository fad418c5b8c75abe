"""Rules on memory that the kernels of the row operators keep, read from their
source: a kernel that is on the multiprocessors while another writes what it
reads, and copies that the two proxies of shared memory make, go wrong too rarely
for a run to show it."""

import os
import re

import pytest

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "numba_mlir_b200", "csrc")


def source(name):
    with open(os.path.join(CSRC, name)) as f:
        return re.sub(r"//[^\n]*", "", f.read())


def functions(text):
    """name -> (parameters, body) of the functions at the top of a file and of
    the structs in it."""
    found = {}
    for m in re.finditer(r"(\w+)\s*\(", text):
        at = close(text, m.end() - 1, "()")
        rest = re.match(r"\s*(const)?\s*(:[^{;]*)?\{", text[at:])
        if rest and m.group(1) not in ("if", "for", "while", "switch"):
            begin = at + rest.end() - 1
            found[m.group(1)] = (text[m.end():at - 1], text[begin:close(text, begin, "{}")])
    return found


def close(text, at, pair):
    depth = 0
    for i in range(at, len(text)):
        depth += (text[i] == pair[0]) - (text[i] == pair[1])
        if depth == 0:
            return i + 1
    raise AssertionError("unbalanced")


# what the sort's kernels leave for the kernels behind them
MADE = ("keys", "order", "place", "kept", "counts", "from", "keysIn", "entriesIn", "p.keys", "p.order", "p.counts")


@pytest.mark.parametrize("file", ["rows.cu", "row_sort.cu"])
def test_what_a_predecessor_writes_is_not_read_as_constant(file):
    every = functions(source(file))
    behind = {n: f for n, f in every.items() if "wait_for_previous()" in f[1]}
    assert {"rows.cu": {"nmb_take_rows_grad", "nmb_dispatch_rows", "nmb_dispatch_rows_bulk"},
            "row_sort.cu": {"nmb_sort_scatter"}}[file] == set(behind)
    # the functions that those call, and what those call
    reached, new = dict(behind), dict(behind)
    while new:
        called = {n: f for n, f in every.items() for _, body in new.values() if re.search(rf"\b{n}\b\s*[<(]", body)}
        new = {n: f for n, f in called.items() if n not in reached}
        reached.update(new)
    for name, (params, body) in reached.items():
        for m in re.finditer(r"__ldg\(", body):
            read = body[m.end():close(body, m.end() - 1, "()") - 1]
            assert not re.match(rf"({'|'.join(map(re.escape, MADE))})\b", read.strip()), f"{name}: __ldg({read})"
        for m in re.finditer(r"const\s+\w+\s*\*\s*__restrict__\s*(\w+)", params):
            assert m.group(1) not in MADE, f"{name}: {m.group(0)}"


@pytest.mark.parametrize("name", ["walk_bulk", "nmb_combine_rows_grad_bulk"])
def test_ordinary_stores_come_before_the_next_copy(name):
    """Where rows are fetched in turns into the same shared memory, edge elements
    are stored there by the thread that issues the place's next bulk copy: a
    fence between the proxies stands in front of that copy."""
    _, body = functions(source("rows.cu"))[name]
    fetches = [m.start() for m in re.finditer(r"fetch_row<LOOSE>\(", body)]
    fence = body.find("nmb::fence_async_smem()")
    assert fetches and 0 <= fence < min(fetches)
    assert re.search(r"if \(LOOSE && (turn > 1|first > 0)\)\s*$", body[:fence])  # from the second turn of a place on


def test_a_block_that_gives_up_waits_for_both_turns():
    """walk_bulk has two turns of copies on their way: a block that gives up on
    one stays for the other, or its copies land in another block's memory."""
    _, body = functions(source("rows.cu"))["walk_bulk"]
    at = body.index("if (!bulk_arrived(")
    gives_up = body[at:body.index("return false", at)]
    assert re.search(r"if \(turn \+ 1 < last\)\s*\(void\)nmb::mbar_wait\(&turns\.bar\[b \^ 1\]", gives_up)


def test_only_kernels_of_one_call_begin_early():
    """Every launch says whether a kernel of the same call stands in front of it:
    the sort's scatters follow a count, a gradient follows a sort only if there are
    entries, copies only where the call has sorted."""
    args = {}
    for file in ("rows.cu", "row_sort.cu"):
        text = source(file)
        for m in re.finditer(r"launchBehind\(", text):
            call = text[m.end():close(text, m.end() - 1, "()") - 1]
            args.setdefault(file, []).append(re.search(r"s\.stream,\s*(\w+),", call).group(1))
    assert args == {"rows.cu": ["behind"] * 3, "row_sort.cu": ["true"]}
    assert "const bool behind = ids->count > 0;" in source("rows.cu")
    assert re.search(r"dispatchRows\(waits, s, x, k, place, offsets \+ groups, out, ids->count > 0\)", source("rows.cu"))
    assert "config.numAttrs = behind ? 1 : 0;" in source("rows_host.h")
