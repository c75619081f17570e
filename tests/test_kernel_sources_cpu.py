"""What the compiler may move above griddepcontrol.wait, checked in the kernels'
sources: in a kernel that waits for its predecessor, loads through a restricted
parameter or by __ldg count as loads of constant data, so neither may reach
data that a kernel on the stream writes."""
import glob
import os
import re

import pytest

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "veltrix-engine_b200", "csrc")
CONSTANT = {"embd", "rope", "w", "qs"}   # weights and the RoPE table: written before any forward


def closing(s, at, pair):
    """Index of the bracket that closes the one at s[at]."""
    depth = 0
    for i in range(at, len(s)):
        depth += (s[i] == pair[0]) - (s[i] == pair[1])
        if depth == 0:
            return i
    raise AssertionError("unbalanced")


def kernels():
    """(file, name, parameters, body) of every __global__ function that waits."""
    for path in sorted(glob.glob(os.path.join(CSRC, "*.cu"))):
        s = re.sub(r"//[^\n]*", "", open(path).read())
        for m in re.finditer(r"__global__", s):
            head = re.compile(r"(k_\w+)\s*\(").search(s, m.end())
            end = closing(s, head.end() - 1, "()")
            brace = s.index("{", end)
            body = s[brace:closing(s, brace, "{}") + 1]
            if "pdl_wait()" in body:
                yield os.path.basename(path), head.group(1), s[head.end():end], body


def test_the_scan_sees_the_kernels():
    names = [k[1] for k in kernels()]
    assert len(names) >= 20 and {"k_embed", "k_rope_kv", "k_qgemv_skinny", "k_kv8_append", "k_splitk_reduce"} <= set(names)


@pytest.mark.parametrize("file,name,params,body", list(kernels()), ids=lambda v: v if len(v) < 30 else "")
def test_waiting_kernels_read_streamed_data_in_order(file, name, params, body):
    for p in params.split(","):
        if "__restrict__" in p:
            assert "const" in p and re.search(r"(\w+)\s*$", p).group(1) in CONSTANT, (file, name, p.strip())
    assert "__ldg(" not in body, (file, name)
