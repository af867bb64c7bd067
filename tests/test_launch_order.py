"""What kernels that are launched close behind others (launch_close) may do before they wait for those, checked on the
sources: such a block may be resident while the kernel before it still runs, so it holds no tensor memory that one of
that kernel's blocks could be waiting for, and no thread ends, or reads what that kernel writes, ahead of its wait."""
import os
import re

import pytest

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "mold_b200", "csrc")


def sources():
    return {f: open(os.path.join(CSRC, f)).read() for f in sorted(os.listdir(CSRC)) if f.endswith((".cu", ".cuh"))}


def kernels():
    """(file, kernel name, body without comments) of every __global__ function."""
    out = []
    for f, s in sources().items():
        s = re.sub(r"//[^\n]*", "", s)
        for m in re.finditer(r"__global__\s+void\s+(?:__launch_bounds__\((?:[^()]|\([^()]*\))*\)\s+)?(\w+)\(", s):
            at = s.index("{", m.end())
            depth, end = 1, at + 1
            while depth:
                depth += {"{": 1, "}": -1}.get(s[end], 0)
                end += 1
            out.append((f, m.group(1), s[at:end]))
    return out


def close_kernels():
    """The kernels that launch_close is given by name or through a local name for an instance."""
    names = set()
    for s in sources().values():
        local = dict(re.findall(r"auto (\w+) = (k_\w+)<", s))
        for x in re.findall(r"launch_close\((?:\w+::)?(\w+)", s):
            names.add(local.get(x, x))
    return [k for k in kernels() if k[1] in names]


def test_kernels_are_found():
    names = {k[1] for k in close_kernels()}
    assert {"k_kv_write", "k_kv_read", "k_attention_paged", "k_attention_varlen", "k_join"} <= names
    assert names == {k[1] for k in kernels() if "wait_before()" in k[2]}


@pytest.mark.parametrize("what", ["tmem_alloc(", "return", "__ldg(", "tma_load", "bulk_load", "cp_async"])
def test_nothing_before_the_wait(what):
    for f, name, body in close_kernels():
        before = body[:body.index("wait_before()")]
        assert what not in before, f"{f}: {name} has {what} ahead of wait_before()"
