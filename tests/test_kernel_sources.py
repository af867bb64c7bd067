"""What the kernels promise and no test on a GPU may provoke, checked on the sources: what kernels that are launched close
behind others (launch_close) do before they wait for those, and what the paged attention does with indices that a call which
gave up has left. A block launched close may be resident while the kernel before it still runs, so it holds no tensor memory
that one of that kernel's blocks could be waiting for, and no thread ends, or reads what that kernel writes, ahead of its
wait."""
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


def test_no_loads_through_the_read_only_path():
    """Its data may not change while a kernel lives, and a kernel that is launched close lives while the one before it
    writes. In the kernels' files, headers for them included."""
    files = {k[0] for k in close_kernels()} | {"kv_cache.cuh", "attn_util.cuh"}
    for f in files:
        s = re.sub(r"//[^\n]*", "", sources()[f])
        assert "__ldg" not in s and ".nc." not in s and "__restrict__" not in s, f


def body(name):
    return next(k[2] for k in kernels() if k[1] == name)


def test_join_checks_the_parts_that_it_finds():
    """A call that gave up a wait, or whose lengths changed under it, leaves parts unwritten: the join takes nothing from the
    workspace as an index that it has not checked, and ends before its first access if it does not fit."""
    b = body("k_join")
    check = b.index("p.blocks - part.first")
    assert "part.first < 0" in b[:check + 40] and check < b.index("p.part_ml[") and check < b.index("p.part_o +")


def test_paged_search_ends_and_checks_what_it_found():
    """Lengths that change while a block searches its first unit may leave it without one: the search ends with the last
    sequence, and neither an index that was never written nor a unit behind the sequence's last is used."""
    b = body("k_attention_paged")
    search = b[b.index("int64_t before = 0"):b.index("b = *s_seq")]
    assert "for (int base = 0; base < p.n_seqs; base += kThreads)" in search
    assert "*s_seq = -1" in b[:b.index("wait_before()")]
    after = b[b.index("b = *s_seq"):b.index("S::tiles_before(at, nt, x0) >=")]
    assert after.index("if (b < 0) return") < after.index("length(b)") and "if (unit >= U) return" in after
