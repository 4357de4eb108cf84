"""Kernels that are set up while the kernel before them still runs read what that
kernel writes.  A ``const __restrict__`` pointer or ``__ldg`` promises the
compiler that the memory keeps its values for the kernel's whole life, which
begins before the writer's ends: such a load may be moved in front of the wait
or be served from a cache that is not kept coherent.  The sources have neither
in these kernels, nor in the device functions that they call."""
import glob
import os
import re

import pytest

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "usaf_b200", "csrc")
WAIT = "wait_for_previous"


def functions(text):
    """Name, head (template to parameters) and body of every device function."""
    text = re.sub(r"//[^\n]*", "", text)
    out = []
    for m in re.finditer(r"__global__|__device__", text):
        brace = text.index("{", m.start())
        head = text[m.start():brace]
        if ";" in head:             # a declaration, or a variable
            continue
        end, depth = brace, 0
        while True:
            depth += {"{": 1, "}": -1}.get(text[end], 0)
            end += 1
            if depth == 0:
                break
        flat = re.sub(r"(__launch_bounds__|__cluster_dims__)\s*\([^)]*\)", "", head)
        name = re.search(r"(\w+)\s*\(", flat)
        out.append((name.group(1) if name else "", head, text[brace:end]))
    return out


def early(functions_):
    """Kernels that wait for the one before them, and what they call."""
    by_name = {}
    for name, head, body in functions_:
        by_name.setdefault(name, []).append((head, body))
    todo = [(n, h, b) for n, h, b in functions_ if "__global__" in h and WAIT in b]
    seen = []
    while todo:
        name, head, body = todo.pop()
        if (name, head, body) in seen:
            continue
        seen.append((name, head, body))
        for called in set(re.findall(r"(\w+)\s*(?:<[^;{}()]*>)?\s*\(", body)):
            todo += [(called, h, b) for h, b in by_name.get(called, ())]
    return seen


FILES = sorted(f for f in glob.glob(os.path.join(CSRC, "*.cu")) if "launch_early" in open(f).read())


def test_the_reader_finds_the_kernels():
    assert {os.path.basename(f) for f in FILES} >= {"norm.cu", "embedding.cu", "adamw.cu"}
    text = """template <typename T> __global__ void __launch_bounds__(256)
    k(const T *__restrict__ a) { wait_for_previous(); get<T>(a); }
    __device__ int get(const int *p) { return __ldg(p); }
    __global__ void other(const int *__restrict__ a) { get(a); }"""
    names = [n for n, _, _ in early(functions(text))]
    assert sorted(names) == ["get", "k"]


@pytest.mark.parametrize("path", FILES, ids=os.path.basename)
def test_no_read_only_promise_in_front_of_the_wait(path):
    shared = [f for h in glob.glob(os.path.join(CSRC, "*.cuh")) for f in functions(open(h).read())]
    found = early(functions(open(path).read()) + shared)
    assert found
    for name, head, body in found:
        assert "__restrict__" not in head, f"{name}: a __restrict__ pointer in a kernel that starts early"
        assert "__ldg" not in body, f"{name}: __ldg in a kernel that starts early"
