"""A CTA's shared memory may only be written by the others of its cluster once it has started: a cluster barrier has to stand before it.

Whether a kernel that lacks it fails depends on how the CTAs happen to start, so the sources are looked at instead."""
import re
from pathlib import Path

import pytest

CSRC = Path(__file__).resolve().parent.parent / "csrc"
REMOTE = re.compile(r"\b(st_cluster_\w+|map_to_cta|st_async_\w+)\(")


def kernels(text):
    for m in re.finditer(r"^__global__ void.*", text, re.M):
        end = text.find("\n}\n", m.start())
        body = re.sub(r"//.*", "", text[m.start():end])
        yield re.search(r"(\w+)\(const __grid_constant__", body).group(1), body


@pytest.mark.parametrize("source", sorted(p.name for p in CSRC.glob("*.cu")))
def test_remote_shared_memory_comes_after_a_cluster_barrier(source):
    for name, body in kernels((CSRC / source).read_text()):
        remote = REMOTE.search(body)
        if remote is None:
            continue
        before = body[:remote.start()]
        assert re.search(r"cluster_arrive(_relaxed)?\(\)", before) and "cluster_wait()" in before, (source, name)


def test_the_kernels_that_use_it_are_found():
    found = {n for p in CSRC.glob("*.cu") for n, b in kernels(p.read_text()) if REMOTE.search(b)}
    assert {"oproj_int4_kernel", "oproj_int4_few_kernel", "mla_pair_kernel"} <= found
