"""CPU: rules that the row operators' kernel sources keep to, read from the sources."""
import glob
import os
import re

import pytest

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "cv-cuda_b200", "csrc")


def _kernels_of_clusters():
    """(name, body without comments) of every kernel that accesses the shared memory of another CTA."""
    found = []
    for path in sorted(glob.glob(os.path.join(CSRC, "*.cu*"))):
        text = re.sub(r"//[^\n]*|/\*.*?\*/", "", open(path, encoding="utf-8").read(), flags=re.S)
        for m in re.finditer(r"__global__[^{;]*?(\w+)\((?:[^(){}]|\([^()]*\))*\)\s*\{", text):
            depth, end = 1, m.end()
            while depth:
                depth += {"{": 1, "}": -1}.get(text[end], 0)
                end += 1
            if "map_shared_rank" in text[m.end():end]:
                found.append((m.group(1), text[m.end():end]))
    return found


def test_kernels_of_clusters_are_found():
    assert {"layernorm_grad_kernel", "embedding_sort_kernel"} <= {name for name, _ in _kernels_of_clusters()}


@pytest.mark.parametrize("name,body", _kernels_of_clusters(), ids=[k[0] for k in _kernels_of_clusters()])
def test_a_cluster_has_started_before_its_shared_memory_is_accessed(name, body):
    """Shared memory of another CTA may be accessed only once that CTA is known to run: a barrier of the cluster comes first."""
    first = body.index("map_shared_rank")
    assert re.search(r"cluster\s*\.\s*(sync|barrier_wait)\s*\(", body[:first]), name
