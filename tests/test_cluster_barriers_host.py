"""Cluster kernels touch their peers' shared memory only once the peers run
(CPU, read from the sources).

CUDA guarantees that the CTAs of a cluster are scheduled together, not that a
CTA has started when another one reaches for its shared memory: a barrier over
the whole cluster has to lie in between. In a kernel's text the first cluster
barrier must come before the first address of a peer (mapa) and before the
first store or bulk copy that goes there."""
import pathlib
import re

import pytest

import recavsr_b200

CSRC = pathlib.Path(recavsr_b200.__file__).parent / "csrc"
PEER = re.compile(r"\bmapa\(|\bst\.shared::cluster|cp\.async\.bulk\.shared::cluster\.shared::cta")
BARRIER = re.compile(r"\bcluster_(?:sync|wait)\(")


def kernels():
    for path in sorted(CSRC.glob("*.cu")):
        text = re.sub(r"//[^\n]*", "", path.read_text())
        starts = [m.start() for m in re.finditer(r"__global__", text)] + [len(text)]
        for begin, end in zip(starts, starts[1:]):
            body = text[begin:end]
            name = re.search(r"(\w+)\(const __grid_constant__", body)
            if PEER.search(body):
                yield pytest.param(body, id=f"{path.stem}-{name.group(1) if name else begin}")


@pytest.mark.parametrize("body", list(kernels()))
def test_cluster_barrier_before_peer_access(body):
    barrier = BARRIER.search(body)
    assert barrier and barrier.start() < PEER.search(body).start()


def test_the_cluster_kernels_are_seen():
    assert len(list(kernels())) >= 4
