"""No-GPU checks of rules that a kernel's source has to keep and that no run shows reliably."""
import pathlib
import re

import pytest

CSRC = pathlib.Path(__file__).resolve().parent.parent / "lattice_b200" / "csrc"


def kernels(path):
    """(name, body) of every kernel of a source file, comments taken out."""
    text = re.sub(r"//[^\n]*", "", path.read_text())
    for m in re.finditer(r"__global__[^;{]*?\b(\w+)\(const [^{;]*\{", text):
        depth, at = 1, m.end()
        while depth:
            depth += {"{": 1, "}": -1}.get(text[at], 0)
            at += 1
        yield m.group(1), text[m.end():at]


@pytest.mark.parametrize("source", sorted(p.name for p in CSRC.glob("*.cu")))
def test_a_cluster_has_started_before_its_shared_memory_is_touched(source):
    """The programming model lets a CTA touch another one's shared memory only once all CTAs of the cluster run: a
    cluster barrier has to lie before the first access."""
    for name, body in kernels(CSRC / source):
        uses = [m.start() for m in re.finditer(r"map_shared_rank|mapa\.|shared::cluster\.b32 ", body)]
        if not uses:
            continue
        waits = [m.start() for m in re.finditer(r"cluster_wait\(\)|cluster\.sync\(\)", body)]
        assert waits and waits[0] < uses[0], f"{source}: {name} maps a peer's shared memory before the cluster is known to run"


def test_the_check_sees_kernels():
    assert {n for n, _ in kernels(CSRC / "lq4_verify.cu")} == {"verify_kernel", "verify_stats_kernel"}
