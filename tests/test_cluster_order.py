"""What one CTA of a cluster tells another, read from the kernels' sources (no GPU): an arrival at the
other's barrier and the wait for it order something between the two only with the cluster's scope."""

import re
from pathlib import Path

CSRC = Path(__file__).resolve().parents[1] / "tessery_b200" / "csrc"
SOURCES = {p.name: p.read_text() for p in sorted([*CSRC.glob("*.cu"), *CSRC.glob("*.cuh")])}


def code(text):
    return re.sub(r"//[^\n]*", "", text)


def test_arrivals_at_another_ctas_barrier_have_the_scope_of_the_cluster():
    found = 0
    for name, text in SOURCES.items():
        for arrive in re.findall(r"mbarrier\.arrive[\w.:]*shared::cluster[\w.:]*", code(text)):
            found += 1
            assert re.search(r"\.(release|relaxed)\.cluster\.", arrive), (name, arrive)
    assert found


def test_a_relaxed_arrival_hands_over_tensor_memory_alone():
    """It orders no other memory: it stands behind the fence of tensor-memory reads, and no rows that
    threads copied are passed between the two CTAs."""
    relaxed = re.findall(r"void (\w+)\([^)]*\) \{\s*asm volatile\(\"mbarrier\.arrive\.relaxed\.cluster",
                         code(SOURCES["tcgen05.cuh"]))
    for name, text in SOURCES.items():
        text = code(text)
        if name == "tcgen05.cuh":
            continue
        for call in relaxed:
            for m in re.finditer(rf"\b{call}\(", text):
                before = text[:m.start()].rsplit("{", 1)[1]
                assert "tc_fence_before();" in before, (name, before)


def test_waits_of_the_pair_are_for_the_cluster():
    text = code(SOURCES["experts_linear.cu"])
    kernel = text[text.index("pair_kernel(const"):text.index("bool make_maps")]
    waits = re.findall(r"\b(?:warp_wait|wait_bar|drain_bar)\b(<true>)?\(", kernel)
    assert len(waits) >= 6 and all(waits)
    assert "mbar_test(" not in kernel and "Gather" not in kernel and "cp.async.cg" not in kernel
    parts = code(SOURCES["linear_parts.cuh"])
    assert re.search(r"if constexpr \(kCluster\)\s+return mbar_test_cluster", parts)
    assert "try_wait.parity.acquire.cluster" in code(SOURCES["tcgen05.cuh"])
