"""Orderings that a run cannot show reliably, checked in the kernels' source:
what a lucky schedule hides is still in the text. CPU only."""
import os
import re

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "krill_b200", "csrc")


def code(name):
    """A source file without its comments."""
    text = open(os.path.join(CSRC, name)).read()
    text = re.sub(r"/\*.*?\*/", "", text, flags=re.S)
    return re.sub(r"//[^\n]*", "", text)


def body(text, signature):
    """The braces' content of the function that `signature` starts."""
    at = text.index("{", text.index(signature))
    depth = 0
    for i in range(at, len(text)):
        depth += {"{": 1, "}": -1}.get(text[i], 0)
        if depth == 0:
            return text[at:i]
    raise AssertionError("unbalanced braces")


def test_block_choice_waits_for_its_cluster_before_remote_stores():
    """A CTA's shared memory may be written by the other CTAs of its cluster
    only once it is known to have started: a cluster barrier stands between the
    kernel's entry and the first store through map_shared_rank."""
    text = body(code("kv_select.cu"), "select_blocks_kernel(SelectParams p)")
    first = text.index("keys[", text.index("map_shared_rank"))
    arrive, wait = text.find("cluster.barrier_arrive("), text.find("cluster.barrier_wait(")
    assert 0 <= arrive < wait < first
    # and no CTA leaves between the two, or the others would wait for it
    assert "return" not in text[arrive:wait]


def test_picked_blocks_are_read_coherently():
    """The sparse decode kernel is resident while the choice before it still
    writes the picked blocks, so they may not be read through the read-only
    path (__ldg), whose data must not change while a kernel runs."""
    text = code("kv_attn.cuh")
    assert "p.sel" in text
    assert not re.search(r"__ldg\(\s*p\.sel\b", text)


def test_mma_issuer_goes_by_its_own_observation():
    """What a barrier's completion orders holds for the threads that observed
    it. The lane that issues the MMAs must be one of them: every lane's test has
    to have succeeded, not any lane's."""
    text = body(code("kv_shared_umma.cu"), "attn_shared_umma_kernel(AttnParams p)")
    polled = re.findall(r"__(any|all)_sync\(\s*0xffffffffu\s*,\s*mbar_\w+", text)
    assert polled and set(polled) == {"all"}
