"""What the sources of the ops in blocks and of the routed layer promise about CTAs that reach into each other, and no run can show (no GPU needed)."""

import re

import pytest

from tests.test_kernel_sources import source


def body(text, kernel):
    """A function's text, from its parameters to its last brace."""
    at = re.search(rf"\b{kernel}\(", text).start()
    begin = end = text.index("{", at)
    level = 0
    while True:
        level += {"{": 1, "}": -1}.get(text[end], 0)
        end += 1
        if not level:
            return text[begin:end]


REACH = r"\bst_cluster_f32\(|\bld_dsmem\(|\bst\.shared::cluster\.|\bbg_load_pair\(|\bbg_commit_pair\(|\bbg_arrive_cluster\(|\brouter_logits\("
MET = r"\bcluster_sync_all\(\)|barrier\.cluster\.wait"


@pytest.mark.parametrize("name,kernel", [("moe_layer.cu", "moe_layer_down_kernel"), ("moe_layer.cu", "router_logits"), ("blocks_gemm.cu", "blocks_gemm_kernel"),
                                         ("blocks_few.cuh", "blocks_few_kernel")])
def test_a_cluster_meets_before_its_ctas_reach_into_each_other(name, kernel):
    """Shared memory of another CTA may be touched once that CTA is known to run: a barrier of the cluster stands before the first such access."""
    text = body(source(name), kernel)
    reach, met = re.search(REACH, text), re.search(MET, text)
    assert reach and met and met.start() < reach.start()


def test_the_routed_layer_s_clusters_arrive_once_for_each_wait():
    for kernel, wait in (("moe_layer_up_kernel", "router_logits"), ("moe_layer_down_kernel", "moe_layer_down_kernel")):
        text = source("moe_layer.cu")
        assert body(text, kernel).count("barrier.cluster.arrive.") == 1 and body(text, wait).count("barrier.cluster.wait.") == 1


def test_no_cta_of_the_products_of_few_rows_holds_tensor_memory_where_its_cluster_meets():
    """Neither the allocation of tensor memory nor a cluster's barrier is bounded.  CTAs that hold the first and wait at the second, beside another kernel's that do the
    same, may wait for each other for good; so tensor memory is given back before the first meeting."""
    text = body(source("blocks_few.cuh"), "blocks_few_kernel")
    assert text.count("tcgen05.alloc.") == text.count("tcgen05.dealloc.") == 1
    assert text.index("tcgen05.alloc.") < text.index("tcgen05.dealloc.") < text.index("cluster_sync_all()")


def test_the_products_of_many_rows_have_an_sm_to_themselves():
    """Their CTAs hold all of an SM's tensor memory while the pair meets: their registers leave no room for another CTA that allocates some (four warps or more)."""
    text = source("blocks_gemm.cu")
    number = lambda name: int(re.search(rf"\b{name} = (\d+)\b", text).group(1))
    assert 65536 - number("BG_THREADS") * number("BG_REGS_LAUNCH") < 4 * 32 * 16
