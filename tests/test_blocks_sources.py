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
