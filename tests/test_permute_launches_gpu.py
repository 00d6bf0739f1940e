"""The launch count that zmoe_permute_launches states, and with it the layer's
statistics, against the kernels of a captured call; results at the sizes where
the form changes."""
import pytest
import torch

from zmoe import synthetic as syn

pytestmark = pytest.mark.gpu


def _ops():
    from zmoe import ops
    return ops


def _kernels(call):
    from cuda.bindings import runtime as rt
    g = torch.cuda.CUDAGraph(keep_graph=True)
    with torch.cuda.graph(g):
        call()
    h = rt.cudaGraph_t(g.raw_cuda_graph())
    err, _, n = rt.cudaGraphGetNodes(h, 0)
    assert err == rt.cudaError_t.cudaSuccess
    err, nodes, n = rt.cudaGraphGetNodes(h, n)
    types = [rt.cudaGraphNodeGetType(v)[1] for v in nodes[:n]]
    return sum(t == rt.cudaGraphNodeType.cudaGraphNodeTypeKernel for t in types)


@pytest.mark.parametrize("T,k,E,H,capacity,want", [
    (1, 4, 60, 2048, 0, 1), (256, 4, 60, 64, 0, 1), (257, 4, 60, 64, 0, 2), (512, 4, 60, 64, 0, 2), (32767, 4, 60, 8, 0, 2),
    (32768, 4, 60, 8, 0, 4), (32768, 4, 60, 0, 0, 3), (700, 4, 60, 0, 0, 1), (512, 1, 8, 64, 40, 3), (512, 1, 8, 0, 40, 2),
    (40, 33, 40, 16, 0, 3), (300, 2, 1025, 8, 0, 3)])
def test_stated_count(T, k, E, H, capacity, want):
    ops = _ops()
    g = torch.Generator().manual_seed(T)
    idx = torch.rand(T, E, generator=g).topk(k, dim=1).indices.to(torch.int32).cuda()
    x = torch.randn(T, H, generator=g).to(torch.bfloat16).cuda() if H else None
    assert ops.permute_launches(T, k, E, H, capacity) == want
    ops.permute(idx.clone(), x, E, capacity, T if capacity else 0)
    torch.cuda.synchronize()
    assert _kernels(lambda: ops.permute(idx, x, E, capacity, T if capacity else 0)) == want


def test_layer_statistics():
    # the same layer, all experts cached, on both sides of the permute's change of form
    from zmoe.layer import MoELayer
    s = syn.LayerShape(hidden=256, num_experts=8, inter=64, topk=4, kind=0, shared_inter=128, shared_gate=True)
    L = MoELayer(s, max_tokens=300, cache_slots=8, transient_slots=0, policy="ZipMoE")
    wr, sg = syn.router_weights(s, std=0.05, seed=1)
    L.set_router(wr, None, sg)
    L.set_shared(*syn.shared_weights(s, std=0.05, seed=2))
    L.load_experts(syn.expert_weights(s, 1, std=0.05, seed=0)[0], num_file_chunks=3)
    x = syn.activations(300, s.hidden, seed=3).cuda()
    for _ in range(2):                                  # every expert decoded once
        L(x)
    L.sync()
    ops, count = _ops(), []
    for T in (256, 257):
        before = L.stats()["launches"]
        L(x[:T])
        L.sync()
        count.append(L.stats()["launches"] - before - ops.permute_launches(T, s.topk, s.num_experts, s.hidden))
    # router, shared FFN 2, grouped FFN 2, combine
    assert count == [6, 6]
