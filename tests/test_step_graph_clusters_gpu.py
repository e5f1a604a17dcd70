"""Steps of one slot whose kernels are the same but whose thread-block clusters are not: an executable graph that is
updated in place would keep the old cluster dimensions, so the record is instantiated anew."""
import pytest
import torch

import soklyn_b200 as sk

pytestmark = pytest.mark.gpu


def test_a_slot_takes_products_whose_sums_are_shared_by_other_numbers_of_blocks(gpu_ctx):
    """128 x 128 outputs, one tile: a sum of 512 is shared by more blocks of a cluster than one of 128."""
    g = torch.Generator(device="cuda")
    g.manual_seed(5)
    nets = []
    for k in (512, 128, 512, 256):
        blk = sk.DenseBlock(gpu_ctx, False, k, 128, 128, sk.InitXavierNormalFunc(k), None, sk.Precision.FP16)
        x = sk.Tensor(torch.randn(128, k, generator=g, device="cuda").half(), sk.Precision.FP16)
        net = sk.FeedForwardNetwork([blk], k)
        nets.append((net, x, net.forward(gpu_ctx, x, 128, False, 1)[-1].data.clone()))
    with gpu_ctx.step_graph(7):                # the slot's first step runs unrecorded
        pass
    before = gpu_ctx.step_graph_stats()
    for _ in range(2):
        for net, x, want in nets:
            with gpu_ctx.step_graph(7):
                out = net.forward(gpu_ctx, x, 128, False, 1)[-1]
            gpu_ctx.synchronize()
            assert torch.equal(out.data, want)
            out.data.zero_()
    after = gpu_ctx.step_graph_stats()
    assert after["launched"] - before["launched"] == 8 and after["instantiated"] - before["instantiated"] > 1
