"""Distance bias, group norm and attention read-out in a model on the GPU: the HIP path against the
CPU path, statically padded batches, and the captured training step.  Tolerances are those of
tests/test_model_gpu.py for the same model without them: three layers of float32 work, whose roundings
(2^-24 each) the batch norms' and the losses' gradients carry to some 1e-4."""
import copy

import pytest
import torch

from hydragnn_amd.data.device_store import DeviceGraphStore
from hydragnn_amd.data.synthetic import degree_histogram, oc20_like
from hydragnn_amd.models.create import create_model
from hydragnn_amd.train.step import TrainStep, batch_loss

pytestmark = pytest.mark.gpu

HEADS = {"graph": [{"type": "branch-0", "architecture": {"num_sharedlayers": 2, "dim_sharedlayers": 50,
                                                         "num_headlayers": 2, "dim_headlayers": [50, 25]}}]}


def _model(samples, **more):
    m = create_model("PNAPlus", 4, 64, [1], 16, "GPS", "multihead", 8, ["graph"], HEADS, "relu", "mae", [1.0], 2,
                     pna_deg=degree_histogram(samples, 10), edge_dim=1, envelope_exponent=5, num_radial=6, radius=10.0,
                     use_gpu=False, dropout=0.0, attn_scope="graph", attn_bias={"unit": 0.25, "max_distance": 48},
                     feature_norm="group", feature_norm_groups=8, graph_pooling="attention", graph_pooling_heads=8,
                     **more)
    g = torch.Generator().manual_seed(1)
    with torch.no_grad():
        for c in m.graph_convs:
            c.attn.rel_bias.copy_(torch.randn(c.attn.rel_bias.shape, generator=g))
    return m


def _store(samples, dev):
    return DeviceGraphStore(samples, dev, head_types=["graph"], head_dims=[1], attn_scope="graph")


def test_gpu_matches_cpu():
    samples = oc20_like(12, seed=3)
    m_cpu = _model(samples)
    m_gpu = copy.deepcopy(m_cpu).cuda()
    idx = list(range(12))
    bc, bg = _store(samples, "cpu").batch(idx), _store(samples, "cuda").batch(idx)
    lc, _ = batch_loss(m_cpu, m_cpu(bc), bc)
    lg, _ = batch_loss(m_gpu, m_gpu(bg), bg)
    lc.backward()
    lg.backward()
    torch.testing.assert_close(lg.cpu(), lc.detach(), rtol=1e-4, atol=1e-4)
    for (n, a), (_, b) in zip(m_gpu.named_parameters(), m_cpu.named_parameters()):
        torch.testing.assert_close(a.grad.cpu(), b.grad, rtol=2e-3, atol=2e-4, msg=n)


def test_a_padded_batch_is_the_batch():
    samples = oc20_like(10, seed=4)
    m = _model(samples).cuda().train()
    m2 = copy.deepcopy(m)
    s = _store(samples, "cuda")
    idx = list(range(10))
    b0, b1 = s.batch(idx), s.batch(idx, Np=1024, Ep=8192)
    l0, _ = batch_loss(m, m(b0), b0)
    l1, _ = batch_loss(m2, m2(b1), b1)
    l0.backward()
    l1.backward()
    torch.testing.assert_close(l1, l0, rtol=1e-5, atol=1e-5)
    for (n, a), (_, b) in zip(m2.named_parameters(), m.named_parameters()):
        torch.testing.assert_close(a.grad, b.grad, rtol=1e-3, atol=1e-5, msg=n)


def test_captured_step_matches_eager():
    samples = oc20_like(64, seed=5)
    m1 = _model(samples).cuda()
    m2 = copy.deepcopy(m1)
    s = _store(samples, "cuda")
    eager = TrainStep(m1, mode="eager")
    graph = TrainStep(m2, mode="graph", node_bucket=4096, edge_bucket=1 << 16)
    graph.prepare(s, 16)
    batches = [list(range(i, i + 16)) for i in range(0, 48, 8)]
    le = [float(eager(s, b)[0]) for b in batches]
    lg = [float(graph(s, b)[0]) for b in batches]
    for a, b in zip(le, lg):
        assert abs(a - b) <= 1e-3 * max(1.0, abs(a)), (le, lg)
