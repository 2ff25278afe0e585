"""The models' distance bias, group norm and attention read-out together (``global_attn_bias``,
``feature_norm``, ``graph_pooling``) on the CPU."""
import copy

import pytest
import torch

from hydragnn_amd.data.graph import collate
from hydragnn_amd.data.synthetic import degree_histogram, oc20_like
from hydragnn_amd.models.create import create_model
from hydragnn_amd.models.layers import AttentionPooling, GroupNorm
from hydragnn_amd.ops.pna import composite_mode

HEADS = {"graph": [{"type": "branch-0", "architecture": {"num_sharedlayers": 1, "dim_sharedlayers": 8,
                                                          "num_headlayers": 1, "dim_headlayers": [8]}}],
         "node": [{"type": "branch-0", "architecture": {"num_headlayers": 1, "dim_headlayers": [8], "type": "mlp"}}]}
BIAS = {"num_buckets": 16, "max_distance": 24, "unit": 0.5}


def _samples(n=4):
    s = oc20_like(n, seed=3, radius=5.0, max_neighbours=8, pe_dim=4, min_atoms=6, max_atoms=14)
    for g in s:
        g.edge_attr = torch.ones(g.edge_index.shape[1], 1)
    return s


def _model(samples, mt="PNAPlus", gps=True, heads=("graph", "node"), **more):
    return create_model(mt, samples[0].x.shape[1], 12, [1] * len(heads), 4, "GPS" if gps else "", "multihead", 2,
                        list(heads), HEADS, "relu", "mse", [1.0] * len(heads), 2,
                        pna_deg=degree_histogram(samples, max_degree=10), edge_dim=1 if gps else None,
                        envelope_exponent=5, num_radial=5, radius=5.0, max_neighbours=8, num_gaussians=8,
                        num_filters=12, max_ell=1, node_max_ell=1, avg_num_neighbors=5.0, correlation=2,
                        use_gpu=False, dropout=0.0, attn_scope="graph", **more)


def _all(**more):
    return dict(attn_bias=BIAS, feature_norm="group", feature_norm_groups=3, graph_pooling="attention",
                graph_pooling_heads=2, **more)


def test_forward_backward_reaches_every_new_parameter():
    samples = _samples()
    m = _model(samples, **_all()).train()
    with torch.no_grad():
        for c in m.graph_convs:
            c.attn.rel_bias.normal_()
    pred = m(collate(samples))
    sum(p.pow(2).mean() for p in pred).backward()
    new = [(n, p) for n, p in m.named_parameters() if "rel_bias" in n or "graph_pooling" in n or "feature_layers" in n]
    assert len([n for n, _ in new if "rel_bias" in n]) == 2 and isinstance(m.graph_pooling, AttentionPooling)
    for n, p in new:
        assert p.grad is not None and torch.isfinite(p.grad).all(), n
        if n != "graph_pooling.kv.bias":  # (its key half moves all scores of a row alike)
            assert p.grad.any(), n


def test_a_zero_bias_is_the_attention_without():
    samples = _samples()
    with_bias, plain = _model(samples, attn_bias=BIAS).eval(), _model(samples).eval()
    state = with_bias.state_dict()
    missing = plain.load_state_dict({k: v for k, v in state.items() if "rel_bias" not in k})
    assert not missing.missing_keys
    b = collate(samples)
    for x, y in zip(with_bias(b), plain(b)):
        torch.testing.assert_close(x, y, rtol=1e-5, atol=1e-6)


def test_a_graph_does_not_depend_on_its_batch():
    """Group norm and the read-out go by graph: in training mode too (batch norm's statistics do not)."""
    samples = _samples()
    m = _model(samples, "PNA", gps=False, feature_norm="group", feature_norm_groups=4, graph_pooling="attention",
               graph_pooling_heads=3).train()
    together = m(collate(samples))
    at = 0
    for i, g in enumerate(samples):
        alone = m(collate([g]))
        n = g.x.shape[0]
        torch.testing.assert_close(alone[0], together[0][i:i + 1], rtol=1e-5, atol=1e-6)
        torch.testing.assert_close(alone[1], together[1][at:at + n], rtol=1e-5, atol=1e-6)
        at += n


def test_moved_and_turned_positions_give_the_same_bias():
    samples = _samples()
    m = _model(samples, **_all()).eval()
    with torch.no_grad():
        for c in m.graph_convs:
            c.attn.rel_bias.normal_()
    b = collate(samples)
    ref = m(b)
    other = copy.deepcopy(b)
    turn = torch.tensor([[0.0, 1.0, 0.0], [-1.0, 0.0, 0.0], [0.0, 0.0, 1.0]])  # exact: no distance changes
    other._store["pos"] = b.pos @ turn
    for x, y in zip(m(other), ref):
        torch.testing.assert_close(x, y, rtol=1e-4, atol=1e-5)


def test_composite_mode_is_twice_differentiable():
    samples = _samples(2)
    m = _model(samples, **_all()).train()
    b = collate(samples)
    b._store["pos"] = b.pos.clone().requires_grad_()
    with composite_mode():
        e = m(b)[0].sum()
        (f,) = torch.autograd.grad(e, b.pos, create_graph=True)
        f.pow(2).sum().backward()
    assert torch.isfinite(m.graph_pooling.queries.grad).all() and m.graph_pooling.queries.grad.any()


def test_configuration_entries_reach_the_model():
    from hydragnn_amd.models.create import create_model_config

    samples = _samples()
    arch = dict(mpnn_type="PNA", input_dim=samples[0].x.shape[1], hidden_dim=12, output_dim=[1], pe_dim=4,
                global_attn_engine="GPS", global_attn_type="multihead", global_attn_heads=2, output_type=["graph"],
                output_heads=HEADS, task_weights=[1.0], num_conv_layers=2, edge_dim=1,
                pna_deg=degree_histogram(samples, max_degree=10), global_attn_scope="graph", global_attn_bias=BIAS,
                feature_norm="group", feature_norm_groups=3, graph_pooling="attention", graph_pooling_heads=2)
    m = create_model_config({"Architecture": arch, "Training": {}}, use_gpu=False)
    assert m.graph_convs[0].attn.rel_bias.shape == (2, 16) and m.graph_convs[0].attn.rel_buckets.unit == 0.5
    assert all(isinstance(n, GroupNorm) and n.groups == 3 for n in m.feature_layers)
    assert m.graph_pooling.heads == 2


@pytest.mark.parametrize("more,what", [
    ({"attn_bias": BIAS, "gps": False}, "global_attn_engine"),
    ({"attn_bias": {"buckets": 4}}, "unknown entries"),
    ({"attn_bias": {"unit": 0.0}}, "unit"),
    ({"feature_norm": "layer"}, "feature_norm"),
    ({"feature_norm": "group", "feature_norm_groups": 5}, "do not divide"),
    ({"feature_norm": "group", "mt": "SchNet", "gps": False}, "no norm between"),
    ({"graph_pooling": "max"}, "graph_pooling"),
    ({"graph_pooling": "attention", "graph_pooling_heads": 5}, "do not divide"),
    ({"graph_pooling": "attention", "heads": ("node",)}, "no graph head"),
    ({"graph_pooling": "attention", "mt": "MACE", "gps": False}, "no graph head"),
])
def test_refusals(more, what):
    with pytest.raises(ValueError, match=what):
        _model(_samples(), **more)


def test_bias_needs_graph_scope_and_positions():
    samples = _samples()
    m = _model(samples, attn_bias=BIAS)
    b = collate(samples)
    b._store["pos"] = None
    with pytest.raises(ValueError, match="positions"):
        m.graph_convs[0](torch.zeros(b.num_nodes, 12), None, m._base_ctx(b))
    with pytest.raises(ValueError, match="scope"):
        create_model("GIN", 4, 12, [1], 4, "GPS", "multihead", 2, ["graph"], HEADS, "relu", "mse", [1.0], 2,
                     use_gpu=False, attn_bias=BIAS)
