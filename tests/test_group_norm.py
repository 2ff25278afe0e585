"""Group norm on the CPU: the plain path against torch's per sequence, and every refusal."""
import math

import pytest
import torch
import torch.nn.functional as F

from hydragnn_amd.ops.norm import group_norm


def _ptr(lens):
    return torch.tensor([0] + list(torch.tensor(lens).cumsum(0)), dtype=torch.int32)


_ACT = {"none": lambda t: t, "relu": torch.relu, "silu": F.silu}


@pytest.mark.parametrize("act", ["none", "relu", "silu"])
def test_plain_path_matches_torch(act):
    lens = [4, 0, 7, 1]
    g = torch.Generator().manual_seed(0)
    x = torch.randn(14, 6, generator=g, dtype=torch.float64) * 2 + 5
    w, b = torch.randn(6, generator=g, dtype=torch.float64), torch.randn(6, generator=g, dtype=torch.float64)
    dy = torch.randn(14, 6, generator=g, dtype=torch.float64)
    x[12:] = math.nan  # behind the last sequence
    leaves = [t.requires_grad_() for t in (x, w, b)]
    out = group_norm(x, 3, w, b, ptr=_ptr(lens), act=act)
    got = torch.autograd.grad(out, leaves, dy)
    at, parts = 0, []
    for n in lens:
        if n:
            parts.append(_ACT[act](F.group_norm(x[at:at + n].t().unsqueeze(0), 3, w, b, 1e-5)[0].t()))
        at += n
    ref = torch.cat(parts)
    torch.testing.assert_close(out[:12], ref, rtol=1e-12, atol=1e-12)
    assert not out[12:].any()
    for a, c in zip(got, torch.autograd.grad(ref, leaves, dy[:12])):
        torch.testing.assert_close(a, torch.nan_to_num(c), rtol=1e-10, atol=1e-10)


def test_without_pointers_each_sample_is_its_own():
    x = torch.randn(3, 4, 5, 8)
    w, b = torch.randn(8), torch.randn(8)
    got = group_norm(x, 4, w, b)
    torch.testing.assert_close(got, F.group_norm(x.permute(0, 3, 1, 2), 4, w, b).permute(0, 2, 3, 1),
                               rtol=1e-5, atol=1e-5)
    assert group_norm(torch.randn(5, 8), 2).shape == (5, 8)
    assert group_norm(torch.randn(0, 8), 2).shape == (0, 8)


@pytest.mark.parametrize("change,what", [
    ({"x": torch.zeros(8)}, "rows, channels"),
    ({"x": torch.zeros(4, 8, dtype=torch.int32)}, "not supported"),
    ({"x": torch.zeros(4, 0)}, "channels"),
    ({"x": torch.zeros(2, 4097)}, "channels"),
    ({"groups": 3}, "do not divide"),
    ({"groups": 0}, "do not divide"),
    ({"groups": 2.0}, "do not divide"),
    ({"act": "tanh"}, "act is"),
    ({"weight": torch.zeros(7)}, "weight is"),
    ({"bias": torch.zeros(8, dtype=torch.float64)}, "bias is"),
    ({"ptr": torch.tensor([0, 4])}, "int32"),
    ({"ptr": torch.tensor([[0, 4]], dtype=torch.int32)}, "int32"),
    ({"ptr": torch.tensor([0, 5], dtype=torch.int32)}, "ascend"),
    ({"ptr": torch.tensor([0, 3, 2], dtype=torch.int32)}, "ascend"),
    ({"x": torch.zeros(2, 2, 8), "ptr": torch.tensor([0, 2], dtype=torch.int32)}, "with ptr"),
])
def test_refusals(change, what):
    with pytest.raises(ValueError, match=what):
        group_norm(**{"x": torch.zeros(4, 8), "groups": 2, **change})
