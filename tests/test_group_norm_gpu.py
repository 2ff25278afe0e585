"""Group norm with an activation on the GPU against 64 bits."""
import math

import pytest
import torch

from hydragnn_amd.ops.norm import group_norm, group_norm_reference

pytestmark = pytest.mark.gpu
DEV = "cuda"
TYPES = [torch.float32, torch.bfloat16, torch.float16]
HALF = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}
U32 = 2.0 ** -24


def _ptr(lens, dev="cpu"):
    return torch.tensor([0] + list(torch.tensor(lens, dtype=torch.long).cumsum(0)), dtype=torch.int32, device=dev)


def _off(got, ref, tol, what, floor=0.0):
    got = got.detach().double().cpu()
    assert got.shape == ref.shape and torch.isfinite(got).all(), what
    off, size = (got - ref).norm().item(), ref.norm().item()
    assert off <= tol * size + floor, f"{what}: off by {off:.3e} of {size:.3e} (tol {tol:.1e})"


def _check(dtype, lens, C, G, act="silu", affine=True, shape=None, mean=3.0):
    g = torch.Generator().manual_seed(0)
    n = sum(lens) + 3 if shape is None else 0
    shape = shape or (n, C)
    x = (torch.randn(shape, generator=g) * 2 + mean * torch.randn(C, generator=g)).to(dtype)
    dy = torch.randn(shape, generator=g).to(dtype)
    params = [torch.randn(C, generator=g), torch.randn(C, generator=g)] if affine else []
    ptr = _ptr(lens) if lens is not None else None
    ref_in = [t.double().requires_grad_() for t in [x, *params]]
    dev = [t.to(DEV).requires_grad_() for t in [x, *params]]
    w = lambda t: t[1:3] if affine else (None, None)  # noqa: E731
    ref = group_norm_reference(ref_in[0], G, *w(ref_in), ptr, 1e-5, act)
    ref_g = torch.autograd.grad(ref, ref_in, dy.double())
    out = group_norm(dev[0], G, *w(dev), ptr=None if ptr is None else ptr.to(DEV), act=act)
    got = torch.autograd.grad(out, dev, dy.to(DEV))
    assert out.dtype == dtype and got[0].dtype == dtype
    # Elementwise work in 32 bits: about 16 roundings of values of the size of xh, w and b (the mean's
    # among them, relative to the deviation that it exceeds by `mean`), then one to the type.
    f32 = 16 * (1 + mean) * U32
    with torch.no_grad():
        _off(out, ref, HALF[dtype] + f32, "out")
        # dx cancels against the group's means: roundings of inv w dy, which dx may be smaller than
        size = dy.double().norm().item()
        _off(got[0], ref_g[0], HALF[dtype] + f32, "dx", floor=f32 * size)
        # sums over n rows: errors grow like the root of n, as the sums of signed values do
        for name, a, b in zip(("dw", "db"), got[1:], ref_g[1:]):
            assert a.dtype == torch.float32
            _off(a, b, 4 * f32, name, floor=f32 * size)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("act", ["none", "relu", "silu"])
@pytest.mark.parametrize("affine", [True, False])
def test_activations(act, dtype, affine):
    _check(dtype, [40, 0, 126, 9], 64, 8, act, affine)
    _check(dtype, [4000, 9000], 64, 8, act, affine)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("C,G", [(1, 1), (3, 1), (7, 7), (12, 3), (40, 4), (96, 1), (100, 25), (320, 32), (2052, 4),
                                 (4096, 4096), (1032, 129)])
def test_channels(C, G, dtype):
    _check(dtype, [30, 5, 0, 64], C, G)
    if C <= 320:
        _check(dtype, [70000 // C + 2500, 11], C, G)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("lens", [[16], [8] * 300, [20000], [5000, 0, 5001, 4097], [9000] + [9] * 40])
def test_lengths(lens, dtype):
    _check(dtype, lens, 24, 3)


@pytest.mark.parametrize("dtype", TYPES)
def test_samples_without_pointers(dtype):
    _check(dtype, None, 32, 4, shape=(3, 5, 7, 32))
    _check(dtype, None, 64, 4, shape=(100, 64))
    _check(dtype, None, 16, 4, shape=(2, 90, 120, 16))


@pytest.mark.parametrize("lens", [[50, 30], [30000, 20000]])
def test_a_mean_far_from_zero(lens):
    """The deviation is a 4096th of the mean: E[x^2] - E[x]^2 in 32 bits would have nothing left."""
    g = torch.Generator().manual_seed(1)
    x = torch.randn(sum(lens), 16, generator=g) + 4096.0
    out = group_norm(x.to(DEV), 4, ptr=_ptr(lens, DEV))
    ref = group_norm_reference(x.double(), 4, None, None, _ptr(lens))
    # the mean itself is a 32-bit number: half a step of 4096 against a deviation of 1, and what it
    # adds to every value of a group
    _off(out, ref, 4096 * U32 + 16 * U32, "out")


def test_a_value_alone_in_its_group_passes_no_gradient():
    for dtype in TYPES:
        x = torch.randn(1, 8, dtype=torch.float32).to(DEV, dtype).requires_grad_()
        w = torch.randn(8, device=DEV, requires_grad=True)
        out = group_norm(x, 8, w, ptr=_ptr([1], DEV))
        dx, dw = torch.autograd.grad(out, (x, w), torch.randn_like(out))
        assert not out.any() and not dx.any() and not dw.any()


@pytest.mark.parametrize("lens", [[20, 30], [9000, 7000]])
@pytest.mark.parametrize("dtype", TYPES)
def test_rows_behind_the_last_sequence(dtype, lens):
    n = sum(lens)
    g = torch.Generator().manual_seed(2)
    x, dy = (torch.randn(n + 40, 24, generator=g).to(DEV, dtype) for _ in range(2))
    res = []
    for dirty in (False, True):
        a, d = x.clone(), dy.clone()
        if dirty:
            a[n:], d[n:] = math.nan, math.inf
        w = torch.ones(24, device=DEV, requires_grad=True)
        out = group_norm(a.requires_grad_(), 3, w, ptr=_ptr(lens, DEV), act="silu")
        res.append([out, *torch.autograd.grad(out, (a, w), d)])
    for a, b in zip(*res):
        assert torch.equal(a, b)
    assert not res[0][0][n:].any() and not res[0][1][n:].any()


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("C", [24, 64])
def test_strided_and_misaligned_rows(C, dtype):
    """Views give the values of copies: the sums' order may go by alignment, the values' size not."""
    for lens in ([40, 9], [6000, 7000]):
        n = sum(lens)
        g = torch.Generator().manual_seed(3)
        wide = torch.randn(n, 2 * C + 1, generator=g).to(DEV, dtype)
        dwide = torch.randn(C, n, generator=g).to(DEV, dtype).t()
        res = []
        for copy in (False, True):
            x = wide[:, 1:C + 1]
            x = (x.contiguous() if copy else x).detach().requires_grad_()
            out = group_norm(x, 4, ptr=_ptr(lens, DEV))
            res.append([out, torch.autograd.grad(out, x, dwide.contiguous() if copy else dwide)[0]])
        for a, b in zip(*res):
            _off(a, b.detach().double().cpu(), HALF[dtype] + 64 * U32, "view")


def test_values_that_are_no_numbers_stay_in_their_graph():
    x = torch.randn(90, 16, device=DEV)
    x[40, 3], x[70, 9] = math.nan, math.inf
    out = group_norm(x, 4, ptr=_ptr([30, 20, 40], DEV))
    assert torch.isfinite(out[:30]).all()
    assert torch.isnan(out[30:50, :4]).all() and torch.isfinite(out[30:50, 4:]).all()
    assert torch.isnan(out[50:, 8:12]).all() and torch.isfinite(out[50:, :8]).all()


@pytest.mark.parametrize("lens", [[30, 50], [9000, 7000]])
def test_captured_step_replays(lens):
    n = sum(lens)
    x, dy = (torch.randn(n + 10, 32, device=DEV).requires_grad_(i == 0) for i in range(2))
    w, b = (torch.randn(32, device=DEV).requires_grad_() for _ in range(2))
    ptr = _ptr(lens, DEV)

    def step():
        out = group_norm(x, 4, w, b, ptr=ptr, act="silu")
        return [out.detach(), *torch.autograd.grad(out, (x, w, b), dy)]

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        static = step()
    for i in range(3):
        with torch.no_grad():
            x.copy_(torch.randn(x.shape, generator=torch.Generator().manual_seed(i)))
        ptr.copy_(_ptr([lens[0] - i, lens[1]], DEV))
        graph.replay()
        torch.cuda.synchronize()
        got = [t.clone() for t in static]
        for a, c in zip(got, step()):
            assert torch.equal(a, c), i


def test_pointers_that_do_not_ascend_stay_inside():
    for n in (60, 20000):
        x = torch.randn(n, 32, device=DEV, requires_grad=True)
        for p in ([0, n + 9, 20], [7, -3, n], [0, n, 4]):
            out = group_norm(x, 4, ptr=torch.tensor(p, dtype=torch.int32, device=DEV))
            torch.autograd.grad(out, x, torch.ones_like(out))
    torch.cuda.synchronize()


def test_no_rows():
    x = torch.randn(0, 8, device=DEV, requires_grad=True)
    w = torch.ones(8, device=DEV, requires_grad=True)
    for p in (_ptr([], DEV), _ptr([0, 0], DEV), None):
        out = group_norm(x, 2, w, ptr=p)
        dx, dw = torch.autograd.grad(out, (x, w), torch.zeros_like(out))
        assert out.shape == dx.shape == (0, 8) and not dw.any()


def test_refusals():
    x = torch.zeros(4, 8, device=DEV)
    with pytest.raises(ValueError, match="int32"):
        group_norm(x, 2, ptr=torch.tensor([0, 4], dtype=torch.int32))
    with pytest.raises(ValueError, match="weight is"):
        group_norm(x, 2, torch.ones(8))
    with pytest.raises(ValueError, match="not supported"):
        group_norm(x.double(), 2)


def _refused():
    import test_group_norm as cpu

    for mark in cpu.test_refusals.pytestmark:
        yield from (c for c in mark.args[1] if c[1] != "ascend")


@pytest.mark.parametrize("change,what", list(_refused()))
def test_the_gpu_refuses_what_the_cpu_refuses(change, what):
    a = {"x": torch.zeros(4, 8), "groups": 2, **change}
    with pytest.raises(ValueError, match=what):
        group_norm(**{n: t.to(DEV) if torch.is_tensor(t) else t for n, t in a.items()})


def test_no_sequences():
    """Every row lies behind the last sequence, whatever their number."""
    for n in (5, 50000):
        x = torch.randn(n, 32, device=DEV, requires_grad=True)
        w = torch.ones(32, device=DEV, requires_grad=True)
        out = group_norm(x, 4, w, ptr=_ptr([], DEV))
        dx, dw = torch.autograd.grad(out, (x, w), torch.ones_like(out))
        assert not out.any() and not dx.any() and not dw.any()


def test_offsets_past_32_bits():
    n, C = 530000, 4096  # 2.2e9 values: the last rows lie beyond 2^31 of them
    x = torch.empty(n, C, device=DEV, dtype=torch.bfloat16)
    x[-700:] = torch.randn(700, C, device=DEV).bfloat16()
    x.requires_grad_()
    ptr = torch.tensor([0, 0, 200], dtype=torch.int32, device=DEV) + (n - 700)
    ptr[0] = 0  # the first sequence's rows hold whatever memory held: only the others are looked at
    ptr = torch.cat([ptr, torch.tensor([n], dtype=torch.int32, device=DEV)])
    out = group_norm(x, 32, ptr=ptr, act="silu")
    small = x.detach()[-700:].clone().requires_grad_()
    ref = group_norm(small, 32, ptr=_ptr([0, 200, 500], DEV), act="silu")
    _off(out[-700:], ref.detach().double().cpu(), HALF[torch.bfloat16] + 64 * U32, "out")
    dy = torch.zeros_like(out)
    dy[-700:] = torch.randn(700, C, device=DEV).bfloat16()
    (dx,) = torch.autograd.grad(out, x, dy)
    (rx,) = torch.autograd.grad(ref, small, dy[-700:].clone())
    _off(dx[-700:], rx.double().cpu(), HALF[torch.bfloat16] + 64 * U32, "dx")
