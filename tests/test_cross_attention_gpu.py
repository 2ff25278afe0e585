"""Ragged cross attention on the GPU against the 64-bit oracle: types, head layouts, lengths, masks,
strides, buckets, gradients, capture."""
import math

import pytest
import torch

from cross_attention_util import HALF, check_norm, check_table, norm_tol, oracle, ptr, score_error
from hydragnn_amd.ops.cross_attention import RelativeBuckets, cross_attention

pytestmark = pytest.mark.gpu
DEV = "cuda"
TYPES = [torch.float32, torch.bfloat16, torch.float16]


def _make(dtype, ql, kl, H, Hk, D, pad=3, seed=0):
    g = torch.Generator().manual_seed(seed)
    nq, nk = sum(ql) + pad, sum(kl) + pad
    return [torch.randn(n, h, D, generator=g).to(dtype) for n, h in ((nq, H), (nk, Hk), (nk, Hk), (nq, H))]


def _bias(kind, nq, nk, H, num=16, far=40, seed=1):
    g = torch.Generator().manual_seed(seed)
    rule = RelativeBuckets(num, far, unit=0.5 if kind == "space" else None)
    if kind == "order":
        pos = [torch.arange(n, dtype=torch.int32) % m for n, m in ((nq, 97), (nk, 89))]
    else:  # half of them on a lattice of the unit, where distances lie on borders
        pos = [torch.randn(n, 3, generator=g) * 4 for n in (nq, nk)]
        for p in pos:
            p[::2] = (p[::2] * 2).round() / 2
    return rule, torch.randn(H, num, generator=g), pos


def _check(dtype, ql, kl, H, Hk, D, kind=None, masked=False, train=True, scale=None):
    q, k, v, do = _make(dtype, ql, kl, H, Hk, D)
    mask = torch.rand(k.shape[0], generator=torch.Generator().manual_seed(2)) > 0.4 if masked else None
    more, cpu, names = {}, {}, ["dq", "dk", "dv"]
    dev = [t.to(DEV).requires_grad_(train) for t in (q, k, v)]
    if kind:
        rule, table, pos = _bias(kind, q.shape[0], k.shape[0], H)
        more = {"buckets": rule, "q_pos": pos[0].to(DEV), "k_pos": pos[1].to(DEV),
                "table": table.to(DEV).requires_grad_(train)}
        cpu = {"table": table, "bucket": rule.buckets(*pos)}
        dev.append(more["table"])
        names.append("dtable")
    out = cross_attention(*dev[:3], ptr(ql, DEV), ptr(kl, DEV), scale=scale,
                          key_mask=None if mask is None else mask.to(DEV), **more)
    assert out.dtype == dtype
    ref = oracle(q, k, v, ql, kl, scale=scale, key_mask=mask, d_out=do if train else None, **cpu)
    n = max(ql + kl)
    far = 0.0 if scale is None else score_error(q, k, scale)
    check_norm(out, ref["out"], norm_tol(dtype, D, n, False, train) + far, "out")
    if not train:
        return
    grads = torch.autograd.grad(out, dev, do.to(DEV))
    # where a row's dS are zero by definition (one key), what is left is the roundings' size
    floor = norm_tol(torch.float32, D, n, True, True) * ref["dv"].norm().item()
    for name, g in zip(names, grads):
        if name == "dtable":
            assert g.dtype == torch.float32
            check_table(g, ref, dtype, name, far)
        else:
            assert g.dtype == dtype
            check_norm(g, ref[name], norm_tol(dtype, D, n, True, True) + far, name, floor)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("D", [1, 8, 20, 32, 33, 64, 96, 128])
def test_head_widths(D, dtype):
    _check(dtype, [70, 0, 5], [130, 7, 64], 4, 2, D)
    _check(dtype, [3, 40], [33, 90], 2, 2, D, train=False)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("H,Hk", [(1, 1), (6, 3), (8, 1), (12, 12), (20, 1), (34, 2)])
def test_head_layouts(H, Hk, dtype):
    _check(dtype, [17, 1, 66], [20, 140, 3], H, Hk, 16, kind="order")
    _check(dtype, [1, 1, 2], [20, 700, 3], H, Hk, 40, train=False, masked=True)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("ql,kl", [([1], [1]), ([1] * 70, [9] * 70), ([1, 1, 1], [1, 0, 2000]), ([200], [1]),
                                   ([0, 300, 0], [0, 300, 0]), ([64, 128, 192], [64, 128, 192]),
                                   ([5] * 130, list(range(130))), ([2, 3], [3000, 4100])])
def test_lengths(ql, kl, dtype):
    _check(dtype, ql, kl, 2, 1, 24)
    _check(dtype, ql, kl, 2, 1, 24, train=False)
    _check(dtype, ql, kl, 4, 4, 64, train=False, kind="order")


@pytest.mark.parametrize("train", [True, False])
@pytest.mark.parametrize("masked", [True, False])
@pytest.mark.parametrize("kind", [None, "order", "space"])
@pytest.mark.parametrize("dtype", TYPES)
def test_masks_and_buckets(dtype, kind, masked, train):
    _check(dtype, [90, 1, 0, 33, 16], [40, 3, 8, 0, 129], 4, 2, 32, kind, masked, train)
    _check(dtype, [1, 2, 1, 1], [40, 3, 200, 0], 4, 1, 64, kind, masked, train)


@pytest.mark.parametrize("kind", ["order", "space"])
@pytest.mark.parametrize("num,far", [(4, 3), (64, 2048), (32, 128)])
def test_bucket_sizes(num, far, kind):
    ql, kl = [80, 3], [70, 150]
    q, k, v, do = _make(torch.bfloat16, ql, kl, 2, 2, 128)
    rule, table, pos = _bias(kind, q.shape[0], k.shape[0], 2, num, far)
    if kind == "order":  # far apart, to where a difference passes 32 bits
        pos[0][:4] = torch.tensor([-2 ** 31, 2 ** 31 - 1, -far, far], dtype=torch.int32)
    else:
        pos[0][0], pos[0][1, 0], pos[1][0, 1] = 3e38, math.inf, math.nan
    leaves = [t.to(DEV).requires_grad_() for t in (q, k, v, table)]
    out = cross_attention(*leaves[:3], ptr(ql, DEV), ptr(kl, DEV), table=leaves[3], buckets=rule,
                          q_pos=pos[0].to(DEV), k_pos=pos[1].to(DEV))
    ref = oracle(q, k, v, ql, kl, table=table, bucket=rule.buckets(*pos), d_out=do)
    check_norm(out, ref["out"], norm_tol(torch.bfloat16, 128, 150, False, True), "out")
    check_table(torch.autograd.grad(out, leaves, do.to(DEV))[3], ref, torch.bfloat16, "dtable")


@pytest.mark.parametrize("dtype", TYPES)
def test_one_direction(dtype):
    ql = [50, 9]
    q, k, v, do = _make(dtype, ql, ql, 2, 2, 16, pad=0)
    rule, table = RelativeBuckets(8, 20, bidirectional=False), torch.randn(2, 8)
    pos = torch.arange(59, dtype=torch.int32)
    out = cross_attention(q.to(DEV), k.to(DEV), v.to(DEV), ptr(ql, DEV), ptr(ql, DEV), table=table.to(DEV),
                          buckets=rule, q_pos=pos.to(DEV), k_pos=pos.to(DEV))
    ref = oracle(q, k, v, ql, ql, table=table, bucket=rule.buckets(pos, pos))
    check_norm(out, ref["out"], norm_tol(dtype, 16, 50, False, False), "out")


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("D", [8, 20, 64])
def test_strided_and_misaligned_views(D, dtype):
    """Views of packed projections and rows that begin anywhere give the very bits of copies."""
    ql, kl, H = [40, 70], [30, 50], 4
    g = torch.Generator().manual_seed(3)
    qkv = torch.randn(111, 3, H, D + 1, generator=g).to(dtype).to(DEV)
    q, k, v = (qkv[1:, i, :, 1:] for i in range(3))
    k, v = k[:83], v[:83]
    do = torch.randn(110, D, H, generator=g).to(dtype).to(DEV).transpose(1, 2)  # its last stride is not 1
    res = []
    for copy in (False, True):
        leaves = [(t.contiguous() if copy else t).detach().requires_grad_() for t in (q, k, v)]
        out = cross_attention(*leaves, ptr(ql, DEV), ptr(kl, DEV))
        res.append([out, *torch.autograd.grad(out, leaves, do.contiguous() if copy else do)])
    for a, b in zip(*res):
        assert torch.equal(a, b)
    ref = oracle(q, k, v, ql, kl, d_out=do)
    check_norm(res[0][0], ref["out"], norm_tol(dtype, D, 70, False, True), "out")


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("train", [True, False])
def test_nothing_masked_or_behind_the_last_sequence_is_seen(dtype, train):
    ql, kl = [1, 40, 3], [70, 33, 200]
    q, k, v, do = (t.to(DEV) for t in _make(dtype, ql, kl, 4, 2, 24))
    mask = torch.rand(k.shape[0], generator=torch.Generator().manual_seed(4)).to(DEV) > 0.5
    mask[70:103] = False  # all keys of the second sequence
    rule, table, pos = _bias("space", q.shape[0], k.shape[0], 4)
    pos = [p.to(DEV) for p in pos]
    res = []
    for dirty in (False, True):
        a, b, c, d, kp = (t.clone() for t in (q, k, v, do, pos[1]))
        if dirty:
            for t in (b, c):
                bad = torch.tensor([math.nan, math.inf, -math.inf], device=DEV, dtype=dtype)
                t[~mask] = bad[torch.arange(int((~mask).sum()), device=DEV) % 3].view(-1, 1, 1)
                t[303:] = math.nan
            a[44:], d[44:], kp[303:], kp[:303][~mask[:303]] = math.nan, math.inf, math.nan, math.inf
        leaves = [t.requires_grad_(train) for t in (a, b, c, table.to(DEV))]
        out = cross_attention(*leaves[:3], ptr(ql, DEV), ptr(kl, DEV), key_mask=mask, table=leaves[3], buckets=rule,
                              q_pos=pos[0], k_pos=kp)
        res.append([out, *(torch.autograd.grad(out, leaves, d) if train else ())])
    for a, b in zip(*res):
        assert torch.equal(a, b)
    out = res[1][0]
    assert torch.equal(out[1:41], torch.zeros_like(out[1:41])) and torch.equal(out[44:], torch.zeros_like(out[44:]))
    if train:
        dq, dk, dv = res[1][1:4]
        assert not dq[1:41].any() and not dq[44:].any() and not dk[~mask].any() and not dv[303:].any()


def test_a_single_key_passes_no_gradient_to_the_scores():
    """With one key p is 1 whatever the score: dq, dk and the table's gradient are zeros, not roundings."""
    for dtype in TYPES:
        q, k, v, do = (t.to(DEV) for t in _make(dtype, [9, 70], [1, 1], 4, 2, 64, pad=0))
        rule, table, pos = _bias("order", 79, 2, 4)
        leaves = [t.requires_grad_() for t in (q, k, v, table.to(DEV))]
        out = cross_attention(*leaves[:3], ptr([9, 70], DEV), ptr([1, 1], DEV), table=leaves[3], buckets=rule,
                              q_pos=pos[0].to(DEV), k_pos=pos[1].to(DEV))
        dq, dk, _, dt = torch.autograd.grad(out, leaves, do)
        assert not dq.any() and not dk.any() and not dt.any()


@pytest.mark.parametrize("dtype", TYPES)
def test_scores_far_apart(dtype):
    """Scores of some thousands: the running maximum, not the exponential, carries them."""
    ql, kl = [33, 1], [200, 300]
    q, k, v, _ = _make(dtype, ql, kl, 2, 2, 64)
    q, k = q * 16, k * 16
    out = cross_attention(*(t.to(DEV) for t in (q, k, v)), ptr(ql, DEV), ptr(kl, DEV))
    ref = oracle(q, k, v, ql, kl)["out"]
    # a score of size s is off by s (sqrt(D) + 8) steps of 32 bits, its p by as much, relatively
    size = (q.float().norm(dim=-1).max() * k.float().norm(dim=-1).max() / 8).item()
    check_norm(out, ref, norm_tol(dtype, 64, 300, False, False) + 4 * 2.0 ** -24 * size * 16, "out")


def test_runs_give_the_same_bits():
    ql, kl = [300, 7, 64], [500, 1, 90]
    q, k, v, do = (t.to(DEV) for t in _make(torch.bfloat16, ql, kl, 8, 2, 64))
    rule, table, pos = _bias("order", q.shape[0], k.shape[0], 8)
    leaves = [t.requires_grad_() for t in (q, k, v, table.to(DEV))]
    runs = []
    for _ in range(3):
        out = cross_attention(*leaves[:3], ptr(ql, DEV), ptr(kl, DEV), table=leaves[3], buckets=rule,
                              q_pos=pos[0].to(DEV), k_pos=pos[1].to(DEV))
        runs.append([out, *torch.autograd.grad(out, leaves, do)])
    for other in runs[1:]:
        for a, b in zip(runs[0], other):
            assert torch.equal(a, b)


def test_leaves_that_want_no_gradient():
    ql, kl = [30, 2], [20, 50]
    q, k, v, do = (t.to(DEV) for t in _make(torch.float32, ql, kl, 2, 1, 16))
    full = [t.clone().requires_grad_() for t in (q, k, v)]
    ref = torch.autograd.grad(cross_attention(*full, ptr(ql, DEV), ptr(kl, DEV)), full, do)
    for want in range(3):
        leaves = [t.clone().requires_grad_(i == want) for i, t in enumerate((q, k, v))]
        out = cross_attention(*leaves, ptr(ql, DEV), ptr(kl, DEV))
        assert torch.equal(torch.autograd.grad(out, leaves[want], do)[0], ref[want])


def test_a_table_in_the_rows_type():
    ql = [20]
    q, k, v, do = (t.to(DEV) for t in _make(torch.bfloat16, ql, ql, 2, 2, 16))
    rule, table, pos = _bias("order", 23, 23, 2)
    t16 = table.to(DEV).bfloat16().requires_grad_()
    t32 = t16.detach().float().requires_grad_()
    outs = [cross_attention(q, k, v, ptr(ql, DEV), ptr(ql, DEV), table=t, buckets=rule, q_pos=pos[0].to(DEV),
                            k_pos=pos[1].to(DEV)) for t in (t16, t32)]
    assert torch.equal(*outs)
    g16, g32 = (torch.autograd.grad(o, t, do)[0] for o, t in zip(outs, (t16, t32)))
    assert g16.dtype == torch.bfloat16 and torch.equal(g16, g32.bfloat16())


def test_another_stream_and_two_calls_at_once():
    ql, kl = [200, 30], [300, 700]
    sets = [[t.to(DEV) for t in _make(torch.bfloat16, ql, kl, 4, 4, 64, seed=s)] for s in range(2)]
    qp, kp = ptr(ql, DEV), ptr(kl, DEV)
    one = [cross_attention(*s[:3], qp, kp) for s in sets]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in sets]
    two = []
    for st, s in zip(streams, sets):
        with torch.cuda.stream(st):
            two.append(cross_attention(*s[:3], qp, kp))
    torch.cuda.synchronize()
    for a, b in zip(one, two):
        assert torch.equal(a, b)


@pytest.mark.parametrize("ql,kl", [([40, 70], [60, 90]), ([1, 1], [3000, 5000])])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_captured_step_replays(dtype, ql, kl):
    q, k, v, do = (t.to(DEV) for t in _make(dtype, ql, kl, 4, 2, 32))
    rule, table, pos = _bias("order", q.shape[0], k.shape[0], 4)
    leaves = [t.requires_grad_() for t in (q, k, v, table.to(DEV))]
    qp, kp = ptr(ql, DEV), ptr(kl, DEV)
    args = dict(buckets=rule, q_pos=pos[0].to(DEV), k_pos=pos[1].to(DEV))

    def step():
        out = cross_attention(*leaves[:3], qp, kp, table=leaves[3], **args)
        res = [out.detach(), *torch.autograd.grad(out, leaves, do)]
        with torch.no_grad():
            res.append(cross_attention(*leaves[:3], qp, kp, table=leaves[3], **args))
        return res

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        static = step()
    lens = [(ql, kl), ([ql[0] - 1, ql[1]], [kl[0] - 30, kl[1]]), ([0, ql[1]], [kl[0], 2])]
    for i, (a, b) in enumerate(lens):  # other lengths and values in the same buffers
        with torch.no_grad():
            for t in leaves:
                t.copy_(torch.randn(t.shape, generator=torch.Generator().manual_seed(10 + i)).to(t))
        qp.copy_(ptr(a, DEV))
        kp.copy_(ptr(b, DEV))
        graph.replay()
        torch.cuda.synchronize()
        got = [t.clone() for t in static]
        for x, y in zip(got, step()):
            assert torch.equal(x, y), i


def test_pointers_that_do_not_ascend_stay_inside():
    """Documented as unspecified: every index is clamped, and the call returns."""
    q, k, v, do = (t.to(DEV).requires_grad_() for t in _make(torch.float32, [40, 30], [50, 20], 2, 2, 16))
    for a, b in (([0, 90, 20], [0, 30, 60]), ([5, -7, 70], [0, 1000, 70]), ([0, 40, 70], [60, 20, 5])):
        out = cross_attention(q, k, v, torch.tensor(a, dtype=torch.int32, device=DEV),
                              torch.tensor(b, dtype=torch.int32, device=DEV))
        torch.autograd.grad(out, (q, k, v), do)
    torch.cuda.synchronize()


def test_refusals():
    q, k, v, _ = (t.to(DEV) for t in _make(torch.float32, [4], [4], 2, 2, 8))
    p = ptr([4], DEV)
    with pytest.raises(ValueError, match="is on"):
        cross_attention(q, k.cpu(), v, p, p)
    with pytest.raises(ValueError, match="is on"):
        cross_attention(q, k, v, p.cpu(), p)
    with pytest.raises(ValueError, match="not supported"):
        cross_attention(q.double(), k.double(), v.double(), p, p)
    out = cross_attention(q.requires_grad_(), k, v, p, p)
    (g,) = torch.autograd.grad(out.sum(), q, create_graph=True)
    with pytest.raises(RuntimeError):
        torch.autograd.grad(g.sum(), q)
    assert HALF[torch.float32] == torch.finfo(torch.float32).eps / 2


def _refused():
    import test_cross_attention as cpu

    for mark in cpu.test_refusals.pytestmark:
        yield from (c for c in mark.args[1] if c[1] != "ascend")


@pytest.mark.parametrize("change,what", list(_refused()))
def test_the_gpu_refuses_what_the_cpu_refuses(change, what):
    import test_cross_attention as cpu

    q, k, v, _, qp, kp = cpu._inputs(dtype=torch.float32)
    a = {"q": q, "k": k, "v": v, "q_ptr": qp, "k_ptr": kp, **change}
    with pytest.raises(ValueError, match=what):
        cross_attention(**{n: t.to(DEV) if torch.is_tensor(t) else t for n, t in a.items()})


def test_no_sequences_and_no_rows():
    q, k, v, do = (t.to(DEV).requires_grad_() for t in _make(torch.bfloat16, [300], [200], 2, 1, 32))
    none = ptr([], DEV)
    out = cross_attention(q, k, v, none, none)
    assert not out.any() and not any(g.any() for g in torch.autograd.grad(out, (q, k, v), do.detach()))
    for a, b in ((q[:0], k), (q, k[:0])):
        a, b = a.detach().requires_grad_(), b.detach().requires_grad_()
        p, r = ptr([a.shape[0]], DEV), ptr([b.shape[0]], DEV)
        out = cross_attention(a, b, b, p, r)
        assert out.shape == a.shape and not out.any()
        assert not any(g.any() for g in torch.autograd.grad(out, (a, b), torch.ones_like(out)))


@pytest.mark.parametrize("rows", [1, 100])
def test_offsets_past_32_bits(rows):
    """The last sequence of a key cache of 2.5e9 elements, by both forms, against a copy of it alone."""
    n, Hk, D, last = 1200000, 16, 128, 100
    k, v = (torch.zeros(n, Hk, D, device=DEV, dtype=torch.bfloat16) for _ in range(2))
    for t in (k, v):
        t[-last:] = torch.randn(last, Hk, D, device=DEV).bfloat16()
    q, do = (torch.randn(rows, Hk, D, device=DEV).bfloat16() for _ in range(2))
    mask = torch.ones(n, dtype=torch.bool, device=DEV)
    mask[-3] = False
    res = []
    for kk, vv, m, first in ((k, v, mask, n - last), (k[-last:].clone(), v[-last:].clone(), mask[-last:].clone(), 0)):
        leaves = [t.requires_grad_() for t in (q.clone(), kk, vv)]
        kp = torch.tensor([0, first, first + last], dtype=torch.int32, device=DEV)
        qp = torch.tensor([0, 0, rows], dtype=torch.int32, device=DEV)
        out = cross_attention(*leaves, qp, kp, key_mask=m)
        g = torch.autograd.grad(out, leaves, do)
        res.append([out.detach(), g[0], g[1][-last:].clone(), g[2][-last:].clone()])
        del out, g, leaves
    # the forms go by sizes, so the sums' order may differ: each side's own roundings
    for a, b in zip(*res):
        check_norm(a, b.double().cpu(), 2 * norm_tol(torch.bfloat16, D, last, True, True), "far")


def test_captured_step_with_much_lds():
    """Heads of 128 with 64 buckets: the kernels' LDS passes 64 KB, which they have to be told of."""
    ql, kl = [40, 70], [60, 90]
    q, k, v, do = (t.to(DEV) for t in _make(torch.bfloat16, ql, kl, 2, 2, 128))
    rule, table, pos = _bias("order", q.shape[0], k.shape[0], 2, 64, 2048)
    leaves = [t.requires_grad_() for t in (q, k, v, table.to(DEV))]
    qp, kp, a, b = ptr(ql, DEV), ptr(kl, DEV), pos[0].to(DEV), pos[1].to(DEV)

    def step():
        out = cross_attention(*leaves[:3], qp, kp, table=leaves[3], buckets=rule, q_pos=a, k_pos=b)
        return [out.detach(), *torch.autograd.grad(out, leaves, do)]

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
            for t in leaves:
                t.copy_(torch.randn(t.shape, generator=torch.Generator().manual_seed(20 + i)).to(t))
        graph.replay()
        torch.cuda.synchronize()
        got = [t.clone() for t in static]
        for x, y in zip(got, step()):
            assert torch.equal(x, y), i


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("scale", [0.0, -0.3, 2.0])
def test_scales(scale, dtype):
    _check(dtype, [40, 3], [70, 130], 4, 2, 32, scale=scale, masked=True)
    _check(dtype, [1, 2], [300, 40], 4, 2, 64, kind="order", scale=scale, masked=True)
