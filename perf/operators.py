"""Workloads of the attention and normalisation operators over ragged batches.

Three operators, each forward and as a training step:

* ``attend``: attention of one ragged batch's rows on another's (``cross_attention``): the queries of
  sequence s see the keys of sequence s, whose number is another one;
* ``bias``: the same with a learned relative position bias, ``table[head, bucket(q_pos, k_pos)]``,
  whose gradient a training step returns too;
* ``norm``: group norm over the rows of each sequence, channels last, with an activation.

``own`` chooses between the framework's operators and their plain form in torch operations.
"""
import math
import random

import torch

own = False

DTYPES = {"fp32": torch.float32, "bf16": torch.bfloat16, "fp16": torch.float16}


def _attend(name, train, dtype, seqs, q_len, k_len, heads, kv_heads, dim, ragged=True, masked=0.0, **more):
    c = {"op": "attend", "train": train, "dtype": dtype, "seqs": seqs, "q_len": q_len, "k_len": k_len,
         "heads": heads, "kv_heads": kv_heads, "dim": dim, "ragged": ragged, "masked": masked}
    if more:
        c.update(op="bias", **more)
    if name:
        c["name"] = name
    return c


def _norm(name, train, dtype, seqs, rows, channels, groups, act):
    c = {"op": "norm", "train": train, "dtype": dtype, "seqs": seqs, "rows": rows, "channels": channels,
         "groups": groups, "act": act}
    if name:
        c["name"] = name
    return c


def listed():
    return [
        # one read-out query for each of 32 molecules of 20 to 126 atoms, 8 heads of 8: latency alone
        _attend("readout fp32", False, "fp32", 32, 1, 126, 8, 8, 8),
        # one token a sequence over long encoder states, 4 query heads to a key head: bytes of the states
        _attend("token bf16", False, "bf16", 16, 1, 16384, 32, 8, 128),
        # a batch of prompts on encoder states with padding keys among them
        _attend("prompt bf16", False, "bf16", 8, 1024, 2048, 16, 16, 64, masked=0.1),
        # the atoms of 32 slabs attend within their slab: the graph transformer's own training step
        _attend("graphs train fp32", True, "fp32", 32, 126, 126, 8, 8, 8),
        # a decoder's cross attention, 4 query heads to a key head, training
        _attend("decoder train bf16", True, "bf16", 8, 1024, 2048, 16, 4, 64, masked=0.1),
        # single precision training on middling lengths
        _attend("decoder train fp32", True, "fp32", 8, 512, 777, 8, 8, 64),
        # distance buckets over the atoms' positions, the graph transformer's training step
        _attend("distance train fp32", True, "fp32", 32, 126, 126, 8, 8, 8, pos="space", buckets=32, far=64),
        # order buckets of a sequence encoder, forward
        _attend("order bf16", False, "bf16", 4, 2048, 2048, 16, 16, 64, pos="order", buckets=32, far=128),
        # the same, training
        _attend("order train bf16", True, "bf16", 4, 2048, 2048, 16, 16, 64, pos="order", buckets=32, far=128),
        # node features of 32 graphs between two layers
        _norm("graphs norm train fp32", True, "fp32", 32, 126, 64, 8, "relu"),
        # wide features of large structures, inference
        _norm("states norm bf16", False, "bf16", 16, 8192, 512, 32, "silu"),
        # the same features in training, few long sequences
        _norm("states norm train fp32", True, "fp32", 4, 20000, 320, 32, "silu"),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    most = [work(c) for c in listed()]
    flops, size = max(w["flops"] for w in most), max(w["bytes"] for w in most)
    while True:
        if rng.random() < 0.3:
            groups = rng.choice([1, 2, 4, 8, 16, 32])
            c = _norm(None, rng.random() < 0.6, rng.choice(["fp32", "bf16", "fp16"]), _log_int(rng, 1, 64),
                      _log_int(rng, 1, 20000), groups * _log_int(rng, 1, 32), groups,
                      rng.choice(["none", "relu", "silu"]))
        else:
            kv = rng.choice([1, 2, 4, 8, 16])
            train = rng.random() < 0.6
            few = rng.random() < 0.3
            more = {}
            if rng.random() < 0.4:
                more = {"pos": rng.choice(["space", "order"]), "buckets": rng.choice([8, 16, 32, 64]),
                        "far": rng.randint(40, 512)}
            c = _attend(None, train, rng.choice(["fp32", "bf16", "fp16"]), _log_int(rng, 1, 64),
                        rng.randint(1, 4) if few else _log_int(rng, 1, 2048),
                        _log_int(rng, 1, 2048 if train else 16384), kv * rng.choice([1, 1, 2, 4]), kv,
                        rng.choice([8, 16, 20, 32, 40, 64, 96, 128]), rng.random() < 0.7,
                        rng.choice([0.0, 0.0, 0.1, 0.4]), **more)
        w = work(c)
        # the plain form's scores of a drawn case stay within a few gigabytes
        pairs = c["seqs"] * c.get("q_len", 0) * c.get("k_len", 0)
        if w["flops"] <= flops and w["bytes"] <= size and pairs * c.get("heads", 0) < 6e8 and \
                pairs * c.get("buckets", 0) < 1.6e9:
            return c


def _lengths(longest, seqs, ragged, salt):
    """Lengths of a case's sequences: they go by the case alone, so that its work is known."""
    if not ragged or longest == 1:
        return [longest] * seqs
    rng = random.Random(longest * 131 + seqs * 7 + salt)
    lens = [rng.randint(max(1, longest // 6), longest) for _ in range(seqs)]
    lens[rng.randrange(seqs)] = longest
    return lens


def _sizes(case):
    if case["op"] == "norm":
        return _lengths(case["rows"], case["seqs"], True, 1), None
    ql = _lengths(case["q_len"], case["seqs"], case["ragged"], 2)
    if case["q_len"] == case["k_len"]:
        return ql, list(ql)
    kl = _lengths(case["k_len"], case["seqs"], case["ragged"], 3)
    if case["ragged"] and case["seqs"] >= 8:
        kl[case["seqs"] // 2] = 0  # a request whose encoder saw nothing
    return ql, kl


def work(case):
    ql, kl = _sizes(case)
    b = 4 if case["dtype"] == "fp32" else 2
    if case["op"] == "norm":
        n = sum(ql) * case["channels"]
        # forward: x in, y out; training also the output's gradient in and x's out
        return {"bytes": n * b * (4 if case["train"] else 2) + 16 * case["channels"],
                "flops": n * (30 if case["train"] else 12)}
    keep = 1.0 - case["masked"]
    pairs = sum(i * j for i, j in zip(ql, kl)) * keep * case["heads"]
    qe, ke = sum(ql) * case["heads"] * case["dim"], sum(kl) * keep * case["kv_heads"] * case["dim"]
    # forward: q, k, v in, out; training: the output's gradient in and three gradients out as well
    size = (2 * qe + 2 * ke + (2 * qe + 2 * ke if case["train"] else 0)) * b
    # a product of the forward is 2 D operations a pair: 2 of them, and 4 more in the backward
    flops = pairs * case["dim"] * (12 if case["train"] else 4)
    if case["op"] == "bias":
        coords = 3 if case["pos"] == "space" else 1
        size += 4 * coords * (sum(ql) + sum(kl)) + 4 * case["heads"] * case["buckets"] * (2 if case["train"] else 1)
        flops += pairs * (2 if case["train"] else 1)
    return {"bytes": float(size), "flops": float(flops)}


UNIT = 0.25  # of the distance buckets


def _ptr(lens, dev):
    p = [0]
    for n in lens:
        p.append(p[-1] + n)
    return torch.tensor(p, dtype=torch.int32, device=dev)


def prepare(case, seed):
    dev = torch.device("cuda")
    g = torch.Generator(device=dev)
    g.manual_seed(int(seed))
    t = DTYPES[case["dtype"]]
    ql, kl = _sizes(case)

    def randn(*shape):
        return torch.randn(*shape, generator=g, device=dev)

    s = {"case": case, "q_ptr": _ptr(ql, dev), "most_q": max(ql)}
    if case["op"] == "norm":
        c = case["channels"]
        # features whose channels lie off zero, each by its own amount
        s["x"] = (randn(sum(ql), c) * (0.5 + randn(c).abs()) + 2.0 * randn(c)).to(t)
        s["weight"], s["bias"] = 1.0 + 0.3 * randn(c), 0.3 * randn(c)
        if case["train"]:
            s["d_out"] = randn(sum(ql), c).to(t)
            s["leaves"] = [s[n].requires_grad_() for n in ("x", "weight", "bias")]
        return s
    h, hk, d = case["heads"], case["kv_heads"], case["dim"]
    pad = 5 if case["ragged"] else 0  # rows behind the last sequence, as a padded batch has them
    nq, nk = sum(ql) + pad, sum(kl) + pad
    s.update(k_ptr=_ptr(kl, dev), most_k=max(kl))
    s["q"], s["k"], s["v"] = randn(nq, h, d).to(t), randn(nk, hk, d).to(t), randn(nk, hk, d).to(t)
    s["key_mask"] = None
    if case["masked"]:
        s["key_mask"] = torch.rand(nk, generator=g, device=dev) >= case["masked"]
    names = ["q", "k", "v"]
    if case["op"] == "bias":
        s["table"] = randn(h, case["buckets"])
        names.append("table")
        if case["pos"] == "space":
            side = 3.0 * max(max(kl), 1) ** (1 / 3)  # atoms at about the density of a solid
            s["k_pos"] = torch.rand(nk, 3, generator=g, device=dev) * side
            s["q_pos"] = s["k_pos"].clone() if ql == kl else torch.rand(nq, 3, generator=g, device=dev) * side
        else:
            s["q_pos"] = torch.cat([torch.arange(n, dtype=torch.int32, device=dev) for n in ql + [pad]])
            s["k_pos"] = torch.cat([torch.arange(n, dtype=torch.int32, device=dev) for n in kl + [pad]])
    if case["train"]:
        s["d_out"] = randn(nq, h, d).to(t)
        s["leaves"] = [s[n].requires_grad_() for n in names]
    return s


def run(state):
    case = state["case"]
    if own:
        return _run_own(state, case)
    with torch.no_grad():
        return _plain_norm(state, case) if case["op"] == "norm" else _plain_attend(state, case)


def _run_own(s, case):
    if case["op"] == "norm":
        from hydragnn_amd.ops.norm import group_norm

        out = group_norm(s["x"], case["groups"], s["weight"], s["bias"], ptr=s["q_ptr"], act=case["act"])
    else:
        from hydragnn_amd.ops.cross_attention import RelativeBuckets, cross_attention

        more = {}
        if case["op"] == "bias":
            rule = RelativeBuckets(case["buckets"], case["far"], unit=UNIT if case["pos"] == "space" else None)
            more = {"table": s["table"], "buckets": rule, "q_pos": s["q_pos"], "k_pos": s["k_pos"]}
        out = cross_attention(s["q"], s["k"], s["v"], s["q_ptr"], s["k_ptr"], key_mask=s["key_mask"], **more)
    if not case["train"]:
        return [out]
    return [out] + list(torch.autograd.grad(out, s["leaves"], s["d_out"]))


# ---------------------------------------------------------------------------- plain forms


def _spread(ptr, longest, rows):
    """Row numbers of a padded [sequences, longest] layout, and which of them are there."""
    at = ptr[:-1].long().view(-1, 1) + torch.arange(longest, device=ptr.device).view(1, -1)
    there = at < ptr[1:].long().view(-1, 1)
    return at.clamp(max=max(rows - 1, 0)), there


def _collect(padded, at, there, rows):
    """The padded layout's rows at their places, zeros where no sequence is."""
    out = padded.new_zeros((rows,) + padded.shape[2:])
    out[at[there]] = padded[there]
    return out


def _bucket(q_pos, k_pos, case):
    """Bucket numbers [..., Lq, Lk]: exact ones for near pairs, spread over the logarithm for far ones."""
    count, far = case["buckets"], case["far"]
    if case["pos"] == "space":
        diff = k_pos.double().unsqueeze(-3) - q_pos.double().unsqueeze(-2)
        dist = torch.sqrt(diff[..., 0] * diff[..., 0] + diff[..., 1] * diff[..., 1] + diff[..., 2] * diff[..., 2])
        n, first = torch.floor(dist / UNIT), 0
    else:
        count = count // 2
        rel = k_pos.double().unsqueeze(-2) - q_pos.double().unsqueeze(-1)
        n, first = rel.abs(), (rel > 0).long() * count
    near = count // 2
    n = n.clamp(max=far)
    # 1e-9 keeps the powers that lie on a border on its upper side
    grown = near + torch.floor(torch.log(n.clamp(min=near) / near) / math.log(far / near) * (count - near) + 1e-9)
    return first + torch.where(n < near, n, grown.clamp(max=count - 1)).long()


def _plain_attend(s, case):
    h, hk, d = case["heads"], case["kv_heads"], case["dim"]
    nq, nk, g = s["q"].shape[0], s["k"].shape[0], h // hk
    qi, q_there = _spread(s["q_ptr"], s["most_q"], nq)
    ki, k_there = _spread(s["k_ptr"], s["most_k"], nk)
    n, lq, lk = qi.shape[0], qi.shape[1], ki.shape[1]
    keep = k_there if s["key_mask"] is None else k_there & s["key_mask"][ki]

    def heads(t, at, groups):  # [rows, H, D] -> [S, Hk, groups * L, D]
        x = t[at].float().view(at.shape[0], at.shape[1], hk, groups, d)
        return x.permute(0, 2, 3, 1, 4).reshape(at.shape[0], hk, groups * at.shape[1], d)

    q, k, v = heads(s["q"], qi, g), heads(s["k"], ki, 1), heads(s["v"], ki, 1)
    scale = 1.0 / math.sqrt(d)
    score = torch.matmul(q, k.transpose(2, 3).contiguous()) * scale  # [S, Hk, G * Lq, Lk]
    bucket = None
    if case["op"] == "bias":
        bucket = _bucket(s["q_pos"][qi], s["k_pos"][ki], case)  # [S, Lq, Lk]
        score += s["table"].t()[bucket].permute(0, 3, 1, 2).reshape(score.shape)
    score.masked_fill_(~keep.view(n, 1, 1, lk), float("-inf"))
    top = score.amax(-1, keepdim=True).clamp(min=-3e38)
    p = torch.exp(score - top)
    del score
    p /= p.sum(-1, keepdim=True).clamp(min=1e-30)  # a row without keys gives zeros
    p *= q_there.view(n, 1, 1, lq, 1).expand(n, hk, g, lq, 1).reshape(n, hk, g * lq, 1)

    def rows(x, at, there, groups, count, like):  # back to [rows, H, D]
        x = x.view(n, hk, groups, at.shape[1], d).permute(0, 3, 1, 2, 4).reshape(n, at.shape[1], hk * groups, d)
        return _collect(x, at, there, count).to(like.dtype)

    out = rows(torch.matmul(p, v), qi, q_there, g, nq, s["q"])
    if not case["train"]:
        return [out]
    do = heads(s["d_out"], qi, g)
    dv = torch.matmul(p.transpose(2, 3).contiguous(), do)
    ds = torch.matmul(do, v.transpose(2, 3).contiguous())
    ds -= (p * ds).sum(-1, keepdim=True)
    ds *= p
    del p
    dq = torch.matmul(ds, k) * scale
    dk = torch.matmul(ds.transpose(2, 3).contiguous(), q) * scale
    res = [out, rows(dq, qi, q_there, g, nq, s["q"]), rows(dk, ki, k_there, 1, nk, s["k"]),
           rows(dv, ki, k_there, 1, nk, s["v"])]
    if bucket is not None:  # a row's sums by bucket, and the long sums over all rows in 64 bits
        hot = (bucket.unsqueeze(-1) == torch.arange(case["buckets"], device=bucket.device)).float()
        by_row = ds.view(n, h, lq, lk).transpose(1, 2).contiguous()
        res.append(torch.matmul(by_row, hot).double().sum((0, 1)).float())
    return res


def _plain_norm(s, case):
    x, w, b, ptr = s["x"], s["weight"], s["bias"], s["q_ptr"]
    rows, c = x.shape
    g = case["groups"]
    at, there = _spread(ptr, s["most_q"], rows)
    n, longest = at.shape
    here = there.view(n, longest, 1, 1).float()
    size = (ptr[1:] - ptr[:-1]).float().view(n, 1, 1, 1) * (c // g)
    xs = x[at].float().view(n, longest, g, c // g)
    mean = (xs * here).sum((1, 3), keepdim=True) / size
    xc = (xs - mean) * here
    inv = torch.rsqrt((xc * xc).sum((1, 3), keepdim=True) / size + 1e-5)
    xh = xc * inv
    z = xh * w.view(g, c // g) + b.view(g, c // g)
    sig = torch.sigmoid(z)
    y = {"none": z, "relu": z.clamp(min=0), "silu": z * sig}[case["act"]]
    out = _collect(y.reshape(n, longest, c), at, there, rows).to(x.dtype)
    if not case["train"]:
        return [out]
    dy = s["d_out"][at].float().view(n, longest, g, c // g) * here
    if case["act"] == "relu":
        dy = dy * (z > 0)
    elif case["act"] == "silu":
        dy = dy * (sig + z * sig * (1 - sig))
    dw = (dy * xh).double().sum((0, 1)).reshape(c).float()
    db = dy.double().sum((0, 1)).reshape(c).float()
    dxh = dy * w.view(g, c // g)
    m1 = dxh.sum((1, 3), keepdim=True) / size
    m2 = (dxh * xh).sum((1, 3), keepdim=True) / size
    dx = inv * (dxh - m1 - xh * m2)
    return [out, _collect(dx.reshape(n, longest, c), at, there, rows).to(x.dtype), dw, db]


# ---------------------------------------------------------------------------- 64 bits


def _exact_buckets(case):
    """The bucket of each whole distance 0..far, in whole numbers only."""
    count = case["buckets"] if case["pos"] == "space" else case["buckets"] // 2
    near, far = count // 2, case["far"]
    res, b = [], 0
    for n in range(far + 1):
        if n < near:
            b = n
        else:
            b = max(b, near)
            # (n / near) ** (count - near) >= (far / near) ** (b + 1 - near), by whole numbers
            while b + 1 < count and n ** (count - near) * near ** (b + 1 - near) >= \
                    far ** (b + 1 - near) * near ** (count - near):
                b += 1
        res.append(b)
    return res


def exact(case, seed):
    s = prepare(case, seed)
    ql, kl = _sizes(case)
    leaves = [t.detach().double().requires_grad_() for t in s.get("leaves", [])]
    if case["op"] == "norm":
        x, w, b = leaves or [s[n].double() for n in ("x", "weight", "bias")]
        parts, at = [], 0
        for n in ql:
            part = x[at:at + n].view(n, case["groups"], -1)
            var, mean = torch.var_mean(part, dim=(0, 2), unbiased=False, keepdim=True)
            z = ((part - mean) / torch.sqrt(var + 1e-5)).reshape(n, -1) * w + b
            parts.append(z if case["act"] == "none" else torch.relu(z) if case["act"] == "relu"
                         else z / (1 + torch.exp(-z)))
            at += n
        out = torch.cat(parts)
    else:
        t = leaves or [s[n].double() for n in (["q", "k", "v", "table"] if case["op"] == "bias" else ["q", "k", "v"])]
        q, k, v = t[:3]
        g = case["heads"] // case["kv_heads"]
        if case["op"] == "bias":
            whole = torch.tensor(_exact_buckets(case), device=q.device)
        parts, a, c = [], 0, 0
        for n, m in zip(ql, kl):
            keep = torch.arange(c, c + m, device=q.device)
            if s["key_mask"] is not None:
                keep = keep[s["key_mask"][c:c + m]]
            if n and keep.numel():
                ks, vs = k[keep].repeat_interleave(g, 1), v[keep].repeat_interleave(g, 1)
                score = torch.matmul(q[a:a + n].transpose(0, 1), ks.permute(1, 2, 0)) / math.sqrt(case["dim"])
                if case["op"] == "bias":
                    qp, kp = s["q_pos"][a:a + n].double(), s["k_pos"][keep].double()
                    if case["pos"] == "space":
                        d = [kp[:, i].view(1, -1) - qp[:, i].view(-1, 1) for i in range(3)]
                        far = torch.sqrt(d[0] * d[0] + d[1] * d[1] + d[2] * d[2]) / UNIT
                        code = whole[far.clamp(max=case["far"]).long()]
                    else:
                        rel = (kp.view(1, -1) - qp.view(-1, 1)).long()
                        code = whole[rel.abs().clamp(max=case["far"])] + (rel > 0) * (case["buckets"] // 2)
                    score = score + t[3][:, code]
                parts.append(torch.matmul(torch.softmax(score, -1), vs.transpose(0, 1)).transpose(0, 1))
            else:
                parts.append(q[a:a + n] * 0.0)
            a, c = a + n, c + m
        parts.append(q[a:] * 0.0)  # rows behind the last sequence
        out = torch.cat(parts)
    if not case["train"]:
        return [out.detach()]
    return [out.detach()] + list(torch.autograd.grad(out, leaves, s["d_out"].double()))
