"""Paged caches for the tests of the decode with attention maps and of the eviction,
and their definitions in 64 bits on the CPU, request by request. Slots that no token
holds are NaN."""
import math

import numpy as np
import torch

FP8 = torch.float8_e4m3fn
EPS32 = 2.0 ** -24


def half_step(dtype):
    """Largest relative error of one rounding to nearest."""
    return torch.finfo(dtype).eps / 2


def paged(lens, hkv, d, ps, kv, layout="tokmajor", seed=0, csr=False, spare=3, scale_k=1.0,
          pairs=True):
    """A cache on the CPU: dict with pools, table (extra columns hold ids outside
    the pool), lengths, scales, and the sequences k / v [hkv, n, d] in 64 bits."""
    g = torch.Generator().manual_seed(seed)
    npg = [-(-n // ps) for n in lens]
    P = sum(npg) + spare
    perm = torch.randperm(P, generator=g).tolist()
    nan = float("nan")
    kp = torch.full((P, hkv, ps, d), nan)
    vp = torch.full((P, hkv, ps, d), nan)
    fp8 = kv == FP8
    ksc = torch.exp2(torch.randint(-6, -2, (P * hkv,), generator=g).float())
    vsc = torch.exp2(torch.randint(-6, -2, (P * hkv,), generator=g).float())
    rows, at, seqs = [], 0, []
    for n, m in zip(lens, npg):
        pages = perm[at:at + m]
        at += m
        rows.append(pages)
        k = torch.randn(hkv, n, d, generator=g) * (60.0 if fp8 else 1.0) * scale_k
        v = torch.randn(hkv, n, d, generator=g) * (60.0 if fp8 else 1.0)
        for b, p in enumerate(pages):
            c = min(ps, n - b * ps)
            kp[p, :, :c] = k[:, b * ps:b * ps + c].clamp(-448, 448)
            vp[p, :, :c] = v[:, b * ps:b * ps + c].clamp(-448, 448)
    kp, vp = kp.to(kv), vp.to(kv)
    for pages, n in zip(rows, lens):
        def seq(pool, sc):
            t = pool.float()[pages].double() if pages else torch.zeros(0, hkv, ps, d).double()
            if fp8:
                t = t * sc.view(P, hkv)[pages].double()[:, :, None, None]
            return t.transpose(0, 1).reshape(hkv, -1, d)[:, :n]
        seqs.append((seq(kp, ksc), seq(vp, vsc)))
    if layout == "dmajor":
        vp = vp.float().transpose(2, 3).contiguous().to(kv)
    if layout == "nhd":     # [P, 2, page, hkv, d] read in place
        both = torch.stack([kp.float().transpose(1, 2), vp.float().transpose(1, 2)], 1).to(kv)
        kp, vp = both[:, 0].permute(0, 2, 1, 3), both[:, 1].permute(0, 2, 1, 3)
    c = dict(k=kp, v=vp, layout="tokmajor" if layout == "nhd" else layout, nhd=layout == "nhd",
             rows=rows, seqs=seqs, P=P, lens=list(lens),
             ctx=torch.tensor(lens, dtype=torch.int32), ks=None, vs=None, pind=None)
    if fp8:
        if pairs:
            both = torch.stack([ksc, vsc], 1).contiguous()
            c["ks"], c["vs"] = both[:, 0], both[:, 1]
        else:
            c["ks"], c["vs"] = ksc, vsc
    if csr:
        c["pind"] = torch.tensor(np.concatenate([[0], np.cumsum(npg)]), dtype=torch.int32)
        c["bt"] = torch.tensor([p for r in rows for p in r] + [P + 7], dtype=torch.int32)
    else:
        width = max(1, max(npg, default=1)) + 2
        bt = torch.full((len(lens), width), P + 7, dtype=torch.int32)
        for r, pages in enumerate(rows):
            bt[r, :len(pages)] = torch.tensor(pages, dtype=torch.int32)
        c["bt"] = bt
    return c


def to_gpu(c):
    """The cache's tensors on the GPU, strided as they are."""
    out = dict(c)
    if c["nhd"]:
        base = c["k"]._base if c["k"]._base is not None else c["k"]
        both = base.cuda()
        out["k"] = both[:, 0].permute(0, 2, 1, 3)
        out["v"] = both[:, 1].permute(0, 2, 1, 3)
    else:
        out["k"], out["v"] = c["k"].cuda(), c["v"].cuda()
    for n in ("bt", "ctx", "pind"):
        out[n] = None if c[n] is None else c[n].cuda()
    if c["ks"] is not None:
        if c["ks"].stride(0) == 2:
            both = torch.stack([c["ks"], c["vs"]], 1).contiguous().cuda()
            out["ks"], out["vs"] = both[:, 0], both[:, 1]
        else:
            out["ks"], out["vs"] = c["ks"].cuda(), c["vs"].cuda()
    return out


def maps(q, k, scale, width):
    """softmax(scale q k^T) in 64 bits, and a bound on the relative error of each of
    its values held in 32 bits: the score's (a dot product of `width` products, at
    most width + 2 roundings of its terms' sum) enters twice (numerator and sum), the
    exponentials' and the divisions' roundings, and the sum's, whose longest chain
    of additions is n / 16 + 40."""
    s = (q @ k.transpose(-1, -2)) * scale
    mag = (q.abs() @ k.abs().transpose(-1, -2)) * scale
    p = torch.softmax(s, -1)
    n = k.shape[-2]
    if n == 0:
        return p, 0.0
    d_s = (width + 2) * EPS32 * mag.amax(-1, keepdim=True) + 4 * EPS32 * s.abs().amax(-1, keepdim=True)
    return p, 2 * d_s + (n / 16 + 40) * EPS32 + 8 * EPS32


def weighted_ref(c, q, weights, counted, decay, sm_scale=None, p_err=0.0, out_dtype=None):
    """(out, bound, weights, bound) of the weighted decode in 64 bits."""
    R, hq, d = q.shape
    hkv = c["seqs"][0][0].shape[0]
    G, ps = hq // hkv, c["k"].shape[2]
    scale = d ** -0.5 if sm_scale is None else sm_scale
    out = torch.full((R, hq, d), float("nan"), dtype=torch.float64)
    bound = torch.zeros(R, hq, d, dtype=torch.float64)
    w = weights.double().clone()
    wb = torch.zeros_like(w)
    for r, (k, v) in enumerate(c["seqs"]):
        n = k.shape[1]
        if n == 0:
            continue
        p, rel = maps(q[r].double().view(hkv, G, d), k, scale, d)
        o = p @ v
        out[r] = o.reshape(hq, d)
        bound[r] = ((p @ v.abs()) * (rel + p_err)).reshape(hq, d)
        t = torch.arange(n)
        pages, slots = torch.tensor(c["rows"][r])[t // ps], t % ps
        add, eb = p.sum(1).t().clone(), (p * rel).sum(1).t().clone()
        cnt = n if counted is None else int(counted[r])
        old = w[pages[:cnt], :, slots[:cnt]] * decay
        add[:cnt] += old
        w[pages, :, slots] = add
        wb[pages, :, slots] = eb + 4 * EPS32 * (add.abs() + p.sum(1).t())
    bound += half_step(out_dtype or q.dtype) * out.abs().nan_to_num() + 1e-30
    return out, bound, w, wb


def diff_ref(c, q, lam, nw, eps, mul, sm_scale=None, p_err=0.0, out_dtype=None):
    """(out, bound) of the differential decode in 64 bits."""
    R, hq, d = q.shape
    hkv, h = c["seqs"][0][0].shape[0], d // 2
    G = hq // hkv
    scale = h ** -0.5 if sm_scale is None else sm_scale
    out = torch.full((R, hq, d), float("nan"), dtype=torch.float64)
    bound = torch.zeros(R, hq, d, dtype=torch.float64)
    for r, (k, v) in enumerate(c["seqs"]):
        if k.shape[1] == 0:
            continue
        qr = q[r].double().view(hkv, G, d)
        p1, r1 = maps(qr[..., :h], k[..., :h], scale, h)
        p2, r2 = maps(qr[..., h:], k[..., h:], scale, h)
        la = lam.double().view(hkv, G, 1)
        o = (p1 - la * p2) @ v
        e = (p1 @ v.abs()) * (r1 + p_err) + la.abs() * (p2 @ v.abs()) * (r2 + p_err) \
            + 3 * EPS32 * ((p1 + la.abs() * p2) @ v.abs())
        if nw is not None:
            inv = 1 / torch.sqrt(o.pow(2).mean(-1, keepdim=True) + eps)
            # d inv / inv is at most |e|_2 |o|_2 / (|o|_2^2 + d eps)
            shift = e.norm(dim=-1, keepdim=True) * o.norm(dim=-1, keepdim=True) \
                / (o.pow(2).sum(-1, keepdim=True) + d * eps)
            e = (e + o.abs() * (shift + 16 * EPS32)) * inv * nw.double().abs()
            o = o * inv * nw.double()
        out[r] = (o * mul).reshape(hq, d)
        bound[r] = (e * abs(mul)).reshape(hq, d) * (1 + 2 ** -10)
    bound += (half_step(out_dtype or q.dtype) + 4 * EPS32) * out.abs().nan_to_num() + 1e-30
    return out, bound


def kept_ref(w, n, m, sink, recent):
    """The slots an eviction keeps of n tokens with weights w [n] (python floats)."""
    late = min(m, recent)
    first = min(sink, m - late)
    mid = list(range(first, n - late))
    key = [(-math.inf if math.isnan(x) else x) for x in w]
    nan = [math.isnan(x) for x in w]
    # heaviest first, NaN behind every number, the lower slot first among equals
    mid.sort(key=lambda t: (nan[t], -key[t], t))
    return list(range(first)) + sorted(mid[:m - first - late]) + list(range(n - late, n))


def close(got, ref, bound, what=""):
    got = got.detach().cpu().double()
    assert torch.equal(got.isnan(), ref.isnan()), what
    off = (got - ref).abs().nan_to_num()
    bad = off > bound
    assert not bad.any(), (what, float(off.max()), float((off / bound.clamp(min=1e-300)).max()))
