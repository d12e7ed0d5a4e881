"""Timed cases of the serving-step operators around a paged KV cache: the
query / key norm with the position rotation (also straight into the cache),
the decode that adds up each cached token's attention weight, the decode of
the difference of two softmax maps, and the eviction of the tokens with the
least weight. Each has a plain form in elementary torch operations and the
call a user makes."""
import math

import numpy as np
import torch

own = False

DEV = "cuda"
DT = {"fp32": torch.float32, "bf16": torch.bfloat16, "fp16": torch.float16,
      "fp8": torch.float8_e4m3fn}
EB = {"fp32": 4, "bf16": 2, "fp16": 2, "fp8": 1}


# -- cases ---------------------------------------------------------------------
def _case(op, name, kv, R, dist, lo, hi, hkv, group, d, page, layout="tokmajor", *, lens=0,
          median=0, **kw):
    c = dict(op=op, kv=kv, R=R, dist=dist, lo=lo, hi=hi, median=median, lens=lens, hkv=hkv,
             group=group, d=d, page=page, layout=layout, **kw)
    if name:
        c["name"] = name
    return c


def _rope(name, kv, R, dist, lo, hi, hkv, group, d, page, layout="tokmajor", *, cache=True,
          held=0, rot=0, interleaved=False, norm=True, **kw):
    """lo..hi new tokens a request, behind up to `held` tokens in the cache."""
    return _case("rope", name, kv, R, dist, lo, hi, hkv, group, d, page, layout, cache=cache,
                 held=held, rot=rot or d, interleaved=interleaved, norm=norm, **kw)


def listed():
    return [
        # one sequence's next token: norm, rotation and cache write, all latency
        _rope("rope_one_token", "bf16", 1, "fixed", 1, 1, 8, 4, 128, 16, held=700),
        # a decode step of a full batch
        _rope("rope_step_batch", "bf16", 256, "fixed", 1, 1, 8, 4, 128, 16, held=500),
        # prompts of odd lengths joining a batch
        _rope("rope_prompts", "bf16", 9, "uniform", 301, 2900, 8, 4, 128, 16, held=0, lens=1),
        # neighbouring-pair rotation of part of a head, into buffers (no cache)
        _rope("rope_partial_fp16", "fp16", 1, "fixed", 4097, 4097, 6, 2, 64, 16, cache=False,
              rot=32, interleaved=True),
        # the uniform decode step of the benchmark's shape, weights kept
        _case("weighted", "weighted_64x2048", "bf16", 64, "fixed", 2048, 2048, 8, 4, 128, 16,
              decay=1.0),
        # ragged contexts in an fp8 cache, weights that fade
        _case("weighted", "weighted_fp8_ragged", "fp8", 96, "lognormal", 3, 4000, 4, 7, 128, 16,
              lens=2, median=900, decay=0.95),
        # a few short chats: latency
        _case("weighted", "weighted_few_short", "fp16", 3, "uniform", 5, 130, 4, 4, 64, 16, lens=3,
              decay=1.0),
        # one long document
        _case("weighted", "weighted_one_long", "bf16", 1, "fixed", 100003, 100003, 8, 4, 128, 16,
              decay=1.0),
        # differential heads of 64 + 64 dims, a ragged batch
        _case("diff", "diff_ragged", "bf16", 48, "uniform", 200, 2900, 8, 2, 128, 16, lens=4,
              norm=True),
        # ... and of 128 + 128 dims, one long context
        _case("diff", "diff_one_long", "bf16", 1, "fixed", 32771, 32771, 6, 2, 256, 16, norm=True),
        # a batch cut to half its tokens
        _case("evict", "evict_32x2048", "bf16", 32, "fixed", 2048, 2048, 8, 1, 128, 16, keep=0.5,
              sink=4, recent=256),
        # one long context cut to an eighth
        _case("evict", "evict_one_long", "bf16", 1, "fixed", 65537, 65537, 8, 1, 128, 16,
              keep=0.125, sink=4, recent=1024),
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 1)))))))


def draw(rng):
    op = rng.choice(["rope", "weighted", "diff", "evict"])
    kv = rng.choice(["bf16", "bf16", "fp16", "fp32"] + (["fp8"] if op != "rope" else ["bf16"]))
    lens = rng.randrange(1, 10 ** 6)
    hkv = rng.choice([1, 2, 3, 4, 5, 8])
    group = rng.choice([1, 2, 3, 4, 7, 8])
    page = rng.choice([16, 16, 32, 64])
    layout = rng.choice(["tokmajor", "tokmajor", "tokmajor", "dmajor"])
    d = rng.choice([64, 128, 128])
    dist = rng.choice(["fixed", "uniform", "lognormal"])
    if op == "rope":
        new = _log_int(rng, 1, 16384)                   # new tokens of the batch, about
        R = min(new, _log_int(rng, 1, 256))
        hi = max(1, new // R)
        rot = rng.choice([d, d, d // 2, d // 4])
        return _rope(None, kv, R, "uniform", max(1, hi // 3), hi, hkv, group, d, page, layout,
                     cache=rng.random() < 0.7, held=rng.randrange(0, 300), rot=rot,
                     interleaved=rng.random() < 0.4, norm=rng.random() < 0.8, lens=lens)
    R = _log_int(rng, 1, 96)
    hi = min(100003, _log_int(rng, 256, 65536 * 3 // hkv) // R + 1)
    lo = hi if dist == "fixed" else max(1, hi // 16)
    kw = dict(lens=lens, median=max(1, hi // 4) if dist == "lognormal" else 0)
    if op == "weighted":
        return _case(op, None, kv, R, dist, lo, hi, hkv, group, d, page, layout,
                     decay=rng.choice([1.0, 0.9]), **kw)
    if op == "diff":
        return _case(op, None, kv, R, dist, lo, hi, hkv, rng.choice([1, 2, 3, 4, 8]),
                     rng.choice([128, 256]), page, layout, norm=rng.random() < 0.8, **kw)
    return _case(op, None, kv, R, dist, lo, hi, hkv, 1, d, page, layout,
                 keep=rng.choice([0.1, 0.3, 0.5, 0.75, 0.95]), sink=rng.choice([0, 1, 4]),
                 recent=rng.choice([0, 16, 100]), **kw)


# -- inputs --------------------------------------------------------------------
def _lens(case):
    rng = np.random.default_rng(100 + case["lens"])
    R, lo, hi = case["R"], case["lo"], case["hi"]
    if case["dist"] == "fixed":
        return np.full(R, hi, np.int64)
    if case["dist"] == "uniform":
        return rng.integers(lo, hi + 1, R).astype(np.int64)
    x = np.exp(rng.normal(np.log(case["median"]), 0.9, R))
    return np.clip(np.rint(x), lo, hi).astype(np.int64)


def _held(case):
    """Tokens each request holds before a rotation's new ones."""
    rng = np.random.default_rng(200 + case["lens"])
    return rng.integers(case["held"] // 4, case["held"] + 1, case["R"]).astype(np.int64)


def _keep(case):
    return np.maximum(1, np.floor(_lens(case) * case["keep"])).astype(np.int64)


def _i32(a):
    return torch.from_numpy(np.ascontiguousarray(a, np.int32)).to(DEV)


def _randn(g, shape, dtype, scale=1.0):
    return (torch.randn(shape, generator=g, device=DEV) * scale).to(dtype)


def _cache(case, g, ctx):
    """Pools that hold ctx tokens a request, on pages in any order; an fp8
    cache with its power-of-two scales."""
    ps, hkv, d, dt = case["page"], case["hkv"], case["d"], DT[case["kv"]]
    npg = -(-ctx // ps)
    P = max(1, int(npg.sum()))
    s = 100.0 if case["kv"] == "fp8" else 1.0
    # a few dims of K are much larger than the others
    big = torch.ones(d, device=DEV)
    big[torch.randperm(d, generator=g, device=DEV)[:max(1, d // 32)]] = 4.0
    k = (torch.randn((P, hkv, ps, d), generator=g, device=DEV) * (s / 4 if s > 1 else 1.0)
         * big).clamp(-440.0, 440.0).to(dt)
    v = torch.randn((P, hkv, d, ps) if case["layout"] == "dmajor" else (P, hkv, ps, d),
                    generator=g, device=DEV)
    v = (v * s).clamp(-440.0, 440.0).to(dt)
    x = dict(k=k, v=v, ks=None, vs=None, ctx=_i32(ctx), layout=case["layout"])
    if case["kv"] == "fp8":
        e = torch.randint(-7, -4, (P * hkv, 2), generator=g, device=DEV)
        pairs = torch.exp2(e.float())
        x["ks"], x["vs"] = pairs[:, 0], pairs[:, 1]
    perm = torch.randperm(P, generator=g, device=DEV).cpu().numpy()
    start = np.cumsum(npg) - npg
    bt = np.zeros((case["R"], max(1, int(npg.max()))), np.int32)
    for r in range(case["R"]):
        bt[r, :npg[r]] = perm[start[r]:start[r] + npg[r]]
    x["bt"] = _i32(bt)
    return x


def _token_weights(g, shape):
    """What a decode adds up: a long tail, many tokens never looked at."""
    w = torch.exp(torch.randn(shape, generator=g, device=DEV) * 2.0 - 3.0)
    return torch.where(torch.rand(shape, generator=g, device=DEV) < 0.15, torch.zeros_like(w), w)


def prepare(case, seed):
    g = torch.Generator(device=DEV).manual_seed(seed)
    hkv, d, ps, R = case["hkv"], case["d"], case["page"], case["R"]
    hq = hkv * case["group"]
    n = _lens(case)
    if case["op"] == "rope":
        held, T, dt = _held(case), int(n.sum()), DT[case["kv"]]
        s = dict(op="rope", cache=case["cache"], interleaved=case["interleaved"], eps=1e-6,
                 qw=None, kw=None, layout=case["layout"])
        if case["cache"]:
            s.update(_cache(case, g, held + n))
            s["v_new"] = None
        # the three parts of one projection's output
        qkv = _randn(g, (T, hq + 2 * hkv, d), dt)
        s["q"], s["k_new"], s["v_new"] = qkv[:, :hq], qkv[:, hq:hq + hkv], qkv[:, hq + hkv:]
        if case["norm"]:
            s["qw"] = 1.0 + 0.2 * torch.randn(d, generator=g, device=DEV)
            s["kw"] = 1.0 + 0.2 * torch.randn(d, generator=g, device=DEV)
        # positions run on from tokens that may no longer be in the cache
        first = held + np.random.default_rng(300 + case["lens"]).integers(0, 5000, R)
        pos = np.concatenate([first[r] + np.arange(n[r]) for r in range(R)])
        s["pos"] = torch.from_numpy(pos.astype(np.int64)).to(DEV)
        half = case["rot"] // 2
        inv = 500000.0 ** (-torch.arange(half, device=DEV, dtype=torch.float64) / half)
        ang = torch.arange(32768, device=DEV, dtype=torch.float64)[:, None] * inv
        s["cos_sin"] = torch.cat([ang.cos(), ang.sin()], 1).float()
        s["app"] = _i32(np.concatenate([[0], np.cumsum(n)]))
        s["most"] = int(n.max())
        return s
    s = _cache(case, g, n)
    s["op"] = case["op"]
    P = s["k"].shape[0]
    if case["op"] != "evict":
        qt = torch.bfloat16 if case["kv"] == "fp8" else DT[case["kv"]]
        s["q"] = _randn(g, (R, hq, d), qt, 1.5)
    if case["op"] == "weighted":
        s["w"] = _token_weights(g, (P, hkv, ps))
        s["decay"] = case["decay"]
        # the newest tokens have no weight yet
        new = np.random.default_rng(400 + case["lens"]).integers(0, 3, R)
        s["counted"] = _i32(np.maximum(0, n - new))
    if case["op"] == "diff":
        s["lam"] = 0.3 + 0.5 * torch.rand(hq, generator=g, device=DEV)
        s["nw"] = 1.0 + 0.2 * torch.randn(d, generator=g, device=DEV) if case["norm"] else None
        s["eps"], s["mul"] = 1e-5, 0.2
    if case["op"] == "evict":
        s["w"] = _token_weights(g, (P, hkv, ps))
        s["w_out"] = torch.zeros_like(s["w"])
        keep = _keep(case)
        s["keep"], s["most"] = _i32(keep), int(keep.max())
        s["sink"], s["recent"] = case["sink"], case["recent"]
    return s


# -- one pass --------------------------------------------------------------------
def run(s):
    if own:
        return _own(s)
    if s["op"] == "rope":
        return _plain_rope(s)
    if s["op"] == "weighted":
        return _plain_weighted(s)
    if s["op"] == "diff":
        return _plain_diff(s)
    return _plain_evict(s)


def _own(s):
    import os
    import sys
    pkg = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))),
                       "sched-pass_amd")
    if pkg not in sys.path:
        sys.path.insert(0, pkg)
    if s["op"] == "rope":
        import rotary
        kw = dict(q_weight=s["qw"], k_weight=s["kw"], eps=s["eps"], interleaved=s["interleaved"])
        if not s["cache"]:
            return list(rotary.qk_norm_rope(s["q"], s["k_new"], s["pos"], s["cos_sin"], **kw))
        q = rotary.append_rotated(s["q"], s["k_new"], s["v_new"], s["pos"], s["cos_sin"], s["app"],
                                  s["ctx"], s["k"], s["v"], s["bt"], v_layout=s["layout"],
                                  max_append=s["most"], **kw)
        return [q, s["k"], s["v"]]
    kw = dict(v_layout=s["layout"], k_scale=s["ks"], v_scale=s["vs"])
    if s["op"] == "weighted":
        import decode_maps
        out = decode_maps.paged_decode_weighted(s["q"], s["k"], s["v"], s["bt"], s["ctx"], s["w"],
                                                counted=s["counted"], decay=s["decay"], **kw)
        return [out, s["w"]]
    if s["op"] == "diff":
        import decode_maps
        return decode_maps.paged_decode_diff(s["q"], s["k"], s["v"], s["bt"], s["ctx"], s["lam"],
                                             norm_weight=s["nw"], eps=s["eps"],
                                             out_scale=s["mul"], **kw)
    import eviction
    kept = eviction.evict(s["k"], s["v"], s["w"], s["bt"], s["ctx"], s["keep"], sink=s["sink"],
                          recent=s["recent"], max_keep=s["most"], weights_out=s["w_out"], **kw)
    return _evict_outputs(s, kept)


def _evict_outputs(s, kept):
    if s["ks"] is None:
        return [kept, s["w_out"], s["k"], s["v"]]
    return [kept, s["w_out"], s["k"], s["v"], s["ks"], s["vs"]]


def _raw(pool):
    return pool.view(torch.uint8) if pool.dtype == torch.float8_e4m3fn else pool


def _norm_rotate(x, weight, c, sn, eps, interleaved):
    x = x.float()
    if weight is not None:
        x = x * torch.rsqrt((x * x).mean(-1, keepdim=True) + eps) * weight
    half = c.shape[-1]
    part, rest = x[..., :2 * half], x[..., 2 * half:]
    a, b = (part[..., 0::2], part[..., 1::2]) if interleaved else (part[..., :half],
                                                                  part[..., half:])
    c, sn = c[:, None], sn[:, None]
    y = (a * c - b * sn, b * c + a * sn)
    y = torch.stack(y, -1).flatten(-2) if interleaved else torch.cat(y, -1)
    return torch.cat([y, rest], -1)


def _plain_rope(s):
    cs = s["cos_sin"][s["pos"]]
    half = cs.shape[1] // 2
    args = (cs[:, :half], cs[:, half:], s["eps"], s["interleaved"])
    q = _norm_rotate(s["q"], s["qw"], *args).to(s["q"].dtype)
    k = _norm_rotate(s["k_new"], s["kw"], *args).to(s["q"].dtype)
    if not s["cache"]:
        return [q, k]
    # row i of request r goes to position ctx[r] - (app[r + 1] - i)
    T, ps = q.shape[0], s["k"].shape[2]
    i = torch.arange(T, device=DEV)
    r = torch.searchsorted(s["app"].long(), i, right=True) - 1
    at = s["ctx"].long()[r] - (s["app"].long()[r + 1] - i)
    page, slot = s["bt"].long()[r, at // ps], at % ps
    s["k"][page, :, slot] = k
    if s["layout"] == "dmajor":
        s["v"][page, :, :, slot] = s["v_new"]
    else:
        s["v"][page, :, slot] = s["v_new"]
    return [q, s["k"], s["v"]]


def _rows(s, pool, scale, dmajor):
    """The batch's tokens as [R, hkv, width * page, d] in 32 bits."""
    P, hkv = pool.shape[:2]
    bt = s["bt"].long()
    x = _raw(pool)[bt]
    x = x.view(pool.dtype).float()
    if dmajor:
        x = x.transpose(3, 4)
    if scale is not None:
        x = x * scale.view(P, hkv)[bt][..., None, None]
    return x.transpose(1, 2).reshape(bt.shape[0], hkv, -1, x.shape[-1])


def _map(q, k, live, scale):
    """softmax(q k^T scale) over the live tokens."""
    x = torch.matmul(q, k.transpose(-1, -2)) * scale
    x = torch.where(live, x, torch.full_like(x, -math.inf))
    x = torch.exp(x - x.amax(-1, keepdim=True))
    return x / x.sum(-1, keepdim=True)


def _plain_weighted(s):
    R, hq, d = s["q"].shape
    k = _rows(s, s["k"], s["ks"], False)
    hkv, N = k.shape[1:3]
    t = torch.arange(N, device=DEV)
    live = (t < s["ctx"][:, None])[:, None, None]
    p = _map(s["q"].float().view(R, hkv, hq // hkv, d), k, live, d ** -0.5)
    del k
    out = torch.matmul(p, _rows(s, s["v"], s["vs"], s["layout"] == "dmajor"))
    old = s["w"][s["bt"].long()].transpose(1, 2).reshape(R, hkv, N)
    old = torch.where(t < s["counted"][:, None, None], old * s["decay"], torch.zeros_like(old))
    new = (old + p.sum(2)).view(R, hkv, -1, s["w"].shape[2]).transpose(1, 2)
    r, t = torch.nonzero(t < s["ctx"][:, None], as_tuple=True)
    ps = s["w"].shape[2]
    s["w"][s["bt"].long()[r, t // ps], :, t % ps] = new[r, t // ps, :, t % ps]
    return [out.reshape(R, hq, d).to(s["q"].dtype), s["w"]]


def _plain_diff(s):
    R, hq, d = s["q"].shape
    k = _rows(s, s["k"], s["ks"], False)
    hkv, N = k.shape[1:3]
    live = (torch.arange(N, device=DEV) < s["ctx"][:, None])[:, None, None]
    q, h = s["q"].float().view(R, hkv, hq // hkv, d), d // 2
    lam = s["lam"].view(1, hkv, hq // hkv, 1)
    p = _map(q[..., :h], k[..., :h], live, h ** -0.5)
    p = p - lam * _map(q[..., h:], k[..., h:], live, h ** -0.5)
    del k
    out = torch.matmul(p, _rows(s, s["v"], s["vs"], s["layout"] == "dmajor"))
    if s["nw"] is not None:
        out = out * torch.rsqrt((out * out).mean(-1, keepdim=True) + s["eps"]) * s["nw"]
    return (out * s["mul"]).reshape(R, hq, d).to(s["q"].dtype)


def _plain_evict(s):
    bt, ctx = s["bt"].long(), s["ctx"].long()[:, None, None]
    P, hkv, ps = s["w"].shape
    R, most = bt.shape[0], s["most"]
    w = s["w"][bt].transpose(1, 2).reshape(R, hkv, -1)
    t = torch.arange(w.shape[2], device=DEV)
    m = torch.minimum(ctx, s["keep"].long()[:, None, None])
    recent = torch.clamp(m, max=s["recent"])
    sink = torch.minimum(torch.full_like(m, s["sink"]), m - recent)
    inf = torch.full_like(w, math.inf)
    key = torch.where((t < sink) | (t >= ctx - recent), inf, w)
    key = torch.where(t < ctx, key, -inf)
    rank = torch.argsort(torch.argsort(key, dim=-1, descending=True, stable=True), dim=-1)
    kept = torch.argsort((rank >= m).int(), dim=-1, stable=True)[..., :most]
    j = torch.arange(kept.shape[2], device=DEV)
    kept = torch.where(j < m, kept, torch.full_like(kept, -1))
    # every row is read before any is written
    r, h, j = torch.nonzero(kept >= 0, as_tuple=True)
    src = kept[r, h, j]
    sp, ss, dp, ds = bt[r, src // ps], src % ps, bt[r, j // ps], j % ps
    s["w_out"][dp, h, ds] = s["w"][sp, h, ss]
    fp8 = s["ks"] is not None
    for pool, scale, dm in ((s["k"], s["ks"], False),
                            (s["v"], s["vs"], s["layout"] == "dmajor")):
        x = _raw(pool)
        rows = x[sp, h, :, ss] if dm else x[sp, h, ss]
        if fp8:
            # a page's scale is the largest of its tokens' old ones
            was = scale[sp * hkv + h]
            top = torch.zeros(P * hkv, device=DEV).scatter_reduce(0, dp * hkv + h, was, "amax")
            now = top[dp * hkv + h]
            vals = rows.view(pool.dtype).float() * (was / now)[:, None]
            rows = vals.clamp(-448.0, 448.0).to(pool.dtype).view(torch.uint8)
            scale.copy_(torch.where(top > 0, top, scale))
        if dm:
            x[dp, h, :, ds] = rows
        else:
            x[dp, h, ds] = rows
    out = torch.full((R, hkv, most), -1, dtype=torch.int32, device=DEV)
    out[..., :kept.shape[2]] = kept
    return _evict_outputs(s, out)


# -- what a pass cannot do without -------------------------------------------------
def work(case):
    n, hkv, d, ps = _lens(case), case["hkv"], case["d"], case["page"]
    hq, eb, T = hkv * case["group"], EB[case["kv"]], int(_lens(case).sum())
    pages = int((-(-n // ps)).sum())
    if case["op"] == "rope":
        rows = hq + hkv + (hkv if case["cache"] else 0)
        b = 2 * T * rows * d * eb + T * (case["rot"] * 4 + 8)
        return {"bytes": b, "flops": T * (hq + hkv) * (4 * d + 3 * case["rot"])}
    if case["op"] == "evict":
        # weights read, kept rows read and written (those of the sinks stay)
        m = np.minimum(n, _keep(case))
        moved = int(np.maximum(0, np.where(m < n, m - case["sink"], 0)).sum())
        b = (T * 4 + int(m.sum()) * 8 + moved * 4 * d * eb) * hkv + 4 * pages
        return {"bytes": b, "flops": T * hkv}
    scales = pages * hkv * 8 if case["kv"] == "fp8" else 0
    qb = 2 if case["kv"] == "fp8" else eb
    b = T * hkv * d * 2 * eb + 4 * pages + scales + 2 * case["R"] * hq * d * qb
    if case["op"] == "weighted":
        return {"bytes": b + T * hkv * 8, "flops": 4 * T * hq * d}
    return {"bytes": b, "flops": 6 * T * hq * d}


# -- the definition in 64 bits, request by request ------------------------------------
def _sequence(x, pool, r, n, scale, dmajor):
    """Request r's first n rows [hkv, n, d] in 64 bits."""
    P, hkv = pool.shape[:2]
    ps = pool.shape[3] if dmajor else pool.shape[2]
    pages = x["bt"][r, :-(-n // ps)].long()
    t = _raw(pool).index_select(0, pages).view(pool.dtype).float().double()
    if dmajor:
        t = t.permute(0, 1, 3, 2)
    if scale is not None:
        t = t * scale.reshape(P, hkv).index_select(0, pages).double().reshape(-1, hkv, 1, 1)
    return t.permute(1, 0, 2, 3).reshape(hkv, -1, t.shape[-1])[:, :n].contiguous()


def exact(case, seed):
    x = prepare(case, seed)
    n = _lens(case)
    if case["op"] == "rope":
        return _exact_rope(case, x, n)
    if case["op"] == "evict":
        return _exact_evict(case, x, n)
    hkv, G, d, dm = case["hkv"], case["group"], case["d"], case["layout"] == "dmajor"
    out = torch.empty(x["q"].shape, dtype=torch.float64, device=DEV)
    w = x["w"].double() if case["op"] == "weighted" else None
    for r in range(case["R"]):
        N = int(n[r])
        k = _sequence(x, x["k"], r, N, x["ks"], False)
        v = _sequence(x, x["v"], r, N, x["vs"], dm)
        q = x["q"][r].double().view(hkv, G, d)
        if case["op"] == "diff":
            a = [torch.softmax(torch.bmm(q[..., c], k[..., c].transpose(1, 2).contiguous())
                               / math.sqrt(d / 2), 2)
                 for c in (slice(0, d // 2), slice(d // 2, d))]
            o = torch.bmm(a[0] - x["lam"].double().view(hkv, G, 1) * a[1], v)
            if case["norm"]:
                o = o / torch.sqrt(o.pow(2).mean(2, keepdim=True) + x["eps"]) * x["nw"].double()
            out[r] = (o * x["mul"]).view(hkv * G, d)
            continue
        p = torch.softmax(torch.bmm(q, k.transpose(1, 2).contiguous()) / math.sqrt(d), 2)
        out[r] = torch.bmm(p, v).view(hkv * G, d)
        at = torch.arange(N, device=DEV)
        pages, slots = x["bt"][r].long()[at // case["page"]], at % case["page"]
        c = int(x["counted"][r])
        add = p.sum(1).t().contiguous()
        add[:c] += case["decay"] * w[pages[:c], :, slots[:c]]
        w[pages, :, slots] = add
    return out if w is None else [out, w]


def _exact_rope(case, x, n):
    half, d = case["rot"] // 2, case["d"]
    cs = x["cos_sin"].double()[x["pos"]]
    turn = torch.complex(cs[:, :half], cs[:, half:])[:, None]

    def rotated(t, weight):
        t = t.double()
        if weight is not None:
            t = t / torch.sqrt(t.pow(2).mean(2, keepdim=True) + x["eps"]) * weight.double()
        i = torch.arange(half, device=DEV)
        lo, hi = (2 * i, 2 * i + 1) if case["interleaved"] else (i, i + half)
        z = torch.complex(t[..., lo], t[..., hi]) * turn
        t = t.clone()
        t[..., lo], t[..., hi] = z.real, z.imag
        return t

    q, k = rotated(x["q"], x["qw"]), rotated(x["k_new"], x["kw"])
    if not case["cache"]:
        return [q, k]
    kp, vp, a = x["k"].double(), x["v"].double(), 0
    ctx = x["ctx"].cpu().numpy()
    for r in range(case["R"]):
        m = int(n[r])
        at = torch.arange(int(ctx[r]) - m, int(ctx[r]), device=DEV)
        pages, slots = x["bt"][r].long()[at // case["page"]], at % case["page"]
        kp[pages, :, slots] = k[a:a + m]
        new = x["v_new"][a:a + m].double()
        if case["layout"] == "dmajor":
            vp[pages, :, :, slots] = new
        else:
            vp[pages, :, slots] = new
        a += m
    return [q, kp, vp]


def _exact_evict(case, x, n):
    P, hkv, ps = x["w"].shape
    fp8, dm = case["kv"] == "fp8", case["layout"] == "dmajor"
    keep, most = _keep(case), x["most"]
    kept = np.full((case["R"], hkv, most), -1, np.int64)
    w = x["w"].cpu().numpy().astype(np.float64)
    bt = x["bt"].cpu().numpy()
    for r in range(case["R"]):
        N = int(n[r])
        m = min(N, int(keep[r]))
        late = min(m, case["recent"])
        first = min(case["sink"], m - late)
        at = np.arange(N)
        rows = w[bt[r, at // ps], :, at % ps]
        mid = at[first:N - late]
        for h in range(hkv):
            # heaviest first, the lower slot first among equals
            best = np.lexsort((mid, -rows[mid, h]))[:m - first - late]
            kept[r, h, :m] = np.concatenate([at[:first], np.sort(mid[best]), at[N - late:]])
    pools = [_raw(t).view(t.dtype).float().double() for t in (x["k"], x["v"])]
    scales = [t.double().clone() for t in (x["ks"], x["vs"])] if fp8 else [None, None]
    w_out = x["w_out"].double()
    for r in range(case["R"]):
        m = min(int(n[r]), int(keep[r]))
        dst = torch.arange(m, device=DEV)
        dp, ds = x["bt"][r].long()[dst // ps], dst % ps
        for h in range(hkv):
            src = torch.from_numpy(kept[r, h, :m]).to(DEV)
            sp, ss = x["bt"][r].long()[src // ps], src % ps
            w_out[dp, h, ds] = x["w"][sp, h, ss].double()
            for t, scale, turned in ((pools[0], scales[0], False), (pools[1], scales[1], dm)):
                rows = t[sp, h, :, ss] if turned else t[sp, h, ss]
                if fp8:
                    old = scale[sp * hkv + h]
                    for p in range(-(-m // ps)):
                        part = slice(p * ps, min(m, (p + 1) * ps))
                        top = old[part].max()
                        rows[part] *= (old[part] / top)[:, None]
                        scale[dp[p * ps] * hkv + h] = top
                if turned:
                    t[dp, h, :, ds] = rows
                else:
                    t[dp, h, ds] = rows
    out = [torch.from_numpy(kept.astype(np.int32)).to(DEV), w_out] + pools
    return out + scales if fp8 else out
