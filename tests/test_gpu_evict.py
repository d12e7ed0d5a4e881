"""Eviction by accumulated attention weight on the GPU: the kept slots, weights,
keys and values against the definition, bit for bit; ties, NaN, infinities and
negative weights; every cache type and layout; what is not touched; and the serving
steps together: rotated append, weighted decode, eviction, and on."""
import ctypes
import math

import pytest
import torch

import eviction
import kv_cache
import sched_abi as abi
import maps_ref as mr
import rotary

pytestmark = pytest.mark.gpu
FP8 = mr.FP8


@pytest.fixture(scope="module", autouse=True)
def lib(schedlib):
    torch.cuda.init()
    return schedlib


def bits(t):
    t = t.detach().cpu().contiguous()
    return t.view({1: torch.uint8, 2: torch.int16, 4: torch.int32}[t.element_size()])


def weights_of(c, hkv, ps, seed, kind):
    g = torch.Generator().manual_seed(seed)
    w = torch.exp(2 * torch.randn(c["P"], hkv, ps, generator=g))
    if kind == "ties":          # few values, many equals
        w = torch.randint(0, 3, w.shape, generator=g).float()
    elif kind == "equal":
        w = torch.full_like(w, 0.25)
    elif kind == "odd":         # signs, zeros of both signs, infinities, NaN
        pick = torch.tensor([0.0, -0.0, 1.0, -1.0, math.inf, -math.inf, math.nan, 1e-40, -1e-40])
        w = pick[torch.randint(0, 9, w.shape, generator=g)]
    elif kind == "close":       # neighbours in the last bits
        w = (torch.randint(0, 40, w.shape, generator=g) + 0x3f800000).int().view(torch.float32)
    return w


def expected(c, w, w_out, keep, sink, recent, max_keep, skip=()):
    """(kept, weights, k, v, ks, vs) after the eviction; pools as raw values."""
    hkv, ps = w.shape[1:]
    k, v = c["k"].clone(), c["v"].clone()
    dm, fp8 = c["layout"] == "dmajor", c["ks"] is not None
    ks, vs = (c["ks"].clone(), c["vs"].clone()) if fp8 else (None, None)
    wo = w_out.clone()
    kept = torch.full((len(c["lens"]), hkv, max_keep), -1, dtype=torch.int32)
    for r, n in enumerate(c["lens"]):
        if r in skip:
            continue
        m = min(n, int(keep[r]), max_keep)
        pages = c["rows"][r]
        for h in range(hkv):
            got = mr.kept_ref([float(w[pages[t // ps], h, t % ps]) for t in range(n)], n, m, sink,
                              recent)
            kept[r, h, :m] = torch.tensor(got, dtype=torch.int32)
            for j, t in enumerate(got):
                wo[pages[j // ps], h, j % ps] = w[pages[t // ps], h, t % ps]
            if m == n:
                continue
            for pool, src, sc, old, turned in ((k, c["k"], ks, c["ks"], False),
                                               (v, c["v"], vs, c["vs"], dm)):
                for b in range(-(-m // ps)):
                    part = got[b * ps:min(m, (b + 1) * ps)]
                    top = max(float(old[pages[t // ps] * hkv + h]) for t in part) if fp8 else 0.0
                    for i, t in enumerate(part):
                        row = src[pages[t // ps], h, :, t % ps] if turned \
                            else src[pages[t // ps], h, t % ps]
                        if fp8:
                            s = float(old[pages[t // ps] * hkv + h])
                            if s != top:
                                x = (row.float() * (s / top)).clamp(-448, 448).to(FP8)
                                row = torch.where(row.float().isnan(), row.view(torch.uint8),
                                                  x.view(torch.uint8)).view(FP8)
                        if turned:
                            pool[pages[b], h, :, i] = row
                        else:
                            pool[pages[b], h, i] = row
                    if fp8:
                        sc[pages[b] * hkv + h] = top
    return kept, wo, k, v, ks, vs


def check(lens, keep, hkv=2, d=64, ps=16, kv=torch.bfloat16, layout="tokmajor", sink=0, recent=0,
          kind="long", max_keep=None, csr=False, inplace=True, seed=1, pairs=True):
    c = mr.paged(lens, hkv, d, ps, kv, layout, seed, csr=csr, pairs=pairs)
    w = weights_of(c, hkv, ps, seed, kind)
    keep_t = torch.tensor(keep, dtype=torch.int32)
    if max_keep is None:
        max_keep = max([1] + [min(a, b) for a, b in zip(lens, keep)])
    w_out = w if inplace else torch.full_like(w, -3.0)
    ref = expected(c, w, w_out, keep, sink, recent, max_keep)
    x = mr.to_gpu(c)
    wg = w.cuda()
    wo = None if inplace else w_out.cuda()
    err = torch.zeros(1, dtype=torch.int32, device="cuda")
    kept = eviction.evict(x["k"], x["v"], wg, x["bt"], x["ctx"], keep_t.cuda(), sink=sink,
                          recent=recent, max_keep=max_keep, weights_out=wo, v_layout=x["layout"],
                          page_indptr=x["pind"], k_scale=x["ks"], v_scale=x["vs"], errors=err)
    torch.cuda.synchronize()
    assert int(err) == 0
    assert torch.equal(kept.cpu(), ref[0]), "kept"
    assert torch.equal(bits(wg if inplace else wo), bits(ref[1])), "weights"
    if not inplace:
        assert torch.equal(bits(wg), bits(w))
    if kv != FP8:
        assert torch.equal(bits(x["k"]), bits(ref[2])) and torch.equal(bits(x["v"]), bits(ref[3]))
    else:
        # a code's zero has either sign's bit; values compare by value, NaN with NaN
        for got, want in ((x["k"], ref[2]), (x["v"], ref[3])):
            assert torch.equal(got.cpu().float().nan_to_num(nan=1e9),
                               want.float().nan_to_num(nan=1e9))
        assert torch.equal(x["ks"].cpu(), ref[4]) and torch.equal(x["vs"].cpu(), ref[5])


LENS = [1, 16, 17, 0, 300, 33, 1500]
KEEP = [1, 7, 17, 5, 100, 0, 1111]


@pytest.mark.parametrize("kv", [torch.float32, torch.bfloat16, torch.float16, FP8])
@pytest.mark.parametrize("layout", ["tokmajor", "dmajor", "nhd"])
def test_types_and_layouts(kv, layout):
    check(LENS, KEEP, kv=kv, layout=layout, sink=2, recent=5)


@pytest.mark.parametrize("kind", ["ties", "equal", "odd", "close"])
@pytest.mark.parametrize("sink,recent", [(0, 0), (3, 20)])
def test_orders(kind, sink, recent):
    check([500, 40, 1025, 2049], [100, 39, 1024, 700], kind=kind, sink=sink, recent=recent, seed=3)


@pytest.mark.parametrize("sink,recent", [(1000, 0), (0, 1000), (1000, 1000), (50, 49), (0, 1)])
def test_sinks_and_recent_beyond_the_kept(sink, recent):
    check([300, 90, 120], [99, 90, 1], sink=sink, recent=recent, kind="ties")


@pytest.mark.parametrize("ps,d", [(4, 4), (12, 20), (32, 128), (256, 96), (16, 256)])
def test_pages_and_dims(ps, d):
    check([700, 9, 260], [300, 4, 259], ps=ps, d=d, hkv=3, sink=1, recent=4)


@pytest.mark.parametrize("kv", [torch.bfloat16, FP8])
def test_page_list_and_separate_weights(kv):
    check(LENS, KEEP, kv=kv, csr=True, inplace=False, pairs=False, sink=1, recent=3)


def test_max_keep_bounds_what_is_kept():
    check([300, 64], [200, 64], max_keep=50, recent=10)
    check([300, 64], [200, 300], max_keep=400)


def test_bounds_beyond_any_table():
    """max_keep, sink and recent past what tables hold; the outputs are what they size."""
    check([300, 64], [200, 300], max_keep=5000, sink=1 << 40, recent=10)
    check([300, 64], [200, 30], max_keep=100000, recent=1 << 40, kv=FP8)
    a = abi.default_evict_args()
    a.num_requests, a.num_kv_heads, a.head_dim, a.page_size = 100, 2, 128, 16
    a.num_pages, a.max_pages, a.k_tok_stride, a.v_dim_stride = 1000, 40, 128, 1
    a.max_keep = 640
    need = abi.load_library().sched_kv_evict_workspace_bytes(ctypes.byref(a))
    a.max_keep = (1 << 31) - 1
    assert abi.load_library().sched_kv_evict_workspace_bytes(ctypes.byref(a)) == need > 0


def test_nothing_to_cut():
    check([100, 5], [100, 1000], max_keep=120)


def test_one_long_request():
    check([20011], [9973], hkv=2, sink=4, recent=128, d=32)
    check([20011], [20010], hkv=1, d=32, kind="ties")


@pytest.mark.parametrize("kind", ["long", "ties", "equal", "odd", "close"])
def test_one_read_of_a_table_of_12288_tokens(kind):
    check([12256, 4097, 12000, 5], [6000, 4096, 11999, 3], hkv=1, d=8, sink=4, recent=64, kind=kind)


@pytest.mark.parametrize("kind", ["long", "ties", "odd"])
def test_stretches(kind):
    """Tables longer than one workgroup's registers, of many tasks."""
    lens = [30000, 12289, 24577, 13] + [50] * 124
    check(lens, [5000, 12288, 100, 7] + [20] * 124, hkv=1, d=4, sink=2, recent=100, kind=kind)


@pytest.mark.parametrize("kind", ["ties", "equal", "odd", "close"])
def test_wide_orders(kind):
    check([13000, 70, 12300, 4096, 8193], [800, 69, 12299, 4095, 4097], hkv=2, d=8, sink=3,
          recent=33, kind=kind)


@pytest.mark.parametrize("kv", [torch.float32, torch.bfloat16, FP8])
@pytest.mark.parametrize("csr,inplace", [(False, True), (True, False)])
def test_wide_types(kv, csr, inplace):
    """Few long requests: the wide selection and the rows in chunks."""
    check([12500, 90, 700], [2500, 80, 650], hkv=2, d=64, kv=kv, csr=csr, inplace=inplace, sink=1,
          recent=50, pairs=False)


def test_wide_without_what_is_not_cut():
    check([12500, 90], [12500, 200], hkv=1, d=8, max_keep=13000)
    check([12500, 90], [12500, 0], hkv=1, d=8, max_keep=13000, inplace=False)
    check([12500, 90], [100, 90], hkv=1, d=8, sink=100, recent=100)


@pytest.mark.parametrize("kv,d", [(torch.float32, 16), (torch.bfloat16, 32), (FP8, 64),
                                  (FP8, 256), (torch.float32, 256), (torch.float16, 96)])
@pytest.mark.parametrize("layout", ["tokmajor", "dmajor"])
def test_rows_in_chunks(kv, d, layout):
    check([2000, 700, 3], [1900, 513, 2], kv=kv, d=d, hkv=2, recent=7, layout=layout)


@pytest.mark.parametrize("kv", [torch.float32, torch.bfloat16, FP8])
@pytest.mark.parametrize("ps,d", [(4, 20), (8, 64), (12, 64), (32, 128), (48, 256), (256, 64)])
def test_turned_values(kv, ps, d):
    """d-major values in pieces of 16 bytes where a page holds whole ones, else by
    element; what is kept ends inside a piece."""
    check([600, 9, 277, 0, 130], [301, 4, 276, 0, 129], kv=kv, ps=ps, d=d, layout="dmajor", sink=1,
          recent=4)


@pytest.mark.parametrize("kv", [torch.bfloat16, FP8])
def test_turned_values_of_more_than_a_stage(kv):
    """Beyond the places that are held at a time, with and without chunks."""
    check([5000, 40], [4100, 30], kv=kv, d=64, layout="dmajor", hkv=1)
    check([3000] + [20] * 259, [2999] + [7] * 259, kv=kv, d=32, layout="dmajor", hkv=1)


def test_another_stream_and_few_rows_in_a_graph():
    """Long and few: tickets and flags are cleared by every run and replay."""
    lens, keep = [14000, 2500], [2000, 1200]
    c = mr.paged(lens, 2, 64, 16, torch.bfloat16, seed=8)
    w = weights_of(c, 2, 16, 8, "long")
    kt = torch.tensor(keep, dtype=torch.int32).cuda()
    a, b = mr.to_gpu(c), mr.to_gpu(c)
    wa, wb = w.cuda(), w.cuda()

    def cut(x, wt, **kw):
        return eviction.evict(x["k"], x["v"], wt, x["bt"], x["ctx"], kt, recent=8, max_keep=2000,
                              v_layout="tokmajor", **kw)

    s = torch.cuda.Stream()
    graphs = []
    for _ in range(2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            graphs.append((g, cut(a, wa)))
    torch.cuda.synchronize()
    for k in range(6):
        g, kept = graphs[k % 2]
        g.replay()
        ref = cut(b, wb, stream=s)
        torch.cuda.synchronize()
        assert torch.equal(kept, ref) and torch.equal(wa, wb), k
        assert torch.equal(bits(a["k"]), bits(b["k"])) and torch.equal(bits(a["v"]), bits(b["v"]))


def test_a_capture_without_a_pool_needs_a_workspace():
    """What such a capture allocated would be freed under its graph: refused, and with a
    workspace that the caller keeps, captured and replayed."""
    hip = ctypes.CDLL("libamdhip64.so")
    c = mr.paged([900, 40], 2, 64, 16, torch.bfloat16, seed=9)
    w = weights_of(c, 2, 16, 9, "long")
    kt = torch.tensor([700, 30], dtype=torch.int32).cuda()
    ref = expected(c, w, w, [700, 30], 0, 0, 700)
    x, wg = mr.to_gpu(c), w.cuda()
    kept = torch.empty(2, 2, 700, dtype=torch.int32, device="cuda")
    ws = torch.empty(1 << 20, dtype=torch.uint8, device="cuda")

    def cut(**kw):
        eviction.evict(x["k"], x["v"], wg, x["bt"], x["ctx"], kt, max_keep=700, kept=kept,
                       v_layout="tokmajor", **kw)

    side = torch.cuda.Stream()
    graph, exe = ctypes.c_void_p(), ctypes.c_void_p()
    torch.cuda.synchronize()
    with torch.cuda.stream(side):
        h = ctypes.c_void_p(side.cuda_stream)
        assert hip.hipStreamBeginCapture(h, 1) == 0         # thread-local mode
        with pytest.raises(RuntimeError, match="workspace"):
            cut()
        cut(workspace=ws)
        assert hip.hipStreamEndCapture(h, ctypes.byref(graph)) == 0
        assert hip.hipGraphInstantiate(ctypes.byref(exe), graph, None, None,
                                       ctypes.c_size_t(0)) == 0
        assert hip.hipGraphLaunch(exe, h) == 0
        side.synchronize()
        assert torch.equal(kept.cpu(), ref[0]) and torch.equal(bits(wg), bits(ref[1]))
        assert torch.equal(bits(x["k"]), bits(ref[2])) and torch.equal(bits(x["v"]), bits(ref[3]))
        assert hip.hipGraphExecDestroy(exe) == 0 and hip.hipGraphDestroy(graph) == 0


def test_a_request_with_a_bad_table_is_left_alone():
    c = mr.paged([200, 100, 90], 2, 64, 16, torch.bfloat16, seed=4)
    w = weights_of(c, 2, 16, 4, "long")
    ref = expected(c, w, w, [50, 40, 30], 0, 0, 50, skip=(0, 2))
    c["bt"][0, 5] = c["P"]
    ctx = c["ctx"].clone()
    ctx[2] = 100000             # its table is shorter
    x, wg = mr.to_gpu(c), w.cuda()
    err = torch.zeros(1, dtype=torch.int32, device="cuda")
    kept = eviction.evict(x["k"], x["v"], wg, x["bt"], ctx.cuda(),
                          torch.tensor([50, 40, 30], dtype=torch.int32).cuda(), max_keep=50,
                          v_layout="tokmajor", errors=err)
    assert int(err) == 4
    assert torch.equal(kept.cpu(), ref[0]) and torch.equal(bits(wg), bits(ref[1]))
    assert torch.equal(bits(x["k"]), bits(ref[2])) and torch.equal(bits(x["v"]), bits(ref[3]))


def test_repeated_eviction_on_a_stream_and_in_a_graph():
    """The same plan replayed: each replay cuts what the last one left."""
    lens, keep = [900, 333], [400, 111]
    c = mr.paged(lens, 2, 128, 16, torch.bfloat16, seed=5)
    w = weights_of(c, 2, 16, 5, "long")
    kt = torch.tensor(keep, dtype=torch.int32).cuda()
    a, b = mr.to_gpu(c), mr.to_gpu(c)
    wa, wb = w.cuda(), w.cuda()

    def cut(x, wt, **kw):
        return eviction.evict(x["k"], x["v"], wt, x["bt"], x["ctx"], kt, recent=8, max_keep=400,
                              v_layout="tokmajor", **kw)

    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        kept = cut(a, wa)
    s = torch.cuda.Stream()
    torch.cuda.synchronize()
    for k in range(4):
        g.replay()
        ref = cut(b, wb, stream=s)
        torch.cuda.synchronize()
        assert torch.equal(kept, ref) and torch.equal(wa, wb), k
        assert torch.equal(bits(a["k"]), bits(b["k"])) and torch.equal(bits(a["v"]), bits(b["v"]))


# -- the steps together ---------------------------------------------------------------
@pytest.mark.parametrize("kv", [torch.bfloat16, FP8])
def test_serving_with_a_bounded_cache(kv):
    """Prompts, then decode steps that append rotated keys, decode with weights and cut
    the cache whenever a request is over its budget: against a model that holds every
    token in a list per (request, kv-head)."""
    R, hq, hkv, d, ps, budget, recent, sink = 3, 4, 2, 128, 16, 64, 8, 2
    src = torch.bfloat16
    cache = kv_cache.PagedKvCache(64, hkv, d, ps, dtype=kv, track_weights=True)
    table = rotary.cos_sin_table(4096, d)
    rids = list("abc")
    for r in rids:
        cache.add_request(r)
    g = torch.Generator().manual_seed(6)
    model = [[[] for _ in range(hkv)] for _ in rids]       # (k row, v row, weight, position)
    free0 = cache.allocator.num_free
    for step in range(40):
        counts = [50, 70, 9] if step == 0 else [1, 1, 1]
        T = sum(counts)
        q = torch.randn(T, hq, d, generator=g).to(src)
        k = torch.randn(T, hkv, d, generator=g).to(src)
        v = torch.randn(T, hkv, d, generator=g).to(src)
        at = cache.positions(rids)
        pos = [at[r] + i for r in range(R) for i in range(counts[r])]
        q_rot = cache.append_rotated(rids, q.cuda(), k.cuda(), v.cuda(), table, counts)
        _, k_rot = rotary.qk_norm_rope(q.cuda(), k.cuda(), torch.tensor(pos).cuda(), table)
        i = 0
        for r in range(R):
            for _ in range(counts[r]):
                for h in range(hkv):
                    model[r][h].append([k_rot[i, h].cpu().double(), v[i, h].double(), 0.0, pos[i]])
                i += 1
        last = torch.tensor([sum(counts[:r + 1]) - 1 for r in range(R)])
        ql = q_rot[last].contiguous()
        out = cache.decode_weighted(ql, rids, out_dtype=torch.float32)
        # an fp8 cache holds values off by 2^-4 of themselves: its model takes the weights
        # and rows the cache has
        bt, ctx = cache.block_table(rids)
        for r in range(R):
            n = len(model[r][0])
            assert int(ctx[r]) == n == cache.lens[rids[r]]
            pages = bt[r, :-(-n // ps)].long()

            def rows(pool, scale):
                t = pool.view(torch.uint8)[pages].view(kv).float().double() if kv == FP8 \
                    else pool[pages].double()
                if scale is not None:
                    t = t * scale.view(-1, hkv)[pages].double()[:, :, None, None]
                return t.transpose(0, 1).reshape(hkv, -1, d)[:, :n].cpu()
            K, V = rows(cache.k_pool, cache.k_scale), rows(cache.v_pool, cache.v_scale)
            W = cache.weights[pages].transpose(0, 1).reshape(hkv, -1)[:, :n].cpu().double()
            for h in range(hkv):
                mk = torch.stack([e[0] for e in model[r][h]])
                mv = torch.stack([e[1] for e in model[r][h]])
                if kv == FP8:
                    # a code is off by 2^-4 of its value or half a subnormal step of its
                    # page's scale, at most twice (an append and a re-encoding)
                    assert ((K[h] - mk).abs() <= 2.0 ** -3 * mk.abs() + 2.0 ** -8).all()
                else:
                    assert torch.equal(K[h], mk) and torch.equal(V[h], mv)
                p, rel = mr.maps(ql[r].cpu().double().view(hkv, hq // hkv, d)[h], K[h], d ** -0.5,
                                 d)
                o = out[r].cpu().double().view(hkv, hq // hkv, d)[h]
                assert ((o - p @ V[h]).abs() <= (p @ V[h].abs()) * (rel + 2.0 ** -16)
                        + 2.0 ** -24).all(), step
                add = p.sum(0)
                old = torch.tensor([e[2] for e in model[r][h]], dtype=torch.float64)
                assert ((W[h] - old - add).abs() <= (p * rel).sum(0)
                        + 4 * mr.EPS32 * (old + add)).all(), step
                for e, x in zip(model[r][h], W[h].tolist()):
                    e[2] = x
        before = cache.lengths(rids)
        if (before > budget + 8).any() or step == 1:
            kept = cache.evict(rids, budget, sink=sink, recent=recent).cpu()
            for r in range(R):
                n = int(before[r])
                m = min(n, budget)
                for h in range(hkv):
                    want = mr.kept_ref([e[2] for e in model[r][h]], n, m, sink, recent)
                    assert kept[r, h, :m].tolist() == want
                    model[r][h] = [model[r][h][t] for t in want]
            assert (cache.lengths(rids) == [min(int(n), budget) for n in before]).all()
            used = sum(len(cache.pages[r]) for r in rids)
            assert used == sum(-(-len(m[0]) // ps) for m in model)
            assert cache.allocator.num_free == free0 - used
    assert (cache.positions(rids) == [50 + 39, 70 + 39, 9 + 39]).all()


def test_cache_refuses_to_cut_tokens_without_a_weight():
    cache = kv_cache.PagedKvCache(16, 1, 64, 16, track_weights=True)
    cache.add_request(0)
    k = torch.randn(40, 1, 64, device="cuda").bfloat16()
    cache.append([0], k, k, [40])
    with pytest.raises(ValueError, match="without a weight"):
        cache.evict([0], 20, recent=10)
    q = torch.randn(1, 2, 64, device="cuda").bfloat16()
    cache.decode_weighted(q, [0])
    cache.append([0], k[:3], k[:3], [3])
    cache.evict([0], 20, recent=10)
    assert cache.lens[0] == 20 and cache.positions([0]).tolist() == [43]
    cache.truncate([0], [18])
    cache.append([0], k[:1], k[:1])
    with pytest.raises(ValueError, match="twice"):
        cache.decode_weighted(q.repeat(2, 1, 1), [0, 0])
    with pytest.raises(ValueError, match="keeps no weights"):
        kv_cache.PagedKvCache(4, 1, 64).evict([], 1)
