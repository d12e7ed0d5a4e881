"""The decode with attention maps handed on (decode_maps) on the GPU against its
definition in 64 bits: every cache type, head dim, group and V layout, ragged
and empty requests, tables of both kinds, strided pools, weights that are fresh,
faded or left alone, streams and graphs, and determinism."""
import pytest
import torch

import decode_maps
import maps_ref as mr
import sched_abi as abi

pytestmark = pytest.mark.gpu
FP8 = mr.FP8
LENS = [1, 16, 17, 0, 300, 33, 700]


@pytest.fixture(scope="module", autouse=True)
def lib(schedlib):
    torch.cuda.init()
    return schedlib


def q_of(kv):
    return torch.bfloat16 if kv == FP8 else kv


def p_err(kind, kv):
    """The matrix cores take a probability as two halves of a 16-bit type: within 2^-16;
    with fp32 values as it is."""
    return 2.0 ** -16 if kind == "mfma" and kv != torch.float32 else 0.0


def make_q(R, hq, d, dt, seed, scale=1.0):
    g = torch.Generator().manual_seed(seed + 1000)
    return (torch.randn(R, hq, d, generator=g) * scale).to(dt)


def run_weighted(c, q, w, counted, decay, flags=0, **kw):
    x = mr.to_gpu(c)
    wg = w.cuda()
    args = dict(v_layout=x["layout"], k_scale=x["ks"], v_scale=x["vs"], page_indptr=x["pind"],
                flags=flags)
    out = decode_maps.paged_decode_weighted(
        q.cuda(), x["k"], x["v"], x["bt"], x["ctx"], wg, decay=decay,
        counted=None if counted is None else counted.cuda(), **args, **kw)
    return out, wg


def check_weighted(lens, hkv, G, d, ps, kv, layout="tokmajor", seed=1, flags=0, csr=False,
                   decay=0.9, out_dtype=None, scale=1.0, pairs=True):
    c = mr.paged(lens, hkv, d, ps, kv, layout, seed, csr=csr, pairs=pairs)
    q = make_q(len(lens), hkv * G, d, q_of(kv), seed, scale)
    g = torch.Generator().manual_seed(seed)
    w = torch.rand(c["P"], hkv, ps, generator=g)
    counted = torch.tensor([max(0, n - (i % 4)) for i, n in enumerate(lens)], dtype=torch.int32)
    # what lies past the counted tokens is not read
    for r, pages in enumerate(c["rows"]):
        for t in range(int(counted[r]), len(pages) * ps):
            w[pages[t // ps], :, t % ps] = float("nan")
    kw = {} if out_dtype is None else dict(out_dtype=out_dtype)
    out, wg = run_weighted(c, q, w, counted, decay, flags, **kw)
    x = mr.to_gpu(c)
    kind = decode_maps.kernel_kind(q.cuda(), x["k"], x["v"], x["bt"] if not csr else
                                   torch.zeros(len(lens), 1, dtype=torch.int32).cuda(),
                                   x["ctx"], v_layout=x["layout"], flags=flags)
    ro, bo, rw, bw = mr.weighted_ref(c, q, w, counted, decay, p_err=p_err(kind, kv),
                                     out_dtype=out.dtype)
    mr.close(out, ro, bo, "out")
    mr.close(wg, rw, bw, "weights")
    # slots that hold no token are the bytes they were
    still = bw == 0
    assert torch.equal(wg.cpu().view(torch.int32)[still], w.view(torch.int32)[still])
    return kind


@pytest.mark.parametrize("kv", [torch.float32, torch.bfloat16, torch.float16, FP8])
@pytest.mark.parametrize("d,G", [(64, 1), (64, 5), (128, 4), (128, 7), (256, 2), (128, 16)])
@pytest.mark.parametrize("flags", [0, abi.FLAG_FORCE_VALU])
def test_weighted_types_and_heads(kv, d, G, flags):
    check_weighted(LENS, 3, G, d, 16, kv, seed=d + G, flags=flags)


def test_weighted_head_dim_32():
    check_weighted(LENS, 2, 3, 32, 16, torch.float32)


@pytest.mark.parametrize("kv", [torch.bfloat16, FP8])
@pytest.mark.parametrize("layout", ["dmajor", "nhd"])
@pytest.mark.parametrize("ps", [16, 48, 256])
def test_weighted_layouts_and_pages(kv, layout, ps):
    check_weighted(LENS, 2, 4, 128, ps, kv, layout, seed=ps)


@pytest.mark.parametrize("d", [64, 128, 256])
@pytest.mark.parametrize("layout,ps", [("dmajor", 48), ("nhd", 16), ("dmajor", 16)])
def test_weighted_fp32_layouts(d, layout, ps):
    assert check_weighted(LENS, 2, 3, d, ps, torch.float32, layout, seed=d + ps) == "mfma"


@pytest.mark.parametrize("kv,d", [(torch.float32, 256), (torch.bfloat16, 256), (FP8, 256),
                                  (torch.float16, 64), (FP8, 64)])
def test_weighted_many_chunks(kv, d):
    """One request of some 40 chunks beside short ones, and a chunk's last token alone."""
    check_weighted([10241, 5, 0, 257], 1, 3, d, 16, kv, seed=d)


def test_weighted_whole_groups_of_chunks():
    """Chunks at the edges where a task is cut or left whole."""
    check_weighted([255, 256, 257, 383, 384, 385, 511, 512, 513], 1, 2, 128, 16, torch.bfloat16)
    check_weighted([127, 128, 129, 191, 192, 193, 255, 256, 257], 1, 2, 128, 16, torch.float32)


@pytest.mark.parametrize("kv", [torch.float32, torch.bfloat16, FP8])
def test_weighted_page_list(kv):
    check_weighted(LENS, 2, 4, 128, 32, kv, csr=True, pairs=False)


@pytest.mark.parametrize("lens", [[1], [15], [4097], [20001, 3], [64] * 70])
def test_weighted_lengths(lens):
    check_weighted(lens, 2, 4, 128, 16, torch.bfloat16, seed=sum(lens))


def test_weighted_peaked_rows():
    """Scores some hundred apart: most weights are 0 or denormal, one is near 1."""
    check_weighted([500, 40], 2, 2, 128, 16, torch.float32, scale=30.0)
    check_weighted([500, 40], 2, 2, 128, 16, torch.bfloat16, scale=30.0)


@pytest.mark.parametrize("out_dtype", [torch.float32, torch.float16])
def test_weighted_output_types(out_dtype):
    check_weighted(LENS, 2, 4, 128, 16, torch.bfloat16, out_dtype=out_dtype)


def test_weighted_sums_to_the_group_size():
    """decay 0 leaves one step's weights: a request's sum over its tokens is the number of
    q-heads of the group (n values, each off by at most 2^-20 of itself here)."""
    c = mr.paged([3000, 31], 4, 128, 16, torch.bfloat16, seed=3)
    q = make_q(2, 24, 128, torch.bfloat16, 3)
    w = torch.rand(c["P"], 4, 16)
    _, wg = run_weighted(c, q, w, None, 0.0)
    for r, pages in enumerate(c["rows"]):
        got = wg.cpu().double()[pages].transpose(0, 1).reshape(4, -1)[:, :c["lens"][r]].sum(1)
        assert ((got - 6).abs() <= 6 * 2.0 ** -14).all()


def check_diff(lens, hkv, G, d, ps, kv, layout="tokmajor", seed=1, flags=0, csr=False, norm=True,
               out_dtype=None, sm_scale=None):
    c = mr.paged(lens, hkv, d, ps, kv, layout, seed, csr=csr)
    q = make_q(len(lens), hkv * G, d, q_of(kv), seed)
    g = torch.Generator().manual_seed(seed)
    lam = torch.rand(hkv * G, generator=g) * 1.5 - 0.5
    nw = 1 + 0.3 * torch.randn(d, generator=g) if norm else None
    x = mr.to_gpu(c)
    out = decode_maps.paged_decode_diff(
        q.cuda(), x["k"], x["v"], x["bt"], x["ctx"], lam.cuda(),
        norm_weight=None if nw is None else nw.cuda(), eps=1e-5, out_scale=0.2,
        v_layout=x["layout"], page_indptr=x["pind"], k_scale=x["ks"], v_scale=x["vs"],
        flags=flags, out_dtype=out_dtype, sm_scale=sm_scale)
    kind = decode_maps.kernel_kind(q.cuda(), x["k"], x["v"], torch.zeros(
        len(lens), 1, dtype=torch.int32).cuda(), x["ctx"], diff=True, v_layout=x["layout"],
        flags=flags)
    ro, bo = mr.diff_ref(c, q, lam, nw, 1e-5, 0.2, sm_scale, p_err(kind, kv), out.dtype)
    mr.close(out, ro, bo, "out")


@pytest.mark.parametrize("kv", [torch.float32, torch.bfloat16, torch.float16, FP8])
@pytest.mark.parametrize("d,G", [(64, 2), (128, 1), (128, 8), (256, 3), (256, 8)])
@pytest.mark.parametrize("flags", [0, abi.FLAG_FORCE_VALU])
def test_diff_types_and_heads(kv, d, G, flags):
    check_diff(LENS, 2, G, d, 16, kv, seed=d + G, flags=flags)


@pytest.mark.parametrize("layout,ps,csr", [("dmajor", 16, False), ("nhd", 32, False),
                                           ("tokmajor", 80, True), ("tokmajor", 64, False)])
@pytest.mark.parametrize("norm", [True, False])
def test_diff_layouts(layout, ps, csr, norm):
    check_diff(LENS, 2, 2, 128, ps, torch.bfloat16, layout, seed=ps, csr=csr, norm=norm)


@pytest.mark.parametrize("d", [64, 128, 256])
@pytest.mark.parametrize("layout,ps,csr", [("dmajor", 48, False), ("nhd", 16, True)])
def test_diff_fp32_layouts(d, layout, ps, csr):
    check_diff(LENS, 2, 3, d, ps, torch.float32, layout, seed=d, csr=csr)


@pytest.mark.parametrize("kv,d", [(torch.float32, 256), (torch.bfloat16, 256), (FP8, 256),
                                  (torch.float16, 64), (FP8, 64)])
def test_diff_many_chunks(kv, d):
    check_diff([10241, 5, 0, 257], 1, 3, d, 16, kv, seed=d)


@pytest.mark.parametrize("lens", [[1], [9000], [130] * 40])
def test_diff_lengths(lens):
    check_diff(lens, 2, 2, 128, 16, torch.float16, seed=len(lens), out_dtype=torch.float32,
               sm_scale=0.2)


def test_diff_lambda_is_the_formula():
    g = torch.Generator().manual_seed(5)
    v = [torch.randn(64, generator=g) * 0.1 for _ in range(4)]
    got = decode_maps.diff_lambda(*[t.cuda() for t in v], 0.8).cpu().double()
    d = [t.double() for t in v]
    ref = torch.exp(d[0] @ d[1]) - torch.exp(d[2] @ d[3]) + 0.8
    # 64-term dots of terms below 0.1, exps near 1: 80 roundings of at most 2
    assert abs(float(got - ref)) <= 160 * mr.EPS32


def test_one_token_is_its_value():
    """A single token has weight 1 whatever its score: the output row is V's."""
    c = mr.paged([1, 1], 2, 128, 16, torch.bfloat16, seed=8)
    q = make_q(2, 4, 128, torch.bfloat16, 8)
    w = torch.zeros(c["P"], 2, 16)
    out, wg = run_weighted(c, q, w, torch.zeros(2, dtype=torch.int32), 1.0)
    for r, (_, v) in enumerate(c["seqs"]):
        want = v[:, 0].repeat_interleave(2, 0)
        assert torch.equal(out[r].cpu().double(), want)
        assert torch.equal(wg.cpu()[c["rows"][r][0], :, 0], torch.full((2,), 2.0))


def test_bits_do_not_depend_on_the_run():
    c = mr.paged([5000, 77, 1200], 2, 128, 16, torch.bfloat16, seed=9)
    q = make_q(3, 8, 128, torch.bfloat16, 9)
    w = torch.rand(c["P"], 2, 16)
    a, wa = run_weighted(c, q, w, None, 0.5)
    for _ in range(3):
        b, wb = run_weighted(c, q, w, None, 0.5)
        assert torch.equal(a, b) and torch.equal(wa, wb)


def test_other_stream_and_given_buffers():
    c = mr.paged([900, 50], 2, 128, 16, torch.bfloat16, seed=10)
    q = make_q(2, 8, 128, torch.bfloat16, 10)
    w = torch.rand(c["P"], 2, 16)
    want, ww = run_weighted(c, q, w, None, 1.0)
    x, wg, qg = mr.to_gpu(c), w.cuda(), q.cuda()
    s = torch.cuda.Stream()
    out = torch.empty_like(qg)
    ws = torch.full((8 << 20,), 255, dtype=torch.uint8, device="cuda")
    torch.cuda.synchronize()
    decode_maps.paged_decode_weighted(qg, x["k"], x["v"], x["bt"], x["ctx"], wg, out=out,
                                      v_layout="tokmajor", stream=s, workspace=ws)
    s.synchronize()
    assert torch.equal(out, want) and torch.equal(wg, ww)


def test_graph_replays_match_eager():
    c = mr.paged([900, 50, 2000], 2, 128, 16, torch.bfloat16, seed=11)
    x = mr.to_gpu(c)
    q = make_q(3, 8, 128, torch.bfloat16, 11).cuda()
    w0 = torch.rand(c["P"], 2, 16).cuda()
    lam = torch.rand(4).cuda()
    wg = w0.clone()
    qd = q[:, :4].contiguous()

    def step(wt):
        o = decode_maps.paged_decode_weighted(q, x["k"], x["v"], x["bt"], x["ctx"], wt, decay=0.5,
                                              v_layout="tokmajor")
        return o, decode_maps.paged_decode_diff(qd, x["k"], x["v"], x["bt"], x["ctx"], lam,
                                                v_layout="tokmajor")

    step(wg)
    torch.cuda.synchronize()
    graphs = []
    for _ in range(2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs = step(wg)
        graphs.append((g, outs))
    wg.copy_(w0)
    we = w0.clone()
    for k in range(6):
        q.normal_(generator=torch.Generator(device="cuda").manual_seed(k))
        qd.copy_(q[:, :4])
        g, outs = graphs[k % 2]
        g.replay()
        ref = step(we)
        torch.cuda.synchronize()
        for a, b in zip(outs, ref):
            assert torch.equal(a.view(torch.int16), b.view(torch.int16)), k
        assert torch.equal(wg, we), k


def test_a_page_outside_the_pool_is_not_followed():
    """Its request's rows mean nothing; the others and every weight elsewhere hold."""
    c = mr.paged([100, 90], 2, 128, 16, torch.bfloat16, seed=12)
    q = make_q(2, 4, 128, torch.bfloat16, 12)
    w = torch.rand(c["P"], 2, 16)
    good, wgood = run_weighted(c, q, w, None, 1.0)
    c["bt"] = c["bt"].clone()
    c["bt"][0, 2], c["bt"][0, 4] = -1, c["P"]
    out, wg = run_weighted(c, q, w, None, 1.0)
    assert torch.equal(out[1], good[1])
    rest = [p for p in range(c["P"]) if p not in c["rows"][0]]
    assert torch.equal(wg[rest], wgood[rest])
    lost = [c["rows"][0][2], c["rows"][0][4]]
    assert torch.equal(wg.cpu()[lost], w[lost])


def test_a_context_past_the_table_is_cut():
    c = mr.paged([64, 40], 2, 64, 16, torch.bfloat16, seed=13)
    q = make_q(2, 2, 64, torch.bfloat16, 13)
    w = torch.rand(c["P"], 2, 16)
    c["bt"] = c["bt"][:, :4].contiguous()
    want, ww = run_weighted(c, q, w, None, 1.0)
    c["ctx"] = torch.tensor([10 ** 9, 40], dtype=torch.int32)
    got, wg = run_weighted(c, q, w, None, 1.0)
    assert torch.equal(got, want) and torch.equal(wg, ww)
    c["ctx"] = torch.tensor([-5, 40], dtype=torch.int32)
    got, wg = run_weighted(c, q, w, None, 1.0)
    assert got[0].isnan().all() and torch.equal(got[1], want[1])
