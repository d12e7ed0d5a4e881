"""Norm of queries and keys with the position rotation on the GPU against the
definition in 64 bits: types, head dims, rotated parts, both pairings, strided and
in-place rows, far positions, and rows that go into the cache."""
import pytest
import torch

import kv_cache
import maps_ref as mr
import rotary

pytestmark = pytest.mark.gpu
TYPES = [torch.float32, torch.bfloat16, torch.float16]


@pytest.fixture(scope="module", autouse=True)
def lib(schedlib):
    torch.cuda.init()
    return schedlib


def ref_rows(x, w, pos, table, eps, inter):
    """(rows, bound) in 64 bits. The bound: the norm's factor is off by at most
    (d + 8) half steps of 32 bits (a sum of d squares in any order, a root, a product), the
    products and sums of the rotation by three more, of the magnitudes that enter;
    then one rounding to the rows' type."""
    d, half = x.shape[-1], table.shape[1] // 2
    y = x.double()
    if w is not None:
        y = y / torch.sqrt(y.pow(2).mean(-1, keepdim=True) + eps) * w.double()
    cs = table.double()[pos]
    c, s = cs[:, None, :half], cs[:, None, half:]
    a, b = (y[..., 0:2 * half:2], y[..., 1:2 * half:2]) if inter else (y[..., :half],
                                                                     y[..., half:2 * half])
    ra, rb = a * c - b * s, b * c + a * s
    ma, mb = (a * c).abs() + (b * s).abs(), (b * c).abs() + (a * s).abs()
    out, mag = y.clone(), y.abs()
    if inter:
        out[..., 0:2 * half:2], out[..., 1:2 * half:2] = ra, rb
        mag[..., 0:2 * half:2], mag[..., 1:2 * half:2] = ma, mb
    else:
        out[..., :half], out[..., half:2 * half] = ra, rb
        mag[..., :half], mag[..., half:2 * half] = ma, mb
    tiny = torch.finfo(x.dtype).smallest_normal * torch.finfo(x.dtype).eps
    return out, (d + 12) * mr.EPS32 * mag + mr.half_step(x.dtype) * out.abs() + tiny


def case(T, hq, hkv, d, dt, seed, w_dtype=torch.float32, norm=True, scale=1.0):
    g = torch.Generator().manual_seed(seed)
    qkv = (torch.randn(T, hq + 2 * hkv, d, generator=g) * scale).to(dt)
    qw = (1 + 0.3 * torch.randn(d, generator=g)).to(w_dtype) if norm else None
    kw = (1 + 0.3 * torch.randn(d, generator=g)).to(w_dtype) if norm else None
    return qkv, qw, kw


def cu(t):
    return None if t is None else t.cuda()


@pytest.mark.parametrize("dt", TYPES)
@pytest.mark.parametrize("inter", [False, True])
@pytest.mark.parametrize("d,rot", [(128, 128), (64, 64), (256, 256), (128, 64), (64, 16),
                                   (96, 96), (80, 20), (36, 34), (4, 2), (32, 32)])
def test_rows(dt, inter, d, rot):
    hq, hkv, T = 5, 2, 7
    qkv, qw, kw = case(T, hq, hkv, d, dt, d + rot)
    table = rotary.cos_sin_table(1000, rot)
    pos = torch.tensor([0, 999, 3, 3, 500, 77, 1])
    x = qkv.cuda()
    q, k = rotary.qk_norm_rope(x[:, :hq], x[:, hq:hq + hkv], pos.cuda(), table, q_weight=cu(qw),
                               k_weight=cu(kw), eps=1e-6, interleaved=inter)
    assert q.is_contiguous() and k.is_contiguous()
    for got, src, w in ((q, qkv[:, :hq], qw), (k, qkv[:, hq:hq + hkv], kw)):
        mr.close(got, *ref_rows(src, w, pos, table.cpu(), 1e-6, inter))
    assert torch.equal(x.cpu(), qkv)


@pytest.mark.parametrize("T", [1, 2, 63, 1000])
@pytest.mark.parametrize("norm", [True, False])
def test_counts_of_tokens(T, norm):
    qkv, qw, kw = case(T, 32, 8, 128, torch.bfloat16, T, norm=norm)
    table = rotary.cos_sin_table(4096, 128, 1e6)
    pos = torch.randint(0, 4096, (T,), dtype=torch.int32)
    x = qkv.cuda()
    q, k = rotary.qk_norm_rope(x[:, :32], x[:, 32:40], pos.cuda(), table, q_weight=cu(qw),
                               k_weight=cu(kw))
    mr.close(q, *ref_rows(qkv[:, :32], qw, pos.long(), table.cpu(), 1e-6, False))
    mr.close(k, *ref_rows(qkv[:, 32:40], kw, pos.long(), table.cpu(), 1e-6, False))


@pytest.mark.parametrize("dt", TYPES)
@pytest.mark.parametrize("inter", [False, True])
@pytest.mark.parametrize("d,rot", [(128, 128), (64, 32), (256, 64), (96, 96), (80, 20)])
def test_many_tokens(dt, inter, d, rot):
    """Enough rows that a lane has several."""
    T, hq, hkv = 3001, 6, 2
    qkv, qw, kw = case(T, hq, hkv, d, dt, d + rot)
    table = rotary.cos_sin_table(4096, rot)
    pos = torch.randint(0, 4096, (T,))
    x = qkv.cuda()
    q, k = rotary.qk_norm_rope(x[:, :hq], x[:, hq:hq + hkv], pos.cuda(), table, q_weight=cu(qw),
                               k_weight=cu(kw), eps=1e-6, interleaved=inter)
    mr.close(q, *ref_rows(qkv[:, :hq], qw, pos, table.cpu(), 1e-6, inter))
    mr.close(k, *ref_rows(qkv[:, hq:hq + hkv], kw, pos, table.cpu(), 1e-6, inter))


def test_on_another_stream():
    qkv, qw, kw = case(50, 8, 2, 128, torch.bfloat16, 12)
    table = rotary.cos_sin_table(64, 128)
    x, pos = qkv.cuda(), torch.arange(50).cuda()
    args = (x[:, :8], x[:, 8:10], pos, table)
    want = rotary.qk_norm_rope(*args, q_weight=cu(qw), k_weight=cu(kw))
    s = torch.cuda.Stream()
    torch.cuda.synchronize()
    with torch.cuda.stream(s):
        got = rotary.qk_norm_rope(*args, q_weight=cu(qw), k_weight=cu(kw))
    s.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(got, want))


@pytest.mark.parametrize("w_dtype", [torch.bfloat16, torch.float16])
def test_weight_types_and_one_sided_norm(w_dtype):
    qkv, qw, _ = case(9, 4, 4, 128, torch.bfloat16, 3, w_dtype=w_dtype)
    table = rotary.cos_sin_table(64, 128)
    pos = torch.arange(9)
    x = qkv.cuda()
    q, k = rotary.qk_norm_rope(x[:, :4], x[:, 4:8], pos.cuda(), table, q_weight=cu(qw))
    mr.close(q, *ref_rows(qkv[:, :4], qw, pos, table.cpu(), 1e-6, False))
    mr.close(k, *ref_rows(qkv[:, 4:8], None, pos, table.cpu(), 1e-6, False))


@pytest.mark.parametrize("inter,rot", [(False, 128), (True, 128), (False, 20)])
def test_in_place(inter, rot):
    qkv, qw, kw = case(33, 8, 2, 128, torch.float16, 4)
    table = rotary.cos_sin_table(64, rot)
    pos = torch.arange(33)
    x = qkv.cuda()
    want = rotary.qk_norm_rope(x[:, :8], x[:, 8:10], pos.cuda(), table, q_weight=cu(qw),
                               k_weight=cu(kw), interleaved=inter)
    got = rotary.qk_norm_rope(x[:, :8], x[:, 8:10], pos.cuda(), table, q_weight=cu(qw),
                              k_weight=cu(kw), interleaved=inter, q_out=x[:, :8],
                              k_out=x[:, 8:10])
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    assert torch.equal(x[:, 10:].cpu(), qkv[:, 10:])        # the values beside them


def test_odd_strides_and_offsets():
    """Rows that start at any element: no wide loads to rely on."""
    dt, T, hq, hkv, d = torch.bfloat16, 6, 3, 2, 64
    qkv, qw, kw = case(T, hq, hkv, d, dt, 6)
    table = rotary.cos_sin_table(64, 64)
    pos = torch.arange(T)
    flat = torch.zeros(T * 700 + 1, dtype=dt, device="cuda")
    q = flat[1:].as_strided((T, hq, d), (699, 67, 1), 1)
    k = flat[1:].as_strided((T, hkv, d), (699, 65, 1), 300)
    q.copy_(qkv[:, :hq])
    k.copy_(qkv[:, hq:hq + hkv])
    gq, gk = rotary.qk_norm_rope(q, k, pos.cuda(), table, q_weight=cu(qw), k_weight=cu(kw))
    mr.close(gq, *ref_rows(qkv[:, :hq], qw, pos, table.cpu(), 1e-6, False))
    mr.close(gk, *ref_rows(qkv[:, hq:hq + hkv], kw, pos, table.cpu(), 1e-6, False))


def test_zero_rows_and_large_values():
    qkv, qw, kw = case(3, 2, 1, 128, torch.bfloat16, 7, scale=1e15)
    qkv[1] = 0
    table = rotary.cos_sin_table(8, 128)
    pos = torch.arange(3)
    x = qkv.cuda()
    q, _ = rotary.qk_norm_rope(x[:, :2], x[:, 2:3], pos.cuda(), table, q_weight=cu(qw),
                               k_weight=cu(kw))
    mr.close(q, *ref_rows(qkv[:, :2], qw, pos, table.cpu(), 1e-6, False))
    assert (q[1] == 0).all()


def test_positions_outside_the_table_are_counted_and_not_written():
    qkv, qw, kw = case(5, 2, 1, 64, torch.bfloat16, 8)
    table = rotary.cos_sin_table(16, 64)
    pos = torch.tensor([0, 16, -1, 15, 1 << 40])
    x = qkv.cuda()
    qo = torch.full((5, 2, 64), 7.0, dtype=torch.bfloat16, device="cuda")
    err = torch.zeros(1, dtype=torch.int32, device="cuda")
    q, _ = rotary.qk_norm_rope(x[:, :2], x[:, 2:3], pos.cuda(), table, q_weight=cu(qw),
                               k_weight=cu(kw), q_out=qo, errors=err)
    assert int(err) == 3
    assert (q[[1, 2, 4]] == 7).all()
    good = [0, 3]
    mr.close(q[good], *ref_rows(qkv[good, :2], qw, pos[good], table.cpu(), 1e-6, False))


# -- into the cache ---------------------------------------------------------------
def fill(counts, held, hkv, d, ps, dt, layout="tokmajor"):
    c = kv_cache.PagedKvCache(256, hkv, d, ps, dtype=dt, v_layout=layout)
    g = torch.Generator(device="cuda").manual_seed(1)
    for r in range(len(counts)):
        c.add_request(r)
    n = sum(held)
    src = torch.bfloat16 if dt == mr.FP8 else dt
    if n:
        k, v = (torch.randn(n, hkv, d, generator=g, device="cuda").to(src) for _ in range(2))
        c.append(list(range(len(counts))), k, v, held)
    return c


@pytest.mark.parametrize("dt", TYPES + [mr.FP8])
@pytest.mark.parametrize("layout", ["tokmajor", "dmajor"])
@pytest.mark.parametrize("counts,held", [([1, 1, 1], [0, 15, 40]), ([37, 0, 5, 16], [3, 9, 0, 16])])
def test_append_matches_the_writer(dt, layout, counts, held):
    """The pools hold what kv_cache.append writes for the rotated keys, bit for bit."""
    hq, hkv, d, ps = 8, 2, 128, 16
    T, src = sum(counts), torch.bfloat16 if dt == mr.FP8 else dt
    qkv, qw, kw = case(T, hq, hkv, d, src, 9)
    x, rids = qkv.cuda(), list(range(len(counts)))
    table = rotary.cos_sin_table(512, d)
    q, k, v = x[:, :hq], x[:, hq:hq + hkv], x[:, hq + hkv:]
    w = dict(q_weight=cu(qw), k_weight=cu(kw))
    a, b = fill(counts, held, hkv, d, ps, dt, layout), fill(counts, held, hkv, d, ps, dt, layout)
    first = a.positions(rids)
    pos = torch.tensor([first[r] + i for r in rids for i in range(counts[r])], dtype=torch.int32)
    err = torch.zeros(1, dtype=torch.int32, device="cuda")
    got = a.append_rotated(rids, q, k, v, table, counts, errors=err, **w)
    q_rot, k_rot = rotary.qk_norm_rope(q, k, pos.cuda(), table, **w)
    b.append(rids, k_rot, v.contiguous(), counts)
    assert torch.equal(got, q_rot) and int(err) == 0
    raw = lambda t: t.view(torch.uint8) if dt == mr.FP8 else t  # noqa: E731
    assert torch.equal(raw(a.k_pool), raw(b.k_pool)) and torch.equal(raw(a.v_pool), raw(b.v_pool))
    if dt == mr.FP8:
        assert torch.equal(a.k_scale, b.k_scale) and torch.equal(a.v_scale, b.v_scale)


@pytest.mark.parametrize("dt", TYPES)
@pytest.mark.parametrize("layout", ["tokmajor", "dmajor"])
@pytest.mark.parametrize("T,held", [(7, 9), (5000, 13)])
@pytest.mark.parametrize("d,ps", [(128, 16), (96, 7)])
def test_append_leaves_the_other_slots(dt, layout, T, held, d, ps):
    """Slots behind the last token, before the first and of other pages keep their bytes."""
    hq, hkv = 4, 2
    n = -(-(held + T) // ps)
    g = torch.Generator().manual_seed(T)
    qkv, qw, kw = case(T, hq, hkv, d, dt, 13)
    kp = torch.randn(n + 2, hkv, ps, d, generator=g).to(dt)
    vp = torch.randn(*((n + 2, hkv, d, ps) if layout == "dmajor" else kp.shape),
                     generator=g).to(dt)
    pages = torch.randperm(n + 2, generator=g)[:n]
    x, kd, vd = qkv.cuda(), kp.cuda(), vp.cuda()
    table = rotary.cos_sin_table(8192, d)
    pos = torch.arange(T) + held
    i32 = lambda v: torch.tensor(v, dtype=torch.int32, device="cuda")  # noqa: E731
    err = torch.zeros(1, dtype=torch.int32, device="cuda")
    q = rotary.append_rotated(x[:, :hq], x[:, hq:hq + hkv], x[:, hq + hkv:], pos.cuda(), table,
                              i32([0, T]), i32([held + T]), kd, vd, pages.int()[None].cuda(),
                              v_layout=layout, q_weight=cu(qw), k_weight=cu(kw), errors=err)
    rq, rk = rotary.qk_norm_rope(x[:, :hq], x[:, hq:hq + hkv], pos.cuda(), table, q_weight=cu(qw),
                                 k_weight=cu(kw))
    at = torch.arange(held, held + T)
    p, s = pages[at // ps], at % ps
    kp[p, :, s] = rk.cpu()
    if layout == "dmajor":
        vp[p, :, :, s] = qkv[:, hq + hkv:]
    else:
        vp[p, :, s] = qkv[:, hq + hkv:]
    assert int(err) == 0 and torch.equal(q, rq)
    assert torch.equal(kd.cpu(), kp) and torch.equal(vd.cpu(), vp)


@pytest.mark.parametrize("layout", ["tokmajor", "dmajor"])
@pytest.mark.parametrize("counts", [[1, 1, 1, 1], [3, 1200, 700, 1100]])
@pytest.mark.parametrize("csr", [False, True])
def test_append_skips_what_has_no_place(layout, counts, csr):
    """Request 1 has a page outside the pool, request 2 a table that is too short (a CSR one
    by its own list); some positions lie outside the rotation's table."""
    dt, hq, hkv, d, ps = torch.bfloat16, 6, 2, 128, 16
    T, R, held = sum(counts), 4, [5, 0, 20, 33]
    g = torch.Generator().manual_seed(T)
    qkv, qw, kw = case(T, hq, hkv, d, dt, 14)
    need = [-(-(h + n) // ps) for h, n in zip(held, counts)]
    have = [n - 1 if r == 2 else n for r, n in enumerate(need)]
    P = sum(need) + 1
    perm = torch.randperm(P, generator=g).tolist()
    rows, at = [], 0
    for n in have:
        rows.append(perm[at:at + n])
        at += n
    rows[1][-1] = P
    kp = torch.randn(P, hkv, ps, d, generator=g).to(dt)
    vp = torch.randn(*((P, hkv, d, ps) if layout == "dmajor" else kp.shape), generator=g).to(dt)
    pos = torch.randint(0, 512, (T,), generator=g)
    pos[torch.rand(T, generator=g) < 0.2] = 512
    pos[0] = 3
    table = rotary.cos_sin_table(512, d)
    app = [0]
    for n in counts:
        app.append(app[-1] + n)
    i32 = lambda v: torch.tensor(v, dtype=torch.int32, device="cuda")  # noqa: E731
    if csr:
        ind = [0]
        for r in rows:
            ind.append(ind[-1] + len(r))
        bt, tk = i32([p for r in rows for p in r]), dict(page_indptr=i32(ind))
    else:
        width = max(need)
        bt, tk = i32([r + [-1] * (width - len(r)) for r in rows]), {}
    x, kd, vd = qkv.cuda(), kp.cuda(), vp.cuda()
    err = torch.zeros(1, dtype=torch.int32, device="cuda")
    qo = torch.full((T, hq, d), 7.0, dtype=dt, device="cuda")
    q = rotary.append_rotated(x[:, :hq], x[:, hq:hq + hkv], x[:, hq + hkv:], pos.cuda(), table,
                              i32(app), i32([h + n for h, n in zip(held, counts)]), kd, vd, bt,
                              v_layout=layout, q_weight=cu(qw), k_weight=cu(kw), errors=err,
                              q_out=qo, **tk)
    rq, rk = rotary.qk_norm_rope(x[:, :hq], x[:, hq:hq + hkv], pos.clamp(max=511).cuda(), table,
                                 q_weight=cu(qw), k_weight=cu(kw))
    rk, bad = rk.cpu(), 0
    for r in range(R):
        for i in range(counts[r]):
            t, b, s = app[r] + i, (held[r] + i) // ps, (held[r] + i) % ps
            if pos[t] == 512:
                bad += 1
                continue
            if b >= len(rows[r]) or rows[r][b] == P:
                bad += hkv
                continue
            kp[rows[r][b], :, s] = rk[t]
            if layout == "dmajor":
                vp[rows[r][b], :, :, s] = qkv[t, hq + hkv:]
            else:
                vp[rows[r][b], :, s] = qkv[t, hq + hkv:]
    ok = pos < 512
    assert torch.equal(q.cpu()[ok], rq.cpu()[ok]) and (q.cpu()[~ok] == 7).all()
    assert torch.equal(kd.cpu(), kp) and torch.equal(vd.cpu(), vp)
    assert int(err) == bad


def test_append_without_a_place_is_counted():
    hq, hkv, d, ps = 2, 3, 64, 16
    qkv, qw, kw = case(20, hq, hkv, d, torch.bfloat16, 10)
    x = qkv.cuda()
    table = rotary.cos_sin_table(64, d)
    kp = torch.full((4, hkv, ps, d), 5.0, dtype=torch.bfloat16, device="cuda")
    vp = kp.clone()
    i32 = lambda v: torch.tensor(v, dtype=torch.int32, device="cuda")  # noqa: E731
    err = torch.zeros(1, dtype=torch.int32, device="cuda")
    # request 0: a page outside the pool for its 4 rows; request 1: 16 good rows of page 2
    q = rotary.append_rotated(x[:, :hq], x[:, hq:hq + hkv], x[:, hq + hkv:],
                              torch.arange(20, device="cuda"), table, i32([0, 4, 20]), i32([4, 16]),
                              kp, vp, i32([[4], [2]]), v_layout="tokmajor", q_weight=cu(qw),
                              k_weight=cu(kw), errors=err)
    assert int(err) == 4 * hkv
    mr.close(q, *ref_rows(qkv[:, :hq], qw, torch.arange(20), table.cpu(), 1e-6, False))
    assert (kp[[0, 1, 3]] == 5).all() and (vp[[0, 1, 3]] == 5).all()
    assert torch.equal(vp[2], x[4:, hq + hkv:].transpose(0, 1))


def test_graph_replays_match_eager():
    hq, hkv, d = 8, 2, 128
    qkv, qw, kw = case(3, hq, hkv, d, torch.bfloat16, 11)
    x = qkv.cuda()
    table = rotary.cos_sin_table(512, d)
    pos = torch.tensor([5, 6, 7], device="cuda")
    w = dict(q_weight=cu(qw), k_weight=cu(kw))
    rotary.qk_norm_rope(x[:, :hq], x[:, hq:hq + hkv], pos, table, **w)
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        out = rotary.qk_norm_rope(x[:, :hq], x[:, hq:hq + hkv], pos, table, **w)
    for k in range(4):
        x.normal_()
        pos += 11
        g.replay()
        ref = rotary.qk_norm_rope(x[:, :hq], x[:, hq:hq + hkv], pos, table, **w)
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(out, ref)), k
