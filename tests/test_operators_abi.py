"""The argument blocks of the decode with attention maps, the norm with rotation and
the eviction without a GPU: their layout as C has it, their defaults, and what the
C entries and the Python calls refuse before anything is launched."""
import ctypes
import os
import subprocess

import pytest
import torch

import decode_maps
import eviction
import kv_cache
import rotary
import sched_abi as abi

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
STRUCTS = [abi.SchedMapsArgs, abi.SchedRotaryArgs, abi.SchedEvictArgs]


def test_struct_layouts_match_c(tmp_path):
    src = tmp_path / "layout.c"
    lines = []
    for s in STRUCTS:
        lines.append(f'printf("%zu\\n", sizeof({s.__name__}));')
        lines += [f'printf("%zu\\n", offsetof({s.__name__}, {n}));' for n, _ in s._fields_]
    src.write_text('#include <stddef.h>\n#include <stdio.h>\n#include "sched_kv.h"\n'
                   "int main(void) {\n" + "\n".join(lines) + "\nreturn 0; }\n")
    exe = tmp_path / "layout"
    subprocess.run(["gcc", "-I", os.path.join(ROOT, "include"), str(src), "-o", str(exe)],
                   check=True)
    got = [int(x) for x in subprocess.run([str(exe)], capture_output=True, text=True,
                                          check=True).stdout.split()]
    want = []
    for s in STRUCTS:
        want.append(ctypes.sizeof(s))
        want += [getattr(s, n).offset for n, _ in s._fields_]
    assert got == want


@pytest.mark.parametrize("name,default", [("maps", abi.default_maps_args),
                                          ("rotary", abi.default_rotary_args),
                                          ("evict", abi.default_evict_args)])
def test_defaults_match(schedlib, name, default):
    c = type(default())()
    getattr(schedlib, f"sched_{name}_default_args")(ctypes.byref(c))
    assert bytes(c) == bytes(default())
    getattr(schedlib, f"sched_{name}_default_args")(None)


PTR = ctypes.c_void_p(0x10000)


def fill(a, **kw):
    for n, t in a._fields_:
        if t is ctypes.c_void_p and n not in ("page_indptr", "k_scale", "v_scale", "errors"):
            setattr(a, n, PTR)
    for n, v in kw.items():
        setattr(a, n, v)
    return a


def maps_args(**kw):
    base = dict(num_requests=2, num_q_heads=8, num_kv_heads=2, head_dim=128, page_size=16,
                bt_stride=4, max_pages=4, num_pages=8, v_dim_stride=1, v_tok_stride=128,
                workspace_bytes=1 << 30)
    return fill(abi.default_maps_args(), **{**base, **kw})


@pytest.mark.parametrize("kw,msg", [
    (dict(abi_version=9), "abi_version"), (dict(op=2), "op 2"), (dict(kv_dtype=7), "dtypes"),
    (dict(q_dtype=abi.FP8_E4M3), "dtypes"), (dict(o_dtype=abi.FP8_E4M3), "dtypes"),
    (dict(num_kv_heads=0), "multiple"), (dict(num_q_heads=7), "multiple"),
    (dict(num_q_heads=34), "at most 16"), (dict(op=1, num_q_heads=18), "at most 8"),
    (dict(head_dim=96), "head_dim"), (dict(op=1, head_dim=32), "head_dim"),
    (dict(page_size=8), "page_size"), (dict(page_size=272), "page_size"),
    (dict(flags=abi.FLAG_SPLIT), "flags"), (dict(num_pages=0), "num_pages"),
    (dict(max_pages=1 << 30, bt_stride=1 << 30), "tables"),
    (dict(ctx_lens=None), "required"), (dict(weights=None), "weights is required"),
    (dict(op=1, lam=None), "lam is required"), (dict(bt_stride=3), "bt_stride"),
    (dict(v_dim_stride=2), "V needs"), (dict(q=ctypes.c_void_p(0x10001)), "aligned"),
    (dict(workspace=None), "workspace"), (dict(workspace_bytes=64), "workspace"),
    (dict(workspace=ctypes.c_void_p(0x10010)), "workspace"),
    (dict(kv_dtype=abi.FP8_E4M3), "k_scale"),
])
def test_maps_refusals(schedlib, kw, msg):
    assert schedlib.sched_decode_maps(ctypes.byref(maps_args(**kw)), None) != 0
    assert msg in abi.last_error()
    assert schedlib.sched_decode_maps(None, None) != 0


def test_maps_nothing_to_do(schedlib):
    assert schedlib.sched_decode_maps(ctypes.byref(maps_args(num_requests=0)), None) == 0
    assert schedlib.sched_decode_maps_workspace_bytes(None) == -1
    assert schedlib.sched_decode_maps_workspace_bytes(ctypes.byref(maps_args())) > 0


def rotary_args(**kw):
    base = dict(num_tokens=4, num_q_heads=4, num_kv_heads=2, head_dim=64, rot_dim=64, max_pos=16,
                cs_stride=64, num_requests=2, page_size=16, bt_stride=2, num_pages=8)
    return fill(abi.default_rotary_args(), **{**base, **kw})


@pytest.mark.parametrize("kw,msg", [
    (dict(abi_version=9), "abi_version"), (dict(dtype=abi.FP8_E4M3), "dtypes"),
    (dict(w_dtype=9), "dtypes"), (dict(num_q_heads=0), "heads"), (dict(num_kv_heads=0), "heads"),
    (dict(head_dim=258), "head_dim"), (dict(head_dim=6), "head_dim"), (dict(rot_dim=0), "rot_dim"),
    (dict(rot_dim=66), "rot_dim"), (dict(rot_dim=7), "rot_dim"), (dict(eps=-1.0), "eps"),
    (dict(eps=float("nan")), "eps"), (dict(q=None), "required"), (dict(max_pos=0), "required"),
    (dict(k_pool=None, k_out=None), "k_out"), (dict(cs_stride=32), "cs_stride"),
    (dict(v=None), "a cache needs"), (dict(append_indptr=None), "a cache needs"),
    (dict(page_size=0), "page_size"), (dict(num_pages=0), "num_pages"), (dict(bt_stride=0), "bt_stride"),
    (dict(k=ctypes.c_void_p(0x10001)), "aligned"), (dict(num_tokens=1 << 31), "num_tokens"),
    (dict(vp_dim_stride=16, vp_tok_stride=2), "V needs"),
])
def test_rotary_refusals(schedlib, kw, msg):
    assert schedlib.sched_qk_norm_rope(ctypes.byref(rotary_args(**kw)), None) != 0
    assert msg in abi.last_error()


def test_rotary_nothing_to_do(schedlib):
    assert schedlib.sched_qk_norm_rope(ctypes.byref(rotary_args(num_tokens=0)), None) == 0
    assert schedlib.sched_qk_norm_rope(ctypes.byref(rotary_args(num_requests=0)), None) == 0
    assert schedlib.sched_qk_norm_rope(None, None) != 0


def evict_args(**kw):
    base = dict(num_requests=2, num_kv_heads=2, head_dim=64, page_size=16, bt_stride=4,
                max_pages=4, max_keep=32, num_pages=8, v_dim_stride=1, v_tok_stride=64,
                workspace_bytes=1 << 20)
    return fill(abi.default_evict_args(), **{**base, **kw})


@pytest.mark.parametrize("kw,msg", [
    (dict(abi_version=9), "abi_version"), (dict(kv_dtype=7), "dtype"),
    (dict(num_kv_heads=0), "kv-heads"), (dict(head_dim=0), "head_dim"),
    (dict(head_dim=260), "head_dim"), (dict(page_size=6), "page_size"),
    (dict(num_pages=0), "num_pages"), (dict(max_keep=1 << 31), "max_keep"),
    (dict(max_pages=1 << 21, bt_stride=1 << 21), "2^24 tokens"),
    (dict(weights=None), "required"), (dict(kept=None), "required"), (dict(bt_stride=3), "bt_stride"),
    (dict(v_dim_stride=2), "V needs"), (dict(k_page_stride=-64), "negative"), (dict(k_pool=ctypes.c_void_p(0x10001)), "aligned"),
    (dict(kv_dtype=abi.FP8_E4M3), "k_scale"),
    (dict(kv_dtype=abi.FP8_E4M3, k_scale=PTR, v_scale=PTR, workspace=None), "workspace"),
    (dict(kv_dtype=abi.FP8_E4M3, k_scale=PTR, v_scale=PTR, workspace_bytes=8), "workspace"),
])
def test_evict_refusals(schedlib, kw, msg):
    assert schedlib.sched_kv_evict(ctypes.byref(evict_args(**kw)), None) != 0
    assert msg in abi.last_error()


def test_evict_nothing_to_do(schedlib):
    assert schedlib.sched_kv_evict(ctypes.byref(evict_args(num_requests=0)), None) == 0
    assert schedlib.sched_kv_evict(None, None) != 0
    assert schedlib.sched_kv_evict_workspace_bytes(None) == -1


# -- the Python calls: their own checks come before any device work ---------------------
def cache(kv=torch.bfloat16, d=64):
    k = torch.zeros(4, 2, 16, d, dtype=kv)
    i32 = lambda *v: torch.tensor(v, dtype=torch.int32)  # noqa: E731
    return dict(q=torch.zeros(1, 4, d, dtype=torch.bfloat16), k=k, v=k.clone(),
                bt=i32(0, 1).view(1, 2), ctx=i32(20), w=torch.zeros(4, 2, 16), keep=i32(5),
                lam=torch.zeros(4))


def weighted(c, **kw):
    return decode_maps.paged_decode_weighted(c["q"], c["k"], c["v"], c["bt"], c["ctx"], c["w"],
                                             v_layout="tokmajor", **kw)


@pytest.mark.parametrize("change,exc,msg", [
    (dict(q=torch.zeros(1, 4, 64, dtype=torch.float64)), TypeError, "q must be"),
    (dict(q=torch.zeros(2, 4, 64)), ValueError, "q must be contiguous"),
    (dict(q=torch.zeros(1, 64, 4).transpose(1, 2)), ValueError, "q must be contiguous"),
    (dict(v=torch.zeros(4, 2, 16, 64)), TypeError, "pool dtypes"),
    (dict(v=torch.zeros(4, 2, 64, 16).bfloat16()), ValueError, "v_pool must be"),
    (dict(bt=torch.zeros(1, 2)), ValueError, "int32"),
    (dict(bt=torch.zeros(2, 2, dtype=torch.int32)), ValueError, "block_table must be"),
    (dict(), ValueError, "device tensor"),
])
def test_python_decode_checks(change, exc, msg):
    with pytest.raises(exc, match=msg):
        weighted({**cache(), **change})


def test_python_weights_and_lambda_checks(monkeypatch):
    monkeypatch.setattr(decode_maps, "check_device", lambda *a, **kw: None)
    c = cache()
    for w in (torch.zeros(4, 2, 8), torch.zeros(4, 2, 16).double(),
              torch.zeros(4, 16, 2).transpose(1, 2)):
        with pytest.raises(ValueError, match="weights must be"):
            weighted({**c, "w": w})
    with pytest.raises(ValueError, match="counted"):
        weighted(c, counted=torch.zeros(2, dtype=torch.int32))
    with pytest.raises(ValueError, match="page_indptr"):
        weighted(c, page_indptr=torch.zeros(3, dtype=torch.int32))
    with pytest.raises(ValueError, match="out must be"):
        weighted(c, out=torch.zeros(1, 4, 32))
    with pytest.raises(ValueError, match="v_layout"):
        decode_maps.paged_decode_weighted(c["q"], c["k"], c["v"], c["bt"], c["ctx"], c["w"],
                                          v_layout="x")
    for kw in (dict(lam=torch.zeros(3)), dict(norm_weight=torch.zeros(32))):
        args = {"lam": c["lam"], **kw}
        with pytest.raises(ValueError, match="must be contiguous float32"):
            decode_maps.paged_decode_diff(c["q"], c["k"], c["v"], c["bt"], c["ctx"],
                                          v_layout="tokmajor", **args)


def test_python_evict_checks(monkeypatch):
    c = cache()

    def cut(**kw):
        return eviction.evict(c["k"], c["v"], kw.pop("w", c["w"]), c["bt"], c["ctx"],
                              kw.pop("keep", c["keep"]), v_layout="tokmajor", **kw)
    with pytest.raises(ValueError, match="device tensor"):
        cut()
    for kw, msg in ((dict(keep=torch.zeros(2, dtype=torch.int32)), "keep_lens"),
                    (dict(sink=-1), "negative"), (dict(recent=-1), "negative"),
                    (dict(w=torch.zeros(4, 2, 4)), "weights must be"),
                    (dict(weights_out=torch.zeros(4, 2, 4)), "weights_out must be"),
                    (dict(weights_out=torch.zeros(2, 4, 16).transpose(0, 1)), "strides"),
                    (dict(max_keep=8, kept=torch.zeros(1, 2, 9, dtype=torch.int32)), "kept must")):
        with pytest.raises(ValueError, match=msg):
            cut(**kw)


def test_python_rotary_checks():
    q, k = torch.zeros(3, 4, 64), torch.zeros(3, 2, 64)
    pos, table = torch.arange(3), rotary.cos_sin_table(8, 64, device="cpu")

    def rope(q=q, k=k, pos=pos, table=table, **kw):
        return rotary.qk_norm_rope(q, k, pos, table, **kw)
    with pytest.raises(ValueError, match="device tensor"):
        rope()
    for kw, exc, msg in ((dict(k=k.half()), TypeError, "rows must all"),
                         (dict(k=torch.zeros(2, 2, 64)), ValueError, "rows must be"),
                         (dict(pos=pos.float()), ValueError, "positions"),
                         (dict(pos=pos[:2]), ValueError, "positions"),
                         (dict(table=table.double()), ValueError, "cos_sin"),
                         (dict(q_weight=torch.zeros(32)), ValueError, "q_weight"),
                         (dict(q_weight=torch.zeros(64), k_weight=torch.zeros(64).half()),
                          TypeError, "two types"),
                         (dict(q_out=torch.zeros(3, 4, 32)), ValueError, "q_out"),
                         (dict(q=torch.zeros(3, 64, 4).transpose(1, 2)), ValueError, "contiguous")):
        with pytest.raises(exc, match=msg):
            rope(**kw)


def test_positions_count_on_after_a_cut():
    c = kv_cache.PagedKvCache(8, 1, 64, 16, device="cpu", track_weights=True)
    c.add_request("a")
    c.lens["a"] = 20
    c._counted[0], c._cut[0] = 20, 7
    assert c.positions(["a"]).tolist() == [27]
    c.lens["a"] = 12
    assert c._counted[0] == 12
    c.release("a")
    c.add_request("b")
    assert c.positions(["b"]).tolist() == [0]


def test_cos_sin_table_is_exact_to_a_rounding():
    t = rotary.cos_sin_table(100000, 8, 1e4, device="cpu")
    ang = torch.arange(100000, dtype=torch.float64)[:, None] * 1e4 ** (-torch.arange(4) / 4.0).double()
    ref = torch.cat([ang.cos(), ang.sin()], 1)
    # one rounding, and the 64-bit angle's own error at 10^5
    assert ((t.double() - ref).abs() <= 2.0 ** -24 * ref.abs() + 1e-10).all()
