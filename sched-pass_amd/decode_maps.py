"""Decode steps whose attention maps are used beyond softmax(q K^T) V, on the pools
and page tables of sched_pd.paged_decode, through the C ABI (`sched_decode_maps` in
include/sched_pd.h):

  * paged_decode_weighted(): the decode, and every cached token's attention weight
    added up per kv-head (what eviction.evict goes by);
  * paged_decode_diff(): the difference of two softmax maps (differential attention)
    with its per-head norm.

Serving calls: one query token per request, nothing differentiated. They take no
levers. Both run on the HIP library only; there is no CPU path.
"""
from __future__ import annotations

import functools
import struct

import torch

import kv_cache
import sched_abi as abi
import sched_pd

_F32 = torch.float32
WORKSPACE = struct.Struct("@PQ")      # workspace, workspace_bytes


def diff_lambda(q1, k1, q2, k2, init: float) -> torch.Tensor:
    """lam of paged_decode_diff from its learned vectors (each [..., head_dim / 2]):
    exp(q1 . k1) - exp(q2 . k2) + init, in fp32. A model computes it once, when its
    weights are loaded, and expands it to [num_q_heads]."""
    dot = lambda a, b: (a.float() * b.float()).sum(-1)  # noqa: E731
    return torch.exp(dot(q1, k1)) - torch.exp(dot(q2, k2)) + init


def _build(op, q, k_pool, v_pool, block_table, ctx_lens, out, out_dtype, v_layout, page_indptr,
           sm_scale, k_scale, v_scale, flags):
    """The checks both operators share: (what their argument blocks begin with, up to the
    values that differ; the rest of the shared ones; the output tensor)."""
    dt = sched_pd._DT
    qd, kd = dt.get(q.dtype), dt.get(k_pool.dtype)
    if qd is None or qd == abi.FP8_E4M3:
        raise TypeError(f"q must be float32, bfloat16 or float16, got {q.dtype}")
    if kd is None or v_pool.dtype != k_pool.dtype:
        raise TypeError(f"pool dtypes {k_pool.dtype}, {v_pool.dtype}")
    ks, vs = k_pool.stride(), v_pool.stride()
    if len(ks) != 4 or len(vs) != 4:
        raise ValueError("pools must have four dims")
    P, hkv, ps, d = k_pool.shape
    if ks[3] != 1:
        raise ValueError("k_pool dims must be contiguous")
    if v_layout == "tokmajor":
        want, vt, vd = (P, hkv, ps, d), vs[2], vs[3]
    elif v_layout == "dmajor":
        want, vt, vd = (P, hkv, d, ps), vs[3], vs[2]
    else:
        raise ValueError(f"v_layout {v_layout!r}")
    if v_pool.shape != want:
        raise ValueError(f"{v_layout} v_pool must be {want}, got {tuple(v_pool.shape)}")
    if vs[3] != 1:
        raise ValueError("v_pool's last dim must be contiguous")
    R = ctx_lens.numel()
    qs = q.shape
    if len(qs) != 3 or qs[0] != R or qs[2] != d or not q.is_contiguous():
        raise ValueError(f"q must be contiguous [{R}, Hq, {d}], got {tuple(qs)}")
    if out is None:
        out = torch.empty(qs, dtype=out_dtype or q.dtype, device=q.device)
    if out.shape != qs or not out.is_contiguous():
        raise ValueError(f"out must be contiguous {tuple(qs)}, got {tuple(out.shape)}")
    od = dt.get(out.dtype)
    if od is None or od == abi.FP8_E4M3:
        raise TypeError(f"out must be float32, bfloat16 or float16, got {out.dtype}")
    stride, pages, indptr = table_of(R, block_table, page_indptr, ctx_lens)
    ksp = vsp = 0
    if kd == abi.FP8_E4M3:
        kv_cache.check_scales(k_scale, v_scale, P * hkv)
        ksp, vsp = k_scale.data_ptr(), v_scale.data_ptr()
        check_device(k_pool, k_scale=k_scale, v_scale=v_scale)
    dev = k_pool.get_device()
    if dev < 0 or q.get_device() != dev or v_pool.get_device() != dev \
            or block_table.get_device() != dev or ctx_lens.get_device() != dev \
            or out.get_device() != dev or page_indptr is not None:
        check_device(k_pool, q=q, out=out, k_pool=k_pool, v_pool=v_pool, block_table=block_table,
                     ctx_lens=ctx_lens, page_indptr=page_indptr)
    head = (abi.MAPS_ABI_VERSION, op, kd, qd, od, R, qs[1], hkv, d, ps, stride, pages, flags,
            0.0 if sm_scale is None else sm_scale)
    tail = (P, q.data_ptr(), out.data_ptr(), k_pool.data_ptr(), v_pool.data_ptr(), ks[0], ks[1],
            ks[2], vs[0], vs[1], vt, vd, ksp, vsp, block_table.data_ptr(), indptr,
            ctx_lens.data_ptr())
    return head, tail, out


_I32 = torch.int32


def table_of(R, block_table, page_indptr, ctx_lens) -> tuple:
    """Check a page table and lengths; (row stride, pages it reaches, page_indptr's
    address or 0)."""
    if block_table.dtype != _I32 or not block_table.is_contiguous():
        raise ValueError("block_table must be contiguous int32")
    if ctx_lens.dtype != _I32 or not ctx_lens.is_contiguous():
        raise ValueError("ctx_lens must be contiguous int32")
    if page_indptr is None:
        shape = block_table.shape
        if len(shape) != 2 or shape[0] != R:
            raise ValueError(f"block_table must be [{R}, max_pages] without page_indptr")
        return shape[1], shape[1], 0
    if page_indptr.dtype != _I32 or not page_indptr.is_contiguous():
        raise ValueError("page_indptr must be contiguous int32")
    if page_indptr.numel() != R + 1:
        raise ValueError("page_indptr needs num_requests + 1 entries")
    return 0, block_table.numel(), page_indptr.data_ptr()


def check_device(like, **tensors) -> None:
    """Raise ValueError unless every tensor lies on `like`'s GPU."""
    dev = like.device
    if dev.type != "cuda":
        raise ValueError(f"k_pool must be a device tensor (got {dev})")
    for what, t in tensors.items():
        if t is not None and t.device != dev:
            raise ValueError(f"{what} must be a device tensor on {dev} (got {t.device})")


def check_weights(weights, P, hkv, ps, what="weights") -> None:
    """Raise unless `weights` holds one fp32 per (page, kv-head, slot)."""
    if weights.dtype != _F32 or weights.shape != (P, hkv, ps) or weights.stride(2) != 1:
        raise ValueError(f"{what} must be float32 [{P}, {hkv}, {ps}] with contiguous slots, got "
                         f"{weights.dtype} {tuple(weights.shape)}")


def scratch(need: int, workspace, device):
    """A workspace of `need` bytes on the current stream: the caller's, or a new one
    (of the graph's own pool under torch.cuda.graph; a capture without such a pool
    has to bring one that lives as long as its graph)."""
    if workspace is not None:
        if workspace.device != device or not workspace.is_contiguous() \
                or workspace.numel() * workspace.element_size() < need:
            raise ValueError(f"workspace must be contiguous on {device} with {need} bytes")
        return workspace
    ws = torch.empty(need, dtype=torch.uint8, device=device)
    if torch.cuda.is_current_stream_capturing() and not sched_pd._in_private_pool(ws):
        raise RuntimeError("a capture outside torch.cuda.graph needs workspace=: memory taken "
                           "here would go to other tensors while the graph still uses it")
    return ws


def on_device(fn):
    """Run fn with its first tensor's GPU current and, if given, `stream` current there, so
    that allocations and the launch are ordered on it."""
    @functools.wraps(fn)
    def run(*args, stream=None, **kw):
        t = args[0] if args else next((v for v in kw.values() if isinstance(v, torch.Tensor)), None)
        dev = t.get_device() if isinstance(t, torch.Tensor) else -1
        if stream is None and (dev < 0 or dev == torch._C._cuda_getDevice()):
            return fn(*args, **kw)
        with torch.cuda.device(dev):
            if stream is None:
                return fn(*args, **kw)
            with torch.cuda.stream(stream):
                return fn(*args, **kw)
    return run


def _launch(block, workspace, device) -> None:
    """Launch a SchedMapsArgs block but for its last two fields, the workspace."""
    need = abi.entry("sched_decode_maps_workspace_bytes")(block + bytes(16))
    if need < 0:
        raise RuntimeError(f"sched_decode_maps failed: {abi.last_error()}")
    ws = scratch(need, workspace, device)
    rc = abi.entry("sched_decode_maps")(
        block + WORKSPACE.pack(ws.data_ptr(), ws.numel() * ws.element_size()), sched_pd._raw_stream(None))
    if rc != 0:
        raise RuntimeError(f"sched_decode_maps failed ({rc}): {abi.last_error()}")


@on_device
def paged_decode_weighted(q, k_pool, v_pool, block_table, ctx_lens, weights, *, counted=None,
                          decay=1.0, out=None, out_dtype=None, v_layout="dmajor",
                          page_indptr=None, sm_scale=None, k_scale=None, v_scale=None, flags=0,
                          workspace=None) -> torch.Tensor:
    """One decode step (sched_pd.paged_decode's output) that also adds up attention
    weights in place: for token t of request r and kv-head h,

        weights = (t < counted[r] ? decay * weights : 0) + sum of the group's softmax(t)

    at the token's page and slot of `weights`, float32 [P, Hkv, page]. `counted`
    (int32 [R]; None: all): how many of the request's tokens have a weight already;
    later slots are written without being read, so fresh pages need no clearing.
    Slots past the context stay as they are. Pages of one call belong to one
    request each. A request without tokens gives NaN rows.

    `stream`: the stream the call's work goes to (default: the current one).
    `workspace`: scratch of sched_decode_maps_workspace_bytes (default: taken from
    torch's allocator)."""
    head, tail, out = _build(abi.MAPS_WEIGHTED, q, k_pool, v_pool, block_table, ctx_lens, out,
                             out_dtype, v_layout, page_indptr, sm_scale, k_scale, v_scale, flags)
    P, hkv, ps, _ = k_pool.shape
    check_weights(weights, P, hkv, ps)
    cnt = 0
    if counted is not None:
        if counted.dtype != _I32 or not counted.is_contiguous() \
                or counted.numel() != ctx_lens.numel():
            raise ValueError(f"counted must be contiguous int32 [{ctx_lens.numel()}]")
        cnt = counted.data_ptr()
    dev = k_pool.get_device()
    if dev < 0 or weights.get_device() != dev or (cnt and counted.get_device() != dev):
        check_device(k_pool, weights=weights, counted=counted)
    ws = weights.stride()
    _launch(abi.packer(abi.SchedMapsArgs, 2)(*head, decay, 0.0, 0.0, *tail, weights.data_ptr(),
                                             ws[0], ws[1], cnt, 0, 0), workspace, k_pool.device)
    return out


@on_device
def paged_decode_diff(q, k_pool, v_pool, block_table, ctx_lens, lam, *, norm_weight=None, eps=1e-5,
                      out_scale=1.0, out=None, out_dtype=None, v_layout="dmajor",
                      page_indptr=None, sm_scale=None, k_scale=None, v_scale=None, flags=0,
                      workspace=None) -> torch.Tensor:
    """One differential decode step. Rows of q [R, Hq, d] and of k_pool hold two maps of
    d / 2 dims side by side, rows of v_pool d dims:

        o = (softmax(s q1 . K1) - lam softmax(s q2 . K2)) V,  s = sm_scale or (d / 2) ** -0.5
        out = out_scale * norm_weight * o / sqrt(mean(o ** 2) + eps)   (per head)

    lam: float32 [Hq] (diff_lambda() computes it from the learned vectors);
    norm_weight: float32 [d], or None for out = out_scale * o. A PagedKvCache of
    head_dim d holds such a layer as it is. A request without tokens gives NaN rows.
    `stream` and `workspace` as paged_decode_weighted's."""
    head, tail, out = _build(abi.MAPS_DIFF, q, k_pool, v_pool, block_table, ctx_lens, out,
                             out_dtype, v_layout, page_indptr, sm_scale, k_scale, v_scale, flags)
    _, hq, d = q.shape
    for t, n, what in ((lam, hq, "lam"), (norm_weight, d, "norm_weight")):
        if t is not None and (t.dtype != _F32 or not t.is_contiguous() or t.numel() != n):
            raise ValueError(f"{what} must be contiguous float32 [{n}]")
    nw = 0 if norm_weight is None else norm_weight.data_ptr()
    dev = k_pool.get_device()
    if dev < 0 or lam.get_device() != dev or (nw and norm_weight.get_device() != dev):
        check_device(k_pool, lam=lam, norm_weight=norm_weight)
    _launch(abi.packer(abi.SchedMapsArgs, 2)(*head, 0.0, eps, out_scale, *tail, 0, 0, 0, 0,
                                             lam.data_ptr(), nw), workspace, k_pool.device)
    return out


def kernel_kind(q, k_pool, v_pool, block_table, ctx_lens, *, diff=False, v_layout="dmajor",
                flags=0) -> str:
    """'mfma' or 'valu': the kernel that streams the cache for such a call."""
    op = abi.MAPS_DIFF if diff else abi.MAPS_WEIGHTED
    fp8 = k_pool.dtype.itemsize == 1
    n = k_pool.shape[0] * k_pool.shape[1]
    s = torch.empty(n, device=k_pool.device) if fp8 else None
    head, tail, _ = _build(op, q, k_pool, v_pool, block_table, ctx_lens, None, None, v_layout,
                           None, None, s, s, flags)
    kind = abi.entry("sched_decode_maps_kernel_kind")(
        abi.packer(abi.SchedMapsArgs)(*head, 0.0, 0.0, 0.0, *tail, 0, 0, 0, 0, 0, 0, 0, 0))
    if kind < 0:
        raise RuntimeError(abi.last_error())
    return {0: "valu", 1: "mfma"}[kind]
