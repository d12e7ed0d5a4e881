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

import ctypes

import torch

import kv_cache
import sched_abi as abi
import sched_pd

_F32 = torch.float32


def diff_lambda(q1, k1, q2, k2, init: float) -> torch.Tensor:
    """lam of paged_decode_diff from its learned vectors (each [..., head_dim / 2]):
    exp(q1 . k1) - exp(q2 . k2) + init, in fp32. A model computes it once, when its
    weights are loaded, and expands it to [num_q_heads]."""
    dot = lambda a, b: (a.float() * b.float()).sum(-1)  # noqa: E731
    return torch.exp(dot(q1, k1)) - torch.exp(dot(q2, k2)) + init


def _build(op, q, k_pool, v_pool, block_table, ctx_lens, out, out_dtype, v_layout, page_indptr,
           sm_scale, k_scale, v_scale, flags):
    """A SchedMapsArgs of what both operators share, and the output tensor."""
    dt = sched_pd._DT
    if q.dtype not in dt or q.dtype.itemsize == 1:
        raise TypeError(f"q must be float32, bfloat16 or float16, got {q.dtype}")
    if k_pool.dtype not in dt or v_pool.dtype != k_pool.dtype:
        raise TypeError(f"pool dtypes {k_pool.dtype}, {v_pool.dtype}")
    if k_pool.dim() != 4 or v_pool.dim() != 4:
        raise ValueError("pools must have four dims")
    P, hkv, ps, d = k_pool.shape
    ks, vs = k_pool.stride(), v_pool.stride()
    if ks[3] != 1:
        raise ValueError("k_pool dims must be contiguous")
    if v_layout == "tokmajor":
        want, inner, vt, vd = (P, hkv, ps, d), vs[3], vs[2], vs[3]
    elif v_layout == "dmajor":
        want, inner, vt, vd = (P, hkv, d, ps), vs[3], vs[3], vs[2]
    else:
        raise ValueError(f"v_layout {v_layout!r}")
    if tuple(v_pool.shape) != want:
        raise ValueError(f"{v_layout} v_pool must be {want}, got {tuple(v_pool.shape)}")
    if inner != 1:
        raise ValueError("v_pool's last dim must be contiguous")
    R = ctx_lens.numel()
    if q.dim() != 3 or q.shape[0] != R or q.shape[2] != d or not q.is_contiguous():
        raise ValueError(f"q must be contiguous [{R}, Hq, {d}], got {tuple(q.shape)}")
    if out is None:
        out = torch.empty(q.shape, dtype=out_dtype or q.dtype, device=q.device)
    if out.shape != q.shape or not out.is_contiguous():
        raise ValueError(f"out must be contiguous {tuple(q.shape)}, got {tuple(out.shape)}")
    if out.dtype not in dt or out.dtype.itemsize == 1:
        raise TypeError(f"out must be float32, bfloat16 or float16, got {out.dtype}")
    a = abi.SchedMapsArgs(
        abi_version=abi.MAPS_ABI_VERSION, op=op, kv_dtype=dt[k_pool.dtype], q_dtype=dt[q.dtype],
        o_dtype=dt[out.dtype], num_requests=R, num_q_heads=q.shape[1], num_kv_heads=hkv,
        head_dim=d, page_size=ps, flags=flags, sm_scale=0.0 if sm_scale is None else sm_scale,
        num_pages=P, q=q.data_ptr(), out=out.data_ptr(), k_pool=k_pool.data_ptr(),
        v_pool=v_pool.data_ptr(), k_page_stride=ks[0], k_head_stride=ks[1], k_tok_stride=ks[2],
        v_page_stride=vs[0], v_head_stride=vs[1], v_tok_stride=vt, v_dim_stride=vd,
        block_table=block_table.data_ptr(), ctx_lens=ctx_lens.data_ptr())
    check_table(a, R, block_table, page_indptr, ctx_lens)
    if a.kv_dtype == abi.FP8_E4M3:
        kv_cache.check_scales(k_scale, v_scale, P * hkv)
        a.k_scale, a.v_scale = k_scale.data_ptr(), v_scale.data_ptr()
        check_device(k_pool, k_scale=k_scale, v_scale=v_scale)
    check_device(k_pool, q=q, out=out, k_pool=k_pool, v_pool=v_pool, block_table=block_table,
                 ctx_lens=ctx_lens, page_indptr=page_indptr)
    return a, out


def check_table(a, R, block_table, page_indptr, ctx_lens) -> None:
    """Check a page table and lengths and fill in a's width and stride."""
    for t, what in ((block_table, "block_table"), (ctx_lens, "ctx_lens"),
                    (page_indptr, "page_indptr")):
        if t is not None and (t.dtype != torch.int32 or not t.is_contiguous()):
            raise ValueError(f"{what} must be contiguous int32")
    if page_indptr is None:
        if block_table.dim() != 2 or block_table.shape[0] != R:
            raise ValueError(f"block_table must be [{R}, max_pages] without page_indptr")
        a.bt_stride = a.max_pages = block_table.shape[1]
    else:
        if page_indptr.numel() != R + 1:
            raise ValueError("page_indptr needs num_requests + 1 entries")
        a.max_pages = block_table.numel()
        a.page_indptr = page_indptr.data_ptr()


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
    if weights.dtype != _F32 or tuple(weights.shape) != (P, hkv, ps) or weights.stride(2) != 1:
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
    """Run fn(pool-like third tensor ...) with that tensor's GPU current and, if given,
    `stream` current there, so that allocations and the launch are ordered on it."""
    import functools

    @functools.wraps(fn)
    def run(*args, stream=None, **kw):
        t = args[1] if len(args) > 1 else None
        other = isinstance(t, torch.Tensor) and t.is_cuda \
            and t.device.index != torch._C._cuda_getDevice()
        if stream is None and not other:
            return fn(*args, **kw)
        with torch.cuda.device(t.device if isinstance(t, torch.Tensor) and t.is_cuda else None):
            if stream is None:
                return fn(*args, **kw)
            with torch.cuda.stream(stream):
                return fn(*args, **kw)
    return run


def _launch(a, workspace, device) -> None:
    lib = abi.load_library()
    need = lib.sched_decode_maps_workspace_bytes(ctypes.byref(a))
    if need < 0:
        raise RuntimeError(f"sched_decode_maps failed: {abi.last_error()}")
    ws = scratch(need, workspace, device)
    a.workspace, a.workspace_bytes = ws.data_ptr(), ws.numel() * ws.element_size()
    rc = lib.sched_decode_maps(ctypes.byref(a), sched_pd._raw_stream(None))
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
    a, out = _build(abi.MAPS_WEIGHTED, q, k_pool, v_pool, block_table, ctx_lens, out, out_dtype,
                    v_layout, page_indptr, sm_scale, k_scale, v_scale, flags)
    check_weights(weights, a.num_pages, a.num_kv_heads, a.page_size)
    a.decay = decay
    a.weights = weights.data_ptr()
    a.w_page_stride, a.w_head_stride = weights.stride(0), weights.stride(1)
    if counted is not None:
        if counted.dtype != torch.int32 or not counted.is_contiguous() \
                or counted.numel() != a.num_requests:
            raise ValueError(f"counted must be contiguous int32 [{a.num_requests}]")
        a.counted = counted.data_ptr()
    check_device(k_pool, weights=weights, counted=counted)
    _launch(a, workspace, k_pool.device)
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
    a, out = _build(abi.MAPS_DIFF, q, k_pool, v_pool, block_table, ctx_lens, out, out_dtype,
                    v_layout, page_indptr, sm_scale, k_scale, v_scale, flags)
    for t, n, what in ((lam, a.num_q_heads, "lam"), (norm_weight, a.head_dim, "norm_weight")):
        if t is not None and (t.dtype != _F32 or not t.is_contiguous() or t.numel() != n):
            raise ValueError(f"{what} must be contiguous float32 [{n}]")
    check_device(k_pool, lam=lam, norm_weight=norm_weight)
    a.eps, a.out_scale = eps, out_scale
    a.lam = lam.data_ptr()
    if norm_weight is not None:
        a.norm_weight = norm_weight.data_ptr()
    _launch(a, workspace, k_pool.device)
    return out


def kernel_kind(q, k_pool, v_pool, block_table, ctx_lens, *, diff=False, v_layout="dmajor",
                flags=0) -> str:
    """'mfma' or 'valu': the kernel that streams the cache for such a call."""
    op = abi.MAPS_DIFF if diff else abi.MAPS_WEIGHTED
    fp8 = k_pool.dtype.itemsize == 1
    n = k_pool.shape[0] * k_pool.shape[1]
    s = torch.empty(n, device=k_pool.device) if fp8 else None
    a, _ = _build(op, q, k_pool, v_pool, block_table, ctx_lens, None, None, v_layout, None, None,
                  s, s, flags)
    kind = abi.load_library().sched_decode_maps_kernel_kind(ctypes.byref(a))
    if kind < 0:
        raise RuntimeError(abi.last_error())
    return {0: "valu", 1: "mfma"}[kind]
