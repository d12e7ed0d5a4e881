"""Eviction of cached tokens by their accumulated attention weight
(`sched_kv_evict` in include/sched_kv.h): per request and kv-head the heaviest tokens
stay, beside the first and the most recent ones, and move down to the front of
the request's pages, in place. decode_maps.paged_decode_weighted adds the weights
up. Runs on the HIP library only; there is no CPU path.
"""
from __future__ import annotations

import torch

import kv_cache
import sched_abi as abi
import sched_pd
from decode_maps import (WORKSPACE, check_device, check_weights, on_device, scratch,
                         table_of)


@on_device
def evict(k_pool, v_pool, weights, block_table, ctx_lens, keep_lens, *, sink=0, recent=0,
          max_keep=None, weights_out=None, v_layout="dmajor", page_indptr=None, k_scale=None,
          v_scale=None, kept=None, errors=None, workspace=None) -> torch.Tensor:
    """Cut request r from ctx_lens[r] = n tokens to m = min(n, keep_lens[r], max_keep).
    Each kv-head keeps the first `sink` and the last `recent` tokens (the recent ones
    first where m holds fewer than both) and, of the others, those with the largest
    weights (float32 [P, Hkv, page]); of equal weights the lower slot, NaN below every
    number. Kept tokens keep their order and move to slots 0..m-1: keys, values and weights
    (to `weights_out`, default in place). Slots from m on are left as they are, a
    request with m == n altogether.

    Returns int32 [R, Hkv, max_keep]: the slots the kept tokens had, then -1 (`kept`
    gives the tensor). max_keep (host; default the table's reach) bounds m and sizes that
    output. The caller's lengths become torch.minimum(ctx_lens, keep_lens); keys carry
    their rotation along, so later tokens' positions go on from the uncut length.

    fp8 caches: a page's scale becomes the largest of its tokens' old ones and codes
    of other scales are encoded anew. A request whose table is too short or names a page
    outside the pool is left alone, its kept rows -1, counted once per kv-head in
    `errors` (int32 [1], optional). Pages of one call belong to one request each.
    `stream`: where the work goes (default: the current stream)."""
    kd = sched_pd._DT.get(k_pool.dtype)
    if kd is None or v_pool.dtype != k_pool.dtype:
        raise TypeError(f"pool dtypes {k_pool.dtype}, {v_pool.dtype}")
    ks, vs = k_pool.stride(), v_pool.stride()
    if len(ks) != 4 or len(vs) != 4:
        raise ValueError("pools must have four dims")
    P, hkv, ps, d = k_pool.shape
    if v_layout not in ("tokmajor", "dmajor"):
        raise ValueError(f"v_layout {v_layout!r}")
    tok = v_layout == "tokmajor"
    want = (P, hkv, ps, d) if tok else (P, hkv, d, ps)
    if v_pool.shape != want:
        raise ValueError(f"{v_layout} v_pool must be {want}, got {tuple(v_pool.shape)}")
    if ks[3] != 1 or vs[3] != 1:
        raise ValueError("the pools' last dims must be contiguous")
    check_weights(weights, P, hkv, ps)
    ws = weights.stride()
    if weights_out is None:
        weights_out = weights
    else:
        check_weights(weights_out, P, hkv, ps, "weights_out")
        if weights_out.stride() != ws:
            raise ValueError("weights_out must have the strides of weights")
    if sink < 0 or recent < 0:
        raise ValueError(f"sink {sink} and recent {recent} must not be negative")
    R = ctx_lens.numel()
    if keep_lens.dtype != torch.int32 or not keep_lens.is_contiguous() or keep_lens.numel() != R:
        raise ValueError(f"keep_lens must be contiguous int32 [{R}]")
    stride, pages, indptr = table_of(R, block_table, page_indptr, ctx_lens)
    max_keep = pages * ps if max_keep is None else int(max_keep)
    if not 0 <= max_keep < 1 << 31:
        raise ValueError(f"max_keep {max_keep}")
    sink, recent = min(int(sink), (1 << 31) - 1), min(int(recent), (1 << 31) - 1)
    if kept is None:
        kept = torch.empty(R, hkv, max_keep, dtype=torch.int32, device=k_pool.device)
    elif kept.dtype != torch.int32 or kept.shape != (R, hkv, max_keep) or not kept.is_contiguous():
        raise ValueError(f"kept must be contiguous int32 [{R}, {hkv}, {max_keep}]")
    ksp = vsp = err = 0
    if kd == abi.FP8_E4M3:
        kv_cache.check_scales(k_scale, v_scale, P * hkv)
        ksp, vsp = k_scale.data_ptr(), v_scale.data_ptr()
        check_device(k_pool, k_scale=k_scale, v_scale=v_scale)
    if errors is not None:
        if errors.dtype not in (torch.int32, torch.uint32) or errors.numel() < 1:
            raise ValueError("errors must be a 32-bit integer tensor")
        err = errors.data_ptr()
    dev = k_pool.get_device()
    if dev < 0 or v_pool.get_device() != dev or weights.get_device() != dev \
            or weights_out.get_device() != dev or block_table.get_device() != dev \
            or ctx_lens.get_device() != dev or keep_lens.get_device() != dev \
            or kept.get_device() != dev or indptr or err:
        check_device(k_pool, k_pool=k_pool, v_pool=v_pool, weights=weights,
                     weights_out=weights_out, block_table=block_table, page_indptr=page_indptr,
                     ctx_lens=ctx_lens, keep_lens=keep_lens, kept=kept, errors=errors)
    block = abi.packer(abi.SchedEvictArgs, 2)(
        abi.EVICT_ABI_VERSION, kd, R, hkv, d, ps, stride, pages, max_keep, sink, recent, 0, P,
        k_pool.data_ptr(), v_pool.data_ptr(), ks[0], ks[1], ks[2], vs[0], vs[1],
        vs[2] if tok else vs[3], vs[3] if tok else vs[2], ksp, vsp, weights.data_ptr(),
        weights_out.data_ptr(), ws[0], ws[1], block_table.data_ptr(), indptr, ctx_lens.data_ptr(),
        keep_lens.data_ptr(), kept.data_ptr(), err)
    need = abi.entry("sched_kv_evict_workspace_bytes")(block + bytes(16))
    if need < 0:
        raise RuntimeError(abi.last_error())
    at = size = 0
    if need:
        scr = scratch(need, workspace, k_pool.device)
        at, size = scr.data_ptr(), scr.numel() * scr.element_size()
    if abi.entry("sched_kv_evict")(block + WORKSPACE.pack(at, size), sched_pd._raw_stream(None)) != 0:
        raise RuntimeError(abi.last_error())
    return kept
