"""Norm of queries and keys per head with the position rotation in the same pass
(`sched_qk_norm_rope` in include/sched_kv.h): into buffers (qk_norm_rope), or the
keys and values straight into a paged cache (append_rotated), which leaves the
queries ready for the decode.

Per head of d dims, in fp32 and rounded once at the end:

    x' = x * weight / sqrt(mean(x ** 2) + eps)          (weight None: x' = x)
    (y_a, y_b) = (x'_a c - x'_b s, x'_b c + x'_a s)

for the pairs (a, b) = (j, j + rot / 2), or (2j, 2j + 1) with interleaved=True, j < rot
/ 2; c and s are cos_sin[position][j] and cos_sin[position][rot / 2 + j]. Dims past
rot pass through. Runs on the HIP library only; there is no CPU path.
"""
from __future__ import annotations

import ctypes

import torch

import kv_cache
import sched_abi as abi
import sched_pd
from decode_maps import check_device, check_table, on_device

_DT = {torch.float32: abi.F32, torch.bfloat16: abi.BF16, torch.float16: abi.F16}


def cos_sin_table(max_pos: int, rot_dim: int, base: float = 10000.0, device="cuda"):
    """The fp32 table [max_pos, rot_dim] of cosines | sines of p * base ** (-2j /
    rot_dim), computed in 64 bits (an fp32 angle of a far position has lost its
    fraction of a turn)."""
    half = rot_dim // 2
    inv = float(base) ** (-torch.arange(half, dtype=torch.float64) / half)
    ang = torch.arange(max_pos, dtype=torch.float64)[:, None] * inv
    return torch.cat([ang.cos(), ang.sin()], 1).float().to(device)


def _build(q, k, v, positions, cos_sin, q_weight, k_weight, eps, interleaved, q_out, errors):
    """A SchedRotaryArgs of the rows and the rotation, and the query output."""
    if q.dtype not in _DT or k.dtype != q.dtype or (v is not None and v.dtype != q.dtype):
        raise TypeError(f"rows must all be float32, bfloat16 or float16, got {q.dtype}, {k.dtype}"
                        f"{'' if v is None else f', {v.dtype}'}")
    if q.dim() != 3 or k.dim() != 3 or q.shape[0] != k.shape[0] or q.shape[2] != k.shape[2]:
        raise ValueError(f"rows must be q [T, Hq, d] and k [T, Hkv, d], got {tuple(q.shape)} and "
                         f"{tuple(k.shape)}")
    if v is not None and v.shape != k.shape:
        raise ValueError(f"v must be {tuple(k.shape)}, got {tuple(v.shape)}")
    T, hq, d = q.shape
    if q_out is None:
        q_out = torch.empty(q.shape, dtype=q.dtype, device=q.device)
    elif q_out.shape != q.shape or q_out.dtype != q.dtype:
        raise ValueError(f"q_out must be {q.dtype} {tuple(q.shape)}")
    qs, ks, qo = q.stride(), k.stride(), q_out.stride()
    if qs[2] != 1 or ks[2] != 1 or qo[2] != 1 or (v is not None and v.stride(2) != 1):
        raise ValueError("row dims must be contiguous")
    if positions.dtype not in (torch.int32, torch.int64) or positions.numel() != T \
            or not positions.is_contiguous():
        raise ValueError(f"positions must be contiguous int32 or int64 [{T}]")
    if cos_sin.dtype != torch.float32 or cos_sin.dim() != 2 or cos_sin.stride(1) != 1:
        raise ValueError("cos_sin must be float32 [max_pos, rot_dim] with contiguous rows")
    a = abi.SchedRotaryArgs(
        abi_version=abi.ROTARY_ABI_VERSION, dtype=_DT[q.dtype], num_tokens=T, num_q_heads=hq,
        num_kv_heads=k.shape[1], head_dim=d, rot_dim=cos_sin.shape[1],
        interleaved=1 if interleaved else 0, pos_i64=positions.dtype == torch.int64,
        max_pos=cos_sin.shape[0], eps=eps, q=q.data_ptr(), k=k.data_ptr(), q_tok_stride=qs[0],
        q_head_stride=qs[1], k_tok_stride=ks[0], k_head_stride=ks[1], q_out=q_out.data_ptr(),
        qo_tok_stride=qo[0], qo_head_stride=qo[1], positions=positions.data_ptr(),
        cos_sin=cos_sin.data_ptr(), cs_stride=cos_sin.stride(0))
    for w, what in ((q_weight, "q_weight"), (k_weight, "k_weight")):
        if w is not None and (w.dtype not in _DT or w.numel() != d or not w.is_contiguous()):
            raise ValueError(f"{what} must be contiguous [{d}]")
    if q_weight is not None and k_weight is not None and q_weight.dtype != k_weight.dtype:
        raise TypeError(f"weights of two types: {q_weight.dtype}, {k_weight.dtype}")
    w = q_weight if q_weight is not None else k_weight
    a.w_dtype = abi.F32 if w is None else _DT[w.dtype]
    if q_weight is not None:
        a.q_weight = q_weight.data_ptr()
    if k_weight is not None:
        a.k_weight = k_weight.data_ptr()
    if errors is not None:
        if errors.dtype not in (torch.int32, torch.uint32) or errors.numel() < 1:
            raise ValueError("errors must be a 32-bit integer tensor")
        a.errors = errors.data_ptr()
    check_device(k, q=q, v=v, q_out=q_out, positions=positions, cos_sin=cos_sin,
                 q_weight=q_weight, k_weight=k_weight, errors=errors)
    return a, q_out


def _launch(a) -> None:
    if abi.load_library().sched_qk_norm_rope(ctypes.byref(a), sched_pd._raw_stream(None)) != 0:
        raise RuntimeError(abi.last_error())


@on_device
def qk_norm_rope(q, k, positions, cos_sin, *, q_weight=None, k_weight=None, eps=1e-6,
                 interleaved=False, q_out=None, k_out=None, errors=None):
    """Norm and rotate q [T, Hq, d] and k [T, Hkv, d] (views of one projection's output
    will do: dims contiguous, any other strides); returns (q_out, k_out), new tensors
    unless given. q_out / k_out may be q / k (in place), else they must not overlap
    the inputs. A token whose position lies outside cos_sin is not written and
    counted in `errors` (int32 [1], optional). `stream`: where the work goes
    (default: the current stream)."""
    a, q_out = _build(q, k, None, positions, cos_sin, q_weight, k_weight, eps, interleaved, q_out,
                      errors)
    if k_out is None:
        k_out = torch.empty(k.shape, dtype=k.dtype, device=k.device)
    elif k_out.shape != k.shape or k_out.dtype != k.dtype or k_out.stride(2) != 1 \
            or k_out.device != k.device:
        raise ValueError(f"k_out must be {k.dtype} {tuple(k.shape)} on {k.device}, dims contiguous")
    a.k_out = k_out.data_ptr()
    a.ko_tok_stride, a.ko_head_stride = k_out.stride(0), k_out.stride(1)
    _launch(a)
    return q_out, k_out


@on_device
def append_rotated(q, k, v, positions, cos_sin, append_indptr, ctx_lens, k_pool, v_pool,
                   block_table, *, q_weight=None, k_weight=None, eps=1e-6, interleaved=False,
                   page_indptr=None, v_layout="dmajor", k_scale=None, v_scale=None, max_append=0,
                   q_out=None, errors=None) -> torch.Tensor:
    """qk_norm_rope() with the key and value rows appended to the cache: the rotated
    queries (returned), and what kv_cache.append() writes for the rotated keys and v.
    Request r's rows append_indptr[r] .. append_indptr[r+1]-1 go to positions ctx_lens[r] - n_r ..
    ctx_lens[r]-1 of its pages (ctx_lens counts tokens after the append; `positions` are
    the rotation's and need not follow them: after an eviction they do not).

    One launch into a cache of the rows' type with token-major V; other caches (fp8,
    d-major V, another type) take qk_norm_rope() and kv_cache.append(), the keys rounded to
    the rows' type in between. `errors` counts tokens with a position outside cos_sin
    and (token, kv-head) pairs that have no place in the cache."""
    if k_pool.dtype != q.dtype or v_layout != "tokmajor" or k_pool.dim() != 4:
        if errors is not None and errors.dtype not in (torch.int32, torch.uint32):
            raise ValueError("errors must be a 32-bit integer tensor")
        a = kv_cache.build_append_args(
            k, v, append_indptr, ctx_lens, k_pool, v_pool, block_table, page_indptr=page_indptr,
            v_layout=v_layout, k_scale=k_scale, v_scale=v_scale, max_append=max_append,
            errors=errors) if k.stride() == v.stride() else None
        q_out, k_rot = qk_norm_rope(q, k, positions, cos_sin, q_weight=q_weight, k_weight=k_weight,
                                    eps=eps, interleaved=interleaved, q_out=q_out, errors=errors)
        del a
        kv_cache.append(k_rot, v.contiguous(), append_indptr, ctx_lens, k_pool, v_pool,
                        block_table, page_indptr=page_indptr, v_layout=v_layout, k_scale=k_scale,
                        v_scale=v_scale, max_append=max_append, errors=errors)
        return q_out
    P, hkv, ps, d = k_pool.shape
    if v_pool.dtype != k_pool.dtype or v_pool.shape != k_pool.shape:
        raise ValueError(f"token-major v_pool must be {k_pool.dtype} {tuple(k_pool.shape)}, got "
                         f"{v_pool.dtype} {tuple(v_pool.shape)}")
    if tuple(k.shape[1:]) != (hkv, d):
        raise ValueError(f"k {tuple(k.shape)} vs pool heads/dims ({hkv}, {d})")
    ks, vs = k_pool.stride(), v_pool.stride()
    if ks[3] != 1 or vs[3] != 1:
        raise ValueError("pool dims must be contiguous")
    a, q_out = _build(q, k, v, positions, cos_sin, q_weight, k_weight, eps, interleaved, q_out,
                      errors)
    R = ctx_lens.numel()
    check_table(a, R, block_table, page_indptr, ctx_lens)
    if append_indptr.dtype != torch.int32 or not append_indptr.is_contiguous() \
            or append_indptr.numel() != R + 1:
        raise ValueError("append_indptr must be contiguous int32 [num_requests + 1]")
    check_device(k, append_indptr=append_indptr, ctx_lens=ctx_lens, k_pool=k_pool, v_pool=v_pool,
                 block_table=block_table, page_indptr=page_indptr)
    a.v = v.data_ptr()
    a.v_tok_stride, a.v_head_stride = v.stride(0), v.stride(1)
    a.num_requests, a.page_size, a.max_append, a.num_pages = R, ps, int(max_append), P
    a.append_indptr, a.ctx_lens = append_indptr.data_ptr(), ctx_lens.data_ptr()
    a.block_table = block_table.data_ptr()
    a.k_pool, a.v_pool = k_pool.data_ptr(), v_pool.data_ptr()
    a.kp_page_stride, a.kp_head_stride, a.kp_tok_stride = ks[:3]
    a.vp_page_stride, a.vp_head_stride, a.vp_tok_stride = vs[:3]
    _launch(a)
    return q_out
