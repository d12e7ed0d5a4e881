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

import torch

import kv_cache
import sched_abi as abi
import sched_pd
from decode_maps import check_device, on_device, table_of

_DT = {torch.float32: abi.F32, torch.bfloat16: abi.BF16, torch.float16: abi.F16}


def cos_sin_table(max_pos: int, rot_dim: int, base: float = 10000.0, device="cuda"):
    """The fp32 table [max_pos, rot_dim] of cosines | sines of p * base ** (-2j /
    rot_dim), computed in 64 bits (an fp32 angle of a far position has lost its
    fraction of a turn)."""
    half = rot_dim // 2
    inv = float(base) ** (-torch.arange(half, dtype=torch.float64) / half)
    ang = torch.arange(max_pos, dtype=torch.float64)[:, None] * inv
    return torch.cat([ang.cos(), ang.sin()], 1).float().to(device)


_ROWS = (0,) * 18        # the block's cache fields without a cache


def _call(q, k, v, positions, cos_sin, q_weight, k_weight, eps, interleaved, q_out, k_out, errors,
          cache=_ROWS):
    """Check the rows and the rotation, launch, and return q_out. `cache`: the block's
    last fields; without one the key rows go to k_out."""
    dt = _DT.get(q.dtype)
    if dt is None or k.dtype != q.dtype or (v is not None and v.dtype != q.dtype):
        raise TypeError(f"rows must all be float32, bfloat16 or float16, got {q.dtype}, {k.dtype}"
                        f"{'' if v is None else f', {v.dtype}'}")
    qsh, ksh = q.shape, k.shape
    if len(qsh) != 3 or len(ksh) != 3 or qsh[0] != ksh[0] or qsh[2] != ksh[2]:
        raise ValueError(f"rows must be q [T, Hq, d] and k [T, Hkv, d], got {tuple(qsh)} and "
                         f"{tuple(ksh)}")
    T, hq, d = qsh
    qs, ks = q.stride(), k.stride()
    vp, vs = 0, (0, 0, 1)
    if v is not None:
        if v.shape != ksh:
            raise ValueError(f"v must be {tuple(ksh)}, got {tuple(v.shape)}")
        vp, vs = v.data_ptr(), v.stride()
    if q_out is None:
        q_out = torch.empty(qsh, dtype=q.dtype, device=q.device)
    elif q_out.shape != qsh or q_out.dtype != q.dtype:
        raise ValueError(f"q_out must be {q.dtype} {tuple(qsh)}")
    qo = q_out.stride()
    if qs[2] != 1 or ks[2] != 1 or qo[2] != 1 or vs[2] != 1:
        raise ValueError("row dims must be contiguous")
    i64 = positions.dtype == torch.int64
    if not (i64 or positions.dtype == torch.int32) or positions.numel() != T \
            or not positions.is_contiguous():
        raise ValueError(f"positions must be contiguous int32 or int64 [{T}]")
    cs = cos_sin.stride()
    if cos_sin.dtype != torch.float32 or len(cs) != 2 or cs[1] != 1:
        raise ValueError("cos_sin must be float32 [max_pos, rot_dim] with contiguous rows")
    qw = kw = wd = 0
    if q_weight is not None:
        qw, wd = _weight(q_weight, d, "q_weight")
    if k_weight is not None:
        kw, kd = _weight(k_weight, d, "k_weight")
        if qw and kd != wd:
            raise TypeError(f"weights of two types: {q_weight.dtype}, {k_weight.dtype}")
        wd = kd
    err = 0
    if errors is not None:
        if errors.dtype not in (torch.int32, torch.uint32) or errors.numel() < 1:
            raise ValueError("errors must be a 32-bit integer tensor")
        err = errors.data_ptr()
    dev = k.get_device()
    if dev < 0 or q.get_device() != dev or positions.get_device() != dev \
            or cos_sin.get_device() != dev or q_out.get_device() != dev \
            or (vp and v.get_device() != dev) or (qw and q_weight.get_device() != dev) \
            or (kw and k_weight.get_device() != dev) or err:
        check_device(k, q=q, v=v, q_out=q_out, positions=positions, cos_sin=cos_sin,
                     q_weight=q_weight, k_weight=k_weight, errors=errors)
    kop, ko = (0, (0, 0)) if k_out is None else (k_out.data_ptr(), k_out.stride())
    block = abi.packer(abi.SchedRotaryArgs)(
        abi.ROTARY_ABI_VERSION, dt, wd, T, hq, ksh[1], d, cos_sin.shape[1],
        1 if interleaved else 0, i64, cos_sin.shape[0], eps, q.data_ptr(), k.data_ptr(), vp, qs[0],
        qs[1], ks[0], ks[1], vs[0], vs[1], q_out.data_ptr(), kop, qo[0], qo[1], ko[0], ko[1], qw,
        kw, positions.data_ptr(), cos_sin.data_ptr(), cs[0], err, *cache)
    if abi.entry("sched_qk_norm_rope")(block, sched_pd._raw_stream(None)) != 0:
        raise RuntimeError(abi.last_error())
    return q_out


def _weight(w, d, what) -> tuple:
    """(address, type) of a norm's weight."""
    dt = _DT.get(w.dtype)
    if dt is None or w.numel() != d or not w.is_contiguous():
        raise ValueError(f"{what} must be contiguous [{d}]")
    return w.data_ptr(), dt


@on_device
def qk_norm_rope(q, k, positions, cos_sin, *, q_weight=None, k_weight=None, eps=1e-6,
                 interleaved=False, q_out=None, k_out=None, errors=None):
    """Norm and rotate q [T, Hq, d] and k [T, Hkv, d] (views of one projection's output
    will do: dims contiguous, any other strides); returns (q_out, k_out), new tensors
    unless given. q_out / k_out may be q / k (in place), else they must not overlap
    the inputs. A token whose position lies outside cos_sin is not written and
    counted in `errors` (int32 [1], optional). `stream`: where the work goes
    (default: the current stream)."""
    if k_out is None:
        k_out = torch.empty(k.shape, dtype=k.dtype, device=k.device)
    elif k_out.shape != k.shape or k_out.dtype != k.dtype or k_out.stride(2) != 1 \
            or k_out.device != k.device:
        raise ValueError(f"k_out must be {k.dtype} {tuple(k.shape)} on {k.device}, dims contiguous")
    return _call(q, k, None, positions, cos_sin, q_weight, k_weight, eps, interleaved, q_out,
                 k_out, errors), k_out


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

    One launch into a cache of the rows' type (two where many tokens go to a d-major V);
    other caches (fp8, another type) take qk_norm_rope() and kv_cache.append(), the keys
    rounded to the rows' type in between, and that writer's zeros behind the last value of
    a d-major V. `errors` counts tokens with a position outside cos_sin and (token,
    kv-head) pairs that have no place in the cache."""
    if v_layout not in ("tokmajor", "dmajor"):
        raise ValueError(f"v_layout must be 'dmajor' or 'tokmajor', got {v_layout!r}")
    if k_pool.dtype != q.dtype or k_pool.dim() != 4:
        q_out, k_rot = qk_norm_rope(q, k, positions, cos_sin, q_weight=q_weight, k_weight=k_weight,
                                    eps=eps, interleaved=interleaved, q_out=q_out, errors=errors)
        kv_cache.append(k_rot, v.contiguous(), append_indptr, ctx_lens, k_pool, v_pool,
                        block_table, page_indptr=page_indptr, v_layout=v_layout, k_scale=k_scale,
                        v_scale=v_scale, max_append=max_append, errors=errors)
        return q_out
    P, hkv, ps, d = k_pool.shape
    dm = v_layout == "dmajor"
    if v_pool.dtype != k_pool.dtype or v_pool.shape != ((P, hkv, d, ps) if dm else k_pool.shape):
        raise ValueError(f"{v_layout} v_pool must be {k_pool.dtype} "
                         f"{(P, hkv, d, ps) if dm else tuple(k_pool.shape)}, got "
                         f"{v_pool.dtype} {tuple(v_pool.shape)}")
    if k.shape[1:] != (hkv, d):
        raise ValueError(f"k {tuple(k.shape)} vs pool heads/dims ({hkv}, {d})")
    ks, vs = k_pool.stride(), v_pool.stride()
    if ks[3] != 1 or vs[3] != 1:
        raise ValueError("pool dims must be contiguous (d-major V: tokens)")
    R = ctx_lens.numel()
    stride, _, indptr = table_of(R, block_table, page_indptr, ctx_lens)
    if append_indptr.dtype != torch.int32 or not append_indptr.is_contiguous() \
            or append_indptr.numel() != R + 1:
        raise ValueError("append_indptr must be contiguous int32 [num_requests + 1]")
    dev = k.get_device()
    if dev < 0 or k_pool.get_device() != dev or v_pool.get_device() != dev \
            or append_indptr.get_device() != dev or ctx_lens.get_device() != dev \
            or block_table.get_device() != dev or indptr:
        check_device(k, append_indptr=append_indptr, ctx_lens=ctx_lens, k_pool=k_pool,
                     v_pool=v_pool, block_table=block_table, page_indptr=page_indptr)
    return _call(q, k, v, positions, cos_sin, q_weight, k_weight, eps, interleaved, q_out, None,
                 errors, (R, ps, stride, int(max_append), P, append_indptr.data_ptr(),
                          ctx_lens.data_ptr(), block_table.data_ptr(), indptr, k_pool.data_ptr(),
                          v_pool.data_ptr(), ks[0], ks[1], ks[2], vs[0], vs[1],
                          1 if dm else vs[2], vs[2] if dm else 1))
