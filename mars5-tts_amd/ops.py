"""Tensor-level wrappers over the C ABI.  torch is plumbing here: device memory
(``data_ptr``), streams and shapes.  No arithmetic happens in this file; every function
enqueues exactly one HIP kernel on ``stream`` (default: torch's current stream)."""
from __future__ import annotations

import ctypes as C
from typing import Optional

import threading

import torch

from . import _lib as L
from ._lib import check, lib

DT_CODE = {torch.float32: L.F32, torch.float16: L.F16, torch.bfloat16: L.BF16}
CODE_DT = {v: k for k, v in DT_CODE.items()}

# How the fp32 engines multiply (process-wide; read when a launch is ENQUEUED, so a captured graph keeps the mode it was
# captured with): "exact" = v_mfma_f32_16x16x4_f32, bitwise an fmaf chain -- the reference instrument; "f16x3" = the same fp32
# operands split into two f16 halves on the fly and three f16 MFMAs per product (csrc/gemm.hip, M5_F32X3): fp32-grade results
# (operand error 2^-22) at several times the rate -- the fast parity-grade mode.  Set with set_f32_products().
_F32_PRODUCTS = "exact"


def set_f32_products(mode: str) -> str:
    """Select the fp32 engines' GEMM arithmetic ("exact" | "f16x3"); returns the previous mode."""
    global _F32_PRODUCTS
    assert mode in ("exact", "f16x3"), mode
    prev, _F32_PRODUCTS = _F32_PRODUCTS, mode
    return prev


def f32_products() -> str:
    return _F32_PRODUCTS


def _gemm_code(dt: torch.dtype) -> int:
    return L.F32X3 if (dt == torch.float32 and _F32_PRODUCTS == "f16x3") else DT_CODE[dt]
DT_NAME = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}


def _p(t: Optional[torch.Tensor]) -> Optional[int]:
    if t is None:
        return None
    assert t.is_cuda, "libmars5_hip operates on device memory only"
    return t.data_ptr()


def cur_stream() -> int:
    return torch.cuda.current_stream().cuda_stream


def _s(stream: Optional[int]) -> int:
    return cur_stream() if stream is None else stream


def gemm(a: torch.Tensor, w: torch.Tensor, out: Optional[torch.Tensor], epi: int, bias: Optional[torch.Tensor] = None,
         scatter: Optional[L.QkvScatter] = None, M: Optional[int] = None, ldc: Optional[int] = None,
         batch: int = 1, sA: int = 0, sW: int = 0, sC: int = 0, sBias: int = 0, stream: Optional[int] = None) -> None:
    """out = a[M,K] @ w[N,K]^T (+bias) with fused epilogue `epi`.  a/w: 2-D, K contiguous."""
    assert a.dtype == w.dtype and a.stride(-1) == 1 and w.stride(-1) == 1
    Mv = a.shape[-2] if M is None else M
    N, K = w.shape[-2], w.shape[-1]
    assert a.shape[-1] == K
    if bias is not None:
        assert bias.dtype == torch.float32
    ld = ldc if ldc is not None else (out.stride(-2) if out is not None else 0)
    check(lib.m5_gemm(_gemm_code(a.dtype), _p(a), a.stride(-2), _p(w), w.stride(-2), _p(bias), _p(out), ld, Mv, N, K, epi,
                      C.byref(scatter) if scatter is not None else None, batch, sA, sW, sC, sBias, _s(stream)), "m5_gemm")


def gemm_dln(a: torch.Tensor, w: torch.Tensor, out: Optional[torch.Tensor], epi: int, dl: Optional[L.DeferredLN], bias: Optional[torch.Tensor] = None,
             scatter: Optional[L.QkvScatter] = None, M: Optional[int] = None, ldc: Optional[int] = None,
             batch: int = 1, sA: int = 0, sW: int = 0, sC: int = 0, sBias: int = 0, stream: Optional[int] = None,
             rt: Optional[L.RowTiles] = None) -> None:
    """``gemm`` with a deferred LayerNorm (include/mars5_hip.h, M5DeferredLN): epi RESIDUAL = the producer (also writes the
    centred copy + row partials), QKV / SWIGLU = a consumer (applies the normalisation in its epilogue); and / or over a
    row-tile list `rt` (M5RowTiles: only the tiles that hold real rows of a padded batch are launched)."""
    assert a.dtype == w.dtype and a.stride(-1) == 1 and w.stride(-1) == 1
    Mv = a.shape[-2] if M is None else M
    N, K = w.shape[-2], w.shape[-1]
    assert a.shape[-1] == K
    if bias is not None:
        assert bias.dtype == torch.float32
    ld = ldc if ldc is not None else (out.stride(-2) if out is not None else 0)
    check(lib.m5_gemm_ex(DT_CODE[a.dtype], _p(a), a.stride(-2), _p(w), w.stride(-2), _p(bias), _p(out), ld, Mv, N, K, epi,
                         C.byref(scatter) if scatter is not None else None, batch, sA, sW, sC, sBias, C.byref(dl) if dl is not None else None,
                         C.byref(rt) if rt is not None else None, _s(stream)), "m5_gemm_ex")


def xattn_scores_dln(x: torch.Tensor, sX: int, a_tab: torch.Tensor, c_tab: torch.Tensor, p_out: torch.Tensor, sP: int, M: int, n_heads: int,
                     Lp: int, batch: int, dl: Optional[L.DeferredLN], stream: Optional[int] = None, rt: Optional[L.RowTiles] = None) -> None:
    """``xattn_scores`` on the centred copy x with the LayerNorm applied in the epilogue (dl.mode = 2) and / or over a row-tile list."""
    N, K = n_heads * Lp, x.shape[-1]
    check(lib.m5_xattn_scores_ex(DT_CODE[x.dtype], _p(x), x.stride(-2), sX, _p(a_tab), N * K, _p(c_tab), N, _p(p_out), p_out.stride(-2), sP,
                                 M, n_heads, Lp, K, batch, C.byref(dl) if dl is not None else None, C.byref(rt) if rt is not None else None,
                                 _s(stream)), "m5_xattn_scores_ex")


def layernorm_mean(x: torch.Tensor, gamma: torch.Tensor, beta: torch.Tensor, eps: float, out: torch.Tensor, mean_out: torch.Tensor,
                   M: Optional[int] = None, stream: Optional[int] = None) -> None:
    """``layernorm`` that also leaves the row means (fp32) in mean_out: the first centre of a deferred-LayerNorm chain."""
    assert x.dtype == torch.float32 and mean_out.dtype == torch.float32 and x.stride(-1) == 1 and out.stride(-1) == 1
    Mv = x.shape[0] if M is None else M
    assert mean_out.numel() >= Mv
    check(lib.m5_layernorm_mean(DT_CODE[out.dtype], _p(x), x.stride(0), _p(gamma), _p(beta), eps, _p(out), out.stride(-2), Mv, x.shape[1],
                                _p(mean_out), _s(stream)), "m5_layernorm_mean")


def layernorm_twice(x: torch.Tensor, gamma: torch.Tensor, beta: torch.Tensor, eps: float, eps2: float, out: torch.Tensor, rows_per_seq: int,
                    n_seq: int = 1, x_seq_stride: int = 0, stream: Optional[int] = None) -> None:
    """out (n_seq * rows_per_seq, D) = normalise(LayerNorm(x; gamma, beta, eps); eps2), no second affine; run s of x starts
    x_seq_stride rows after run s - 1 (include/mars5_hip.h)."""
    assert x.dtype == torch.float32 and x.stride(-1) == 1 and out.stride(-1) == 1
    check(lib.m5_layernorm_twice(DT_CODE[out.dtype], _p(x), x.stride(0), _p(gamma), _p(beta), eps, eps2, _p(out), out.stride(-2), rows_per_seq, n_seq,
                                 x_seq_stride, x.shape[1], _s(stream)), "m5_layernorm_twice")


def gemm_q_cross_attn(a: torch.Tensor, w: torch.Tensor, bias: Optional[torch.Tensor], n_heads: int, mem_table: torch.Tensor, max_le: int,
                      rows_per_seq: int, step: torch.Tensor, scale: float, out: torch.Tensor, stream: Optional[int] = None) -> bool:
    """out = cross-attention of the projected queries a @ w^T + bias against short pre-projected memories, one launch.
    mem_table (n_seq, 6) int64 device (include/mars5_hip.h).  False if the shape is not eligible (nothing launched)."""
    assert a.dtype == w.dtype == out.dtype and mem_table.dtype == torch.int64 and mem_table.is_contiguous()
    if L.tool_knob("M5_GEMM_XATTN", "0") != "1":    # tools build only (the product library does not export it): measured slower inside the NAR step (csrc/gemm16.hip)
        return False
    st = lib.m5_gemm_q_cross_attn(DT_CODE[a.dtype], _p(a), a.stride(0), _p(w), w.stride(0), _p(bias), a.shape[0], n_heads, w.shape[1],
                                  _p(mem_table), max_le, rows_per_seq, _p(step), scale, _p(out), out.stride(0), _s(stream))
    if st == L.M5_ERR_UNSUPPORTED:
        return False
    check(st, "m5_gemm_q_cross_attn")
    return True


def xattn_absorb(dtype: torch.dtype, tab_seq: torch.Tensor, tab_layer: torch.Tensor, n_layers: int, n_seq: int, n_heads: int, D: int, Lp: int,
                 step: torch.Tensor, scale: float, stream: Optional[int] = None) -> None:
    """Build the absorbed cross-attention operands (A, c, B^T) of every (layer, sequence) for the memory block of step *step."""
    assert tab_seq.dtype == torch.int64 and tab_layer.dtype == torch.int64 and tab_seq.is_contiguous() and tab_layer.is_contiguous()
    check(lib.m5_xattn_absorb(DT_CODE[dtype], _p(tab_seq), _p(tab_layer), n_layers, n_seq, n_heads, D, Lp, _p(step), scale, _s(stream)),
          "m5_xattn_absorb")


def xattn_scores(x: torch.Tensor, sX: int, a_tab: torch.Tensor, c_tab: torch.Tensor, p_out: torch.Tensor, sP: int, M: int, n_heads: int,
                 Lp: int, batch: int, stream: Optional[int] = None) -> None:
    """p_out[b] = per-head softmax(x[b] a_tab[b]^T + c_tab[b]): x (rows, K) with batch stride sX rows*K elements given in elements."""
    N, K = n_heads * Lp, x.shape[-1]
    check(lib.m5_xattn_scores(DT_CODE[x.dtype], _p(x), x.stride(-2), sX, _p(a_tab), N * K, _p(c_tab), N, _p(p_out), p_out.stride(-2), sP,
                              M, n_heads, Lp, K, batch, _s(stream)), "m5_xattn_scores")


def gemm_residual_ln(a: torch.Tensor, w: torch.Tensor, x: torch.Tensor, bias: Optional[torch.Tensor], gamma: torch.Tensor,
                     beta: torch.Tensor, eps: float, xn: torch.Tensor, scratch: torch.Tensor, tag: int = 0,
                     tag_step: Optional[torch.Tensor] = None, stream: Optional[int] = None) -> bool:
    """x += a @ w^T + bias and xn = LayerNorm(x) in one launch.  False if the shape is not eligible for the fused kernel
    (nothing was launched; run gemm + layernorm instead).  Consecutive calls on one `scratch` need different launch tags
    (tag, or the device counter `tag_step` under graph replay): see include/mars5_hip.h."""
    assert a.dtype == w.dtype == xn.dtype and x.dtype == torch.float32 and scratch.dtype == torch.uint8
    if L.tool_knob("M5_GEMM_LN", "0") != "1":       # tools build only (the product library does not export it): measured slower than GEMM + LayerNorm launches (csrc/gemm16.hip)
        return False
    N, K = w.shape
    st = lib.m5_gemm_residual_ln(DT_CODE[a.dtype], _p(a), a.stride(0), _p(w), w.stride(0), _p(bias), _p(x), x.stride(0), a.shape[0], N, K,
                                 _p(gamma), _p(beta), eps, _p(xn), xn.stride(0), _p(scratch), scratch.numel(), _p(tag_step), tag, _s(stream))
    if st == L.M5_ERR_UNSUPPORTED:
        return False
    check(st, "m5_gemm_residual_ln")
    return True


def layernorm(x: torch.Tensor, gamma: torch.Tensor, beta: torch.Tensor, eps: float, out: torch.Tensor,
              n_affine: int = 1, affine_stride: int = 0, y_affine_stride: int = 0, M: Optional[int] = None,
              stream: Optional[int] = None) -> None:
    assert x.dtype == torch.float32 and x.stride(-1) == 1 and out.stride(-1) == 1
    Mv = x.shape[0] if M is None else M
    ldy = out.stride(-2)
    check(lib.m5_layernorm(DT_CODE[out.dtype], _p(x), x.stride(0), _p(gamma), _p(beta), eps, _p(out), ldy, Mv, x.shape[1],
                           n_affine, affine_stride, y_affine_stride, _s(stream)), "m5_layernorm")


def rmsnorm(x: torch.Tensor, w: torch.Tensor, eps: float, out: torch.Tensor, stream: Optional[int] = None) -> None:
    assert x.dtype == torch.float32 and x.stride(-1) == 1
    check(lib.m5_rmsnorm(DT_CODE[out.dtype], _p(x), x.stride(0), _p(w), eps, _p(out), out.stride(0), x.shape[0], x.shape[1],
                         _s(stream)), "m5_rmsnorm")


def attention(dtype: torch.dtype, args: L.AttnArgs, stream: Optional[int] = None) -> None:
    check(lib.m5_attention(_gemm_code(dtype), C.byref(args), _s(stream)), "m5_attention")


def gather_rows(out: torch.Tensor, table: torch.Tensor, idx: torch.Tensor, alpha: Optional[torch.Tensor] = None,
                pe: Optional[torch.Tensor] = None, pos: Optional[torch.Tensor] = None, add: Optional[torch.Tensor] = None,
                add_idx: Optional[torch.Tensor] = None, stream: Optional[int] = None) -> None:
    assert out.dtype == torch.float32 and table.dtype == torch.float32 and idx.dtype == torch.int64
    R, D = out.shape
    assert table.shape[1] == D and table.is_contiguous()
    check(lib.m5_gather_rows(_p(out), out.stride(0), R, D, _p(table), _p(idx), _p(alpha), _p(pe), _p(pos), _p(add),
                             _p(add_idx), _s(stream)), "m5_gather_rows")


def chunked_embed(out: torch.Tensor, tables: torch.Tensor, codes: Optional[torch.Tensor], lead_row: Optional[torch.Tensor],
                  alpha: Optional[torch.Tensor], pe: Optional[torch.Tensor], add: Optional[torch.Tensor] = None,
                  add_index: Optional[torch.Tensor] = None, rows: Optional[int] = None, stream: Optional[int] = None) -> None:
    """out (n_rep, Rr, D) fp32, the first R = `rows` (default Rr) rows of every rep are written;
    tables (n_q, n_codes, D/n_q); codes (R-lead, n_q) int64."""
    assert out.dtype == torch.float32 and out.is_contiguous() and tables.is_contiguous()
    n_rep, Rr, D = out.shape
    R = Rr if rows is None else rows
    assert R <= Rr
    n_q, n_codes, _ = tables.shape
    if codes is not None:
        assert codes.dtype == torch.int64 and codes.is_contiguous()
    check(lib.m5_chunked_embed(_p(out), Rr * D, n_rep, R, D, n_q, n_codes, _p(tables), _p(codes), _p(lead_row), _p(alpha),
                               _p(pe), _p(add), _p(add_index), _s(stream)), "m5_chunked_embed")


def rope_cache(qkv: torch.Tensor, n_heads: int, pos0: int, rope: torch.Tensor, q_out: torch.Tensor, kcache: torch.Tensor,
               vcache: torch.Tensor, cache_hs: int, window: int, vt_out: torch.Tensor, vt_hs: int, vt_ds: int,
               stream: Optional[int] = None) -> None:
    check(lib.m5_rope_cache(DT_CODE[qkv.dtype], _p(qkv), qkv.shape[0], n_heads, pos0, _p(rope), _p(q_out), _p(kcache),
                            _p(vcache), cache_hs, window, _p(vt_out), vt_hs, vt_ds, _s(stream)), "m5_rope_cache")


def ar_gemv(dtype: torch.dtype, pro: int, epi: int, args: L.GemvArgs, stream: Optional[int] = None) -> None:
    check(lib.m5_ar_gemv(DT_CODE[dtype], pro, epi, C.byref(args), _s(stream)), "m5_ar_gemv")


def ar_layers_persistent(dtype: torch.dtype, args: L.ArMegaArgs, stream: Optional[int] = None) -> int:
    """All Mistral layers of one decode step as one persistent launch (csrc/ar_mega.hip).  Returns the C status: M5_OK, or
    M5_ERR_UNSUPPORTED when the geometry / device does not allow it (the caller then enqueues the per-launch form)."""
    rc = lib.m5_ar_layers_persistent(DT_CODE[dtype], C.byref(args), _s(stream))
    if rc not in (L.M5_OK, L.M5_ERR_UNSUPPORTED):
        check(rc, "m5_ar_layers_persistent")
    return rc


def ar_rope_cache_batch(qkv: torch.Tensor, n_heads: int, rope: torch.Tensor, state: torch.Tensor, qbuf: torch.Tensor,
                        kcache: torch.Tensor, vcache: torch.Tensor, cache_bs: int, cache_hs: int, window: int,
                        stream: Optional[int] = None) -> None:
    """qkv (B, 3D) dtype; state (B, ST_WORDS) int32; qbuf (B, D); k/vcache: this layer's [h][W][64] block of
    sequence 0, sequence b at + b*cache_bs elements."""
    B = qkv.shape[0]
    check(lib.m5_ar_rope_cache_batch(DT_CODE[qkv.dtype], _p(qkv), B, n_heads, _p(rope), _p(state), state.stride(0), _p(qbuf),
                                     qbuf.stride(0), _p(kcache), _p(vcache), cache_bs, cache_hs, window, _s(stream)),
          "m5_ar_rope_cache_batch")


def ar_qkv_rope_batch(xn: torch.Tensor, wqkv: torch.Tensor, n_heads: int, rope: torch.Tensor, state: torch.Tensor, qbuf: torch.Tensor,
                      kcache: torch.Tensor, vcache: torch.Tensor, cache_bs: int, cache_hs: int, window: int, qkv_tmp: torch.Tensor,
                      stream: Optional[int] = None) -> None:
    """Batched decode QKV projection + RoPE + cache write: xn (B, K) dtype, wqkv (3D, K)."""
    check(lib.m5_ar_qkv_rope_batch(DT_CODE[xn.dtype], _p(xn), xn.stride(0), _p(wqkv), wqkv.stride(0), xn.shape[0], n_heads, xn.shape[1],
                                   _p(rope), _p(state), state.stride(0), _p(qbuf), qbuf.stride(0), _p(kcache), _p(vcache), cache_bs,
                                   cache_hs, window, _p(qkv_tmp), _s(stream)), "m5_ar_qkv_rope_batch")


def ar_attn_combine_batch(part: torch.Tensor, n_heads: int, nsplit: int, state: torch.Tensor, out: torch.Tensor,
                          stream: Optional[int] = None) -> None:
    """part (B, H, nsplit, ATTN_PART) fp32 -> out (B, D) dtype."""
    B = part.shape[0]
    check(lib.m5_ar_attn_combine_batch(DT_CODE[out.dtype], _p(part), part.stride(0), B, n_heads, nsplit, _p(state), state.stride(0),
                                       _p(out), out.stride(0), _s(stream)), "m5_ar_attn_combine_batch")


def ar_attn_decode(dtype: torch.dtype, args: L.AttnDecodeArgs, stream: Optional[int] = None) -> None:
    check(lib.m5_ar_attn_decode(DT_CODE[dtype], C.byref(args), _s(stream)), "m5_ar_attn_decode")


def ar_sample(args: L.SampleArgs, stream: Optional[int] = None) -> None:
    check(lib.m5_ar_sample(C.byref(args), _s(stream)), "m5_ar_sample")


def nar_sample(args: L.NarSampleArgs, stream: Optional[int] = None) -> None:
    check(lib.m5_nar_sample(C.byref(args), _s(stream)), "m5_nar_sample")


def nar_uniforms(args: L.NarUniformArgs, stream: Optional[int] = None) -> None:
    check(lib.m5_nar_uniforms(C.byref(args), _s(stream)), "m5_nar_uniforms")


# ---- paged serving (include/mars5_paged.h: M5Paged*Args, M5DraftVerifyArgs).  The tensors of a call live on one device, which need not be
# the current one; `stream` (a raw handle of that device) defaults to torch's current stream there.  A decode step makes dozens of these
# calls, each of them a few microseconds long on the GPU: the checks are written out inline, without helpers per tensor.
_raw_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None) or (lambda idx: torch.cuda.current_stream(idx).cuda_stream)
_current_device = getattr(torch._C, "_cuda_getDevice", None) or torch.cuda.current_device
_plan, _rope, _attn, _verify = lib.m5_paged_plan, lib.m5_paged_rope_cache, lib.m5_paged_attention, lib.m5_draft_verify
_plan_args, _rope_args, _attn_args, _verify_args = (L.packed(c) for c in (L.PagedPlanArgs, L.PagedRopeArgs, L.PagedAttnArgs, L.DraftVerifyArgs))
_I32, _I64, _F32 = torch.int32, torch.int64, torch.float32
_NO_DEVICE = "libmars5_hip operates on device memory only"
_DEVICES = "the tensors of a call live on one device"


def _launch(fn, what: str, lead: tuple, args, idx: int, stream: Optional[int]) -> None:
    if stream is None:
        stream = _raw_stream(idx)
    if idx == _current_device():
        rc = fn(*lead, args, stream)
    else:
        with torch.cuda.device(idx):
            rc = fn(*lead, args, stream)
    if rc:
        check(rc, what)


def _caches(k_cache: torch.Tensor, v_cache: torch.Tensor, dtype: torch.dtype, n_kv_heads: int, head_dim: int) -> tuple:
    """(n_blocks, block_size, k pointer and strides, v pointer and strides) of caches (n_blocks, n_kv_heads, block_size, head_dim)."""
    shape = k_cache.shape
    assert k_cache.dtype == v_cache.dtype == dtype and v_cache.shape == shape and len(shape) == 4, "caches: (n_blocks, n_kv_heads, block_size, head_dim), the rows' type"
    assert shape[1] == n_kv_heads and shape[3] == head_dim, f"cache {tuple(shape)} for {n_kv_heads} kv heads of {head_dim}"
    kb, kh, ks, k1 = k_cache.stride()
    vb, vh, vs, v1 = v_cache.stride()
    assert k1 == v1 == 1, "caches: features are contiguous"
    return shape[0], shape[2], (k_cache.data_ptr(), kb, kh, ks), (v_cache.data_ptr(), vb, vh, vs)


def paged_plan(seq_len: torch.Tensor, keep_len: torch.Tensor, new_len: torch.Tensor, block_table: torch.Tensor, free_blocks: torch.Tensor,
               state: torch.Tensor, block_size: int, q_start: torch.Tensor, slot_map: Optional[torch.Tensor] = None,
               positions: Optional[torch.Tensor] = None, stream: Optional[int] = None) -> None:
    """One step of a paged cache: request b keeps keep_len[b] of its seq_len[b] positions and adds new_len[b]; block_table
    (n_seq, width), the free stack (free_blocks, state[PST_FREE]) and seq_len are brought up to date, q_start (n_seq + 1,),
    slot_map and positions (n_rows,) describe the step's rows (None: not wanted).  All int32.  state (PST_WORDS,): zero-filled once,
    then state[PST_FREE] = the number of free ids; state[PST_STATUS] != 0 afterwards: nothing was done (include/mars5_paged.h).
    keep_len may be seq_len itself (all is kept); otherwise the tensors must not overlap.  One launch."""
    idx, (B,), (n_blocks,) = seq_len.get_device(), seq_len.shape, free_blocks.shape
    assert idx >= 0, _NO_DEVICE
    assert (idx == keep_len.get_device() == new_len.get_device() == block_table.get_device() == free_blocks.get_device() == state.get_device() ==
            q_start.get_device()), _DEVICES
    assert (seq_len.dtype == keep_len.dtype == new_len.dtype == block_table.dtype == free_blocks.dtype == state.dtype == q_start.dtype == _I32), "int32 tensors"
    assert keep_len.shape == new_len.shape == (B,) and q_start.shape == (B + 1,) and state.shape == (L.PST_WORDS,), "keep_len, new_len (n_seq,), q_start (n_seq + 1,), state (PST_WORDS,)"
    assert (seq_len.is_contiguous() and keep_len.is_contiguous() and new_len.is_contiguous() and free_blocks.is_contiguous() and state.is_contiguous() and
            q_start.is_contiguous()), "contiguous tensors (a table's rows may lie apart)"
    assert block_table.dim() == 2 and block_table.shape[0] == B and block_table.stride(1) == 1, "block_table: (n_seq, width)"
    assert (slot_map is None) == (positions is None), "slot_map and positions go together"
    n_rows = slots = where = 0
    if slot_map is not None:
        (n_rows,) = slot_map.shape
        assert n_rows > 0, "slot_map of no rows: pass None"
        assert idx == slot_map.get_device() == positions.get_device(), _DEVICES
        assert slot_map.dtype == positions.dtype == _I32 and positions.shape == (n_rows,) and slot_map.is_contiguous() and positions.is_contiguous(), "slot_map, positions: (n_rows,) int32"
        slots, where = slot_map.data_ptr(), positions.data_ptr()
    args = _plan_args(seq_len.data_ptr(), keep_len.data_ptr(), new_len.data_ptr(), B, block_table.shape[1], n_blocks, block_size, n_rows,
                      block_table.data_ptr(), block_table.stride(0), free_blocks.data_ptr(), state.data_ptr(), q_start.data_ptr(), slots, where)
    _launch(_plan, "m5_paged_plan", (), C.byref(args), idx, stream)


def paged_rope_cache(qkv: torch.Tensor, n_heads: int, n_kv_heads: int, rope: torch.Tensor, positions: torch.Tensor, slot_map: torch.Tensor,
                     q_out: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor, q_norm: Optional[torch.Tensor] = None,
                     k_norm: Optional[torch.Tensor] = None, eps: float = 1e-5, interleaved: bool = True, stream: Optional[int] = None) -> None:
    """``rope_cache`` for a paged cache: qkv (n_rows, (n_heads + 2 n_kv_heads) head_dim) -> RMSNorm of every q / k head (weights fp32
    (head_dim,), None = none), rotation by rope (n_pos, n_pairs, 2) fp32 (tables.rope_table) at positions, q -> q_out
    (n_rows, n_heads, head_dim), k / v -> slot_map of the caches (n_blocks, n_kv_heads, block_size, head_dim), any strides with
    contiguous features.  Rows of slot or position -1 are skipped; slots must be distinct; q_out may be
    the q part of qkv itself.  One launch."""
    idx, (rows, width), dt, out_shape = qkv.get_device(), qkv.shape, qkv.dtype, q_out.shape
    hd = out_shape[2]
    assert idx >= 0, _NO_DEVICE
    assert (idx == rope.get_device() == positions.get_device() == slot_map.get_device() == q_out.get_device() == k_cache.get_device() ==
            v_cache.get_device()), _DEVICES
    assert width == (n_heads + 2 * n_kv_heads) * hd, f"qkv has {width} columns, {n_heads} + 2 * {n_kv_heads} heads of {hd} need others"
    assert q_out.dtype == dt and out_shape == (rows, n_heads, hd), "q_out: (n_rows, n_heads, head_dim), qkv's type"
    assert rope.dtype == _F32 and rope.dim() == 3 and rope.shape[2] == 2 and rope.is_contiguous(), "rope: (n_pos, n_pairs, 2) fp32"
    assert positions.dtype == slot_map.dtype == _I32 and positions.shape == slot_map.shape == (rows,), "positions, slot_map: (n_rows,) int32"
    assert positions.is_contiguous() and slot_map.is_contiguous() and qkv.stride(1) == 1
    q_rs, q_hs, q1 = q_out.stride()
    assert q1 == 1, "q_out: features are contiguous"
    n_blocks, block_size, k, v = _caches(k_cache, v_cache, dt, n_kv_heads, hd)
    qw = kw = 0
    if q_norm is not None:
        assert q_norm.dtype == _F32 and q_norm.shape == (hd,) and q_norm.is_contiguous() and q_norm.get_device() == idx, "q_norm: (head_dim,) fp32"
        qw = q_norm.data_ptr()
    if k_norm is not None:
        assert k_norm.dtype == _F32 and k_norm.shape == (hd,) and k_norm.is_contiguous() and k_norm.get_device() == idx, "k_norm: (head_dim,) fp32"
        kw = k_norm.data_ptr()
    if rows == 0:
        return
    args = _rope_args(qkv.data_ptr(), qkv.stride(0), rows, n_heads, n_kv_heads, hd, qw, kw, eps, rope.data_ptr(), rope.shape[0], rope.shape[1], interleaved,
                      positions.data_ptr(), slot_map.data_ptr(), q_out.data_ptr(), q_rs, q_hs, *k, *v, n_blocks, block_size)
    _launch(_rope, "m5_paged_rope_cache", (DT_CODE[dt],), C.byref(args), idx, stream)


def _paged_attn_args(q, k_cache, v_cache, block_table, seq_len, q_start, out, scale, window, max_new, workspace) -> tuple:
    idx, (rows, heads, hd), (B,), dt = q.get_device(), q.shape, seq_len.shape, q.dtype
    assert idx >= 0, _NO_DEVICE
    assert (idx == k_cache.get_device() == v_cache.get_device() == block_table.get_device() == seq_len.get_device() == q_start.get_device() ==
            out.get_device()), _DEVICES
    assert out.dtype == dt and out.shape == q.shape, "out: q's shape and type"
    q_rs, q_hs, q1 = q.stride()
    o_rs, o_hs, o1 = out.stride()
    assert q1 == o1 == 1, "q, out: features are contiguous"
    kv = k_cache.shape[1]
    n_blocks, block_size, k, v = _caches(k_cache, v_cache, dt, kv, hd)
    assert heads % kv == 0, f"{heads} query heads over {kv} kv heads"
    assert seq_len.dtype == q_start.dtype == block_table.dtype == _I32 and q_start.shape == (B + 1,) and seq_len.is_contiguous() and q_start.is_contiguous(), \
        "seq_len (n_seq,), q_start (n_seq + 1,), block_table (n_seq, width): int32"
    assert block_table.dim() == 2 and block_table.shape[0] == B and block_table.stride(1) == 1, "block_table: (n_seq, width)"
    assert window >= 0 and (scale is None or scale > 0)
    ws = ws_bytes = 0
    if workspace is not None:
        assert workspace.dtype == torch.uint8 and workspace.dim() == 1 and workspace.is_contiguous() and workspace.get_device() == idx, "workspace: zero-filled uint8 bytes"
        ws, ws_bytes = workspace.data_ptr(), workspace.shape[0]
    return idx, _attn_args(q.data_ptr(), q_rs, q_hs, *k, *v, block_table.data_ptr(), block_table.stride(0), block_table.shape[1], n_blocks, block_size,
                           B, rows, rows if max_new is None else max_new, heads, kv, hd, window, seq_len.data_ptr(), q_start.data_ptr(),
                           hd ** -0.5 if scale is None else scale, out.data_ptr(), o_rs, o_hs, ws, ws_bytes)


def paged_attention(q: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor, block_table: torch.Tensor, seq_len: torch.Tensor,
                    q_start: torch.Tensor, out: torch.Tensor, scale: Optional[float] = None, window: int = 0, max_new: Optional[int] = None,
                    workspace: Optional[torch.Tensor] = None, stream: Optional[int] = None) -> None:
    """out (n_rows, n_heads, head_dim) = causal attention of every request's new rows q over its seq_len[b] cached positions (the
    rows' own included), optionally through a sliding window.  Rows from q_start[-1] on are padding.  scale: 1 / sqrt(head_dim).
    max_new: upper bound of the new tokens of one request (speed only).  workspace: uint8, zero-filled once, one for every call
    that may be in flight at a time; without it keys are not split over workgroups (paged_attention_workspace: how much).
    One launch."""
    if q.shape[0] == 0:
        return
    idx, args = _paged_attn_args(q, k_cache, v_cache, block_table, seq_len, q_start, out, scale, window, max_new, workspace)
    _launch(_attn, "m5_paged_attention", (DT_CODE[q.dtype],), C.byref(args), idx, stream)


def paged_attention_workspace(q: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor, block_table: torch.Tensor, seq_len: torch.Tensor,
                              q_start: torch.Tensor, out: torch.Tensor, window: int = 0, max_new: Optional[int] = None) -> int:
    """Bytes of workspace that paged_attention can use for tensors of these shapes (it works with fewer)."""
    _, args = _paged_attn_args(q, k_cache, v_cache, block_table, seq_len, q_start, out, None, window, max_new, None)
    n = L.i64(0)
    check(lib.m5_paged_attention_workspace(DT_CODE[q.dtype], C.byref(args), C.byref(n)), "m5_paged_attention_workspace")
    return int(n.value)


def draft_verify(target: torch.Tensor, draft: Optional[torch.Tensor], tokens: torch.Tensor, row_start: torch.Tensor, uniforms: torch.Tensor,
                 noise: torch.Tensor, out_tokens: torch.Tensor, n_out: torch.Tensor, seq_len: Optional[torch.Tensor] = None,
                 keep_len: Optional[torch.Tensor] = None, workspace: Optional[torch.Tensor] = None, stream: Optional[int] = None,
                 plan_state: Optional[torch.Tensor] = None) -> None:
    """Speculative sampling from given random numbers: target / draft (n_rows, vocab) probabilities (draft None: certain drafts),
    tokens (n_rows,) int64 the tokens that were fed, row_start (n_seq + 1,) int32, uniforms (n_rows,) and noise (n_seq, vocab)
    fp32 (U[0, 1) and Exp(1)).  out_tokens (n_seq, width) int64 = accepted drafts, one drawn token, -1; n_out (n_seq,) int32;
    keep_len = seq_len - rows + n_out for the next paged_plan.  workspace: DRAFT_WS_BYTES per request (uint8, zero-filled once, one
    for every call that may be in flight at a time), or None.  plan_state: the state of the step's paged_plan; if that refused the
    step, nothing is verified and keep_len (the tensor that the plan was given) stays as it was.  row_start is the plan's q_start only in
    steps without prompt chunks: of those, the last row alone is verified (include/mars5_paged.h).  One launch."""
    idx, (rows, V), (B,), dt = target.get_device(), target.shape, n_out.shape, target.dtype
    assert idx >= 0, _NO_DEVICE
    assert (idx == tokens.get_device() == row_start.get_device() == uniforms.get_device() == noise.get_device() == out_tokens.get_device() ==
            n_out.get_device()), _DEVICES
    assert rows > 0 and target.stride(1) == 1, "target: (n_rows, vocab)"
    assert tokens.dtype == _I64 and tokens.shape == (rows,) and tokens.is_contiguous(), "tokens: (n_rows,) int64"
    assert uniforms.dtype == noise.dtype == _F32 and uniforms.shape == (rows,) and uniforms.is_contiguous() and noise.shape == (B, V) and noise.stride(1) == 1, \
        "uniforms (n_rows,), noise (n_seq, vocab): fp32"
    assert out_tokens.dtype == _I64 and out_tokens.dim() == 2 and out_tokens.shape[0] == B and out_tokens.stride(1) == 1, "out_tokens: (n_seq, width) int64"
    assert row_start.dtype == n_out.dtype == _I32 and row_start.shape == (B + 1,) and row_start.is_contiguous() and n_out.is_contiguous(), "row_start (n_seq + 1,), n_out (n_seq,): int32"
    assert (seq_len is None) == (keep_len is None), "seq_len and keep_len go together"
    q = q_rs = held = kept = ws = ws_bytes = words = 0
    if draft is not None:
        assert draft.shape == target.shape and draft.dtype == dt and draft.stride(1) == 1 and draft.get_device() == idx, "draft: target's shape and type"
        q, q_rs = draft.data_ptr(), draft.stride(0)
    if seq_len is not None:
        assert idx == seq_len.get_device() == keep_len.get_device(), _DEVICES
        assert seq_len.dtype == keep_len.dtype == _I32 and seq_len.shape == keep_len.shape == (B,) and seq_len.is_contiguous() and keep_len.is_contiguous(), "seq_len, keep_len: (n_seq,) int32"
        held, kept = seq_len.data_ptr(), keep_len.data_ptr()
    if workspace is not None:
        assert workspace.dtype == torch.uint8 and workspace.dim() == 1 and workspace.is_contiguous() and workspace.get_device() == idx, "workspace: zero-filled uint8 bytes"
        ws, ws_bytes = workspace.data_ptr(), workspace.shape[0]
    if plan_state is not None:
        assert plan_state.dtype == _I32 and plan_state.shape == (L.PST_WORDS,) and plan_state.is_contiguous() and plan_state.get_device() == idx, "plan_state: (PST_WORDS,) int32"
        words = plan_state.data_ptr()
    args = _verify_args(target.data_ptr(), target.stride(0), q, q_rs, rows, V, B, out_tokens.shape[1], tokens.data_ptr(), row_start.data_ptr(), uniforms.data_ptr(),
                        noise.data_ptr(), noise.stride(0), out_tokens.data_ptr(), out_tokens.stride(0), n_out.data_ptr(), held, kept, ws, ws_bytes, words)
    _launch(_verify, "m5_draft_verify", (DT_CODE[dt],), C.byref(args), idx, stream)


def expand_tokens(tokens: torch.Tensor, n_text: int, off: torch.Tensor, vals: torch.Tensor, max_run: int,
                  stream: Optional[int] = None) -> torch.Tensor:
    """AR token ids (n,) int64 -> codebook-0 frames (G,) int64 through the CSR expansion table (off int32 (V+1,), vals int64):
    one launch, then a 4-byte read-back of G (the NAR buffers are sized by it)."""
    assert tokens.dtype == torch.int64 and off.dtype == torch.int32 and vals.dtype == torch.int64 and tokens.is_contiguous()
    n = int(tokens.shape[0])
    if n == 0:
        return torch.empty(0, dtype=torch.int64, device=tokens.device)
    cap = max(n * max(max_run, 1), 1)
    out = torch.empty(cap, dtype=torch.int64, device=tokens.device)
    total = torch.zeros(1, dtype=torch.int32, device=tokens.device)
    check(lib.m5_expand_tokens(_p(tokens), n, n_text, _p(off), _p(vals), off.shape[0] - 1, _p(out), cap, _p(total), _s(stream)), "m5_expand_tokens")
    return out[: int(total.item())]


def trim_bounds(y: torch.Tensor, top_db: float, frame_length: int = 2048, hop_length: int = 512, stream: Optional[int] = None) -> torch.Tensor:
    """[start, end) (int32 (2,), device) of the non-silent part of the mono fp32 device signal y (n,): two launches."""
    assert y.dtype == torch.float32 and y.dim() == 1 and y.is_contiguous()
    n = int(y.shape[0])
    nf = 1 + n // hop_length
    power = torch.empty(nf, dtype=torch.float32, device=y.device)
    bounds = torch.zeros(2, dtype=torch.int32, device=y.device)
    check(lib.m5_trim_bounds(_p(y), n, frame_length, hop_length, float(top_db), _p(power), nf, _p(bounds), _s(stream)), "m5_trim_bounds")
    return bounds


def copy_d2d(dst: torch.Tensor, src: torch.Tensor, stream: Optional[int] = None) -> None:
    """dst = src (contiguous device tensors of the same size and dtype) as a stream-ordered device copy of this library --
    capturable, and plannable (a torch ``copy_`` is neither visible to a stage plan nor free of an ATen launch)."""
    assert dst.is_contiguous() and src.is_contiguous() and dst.dtype == src.dtype and dst.numel() == src.numel()
    check(lib.m5_copy_d2d(_p(dst), _p(src), dst.numel() * dst.element_size(), _s(stream)), "m5_copy_d2d")


class StagePlan:
    """A stage of the hot path as ONE C call (include/mars5_hip.h: m5_nar_step / m5_ar_decode_step / m5_stage_run).  The
    host engine runs its enqueue code once under ``recording()`` -- every launch that would have gone to the library is
    appended to the plan instead -- and from then on ``run(stream)`` enqueues the whole stage from C.  The tensors the
    recorded launches point to must stay alive and in place (the engines' sessions own them); `keep` holds extra references."""

    KINDS = {"nar_step": "m5_nar_step", "ar_decode_step": "m5_ar_decode_step", "stage": "m5_stage_run"}

    def __init__(self, kind: str):
        assert kind in self.KINDS, kind
        self.kind, self._rec, self._c, self.keep = kind, None, None, []

    def recording(self):
        plan = self

        class _Ctx:
            def __enter__(self_c):
                assert getattr(L._REC, "plan", None) is None, "a stage plan is already being recorded on this thread"
                plan._rec = L.PlanRecorder()
                L._REC.plan = plan._rec
                return plan

            def __exit__(self_c, *exc):
                L._REC.plan = None
                if exc[0] is None:
                    plan._finish()
                return False
        return _Ctx()

    def _finish(self) -> None:
        rec = self._rec
        n = len(rec.ops)
        arr = (L.PlanOp * max(n, 1))()
        for i, (fn, slots) in enumerate(rec.ops):
            arr[i].fn, arr[i].n_args = fn, len(slots)
            for j, v in enumerate(slots):
                arr[i].a[j] = v if v < (1 << 63) else v - (1 << 64)
        arena = (C.c_ubyte * max(len(rec.arena), 1)).from_buffer_copy(bytes(rec.arena) or b"\0")
        self._failed = L.i32(-1)
        self._arr, self._arena = arr, arena
        self._c = L.StagePlanC(ops=arr, n_ops=n, arena=C.cast(arena, C.c_void_p), arena_bytes=len(rec.arena), failed_op=C.pointer(self._failed))
        self.n_ops = n

    def run(self, stream: Optional[int] = None, raise_on_error: bool = True) -> int:
        assert self._c is not None, "record the plan first"
        rc = getattr(lib, self.KINDS[self.kind])(C.byref(self._c), _s(stream))
        if rc != L.M5_OK and raise_on_error:
            check(rc, f"{self.KINDS[self.kind]} (op {int(self._failed.value)} of {self.n_ops})")
        return rc


def add_int(p: torch.Tensor, delta: int, stream: Optional[int] = None) -> None:
    assert p.dtype == torch.int32
    check(lib.m5_add_int(_p(p), delta, _s(stream)), "m5_add_int")


def mark(label: str, stream: Optional[int] = None) -> None:
    """Hook in front of launches that do not go through this module (torch copies inside a captured step): a no-op in the
    product; bench.py's in-graph timing replaces it with a clock stamp so that those launches get their own interval."""
    return None


def clock_stamp(slots: torch.Tensor, i: int, stream: Optional[int] = None) -> None:
    """slots[i] (int64, device) = the 100 MHz wall clock when this one-lane launch runs (in-graph timing, bench roofline leg)."""
    assert slots.dtype == torch.int64 and slots.is_cuda and 0 <= i < slots.numel()
    check(lib.m5_clock_stamp(slots.data_ptr() + 8 * i, _s(stream)), "m5_clock_stamp")


def use_on(t: Optional[torch.Tensor], stream: torch.cuda.Stream) -> Optional[torch.Tensor]:
    """`t` is about to be read by launches on `stream` although another stream's allocation may back it (a caller's temporary made on
    the current stream and dropped as soon as the call returns): tell torch's caching allocator, which otherwise hands the block to
    the next allocation of ITS stream while `stream` has not read it yet.  Round 5 found exactly that: the text ids of `tts()` -- a
    temporary of the default stream, gathered on the NAR stream -- were overwritten once the host no longer waited for the
    conditioning, and the gather read through garbage indices (a memory fault)."""
    if t is not None and t.is_cuda:
        t.record_stream(stream)
    return t


_SESSION_TLS = threading.local()      # per host thread: {(device index, role): stream}; the entries die with their thread


def session_stream(dev, role: str) -> torch.cuda.Stream:
    """The long-lived stream of one role ("ar", "nar", "nar_lane1", ...) on one device for the calling host thread.
    Sessions used to make a fresh ``torch.cuda.Stream()`` each: torch hands those out of a pool of 32, and its caching
    allocator keeps freed blocks PER STREAM, so the ~1.2 GB of per-utterance state (hoisted conditioning, workspaces, KV cache)
    was hipMalloc'ed again for every utterance until the pool wrapped around -- 50 ms of host time per utterance in front of the
    decode (tools/host_profile.py).  With one stream per role the blocks of the previous utterance are reused.  Roles keep the
    concurrency that exists (AR decode beside NAR conditioning; two batch groups in flight); host threads keep their own streams.
    Consequence to know about: two sessions of the SAME role made on one host thread without an explicit `stream=` share this
    stream and therefore run one after the other -- pass each its own ``torch.cuda.Stream`` (as ``tts_batch_from_codes`` does
    for its groups in flight) to overlap them.  The table is thread-local (no lock, no growth in thread-per-request servers:
    a dead thread's entries go with it); every stream that stays alive keeps its own pool of cached allocator blocks
    (``torch.cuda.empty_cache()`` returns them)."""
    d = torch.device(dev)
    idx = d.index if d.index is not None else torch.cuda.current_device()
    tab = getattr(_SESSION_TLS, "streams", None)
    if tab is None:
        tab = _SESSION_TLS.streams = {}
    st = tab.get((idx, role))
    if st is None:
        st = tab[(idx, role)] = torch.cuda.Stream(device=idx)
    return st


class Graph:
    """A captured hipGraph of libmars5_hip launches (m5_graph_* helpers)."""

    def __init__(self):
        self.exec = C.c_void_p(None)

    @staticmethod
    def begin(stream: int) -> None:
        check(lib.m5_graph_begin(stream), "m5_graph_begin")

    def end(self, stream: int) -> "Graph":
        check(lib.m5_graph_end(stream, C.byref(self.exec)), "m5_graph_end")
        return self

    def launch(self, stream: int) -> None:
        check(lib.m5_graph_launch(self.exec, stream), "m5_graph_launch")

    def __del__(self):
        try:
            if self.exec and self.exec.value:
                lib.m5_graph_destroy(self.exec)
        except Exception:
            pass


class Event:
    def __init__(self):
        self.ev = C.c_void_p(None)
        check(lib.m5_event_create(C.byref(self.ev)), "m5_event_create")

    def record(self, stream: int) -> None:
        check(lib.m5_event_record(self.ev, stream), "m5_event_record")

    def elapsed_ms(self, stop: "Event") -> float:
        ms = C.c_float(0)
        check(lib.m5_event_elapsed_ms(self.ev, stop.ev, C.byref(ms)), "m5_event_elapsed_ms")
        return float(ms.value)

    def __del__(self):
        try:
            if self.ev and self.ev.value:
                lib.m5_event_destroy(self.ev)
        except Exception:
            pass
