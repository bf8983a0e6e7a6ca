"""Torch-tensor front end of the C ABI: shape/dtype checks, then one call.

Each function mirrors one reference kernel (named in its docstring) and
launches on torch's current CUDA stream, so the calls compose with torch
streams and can be captured into CUDA graphs.  Outputs may be passed in
(``out=``) so that a decode step allocates nothing.
"""
from __future__ import annotations

from typing import Optional

import torch

from ._lib import binding, binding_q8, call, check, lib

FP16 = torch.float16


def _stream() -> int:
    return torch.cuda.current_stream().cuda_stream


def _dev(t: torch.Tensor, name: str, dtype=None):
    if not t.is_cuda:
        raise RuntimeError(f"{name} must be a CUDA tensor (the decode path has no CPU fallback)")
    if dtype is not None and t.dtype != dtype:
        raise TypeError(f"{name}: expected {dtype}, got {t.dtype}")
    if not t.is_contiguous():
        raise ValueError(f"{name} must be contiguous")
    return t.data_ptr()


def _x2d(x: torch.Tensor):
    x2 = x if x.dim() == 2 else x.reshape(1, -1)
    return x2, x2.shape[0]


def gemv_q4(packed, scales, x, rows: int, k: int, out: Optional[torch.Tensor] = None):
    """kernels/quant_matmul.metal `gemv_q4_0`: y[b] = W x[b] (fp32 accumulate)."""
    x2, B = _x2d(x)
    y = out if out is not None else torch.empty(B, rows, dtype=FP16, device=x.device)
    call("lmps_gemv_q4_0", _dev(packed, "packed", torch.uint8), _dev(scales, "scales", FP16),
         _dev(x2, "x", FP16), k, _dev(y, "y", FP16), rows, rows, k, B, _stream())
    return y if x.dim() == 2 else y.reshape(-1)


def gemv_q4_bias(packed, scales, bias, x, rows: int, k: int, out=None):
    x2, B = _x2d(x)
    y = out if out is not None else torch.empty(B, rows, dtype=FP16, device=x.device)
    call("lmps_gemv_q4_bias", _dev(packed, "packed", torch.uint8), _dev(scales, "scales", FP16),
         _dev(bias, "bias", FP16), _dev(x2, "x", FP16), k, _dev(y, "y", FP16), rows, rows, k, B,
         _stream())
    return y if x.dim() == 2 else y.reshape(-1)


def gemv_q4_residual(packed, scales, x, residual, rows: int, k: int, out=None):
    """GEMV + kernels/residual.metal: out = residual + fp16(W x).  out may be residual."""
    x2, B = _x2d(x)
    r2 = residual if residual.dim() == 2 else residual.reshape(1, -1)
    y = out if out is not None else torch.empty(B, rows, dtype=FP16, device=x.device)
    call("lmps_gemv_q4_residual", _dev(packed, "packed", torch.uint8), _dev(scales, "scales", FP16),
         _dev(x2, "x", FP16), k, _dev(r2, "residual", FP16), _dev(y, "y", FP16), rows, rows, k, B,
         _stream())
    return y if x.dim() == 2 else y.reshape(-1)


def gemv_q4_swiglu(gate_packed, gate_scales, up_packed, up_scales, x, rows: int, k: int, out=None):
    """gate/up GEMVs + kernels/swiglu.metal in one pass."""
    x2, B = _x2d(x)
    y = out if out is not None else torch.empty(B, rows, dtype=FP16, device=x.device)
    call("lmps_gemv_q4_swiglu", _dev(gate_packed, "gate_packed", torch.uint8),
         _dev(gate_scales, "gate_scales", FP16), _dev(up_packed, "up_packed", torch.uint8),
         _dev(up_scales, "up_scales", FP16), _dev(x2, "x", FP16), k, _dev(y, "y", FP16), rows,
         rows, k, B, _stream())
    return y if x.dim() == 2 else y.reshape(-1)


def lm_head_argmax(packed, scales, x, rows: int, k: int, keys: torch.Tensor, ids: torch.Tensor,
                   logits: Optional[torch.Tensor] = None):
    """runners/engine.py:171-181 on the device: Q4 LM head + first-index argmax."""
    x2, B = _x2d(x)
    call("lmps_lm_head_argmax", _dev(packed, "packed", torch.uint8), _dev(scales, "scales", FP16),
         _dev(x2, "x", FP16), k, _dev(logits, "logits", FP16) if logits is not None else None,
         _dev(keys, "keys", torch.int64), _dev(ids, "ids", torch.int32), rows, k, B, _stream())
    return ids


def rms_norm(x, gamma, eps: float = 1e-6, out=None):
    """kernels/rms_norm.metal `rms_norm_q4` (full-vector reduction)."""
    x2, B = _x2d(x)
    y = out if out is not None else torch.empty_like(x2)
    call("lmps_rms_norm", _dev(x2, "x", FP16), _dev(gamma, "gamma", FP16), _dev(y, "out", FP16),
         x2.shape[1], B, float(eps), _stream())
    return y if x.dim() == 2 else y.reshape(-1)


def rope_(vec, pos, inv_freq, n_heads: int, head_dim: int, style: int = 0):
    """kernels/rope.metal `apply_rope_q4`, in place, per-row position."""
    v2, B = _x2d(vec)
    call("lmps_rope", _dev(v2, "vec", FP16), _dev(pos, "pos", torch.int32),
         _dev(inv_freq, "inv_freq", torch.float32), n_heads, head_dim, B, style, _stream())
    return vec


def residual_add(x, y, out=None):
    o = out if out is not None else torch.empty_like(x)
    call("lmps_residual_add", _dev(x, "x", FP16), _dev(y, "y", FP16), _dev(o, "out", FP16),
         x.numel(), _stream())
    return o


def swiglu(gate, up, out=None):
    o = out if out is not None else torch.empty_like(gate)
    call("lmps_swiglu", _dev(gate, "gate", FP16), _dev(up, "up", FP16), _dev(o, "out", FP16),
         gate.numel(), _stream())
    return o


def swiglu_rows(gate_up, n: int, out):
    """out[r] = silu(gate_up[r, :n]) * gate_up[r, n:2n] (a fused gate|up GEMM output)."""
    call("lmps_swiglu_rows", _dev(gate_up, "gate_up", FP16), gate_up.shape[-1], gate_up.shape[0], n,
         _dev(out, "out", FP16), out.shape[-1], _stream())
    return out


def embed_gather(table, ids, out, bad: Optional[torch.Tensor] = None):
    V, D = table.shape
    call("lmps_embed_gather", _dev(table, "table", FP16), _dev(ids, "ids", torch.int32),
         _dev(out, "out", FP16), D, V, ids.numel(),
         _dev(bad, "bad", torch.int32) if bad is not None else None, _stream())
    return out


def attention_scores(q, k_cache, seq_len: int, n_q_heads: int, n_kv_heads: int, head_dim: int, out=None):
    s = out if out is not None else torch.empty(n_q_heads, seq_len, dtype=torch.float32, device=q.device)
    call("lmps_attention_scores", _dev(q, "q", FP16), _dev(k_cache, "k_cache", FP16),
         _dev(s, "scores", torch.float32), seq_len, n_q_heads, n_kv_heads, head_dim, _stream())
    return s


def softmax_(scores, seq_len: int, n_heads: int):
    call("lmps_softmax", _dev(scores, "scores", torch.float32), seq_len, n_heads, _stream())
    return scores


def attn_weighted_sum(scores, v_cache, seq_len: int, n_q_heads: int, n_kv_heads: int, head_dim: int, out=None):
    o = out if out is not None else torch.empty(n_q_heads * head_dim, dtype=FP16, device=scores.device)
    call("lmps_attn_weighted_sum", _dev(scores, "scores", torch.float32), _dev(v_cache, "v_cache", FP16),
         _dev(o, "out", FP16), seq_len, n_q_heads, n_kv_heads, head_dim, _stream())
    return o


def rope_kv_append(qkv, pos, inv_freq, q_out, k_pool, v_pool, block_table, page_size: int,
                   n_q_heads: int, n_kv_heads: int, head_dim: int, style: int = 0):
    B = qkv.shape[0]
    call("lmps_rope_kv_append", _dev(qkv, "qkv", FP16), _dev(pos, "pos", torch.int32),
         _dev(inv_freq, "inv_freq", torch.float32), _dev(q_out, "q_out", FP16),
         _dev(k_pool, "k_pool", FP16), _dev(v_pool, "v_pool", FP16),
         _dev(block_table, "block_table", torch.int32), block_table.shape[1], page_size,
         n_q_heads, n_kv_heads, head_dim, B, style, _stream())
    return q_out


def gqa_decode_attention_rope(qkv, pos, inv_freq, k_pool, v_pool, block_table, seq_lens, out, workspace,
                              page_size: int, n_q_heads: int, n_kv_heads: int, head_dim: int,
                              max_seq_len: int, n_splits: int, style: int = 0):
    """rope_kv_append + gqa_decode_attention in one launch (seq_lens = pos + 1)."""
    B = qkv.shape[0]
    ws_ptr = workspace.data_ptr() if workspace is not None and workspace.numel() else None
    ws_bytes = workspace.numel() * workspace.element_size() if workspace is not None else 0
    call("lmps_gqa_decode_attention_rope", _dev(qkv, "qkv", FP16), _dev(pos, "pos", torch.int32),
         _dev(inv_freq, "inv_freq", torch.float32), style, _dev(k_pool, "k_pool", FP16),
         _dev(v_pool, "v_pool", FP16), _dev(block_table, "block_table", torch.int32),
         _dev(seq_lens, "seq_lens", torch.int32), _dev(out, "out", FP16), ws_ptr, ws_bytes,
         block_table.shape[1], page_size, n_q_heads, n_kv_heads, head_dim, B, max_seq_len, n_splits, _stream())
    return out


def attention_splits(batch: int, n_kv_heads: int, max_seq_len: int, page_size: int) -> int:
    return int(lib().lmps_gqa_attention_splits(batch, n_kv_heads, max_seq_len, page_size))


def attention_workspace_size(batch: int, n_q_heads: int, head_dim: int, n_splits: int) -> int:
    return int(lib().lmps_gqa_attention_workspace_size(batch, n_q_heads, head_dim, n_splits))


def gqa_decode_attention(q, k_pool, v_pool, block_table, seq_lens, out, workspace,
                         page_size: int, n_q_heads: int, n_kv_heads: int, head_dim: int,
                         max_seq_len: int, n_splits: int):
    """Fused attention.metal + softmax.metal + attn_sum.metal over the paged cache."""
    B = q.shape[0]
    ws_ptr = workspace.data_ptr() if workspace is not None and workspace.numel() else None
    ws_bytes = workspace.numel() * workspace.element_size() if workspace is not None else 0
    call("lmps_gqa_decode_attention", _dev(q, "q", FP16), _dev(k_pool, "k_pool", FP16),
         _dev(v_pool, "v_pool", FP16), _dev(block_table, "block_table", torch.int32),
         _dev(seq_lens, "seq_lens", torch.int32), _dev(out, "out", FP16), ws_ptr, ws_bytes,
         block_table.shape[1], page_size, n_q_heads, n_kv_heads, head_dim, B, max_seq_len,
         n_splits, _stream())
    return out


def q4_pack_device(w: torch.Tensor):
    """utils/pack_weights.py `pack_tensor_4bit` on the device (bit-exact)."""
    n = w.numel()
    groups = (n + 31) // 32
    packed = torch.empty(groups * 16, dtype=torch.uint8, device=w.device)
    scales = torch.empty(groups, dtype=FP16, device=w.device)
    call("lmps_q4_pack", _dev(w, "w", torch.float32), n, packed.data_ptr(), scales.data_ptr(), _stream())
    return packed, scales


def decode_advance(next_ids, tokens, pos, seq_lens, history=None, step=None):
    B = tokens.numel()
    max_steps = history.shape[0] if history is not None else 0
    call("lmps_decode_advance", _dev(next_ids, "next", torch.int32), _dev(tokens, "tokens", torch.int32),
         _dev(pos, "pos", torch.int32), _dev(seq_lens, "seq_lens", torch.int32),
         _dev(history, "history", torch.int32) if history is not None else None,
         _dev(step, "step", torch.int32) if step is not None else None, max_steps, B, _stream())


EPI_NONE, EPI_BIAS, EPI_RESIDUAL, EPI_SWIGLU = 0, 1, 2, 3


def w4a16_gemm_workspace_size(m: int, n: int) -> int:
    return int(lib().lmps_w4a16_gemm_workspace_size(m, n))


def w4a16_gemm(x, packed, scales, n: int, k: int, *, bias=None, residual=None, swiglu: bool = False, out=None,
               error: Optional[torch.Tensor] = None, workspace: Optional[torch.Tensor] = None):
    """tcgen05 W4A16 GEMM: out[m] = x[m] . W^T (+ bias | residual + fp16(.)).

    x is fp16 [m, k] (token-major); W the Q4 [n, k] layout.  Used where the
    projections of many tokens at once are dense contractions (prefill, large
    batches).  ``swiglu``: W's rows interleave gate and up rows and out[m, t] =
    SwiGLU(gate row t, up row t), n / 2 columns (interleave_rows builds W).
    Calls with m < 128 split K inside a thread-block cluster; ``workspace`` is
    accepted for API stability and unused."""
    x2, m = _x2d(x)
    y = out if out is not None else torch.empty(m, n // 2 if swiglu else n, dtype=FP16, device=x.device)
    epi, b_ptr, r_ptr, ldr = (EPI_SWIGLU if swiglu else EPI_NONE), None, None, 0
    if swiglu and (bias is not None or residual is not None):
        raise ValueError("the SwiGLU epilogue takes no bias or residual")
    if bias is not None:
        epi, b_ptr = EPI_BIAS, _dev(bias, "bias", FP16)
    if residual is not None:
        if bias is not None:
            raise ValueError("bias and residual epilogues are exclusive")
        r2 = residual if residual.dim() == 2 else residual.reshape(1, -1)
        epi, r_ptr, ldr = EPI_RESIDUAL, _dev(r2, "residual", FP16), r2.shape[1]
    err = error if error is not None else torch.zeros(1, dtype=torch.int32, device=x.device)
    ws_ptr, ws_bytes = None, 0
    if workspace is not None and workspace.numel() > 0:
        ws_ptr, ws_bytes = _dev(workspace, "workspace", torch.uint8), workspace.numel()
    call("lmps_w4a16_gemm", _dev(x2, "x", FP16), x2.shape[1], _dev(packed, "packed", torch.uint8),
         _dev(scales, "scales", FP16), b_ptr, r_ptr, ldr, _dev(y, "y", FP16), y.shape[-1], m, n, k, epi,
         _dev(err, "error", torch.int32), ws_ptr, ws_bytes, _stream())
    return y


def argmax_rows(logits, n: int, ids):
    """First-index argmax of each fp16 row of logits[:, :n] into int32 ids."""
    call("lmps_argmax_rows", _dev(logits, "logits", FP16), logits.shape[-1], logits.shape[0], n,
         _dev(ids, "ids", torch.int32), _stream())
    return ids


def sample_rows(logits, n: int, top_k: int, temperature: float, seed: int, offset: int, ids, ids2=None):
    """Top-k / temperature sample of each fp16 row of logits[:, :n] into int32
    ids (and ids2): seeded Philox draw, reproducible (see include/llamamps_b200.h)."""
    call("lmps_sample_rows", _dev(logits, "logits", FP16), logits.shape[-1], logits.shape[0], n, int(top_k),
         float(temperature), int(seed) & 0xFFFFFFFFFFFFFFFF, int(offset) & 0xFFFFFFFFFFFFFFFF,
         _dev(ids, "ids", torch.int32), _dev(ids2, "ids2", torch.int32) if ids2 is not None else None,
         _stream())
    return ids


def prefill_attention(q, k_pool, v_pool, block_table, out, batch: int, seq_len: int, page_size: int,
                      n_q_heads: int, n_kv_heads: int, head_dim: int, *, error: Optional[torch.Tensor] = None,
                      tcgen05: Optional[bool] = None):
    """Causal attention of every prompt position (q rows b*seq_len + p) over the paged cache.

    On the tcgen05 kernel (S and O in tensor memory, TMA-loaded K/V) where it
    takes the shape -- head_dim 128, page_size a multiple of 64, an even
    query-head group -- else on the mma.sync kernel; ``tcgen05`` forces one.
    ``error`` (int32 [1]) receives the tcgen05 kernel's wait-timeout flag."""
    fits = head_dim == 128 and page_size % 64 == 0 and (n_q_heads // n_kv_heads) % 2 == 0
    if tcgen05 is None:
        tcgen05 = fits
    if tcgen05:
        n_pages = k_pool.numel() // (n_kv_heads * page_size * head_dim)
        err = error if error is not None else torch.zeros(1, dtype=torch.int32, device=q.device)
        call("lmps_prefill_attention_tcgen05", _dev(q, "q", FP16), q.shape[-1], _dev(k_pool, "k_pool", FP16),
             _dev(v_pool, "v_pool", FP16), n_pages, _dev(block_table, "block_table", torch.int32),
             block_table.shape[1], page_size, _dev(out, "out", FP16), out.shape[-1], batch, seq_len, n_q_heads,
             n_kv_heads, head_dim, _dev(err, "error", torch.int32), _stream())
        return out
    call("lmps_prefill_attention", _dev(q, "q", FP16), q.shape[-1], _dev(k_pool, "k_pool", FP16),
         _dev(v_pool, "v_pool", FP16), _dev(block_table, "block_table", torch.int32), block_table.shape[1],
         page_size, _dev(out, "out", FP16), out.shape[-1], batch, seq_len, n_q_heads, n_kv_heads, head_dim,
         _stream())
    return out


# -- 4-bit KV cache -----------------------------------------------------------
Q4_ROW_BYTES = 72          # a cached row of 128 elements: 64 code bytes and 4 fp16 scales
Q4_ERR_TIMEOUT, Q4_ERR_PAGE, Q4_ERR_POSITION = 1, 2, 4
_U8, _I32, _F32 = torch.uint8, torch.int32, torch.float32


def raise_q4_error(bits: int) -> None:
    """RuntimeError for the Q4_ERR_* bits of a 4-bit cache kernel's error word (none: no error)."""
    if bits:
        names = [n for b, n in ((Q4_ERR_TIMEOUT, "a wait for the tensor core timed out"),
                                (Q4_ERR_PAGE, "a block table entry outside the pool"),
                                (Q4_ERR_POSITION, "a position outside the cache")) if bits & b]
        raise RuntimeError("4-bit KV cache: " + ", ".join(names))


def _q4_explain(dev: int, named) -> None:
    """Raises for the first of (name, tensor, dtype, elements) that is not on
    device ``dev`` (the first argument's), of this type, contiguous and of
    this many elements (at least, for a negative number)."""
    for name, t, dtype, n in named:
        if not t.is_cuda:
            raise RuntimeError(f"{name} must be a CUDA tensor (the decode path has no CPU fallback)")
        if t.get_device() != dev:
            raise ValueError(f"{name} is on another device than the call's other tensors")
        if t.dtype is not dtype:
            raise TypeError(f"{name}: expected {dtype}, got {t.dtype}")
        if not t.is_contiguous():
            raise ValueError(f"{name} must be contiguous")
        if t.numel() != n if n >= 0 else t.numel() < -n:
            raise ValueError(f"{name}: {t.numel()} elements, expected {abs(n)}")


def _q4_arg(t: torch.Tensor, name: str, dtype, dev: int, n: int) -> int:
    """Address of an argument after :func:`_q4_explain`'s checks (the attribute
    reads are most of an eager call's host time: 0.06 us each, 5 a tensor)."""
    m = t.numel()
    if t.dtype is dtype and t.get_device() == dev and dev >= 0 and (m == n or m >= -n > 0) and t.is_contiguous():
        return t.data_ptr()
    _q4_explain(dev, ((name, t, dtype, n),))
    raise RuntimeError(f"{name} must be a CUDA tensor")


def _q4_cache(k_pool, v_pool, block_table, dev: int, page_size: int, n_kv_heads: int, rows: int):
    """(k, v, n_pages, block_table, max_pages) of one layer's pools and a table of ``rows`` rows at least."""
    shape, table = k_pool.shape, block_table.shape
    if len(shape) != 3 or shape[1] != n_kv_heads or shape[2] != page_size * Q4_ROW_BYTES or v_pool.shape != shape:
        raise ValueError(f"pools: shapes {tuple(shape)} and {tuple(v_pool.shape)}, expected [n_pages, {n_kv_heads}, "
                         f"{page_size * Q4_ROW_BYTES}]")
    if len(table) != 2 or table[0] < rows:
        raise ValueError(f"block_table: shape {tuple(table)}, expected [{rows}, max_pages]")
    if not (k_pool.dtype is _U8 and v_pool.dtype is _U8 and block_table.dtype is _I32
            and k_pool.get_device() == v_pool.get_device() == block_table.get_device() == dev and dev >= 0
            and k_pool.is_contiguous() and v_pool.is_contiguous() and block_table.is_contiguous()):
        _q4_explain(dev, (("k_pool", k_pool, _U8, -1), ("v_pool", v_pool, _U8, -1),
                          ("block_table", block_table, _I32, -1)))
    return k_pool.data_ptr(), v_pool.data_ptr(), shape[0], block_table.data_ptr(), table[1]


def _q4_workspace(workspace, dev: int):
    if workspace is None:
        return None, 0
    n = workspace.numel()
    return (_q4_arg(workspace, "workspace", _U8, dev, n), n) if n else (None, 0)


def _q4_done(status, name: str) -> bool:
    """Whether the binding made the call (None: it found something to diagnose, and the call goes the checked
    way through ctypes)."""
    if status is None:
        return False
    if status:
        check(status, name)
    return True


def _q4_call(name: str, dev: int, *args) -> None:
    """The call on the current stream of the tensors' device."""
    if dev == torch._C._cuda_getDevice():
        status = getattr(lib(), name)(*args, torch._C._cuda_getCurrentRawStream(dev))
    else:
        with torch.cuda.device(dev):
            status = getattr(lib(), name)(*args, torch._C._cuda_getCurrentRawStream(dev))
    if status:
        check(status, name)


def rope_kv_append_q4(qkv, pos, inv_freq, q_out, k_pool, v_pool, block_table, page_size: int,
                      n_q_heads: int, n_kv_heads: int, head_dim: int, style: int = 0, *,
                      k_out: Optional[torch.Tensor] = None, v_out: Optional[torch.Tensor] = None,
                      error: Optional[torch.Tensor] = None):
    """rope_kv_append into the 4-bit cache: rotated q to ``q_out``, rotated K
    and V rows quantised to position ``pos[r]`` of the pages of row r of
    ``block_table``; ``k_out`` / ``v_out`` receive the values the cache then
    holds.  Rows with pos < 0 are skipped.  ``error`` (int32 [1]) collects
    Q4_ERR_PAGE / Q4_ERR_POSITION bits."""
    if _q4_done(binding().append(qkv, pos, inv_freq, q_out, k_pool, v_pool, block_table, page_size, n_q_heads,
                                 n_kv_heads, head_dim, style, k_out, v_out, error), "lmps_rope_kv_append_q4"):
        return q_out
    dev, rows = qkv.get_device(), qkv.shape[0]
    q_n, kv_n = rows * n_q_heads * head_dim, rows * n_kv_heads * head_dim
    a_qkv = _q4_arg(qkv, "qkv", FP16, dev, q_n + 2 * kv_n)
    cache = _q4_cache(k_pool, v_pool, block_table, dev, page_size, n_kv_heads, rows)
    _q4_call("lmps_rope_kv_append_q4", dev, a_qkv, _q4_arg(pos, "pos", _I32, dev, -rows),
             _q4_arg(inv_freq, "inv_freq", _F32, dev, head_dim // 2), _q4_arg(q_out, "q_out", FP16, dev, q_n),
             _q4_arg(k_out, "k_out", FP16, dev, kv_n) if k_out is not None else None,
             _q4_arg(v_out, "v_out", FP16, dev, kv_n) if v_out is not None else None, *cache,
             page_size, n_q_heads, n_kv_heads, head_dim, rows, style,
             _q4_arg(error, "error", _I32, dev, -1) if error is not None else None)
    return q_out


def attention_q4_splits(batch: int, n_kv_heads: int, max_seq_len: int) -> int:
    return int(lib().lmps_attention_q4_splits(batch, n_kv_heads, max_seq_len))


def attention_q4_launches(n_splits: int, max_seq_len: int) -> int:
    """Kernels of a decode attention call over the 4-bit cache: 1 unsplit or split within a thread-block
    cluster, 2 where pieces are merged by a second one."""
    return int(lib().lmps_attention_q4_launches(n_splits, max_seq_len))


def attention_q4_workspace_size(batch: int, n_q_heads: int, head_dim: int, n_splits: int) -> int:
    return int(lib().lmps_attention_q4_workspace_size(batch, n_q_heads, head_dim, n_splits))


def gqa_decode_attention_q4(q, k_pool, v_pool, block_table, seq_lens, out, workspace, page_size: int,
                            n_q_heads: int, n_kv_heads: int, head_dim: int, max_seq_len: int, n_splits: int, *,
                            error: Optional[torch.Tensor] = None):
    """gqa_decode_attention over the 4-bit cache: one query row per sequence
    over its first ``seq_lens[b]`` positions (0: zeros)."""
    if _q4_done(binding().decode(q, k_pool, v_pool, block_table, seq_lens, out, workspace, page_size, n_q_heads,
                                 n_kv_heads, head_dim, max_seq_len, n_splits, error), "lmps_gqa_decode_attention_q4"):
        return out
    dev, B = q.get_device(), q.shape[0]
    n = B * n_q_heads * head_dim
    a_q = _q4_arg(q, "q", FP16, dev, n)
    kp, vp, n_pages, bt, max_pages = _q4_cache(k_pool, v_pool, block_table, dev, page_size, n_kv_heads, B)
    ws, ws_bytes = _q4_workspace(workspace, dev)
    _q4_call("lmps_gqa_decode_attention_q4", dev, a_q, kp, vp, n_pages, bt,
             _q4_arg(seq_lens, "seq_lens", _I32, dev, -B), _q4_arg(out, "out", FP16, dev, n), ws, ws_bytes,
             max_pages, page_size, n_q_heads, n_kv_heads, head_dim, B, max_seq_len, n_splits,
             _q4_arg(error, "error", _I32, dev, -1) if error is not None else None)
    return out


def gqa_decode_attention_rope_q4(qkv, pos, inv_freq, k_pool, v_pool, block_table, seq_lens, out, workspace,
                                 page_size: int, n_q_heads: int, n_kv_heads: int, head_dim: int,
                                 max_seq_len: int, n_splits: int, style: int = 0, *,
                                 error: Optional[torch.Tensor] = None):
    """rope_kv_append_q4 + gqa_decode_attention_q4 in one call (seq_lens = pos + 1)."""
    if _q4_done(binding().step(qkv, pos, inv_freq, k_pool, v_pool, block_table, seq_lens, out, workspace, page_size,
                               n_q_heads, n_kv_heads, head_dim, max_seq_len, n_splits, style, error),
                "lmps_gqa_decode_attention_rope_q4"):
        return out
    dev, B = qkv.get_device(), qkv.shape[0]
    n = B * n_q_heads * head_dim
    a_qkv = _q4_arg(qkv, "qkv", FP16, dev, n + 2 * B * n_kv_heads * head_dim)
    kp, vp, n_pages, bt, max_pages = _q4_cache(k_pool, v_pool, block_table, dev, page_size, n_kv_heads, B)
    ws, ws_bytes = _q4_workspace(workspace, dev)
    _q4_call("lmps_gqa_decode_attention_rope_q4", dev, a_qkv, _q4_arg(pos, "pos", _I32, dev, -B),
             _q4_arg(inv_freq, "inv_freq", _F32, dev, head_dim // 2), style, kp, vp, n_pages, bt,
             _q4_arg(seq_lens, "seq_lens", _I32, dev, -B), _q4_arg(out, "out", FP16, dev, n), ws, ws_bytes,
             max_pages, page_size, n_q_heads, n_kv_heads, head_dim, B, max_seq_len, n_splits,
             _q4_arg(error, "error", _I32, dev, -1) if error is not None else None)
    return out


def prefill_q4_splits(batch: int, seq_len: int, n_q_heads: int, n_kv_heads: int, max_seq_len: int) -> int:
    return int(lib().lmps_prefill_q4_splits(batch, seq_len, n_q_heads, n_kv_heads, max_seq_len))


def prefill_q4_workspace_size(batch: int, seq_len: int, n_q_heads: int, head_dim: int, n_splits: int) -> int:
    return int(lib().lmps_prefill_q4_workspace_size(batch, seq_len, n_q_heads, head_dim, n_splits))


def prefill_attention_q4(q, k_pool, v_pool, block_table, out, batch: int, seq_len: int, page_size: int,
                         n_q_heads: int, n_kv_heads: int, head_dim: int, max_seq_len: int, *,
                         starts: Optional[torch.Tensor] = None, q_lens: Optional[torch.Tensor] = None,
                         workspace: Optional[torch.Tensor] = None, n_splits: int = 1,
                         error: Optional[torch.Tensor] = None):
    """Causal attention of many queries a sequence over the 4-bit cache: row
    b * seq_len + i of ``q`` is the query at position ``starts[b] + i`` (0 + i
    without ``starts``) for i < ``q_lens[b]`` (seq_len without); other rows of
    ``out`` stay as they were.  The K and V of all these positions are already
    in the cache; starts + q_lens <= ``max_seq_len``.  Without ``error`` the
    call waits for the kernel and raises what it reports (so a graph capture
    needs one)."""
    if error is None and q.is_cuda:
        if torch.cuda.is_current_stream_capturing():
            raise ValueError("error: a captured prefill_attention_q4 needs an int32 error word")
        error = torch.zeros(1, dtype=_I32, device=q.device)
        prefill_attention_q4(q, k_pool, v_pool, block_table, out, batch, seq_len, page_size, n_q_heads, n_kv_heads,
                             head_dim, max_seq_len, starts=starts, q_lens=q_lens, workspace=workspace,
                             n_splits=n_splits, error=error)
        raise_q4_error(int(error.item()))
        return out
    if _q4_done(binding().prefill(q, k_pool, v_pool, block_table, out, batch, seq_len, page_size, n_q_heads, n_kv_heads,
                                  head_dim, max_seq_len, starts, q_lens, workspace, n_splits, error),
                "lmps_prefill_attention_q4"):
        return out
    dev = q.get_device()
    n = batch * seq_len * n_q_heads * head_dim
    a_q = _q4_arg(q, "q", FP16, dev, n)
    kp, vp, n_pages, bt, max_pages = _q4_cache(k_pool, v_pool, block_table, dev, page_size, n_kv_heads, batch)
    ws, ws_bytes = _q4_workspace(workspace, dev)
    _q4_call("lmps_prefill_attention_q4", dev, a_q, kp, vp, n_pages, bt,
             _q4_arg(starts, "starts", _I32, dev, -batch) if starts is not None else None,
             _q4_arg(q_lens, "q_lens", _I32, dev, -batch) if q_lens is not None else None,
             _q4_arg(out, "out", FP16, dev, n), ws, ws_bytes, max_pages, page_size, n_q_heads, n_kv_heads,
             head_dim, batch, seq_len, max_seq_len, n_splits, _q4_arg(error, "error", _I32, dev, -1))
    return out


# -- 8-bit linear layers -------------------------------------------------------
_I8 = torch.int8


def _q8_arg(t: torch.Tensor, name: str, dtype, dev: int, rows: int, k: int):
    """Address and row stride of ``t`` as ``rows`` rows of ``k`` elements, or the error that says why it is none."""
    if not isinstance(t, torch.Tensor):
        raise TypeError(f"{name}: expected a tensor, got {type(t).__name__}")
    if not t.is_cuda:
        raise RuntimeError(f"{name} must be a CUDA tensor (the decode path has no CPU fallback)")
    if t.get_device() != dev:
        raise ValueError(f"{name} is on another device than the call's other tensors")
    if t.dtype != dtype:
        raise TypeError(f"{name}: expected {dtype}, got {t.dtype}")
    if tuple(t.shape) != (rows, k) and not (rows == 1 and tuple(t.shape) == (k,)):
        raise ValueError(f"{name}: shape {tuple(t.shape)}, expected [{rows}, {k}]")
    if k > 1 and t.stride(-1) != 1:
        raise ValueError(f"{name}: the elements of a row must be side by side")
    ld = t.stride(0) if rows > 1 else -(-k // 16) * 16
    if ld < k:
        raise ValueError(f"{name}: rows must not overlap (stride {ld} for {k} elements)")
    if max(ld, rows, k) > 0x7FFFFFFF:
        raise ValueError(f"{name}: {rows} rows of {k} elements, {ld} apart: more than 32 bits")
    return t.data_ptr(), ld


def _q8_vector(t: torch.Tensor, name: str, dtype, dev: int, n: int) -> int:
    if isinstance(t, torch.Tensor) and (t.numel() != n or not t.is_contiguous()):
        raise ValueError(f"{name}: expected {n} contiguous elements, got shape {tuple(t.shape)}")
    return _q8_arg(t.reshape(-1) if isinstance(t, torch.Tensor) else t, name, dtype, dev, 1, n)[0]


def _q8_shape(t: torch.Tensor, name: str):
    if not isinstance(t, torch.Tensor):
        raise TypeError(f"{name}: expected a tensor, got {type(t).__name__}")
    if t.dim() not in (1, 2) or t.shape[-1] == 0:
        raise ValueError(f"{name}: shape {tuple(t.shape)}, expected [rows, k] or [k]")
    return (1 if t.dim() == 1 else t.shape[0]), t.shape[-1]


def _q8_outputs(x: torch.Tensor, codes, scales):
    """Codes (rows start at multiples of 16 bytes) and scales for x's rows where they are not given."""
    rows, k = _q8_shape(x, "x")
    if codes is None:
        codes = torch.empty(rows, -(-k // 16) * 16, dtype=_I8, device=x.device)[:, :k]
        codes = codes if x.dim() == 2 else codes[0]
    return codes, torch.empty(rows, dtype=_F32, device=x.device) if scales is None else scales


def quantise_rows_q8(x, codes: Optional[torch.Tensor] = None, scales: Optional[torch.Tensor] = None, *,
                     values: Optional[torch.Tensor] = None):
    """Rows of fp16 ``x`` ([rows, k], or [k]; any row stride, k up to 2^30) as int8 codes in
    [-127, 127] and one fp32 scale each, max|row| / 127: (codes, scales).  A
    zero row has scale 0, a row with a NaN or an infinity scale NaN.  Without
    ``codes``, the result's rows start at multiples of 16 bytes, as
    :func:`w8a8_gemm` needs them.  ``values`` (fp16) receives code * scale."""
    if codes is None or scales is None:
        codes, scales = _q8_outputs(x, codes, scales)
    if _q4_done(binding_q8().quantise(x, codes, scales, values), "lmps_quantise_rows_q8"):
        return codes, scales
    rows, k = _q8_shape(x, "x")
    dev = x.get_device()
    a_x, ldx = _q8_arg(x, "x", FP16, dev, rows, k)
    a_c, ldc = _q8_arg(codes, "codes", _I8, dev, rows, k)
    a_v, ldv = _q8_arg(values, "values", FP16, dev, rows, k) if values is not None else (None, 0)
    a_s = _q8_vector(scales, "scales", _F32, dev, rows)
    if rows:
        _q4_call("lmps_quantise_rows_q8", dev, a_x, ldx, a_c, ldc, a_s, a_v, ldv, rows, k)
    return codes, scales


def rms_norm_q8(x, gamma, eps: float = 1e-6, *, residual: Optional[torch.Tensor] = None,
                sum_out: Optional[torch.Tensor] = None, codes: Optional[torch.Tensor] = None,
                scales: Optional[torch.Tensor] = None, values: Optional[torch.Tensor] = None):
    """:func:`rms_norm` with its output in 8 bits, as :func:`quantise_rows_q8`
    gives it (of the unrounded norm): (codes, scales).  With ``residual`` the
    norm is of s = fp16(residual + x), which ``sum_out`` receives: (codes,
    scales, sum).  ``sum_out`` may be ``residual`` or ``x`` itself.  A row's
    scale may differ in its last bits between calls of different size (the
    order of additions in its sum of squares), its codes do not."""
    if codes is None or scales is None:
        codes, scales = _q8_outputs(x, codes, scales)
    if residual is None:
        if sum_out is not None:
            raise ValueError("sum_out: only with a residual")
    elif sum_out is None:
        sum_out = torch.empty_like(x, memory_format=torch.contiguous_format)
    eps = float(eps)
    done = (codes, scales) if residual is None else (codes, scales, sum_out)
    if _q4_done(binding_q8().norm(x, gamma, eps, residual, sum_out, codes, scales, values), "lmps_rms_norm_q8"):
        return done
    rows, k = _q8_shape(x, "x")
    dev = x.get_device()
    a_x, ldx = _q8_arg(x, "x", FP16, dev, rows, k)
    a_g = _q8_vector(gamma, "gamma", FP16, dev, k)
    a_r, ldr = _q8_arg(residual, "residual", FP16, dev, rows, k) if residual is not None else (None, 0)
    a_o, lds = _q8_arg(sum_out, "sum_out", FP16, dev, rows, k) if residual is not None else (None, 0)
    a_c, ldc = _q8_arg(codes, "codes", _I8, dev, rows, k)
    a_v, ldv = _q8_arg(values, "values", FP16, dev, rows, k) if values is not None else (None, 0)
    a_s = _q8_vector(scales, "scales", _F32, dev, rows)
    if rows:
        _q4_call("lmps_rms_norm_q8", dev, a_x, ldx, a_r, ldr, a_o, lds, a_g, eps, a_c, ldc, a_s, a_v, ldv, rows, k)
    return done


def w8a8_gemm(codes, scales, w_codes, w_scales, *, bias: Optional[torch.Tensor] = None,
              residual: Optional[torch.Tensor] = None, swiglu: bool = False, out: Optional[torch.Tensor] = None,
              error: Optional[torch.Tensor] = None):
    """out[t] = scales[t] * w_scales * (w_codes . codes[t]) (+ bias) (+ residual[t]),
    rounded to fp16 once: int8 rows ([m, k], or [k]) with a scale for each
    token, weights [n, k] with a scale for each channel (both as
    :func:`quantise_rows_q8` makes them: rows at multiples of 16 bytes, k up to
    131071).  ``swiglu``: the n gate rows of ``w_codes`` are followed by n up
    rows, out[t] = silu(gate) * up, without bias or residual.  ``out`` may be
    ``residual``.  ``error`` (int32 [1]) is set to 1 if a wait on the device ran
    out; without it the call waits for the kernel and raises that (so a graph
    capture needs one)."""
    gated = 1 if swiglu else 0
    if out is not None and error is not None and _q4_done(
            binding_q8().gemm(codes, scales, w_codes, w_scales, bias, residual, gated, out, error), "lmps_w8a8_gemm"):
        return out
    m, k = _q8_shape(codes, "codes")
    w_rows, _ = _q8_shape(w_codes, "w_codes")
    if gated and w_rows % 2:
        raise ValueError(f"w_codes: {w_rows} rows, expected as many gate rows as up rows")
    if gated and (bias is not None or residual is not None):
        raise ValueError("the SwiGLU epilogue takes no bias or residual")
    n = w_rows // 2 if gated else w_rows
    if (out is None or error is None) and codes.is_cuda:
        word = error
        if out is None:
            out = torch.empty((m, n) if codes.dim() == 2 else (n,), dtype=FP16, device=codes.device)
        if error is None:
            if torch.cuda.is_current_stream_capturing():
                raise ValueError("error: a captured w8a8_gemm needs an int32 error word")
            word = torch.zeros(1, dtype=_I32, device=codes.device)
        w8a8_gemm(codes, scales, w_codes, w_scales, bias=bias, residual=residual, swiglu=swiglu, out=out, error=word)
        if error is None and int(word.item()):
            raise RuntimeError("w8a8_gemm: a wait for the tensor core timed out")
        return out
    dev = codes.get_device()
    a_x, ldx = _q8_arg(codes, "codes", _I8, dev, m, k)
    a_w, ldw = _q8_arg(w_codes, "w_codes", _I8, dev, w_rows, k)
    a_xs = _q8_vector(scales, "scales", _F32, dev, m)
    a_ws = _q8_vector(w_scales, "w_scales", _F32, dev, w_rows)
    a_b = _q8_vector(bias, "bias", FP16, dev, n) if bias is not None else None
    a_r, ldr = _q8_arg(residual, "residual", FP16, dev, m, n) if residual is not None else (None, 0)
    a_y, ldy = _q8_arg(out, "out", FP16, dev, m, n)
    a_e = _q8_vector(error, "error", _I32, dev, error.numel() if isinstance(error, torch.Tensor) else 1)
    for name, at, ld in (("codes", a_x, ldx), ("w_codes", a_w, ldw)):
        if at % 16 or ld % 16:
            raise ValueError(f"{name}: rows must start at multiples of 16 bytes")
    if m and n:
        _q4_call("lmps_w8a8_gemm", dev, a_x, ldx, a_xs, a_w, ldw, a_ws, a_b, a_r, ldr, a_y, ldy, m, n, k, gated, a_e)
    return out


# -- two-way tensor parallelism over peer memory ----------------------------
class PeerExchange:
    """This rank's exchange buffer and the peer's, mapped through CUDA IPC,
    for :func:`tp2_allreduce_residual` (``n_sites`` call sites of at most
    ``max_n`` fp16 elements).  ``handle()`` gives the 64 bytes to send to the
    peer, ``connect(peer_handle)`` maps the peer's buffer.  ``close()``
    unmaps and frees; call it on both ranks after a barrier, with no call in
    flight on either GPU."""

    def __init__(self, n_sites: int, max_n: int, device, wait_ns: int = 0):
        import ctypes
        self.n_sites, self.max_n, self.device = n_sites, max_n, torch.device(device)
        # limit of every wait for the peer, in GPU global-timer nanoseconds (0: 5 s)
        self.wait_ns = int(wait_ns)
        nbytes = lib().lmps_tp2_comm_bytes(n_sites, max_n)
        if nbytes == 0:
            raise ValueError("max_n must be a positive multiple of 8")
        with torch.cuda.device(self.device):
            p = ctypes.c_void_p()
            call("lmps_comm_alloc", nbytes, ctypes.byref(p))
            self.comm = p.value
            self.seen = torch.zeros(n_sites * 64, dtype=torch.int32, device=self.device)
        self.peer = None

    def handle(self) -> bytes:
        import ctypes
        buf = ctypes.create_string_buffer(64)
        with torch.cuda.device(self.device):
            call("lmps_ipc_handle", self.comm, buf)
        return buf.raw

    def connect(self, peer_handle: bytes) -> None:
        import ctypes
        if len(peer_handle) != 64:
            raise ValueError("an IPC handle is 64 bytes")
        p = ctypes.c_void_p()
        with torch.cuda.device(self.device):
            call("lmps_ipc_open", ctypes.create_string_buffer(peer_handle, 64), ctypes.byref(p))
        self.peer = p.value

    def close(self) -> None:
        with torch.cuda.device(self.device):
            if self.peer is not None:
                call("lmps_ipc_close", self.peer)
                self.peer = None
            if self.comm is not None:
                call("lmps_comm_free", self.comm)
                self.comm = None


def tp2_allreduce_residual(part, x, ex: PeerExchange, site: int, error):
    """x <- x + (part + the peer's part) through the peer's mapped buffer.
    A wait for the peer longer than ``ex.wait_ns`` sets ``error``."""
    if ex.peer is None:
        raise RuntimeError("the peer exchange is not connected")
    call("lmps_tp2_allreduce_residual", _dev(part, "part", FP16), _dev(x, "x", FP16), part.numel(), ex.comm,
         ex.peer, _dev(ex.seen, "seen", torch.int32), site, ex.n_sites, ex.max_n,
         _dev(error, "error", torch.int32), ex.wait_ns, _stream())
    return x


def tp2_argmax_exchange(logits, local_ids, row_offset: int, ids, ex: PeerExchange, site: int, error):
    """The global first-index argmax of a vocabulary split between two ranks:
    this rank's fp16 logits [B, ld] and local argmax ids in, the winner over
    both ranks' rows (global row numbers) out, on both ranks."""
    if ex.peer is None:
        raise RuntimeError("the peer exchange is not connected")
    B = local_ids.numel()
    call("lmps_tp2_argmax_exchange", _dev(logits, "logits", FP16), logits.shape[-1],
         _dev(local_ids, "local_ids", torch.int32), B, int(row_offset), _dev(ids, "ids", torch.int32), ex.comm,
         ex.peer, _dev(ex.seen, "seen", torch.int32), site, ex.n_sites, ex.max_n, _dev(error, "error", torch.int32),
         ex.wait_ns, _stream())
    return ids


def gemv_q4_tp2_residual(packed, scales, a, rows: int, k: int, x, part, ex: PeerExchange, site: int, error):
    """One kernel: part = W a (this rank's K slice, fp16), stored into the
    peer's receive slot over NVLink, then x <- x + (part + the peer's part)
    after a per-CTA hand-off with the peer's same CTA."""
    if ex.peer is None:
        raise RuntimeError("the peer exchange is not connected")
    a2, B = _x2d(a)
    call("lmps_gemv_q4_tp2_residual", _dev(packed, "packed", torch.uint8), _dev(scales, "scales", FP16),
         _dev(a2, "a", FP16), a2.shape[1], _dev(x, "x", FP16), _dev(part, "part", FP16), rows, k, B, ex.comm,
         ex.peer, _dev(ex.seen, "seen", torch.int32), site, ex.n_sites, ex.max_n,
         _dev(error, "error", torch.int32), ex.wait_ns, _stream())
    return x

