"""The path's kernels on caller-owned device tensors (torch is only the allocator here).

Each function forwards to one operator entry point of include/relay_b200.h on the current
CUDA stream of torch. Used by the parity tests and by bench.py at shapes the model-level
path does not reach; the backend (backend.py) calls the same kernels internally.
"""
from __future__ import annotations

import ctypes as C
from dataclasses import dataclass
from typing import Optional

import torch

from . import _lib
from ._lib import CAttnShape, CTokenMeta


def _p(t: Optional[torch.Tensor]):
    return None if t is None else C.c_void_p(t.data_ptr())


def _stream():
    return C.c_void_p(torch.cuda.current_stream().cuda_stream)


def _raw_stream(device: int) -> int:
    # the current stream's handle without building a torch.cuda.Stream for it (3 us a call)
    return torch._C._cuda_getCurrentRawStream(device)


def _dev_i32(a, device) -> torch.Tensor:
    return torch.as_tensor(a, dtype=torch.int32).to(device).contiguous()


@dataclass
class TokenMeta:
    """Device copies of the batch's position metadata (engine/src/cuda_kernels.cuh:16-26)."""

    pos: torch.Tensor
    seq: torch.Tensor
    table_off: torch.Tensor
    tables: torch.Tensor

    @staticmethod
    def from_host(pos, seq, table_off, tables, device="cuda") -> "TokenMeta":
        return TokenMeta(*(_dev_i32(a, device) for a in (pos, seq, table_off, tables)))

    def c(self) -> CTokenMeta:
        return CTokenMeta(self.pos.data_ptr(), self.seq.data_ptr(), self.table_off.data_ptr(), self.tables.data_ptr())


def attn_shape(heads, kv_heads, head_dim, block_size, q_stride=None, o_stride=None) -> CAttnShape:
    q_stride = (heads + 2 * kv_heads) * head_dim if q_stride is None else q_stride
    o_stride = heads * head_dim if o_stride is None else o_stride
    return CAttnShape(heads, kv_heads, head_dim, block_size, q_stride, o_stride)


def decode_scratch_bytes(shape: CAttnShape, n_decode: int, max_ctx: int) -> int:
    return _lib.lib().rb200_decode_scratch_bytes(C.byref(shape), n_decode, max_ctx)


def decode_plan(shape: CAttnShape, n_decode: int, max_ctx: int):
    """(keys per slice, slices per context, bytes of partial results) of such a decode launch."""
    sl, parts = C.c_int32(0), C.c_int32(0)
    nbytes = _lib.lib().rb200_decode_plan(C.byref(shape), n_decode, max_ctx, C.byref(sl), C.byref(parts))
    return sl.value, parts.value, nbytes


def decode_attention(shape: CAttnShape, q: torch.Tensor, meta: TokenMeta, decode_tokens: torch.Tensor, max_ctx: int,
                     k_pool: torch.Tensor, v_pool: torch.Tensor, out: torch.Tensor,
                     scratch: Optional[torch.Tensor] = None) -> torch.Tensor:
    n = decode_tokens.numel()
    if scratch is None:
        scratch = torch.empty(max(decode_scratch_bytes(shape, n, max_ctx), 16), dtype=torch.uint8, device=q.device)
    m = meta.c()
    _lib.check(_lib.lib().rb200_decode_attention(C.byref(shape), _p(q), C.byref(m), _p(decode_tokens), n, max_ctx,
                                                 _p(k_pool), _p(v_pool), _p(scratch), scratch.numel(), _p(out), _stream()))
    return out


def decode_attention_static(shape: CAttnShape, q, meta: TokenMeta, decode_tokens, max_ctx: int, k_pool, v_pool,
                            out) -> torch.Tensor:
    """decode_attention without caller scratch: the partial results go to the fixed buffer
    inside the library (at most _lib.STATIC_DECODE_SCRATCH_BYTES; larger batches raise
    ValueError). Allocates nothing; calls sharing a GPU must not overlap."""
    m = meta.c()
    _lib.check(_lib.lib().rb200_decode_attention_static(C.byref(shape), _p(q), C.byref(m), _p(decode_tokens),
                                                        decode_tokens.numel(), max_ctx, _p(k_pool), _p(v_pool), _p(out),
                                                        _stream()))
    return out


def _here(op: str, name: str, t: torch.Tensor) -> int:
    """The current CUDA device, which an operator's tensors have to be on; `t` is the first of them."""
    here = t.get_device()
    if here < 0 or here != torch._C._cuda_getDevice():
        raise ValueError(f"{op}: {name} must be on the current CUDA device, not on {t.device}")
    return here


def _plain(here: int, dtype: torch.dtype, *tensors) -> bool:
    """Whether each tensor has that type, is contiguous and lies on device `here`; None passes."""
    for t in tensors:
        if t is not None and (t.dtype is not dtype or t.get_device() != here or not t.is_contiguous()):
            return False
    return True


def _complain(op: str, here: int, *named) -> None:
    """Says what is wrong with the first (name, tensor, dtype, whole) that is not of that type on device `here`, with
    contiguous rows or, where `whole`, contiguous altogether."""
    for name, t, dtype, whole in named:
        if t is None:
            continue
        if t.dtype is not dtype:
            raise ValueError(f"{op}: {name} must be {dtype}, not {t.dtype}")
        if t.get_device() != here:
            raise ValueError(f"{op}: {name} must be on the current CUDA device {here}, not on {t.device}")
        if not t.is_contiguous() and (whole or t.dim() != 2 or (t.size(1) > 1 and t.stride(1) != 1)):
            raise ValueError(f"{op}: {name} must be contiguous" if whole else f"{op}: the rows of {name} must be contiguous")


def _check_meta(op: str, here: int, meta: TokenMeta, tokens: int) -> None:
    if not _plain(here, torch.int32, meta.pos, meta.seq, meta.table_off, meta.tables):
        _complain(op, here, *((name, getattr(meta, name), torch.int32, True) for name in ("pos", "seq", "table_off", "tables")))
    if meta.pos.numel() < tokens or meta.seq.numel() < tokens:
        raise ValueError(f"{op}: the metadata must have an entry for each token")


def _check_pools(op: str, here: int, page, k_pool, v_pool) -> None:
    if not _plain(here, torch.float16, k_pool, v_pool):
        _complain(op, here, ("k_pool", k_pool, torch.float16, True), ("v_pool", v_pool, torch.float16, True))
    dims = k_pool.shape
    if dims[1:] != page or v_pool.shape != dims:
        raise ValueError(f"{op}: the pools must be [blocks, kv_heads, block_size, head_dim] tensors")


def _row_stride(t: torch.Tensor) -> int:
    return t.size(1) if t.is_contiguous() else t.stride(0)


def _ptr(t: Optional[torch.Tensor]):
    return None if t is None else t.data_ptr()


def shared_prefix_scratch_bytes(shape: CAttnShape, n_decode: int, n_groups: int, max_prefix: int, max_suffix: int) -> int:
    return _lib.lib().rb200_shared_prefix_scratch_bytes(C.byref(shape), n_decode, n_groups, max_prefix, max_suffix)


def shared_prefix_attention(shape: CAttnShape, q: torch.Tensor, meta: TokenMeta, decode_tokens: torch.Tensor,
                            group_off: torch.Tensor, prefix_len: torch.Tensor, max_prefix: int, max_suffix: int,
                            k_pool: torch.Tensor, v_pool: torch.Tensor, out: torch.Tensor,
                            scratch: Optional[torch.Tensor] = None) -> torch.Tensor:
    """decode_attention for groups of sequences whose contexts begin with the same keys: entries
    group_off[g] .. group_off[g + 1] - 1 of decode_tokens share their first prefix_len[g] keys, which
    are read once for the group. max_prefix / max_suffix (the longest shared part, the most keys
    behind it) only decide how the work is split. A step captured as a graph passes its own scratch."""
    op = "shared_prefix_attention"
    here, n, n_groups, rows = _here(op, "q", q), decode_tokens.numel(), prefix_len.numel(), meta.pos.numel()
    if not (_plain(here, torch.int32, decode_tokens, group_off, prefix_len) and _plain(here, torch.float32, q) and
            _plain(here, torch.float16, out) and _plain(here, torch.uint8, scratch)):
        i32 = torch.int32
        _complain(op, here, ("decode_tokens", decode_tokens, i32, True), ("group_off", group_off, i32, True),
                  ("prefix_len", prefix_len, i32, True), ("q", q, torch.float32, False), ("out", out, torch.float16, False),
                  ("scratch", scratch, torch.uint8, True))
    _check_meta(op, here, meta, rows)
    _check_pools(op, here, (shape.kv_heads, shape.block_size, shape.head_dim), k_pool, v_pool)
    if group_off.numel() != n_groups + 1:
        raise ValueError(f"{op}: group_off must have one entry more than prefix_len")
    width = shape.heads * shape.head_dim
    dims = q.shape
    if len(dims) != 2 or dims[0] < rows or dims[1] < width or (rows > 1 and q.stride(0) != shape.q_stride):
        raise ValueError(f"{op}: q must have the batch's rows, {shape.q_stride} values apart")
    dims = out.shape
    if len(dims) != 2 or dims[0] < rows or dims[1] < width or (rows > 1 and out.stride(0) != shape.o_stride):
        raise ValueError(f"{op}: out must have the batch's rows, {shape.o_stride} values apart")
    L, sh, m = _lib.lib(), C.byref(shape), meta.c()
    if scratch is None:
        need = L.rb200_shared_prefix_scratch_bytes(sh, n, n_groups, max_prefix, max_suffix)
        scratch = torch.empty(need, dtype=torch.uint8, device=q.device) if need else None
    _lib.check(L.rb200_shared_prefix_attention(
        sh, q.data_ptr(), C.byref(m), decode_tokens.data_ptr(), n, group_off.data_ptr(), prefix_len.data_ptr(), n_groups, max_prefix,
        max_suffix, k_pool.data_ptr(), v_pool.data_ptr(), _ptr(scratch), 0 if scratch is None else scratch.numel(), out.data_ptr(),
        _raw_stream(here)))
    return out


def prefill_attention(shape: CAttnShape, q, meta: TokenMeta, tiles: torch.Tensor, k_pool, v_pool, out) -> torch.Tensor:
    m = meta.c()
    _lib.check(_lib.lib().rb200_prefill_attention(C.byref(shape), _p(q), C.byref(m), _p(tiles), tiles.numel() // 2,
                                                  _p(k_pool), _p(v_pool), _p(out), _stream()))
    return out


def reference_attention(shape: CAttnShape, q, meta: TokenMeta, n_tokens: int, k_pool, v_pool, out) -> torch.Tensor:
    m = meta.c()
    _lib.check(_lib.lib().rb200_reference_attention(C.byref(shape), _p(q), C.byref(m), n_tokens, _p(k_pool), _p(v_pool),
                                                    _p(out), _stream()))
    return out


def gemv_scratch(N: int, K: int, device="cuda") -> torch.Tensor:
    return torch.zeros(_lib.lib().rb200_gemv_scratch_bytes(N, K), dtype=torch.uint8, device=device)


def gemv_int8(wq, scale, x, y, beta=0.0, scratch=None) -> torch.Tensor:
    """y[T,N] (+)= scale * (wq[N,K] . x[T,K]); T <= 8."""
    N, K = wq.shape
    T = x.shape[0]
    scratch = gemv_scratch(N, K, wq.device) if scratch is None else scratch
    _lib.check(_lib.lib().rb200_gemv_int8(_p(wq), _p(scale), _p(x), _p(y), T, K, N, wq.stride(0), x.stride(0), beta,
                                          _p(scratch), scratch.numel(), _stream()))
    return y


def gemv_f16(w, x, y, beta=0.0, scratch=None) -> torch.Tensor:
    N, K = w.shape
    T = x.shape[0]
    scratch = gemv_scratch(N, K, w.device) if scratch is None else scratch
    _lib.check(_lib.lib().rb200_gemv_f16(_p(w), _p(x), _p(y), T, K, N, w.stride(0), x.stride(0), beta, _p(scratch),
                                         scratch.numel(), _stream()))
    return y


def gemm(w, x, y, beta=0.0, scale=None) -> torch.Tensor:
    """y[T,N] (+)= x[T,K] w[N,K]^T; w fp16, or int8 with per-row `scale`."""
    N, K = w.shape
    T = x.shape[0]
    i8 = w.dtype == torch.int8
    _lib.check(_lib.lib().rb200_gemm(None if i8 else _p(w), _p(w) if i8 else None, _p(scale), _p(x), _p(y), T, K, N,
                                     w.stride(0), x.stride(0), beta, _stream()))
    return y


def gemm_status() -> int:
    return _lib.lib().rb200_gemm_status()


def rmsnorm(x, w, out, eps, rows=None) -> torch.Tensor:
    R = out.shape[0]
    _lib.check(_lib.lib().rb200_rmsnorm(_p(x), _p(rows), _p(w), _p(out), R, x.shape[1], out.stride(0), eps, _stream()))
    return out


def embed(tokens, table, x) -> torch.Tensor:
    _lib.check(_lib.lib().rb200_embed(_p(tokens), _p(table), _p(x), tokens.numel(), x.shape[1], table.stride(0), _stream()))
    return x


def qkv_post(qkv, bias, inv_freq, meta: TokenMeta, k_pool, v_pool, heads, kv_heads, head_dim, block_size) -> None:
    m = meta.c()
    _lib.check(_lib.lib().rb200_qkv_post(_p(qkv), _p(bias), _p(inv_freq), C.byref(m), qkv.shape[0], _p(k_pool), _p(v_pool),
                                         heads, kv_heads, head_dim, block_size, _stream()))


def qkv_norm_post(qkv, bias, q_norm, k_norm, eps, inv_freq, meta: TokenMeta, q_out, k_pool, v_pool, heads, kv_heads, head_dim,
                  block_size, rot_dim=None) -> torch.Tensor:
    """qkv_post with an RMS norm over each query and key head (q_norm, k_norm [head_dim], or None) ahead of
    the rotation of its first rot_dim values (default: all): q to q_out (which may be qkv), k and v to
    their pages. A token with seq or pos below 0 is padding."""
    op, f32, rot = "qkv_norm_post", torch.float32, head_dim if rot_dim is None else rot_dim
    here = _here(op, "qkv", qkv)
    if not _plain(here, f32, qkv, bias, q_norm, k_norm, inv_freq, q_out):
        _complain(op, here, ("qkv", qkv, f32, False), ("bias", bias, f32, True), ("q_norm", q_norm, f32, True),
                  ("k_norm", k_norm, f32, True), ("inv_freq", inv_freq, f32, True), ("q_out", q_out, f32, False))
    width = (heads + 2 * kv_heads) * head_dim
    dims, q_dims = qkv.shape, q_out.shape
    if len(dims) != 2 or dims[1] < width:
        raise ValueError(f"{op}: qkv must be [tokens, (heads + 2 kv_heads) head_dim]")
    T = dims[0]
    if len(q_dims) != 2 or q_dims[0] < T or q_dims[1] < heads * head_dim:
        raise ValueError(f"{op}: q_out must be [tokens, heads head_dim]")
    _check_meta(op, here, meta, T)
    _check_pools(op, here, (kv_heads, block_size, head_dim), k_pool, v_pool)
    if bias is not None and bias.numel() != width:
        raise ValueError(f"{op}: bias must have {width} values")
    if (q_norm is not None and q_norm.numel() != head_dim) or (k_norm is not None and k_norm.numel() != head_dim):
        raise ValueError(f"{op}: q_norm and k_norm must have {head_dim} values")
    if inv_freq is not None and inv_freq.numel() != rot // 2:
        raise ValueError(f"{op}: inv_freq must have {rot // 2} values")
    m = meta.c()
    _lib.check(_lib.lib().rb200_qkv_norm_post(
        qkv.data_ptr(), _row_stride(qkv), _ptr(bias), _ptr(q_norm), _ptr(k_norm), eps, _ptr(inv_freq), rot, C.byref(m), T,
        q_out.data_ptr(), _row_stride(q_out), k_pool.data_ptr(), v_pool.data_ptr(), heads, kv_heads, head_dim, block_size,
        _raw_stream(here)))
    return q_out


def silu_mul(gu, act) -> torch.Tensor:
    T, I2 = gu.shape
    _lib.check(_lib.lib().rb200_silu_mul(_p(gu), _p(act), T, I2 // 2, act.stride(0), _stream()))
    return act


def f32_to_f16(x, out) -> torch.Tensor:
    _lib.check(_lib.lib().rb200_f32_to_f16(_p(x), _p(out), x.numel(), _stream()))
    return out


def kv_gather(k_pool, v_pool, blocks, block_bytes, staging) -> torch.Tensor:
    _lib.check(_lib.lib().rb200_kv_gather(_p(k_pool), _p(v_pool), _p(blocks), blocks.numel(), block_bytes, _p(staging),
                                          _stream()))
    return staging


def kv_scatter(k_pool, v_pool, blocks, block_bytes, staging) -> None:
    _lib.check(_lib.lib().rb200_kv_scatter(_p(k_pool), _p(v_pool), _p(blocks), blocks.numel(), block_bytes, _p(staging),
                                           _stream()))


def argmax_rows(logits, token_out, logit_out=None):
    R, V = logits.shape
    _lib.check(_lib.lib().rb200_argmax_rows(_p(logits), R, V, _p(token_out), _p(logit_out), _stream()))
    return token_out


def adjust_logits(logits, out, penalties=None, history=None, history_len=None, prompt_len=None, bias_ids=None, bias_values=None,
                  bias_len=None, mask=None) -> torch.Tensor:
    """What a request asks of its logits [R][V] ahead of the sampler, to `out` (which may be `logits`):
    penalties ([R][4] float32: repetition, presence, frequency, 0) by the row's first history_len tokens
    of history [R][.], of which the first prompt_len are the prompt; bias_values for the first bias_len
    of bias_ids [R][.], the last entry of a token counting; and a mask [R][ceil(V / 32)] of int32 words,
    whose 0 bits become -inf. Ids outside the vocabulary are passed over."""
    op, f32, i32 = "adjust_logits", torch.float32, torch.int32
    here = _here(op, "logits", logits)
    if not (_plain(here, f32, logits, out, penalties, bias_values) and
            _plain(here, i32, history, history_len, prompt_len, bias_ids, bias_len, mask)):
        _complain(op, here, ("logits", logits, f32, False), ("out", out, f32, False), ("penalties", penalties, f32, True),
                  ("history", history, i32, True), ("history_len", history_len, i32, True), ("prompt_len", prompt_len, i32, True),
                  ("bias_ids", bias_ids, i32, True), ("bias_values", bias_values, f32, True), ("bias_len", bias_len, i32, True),
                  ("mask", mask, i32, False))
    if logits.dim() != 2 or out.shape != logits.shape:
        raise ValueError(f"{op}: logits and out must both be [rows, vocabulary]")
    R, V = logits.shape
    if penalties is not None:
        if history is None or history_len is None or penalties.shape != (R, 4):
            raise ValueError(f"{op}: penalties must be [rows, 4] and need a history")
        if history.dim() != 2 or history.size(0) != R or history_len.numel() != R or (prompt_len is not None and prompt_len.numel() != R):
            raise ValueError(f"{op}: history must be [rows, tokens] with a length, and a prompt length, for each row")
    if bias_ids is not None:
        if bias_values is None or bias_len is None or bias_ids.shape != bias_values.shape:
            raise ValueError(f"{op}: bias_ids need values of the same shape and lengths")
        if bias_ids.dim() != 2 or bias_ids.size(0) != R or bias_len.numel() != R:
            raise ValueError(f"{op}: bias_ids must be [rows, entries] with a length for each row")
    if mask is not None and (mask.dim() != 2 or mask.size(0) != R or mask.size(1) * 32 < V):
        raise ValueError(f"{op}: mask must be [rows, ceil(vocabulary / 32)]")
    _lib.check(_lib.lib().rb200_adjust_logits(
        logits.data_ptr(), _row_stride(logits), out.data_ptr(), _row_stride(out), R, V, _ptr(penalties), _ptr(history),
        0 if penalties is None else history.size(1), _ptr(history_len), _ptr(prompt_len), _ptr(bias_ids), _ptr(bias_values),
        0 if bias_ids is None else bias_ids.size(1), _ptr(bias_len), _ptr(mask), 0 if mask is None else _row_stride(mask),
        _raw_stream(here)))
    return out


def sample_rows(logits, params: torch.Tensor, token_out, logprob_out=None):
    """The device sampler on logits [R][V]; `params`: a device uint8 tensor holding R
    rb200_sampling_params (32 bytes each); logprob_out: float64 [R] or None."""
    R, V = logits.shape
    _lib.check(_lib.lib().rb200_sample_rows(_p(logits), R, V, _p(params), _p(token_out), _p(logprob_out), _stream()))
    return token_out
