"""torch-facing wrappers over the sm_100a kernel library (``include/hds_b200.h``).

Every function takes CUDA tensors, launches on the current stream and returns immediately; there
is no hidden allocation unless an ``out=`` argument is omitted or the function's docstring says so. These wrappers are the ONLY way the
framework runs compute on the device — there is no eager-PyTorch fallback behind them (the fp32
PyTorch restatements used as test oracles live in :mod:`hcache_deepspeed_b200.ops.reference`).

Reference counterparts: the ``DSKernelBase`` callables under
``deepspeed/inference/v2/kernels/{core_ops,ragged_ops}/`` (e.g. ``core_ops/blas_kernels/blas.py``,
``ragged_ops/linear_blocked_kv_rotary/blocked_kv_rotary.py``).
"""
from __future__ import annotations

import contextlib
import ctypes
import functools
from typing import Optional, Sequence, Tuple

import torch

from . import native
from .plans import ADAPTER_FEW, MAX_SCALE, AdapterPlan, SharedPrefixPlan  # noqa: F401

ACT_IDENTITY, ACT_GELU, ACT_RELU, ACT_SILU, ACT_GELU_TANH, ACT_SWIGLU_CLAMPED, ACT_RELU2 = 0, 1, 2, 3, 4, 5, 6
ACT_CODES = {"identity": 0, None: 0, "gelu": 1, "relu": 2, "silu": 3, "gelu_tanh": 4, "gelu_new": 4,
             "gelu_pytorch_tanh": 4, "swish": 3, "swiglu_clamped": 5, "relu2": 6}

EPI_STORE, EPI_GATED, EPI_ACCUM = 0, 1, 2

#: counts launches of our own kernels (bench.py reports it as ``gpu_launches``)
launch_count = 0


def _dt(t: torch.Tensor) -> int:
    if t.dtype == torch.bfloat16:
        return 0
    if t.dtype == torch.float16:
        return 1
    raise TypeError(f"unsupported activation dtype {t.dtype}: the sm_100a kernels take bf16 or fp16")


def _dt3(t: torch.Tensor) -> int:
    """dtype code of the kernels that also take fp32."""
    return 2 if t.dtype == torch.float32 else _dt(t)


def _p(t: Optional[torch.Tensor]):
    return None if t is None else t.data_ptr()


def _stream() -> int:
    return torch.cuda.current_stream().cuda_stream


def _count(n: int = 1) -> None:
    global launch_count
    launch_count += n


def _check_2d(t: torch.Tensor, name: str) -> None:
    if t.dim() != 2 or t.stride(1) != 1:
        raise ValueError(f"{name} must be 2-D with a contiguous last dimension, got {tuple(t.shape)} / {t.stride()}")


class TiledWeight:
    """A weight matrix ``[N, K]`` stored pre-tiled for TMA: ``data[ceil(N/32), ceil(K/64), 32, 64]`` so that the
    32x64 block a GEMM tile needs per k-step is one contiguous 4 KB chunk (zero padded at the edges). Streaming a
    row-major weight fetches 128-byte segments 2*K bytes apart — poor DRAM page locality for decode-size GEMMs
    that are pure weight streaming; the tiled layout makes every fetch sequential."""

    def __init__(self, data: torch.Tensor, n: int, k: int):
        self.data, self.n, self.k = data, n, k

    @staticmethod
    def from_dense(w: torch.Tensor) -> "TiledWeight":
        n, k = w.shape
        np_, kp = -(-n // 32) * 32, -(-k // 64) * 64
        if (np_, kp) != (n, k):
            wp = w.new_zeros((np_, kp))
            wp[:n, :k] = w
            w = wp
        data = w.view(np_ // 32, 32, kp // 64, 64).permute(0, 2, 1, 3).contiguous()
        return TiledWeight(data, n, k)

    def to_dense(self) -> torch.Tensor:
        s, kb = self.data.shape[0], self.data.shape[1]
        return self.data.permute(0, 2, 1, 3).reshape(s * 32, kb * 64)[:self.n, :self.k]

    def rows_from(self, start: int) -> "TiledWeight":
        """Zero-copy view of rows ``[start, n)`` (start must be a multiple of 32)."""
        assert start % 32 == 0
        return TiledWeight(self.data[start // 32:], self.n - start, self.k)

    @property
    def shape(self):
        return (self.n, self.k)

    @property
    def dtype(self):
        return self.data.dtype

    @property
    def device(self):
        return self.data.device

    def data_ptr(self) -> int:
        return self.data.data_ptr()


def _w(w):
    """(pointer, ldw) of a weight operand: ldw = -1 marks the tiled layout for the C ABI."""
    if isinstance(w, TiledWeight):
        return w.data.data_ptr(), -1
    return w.data_ptr(), w.stride(0)


def gemm_splitk_workspace_bytes(M: int, N: int) -> int:
    return int(native.cuda_lib().hds_gemm_splitk_workspace_bytes(M, N))


def gemm(a: torch.Tensor, w: torch.Tensor, bias: Optional[torch.Tensor] = None, act: int = ACT_IDENTITY,
         gated: bool = False, out: Optional[torch.Tensor] = None, bn: int = 0, splits: int = 0,
         workspace: Optional[torch.Tensor] = None, limit: float = 0.0) -> torch.Tensor:
    """``out = epilogue(a @ w.T + bias)`` on the tcgen05 GEMM. ``gated``: interleaved (gate, up) columns.
    ``workspace`` (zero-initialised uint8 scratch): lets the token-major kernel split K for decode-size M; up to 64 tokens the
    feature-major one splits without (``splits=1``: none does). ``limit``: the bound of ``ACT_SWIGLU_CLAMPED``. fp32 operands take the plain fp32 kernel."""
    _check_2d(a, "a")
    M, K = a.shape
    N = w.shape[0]
    assert w.shape[1] == K and w.dtype == a.dtype
    wp, ldw = _w(w)
    n_out = N // 2 if gated else N
    if out is None:
        out = torch.empty((M, n_out), dtype=a.dtype, device=a.device)
    _check_2d(out, "out")
    if a.dtype == torch.float32:
        return _gemm_f32(a, w, out, EPI_GATED if gated else EPI_STORE, act, limit, bias=bias)
    lib = native.cuda_lib()
    if act == ACT_SWIGLU_CLAMPED:
        native.check(lib.hds_gemm_next_act_limit(limit), "hds_gemm_next_act_limit")
    rc = lib.hds_gemm(_p(a), a.stride(0), wp, ldw, M, N, K, _dt(a), EPI_GATED if gated else EPI_STORE,
                      act, _p(bias), _p(out), out.stride(0), bn, splits, _p(workspace),
                      0 if workspace is None else workspace.numel() * workspace.element_size(), _stream())
    native.check(rc, "hds_gemm")
    _count()
    return out


def _gemm_f32(a: torch.Tensor, w: torch.Tensor, out: torch.Tensor, epilogue: int, act: int, limit: float,
              group_off: Optional[torch.Tensor] = None, n_groups: int = 0, bias: Optional[torch.Tensor] = None) -> torch.Tensor:
    M, K = a.shape
    N = w.shape[0] // max(1, n_groups)
    assert w.dtype == torch.float32 and w.shape[1] == K and out.dtype == torch.float32
    rc = native.cuda_lib().hds_gemm_f32(_p(a), a.stride(0), _p(w), w.stride(0), M, N, K, epilogue, act, limit, _p(out), out.stride(0),
                                        _p(group_off), n_groups, _p(bias), _stream())
    native.check(rc, "hds_gemm_f32")
    _count()
    return out


def gemm_accum(a: torch.Tensor, w: torch.Tensor, accum: torch.Tensor, bias: Optional[torch.Tensor] = None,
               peer_ptrs: Optional[Sequence[int]] = None, multicast_ptr: Optional[int] = None, bn: int = 0,
               splits: int = 0) -> None:
    """``accum (fp32) += a @ w.T``. With ``peer_ptrs`` / ``multicast_ptr`` the epilogue adds its tile into every
    tensor-parallel rank's buffer (``red.sys`` / ``multimem.red``: the push form of GEMM -> all-reduce; the serving path
    uses the pull form — local accumulation, flag signal, reduction in :func:`norm_tp`)."""
    _check_2d(a, "a")
    M, K = a.shape
    N = w.shape[0]
    assert accum.dtype == torch.float32 and accum.stride(-1) == 1
    if a.dtype == torch.float32:
        assert peer_ptrs is None and multicast_ptr is None
        _gemm_f32(a, w, accum, EPI_ACCUM, ACT_IDENTITY, 0.0, bias=bias)
        return
    wp, ldw = _w(w)
    if multicast_ptr is not None:
        ptrs, mode = [multicast_ptr], 2
    elif peer_ptrs is not None:
        ptrs, mode = list(peer_ptrs), 1
    else:
        ptrs, mode = [accum.data_ptr()], 0
    arr = (ctypes.c_void_p * len(ptrs))(*ptrs)
    lib = native.cuda_lib()
    rc = lib.hds_gemm_accum(_p(a), a.stride(0), wp, ldw, M, N, K, _dt(a), _p(bias), arr, len(ptrs), mode,
                            accum.stride(0) if accum.dim() == 2 else N, bn, splits, _stream())
    native.check(rc, "hds_gemm_accum")
    _count()


def restore_kv_proj(latents: torch.Tensor, w_kv: torch.Tensor, kv_cache_layer: torch.Tensor, tok_pos: torch.Tensor,
                    tok_slot: torch.Tensor, inv_freq: Optional[torch.Tensor], n_kv_heads: int, head_dim: int,
                    block_size: int, bias_kv: Optional[torch.Tensor] = None) -> None:
    """HCache restore of one layer: K/V projection + RoPE + paged KV write in one tcgen05 kernel."""
    _check_2d(latents, "latents")
    T, H = latents.shape
    lib = native.cuda_lib()
    wp, ldw = _w(w_kv)
    rc = lib.hds_restore_kv_proj(_p(latents), latents.stride(0), wp, ldw, T, H, _dt(latents),
                                 _p(bias_kv), _p(kv_cache_layer), _p(tok_pos), _p(tok_slot), _p(inv_freq), n_kv_heads,
                                 head_dim, block_size, 0 if inv_freq is None else 1, _stream())
    native.check(rc, "hds_restore_kv_proj")
    _count()


def restore_kv_proj_peers(peer_ptrs: Sequence[int], rows_per_peer: int, T: int, H: int, dtype: torch.dtype, w_kv,
                          kv_cache_layer: torch.Tensor, tok_pos: torch.Tensor, tok_slot: torch.Tensor,
                          inv_freq: Optional[torch.Tensor], n_kv_heads: int, head_dim: int, block_size: int,
                          bias_kv: Optional[torch.Tensor] = None) -> None:
    """TP restore: latents row-sharded over peers' symmetric buffers, gathered by the kernel's TMA loads."""
    arr = (ctypes.c_void_p * len(peer_ptrs))(*peer_ptrs)
    wp, ldw = _w(w_kv)
    lib = native.cuda_lib()
    rc = lib.hds_restore_kv_proj_peers(arr, len(peer_ptrs), rows_per_peer, H, wp, ldw, T, H,
                                       0 if dtype == torch.bfloat16 else 1, _p(bias_kv), _p(kv_cache_layer), _p(tok_pos),
                                       _p(tok_slot), _p(inv_freq), n_kv_heads, head_dim, block_size,
                                       0 if inv_freq is None else 1, _stream())
    native.check(rc, "hds_restore_kv_proj_peers")
    _count()


def qkv_rope_proj(x: torch.Tensor, w_qkv: torch.Tensor, q_out: torch.Tensor, kv_cache_layer: torch.Tensor,
                  tok_pos: torch.Tensor, tok_slot: torch.Tensor, inv_freq: Optional[torch.Tensor], n_q_heads: int,
                  n_kv_heads: int, head_dim: int, block_size: int, bias_qkv: Optional[torch.Tensor] = None,
                  amp: Optional[torch.Tensor] = None) -> None:
    """Forward QKV projection with RoPE + KV-append fused into the GEMM epilogue. ``n_kv_heads`` = 0: queries alone, no pages.
    ``amp`` (like ``inv_freq``): factors of the rotated pairs."""
    _check_2d(x, "x")
    T, H = x.shape
    lib = native.cuda_lib()
    wp, ldw = _w(w_qkv)
    rc = lib.hds_qkv_rope_proj(_p(x), x.stride(0), wp, ldw, T, H, _dt(x), _p(bias_qkv), _p(q_out),
                               _p(kv_cache_layer), _p(tok_pos), _p(tok_slot), _p(inv_freq), _p(amp), n_q_heads, n_kv_heads,
                               head_dim, block_size, 0 if inv_freq is None else 1, _stream())
    native.check(rc, "hds_qkv_rope_proj")
    _count()


def norm(x: torch.Tensor, gamma: torch.Tensor, out: torch.Tensor, *, beta: Optional[torch.Tensor] = None,
         delta: Optional[torch.Tensor] = None, zero_delta: bool = False, res_out: Optional[torch.Tensor] = None,
         row_idx: Optional[torch.Tensor] = None, rows: Optional[int] = None, eps: float = 1e-5,
         layer_norm: bool = False, post_norm: bool = False, fp8: Optional[Tuple[torch.Tensor, torch.Tensor]] = None) -> torch.Tensor:
    """RMSNorm / LayerNorm with fused residual add (``delta`` may be the fp32 partial-sum buffer of
    :func:`gemm_accum`, which is consumed and optionally re-zeroed) and optional row gather. ``fp8``: (codes, scales) that get what
    :func:`quantize_fp8_rows` would make of ``out``."""
    cols = x.shape[-1]
    n = rows if rows is not None else (row_idx.numel() if row_idx is not None else x.numel() // cols)
    lib, dt, stream = native.cuda_lib(), _dt(x), _stream()
    if fp8 is not None:       # (last: what is armed has to meet its norm)
        q, scales = fp8
        assert q.dtype == torch.uint8 and scales.dtype == torch.float32 and q.shape == (n, cols) and scales.numel() >= n and scales.is_contiguous()
        native.check(lib.hds_norm_next_fp8(_p(q), q.stride(0), _p(scales)), "hds_norm_next_fp8")
    rc = lib.hds_norm(_p(x), x.stride(-2) if x.dim() > 1 else cols, _p(delta),
                      1 if (delta is not None and delta.dtype == torch.float32) else 0, 1 if zero_delta else 0,
                      _p(res_out), _p(out), out.stride(-2) if out.dim() > 1 else cols, _p(gamma), _p(beta), _p(row_idx),
                      n, cols, eps, 1 if layer_norm else 0, 1 if post_norm else 0, dt, stream)
    native.check(rc, "hds_norm")
    _count()
    return out


def _ptr_array(ptrs: Optional[Sequence[int]]):
    if ptrs is None:
        return None
    return (ctypes.c_void_p * len(ptrs))(*[int(p) for p in ptrs])


def norm_tp(ctx: int, x: torch.Tensor, gamma: torch.Tensor, out: torch.Tensor, src_ptrs: Sequence[int], *,
            src_mc: Optional[int] = None, partial_16bit: bool = False, zero_buf: Optional[torch.Tensor] = None,
            beta: Optional[torch.Tensor] = None, res_out: Optional[torch.Tensor] = None, out_ptrs: Optional[Sequence[int]] = None,
            out_mc: Optional[int] = None, row0: int = 0, n_rows: Optional[int] = None, wait: bool = True, signal: bool = False,
            eps: float = 1e-5, layer_norm: bool = False) -> torch.Tensor:
    """The collective after a row-parallel GEMM fused with residual add + norm (``hds_norm_tp``): all-reduce shape
    (``out_ptrs`` / ``out_mc`` unset: every rank reduces all rows) or reduce-scatter + all-gather shape (this rank reduces
    rows ``[row0, row0 + n_rows)`` and writes their normalised values into every rank's ``out``)."""
    cols = x.shape[-1]
    total = x.numel() // cols
    n = total if n_rows is None else n_rows
    lib = native.cuda_lib()
    rc = lib.hds_norm_tp(ctx, int(wait), int(signal), _p(x), x.stride(-2) if x.dim() > 1 else cols, _ptr_array(src_ptrs),
                         src_mc, int(partial_16bit), _p(zero_buf), _p(res_out), _p(out), out.stride(-2) if out.dim() > 1 else cols,
                         _ptr_array(out_ptrs), out_mc, row0, n, total, _p(gamma), _p(beta), cols, eps, 1 if layer_norm else 0,
                         _dt(x), _stream())
    native.check(rc, "hds_norm_tp")
    _count()
    return out


# ---- tensor-parallel flag protocol (tp_comm.cu) ------------------------------------------------------------------------
def tp_ctx_create(rank: int, n_ranks: int, pad_ptrs: Sequence[int]) -> int:
    ctx = native.cuda_lib().hds_tp_ctx_create(rank, n_ranks, _ptr_array(pad_ptrs))
    if ctx < 0:
        native.check(ctx, "hds_tp_ctx_create")
    return ctx


def tp_ctx_destroy(ctx: int) -> None:
    native.cuda_lib().hds_tp_ctx_destroy(ctx)


def tp_arm(ctx: int, wait: bool, signal: bool) -> None:
    """Attach a flag wait / signal to the NEXT GEMM-family kernel this thread launches (see ``hds_tp_arm``)."""
    native.check(native.cuda_lib().hds_tp_arm(ctx, int(wait), int(signal)), "hds_tp_arm")


def tp_disarm() -> bool:
    return bool(native.cuda_lib().hds_tp_disarm())


def tp_signal(ctx: int) -> None:
    native.check(native.cuda_lib().hds_tp_signal(ctx, _stream()), "hds_tp_signal")
    _count()


def tp_wait(ctx: int) -> None:
    native.check(native.cuda_lib().hds_tp_wait(ctx, _stream()), "hds_tp_wait")
    _count()


def tp_gather_cols(ctx: int, out: torch.Tensor, src_ptrs: Sequence[int], ld_src: int, col0: Sequence[int],
                   width: Sequence[int], rows: int, wait: bool = True) -> torch.Tensor:
    """``out[:rows, col0[p]:col0[p]+width[p]] = rank p's slice`` for every rank (vocabulary-sharded logits all-gather)."""
    n = len(src_ptrs)
    c0 = (ctypes.c_int32 * n)(*col0)
    wd = (ctypes.c_int32 * n)(*width)
    rc = native.cuda_lib().hds_tp_gather_cols(ctx, int(wait), _p(out), out.stride(0), _ptr_array(src_ptrs), ld_src, c0, wd, rows,
                                              out.element_size(), _stream())
    native.check(rc, "hds_tp_gather_cols")
    _count()
    return out


def rope_kv_append(qkv: torch.Tensor, q_out: torch.Tensor, kv_cache_layer: torch.Tensor, tok_pos: torch.Tensor,
                   tok_slot: torch.Tensor, inv_freq: Optional[torch.Tensor], n_q_heads: int, n_kv_heads: int,
                   head_dim: int, rotary_dim: int, block_size: int) -> None:
    _check_2d(qkv, "qkv")
    lib = native.cuda_lib()
    rc = lib.hds_rope_kv_append(_p(qkv), qkv.stride(0), _p(q_out), _p(kv_cache_layer), _p(tok_pos), _p(tok_slot),
                                _p(inv_freq), qkv.shape[0], n_q_heads, n_kv_heads, head_dim, rotary_dim, block_size,
                                0 if inv_freq is None else 1, _dt(qkv), _stream())
    native.check(rc, "hds_rope_kv_append")
    _count()


def embed(ids: torch.Tensor, weight: torch.Tensor, out: torch.Tensor, pos_weight: Optional[torch.Tensor] = None,
          tok_pos: Optional[torch.Tensor] = None, pos_offset: int = 0) -> torch.Tensor:
    assert ids.dtype == torch.int32
    lib = native.cuda_lib()
    rc = lib.hds_embed(_p(ids), _p(weight), _p(pos_weight), _p(tok_pos), pos_offset,
                       0 if pos_weight is None else pos_weight.shape[0], _p(out), ids.numel(), weight.shape[1],
                       weight.shape[0], _dt(weight), _stream())
    native.check(rc, "hds_embed")
    _count()
    return out


def gather_rows(x: torch.Tensor, row_idx: torch.Tensor, out: torch.Tensor) -> torch.Tensor:
    lib = native.cuda_lib()
    rc = lib.hds_gather_rows(_p(x), _p(row_idx), _p(out), row_idx.numel(), x.shape[-1] * x.element_size() // 2, _stream())
    native.check(rc, "hds_gather_rows")
    _count()
    return out


def argmax(logits: torch.Tensor, out_ids: Optional[torch.Tensor] = None) -> torch.Tensor:
    _check_2d(logits, "logits")
    if out_ids is None:
        out_ids = torch.empty((logits.shape[0],), dtype=torch.int32, device=logits.device)
    code = 2 if logits.dtype == torch.float32 else _dt(logits)
    lib = native.cuda_lib()
    rc = lib.hds_argmax(_p(logits), logits.stride(0), logits.shape[0], logits.shape[1], _p(out_ids), None, code,
                        _stream())
    native.check(rc, "hds_argmax")
    _count()
    return out_ids


def kv_blocks_copy(cache: torch.Tensor, staging: torch.Tensor, block_ids: torch.Tensor, to_staging: bool) -> None:
    """cache: [layers, blocks, 2, kvh, bs, d]; staging: [n_sel, layers, 2, kvh, bs, d]."""
    n_layers = cache.shape[0]
    block_bytes = cache[0, 0].numel() * cache.element_size()
    layer_stride = cache.stride(0) * cache.element_size()
    lib = native.cuda_lib()
    rc = lib.hds_kv_blocks_copy(_p(cache), _p(staging), _p(block_ids), block_ids.numel(), n_layers, block_bytes,
                                layer_stride, 1 if to_staging else 0, _stream())
    native.check(rc, "hds_kv_blocks_copy")
    _count()


def p2p_gather_rows(dst: torch.Tensor, peer_ptrs: Sequence[int], rows_per_peer: int, n_rows: int, my_rank: int) -> None:
    """Fill ``dst[:n_rows]`` rows owned by other TP ranks from their symmetric buffers (one launch, NVLink loads)."""
    arr = (ctypes.c_void_p * len(peer_ptrs))(*peer_ptrs)
    lib = native.cuda_lib()
    rc = lib.hds_p2p_gather_rows(_p(dst), arr, len(peer_ptrs), rows_per_peer, n_rows, dst.shape[-1] * dst.element_size(),
                                 my_rank, _stream())
    native.check(rc, "hds_p2p_gather_rows")
    _count()


def cvt_f32(src: torch.Tensor, dst: torch.Tensor, zero_src: bool = False) -> torch.Tensor:
    lib = native.cuda_lib()
    rc = lib.hds_cvt_f32(_p(src), _p(dst), src.numel(), 1 if zero_src else 0, _dt(dst), _stream())
    native.check(rc, "hds_cvt_f32")
    _count()
    return dst


def splitkv_workspace_bytes(n_items: int, n_q_heads: int, n_kv_heads: int, head_dim: int, max_splits: int,
                            rows_per_item: int) -> int:
    return int(native.cuda_lib().hds_paged_attention_splitkv_workspace_bytes(n_items, n_q_heads, n_kv_heads, head_dim,
                                                                             max_splits, rows_per_item))


def _arm_alibi(lib, alibi: Optional[torch.Tensor], n_q_heads: int, window: int = 0, keep_first: int = 0,
               out: Optional[torch.Tensor] = None, sink: Optional[torch.Tensor] = None, sigmoid_bias: Optional[torch.Tensor] = None,
               gate: Optional[torch.Tensor] = None, softcap: float = 0.0) -> None:
    """Options of the next attention launch of this thread, consumed by that launch: ALiBi slopes, sliding window and kept
    first tokens, the stride of ``out`` when its rows (``[T, n_q_heads * head_dim]``) are not dense, softmax sinks, the biases of
    sigmoid weights, the output gate, the bound of the scores."""
    if softcap:
        native.check(lib.hds_attention_next_softcap(float(softcap)), "hds_attention_next_softcap")
    for t, fn in ((sink, "hds_attention_next_sink"), (sigmoid_bias, "hds_attention_next_sigmoid")):
        if t is not None:
            assert t.dtype == torch.float32 and t.is_cuda and t.is_contiguous() and t.numel() == n_q_heads
            native.check(getattr(lib, fn)(_p(t)), fn)
    if gate is not None:
        _check_2d(gate, "gate")
        native.check(lib.hds_attention_next_gate(_p(gate), gate.stride(0)), "hds_attention_next_gate")
    if keep_first:
        native.check(lib.hds_attention_next_keep_first(int(keep_first)), "hds_attention_next_keep_first")
    if out is not None and out.dim() == 2 and out.stride(0) != out.shape[1]:
        native.check(lib.hds_attention_next_out_stride(out.stride(0)), "hds_attention_next_out_stride")
    if window:
        native.check(lib.hds_attention_next_window(int(window)), "hds_attention_next_window")
    if alibi is None:
        return
    assert alibi.dtype == torch.float32 and alibi.is_cuda and alibi.is_contiguous() and alibi.numel() == n_q_heads
    native.check(lib.hds_attention_next_alibi(_p(alibi)), "hds_attention_next_alibi")


def paged_attention_splitkv(q: torch.Tensor, out: torch.Tensor, kv_cache_layer: torch.Tensor,
                            block_tables: torch.Tensor, items: torch.Tensor, n_items: int, rows_per_item: int,
                            n_q_heads: int, n_kv_heads: int, head_dim: int, block_size: int, n_splits: int,
                            scale: float, workspace: Optional[torch.Tensor], alibi: Optional[torch.Tensor] = None,
                            window: int = 0, keep_first: int = 0, sink: Optional[torch.Tensor] = None,
                            sigmoid_bias: Optional[torch.Tensor] = None, gate: Optional[torch.Tensor] = None, softcap: float = 0.0,
                            grouped: bool = False) -> None:
    """kv_cache_layer: [blocks, 2, kvh, bs, d]; items: int32 [n, 4] = (seq, q_row0, n_q, pos0). ``alibi``: fp32 [n_q_heads]
    slopes; score += slope * (key position - query position). ``window``: sliding-window attention, keys (p - window, p] and
    the first ``keep_first`` ones. ``sink``, ``sigmoid_bias`` (fp32 [n_q_heads]) and ``gate`` (rows like ``out``'s): see
    ``hds_attention_next_sink``. ``grouped``: the kernel for query heads that share their keys (``hds_paged_attention_group``)."""
    lib = native.cuda_lib()
    _arm_alibi(lib, alibi, n_q_heads, window, keep_first, out, sink, sigmoid_bias, gate, softcap)
    fn = lib.hds_paged_attention_group if grouped else lib.hds_paged_attention_splitkv
    rc = fn(_p(q), _p(out), _p(kv_cache_layer), kv_cache_layer.shape[0], _p(block_tables), block_tables.stride(0), _p(items), n_items,
            rows_per_item, n_q_heads, n_kv_heads, head_dim, block_size, n_splits, scale, _p(workspace),
            0 if workspace is None else workspace.numel() * workspace.element_size(), _dt(q), _stream())
    native.check(rc, "hds_paged_attention_splitkv")
    _count()


def prefill_workspace_bytes(n_items: int, n_q_heads: int, head_dim: int, n_splits: int) -> int:
    return int(native.cuda_lib().hds_paged_attention_prefill_workspace_bytes(n_items, n_q_heads, head_dim, n_splits))


def paged_attention_prefill(q: torch.Tensor, out: torch.Tensor, kv_cache_layer: torch.Tensor,
                            block_tables: torch.Tensor, items: torch.Tensor, n_items: int, n_q_heads: int,
                            n_kv_heads: int, head_dim: int, block_size: int, scale: float, n_splits: int = 1,
                            workspace: Optional[torch.Tensor] = None, packed: bool = False,
                            alibi: Optional[torch.Tensor] = None, window: int = 0, keep_first: int = 0, sink: Optional[torch.Tensor] = None,
                            sigmoid_bias: Optional[torch.Tensor] = None, gate: Optional[torch.Tensor] = None, softcap: float = 0.0) -> None:
    """tcgen05 paged attention. ``packed``: grouped-query decode form — one CTA per (item, KV head) whose MMA rows are
    the group's (token, query head) pairs (``hds_paged_attention_packed``). ``alibi``: fp32 [n_q_heads] slopes;
    ``window``: sliding-window attention."""
    lib = native.cuda_lib()
    _arm_alibi(lib, alibi, n_q_heads, window, keep_first, out, sink, sigmoid_bias, gate, softcap)
    fn = lib.hds_paged_attention_packed if packed else lib.hds_paged_attention_prefill
    rc = fn(_p(q), _p(out), _p(kv_cache_layer), kv_cache_layer.shape[0], _p(block_tables),
                                         block_tables.stride(0), _p(items), n_items, q.shape[0], n_q_heads, n_kv_heads,
                                         head_dim, block_size, scale, n_splits, _p(workspace),
                                         0 if workspace is None else workspace.numel() * workspace.element_size(),
                                         _dt(q), _stream())
    native.check(rc, "hds_paged_attention_prefill")
    _count()


# ------------------------------------------------------------------------------------------------
# mixture of experts (ref: ragged_ops/top_k_gating, moe_scatter, moe_gather, cutlass_ops/moe_gemm)
# ------------------------------------------------------------------------------------------------
#: most (token, expert) choices of a step whose expert GEMMs stream weights feature-major, 64 rows being the widest token tile
MOE_FEW = 64


def _moe_few(choices: int, K: int, gated: bool) -> bool:
    """The token tile has room for all choices at one expert. Gated, and more than 32 wide, its epilogue costs more than a short weight row
    saves: 64 choices of 64 experts of 2816 x 1024 55.1 us token-major and 66.0 feature-major, 128 of 1536 x 768 36.2 and 43.7, 16 of 2816 x
    2048 46.1 and 47.2; 64 of 7168 x 4096 486 and 428. Plain ones gain at all sizes (64 of 2048 x 1408 56.5 and 55.5)."""
    return 0 < choices <= MOE_FEW and (not gated or choices <= 32 or K >= 4096)


def moe_padded_rows(n_tokens: int, n_experts: int, top_k: int) -> int:
    """Row capacity of the scattered activation buffer (each expert's range is padded to 128 rows)."""
    return int(native.cuda_lib().hds_moe_padded_rows(n_tokens, n_experts, top_k))


def moe_topk_gating(logits: torch.Tensor, top_k: int, normalize: bool, scores: torch.Tensor, expert_ids: torch.Tensor,
                    offsets: torch.Tensor, counts: torch.Tensor, bias: Optional[torch.Tensor] = None, scale: float = 1.0,
                    clear: bool = False, sigmoid: bool = False, biased: bool = False) -> None:
    """Softmax (or ``sigmoid``) + top-k per token; ``counts`` (int32 [E], zero on entry) is incremented per assignment. ``bias`` (fp32 [E]) is added
    to the scores that choose (``biased``: to the logits, which choose), ``scale`` multiplies the scores returned, ``clear`` zeroes (fp32) logits once read."""
    T, E = logits.shape
    code = 2 if logits.dtype == torch.float32 else _dt(logits)
    rc = native.cuda_lib().hds_moe_topk_gating(_p(logits), logits.stride(0), T, E, top_k, int(normalize), 2 if biased else int(sigmoid), _p(bias), scale,
                                                 int(clear), code, _p(scores),
                                               _p(expert_ids), _p(offsets), _p(counts), _stream())
    native.check(rc, "hds_moe_topk_gating")
    _count()


def moe_scatter(x: torch.Tensor, xs: torch.Tensor, expert_ids: torch.Tensor, offsets: torch.Tensor, counts: torch.Tensor,
                pad_off: torch.Tensor, mapped_slots: torch.Tensor, top_k: int, scores: Optional[torch.Tensor] = None) -> None:
    """Build ``pad_off`` (int32 [E+1]) from ``counts`` (re-zeroed) and copy every token row, times its ``scores`` if given, to its k
    expert rows."""
    T, H = x.shape
    E = counts.numel()
    r = x.element_size() // 2      # the kernel moves 16-bit units
    H *= r
    rc = native.cuda_lib().hds_moe_scatter(_p(x), x.stride(0) * r, _p(xs), xs.stride(0) * r, _p(expert_ids), _p(offsets), _p(counts),
                                           _p(pad_off), _p(mapped_slots), T, E, top_k, H, _p(scores), _dt3(x), _stream())
    native.check(rc, "hds_moe_scatter")
    _count(2)


def moe_gemm(a: torch.Tensor, w_stacked: torch.Tensor, pad_off: torch.Tensor, n_experts: int, out: torch.Tensor,
             act: int = ACT_IDENTITY, gated: bool = False, limit: float = 0.0, choices: int = 0) -> torch.Tensor:
    """Grouped GEMM: rows of ``a`` in expert e's range times ``w_stacked[e*N:(e+1)*N]``ᵀ (``w_stacked``: [E*N, K]). ``choices`` (0: not
    known): how many rows live in all; few of them take the kernel that streams the weights."""
    _check_2d(a, "a")
    _check_2d(out, "out")
    rows, K = a.shape
    N = w_stacked.shape[0] // n_experts
    assert w_stacked.shape[1] == K and rows % 128 == 0 and out.shape[0] >= rows
    if a.dtype == torch.float32:
        return _gemm_f32(a, w_stacked, out, EPI_GATED if gated else EPI_STORE, act, limit, pad_off, n_experts)
    if act == ACT_SWIGLU_CLAMPED:
        native.check(native.cuda_lib().hds_gemm_next_act_limit(limit), "hds_gemm_next_act_limit")
    if _moe_few(choices, K, gated):
        rc = native.cuda_lib().hds_moe_gemm_few(_p(a), a.stride(0), _p(w_stacked), w_stacked.stride(0), _p(pad_off), n_experts, choices,
                                                choices, rows, N, K, _dt(a), EPI_GATED if gated else EPI_STORE, act, _p(out),
                                                out.stride(0), _stream())
        native.check(rc, "hds_moe_gemm_few")
        _count()
        return out
    rc = native.cuda_lib().hds_moe_gemm(_p(a), a.stride(0), _p(w_stacked), w_stacked.stride(0), _p(pad_off), n_experts, rows,
                                        N, K, _dt(a), EPI_GATED if gated else EPI_STORE, act, _p(out), out.stride(0),
                                        _stream())
    native.check(rc, "hds_moe_gemm")
    _count()
    return out


def gemm_2sm(a: torch.Tensor, w: torch.Tensor, out: Optional[torch.Tensor] = None, bias: Optional[torch.Tensor] = None,
             act: int = ACT_IDENTITY, gated: bool = False, bn: int = 0) -> torch.Tensor:
    """``out = epilogue(a @ w.T + bias)`` on the CTA-pair kernel (``tcgen05.mma.cta_group::2``: two SMs per 256 x bn tile)."""
    _check_2d(a, "a")
    _check_2d(w, "w")
    M, K = a.shape
    N = w.shape[0]
    if out is None:
        out = torch.empty(M, N // 2 if gated else N, dtype=a.dtype, device=a.device)
    rc = native.cuda_lib().hds_gemm_2sm(_p(a), a.stride(0), _p(w), w.stride(0), M, N, K, _dt(a),
                                        EPI_GATED if gated else EPI_STORE, act, _p(bias), _p(out), out.stride(0), bn, _stream())
    native.check(rc, "hds_gemm_2sm")
    _count()
    return out


def quantize_fp8_rows(x: torch.Tensor, q: Optional[torch.Tensor] = None,
                      scales: Optional[torch.Tensor] = None) -> Tuple[torch.Tensor, torch.Tensor]:
    """Row-wise E4M3 quantisation: ``q[r] = e4m3(x[r] / scales[r])`` with ``scales[r] = amax(x[r]) / 448``.
    Rows are tokens for activations and output channels for weights. ``q`` is ``uint8`` storage of the fp8 codes."""
    _check_2d(x, "x")
    rows, K = x.shape
    if q is None:
        q = torch.empty(rows, K, dtype=torch.uint8, device=x.device)
    if scales is None:
        scales = torch.empty(rows, dtype=torch.float32, device=x.device)
    rc = native.cuda_lib().hds_quantize_fp8_rows(_p(x), x.stride(0), rows, K, _dt(x), _p(q), q.stride(0), _p(scales),
                                                 _stream())
    native.check(rc, "hds_quantize_fp8_rows")
    _count()
    return q, scales


def gemm_fp8(aq: torch.Tensor, a_scale: torch.Tensor, wq: torch.Tensor, w_scale: torch.Tensor, out: torch.Tensor,
             bias: Optional[torch.Tensor] = None, act: int = ACT_IDENTITY, gated: bool = False, bn: int = 0,
             workspace: Optional[torch.Tensor] = None, splits: int = 0, w_fmt: int = 0) -> torch.Tensor:
    """``out = epilogue((aq @ wq.T) * a_scale[:, None] * w_scale[None, :] + bias)`` with E4M3 operands on
    ``tcgen05.mma.kind::f8f6f4`` (fp32 accumulation in TMEM). ``aq``: [M, K] uint8, ``wq``: [N, K] uint8.
    M <= 64 with ``bn == 0`` takes the feature-major weight-streaming kernel, which splits K for a caller that gives a ``workspace`` of
    at least :func:`gemm_fp8_skinny_workspace_bytes` (it is not written: the parts meet in a cluster)."""
    _check_2d(aq, "aq")
    _check_2d(wq, "wq")
    _check_2d(out, "out")
    M, K = aq.shape
    N = wq.shape[0]
    # w_fmt 1: E3M2 (FP6) weights packed 6 bits each — [N, 3K/4] bytes, unpacked by the TMA on the way to shared memory
    assert wq.shape[1] == (K * 3 // 4 if w_fmt == 1 else K) and aq.dtype == torch.uint8 and wq.dtype == torch.uint8
    assert a_scale.dtype == torch.float32 and w_scale.dtype == torch.float32
    lib = native.cuda_lib()
    if w_fmt:
        native.check(lib.hds_fp8_next_weight_format(w_fmt), "hds_fp8_next_weight_format")
    if M <= 64 and bn == 0:
        rc = lib.hds_gemm_fp8_skinny(_p(aq), aq.stride(0), _p(a_scale), _p(wq), wq.stride(0), _p(w_scale), M, N, K, _dt(out),
                                     EPI_GATED if gated else EPI_STORE, act, _p(bias), _p(out), out.stride(0), None, 0,
                                     _p(workspace), 0 if workspace is None else workspace.numel(), splits, _stream())
        native.check(rc, "hds_gemm_fp8_skinny")
    else:
        rc = lib.hds_gemm_fp8(_p(aq), aq.stride(0), _p(a_scale), _p(wq), wq.stride(0), _p(w_scale), M, N, K, _dt(out),
                              EPI_GATED if gated else EPI_STORE, act, _p(bias), _p(out), out.stride(0), bn, _stream())
        native.check(rc, "hds_gemm_fp8")
    _count()
    return out


def gemm_fp8_skinny_workspace_bytes(M: int, N: int) -> int:
    nt = 16 if M <= 16 else 32 if M <= 32 else 64
    n_tiles = (N + 127) // 128
    return ((n_tiles * 128 * nt * 4 + 255) & ~255) + n_tiles * 16


def gemm_fp8_accum(aq: torch.Tensor, a_scale: torch.Tensor, wq: torch.Tensor, w_scale: torch.Tensor, accum: torch.Tensor,
                   bias: Optional[torch.Tensor] = None, out_dtype: torch.dtype = torch.bfloat16, splits: int = 0,
                   w_fmt: int = 0) -> torch.Tensor:
    """``accum (fp32) += (aq @ wq.T) * scales (+ bias once)`` for M <= 64 (decode): split-K partial sums go straight
    into ``accum`` with fp32 atomics, no scratch."""
    M, K = aq.shape
    N = wq.shape[0]
    assert accum.dtype == torch.float32 and M <= 64
    dt = 0 if out_dtype == torch.bfloat16 else 1
    if w_fmt:
        native.check(native.cuda_lib().hds_fp8_next_weight_format(w_fmt), "hds_fp8_next_weight_format")
    rc = native.cuda_lib().hds_gemm_fp8_skinny(_p(aq), aq.stride(0), _p(a_scale), _p(wq), wq.stride(0), _p(w_scale), M, N, K, dt,
                                               2, ACT_IDENTITY, _p(bias), None, 0, _p(accum), accum.stride(0), None, 0, splits,
                                               _stream())
    native.check(rc, "hds_gemm_fp8_skinny")
    _count()
    return accum


def moe_gather(y: torch.Tensor, mapped_slots: torch.Tensor, scores: torch.Tensor, out: torch.Tensor) -> None:
    """``out[t] += sum_j scores[t, j] * y[mapped_slots[t, j]]`` (``out`` fp32)."""
    T, k = mapped_slots.shape
    assert out.dtype == torch.float32
    rc = native.cuda_lib().hds_moe_gather(_p(y), y.stride(0), _p(mapped_slots), _p(scores), _p(out), out.stride(0), T, k,
                                          y.shape[1], _dt(y), _stream())
    native.check(rc, "hds_moe_gather")
    _count()


def moe_gather_shared(y: torch.Tensor, mapped_slots: torch.Tensor, scores: torch.Tensor, x: torch.Tensor, w_gate: torch.Tensor,
                      ys: torch.Tensor, out: torch.Tensor) -> None:
    """``moe_gather`` and a shared expert: ``out[t] += ... + sigmoid(x[t] . w_gate) * ys[t]`` (``out`` fp32, ``w_gate`` [1, H])."""
    T, k = mapped_slots.shape
    H = y.shape[1]
    assert out.dtype == torch.float32 and x.dtype == w_gate.dtype == ys.dtype == y.dtype
    assert x.shape == (T, H) and ys.shape == (T, H) and w_gate.numel() == H and w_gate.is_contiguous()
    rc = native.cuda_lib().hds_moe_gather_shared(_p(y), y.stride(0), _p(mapped_slots), _p(scores), _p(x), x.stride(0), _p(w_gate), _p(ys),
                                                 ys.stride(0), _p(out), out.stride(0), T, k, H, _dt(y), _stream())
    native.check(rc, "hds_moe_gather_shared")
    _count()


# ------------------------------------------------------------------------------------------------
# expert choice by table, fp32 residual stream, state-space mixers, generic attention
# ------------------------------------------------------------------------------------------------
def moe_table_route(ids: torch.Tensor, table: torch.Tensor, n_experts: int, scores: torch.Tensor, expert_ids: torch.Tensor,
                    offsets: torch.Tensor, counts: torch.Tensor) -> None:
    """Experts of every token from ``table`` (int32 [vocab, top]) with equal weights; ``counts`` as in moe_topk_gating."""
    assert ids.dtype == torch.int32 and table.dtype == torch.int32
    rc = native.cuda_lib().hds_moe_table_route(_p(ids), _p(table), table.shape[0], ids.numel(), n_experts, table.shape[1], _p(scores),
                                               _p(expert_ids), _p(offsets), _p(counts), _stream())
    native.check(rc, "hds_moe_table_route")
    _count()


def moe_combine(y: torch.Tensor, mapped_slots: torch.Tensor, scores: Optional[torch.Tensor], base: Optional[torch.Tensor],
                out: torch.Tensor) -> torch.Tensor:
    """``out[t] = base[t] + sum_j scores[t, j] * y[mapped_slots[t, j]]`` (``out`` fp32, stored; ``base`` optional, or ``out``
    itself: added in place; ``scores`` None: ones)."""
    T, k = mapped_slots.shape
    assert out.dtype == torch.float32
    accumulate = base is not None and base.data_ptr() == out.data_ptr()
    if accumulate:
        base = None
    assert base is None or base.dtype == y.dtype
    rc = native.cuda_lib().hds_moe_combine(_p(y), y.stride(0), _p(mapped_slots), _p(scores), _p(base),
                                           0 if base is None else base.stride(0), _p(out), out.stride(0), T, k, y.shape[1],
                                             int(accumulate), _dt3(y), _stream())
    native.check(rc, "hds_moe_combine")
    _count()
    return out


def embed_f32(ids: torch.Tensor, weight: torch.Tensor, out: torch.Tensor, gamma: Optional[torch.Tensor] = None,
              cols: Optional[int] = None, eps: float = 1e-5, scale: float = 1.0) -> torch.Tensor:
    """Embedding rows in fp32, times ``scale``; with ``gamma`` RMS-normed over their first ``cols`` values and weighted instead."""
    assert ids.dtype == torch.int32 and out.dtype == torch.float32
    rc = native.cuda_lib().hds_embed_f32(_p(ids), _p(weight), _p(gamma), _p(out), ids.numel(), weight.shape[1], weight.shape[0],
                                         weight.shape[1] if cols is None else cols, eps, scale, _dt3(weight), _stream())
    native.check(rc, "hds_embed_f32")
    _count()
    return out


def norm_residual(resid: torch.Tensor, gamma: torch.Tensor, out: torch.Tensor, delta: Optional[torch.Tensor] = None,
                  factor: float = 1.0, post: Optional[torch.Tensor] = None, cols: Optional[int] = None, eps: float = 1e-5,
                  store_resid: bool = True, groups: int = 1, delta2: Optional[torch.Tensor] = None,
                  post2: Optional[torch.Tensor] = None) -> torch.Tensor:
    """``resid += norm(factor * delta) * post`` (without ``post``: ``resid += factor * delta``), ``+= norm(delta2) * post2`` on the
    fp32 stream, ``out = norm(resid) * gamma``, that norm over each of ``groups`` equal parts of a row (``hds_norm_residual``)."""
    rows, width = resid.shape
    assert resid.stride(0) == out.stride(0) and (delta is None or delta.stride(0) == resid.stride(0))
    assert delta is None or delta.dtype in (torch.float32, out.dtype)
    assert delta2 is None or (delta2.dtype == delta.dtype and delta2.stride(0) == resid.stride(0))
    rc = native.cuda_lib().hds_norm_residual(_p(resid), _p(delta), 1 if (delta is not None and delta.dtype == torch.float32) else 0,
                                             factor, _p(post), _p(gamma), _p(out), resid.stride(0), rows,
                                             width if cols is None else cols, width, eps, 1 if store_resid else 0, groups, _p(delta2), _p(post2),
                                             _dt3(out), _stream())
    native.check(rc, "hds_norm_residual")
    _count()
    return out


def gated_norm(y: torch.Tensor, z: torch.Tensor, weight: torch.Tensor, out: torch.Tensor, groups: int, eps: float,
               scale: float = 1.0, gate_after: bool = False) -> torch.Tensor:
    """``out = scale * weight * v / rms(v)``, ``v = y * silu(z)``, rms per part of a row (``groups`` equal parts); ``gate_after``:
    ``out = scale * weight * y / rms(y) * silu(z)``."""
    rc = native.cuda_lib().hds_gated_norm(_p(y), y.stride(0), _p(z), z.stride(0), _p(weight), _p(out), out.stride(0), y.shape[0],
                                          y.shape[1], groups, eps, scale, int(gate_after), _dt3(out), _stream())
    native.check(rc, "hds_gated_norm")
    _count()
    return out


SCAN_AUTO, SCAN_TOKENS, SCAN_CHUNKED = 0, 1, 2


def state_space(proj: torch.Tensor, conv_w: torch.Tensor, conv_b: torch.Tensor, dt_bias: torch.Tensor, decay: torch.Tensor,
                skip: torch.Tensor, state: torch.Tensor, conv_state: torch.Tensor, spans: torch.Tensor, n_single: int, groups: int,
                u: torch.Tensor, dt: torch.Tensor, y: torch.Tensor, method: int = SCAN_AUTO) -> torch.Tensor:
    """Convolution and recurrence of a state-space mixer over a ragged batch (``hds_state_space``). ``state``
    [slots, heads, vdim, state], ``conv_state`` [slots, taps, channels]; ``spans`` int32 [n_seqs, 4]."""
    T = proj.shape[0]
    _, heads, vdim, n = state.shape
    taps = conv_w.shape[0]
    rc = native.cuda_lib().hds_state_space(_p(proj), proj.stride(0), _p(conv_w), _p(conv_b), _p(dt_bias), _p(decay), _p(skip), _p(state),
                                           _p(conv_state), _p(spans), spans.shape[0], n_single, T, heads, vdim, n, groups, taps, _p(u),
                                           u.stride(0), _p(dt), _p(y), method, _dt3(proj), _stream())
    native.check(rc, "hds_state_space")
    n_multi = spans.shape[0] - n_single
    _count((2 if n_multi else 0) + (1 if n_single else 0))
    return y


def paged_attention_generic(q: torch.Tensor, out: torch.Tensor, kv_cache_layer: torch.Tensor, block_tables: torch.Tensor,
                            tok_seq: torch.Tensor, tok_pos: torch.Tensor, n_q_heads: int, n_kv_heads: int, head_dim: int,
                            block_size: int, scale: float, window: int = 0, keep_first: int = 0, value_dim: int = 0,
                            spans: Optional[torch.Tensor] = None, limit: int = 0, sink: Optional[torch.Tensor] = None,
                            sigmoid_bias: Optional[torch.Tensor] = None, gate: Optional[torch.Tensor] = None, softcap: float = 0.0) -> None:
    """fp32-arithmetic attention for any operand type and head size (``hds_paged_attention_generic``). ``value_dim`` > 0: pages of
    one plane, the first ``value_dim`` values of a key row are its value. ``spans``: skip sequences of more than ``limit`` tokens."""
    _arm_alibi(native.cuda_lib(), None, n_q_heads, sink=sink, sigmoid_bias=sigmoid_bias, gate=gate, softcap=softcap)
    rc = native.cuda_lib().hds_paged_attention_generic(_p(q), _p(out), out.stride(0), _p(kv_cache_layer), _p(block_tables),
                                                       block_tables.stride(0), _p(tok_seq), _p(tok_pos), q.shape[0], n_q_heads,
                                                       n_kv_heads, head_dim, block_size, scale, window, keep_first, value_dim, _p(spans),
                                                       limit, _dt3(q), _stream())
    native.check(rc, "hds_paged_attention_generic")
    _count()


def kv_append_generic(qkv: torch.Tensor, q_out: torch.Tensor, kv_cache_layer: torch.Tensor, tok_slot: torch.Tensor, n_q_heads: int,
                      n_kv_heads: int, head_dim: int, block_size: int) -> None:
    rc = native.cuda_lib().hds_kv_append_generic(_p(qkv), qkv.stride(0), _p(q_out), _p(kv_cache_layer), _p(tok_slot), qkv.shape[0],
                                                 n_q_heads, n_kv_heads, head_dim, block_size, qkv.element_size(), _stream())
    native.check(rc, "hds_kv_append_generic")
    _count()


# ------------------------------------------------------------------------------------------------
# latent attention, gated delta rule
# ------------------------------------------------------------------------------------------------
def latent_append(proj: torch.Tensor, q_out: Optional[torch.Tensor], pages: Optional[torch.Tensor], tok_pos: torch.Tensor,
                  tok_slot: torch.Tensor, heads: int, dim: int, rot_dim: int, head_width: int, rank: int, freq: torch.Tensor,
                  norm_w: Optional[torch.Tensor], eps: float) -> None:
    """Rotated queries to ``q_out`` [T, heads * head_width] and normed latents with their rotated key part to their ``pages``
    [blocks, 1, 1, bs, width], from ``proj`` = [q heads | latent | key part] (either output optional)."""
    width = rank + rot_dim if pages is None else pages.shape[4]
    rc = native.cuda_lib().hds_latent_append(_p(proj), proj.stride(0), _p(q_out), _p(pages), _p(tok_pos), _p(tok_slot), proj.shape[0], heads,
                                             dim, rot_dim, head_width, rank, width, _p(freq), _p(norm_w), eps, _dt3(proj), _stream())
    native.check(rc, "hds_latent_append")
    _count()


def head_matmul(x: torch.Tensor, w: torch.Tensor, out: torch.Tensor, tok_seq: torch.Tensor, spans: torch.Tensor, limit: int, in_width: int,
                out_width: int, copy: int = 0) -> torch.Tensor:
    """``out[t, h, :N] = x[t, h, :K] @ w[h]`` for ``w`` [heads, K, N]; then ``copy`` input values from place K on, then zeros. Rows of a
    head are ``in_width`` / ``out_width`` wide. Tokens of sequences with more than ``limit`` new tokens are skipped."""
    heads, K, N = w.shape
    rc = native.cuda_lib().hds_head_matmul(_p(x), x.stride(0), in_width, _p(w), _p(out), out.stride(0), out_width, _p(tok_seq), _p(spans), limit,
                                           x.shape[0], heads, K, N, copy, _dt3(x), _stream())
    native.check(rc, "hds_head_matmul")
    _count()
    return out


def latent_attention_supported(rank: int, page_width: int) -> bool:
    """Does the tensor-core kernel take latents of this size (else: :func:`paged_attention_generic`)?"""
    return bool(native.cuda_lib().hds_paged_attention_latent_supported(rank, page_width))


def latent_attention_ctas(item_tokens: int, heads: int, rank: int, page_width: int) -> Tuple[int, int]:
    """(CTAs per item and split, keys per tile) of :func:`paged_attention_latent`."""
    tile = ctypes.c_int(0)
    n = native.cuda_lib().hds_paged_attention_latent_ctas(item_tokens, heads, rank, page_width, ctypes.byref(tile))
    return int(n), tile.value


def latent_attention_workspace_bytes() -> int:
    return int(native.cuda_lib().hds_paged_attention_latent_workspace_bytes())


def paged_attention_latent(q: torch.Tensor, out: torch.Tensor, pages: torch.Tensor, block_tables: torch.Tensor, items: torch.Tensor,
                           n_items: int, item_tokens: int, heads: int, rank: int, block_size: int, n_splits: int, scale: float,
                           workspace: torch.Tensor, window: int = 0) -> None:
    """tcgen05 attention in the latent space: ``q`` [T, heads * width], ``pages`` [blocks, 1, 1, bs, width], ``out`` [T, heads * rank].
    items: at most ``item_tokens`` tokens each."""
    rc = native.cuda_lib().hds_paged_attention_latent(_p(q), _p(out), _p(pages), pages.shape[0], _p(block_tables), block_tables.stride(0),
                                                      _p(items), n_items, item_tokens, q.shape[0], heads, rank, pages.shape[4], block_size,
                                                      scale, window, n_splits, _p(workspace), workspace.numel(), _dt(q), _stream())
    native.check(rc, "hds_paged_attention_latent")
    _count()


def delta_workspace_bytes(n_tokens: int, n_seqs: int, heads: int, groups: int) -> int:
    """Scratch of the chunked delta rule for batches of up to ``n_tokens`` tokens in ``n_seqs`` sequences."""
    return int(native.cuda_lib().hds_delta_workspace_bytes(n_tokens, n_seqs, heads, groups))


def delta_rule(proj: torch.Tensor, conv_w: torch.Tensor, conv_b: torch.Tensor, dt_bias: torch.Tensor, decay: torch.Tensor, state: torch.Tensor,
               conv_state: torch.Tensor, spans: torch.Tensor, n_single: int, groups: int, u: torch.Tensor, dt: torch.Tensor, y: torch.Tensor,
               out: Optional[torch.Tensor], norm_w: torch.Tensor, eps: float, workspace: Optional[torch.Tensor] = None,
               method: int = SCAN_AUTO) -> torch.Tensor:
    """Convolution and recurrence of a gated delta rule over a ragged batch (``hds_delta_rule``), and, with ``out``, the norm and gate
    behind it. ``state`` [slots, heads, vdim, dim]. Without ``out`` (or when sequences bring several tokens) ``y`` holds the read-outs."""
    T = proj.shape[0]
    _, heads, vdim, n = state.shape
    rc = native.cuda_lib().hds_delta_rule(_p(proj), proj.stride(0), _p(conv_w), _p(conv_b), _p(dt_bias), _p(decay), _p(state), _p(conv_state),
                                          _p(spans), spans.shape[0], n_single, T, heads, vdim, n, groups, conv_w.shape[0], _p(u), u.stride(0),
                                          _p(dt), _p(y), _p(out), 0 if out is None else out.stride(0), _p(norm_w), eps, _p(workspace),
                                          0 if workspace is None else workspace.numel(), method, _dt3(proj), _stream())
    native.check(rc, "hds_delta_rule")
    _count((2 if spans.shape[0] > n_single else 0) + (1 if n_single else 0))
    if out is not None and n_single < spans.shape[0]:
        gated_norm(y, proj[:, :heads * vdim], norm_w, out, heads, eps, gate_after=True)
    return y


# ------------------------------------------------------------------------------------------------
# attention inputs, minGRU, gated linear attention
# ------------------------------------------------------------------------------------------------
def attention_append(qkv: torch.Tensor, q_out: torch.Tensor, kv_cache_layer: Optional[torch.Tensor], tok_pos: torch.Tensor, tok_slot: torch.Tensor,
                     n_q_heads: int, n_kv_heads: int, head_dim: int, block_size: int, freq: Optional[torch.Tensor],
                     q_norm: Optional[torch.Tensor] = None, k_norm: Optional[torch.Tensor] = None, q_cols: int = 0, k_cols: int = 0,
                     eps: float = 0.0, first: Optional[torch.Tensor] = None, share: Optional[torch.Tensor] = None,
                     amp: Optional[torch.Tensor] = None) -> None:
    """Projected rows ``qkv`` = [q heads | k heads | v heads] -> normed and rotated queries, page rows with mixed values
    (``hds_attention_append``). ``n_kv_heads`` = 0: queries alone, no pages."""
    _check_2d(qkv, "qkv")
    assert n_kv_heads == 0 or (kv_cache_layer.shape[4] == head_dim and kv_cache_layer.shape[3] == block_size)
    assert first is None or (first.shape[:4] == kv_cache_layer.shape[:4] and first.is_contiguous())
    rc = native.cuda_lib().hds_attention_append(_p(qkv), qkv.stride(0), _p(q_out), _p(kv_cache_layer), _p(tok_pos), _p(tok_slot), qkv.shape[0],
                                                n_q_heads, n_kv_heads, head_dim, block_size, _p(freq), _p(amp), _p(q_norm), _p(k_norm), q_cols, k_cols,
                                                eps, _p(first), 0 if first is None else first.shape[4], _p(share), _dt3(qkv), _stream())
    native.check(rc, "hds_attention_append")
    _count()


def mix_cached_values(kv_cache_layer: torch.Tensor, first: torch.Tensor, tok_slot: torch.Tensor, share: torch.Tensor, n_kv_heads: int,
                      head_dim: int, block_size: int) -> None:
    """The tokens' cached values become (1 - share) of themselves plus ``share`` of those in ``first``."""
    assert first.shape[:4] == kv_cache_layer.shape[:4] and kv_cache_layer.shape[3] == block_size
    rc = native.cuda_lib().hds_mix_cached_values(_p(kv_cache_layer), _p(first), first.shape[4], _p(tok_slot), _p(share), tok_slot.numel(),
                                                 n_kv_heads, head_dim, block_size, _dt3(kv_cache_layer), _stream())
    native.check(rc, "hds_mix_cached_values")
    _count()


def gru_workspace_bytes(n_tokens: int, n_seqs: int, width: int) -> int:
    return int(native.cuda_lib().hds_gru_workspace_bytes(n_tokens, n_seqs, width))


def gru(proj: torch.Tensor, bias: torch.Tensor, state: torch.Tensor, spans: torch.Tensor, n_single: int, out: Optional[torch.Tensor],
        workspace: Optional[torch.Tensor]) -> None:
    """minGRU of ``proj`` = [z | u | output gate] over a ragged batch (``hds_gru``); ``state`` [slots, ..., width] fp32."""
    _check_2d(proj, "proj")
    width = bias.numel() // 2
    assert proj.shape[1] == 3 * width and state[0].numel() == width
    rc = native.cuda_lib().hds_gru(_p(proj), proj.stride(0), _p(bias), _p(state), _p(spans), spans.shape[0], n_single, proj.shape[0], width,
                                   _p(out), 0 if out is None else out.stride(0), _p(workspace), 0 if workspace is None else workspace.numel(),
                                   _dt3(proj), _stream())
    native.check(rc, "hds_gru")
    _count((3 if out is not None else 2) * (spans.shape[0] > n_single) + (n_single > 0))


def linear_attention_workspace_bytes(n_tokens: int, n_seqs: int, heads: int, vdim: int, dim: int) -> int:
    """Scratch of the chunked form for batches of up to ``n_tokens`` tokens in ``n_seqs`` sequences (0: not for this shape)."""
    return int(native.cuda_lib().hds_linear_attention_workspace_bytes(n_tokens, n_seqs, heads, vdim, dim))


def linear_attention(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, gate: torch.Tensor, z: torch.Tensor, bias: torch.Tensor, inv_tau: float,
                     state: torch.Tensor, spans: torch.Tensor, n_single: int, y: torch.Tensor, out: Optional[torch.Tensor],
                     norm_w: torch.Tensor, eps: float, workspace: Optional[torch.Tensor] = None, method: int = SCAN_AUTO) -> None:
    """Gated linear attention over a ragged batch, with the norm and gate behind (``hds_linear_attention``). ``state``
    [slots, heads, vdim, dim] fp32; ``y`` fp32 scratch; ``out`` None: advance the state alone."""
    T = q.shape[0]
    _, heads, vdim, dim = state.shape
    assert q.stride(0) == k.stride(0) == v.stride(0) == gate.stride(0) and bias.numel() == heads * dim
    done = ctypes.c_int(1)
    rc = native.cuda_lib().hds_linear_attention(_p(q), _p(k), _p(v), _p(gate), q.stride(0), _p(z), z.stride(0), _p(bias), inv_tau, _p(state),
                                                _p(spans), spans.shape[0], n_single, T, heads, vdim, dim, _p(y), y.stride(0), _p(out),
                                                0 if out is None else out.stride(0), _p(norm_w), eps, _p(workspace),
                                                0 if workspace is None else workspace.numel(), method, ctypes.addressof(done), _dt3(q), _stream())
    native.check(rc, "hds_linear_attention")
    _count((3 if out is not None else 2) * (spans.shape[0] > n_single) + (n_single > 0))
    if out is not None and not done.value:
        gated_norm(y[:, :heads * vdim], gate[:, :heads * vdim], norm_w, out, heads, eps, gate_after=True)


def retention_workspace_bytes(n_tokens: int, n_seqs: int, heads: int, vdim: int, dim: int) -> int:
    """Scratch of the chunked form for batches of up to ``n_tokens`` tokens in ``n_seqs`` sequences (0: not for this shape)."""
    return int(native.cuda_lib().hds_retention_workspace_bytes(n_tokens, n_seqs, heads, vdim, dim))


def retention(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, gate: torch.Tensor, log2_decay: torch.Tensor, freq: Optional[torch.Tensor],
              amp: Optional[torch.Tensor], k_scale: float, norm_cols: int, state: torch.Tensor, spans: torch.Tensor, n_single: int, y: torch.Tensor,
              out: Optional[torch.Tensor], ones: torch.Tensor, eps: float, workspace: Optional[torch.Tensor] = None, method: int = SCAN_AUTO) -> None:
    """Retention over a ragged batch, with the norm and gate behind (``hds_retention``). ``state`` [slots, heads, vdim, dim] fp32; heads
    hold ``norm_cols`` values and zeros; ``freq`` None: q and k have been turned; ``y`` fp32 scratch; ``out`` None: advance the state
    alone; ``ones``: as many as a row of v has values."""
    T = q.shape[0]
    _, heads, vdim, dim = state.shape
    assert q.stride(0) == k.stride(0) and v.stride(0) == gate.stride(0) and log2_decay.numel() == heads and (freq is None or freq.numel() == dim // 2)
    done = ctypes.c_int(1)
    rc = native.cuda_lib().hds_retention(_p(q), _p(k), q.stride(0), _p(v), _p(gate), v.stride(0), _p(log2_decay), _p(freq), _p(amp), k_scale, norm_cols,
                                         _p(state), _p(spans), spans.shape[0], n_single, T, heads, vdim, dim, _p(y), y.stride(0), _p(out),
                                         0 if out is None else out.stride(0), eps, _p(workspace), 0 if workspace is None else workspace.numel(),
                                         method, ctypes.addressof(done), _dt3(q), _stream())
    native.check(rc, "hds_retention")
    _count((2 if out is not None else 1) * (spans.shape[0] > n_single) + (n_single > 0))
    if out is not None and not done.value:
        r = vdim / norm_cols          # mean over a padded row * r = mean over the head
        gated_norm(y[:, :heads * vdim], gate, ones, out, heads, eps / r, r**-0.5, gate_after=True)


def retention_stuck() -> bool:
    """Has a wait inside retention's kernels ever run out of time? (Synchronizes.)"""
    flag = ctypes.c_int(0)
    native.check(native.cuda_lib().hds_retention_status(ctypes.addressof(flag)), "hds_retention_status")
    return bool(flag.value)


# ------------------------------------------------------------------------------------------------
# batches of many requests: adapters beside a projection, attention behind a shared prefix, controls on logits
# ------------------------------------------------------------------------------------------------
# (A step makes hundreds of these calls: their checks read each attribute once, and a stream is asked for by its number. A Stream object and
# a device guard alone cost 5 us of the 22 that a call took; it takes 12 to 17 so.)
_raw_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None)      # (a build of torch for the CPU alone has no such name, and no call)
_I32, _F32, _LOGITS = torch.int32, torch.float32, (torch.bfloat16, torch.float16, torch.float32)


def _place(t: torch.Tensor, name: str) -> int:
    if not t.is_cuda:
        raise ValueError(f"{name} must be a CUDA tensor")
    return t.get_device()


def _elsewhere(index: int, **tensors: Optional[torch.Tensor]) -> None:
    """Name the tensor that is not on the call's device."""
    for name, t in tensors.items():
        if t is not None and t.get_device() != index:
            raise ValueError(f"{name} is on {t.device}, the call is on cuda:{index}")


_HERE = contextlib.nullcontext()


def _on(index: int):
    """The call's device as the current one, where it is not that anyway."""
    return _HERE if index == torch._C._cuda_getDevice() else torch.cuda.device(index)


def _rows(t: torch.Tensor, name: str) -> int:
    """Elements between the rows of a 2-D tensor whose last dimension is contiguous (of a single row: its width)."""
    st, shape = t.stride(), t.shape
    if len(st) != 2 or st[1] != 1 and shape[1] > 1:
        raise ValueError(f"{name} must be 2-D with a contiguous last dimension, got {tuple(shape)} / {st}")
    return st[0] if shape[0] > 1 else shape[1]


def _rows_apart(t: torch.Tensor, name: str) -> int:
    """The same where no two rows may share memory: of a tensor that is written, or that tensor maps describe."""
    ld, (rows, width) = _rows(t, name), t.shape
    if ld < width and rows > 1:
        raise ValueError(f"rows of {name} share memory: {(rows, width)} / {t.stride()}")
    return ld


@functools.lru_cache(maxsize=1024)
def _adapter_parts(index: int, tiles: int, width: int) -> int:
    return native.cuda_lib().hds_adapter_parts(tiles, width)       # (of the current device, which is number `index`)


def adapter_add(base: torch.Tensor, x: torch.Tensor, down: torch.Tensor, up: torch.Tensor, scales: torch.Tensor, plan: AdapterPlan,
                out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """``out[t] = base[t] + scales[i] * (x[t] @ down[i].T) @ up[i].T`` with row t's own adapter ``i`` (``plan``), ``out[t] = base[t]`` for a row
    without one. ``base`` [T, N] (the shared projection's output), ``x`` [T, K], ``down`` [adapters, R, K], ``up`` [adapters, N, R], 16-bit;
    ``scales`` fp32 [adapters]. K, N and R are multiples of 8, R at most 256. ``out`` may be ``base`` or ``x``. With more than 16 rows of an
    adapter the call allocates scratch."""
    index = _place(x, "x")
    ld_x, ld_base, dt, dtype = _rows(x, "x"), _rows(base, "base"), _dt(x), x.dtype
    (T, K), (rows, N) = x.shape, base.shape
    if down.dim() != 3 or up.dim() != 3 or not down.is_contiguous() or not up.is_contiguous():
        raise ValueError("down and up must be contiguous [adapters, rank, K] and [adapters, N, rank]")
    n, R, width = down.shape
    if rows != T or width != K or up.shape != (n, N, R) or scales.shape != (n, ):
        raise ValueError(f"shapes do not agree: base {tuple(base.shape)}, x {tuple(x.shape)}, down {tuple(down.shape)}, up {tuple(up.shape)}, "
                         f"scales {tuple(scales.shape)}")
    if base.dtype != dtype or down.dtype != dtype or up.dtype != dtype or scales.dtype != torch.float32 or not scales.is_contiguous():
        raise TypeError("base, x, down and up have one type, scales are contiguous fp32")
    if R % 8 or not 8 <= R <= 256 or K % 8 or N % 8 or not 0 < K < 1 << 24 or not 0 < N < 1 << 24:
        raise ValueError(f"K, N and the rank are multiples of 8, the rank at most 256, K and N below 2^24; got {K}, {N}, {R}")
    if plan.n_rows != T or plan.n_adapters != n:
        raise ValueError(f"the plan is for {plan.n_rows} rows of {plan.n_adapters} adapters, the call has {T} of {n}")
    if out is None:
        out, ld_out = x.new_empty((T, N)), N
    else:
        ld_out = _rows_apart(out, "out")
        if out.shape != (T, N) or out.dtype != dtype:
            raise ValueError("out must be like base")
    if not index == base.get_device() == down.get_device() == up.get_device() == scales.get_device() == out.get_device():
        _elsewhere(index, base=base, down=down, up=up, scales=scales, out=out)
    if plan.index != index:
        raise ValueError(f"the plan is on {plan.device}, the call is on cuda:{index}")
    p_base, p_out = base.data_ptr(), out.data_ptr()
    count = plan.n_tiles if p_out == p_base and ld_out == ld_base else plan.n_tiles_and_bare
    if count == 0:
        return out
    lib = native.cuda_lib()
    with _on(index):
        stream = _raw_stream(index)
        plan.used_on(stream)
        ws, n_bytes = None, 0
        if plan.tile_rows > ADAPTER_FEW:
            n_bytes = _adapter_parts(index, count, K) * T * R * 4
            ws = x.new_empty(n_bytes // 2)       # of this call alone: a plan may be in use on several streams, and in graphs
        rc = lib.hds_adapter_add(p_base, ld_base, x.data_ptr(), ld_x, down.data_ptr(), up.data_ptr(), scales.data_ptr(), n, R, K, N, T,
                                 plan.tiles_ptr, plan.rows_ptr, count, plan.tile_rows, p_out, ld_out, _p(ws), n_bytes, dt, stream)
    if rc:
        native.check(rc, "hds_adapter_add")
    _count(1 if ws is None else 2)
    return out


def paged_attention_shared(q: torch.Tensor, out: torch.Tensor, kv_cache_layer: torch.Tensor, block_tables: torch.Tensor, plan: SharedPrefixPlan,
                           scale: float) -> torch.Tensor:
    """Causal attention of a batch whose sequences share prefixes (``plan``), each prefix read once for its group. ``q`` and ``out``
    [rows, n_q_heads * head_dim], a sequence's new tokens being neighbouring rows in the plan's order; rows behind the last sequence are left as they
    are. For few new tokens per sequence: from about 64 on, ``paged_attention_prefill`` is faster though it reads the prefix per sequence (16 sequences
    of 32 heads on 8 behind 4096 keys: 36 and 135 us with 16 new tokens each, 149 and 139 with 64, 5099 and 1101 with 1000). The prefix' weights are
    rounded to 16 bits, which puts outputs further from 64 bits than those of the per-sequence decode kernels (0.0023 and 0.0017 of them in bf16). As
    with those, infinite or NaN values of a new token reach the rows ahead of it in its sequence, to which it has a weight of 0.
    ``kv_cache_layer`` [blocks, 2, n_kv_heads, block_size, head_dim] holds the new tokens' keys already; ``block_tables`` int32
    [sequences, stride]. head_dim 64 or 128, 16-bit. ``out`` may be ``q``, and overlaps no operand otherwise. A group's pages are those that its first sequence's table names. ``scale`` from 0 to below 2^127.
    The call allocates its scratch."""
    index, cache = _place(q, "q"), kv_cache_layer.shape
    ld_q, ld_out, dt, dtype = _rows_apart(q, "q"), _rows_apart(out, "out"), _dt(q), q.dtype
    d, H, rows = plan.head_dim, plan.n_q_heads, plan.rows
    if d not in (64, 128):
        raise ValueError(f"head_dim must be 64 or 128, got {d}")
    (q_rows, q_width), (out_rows, out_width) = q.shape, out.shape
    if q_width != H * d or q_rows < rows or out_width != q_width or out_rows < rows:
        raise ValueError(f"q and out need {rows} rows of {H} x {d}, got {tuple(q.shape)} and {tuple(out.shape)}")
    if out.dtype != dtype or kv_cache_layer.dtype != dtype:
        raise TypeError("q, out and the cache have one type")
    blocks = cache[0] if len(cache) == 5 else 0
    if cache != (blocks, 2, plan.n_kv_heads, plan.block_size, d) or not kv_cache_layer.is_contiguous():
        raise ValueError(f"the cache must be contiguous [blocks, 2, {plan.n_kv_heads}, {plan.block_size}, {d}], got {tuple(cache)}")
    ld_tables, (n_tables, width) = _rows(block_tables, "block_tables"), block_tables.shape
    if block_tables.dtype != torch.int32 or n_tables < plan.n_seqs or width < plan.max_blocks or ld_tables >= 1 << 31:
        raise ValueError(f"block_tables must be int32 [{plan.n_seqs}, at least {plan.max_blocks}], rows less than 2^31 apart, got {block_tables.dtype} "
                         f"{tuple(block_tables.shape)} / {block_tables.stride()}")
    if not index == out.get_device() == kv_cache_layer.get_device() == block_tables.get_device():
        _elsewhere(index, out=out, kv_cache_layer=kv_cache_layer, block_tables=block_tables)
    if plan.index != index:
        raise ValueError(f"the plan is on {plan.device}, the call is on cuda:{index}")
    if not 0.0 <= scale < MAX_SCALE:
        raise ValueError(f"scale must be below 2^127 and not negative, got {scale}")
    if rows == 0:
        return out
    lib = native.cuda_lib()
    with _on(index):
        stream = _raw_stream(index)
        plan.used_on(stream)
        n_bytes = plan.workspace_bytes
        if not n_bytes:
            n_bytes = plan.workspace_bytes = lib.hds_paged_attention_shared_workspace_bytes(rows, H, d, plan.n_tiles, plan.p_splits, plan.n_units, plan.n_workers)
        ws = q.new_empty(n_bytes // 2)       # of this call alone: a plan may be in use on several streams, and in graphs
        rc = lib.hds_paged_attention_shared(q.data_ptr(), ld_q, out.data_ptr(), ld_out, rows, kv_cache_layer.data_ptr(), blocks, block_tables.data_ptr(), ld_tables,
                                            plan.tiles_ptr, plan.n_tiles, plan.p_splits, plan.items_ptr, plan.workers_ptr, plan.n_workers, plan.units_ptr,
                                            plan.n_units, plan.rows_ptr, H, plan.n_kv_heads, d, plan.block_size, scale, ws.data_ptr(), n_bytes, dt,
                                            stream)
    if rc:
        native.check(rc, "hds_paged_attention_shared")
    _count(2)
    return out


def _check_rows(t: torch.Tensor, name: str, dtype: torch.dtype, rows: Optional[int], cols: int = 0) -> int:
    ld = _rows(t, name)
    shape = t.shape
    if t.dtype != dtype or rows is not None and shape[0] != rows or shape[1] < cols:
        raise ValueError(f"{name} must be {dtype} [{'masks' if rows is None else rows}, {f'at least {cols}' if cols else 'any'}], got {t.dtype} {tuple(shape)}")
    return ld


def _check_each(t: Optional[torch.Tensor], name: str, dtype: torch.dtype, n: int) -> None:
    if t is not None and (t.dtype != dtype or t.shape != (n, ) or not t.is_contiguous()):
        raise ValueError(f"{name} must be contiguous {dtype} [{n}], got {t.dtype} {tuple(t.shape)}")


def _check_controls(logits: torch.Tensor, out: torch.Tensor, history, history_len, prompt_len, repetition, presence, frequency, bias_ids, bias, mask,
                    mask_rows) -> Tuple[int, ...]:
    """What :func:`logit_controls` takes, and the restatement in torch: elements between the rows of logits, out, history, bias_ids, bias and mask;
    history places, biases and masks."""
    ld, ld_out, shape, dtype, index = _rows(logits, "logits"), _rows_apart(out, "out"), logits.shape, logits.dtype, logits.get_device()
    n, V = shape
    if dtype not in _LOGITS:
        raise TypeError(f"unsupported logits dtype {dtype}: bf16, fp16 or fp32")
    if out.shape != shape or out.dtype != dtype:
        raise ValueError("out must be like logits")
    if n > 65535 or V >= 1 << 30:
        raise ValueError("at most 65535 rows and a vocabulary below 2^30")
    ld_history = ld_ids = ld_bias = ld_mask = places = n_bias = n_masks = 0
    here, each = out.get_device() == index, (n, )
    if history is not None and history_len is not None:
        ld_history, places = _check_rows(history, "history", _I32, n), history.shape[1]
        here = here and history.get_device() == index
        if history_len.dtype is not _I32 or history_len.shape != each or not history_len.is_contiguous():
            _check_each(history_len, "history_len", _I32, n)
        here = here and history_len.get_device() == index
        if prompt_len is not None:
            if prompt_len.dtype is not _I32 or prompt_len.shape != each or not prompt_len.is_contiguous():
                _check_each(prompt_len, "prompt_len", _I32, n)
            here = here and prompt_len.get_device() == index
        for t in (repetition, presence, frequency):
            if t is not None:
                if t.dtype is not _F32 or t.shape != each or not t.is_contiguous():
                    for wrong, name in ((repetition, "repetition"), (presence, "presence"), (frequency, "frequency")):
                        _check_each(wrong, name, _F32, n)
                here = here and t.get_device() == index
    elif history is not None or history_len is not None:
        raise ValueError("a history comes with its lengths")
    elif prompt_len is not None or repetition is not None or presence is not None or frequency is not None:
        raise ValueError("penalties need a history")
    if bias is not None and bias_ids is not None:
        ld_ids, ld_bias, n_bias = _check_rows(bias_ids, "bias_ids", _I32, n), _check_rows(bias, "bias", _F32, n), bias.shape[1]
        if bias_ids.shape[1] != n_bias:
            raise ValueError("bias and bias_ids have one shape")
        here = here and bias.get_device() == bias_ids.get_device() == index
    elif bias is not None or bias_ids is not None:
        raise ValueError("biases come with their tokens")
    if mask is not None:
        ld_mask, n_masks = _check_rows(mask, "mask", _I32, n if mask_rows is None else None, -(-V // 32)), mask.shape[0]
        _check_each(mask_rows, "mask_rows", _I32, n)
        here = here and mask.get_device() == index and (mask_rows is None or mask_rows.get_device() == index)
    elif mask_rows is not None:
        raise ValueError("mask_rows needs masks")
    if places >= 1 << 30 or n_bias >= 1 << 30 or n_masks >= 1 << 30:       # (the library takes them as 32-bit numbers)
        raise ValueError("histories, biases and masks: fewer than 2^30")
    if not here:
        _elsewhere(index, out=out, history=history, history_len=history_len, prompt_len=prompt_len, repetition=repetition, presence=presence,
                   frequency=frequency, bias_ids=bias_ids, bias=bias, mask=mask, mask_rows=mask_rows)
    return ld, ld_out, ld_history, ld_ids, ld_bias, ld_mask, places, n_bias, n_masks


def logit_controls(logits: torch.Tensor, out: Optional[torch.Tensor] = None, *, history: Optional[torch.Tensor] = None,
                   history_len: Optional[torch.Tensor] = None, prompt_len: Optional[torch.Tensor] = None, repetition: Optional[torch.Tensor] = None,
                   presence: Optional[torch.Tensor] = None, frequency: Optional[torch.Tensor] = None, bias_ids: Optional[torch.Tensor] = None,
                   bias: Optional[torch.Tensor] = None, mask: Optional[torch.Tensor] = None, mask_rows: Optional[torch.Tensor] = None) -> torch.Tensor:
    """What every row's request lays on its logits ``[n, vocab]``, in this order (``out`` may be ``logits``, and
    overlaps no operand otherwise):

    ``repetition`` fp32 [n]: logits of tokens in the row's history are divided by it where positive, multiplied where not; ``frequency`` and
    ``presence`` fp32 [n]: taken off once per time that the token stands in the answer, and once if it does. ``history`` int32 [n, places] holds
    a row's tokens, the first ``history_len[i]`` of them, and of these the first ``prompt_len[i]`` are its prompt (default: none). ``bias``
    fp32 [n, k] is added to the logits of the tokens ``bias_ids`` int32 [n, k] (of a token given twice the last one counts;
    beyond some hundred per row a mask is the better way to forbid: 1000 biases in 64 rows of 32000 take 17 us, 5000 take 473). ``mask`` int32
    [masks, words]: bit v % 32 of word v // 32 allows token v, the others get -inf; ``mask_rows`` int32 [n]: the row's mask, or -1 for none
    (default: mask i for row i). Ids that are no tokens (-1 as padding) are passed over."""
    index = _place(logits, "logits")
    if out is None:
        out = logits.new_empty(logits.shape)
    ld, ld_out, ld_history, ld_ids, ld_bias, ld_mask, places, n_bias, n_masks = _check_controls(
        logits, out, history, history_len, prompt_len, repetition, presence, frequency, bias_ids, bias, mask, mask_rows)
    n, V = logits.shape
    with _on(index):
        rc = native.cuda_lib().hds_logit_controls(logits.data_ptr(), ld, out.data_ptr(), ld_out, n, V, _p(history), ld_history, places, _p(history_len),
                                                  _p(prompt_len), _p(repetition), _p(presence), _p(frequency), _p(bias_ids), ld_ids, _p(bias), ld_bias,
                                                  n_bias, _p(mask), ld_mask, n_masks, _p(mask_rows), _dt3(logits), _raw_stream(index))
    if rc:
        native.check(rc, "hds_logit_controls")
    _count(1 if n and V else 0)
    return out
