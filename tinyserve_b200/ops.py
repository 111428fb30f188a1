"""Torch-facing wrappers over the C-ABI kernels.

These functions take CUDA tensors, call ``libtsb_moe.so`` on the current CUDA
stream and return CUDA tensors.  CPU tensors are rejected: there is no CPU
path in the product.
"""
from __future__ import annotations

import ctypes

import torch

from . import _lib
from .formats import FORMATS, TSB_MXFP4, mxfp4_split

_DT = {torch.float32: _lib.DT_F32, torch.bfloat16: _lib.DT_BF16, torch.float16: _lib.DT_F16}


def _ptr(t: torch.Tensor | None) -> int | None:
    return None if t is None else t.data_ptr()


def _stream(device: torch.device) -> int:
    return torch.cuda.current_stream(device).cuda_stream


def _require_cuda(*ts: torch.Tensor | None) -> None:
    for t in ts:
        if t is not None and not t.is_cuda:
            raise RuntimeError("tinyserve_b200 kernels need CUDA tensors")


def _require_one_device(first: torch.Tensor, *others: torch.Tensor | None) -> None:
    device = first.get_device()
    if device >= 0:
        for t in others:
            if t is not None and t.get_device() != device:
                break
        else:
            return
    raise RuntimeError("tinyserve_b200 kernels need CUDA tensors, all on one device")


def dequant(fmt: int, w: torch.Tensor, scales: torch.Tensor | None, rows: int, cols: int,
            dtype: torch.dtype = torch.float32) -> torch.Tensor:
    """Bit-exact dequantisation (same values as ``dequant_tensor`` /
    ``dequant_mxfp4_no_transpose``) of a [rows, cols] weight."""
    _require_cuda(w, scales)
    if dtype not in (torch.float32, torch.bfloat16):
        raise ValueError("dequant dtype must be float32 or bfloat16")
    out = torch.empty(rows, cols, dtype=dtype, device=w.device)
    _lib.check(_lib.lib().tsb_dequant(fmt, _ptr(w), _ptr(scales), rows, cols, _ptr(out), _DT[dtype],
                                      _stream(w.device)))
    return out


def quant_matvec(fmt: int, w: torch.Tensor, scales: torch.Tensor | None, out_features: int, in_features: int,
                 x: torch.Tensor, out_dtype: torch.dtype | None = None,
                 dev_err: torch.Tensor | None = None) -> torch.Tensor:
    """y[M, N] = x[M, K] @ W[N, K]^T with W quantised; x is fp32/bf16/fp16 [M, K]."""
    _require_cuda(w, scales, x)
    if x.dim() == 1:
        x = x.view(1, -1)
    x = x.contiguous()
    M = x.shape[0]
    if x.shape[1] != in_features:
        raise ValueError(f"x has {x.shape[1]} features, expected {in_features}")
    y = torch.empty(M, out_features, dtype=out_dtype or x.dtype, device=x.device)
    _lib.check(_lib.lib().tsb_quant_matvec(
        fmt, _ptr(w), _ptr(scales), out_features, in_features, _ptr(x), _DT[x.dtype], M, in_features,
        _ptr(y), _DT[y.dtype], out_features, _ptr(dev_err), _stream(x.device)))
    return y


def weight_bytes(fmt: int, rows: int, cols: int) -> tuple[int, int]:
    d, s = ctypes.c_int64(), ctypes.c_int64()
    _lib.check(_lib.lib().tsb_weight_bytes(fmt, rows, cols, ctypes.byref(d), ctypes.byref(s)))
    return d.value, s.value


# ---------------------------------------------------------------------------
# A paged KV cache, attention over it and token sampling: the operators of a
# serving step (tinyserve/paged_kv_cache.py:20-122; sliding window with
# visible first tokens, tinyserve/static_kv_cache.py:282-389).
# ---------------------------------------------------------------------------
_paged_ws: dict[tuple[int, int, int], torch.Tensor] = {}                   # by device, head size, stream
_captured_ws: dict[tuple[int, int, int], tuple[int, torch.Tensor]] = {}    # of the capture that is under way there
_PAGED_ZEROED = 64 * 1024  # TSB_PAGED_ZEROED


def paged_workspace(device: torch.device, head_dim: int) -> torch.Tensor:
    """Zero-initialised scratch of the paged operators.  One workspace serves
    successive calls on one stream; the operators keep one per (device,
    stream) unless they are given another.  A graph captured on a stream where
    they keep none holds scratch of its own."""
    n = _lib.lib().tsb_paged_workspace(head_dim)
    if n == 0:
        raise RuntimeError("head_dim must be 64 or 128")
    ws = torch.empty(n, dtype=torch.uint8, device=device)
    ws[:_PAGED_ZEROED].zero_()
    return ws


def _paged_workspace(device: torch.device, head_dim: int, stream: int) -> torch.Tensor:
    key = (device.index, head_dim, stream)
    ws = _paged_ws.get(key)
    if ws is not None:
        return ws
    capture = ctypes.c_uint64()
    _lib.check(_lib.lib().tsb_capture_id(stream, ctypes.byref(capture)))
    if capture.value == 0:
        ws = _paged_ws[key] = paged_workspace(device, head_dim)
        return ws
    # Memory of the graph's, zeroed where the graph runs: nothing outside it may
    # go by it, and another capture on this stream takes its own.
    held = _captured_ws.get(key)
    if held is None or held[0] != capture.value:
        _captured_ws.pop(key, None)
        held = _captured_ws[key] = (capture.value, paged_workspace(device, head_dim))
    return held[1]


_raw_stream = torch._C._cuda_getCurrentRawStream if hasattr(torch._C, "_cuda_getCurrentRawStream") else None


def _stream_of(t: torch.Tensor) -> int:
    """The current stream of a tensor's device, without the Stream object."""
    return _raw_stream(t.get_device()) if _raw_stream else _stream(t.device)


def paged_device_error(workspace: torch.Tensor | None = None, device: torch.device | None = None) -> int:
    """Read and clear the device error word of a workspace, or of every
    workspace the paged operators keep for ``device`` (of a stream's graphs with
    scratch of their own, the last captured one's): 0 when the batches were
    consistent, 2 when one named a page outside the pool or a length beyond
    its table, 1 when a wait inside a kernel gave up.  After an error the
    workspace is made sound again.  Synchronises."""
    if workspace is None:
        device = torch.device("cuda" if device is None else device)
        index = torch.cuda.current_device() if device.index is None else device.index
        kept = list(_paged_ws.items()) + [(key, ws) for key, (_, ws) in _captured_ws.items()]
        held = [ws for key, ws in kept if key[0] == index]
    else:
        held = [workspace]
    code = 0
    for ws in held:
        torch.cuda.synchronize(ws.device)
        c = ctypes.c_int32()
        _lib.check(_lib.lib().tsb_read_device_error(ws.data_ptr(), ctypes.byref(c), _stream(ws.device)))
        if c.value:
            ws[:_PAGED_ZEROED].zero_()  # a call that gave up leaves counts of finished parts
            torch.cuda.synchronize(ws.device)
        code = code or c.value
    return code


def _paged_call(rows: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor, page_table: torch.Tensor,
                cu_q: torch.Tensor, kv_lens: torch.Tensor, max_q: int, workspace: torch.Tensor | None):
    """The C structs of a paged call (kept alive by the caller), after the
    checks that need the tensors themselves."""
    _require_one_device(rows, k_cache, v_cache, page_table, cu_q, kv_lens, workspace)
    if workspace is not None and (workspace.dtype != torch.uint8 or not workspace.is_contiguous()):
        raise ValueError("workspace must be contiguous uint8")
    dtype, held = rows.dtype, k_cache.dtype
    if dtype != torch.bfloat16 and dtype != torch.float16:
        raise TypeError("tokens must be bfloat16 or float16")
    if held != dtype and held != torch.float8_e4m3fn:
        raise TypeError("the cache must hold the tokens' dtype or float8_e4m3fn")
    shape, strides, table = k_cache.shape, k_cache.stride(), page_table.shape
    if len(shape) != 4 or v_cache.shape != shape or v_cache.stride() != strides or v_cache.dtype != held:
        raise ValueError("k_cache and v_cache must be alike: [pages, kv_heads, page_size, head_dim]")
    if strides[3] != 1:
        raise ValueError("the caches' last dimension must be contiguous")
    if len(table) != 2 or page_table.dtype != torch.int32 or (table[1] > 1 and page_table.stride(1) != 1):
        raise ValueError("page_table must be int32 [sequences, pages] with contiguous rows")
    n_seqs, width = table
    if (cu_q.dtype != torch.int32 or kv_lens.dtype != torch.int32 or cu_q.shape != (n_seqs + 1,)
            or kv_lens.shape != (n_seqs,) or not cu_q.is_contiguous() or not kv_lens.is_contiguous()):
        raise ValueError("cu_q and kv_lens must be contiguous int32 of sequences + 1 and sequences entries")
    cache = _lib.TsbPagedCache(k_cache.data_ptr(), v_cache.data_ptr(), strides[0], strides[1], strides[2], shape[0],
                               shape[2], shape[1], shape[3], _DT[dtype], 0 if held == dtype else 1)
    batch = _lib.TsbPagedBatch(page_table.data_ptr(), cu_q.data_ptr(), kv_lens.data_ptr(),
                               page_table.stride(0) if n_seqs > 1 else width, width, n_seqs, rows.shape[0], max_q)
    return cache, batch


def paged_kv_store(qkv: torch.Tensor, cos: torch.Tensor, sin: torch.Tensor, k_cache: torch.Tensor,
                   v_cache: torch.Tensor, page_table: torch.Tensor, cu_q: torch.Tensor, kv_lens: torch.Tensor, *,
                   n_q_heads: int, q_out: torch.Tensor | None = None,
                   workspace: torch.Tensor | None = None) -> torch.Tensor:
    """Rotate a fused projection's queries and keys and put keys and values into
    their pages; returns the rotated queries [N, n_q_heads, D].

    qkv         [N, (n_q_heads + 2 kv_heads) * D] bf16 / f16, contiguous rows: the new tokens of all sequences
    cos, sin    [positions, D / 2] fp32, bf16 or f16; halves rotated (the GPT-OSS convention)
    k_cache, v_cache  [pages, kv_heads, page_size, D] of qkv's dtype or float8_e4m3fn, any strides with a
                contiguous last dimension; D 64 or 128
    page_table  int32 [B, pages per sequence]
    cu_q        int32 [B + 1]: rows of sequence b are cu_q[b] .. cu_q[b + 1] - 1
    kv_lens     int32 [B]: positions held once the new tokens are in; those are its last ones
    workspace   scratch of ``paged_workspace`` instead of the stream's own
    Rows that belong to no sequence are not written (in a new q_out they hold anything).
    """
    n, d = qkv.shape[0], k_cache.shape[-1]
    cache, batch = _paged_call(qkv, k_cache, v_cache, page_table, cu_q, kv_lens, n, workspace)
    if qkv.dim() != 2 or qkv.shape[1] != (n_q_heads + 2 * cache.n_kv_heads) * d or (n and qkv.stride(1) != 1):
        raise ValueError("qkv must be [tokens, (n_q_heads + 2 kv_heads) * head_dim] with contiguous rows")
    if (cos.dim() != 2 or cos.shape != sin.shape or cos.dtype != sin.dtype or cos.shape[1] * 2 != d
            or cos.dtype not in _DT or not cos.is_contiguous() or not sin.is_contiguous()):
        raise ValueError("cos and sin must be contiguous [positions, head_dim / 2] of fp32, bf16 or f16")
    _require_one_device(qkv, cos, sin, q_out)
    if q_out is None:
        q_out = torch.empty(n, n_q_heads, d, dtype=qkv.dtype, device=qkv.device)
    elif q_out.shape != (n, n_q_heads, d) or q_out.dtype != qkv.dtype or not q_out.is_contiguous():
        raise ValueError("q_out must be contiguous [tokens, n_q_heads, head_dim] of qkv's dtype")
    stream = _stream_of(qkv)
    ws = _paged_workspace(qkv.device, d, stream) if workspace is None else workspace
    row = qkv.stride(0) if n > 1 else qkv.shape[1]
    _lib.check(_lib.lib().tsb_paged_kv_store(
        ctypes.byref(cache), ctypes.byref(batch), qkv.data_ptr(), row, n_q_heads,
        cos.data_ptr(), sin.data_ptr(), _DT[cos.dtype], cos.shape[0], q_out.data_ptr(), ws.data_ptr(), ws.numel(),
        stream))
    return q_out


def paged_attention(q: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor, page_table: torch.Tensor,
                    cu_q: torch.Tensor, kv_lens: torch.Tensor, max_q: int, *, scale: float | None = None,
                    window: int = 0, keep_first: int = 0, sinks: torch.Tensor | None = None,
                    out: torch.Tensor | None = None, workspace: torch.Tensor | None = None) -> torch.Tensor:
    """Causal attention of a ragged batch of new tokens (prompt chunks and
    single decode tokens together) over the pages; [N, n_q_heads, D].

    q           [N, n_q_heads, D] bf16 / f16, last dimension contiguous
    max_q       upper bound of the new tokens of any sequence
    window      0: every earlier position; else the last ``window`` positions and the first ``keep_first``
    sinks       fp32 [n_q_heads]: a logit per head that joins the softmax denominator only
    The other arguments are paged_kv_store's.  A token that sees nothing gives zeros; rows that belong to no sequence
    are not written (in a new ``out`` they hold anything).
    """
    cache, batch = _paged_call(q, k_cache, v_cache, page_table, cu_q, kv_lens, max_q, workspace)
    n, d = q.shape[0], cache.head_dim
    if q.dim() != 3 or q.shape[2] != d or (n and q.stride(2) != 1):
        raise ValueError("q must be [tokens, n_q_heads, head_dim] with a contiguous last dimension")
    if sinks is not None and (sinks.dtype != torch.float32 or sinks.shape != (q.shape[1],) or not sinks.is_contiguous()
                              or sinks.get_device() != q.get_device()):
        raise ValueError("sinks must be fp32 [n_q_heads] on the GPU")
    if out is None:
        out = torch.empty(n, q.shape[1], d, dtype=q.dtype, device=q.device)
    elif out.shape != q.shape or out.dtype != q.dtype or not out.is_contiguous() or out.device != q.device:
        raise ValueError("out must be contiguous, like q")
    stream = _stream_of(q)
    ws = _paged_workspace(q.device, d, stream) if workspace is None else workspace
    _lib.check(_lib.lib().tsb_paged_attention(
        ctypes.byref(cache), ctypes.byref(batch), q.data_ptr(), q.stride(0), q.stride(1), q.shape[1], window,
        keep_first, None if sinks is None else sinks.data_ptr(), d ** -0.5 if scale is None else scale,
        out.data_ptr(), ws.data_ptr(), ws.numel(), stream))
    return out


def sample_tokens(logits: torch.Tensor, noise: torch.Tensor | None = None, *,
                  temperature: torch.Tensor | None = None, top_k: torch.Tensor | None = None,
                  top_p: torch.Tensor | None = None,
                  min_p: torch.Tensor | None = None) -> tuple[torch.Tensor, torch.Tensor]:
    """Draw one token per row of logits [B, V] (fp32 / bf16 / f16, contiguous
    rows); returns (tokens int64 [B], logprobs fp32 [B]).

    noise        fp32 [B, V] exponential variates (``torch.empty(B, V).exponential_()``): the kept token with
                 the largest scaled logit - log(noise) is drawn.  None: every row takes its best token.
    temperature  fp32 [B] (None: 1); rows <= 0 take their best token
    top_k        int32 [B], <= 0: all;  top_p fp32 [B], >= 1: all;  min_p fp32 [B], <= 0: all (None: all).
                 Equal logits rank by index; top_p counts the mass that top_k keeps; min_p is relative to
                 the best token; the best token is always kept.
    logprobs     of the drawn tokens under the row's softmax at its temperature, before the filters
    """
    _require_one_device(logits, noise, temperature, top_k, top_p, min_p)
    if logits.dim() != 2 or logits.dtype not in _DT:
        raise ValueError("logits must be [rows, vocabulary] of fp32, bf16 or f16")
    rows, vocab = logits.shape
    if vocab == 0:
        raise ValueError("the vocabulary is empty")
    if vocab > 1 and logits.stride(1) != 1:
        raise ValueError("logits must have contiguous rows")
    if noise is not None and (noise.shape != logits.shape or noise.dtype != torch.float32
                              or (vocab > 1 and noise.stride(1) != 1)):
        raise ValueError("noise must be fp32, shaped like logits, with contiguous rows")
    for name, t, dt in (("temperature", temperature, torch.float32), ("top_k", top_k, torch.int32),
                        ("top_p", top_p, torch.float32), ("min_p", min_p, torch.float32)):
        if t is not None and (t.shape != (rows,) or t.dtype != dt or not t.is_contiguous()):
            raise ValueError(f"{name} must be contiguous {dt} of one entry per row")
    tokens = torch.empty(rows, dtype=torch.int64, device=logits.device)
    logprobs = torch.empty(rows, dtype=torch.float32, device=logits.device)
    row = logits.stride(0) if rows > 1 else vocab
    noise_row = 0 if noise is None else noise.stride(0) if rows > 1 else vocab
    _lib.check(_lib.lib().tsb_sample(
        logits.data_ptr(), _DT[logits.dtype], rows, vocab, row, _ptr(noise), noise_row, _ptr(temperature),
        _ptr(top_k), _ptr(top_p), _ptr(min_p), tokens.data_ptr(), logprobs.data_ptr(), _stream_of(logits)))
    return tokens, logprobs


# ---------------------------------------------------------------------------
# Drop-in for torch.ops.tinyserve_ggml.ggml_mul_mat_vec
# (tinyserve/csrc/ggml_ops.cu:461-574): same schema, argument meaning, output
# dtype and error messages; callers ggml_forward.py:103-115 and
# ggml_linear.py:77-100 keep working unchanged.
# ---------------------------------------------------------------------------
def ggml_mul_mat_vec(activation: torch.Tensor, weight_data: torch.Tensor, ggml_type: int,
                     out_features: int, in_features: int) -> torch.Tensor:
    if not activation.is_cuda:
        raise RuntimeError("activation must be on CUDA")
    if not weight_data.is_cuda:
        raise RuntimeError("weight_data must be on CUDA")
    if weight_data.dtype != torch.uint8:
        raise RuntimeError("weight_data must be uint8")
    if ggml_type not in FORMATS or ggml_type == TSB_MXFP4:
        raise RuntimeError(f"Unsupported ggml_type: {ggml_type}. Supported: Q8_0(8), Q4_K(12), Q5_K(13), Q6_K(14)")
    _, bb, be = FORMATS[ggml_type]
    if in_features % 32 or (out_features * in_features) % be:
        raise RuntimeError(f"in_features ({in_features}) must be divisible by block_elements ({be})")
    expected = out_features * in_features // be * bb
    if weight_data.numel() < expected:
        raise RuntimeError(f"weight_data too small: got {weight_data.numel()} bytes, expected {expected}")
    act = activation.contiguous().view(-1)
    if act.numel() < in_features:
        raise RuntimeError(f"activation too small: got {act.numel()} elements, expected {in_features}")
    if act.dtype not in _DT:
        act = act.float()
    y = quant_matvec(ggml_type, weight_data, None, out_features, in_features, act[:in_features].view(1, -1),
                     out_dtype=activation.dtype if activation.dtype in _DT else torch.float32)
    return y.view(1, out_features).to(activation.dtype)


_registered = False


def register_torch_op() -> None:
    """Register ``torch.ops.tinyserve_ggml.ggml_mul_mat_vec`` (schema of ggml_ops.cu:571-574)."""
    global _registered
    if _registered or hasattr(torch.ops, "tinyserve_ggml") and hasattr(torch.ops.tinyserve_ggml, "ggml_mul_mat_vec"):
        _registered = True
        return
    lib = torch.library.Library("tinyserve_ggml", "DEF")
    lib.define("ggml_mul_mat_vec(Tensor activation, Tensor weight_data, int ggml_type, int out_features, "
               "int in_features) -> Tensor")
    lib.impl("ggml_mul_mat_vec", ggml_mul_mat_vec, "CUDA")
    register_torch_op._lib = lib  # keep the Library object alive
    _registered = True


def mxfp4_weight_views(blocks: torch.Tensor, scales: torch.Tensor, rows: int, cols: int):
    """Validate MXFP4 tensors of a [rows, cols] weight (blocks [rows, cols/32, 16], scales [rows, cols/32])."""
    nb, ns = mxfp4_split(rows, cols)
    if blocks.numel() != nb or scales.numel() != ns:
        raise ValueError(f"MXFP4 [{rows},{cols}] needs {nb} block bytes and {ns} scale bytes")
    return blocks, scales
