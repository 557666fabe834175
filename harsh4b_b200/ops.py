"""Operator-level wrappers over the C ABI, on torch CUDA tensors.

Each function mirrors one call the reference's CPU path makes (the C ABI
declarations in include/harsh4b_b200.h cite the reference lines). Inputs
must already be CUDA tensors; nothing here copies to or from the host.
"""
from __future__ import annotations

import ctypes
from functools import lru_cache

import torch

from ._lib import PagedKvDesc, check, lib, stream_handle


def _dev(tensor: torch.Tensor, dtype: torch.dtype, name: str) -> int:
    if not isinstance(tensor, torch.Tensor) or not tensor.is_cuda:
        raise ValueError(f"{name} must be a CUDA tensor")
    if tensor.dtype != dtype:
        raise ValueError(f"{name} must be {dtype}, got {tensor.dtype}")
    if not tensor.is_contiguous():
        raise ValueError(f"{name} must be contiguous")
    return tensor.data_ptr()


def int4_i8_gemv(x8: torch.Tensor, weights: torch.Tensor, scales: torch.Tensor, activation_scale: float,
                 *, out: torch.Tensor | None = None, acc: torch.Tensor | None = None):
    """litespark_int4_i8_gemv on the GPU: returns (fp32 out[rows], int32 acc[rows] or None)."""
    rows, packed = weights.shape
    out = torch.empty(rows, dtype=torch.float32, device=weights.device) if out is None else out
    check(lib().h4b_int4_i8_gemv(_dev(x8, torch.int8, "x8"), _dev(weights, torch.uint8, "weights"),
                                 _dev(scales, torch.float32, "scales"), float(activation_scale),
                                 _dev(out, torch.float32, "out"),
                                 _dev(acc, torch.int32, "acc") if acc is not None else None,
                                 rows, 2 * packed, stream_handle()), "h4b_int4_i8_gemv")
    return out, acc


def int4_gemv_fused_quant(values: torch.Tensor, weights: torch.Tensor, scales: torch.Tensor,
                          *, out: torch.Tensor | None = None, acc: torch.Tensor | None = None,
                          scale: torch.Tensor | None = None, pdl: bool = False):
    """quantize_activation + int4 GEMV in one kernel: returns (out, acc, act_scale tensor[1]).
    pdl=True launches with programmatic dependent launch (H4B_LAUNCH_PDL)."""
    rows, packed = weights.shape
    out = torch.empty(rows, dtype=torch.float32, device=weights.device) if out is None else out
    scale = torch.empty(1, dtype=torch.float32, device=weights.device) if scale is None else scale
    check(lib().h4b_int4_gemv_fused_quant_ex(_dev(values, torch.float32, "values"),
                                             _dev(weights, torch.uint8, "weights"),
                                             _dev(scales, torch.float32, "scales"), _dev(out, torch.float32, "out"),
                                             _dev(acc, torch.int32, "acc") if acc is not None else None,
                                             _dev(scale, torch.float32, "scale"), rows, 2 * packed,
                                             1 if pdl else 0, stream_handle()),
          "h4b_int4_gemv_fused_quant_ex")
    return out, acc, scale


def quantize_activation(values: torch.Tensor, quantized: torch.Tensor | None = None):
    """Returns (int8 tensor, dequant scale tensor[1])."""
    quantized = torch.empty(values.numel(), dtype=torch.int8, device=values.device) if quantized is None else quantized
    if quantized.numel() < values.numel():
        raise ValueError("int8 output buffer is smaller than the activation")
    scale = torch.empty(1, dtype=torch.float32, device=values.device)
    check(lib().h4b_quantize_activation(_dev(values, torch.float32, "values"),
                                        _dev(quantized, torch.int8, "quantized"), scale.data_ptr(),
                                        values.numel(), stream_handle()), "h4b_quantize_activation")
    return quantized, scale


def rmsnorm(x: torch.Tensor, weight: torch.Tensor, eps: float, out: torch.Tensor | None = None) -> torch.Tensor:
    out = torch.empty_like(x) if out is None else out
    check(lib().h4b_rmsnorm(_dev(x, torch.float32, "x"), _dev(weight, torch.float32, "weight"),
                            _dev(out, torch.float32, "out"), x.numel(), float(eps), stream_handle()), "h4b_rmsnorm")
    return out


def add_inplace(x: torch.Tensor, y: torch.Tensor) -> torch.Tensor:
    check(lib().h4b_add_inplace(_dev(x, torch.float32, "x"), _dev(y, torch.float32, "y"), x.numel(),
                                stream_handle()), "h4b_add_inplace")
    return x


def gqa_decode(query: torch.Tensor, keys: torch.Tensor, values: torch.Tensor, context: int,
               kv_heads: int, groups: int, *, scores: torch.Tensor | None = None,
               out: torch.Tensor | None = None) -> torch.Tensor:
    """litespark_gqa_decode on the GPU; keys/values fp32 [capacity, kv_heads, head_dim]."""
    capacity, _, head_dim = keys.shape
    q_heads = kv_heads * groups
    scores = torch.empty(q_heads * capacity, dtype=torch.float32, device=query.device) if scores is None else scores
    out = torch.empty(q_heads, head_dim, dtype=torch.float32, device=query.device) if out is None else out
    check(lib().h4b_gqa_decode(_dev(query, torch.float32, "query"), _dev(keys, torch.float32, "keys"),
                               _dev(values, torch.float32, "values"), _dev(scores, torch.float32, "scores"),
                               _dev(out, torch.float32, "out"), context, kv_heads, groups, head_dim, capacity,
                               stream_handle()), "h4b_gqa_decode")
    return out


def gqa_decode_noalloc(query: torch.Tensor, keys: torch.Tensor, values: torch.Tensor, context: int,
                       kv_heads: int, groups: int, *, out: torch.Tensor | None = None) -> torch.Tensor:
    """gqa_decode without a scratch buffer, for callers that cannot allocate
    device memory when attention runs (see h4b_gqa_decode_noalloc in
    include/harsh4b_b200.h): the split partials live in a fixed 1 MiB array
    inside the library, so concurrent calls on different streams race."""
    head_dim = keys.shape[-1]
    if out is None:
        raise ValueError("gqa_decode_noalloc allocates nothing: pass `out` (q_heads x head_dim fp32)")
    check(lib().h4b_gqa_decode_noalloc(_dev(query, torch.float32, "query"), _dev(keys, torch.float32, "keys"),
                                       _dev(values, torch.float32, "values"), _dev(out, torch.float32, "out"),
                                       context, kv_heads, groups, head_dim, stream_handle()),
          "h4b_gqa_decode_noalloc")
    return out


def embedding(token: torch.Tensor, table: torch.Tensor, scales: torch.Tensor,
              out: torch.Tensor | None = None) -> torch.Tensor:
    vocab, packed = table.shape
    out = torch.empty(2 * packed, dtype=torch.float32, device=table.device) if out is None else out
    check(lib().h4b_embedding(_dev(token, torch.int32, "token"), _dev(table, torch.uint8, "table"),
                              _dev(scales, torch.float32, "scales"), _dev(out, torch.float32, "out"), vocab,
                              2 * packed, stream_handle()), "h4b_embedding")
    return out


def argmax(logits: torch.Tensor, out: torch.Tensor | None = None) -> torch.Tensor:
    out = torch.empty(1, dtype=torch.int32, device=logits.device) if out is None else out
    check(lib().h4b_argmax(_dev(logits, torch.float32, "logits"), logits.numel(), _dev(out, torch.int32, "out"),
                           stream_handle()), "h4b_argmax")
    return out


def sample(logits: torch.Tensor, generated: torch.Tensor | None, uniform: float, *, temperature: float = 0.7,
           top_k: int = 50, top_p: float = 0.9, repetition_penalty: float = 1.15, out: torch.Tensor | None = None,
           scratch: torch.Tensor | None = None, return_candidates: bool = False):
    """h4b_sample: one token from fp32 logits (penalised IN PLACE) on the GPU.
    `generated` holds distinct int32 ids (or None); `uniform` is a draw in
    [0, 1) from the caller's generator. Returns the int32 token tensor[1]
    (and the candidate ids / probabilities when asked)."""
    vocab = logits.numel()
    out = torch.empty(1, dtype=torch.int32, device=logits.device) if out is None else out
    k = min(top_k if top_k > 0 else 50, vocab)
    if scratch is None:
        nbytes = int(lib().h4b_sample_scratch_bytes(vocab, top_k))
        if nbytes < 0:
            check(nbytes, "h4b_sample_scratch_bytes")
        scratch = torch.empty(max(nbytes, 16), dtype=torch.uint8, device=logits.device)
    ids = torch.empty(k, dtype=torch.int32, device=logits.device) if return_candidates else None
    probs = torch.empty(k, dtype=torch.float32, device=logits.device) if return_candidates else None
    n_gen = 0 if generated is None else generated.numel()
    check(lib().h4b_sample(_dev(logits, torch.float32, "logits"), vocab,
                           _dev(generated, torch.int32, "generated") if n_gen else None, n_gen, float(temperature),
                           int(top_k), float(top_p), float(repetition_penalty), float(uniform),
                           _dev(out, torch.int32, "out"), ids.data_ptr() if ids is not None else None,
                           probs.data_ptr() if probs is not None else None, scratch.data_ptr(), stream_handle()),
          "h4b_sample")
    return (out, ids, probs) if return_candidates else out


def quantize_rows(values: torch.Tensor):
    """Per-token int8 quantisation of fp32 [M, K]: returns (x8, scales[M], sums[M])."""
    rows, width = values.shape
    x8 = torch.empty(rows, width, dtype=torch.int8, device=values.device)
    scales = torch.empty(rows, dtype=torch.float32, device=values.device)
    sums = torch.empty(rows, dtype=torch.int32, device=values.device)
    check(lib().h4b_quantize_rows(_dev(values, torch.float32, "values"), x8.data_ptr(), scales.data_ptr(),
                                  sums.data_ptr(), rows, width, stream_handle()), "h4b_quantize_rows")
    return x8, scales, sums


GEMM_KERNELS = {"auto": 0, "tcgen05": 1, "mma_sync": 2}


def int4_gemm(x8: torch.Tensor, act_scales: torch.Tensor, act_sums: torch.Tensor, weights: torch.Tensor,
              scales: torch.Tensor, out: torch.Tensor | None = None, kernel: str = "auto") -> torch.Tensor:
    """h4b_int4_gemm_ex: fp32 [M, N] from int8 activations [M, K] and int4
    weights [N, K/2]; `kernel` picks tcgen05, mma.sync or the automatic choice."""
    tokens, width = x8.shape
    rows = weights.shape[0]
    out = torch.empty(tokens, rows, dtype=torch.float32, device=x8.device) if out is None else out
    check(lib().h4b_int4_gemm_ex(_dev(x8, torch.int8, "x8"), _dev(act_scales, torch.float32, "act_scales"),
                                 _dev(act_sums, torch.int32, "act_sums"), _dev(weights, torch.uint8, "weights"),
                                 _dev(scales, torch.float32, "scales"), _dev(out, torch.float32, "out"), tokens,
                                 rows, width, GEMM_KERNELS[kernel], stream_handle()), "h4b_int4_gemm_ex")
    return out


def int4_gemm_acc(x8: torch.Tensor, act_scales: torch.Tensor, act_sums: torch.Tensor, weights: torch.Tensor,
                  scales: torch.Tensor, acc: torch.Tensor, out: torch.Tensor | None = None,
                  residual: bool = False) -> torch.Tensor:
    """h4b_int4_gemm_acc: int4_gemm with the K sum split over CTAs through the
    zeroed int32 buffer `acc` [M, N] (left zero); `residual` adds into `out`."""
    tokens, width = x8.shape
    rows = weights.shape[0]
    if residual and out is None:
        raise ValueError("residual needs out")
    if acc.numel() < tokens * rows:
        raise ValueError(f"acc holds {acc.numel()} int32, needs {tokens * rows}")
    out = torch.empty(tokens, rows, dtype=torch.float32, device=x8.device) if out is None else out
    check(lib().h4b_int4_gemm_acc(_dev(x8, torch.int8, "x8"), _dev(act_scales, torch.float32, "act_scales"),
                                  _dev(act_sums, torch.int32, "act_sums"), _dev(weights, torch.uint8, "weights"),
                                  _dev(scales, torch.float32, "scales"), _dev(out, torch.float32, "out"),
                                  _dev(acc, torch.int32, "acc"), tokens, rows, width, 1 if residual else 0,
                                  stream_handle()), "h4b_int4_gemm_acc")
    return out


def int4_gemm_rows(values: torch.Tensor, weights: torch.Tensor, scales: torch.Tensor,
                   kernel: str = "auto") -> torch.Tensor:
    """fp32 [M, K] -> fp32 [M, N]: per-token quantisation, then the batched GEMM."""
    x8, act_scales, sums = quantize_rows(values)
    return int4_gemm(x8, act_scales, sums, weights, scales, kernel=kernel)


def int4_gemv_absmax(values: torch.Tensor, absmax: torch.Tensor, weights: torch.Tensor, scales: torch.Tensor,
                     acc: torch.Tensor, out: torch.Tensor | None = None) -> torch.Tensor:
    """Quantise with a given device absmax, GEMV, int32 row sums into `acc`."""
    rows, packed = weights.shape
    check(lib().h4b_int4_gemv_absmax(_dev(values, torch.float32, "values"), _dev(absmax, torch.float32, "absmax"),
                                     _dev(weights, torch.uint8, "weights"), _dev(scales, torch.float32, "scales"),
                                     _dev(out, torch.float32, "out") if out is not None else None,
                                     _dev(acc, torch.int32, "acc"), rows, 2 * packed, stream_handle()),
          "h4b_int4_gemv_absmax")
    return acc


def residual_acc(x: torch.Tensor, acc: torch.Tensor, absmax: torch.Tensor, scales: torch.Tensor) -> torch.Tensor:
    """x += float(acc) * dequant(absmax) * scales (in place)."""
    check(lib().h4b_residual_acc(_dev(x, torch.float32, "x"), _dev(acc, torch.int32, "acc"),
                                 _dev(absmax, torch.float32, "absmax"), _dev(scales, torch.float32, "scales"),
                                 x.numel(), stream_handle()), "h4b_residual_acc")
    return x


# ---- paged K/V cache -------------------------------------------------------------
# A decode step calls these once a layer, so what they do on the host is kept
# to a few microseconds: one pass over the tensors' attributes, one C call.
_PAGED_DTYPES = {torch.float16: 1, torch.bfloat16: 2}  # H4B_FP16, H4B_BF16


def _on(tensor: torch.Tensor, dtype: torch.dtype, name: str, device: int) -> int:
    """Data pointer of a contiguous tensor on CUDA device `device`."""
    try:
        if tensor.get_device() == device and tensor.dtype is dtype and tensor.is_contiguous() and device >= 0:
            return tensor.data_ptr()
    except AttributeError:  # not a tensor
        pass
    _dev(tensor, dtype, name)
    raise ValueError(f"{name} must be on the device of the other tensors, cuda:{device}, got {tensor.device}")


def _rows(tensor: torch.Tensor, dtype: torch.dtype, name: str, device: int) -> int:
    """Data pointer of a tensor on CUDA device `device` whose rows (dim 0) may be strided."""
    if isinstance(tensor, torch.Tensor) and tensor.get_device() == device >= 0 and tensor.dtype is dtype \
            and (tensor.is_contiguous() or tensor[:1].squeeze(0).is_contiguous()):
        return tensor.data_ptr()
    _on(tensor[:1].squeeze(0) if isinstance(tensor, torch.Tensor) else tensor, dtype, name, device)
    raise ValueError(f"{name} must be contiguous within each row")


def _raw_stream(index: int) -> int:
    """The current stream's handle, as stream_handle() but without the stream object."""
    return torch._C._cuda_getCurrentRawStream(index)


def _here(device: int) -> int:
    """The current stream of the tensors' device, which has to be the current
    one: the library launches there."""
    current = torch.cuda.current_device()
    if device != current:
        raise ValueError(f"the tensors must be on the current device, cuda:{current}, not cuda:{device}")
    return _raw_stream(device)


def _paged(k_pages, v_pages, page_table, q_offsets, kv_lens, tokens: int) -> PagedKvDesc:
    """The h4b_paged_kv of one layer's pages and a batch's tables."""
    dtype = k_pages.dtype
    code = _PAGED_DTYPES.get(dtype)
    if code is None:
        raise ValueError(f"k_pages must be float16 or bfloat16, got {dtype}")
    shape, table = k_pages.shape, page_table.shape
    if len(shape) != 4 or shape != v_pages.shape:
        raise ValueError("k_pages and v_pages must be [pages][kv_heads][page_size][head_dim]")
    sequences = kv_lens.numel()
    if len(table) != 2 or table[0] != sequences or q_offsets.numel() != sequences + 1:
        raise ValueError("page_table must be [sequences][pages each], q_offsets [sequences + 1], kv_lens [sequences]")
    device = k_pages.get_device()
    return PagedKvDesc(_on(k_pages, dtype, "k_pages", device), _on(v_pages, dtype, "v_pages", device),
                       _on(page_table, torch.int32, "page_table", device),
                       _on(q_offsets, torch.int32, "q_offsets", device),
                       _on(kv_lens, torch.int32, "kv_lens", device), code, shape[0], shape[2], shape[1], shape[3],
                       sequences, table[1], tokens)


def paged_append(qkv: torch.Tensor, k_pages: torch.Tensor, v_pages: torch.Tensor, page_table: torch.Tensor,
                 q_offsets: torch.Tensor, kv_lens: torch.Tensor, *, heads: int, norm_q: torch.Tensor | None = None,
                 norm_k: torch.Tensor | None = None, eps: float = 1e-6, rope_cos: torch.Tensor | None = None,
                 rope_sin: torch.Tensor | None = None, out: torch.Tensor | None = None) -> torch.Tensor:
    """h4b_paged_append: the new tokens' k and v into one layer's pages, their
    q heads back. `qkv` holds `heads` q heads, the k heads and the v heads of
    every new token ([tokens][(heads + 2 kv_heads) * head_dim], fp32 or the
    cache's type, rows may be strided); q and k are RMS-normalised with
    `norm_q` / `norm_k` and rotated with `rope_cos` / `rope_sin` where given.
    Returns q [tokens][heads][head_dim] in the cache's type."""
    tokens, width = qkv.shape if qkv.dim() == 2 else (0, -1)
    dtype, source, device = k_pages.dtype, qkv.dtype, k_pages.get_device()
    kv = _paged(k_pages, v_pages, page_table, q_offsets, kv_lens, tokens)
    head_dim = kv.head_dim
    if width != (heads + 2 * kv.kv_heads) * head_dim:
        raise ValueError("qkv must be [tokens][(heads + 2 kv_heads) * head_dim]")
    if source is not torch.float32 and source is not dtype:
        raise ValueError(f"qkv must be float32 or {dtype}, got {source}")
    if out is None:
        out = torch.empty((tokens, heads, head_dim), dtype=dtype, device=qkv.device)
    elif out.shape != (tokens, heads, head_dim):
        raise ValueError("out must be [tokens][heads][head_dim]")
    weights = [None, None]
    for k, (name, norm) in enumerate((("norm_q", norm_q), ("norm_k", norm_k))):
        if norm is not None:
            if norm.numel() != head_dim:
                raise ValueError(f"{name} must hold head_dim values")
            weights[k] = _on(norm, torch.float32, name, device)
    cos = sin = None
    positions = 0
    if rope_cos is not None or rope_sin is not None:
        if rope_cos is None or rope_sin is None or rope_cos.shape != rope_sin.shape or rope_cos.dim() != 2 \
                or rope_cos.shape[1] != head_dim // 2:
            raise ValueError("rope_cos and rope_sin must be [positions][head_dim / 2]")
        positions = rope_cos.shape[0]
        cos, sin = _on(rope_cos, torch.float32, "rope_cos", device), _on(rope_sin, torch.float32, "rope_sin", device)
    check(lib().h4b_paged_append(ctypes.byref(kv), _rows(qkv, source, "qkv", device),
                                 0 if source is torch.float32 else kv.dtype, qkv.stride(0) if tokens > 1 else width, heads,
                                 weights[0], weights[1], eps, cos, sin, positions, _rows(out, dtype, "out", device),
                                 out.stride(0) if tokens > 1 else heads * head_dim, _here(device)), "h4b_paged_append")
    return out


@lru_cache(None)
def _paged_workspace_bytes(head_dim: int, device: int) -> int:
    with torch.cuda.device(device):
        nbytes = int(lib().h4b_paged_attention_workspace_bytes(head_dim))
    if nbytes < 0:
        check(nbytes, "h4b_paged_attention_workspace_bytes")
    return nbytes


def paged_workspace(head_dim: int = 128, device=None) -> torch.Tensor:
    """A workspace for paged_attention calls that follow each other (one
    stream): zeroed once, every call leaves it ready for the next."""
    device = torch.device("cuda", torch.cuda.current_device()) if device is None else torch.device(device)
    index = torch.cuda.current_device() if device.index is None else device.index
    return torch.zeros(_paged_workspace_bytes(head_dim, index), dtype=torch.uint8, device=device)


def paged_attention(q: torch.Tensor, k_pages: torch.Tensor, v_pages: torch.Tensor, page_table: torch.Tensor,
                    q_offsets: torch.Tensor, kv_lens: torch.Tensor, *, max_query: int | None = None, window: int = 0,
                    sinks: int = 0, scale: float | None = None, out: torch.Tensor | None = None,
                    lse: torch.Tensor | None = None, workspace: torch.Tensor | None = None) -> torch.Tensor:
    """h4b_paged_attention: causal attention of a ragged batch's new tokens
    (q [tokens][heads][head_dim], rows may be strided; sequence b's are rows
    q_offsets[b] .. q_offsets[b + 1] - 1) over their sequences' pages, which
    hold the new tokens already (paged_append). `window` > 0: a token sees the
    last `window` keys (itself among them) and the first `sinks`. `max_query`
    is the longest chunk to expect (it picks the kernel; by default 1 when
    there are no more rows than sequences, else all rows). `scale` is positive
    (1 / sqrt(head_dim) by default). `lse`, if given, receives the float32
    [tokens][heads] log-sum-exp. `workspace`: from paged_workspace, kept between
    calls (one is made per call otherwise)."""
    if q.dim() != 3:
        raise ValueError("q must be [tokens][heads][head_dim]")
    tokens, heads, head_dim = shape = q.shape
    dtype, device = k_pages.dtype, k_pages.get_device()
    kv = _paged(k_pages, v_pages, page_table, q_offsets, kv_lens, tokens)
    if head_dim != kv.head_dim or heads % kv.kv_heads:
        raise ValueError("q must have the cache's head_dim and a multiple of its kv heads")
    if out is None:
        out = torch.empty(shape, dtype=dtype, device=q.device)
    elif out.shape != shape:
        raise ValueError("out must have q's shape")
    if lse is not None and lse.shape != (tokens, heads):
        raise ValueError("lse must be [tokens][heads]")
    if max_query is None:
        max_query = 1 if tokens <= kv.sequences else tokens
    if workspace is None:
        workspace = paged_workspace(head_dim, q.device)
    if max(window, sinks, max_query) > 0x7fffffff or min(window, sinks, max_query) < -0x80000000:
        raise ValueError("window, sinks and max_query must fit 32 bits")
    width = heads * head_dim
    several = tokens > 1
    check(lib().h4b_paged_attention(ctypes.byref(kv), _rows(q, dtype, "q", device), q.stride(0) if several else width,
                                    heads, head_dim ** -0.5 if scale is None else scale, window, sinks, max_query,
                                    _rows(out, dtype, "out", device), out.stride(0) if several else width,
                                    None if lse is None else _on(lse, torch.float32, "lse", device),
                                    _on(workspace, torch.uint8, "workspace", device), workspace.numel(),
                                    _here(device)), "h4b_paged_attention")
    return out


def copy_pages(k_pages: torch.Tensor, v_pages: torch.Tensor, src: torch.Tensor, dst: torch.Tensor) -> None:
    """h4b_pages_copy: page src[i] to page dst[i] in every layer of
    [layers][pages][kv_heads][page_size][head_dim] (or one layer's [pages]...)
    caches of any type; int32 ids on the device. No page may be the
    destination of two moves, nor a source and a destination."""
    shape, dtype, count, device = k_pages.shape, k_pages.dtype, src.numel(), k_pages.get_device()
    if shape != v_pages.shape or len(shape) not in (4, 5):
        raise ValueError("k_pages and v_pages must be [layers][pages][kv_heads][page_size][head_dim]")
    if count != dst.numel():
        raise ValueError("src and dst must hold as many page ids")
    pages, kv_heads, page_size, head_dim = shape[-4:]
    check(lib().h4b_pages_copy(_on(k_pages, dtype, "k_pages", device), _on(v_pages, dtype, "v_pages", device),
                               shape[0] if len(shape) == 5 else 1, pages,
                               kv_heads * page_size * head_dim * k_pages.element_size(),
                               _on(src, torch.int32, "src", device), _on(dst, torch.int32, "dst", device), count,
                               _here(device)), "h4b_pages_copy")
