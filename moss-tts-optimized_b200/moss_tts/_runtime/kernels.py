"""Decode operators with the reference's module-level signatures, on B200 CUDA kernels.

Mirrors ``src/moss_tts/_runtime/kernels.py`` of the reference: ``embedding_sum``,
``rmsnorm``, ``add_rmsnorm``, ``linear_decode``, ``silu_mul`` and
``qk_rope_decode`` keep their names, arguments and return values. All launches
go to PyTorch's current CUDA stream, outputs are allocated with ``torch.empty``
(as the reference does), and there is no CPU fallback: the C library must be
built and the tensors must live on a CUDA device.
"""
import torch

from . import native

_ATTN_SPLITS = 16


def _cuda(*tensors):
    dev = None
    for t in tensors:
        if t is None:
            continue
        if not isinstance(t, torch.Tensor) or not t.is_cuda:
            raise ValueError("CUDA tensors required (there is no CPU path)")
        if dev is None:
            dev = t.device
        elif t.device != dev:
            raise ValueError("All tensors must be on the same CUDA device")
        if not t.is_contiguous():
            raise ValueError("Contiguous tensors required")
    return dev


def _bf16(*tensors):
    for t in tensors:
        if t is not None and t.dtype != torch.bfloat16:
            raise ValueError("bf16 tensors required")


def embedding_sum(ids, text_weight, audio_weight):
    """Text embedding + 32 audio-codebook embeddings, bf16 rounding after each add.

    Same contract as the reference (``kernels.py:21-26``): ``ids`` int64
    ``[..., 1 + n_vq]``, ``text_weight`` ``[V, H]``, ``audio_weight`` ``[n_vq, V_a, H]``.
    """
    ids = ids.contiguous()
    _cuda(ids, text_weight, audio_weight)
    _bf16(text_weight, audio_weight)
    if ids.dtype != torch.long or ids.shape[-1] != audio_weight.shape[0] + 1:
        raise ValueError("ids must be int64 [..., 1 + n_vq]")
    h = text_weight.shape[-1]
    out = torch.empty((*ids.shape[:-1], h), device=ids.device, dtype=text_weight.dtype)
    tokens = ids.numel() // ids.shape[-1]
    native.call("mt_embedding_sum", ids.data_ptr(), text_weight.data_ptr(), audio_weight.data_ptr(),
                out.data_ptr(), tokens, h, text_weight.shape[0], audio_weight.shape[1],
                audio_weight.shape[0], None, 0, native.stream_of(ids))
    return out


def rmsnorm(x, weight, eps):
    """Qwen3 RMSNorm over the last dimension (``kernels.py:62-66``)."""
    x = x.contiguous()
    _cuda(x, weight)
    _bf16(x, weight)
    y = torch.empty_like(x)
    native.call("mt_rmsnorm", x.data_ptr(), None, weight.data_ptr(), None, y.data_ptr(),
                x.numel() // x.shape[-1], x.shape[-1], float(eps), 0, native.stream_of(x))
    return y


def add_rmsnorm(x, residual, weight, eps):
    """``(summed, normalized)`` with ``summed = bf16(x + residual)`` (``kernels.py:85-90``)."""
    x, residual = x.contiguous(), residual.contiguous()
    _cuda(x, residual, weight)
    _bf16(x, residual, weight)
    if x.shape != residual.shape:
        raise ValueError("x and residual shapes differ")
    summed, normalized = torch.empty_like(x), torch.empty_like(x)
    native.call("mt_rmsnorm", x.data_ptr(), residual.data_ptr(), weight.data_ptr(), summed.data_ptr(),
                normalized.data_ptr(), x.numel() // x.shape[-1], x.shape[-1], float(eps), 0,
                native.stream_of(x))
    return summed, normalized


def linear_decode(x, w):
    """bf16 GEMV for up to 8 rows (``kernels.py:102-108``); fp32 accumulation."""
    x = x.contiguous()
    _cuda(x, w)
    _bf16(x, w)
    n, k = w.shape
    rows = x.numel() // x.shape[-1]
    if x.shape[-1] != k or rows > 8:
        raise ValueError("linear_decode expects [..., K] with at most 8 rows")
    y = torch.empty((*x.shape[:-1], n), dtype=x.dtype, device=x.device)
    native.call("mt_bf16_linear", x.data_ptr(), None, None, 0.0, None, w.data_ptr(), y.data_ptr(),
                rows, n, k, 0, 0, native.stream_of(x))
    return y


def silu_mul(x):
    """``bf16(bf16(silu(gate)) * up)`` for ``x = gate || up`` (``kernels.py:132-139``)."""
    x = x.contiguous()
    _cuda(x)
    _bf16(x)
    n = x.shape[-1] // 2
    y = torch.empty((*x.shape[:-1], n), dtype=x.dtype, device=x.device)
    native.call("mt_silu_mul", x.data_ptr(), y.data_ptr(), x.numel() // x.shape[-1], n, 0,
                native.stream_of(x))
    return y


class AttentionScratch:
    """Per-device scratch for the split-K decode attention (partials, LSE, tickets)."""

    def __init__(self, device, batch, nq, nkv, splits):
        rep = nq // nkv
        self.splits = splits
        self.partial = torch.empty(batch * nkv * splits * rep * 128, device=device, dtype=torch.float32)
        self.lse = torch.empty(batch * nkv * splits * rep, device=device, dtype=torch.float32)
        self.tickets = torch.zeros(batch * nkv, device=device, dtype=torch.int32)


_scratch = {}


def qk_rope_decode(qkv, q_weight, k_weight, cos, sin, cache, layer_idx, position, eps, backend=None,
                   block=128, warps=4, context_capacity=None, quantize_output=False,
                   native_attention=False, pdl=None):
    """QK-norm + RoPE + KV-cache write + split-K decode attention for one token.

    Same call signature as the reference (``kernels.py:211-251``). ``cos``/``sin`` are the
    bf16 RoPE tables ``[max_len, 128]`` (rows selected on the device by ``position``);
    ``cache`` exposes ``cache.layers[layer_idx].keys/.values`` of shape ``[1, nkv, L, 128]``.
    Returns the attention output ``[1, 1, nq * 128]``. The reference's tile/warp/backend
    knobs select Triton variants and are validated but otherwise unused; int8 output
    quantization (``quantize_output``) belongs to the W4A8 path and is rejected.
    """
    if backend is not None or quantize_output or pdl:
        raise ValueError("Only the native fused B200 attention is available")
    kc, vc = cache.layers[layer_idx].keys, cache.layers[layer_idx].values
    _cuda(qkv, q_weight, k_weight, cos, sin, kc, vc, position)
    _bf16(qkv, q_weight, k_weight, cos, sin, kc, vc)
    if kc.ndim != 4 or kc.shape[0] != 1 or kc.shape[-1] != 128 or vc.shape != kc.shape:
        raise ValueError("KV cache must be [1, nkv, L, 128]")
    nkv, length = kc.shape[1], kc.shape[2]
    nq = qkv.shape[-1] // 128 - 2 * nkv
    if position.dtype != torch.long or position.numel() != 1:
        raise ValueError("position must be a one-element int64 CUDA tensor")
    if cos.shape != (length, 128) or sin.shape != cos.shape:
        raise ValueError("RoPE tables must be [L, 128]")
    capacity = length if context_capacity is None else context_capacity
    if not 0 < capacity <= length:
        raise ValueError("Invalid decode attention capacity")
    key = (qkv.device, nq, nkv)
    scratch = _scratch.get(key)
    if scratch is None:
        scratch = _scratch[key] = AttentionScratch(qkv.device, 1, nq, nkv, _ATTN_SPLITS)
    out = torch.empty((1, 1, nq * 128), device=qkv.device, dtype=qkv.dtype)
    native.call("mt_attention_decode", qkv.data_ptr(), q_weight.data_ptr(), k_weight.data_ptr(),
                cos.data_ptr(), sin.data_ptr(), position.data_ptr(), kc.data_ptr(), vc.data_ptr(),
                out.data_ptr(), scratch.partial.data_ptr(), scratch.lse.data_ptr(),
                scratch.tickets.data_ptr(), 1, nq, nkv, length, scratch.splits, float(eps), None, 0,
                native.stream_of(qkv))
    return out


# ---------------------------------------------------------------------------- paged key-value cache
# A call of a few rows runs for 5 to 10 microseconds on the GPU, and Python's checks are what it waits for:
# they read every attribute once and compare devices by index.
_TYPES = {torch.bfloat16: 0, torch.float16: 1}
_DIMS = (64, 128)
_PAGE_SIZES = (16, 32, 64, 128, 256)
_current_device = torch.cuda.current_device
# the address alone, without a Stream object, where torch has the (private) function for it
_raw_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None) or (
    lambda dev: torch.cuda.current_stream(dev).cuda_stream)


def _strides3(name, t, heads, d):
    """Row and head stride of ``t`` ``[rows, heads, D]``, whose D elements are adjacent."""
    row, head, one = t.stride()
    if t.shape[0] <= 1:  # the stride of a dimension of one says nothing
        row = heads * d
    if heads <= 1:
        head = d
    if one != 1 or (row | head) & 7 or row <= 0 or head <= 0 or row >= 1 << 31 or head >= 1 << 31 or t.data_ptr() & 15:
        raise ValueError(f"{name}: D must be adjacent, rows and heads 16-byte aligned and not broadcast")
    return row, head


def _no_backward(a, b, c=None):
    if (a.requires_grad or b.requires_grad or c is not None and c.requires_grad) and torch.is_grad_enabled():
        raise ValueError("There is no backward pass: inputs that require a gradient need torch.no_grad()")


def _query(q, nkv, d):
    """(tokens, heads, row stride, head stride, device index) of the queries."""
    if not isinstance(q, torch.Tensor) or not q.is_cuda:
        raise ValueError("CUDA tensors required (there is no CPU path)")
    if q.dtype not in _TYPES:
        raise ValueError("bf16 or fp16 tensors required")
    if q.ndim != 3:
        raise ValueError("q must be [rows, heads, D]")
    tokens, nq, dq = q.shape
    if dq != d or d not in _DIMS:
        raise ValueError("head_dim must be 64 or 128, the same for queries and keys")
    if nq == 0 or nkv == 0 or nq % nkv or nq // nkv > 64:
        raise ValueError("Query heads must be 1 to 64 times the key heads")
    return tokens, nq, *_strides3("q", q, nq, d), q.get_device()


def _ints(name, t, n, dev):
    """The address of an int32 vector of ``n`` elements (lengths or offsets)."""
    if t.dtype is not torch.int32 or t.shape != (n,) or t.get_device() != dev or not t.is_contiguous():
        raise ValueError(f"{name} must be a contiguous int32 vector of {n} elements on the queries' device")
    return t.data_ptr()


def _status(status, dev):
    if status is None:
        return None
    if status.dtype is not torch.int32 or status.numel() != 1 or status.get_device() != dev:
        raise ValueError("status must be a one-element int32 tensor on the queries' device")
    return status.data_ptr()


def _out(out, shape, like):
    if out is None:
        return torch.empty(shape, device=like.device, dtype=like.dtype)
    if out.shape != shape or out.dtype is not like.dtype or out.get_device() != like.get_device() \
            or not out.is_contiguous() or out.data_ptr() & 31:
        raise ValueError(f"out must be a contiguous, 32-byte aligned {like.dtype} tensor {tuple(shape)} on the "
                         "queries' device")
    return out


def _extent(t):
    """The addresses of a tensor's first byte and behind its last."""
    first = t.data_ptr()
    if not t.numel():
        return first, first
    n = 1
    for size, stride in zip(t.shape, t.stride()):
        n += (size - 1) * stride
    return first, first + n * t.element_size()


def _apart(written, read):
    """Says which output lies in an input's memory, where that is what an entry point has refused: rows are read
    by other blocks than the one that writes them, and some a second time."""
    for name, w in written.items():
        first, past = _extent(w)
        for other, t in (written | read).items():
            # (keys and values may lie side by side)
            if t is not None and name != other and {name, other} != {"k_pages", "v_pages"} \
                    and _extent(t)[0] < past and _extent(t)[1] > first:
                raise ValueError(f"{name} must not lie in the memory of {other}")


def _paged(k_pages, v_pages, page_table, kv_lens, dtype, dev):
    """(``mt_paged_kv`` of one layer's pages as bytes, batch, most tokens of a sequence)."""
    shape = k_pages.shape
    if len(shape) != 4 or v_pages.shape != shape:
        raise ValueError("k_pages and v_pages must be [pages, heads, page_size, D]")
    pages, heads, size, d = shape
    if size not in _PAGE_SIZES:
        raise ValueError("page_size must be a power of two, 16 to 256")
    if d not in _DIMS:
        raise ValueError("head_dim must be 64 or 128, the same for queries and keys")
    if pages < 1 or pages >= 1 << 31 or heads < 1:
        raise ValueError("The cache has no pages")
    if k_pages.dtype is not dtype or v_pages.dtype is not dtype or k_pages.get_device() != dev \
            or v_pages.get_device() != dev:
        raise ValueError("The pages must have the queries' type and device")
    kp, kh, kr, k1 = k_pages.stride()
    vp, vh, vr, v1 = v_pages.stride()
    if pages == 1:  # the stride of a dimension of one says nothing
        kp = vp = heads * size * d
    if heads == 1:
        kh = vh = size * d
    k, v = k_pages.data_ptr(), v_pages.data_ptr()
    if k1 != 1 or v1 != 1 or (kp | kh | kr | vp | vh | vr) & 7 or (k | v) & 15 or min(kp, kh, kr, vp, vh, vr) <= 0:
        raise ValueError("pages: D must be adjacent, pages, heads and rows 16-byte aligned and not broadcast")
    if page_table.dtype is not torch.int32 or page_table.ndim != 2 or page_table.get_device() != dev:
        raise ValueError("page_table must be int32 [batch, max_pages] on the queries' device")
    batch, most = page_table.shape
    row, one = page_table.stride()
    if batch < 1 or most < 1 or most * size > 1 << 30 or (one != 1 and most > 1):
        raise ValueError("page_table must have rows of 1 or more adjacent entries, for up to 2^30 tokens")
    return native.PAGED_KV.pack(k, v, page_table.data_ptr(), _ints("kv_lens", kv_lens, batch, dev), kp, kh, kr, vp, vh,
                                vr, row, pages, heads, size, d, most, batch, _TYPES[dtype]), batch, most * size


def _call_on(dev, name, *args, workspace=None, apart=None):
    """``native.call`` on device ``dev`` and its current stream; ``workspace`` (function, arguments) gives the
    bytes of a workspace, which comes last before the status, flags and stream. It is taken from torch's
    allocator for the one call, so that calls on other streams and captured graphs have one each. ``apart()``
    gives the tensors that are written and those that are read, by name, for a call that is refused."""
    if _current_device() != dev:
        with torch.cuda.device(dev):
            return _call_on(dev, name, *args, workspace=workspace, apart=apart)
    if workspace is not None:
        n = workspace[0](*workspace[1:])
        held = torch.empty(n, device=torch.device("cuda", dev), dtype=torch.uint8) if n else None
        args = [held.data_ptr() if a is _WORKSPACE and n else None if a is _WORKSPACE else a for a in args]
    try:
        native.call(name, *args, _raw_stream(dev))
    except RuntimeError:
        _apart(*apart())
        raise


_WORKSPACE = object()  # stands for the workspace's address in _call_on's arguments


def qk_rope_paged(qkv, q_weight, k_weight, cos, sin, k_pages, v_pages, page_table, kv_lens, cu_seqlens, eps, *,
                  out=None, status=None):
    """QK-norm + RoPE of packed new tokens and their write into a paged key-value cache.

    ``qkv`` ``[tokens, (nq + 2 nkv) * D]`` (bf16 or fp16, rows may be strided); ``cos`` / ``sin`` the RoPE
    tables ``[max_len, D]`` in that type or fp32. Key j of sequence b lies in row ``j % page_size`` of page
    ``page_table[b, j // page_size]`` (int32 ``[batch, max_pages]``) of ``k_pages`` / ``v_pages``
    ``[pages, nkv, page_size, D]`` (any strides with adjacent D; page_size a power of two, 16 to 256; D 64 or
    128). ``kv_lens`` int32 ``[batch]`` counts each sequence's tokens with the new ones; ``cu_seqlens`` int32
    ``[batch + 1]`` are the new tokens' offsets in ``qkv``, or None for one token per sequence, where a sequence
    of length 0 is an empty slot: zeros in its query row, nothing in the pages. Returns the rotated queries
    ``[tokens, nq, D]`` (in ``out`` if given, which has memory of its own); rows behind the last
    sequence are not written.

    Unlike ``qk_rope_decode``, whose intermediate roundings are the reference's, this rounds once, at the
    store. A page that is written must belong to one sequence. ``status`` (int32, one element) takes 1 for a
    position outside the tables (nothing is written for it) and 3 for a page id outside the cache.
    """
    if not isinstance(qkv, torch.Tensor) or not qkv.is_cuda:
        raise ValueError("CUDA tensors required (there is no CPU path)")
    dtype, dev = qkv.dtype, qkv.get_device()
    if dtype not in _TYPES or qkv.ndim != 2:
        raise ValueError("qkv must be bf16 or fp16 [tokens, (nq + 2 nkv) * D]")
    _no_backward(qkv, q_weight, k_weight)
    tokens, width = qkv.shape
    row, one = qkv.stride()
    if tokens <= 1:
        row = width
    if one != 1 or row & 7 or row < width or row >= 1 << 31 or qkv.data_ptr() & 15:
        raise ValueError("qkv must have adjacent elements in 16-byte aligned rows")
    _no_backward(k_pages, v_pages)
    kv, batch, _ = _paged(k_pages, v_pages, page_table, kv_lens, dtype, dev)
    nkv, d = k_pages.shape[1], k_pages.shape[3]
    nq = width // d - 2 * nkv
    if width % d or nq < 1:
        raise ValueError("qkv must hold nq >= 1 query heads and the cache's key and value heads")
    for w in (q_weight, k_weight):
        if w.dtype is not dtype or w.shape != (d,) or w.get_device() != dev or not w.is_contiguous() or w.data_ptr() & 15:
            raise ValueError("q_weight and k_weight must be contiguous [D], of qkv's type and device")
    table, kind = cos.shape, cos.dtype
    if len(table) != 2 or table[1] != d or table[0] < 1 or sin.shape != table:
        raise ValueError("RoPE tables must be [max_len, D]")
    if (kind is not dtype and kind is not torch.float32) or sin.dtype is not kind or cos.get_device() != dev \
            or sin.get_device() != dev or not cos.is_contiguous() or not sin.is_contiguous() \
            or (cos.data_ptr() | sin.data_ptr()) & 15:
        raise ValueError("RoPE tables must be contiguous, in qkv's type or fp32, on its device")
    if cu_seqlens is None and tokens != batch:
        raise ValueError("Without cu_seqlens there is one token per sequence")
    cu = None if cu_seqlens is None else _ints("cu_seqlens", cu_seqlens, batch + 1, dev)
    st = _status(status, dev)
    out = _out(out, (tokens, nq, d), qkv)
    if tokens:
        _call_on(dev, "mt_qk_rope_paged", qkv.data_ptr(), q_weight.data_ptr(), k_weight.data_ptr(), cos.data_ptr(),
                 sin.data_ptr(), table[0], 1 if kind is torch.float32 else 0, kv, cu, tokens, nq, row, out.data_ptr(),
                 eps, st, 0,
                 apart=lambda: ({"out": out, "k_pages": k_pages, "v_pages": v_pages},
                                {"qkv": qkv, "q_weight": q_weight, "k_weight": k_weight, "cos": cos, "sin": sin,
                                 "page_table": page_table, "kv_lens": kv_lens, "cu_seqlens": cu_seqlens}))
    return out


def paged_attention_decode(q, k_pages, v_pages, page_table, kv_lens, *, scale=None, out=None, status=None):
    """Attention of one new token per sequence over a paged key-value cache (``qk_rope_paged``'s).

    ``q`` ``[batch, nq, D]`` (bf16 or fp16; rows and heads may be strided); query head h reads key head
    ``h // (nq / nkv)``. Returns ``softmax(scale q k^T) v`` over keys ``0 .. kv_lens[b] - 1``, ``[batch, nq, D]``
    (in ``out`` if given, which has memory of its own); ``scale`` defaults to ``1 / sqrt(D)``. A sequence of
    length 0 gives zeros; an infinite value may leave NaN.
    ``status`` as in ``qk_rope_paged``: a length beyond the page table (1) is cut, a page id outside the
    cache (3) reads as zeros.
    """
    _, nkv, _, d = k_pages.shape
    rows, nq, row, head, dev = _query(q, nkv, d)
    _no_backward(q, k_pages, v_pages)
    kv, batch, _ = _paged(k_pages, v_pages, page_table, kv_lens, q.dtype, dev)
    if rows != batch:
        raise ValueError("page_table must have a row for each query row")
    st = _status(status, dev)
    out = _out(out, (batch, nq, d), q)
    _call_on(dev, "mt_paged_attention_decode", q.data_ptr(), row, head, kv, nq, d ** -0.5 if scale is None else scale,
             out.data_ptr(), _WORKSPACE, st, 0, workspace=(native.paged_decode_workspace, dev),
             apart=lambda: ({"out": out}, {"the queries": q, "k_pages": k_pages, "v_pages": v_pages,
                                           "page_table": page_table, "kv_lens": kv_lens}))
    return out


def packed_attention(q, k, v, cu_seqlens_q, cu_seqlens_k=None, *, causal=True, scale=None, out=None):
    """Attention of packed sequences of different lengths, causal or over all of a sequence's keys.

    ``q`` ``[tokens, nq, D]``, ``k`` and ``v`` ``[tokens_k, nkv, D]`` (bf16 or fp16, D 64 or 128; rows and heads
    may be strided, so slices of one ``q | k | v`` projection do); ``cu_seqlens_q`` / ``cu_seqlens_k`` int32
    ``[batch + 1]`` row offsets, the second None where they are the same. The last query of a sequence stands
    at its last key: with ``causal``, query i of n sees keys ``0 .. len - n + i``; a query without a key gives
    zeros. Returns ``[tokens, nq, D]`` (in ``out`` if given, which has memory of its own); rows outside every
    sequence are not written.
    """
    shape = k.shape
    if len(shape) != 3 or v.shape != shape:
        raise ValueError("k and v must be [tokens, nkv, D]")
    tokens_k, nkv, d = shape
    tokens, nq, row, head, dev = _query(q, nkv, d)
    _no_backward(q, k, v)
    dtype = q.dtype
    if k.dtype is not dtype or v.dtype is not dtype or k.get_device() != dev or v.get_device() != dev:
        raise ValueError("k and v must have the queries' type and device")
    k_row, k_head = _strides3("k", k, nkv, d)
    v_row, v_head = _strides3("v", v, nkv, d)
    batch = cu_seqlens_q.numel() - 1
    if batch < 1:
        raise ValueError("cu_seqlens_q must hold batch + 1 offsets of 1 or more sequences")
    cu_q = _ints("cu_seqlens_q", cu_seqlens_q, batch + 1, dev)
    cu_k = cu_q if cu_seqlens_k is None else _ints("cu_seqlens_k", cu_seqlens_k, batch + 1, dev)
    out = _out(out, (tokens, nq, d), q)
    if tokens == 0:
        return out
    if tokens_k == 0:  # no key anywhere: every row of a sequence is zero, as the kernel would leave it
        k, v, tokens_k, nkv, k_row, k_head, v_row, v_head = q, q, tokens, nq, row, head, row, head
        none = torch.zeros(batch + 1, device=q.device, dtype=torch.int32)
        cu_k = none.data_ptr()
    _call_on(dev, "mt_packed_attention", q.data_ptr(), row, head, k.data_ptr(), k_row, k_head, v.data_ptr(), v_row,
             v_head, cu_q, cu_k, batch, tokens, tokens_k, nq, nkv, d, _TYPES[dtype], 1 if causal else 0,
             d ** -0.5 if scale is None else scale, out.data_ptr(), _WORKSPACE, 0,
             workspace=(native.prompt_workspace, tokens, batch, tokens_k, nq, nkv, d),
             apart=lambda: ({"out": out}, {"the queries": q, "k": k, "v": v, "cu_seqlens_q": cu_seqlens_q,
                                           "cu_seqlens_k": cu_seqlens_k}))
    return out


def paged_attention_prompt(q, k_pages, v_pages, page_table, kv_lens, cu_seqlens, *, scale=None, out=None, status=None):
    """Causal attention of packed prompts, or chunks of them, over a paged key-value cache.

    ``q`` ``[tokens, nq, D]`` are the newest tokens of every sequence, rows ``cu_seqlens[b] ..
    cu_seqlens[b + 1] - 1`` (int32 ``[batch + 1]``) of the last ``kv_lens[b]`` positions; their keys and values
    are in the pages already (``qk_rope_paged``). Query i of n sees keys ``0 .. kv_lens[b] - n + i``. Otherwise
    as ``packed_attention``, with ``paged_attention_decode``'s cache and ``status``.
    """
    _, nkv, _, d = k_pages.shape
    tokens, nq, row, head, dev = _query(q, nkv, d)
    _no_backward(q, k_pages, v_pages)
    kv, batch, most = _paged(k_pages, v_pages, page_table, kv_lens, q.dtype, dev)
    cu = _ints("cu_seqlens", cu_seqlens, batch + 1, dev)
    st = _status(status, dev)
    out = _out(out, (tokens, nq, d), q)
    if tokens:
        _call_on(dev, "mt_paged_attention_prompt", q.data_ptr(), row, head, kv, cu, tokens, nq,
                 d ** -0.5 if scale is None else scale, out.data_ptr(), _WORKSPACE, st, 0,
                 workspace=(native.prompt_workspace, tokens, batch, most, nq, nkv, d),
                 apart=lambda: ({"out": out}, {"the queries": q, "k_pages": k_pages, "v_pages": v_pages,
                                               "page_table": page_table, "kv_lens": kv_lens, "cu_seqlens": cu_seqlens}))
    return out
