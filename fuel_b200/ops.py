"""Kernel-level entry points on torch CUDA tensors.

torch supplies device memory and the current stream only; every operation is one
call into libfuelq.so through the C ABI of include/fuelq.h. Function names follow
the reference's quantized storage API (fuel-backend-contract/src/quantized.rs:29-103).
"""
from __future__ import annotations

import torch

from . import _lib
from .ggml import GgmlDType

_L = _lib.lib
_raw_stream = torch._C._cuda_getCurrentRawStream   # the handle alone: a Stream object costs microseconds
_OUT_TYPES = {torch.float32: GgmlDType.F32, torch.float16: GgmlDType.F16, torch.bfloat16: GgmlDType.BF16}
_TYPE_IDS = {t: int(g) for t, g in _OUT_TYPES.items()}
_current_device = torch._C._cuda_getDevice
_I32, _F32 = torch.int32, torch.float32


def _stream() -> int:
    return _raw_stream(torch.cuda.current_device())


def _need_cuda(t: torch.Tensor, name: str) -> None:
    if not t.is_cuda:
        raise ValueError(f"{name} must be a CUDA tensor (there is no CPU path)")
    if not t.is_contiguous():
        raise ValueError(f"{name} must be contiguous")  # fuel-cpu-backend/src/quantized.rs:96-98


def storage_bytes(dtype: GgmlDType, elem_count: int) -> int:
    bs = dtype.block_size()
    if elem_count % bs:
        raise ValueError(f"{elem_count} elements is not a multiple of the {dtype.name} block size {bs}")
    return elem_count // bs * dtype.type_size()


def quantize_act(weight_dtype: GgmlDType, x: torch.Tensor) -> torch.Tensor:
    """Rows of x [.., k] -> the reference's Q8_K / Q8_1 / Q8_0 activation blocks (uint8 stream)."""
    _need_cuda(x, "x")
    k = x.shape[-1]
    m = x.numel() // k
    act = (GgmlDType.Q8K if weight_dtype in (GgmlDType.Q2K, GgmlDType.Q3K, GgmlDType.Q4K, GgmlDType.Q5K, GgmlDType.Q6K)
           else GgmlDType.Q8_1 if weight_dtype in (GgmlDType.Q4_1, GgmlDType.Q5_1) else GgmlDType.Q8_0)
    if k % act.block_size():
        _lib.check(_lib.INVALID_PROBLEM, "quantize_act")
    out = torch.empty(storage_bytes(act, m * k), dtype=torch.uint8, device=x.device)
    with torch.cuda.device(x.device):
        _lib.check(_L.fuelq_quantize_act(int(weight_dtype), m, k, x.data_ptr(), out.data_ptr(), _stream()),
                   "fuelq_quantize_act")
    return out


def quantize_act_packed(weight_dtype: GgmlDType, x: torch.Tensor) -> torch.Tensor:
    _need_cuda(x, "x")
    k = x.shape[-1]
    m = x.numel() // k
    nbytes = _L.fuelq_act_packed_bytes(int(weight_dtype), m, k)
    out = torch.empty(max(nbytes, 16), dtype=torch.uint8, device=x.device)
    with torch.cuda.device(x.device):
        _lib.check(_L.fuelq_quantize_act_packed(int(weight_dtype), m, k, x.data_ptr(), out.data_ptr(), nbytes,
                                                _stream()), "fuelq_quantize_act_packed")
    return out


def qmatmul(dtype: GgmlDType, w_blocks: torch.Tensor, n: int, x: torch.Tensor,
            out: torch.Tensor | None = None, workspace: torch.Tensor | None = None) -> torch.Tensor:
    """y[.., n] = x[.., k] . W[n, k]^T, W as GGUF blocks (uint8 stream of n rows)."""
    _need_cuda(x, "x")
    _need_cuda(w_blocks, "w_blocks")
    if x.dtype != torch.float32:
        raise ValueError("activations must be float32")
    k = x.shape[-1]
    m = x.numel() // k if k else 0
    if k % dtype.block_size() == 0 and w_blocks.numel() != storage_bytes(dtype, n * k):
        raise ValueError(f"weight bytes={w_blocks.numel()} doesn't match n={n} x k={k} {dtype.name}")
    if out is None:
        out = torch.empty(*x.shape[:-1], n, dtype=torch.float32, device=x.device)
    ws_bytes = _L.fuelq_qmatmul_workspace_bytes(int(dtype), m, n, k)
    if workspace is None:
        workspace = torch.empty(max(ws_bytes, 16), dtype=torch.uint8, device=x.device)
    with torch.cuda.device(x.device):
        _lib.check(_L.fuelq_qmatmul(int(dtype), m, n, k, w_blocks.data_ptr(), x.data_ptr(), out.data_ptr(),
                                    workspace.data_ptr(), workspace.numel(), _stream()), "fuelq_qmatmul")
    return out


def qmatmul_host(dtype: GgmlDType, w_blocks: torch.Tensor, n: int, x_host: torch.Tensor,
                 out_host: torch.Tensor | None = None, workspace: torch.Tensor | None = None) -> torch.Tensor:
    """qmatmul for HOST activations and a HOST result (CPU tensors; pinned ones keep the call asynchronous and, when
    small, are read and written in place by the kernels). Enqueued on the current stream of the weights' device;
    synchronize that stream before reading the result."""
    _need_cuda(w_blocks, "w_blocks")
    if x_host.is_cuda or x_host.dtype != torch.float32 or not x_host.is_contiguous():
        raise ValueError("x_host must be a contiguous float32 CPU tensor")
    k = x_host.shape[-1]
    m = x_host.numel() // k if k else 0
    if out_host is None:
        out_host = torch.empty(*x_host.shape[:-1], n, dtype=torch.float32, pin_memory=x_host.is_pinned())
    ws_bytes = _L.fuelq_qmatmul_host_workspace_bytes(int(dtype), m, n, k)
    if workspace is None:
        workspace = torch.empty(max(ws_bytes, 256), dtype=torch.uint8, device=w_blocks.device)
    with torch.cuda.device(w_blocks.device):
        _lib.check(_L.fuelq_qmatmul_host(int(dtype), m, n, k, w_blocks.data_ptr(), x_host.data_ptr(), out_host.data_ptr(),
                                         workspace.data_ptr(), workspace.numel(), _stream()), "fuelq_qmatmul_host")
    return out_host


def qmatmul_packed(dtype: GgmlDType, w_blocks: torch.Tensor, n: int, k: int, m: int, packed_act: torch.Tensor,
                   out: torch.Tensor) -> torch.Tensor:
    with torch.cuda.device(out.device):
        _lib.check(_L.fuelq_qmatmul_packed(int(dtype), m, n, k, w_blocks.data_ptr(), packed_act.data_ptr(),
                                           out.data_ptr(), _stream()), "fuelq_qmatmul_packed")
    return out


def quantize_weights(dtype: GgmlDType, w: torch.Tensor) -> torch.Tensor:
    """f32 weights (any shape, row length a multiple of the block) -> GGUF block bytes, on the device."""
    _need_cuda(w, "w")
    if w.dtype != torch.float32:
        raise ValueError("only f32 can be quantized")  # fuel-cuda-backend/src/quantized.rs:414-418
    out = torch.empty(storage_bytes(dtype, w.numel()), dtype=torch.uint8, device=w.device)
    with torch.cuda.device(w.device):
        _lib.check(_L.fuelq_quantize_weights(int(dtype), w.numel(), w.data_ptr(), out.data_ptr(), _stream()),
                   "fuelq_quantize_weights")
    return out


def dequantize(dtype: GgmlDType, blocks: torch.Tensor, elem_count: int,
               out_dtype: torch.dtype = torch.float32) -> torch.Tensor:
    _need_cuda(blocks, "blocks")
    out = torch.empty(elem_count, dtype=out_dtype, device=blocks.device)
    with torch.cuda.device(blocks.device):
        _lib.check(_L.fuelq_dequantize(int(dtype), elem_count, blocks.data_ptr(), out.data_ptr(),
                                       int(_OUT_TYPES[out_dtype]), _stream()), "fuelq_dequantize")
    return out


# ---- attention for batches of sequences: a paged key-value cache, whole packed prompts

# (these run at every call of a decode step, where a look at a tensor's shape or type is a tenth of a microsecond: each is
# looked at once and handed on)
def _heads(t: torch.Tensor, name: str, dtype: torch.dtype, dev: int):
    """Checks a [rows, heads, head_dim] tensor on device `dev` whose rows may lie apart; its row stride in elements, its shape."""
    shape = t.shape
    if dev < 0 or t.get_device() != dev:
        raise ValueError(f"{name} must be a CUDA tensor on the device of the other operands (there is no CPU path)")
    if t.dtype is not dtype or len(shape) != 3:
        raise ValueError(f"{name} must be a {dtype} tensor of [rows, heads, head_dim]")
    rows, heads, hd = shape
    row, head, one = t.stride()
    if one != 1 or (head != hd and heads > 1):
        raise ValueError(f"the heads of a row of {name} must be contiguous")
    return row if rows > 1 else heads * hd, shape


def _indices(t: torch.Tensor, name: str, dims: int, dev: int):
    """Checks an int32 tensor of indices; its shape."""
    shape = t.shape
    if t.dtype is not _I32 or t.get_device() != dev or len(shape) != dims or not t.is_contiguous():
        raise ValueError(f"{name} must be a contiguous int32 tensor of {dims} dimension(s) on the device of the other operands")
    return shape


def _paged(kcache: torch.Tensor, vcache: torch.Tensor, dev: int):
    """Checks a paged cache; (pages, kv heads, page size, head_dim), the type's number."""
    shape, dtype = kcache.shape, kcache.dtype
    if len(shape) != 4 or shape != vcache.shape or vcache.dtype is not dtype or dtype not in _TYPE_IDS:
        raise ValueError("the caches must be two f32, f16 or bf16 tensors of [pages, kv_heads, page_size, head_dim]")
    if kcache.get_device() != dev or vcache.get_device() != dev or not kcache.is_contiguous() or not vcache.is_contiguous():
        raise ValueError("the caches must be contiguous, on the device of the other operands")
    return shape, _TYPE_IDS[dtype]


def _result(out: torch.Tensor | None, shape, dtype: torch.dtype, dev: int, name: str) -> torch.Tensor:
    if out is None:
        return torch.empty(shape, dtype=dtype, device=torch.device("cuda", dev))
    if out.shape != shape or out.dtype is not dtype or out.get_device() != dev or not out.is_contiguous():
        raise ValueError(f"{name} must be a contiguous {dtype} tensor of {tuple(shape)} on the device of the operands")
    return out


def _scratch(workspace: torch.Tensor | None, nbytes: int, like: torch.Tensor) -> torch.Tensor:
    if workspace is None:
        return torch.empty(max(nbytes, 16), dtype=torch.uint8, device=like.device)
    if workspace.get_device() != like.get_device() or not workspace.is_contiguous():
        raise ValueError("the workspace must be contiguous, on the device of the operands")
    return workspace


def paged_append(k: torch.Tensor, v: torch.Tensor, kcache: torch.Tensor, vcache: torch.Tensor, page_table: torch.Tensor,
                 positions: torch.Tensor, cos: torch.Tensor, sin: torch.Tensor, *, seq_ids: torch.Tensor | None = None,
                 q: torch.Tensor | None = None, q_out: torch.Tensor | None = None,
                 k_out: torch.Tensor | None = None) -> torch.Tensor | None:
    """Keys k [rows, kv_heads, head_dim], rotated by positions[row], and values v go to that position of sequence
    seq_ids[row] (None: sequence `row`) in the paged caches [pages, kv_heads, page_size, head_dim]; page_table is
    [sequences, pages of the longest]. Rows with a negative position or sequence number are padding. Returns the rotated
    queries (q_out, or a new tensor) if q is given; k_out, if given, receives the rotated keys. The rows of q, k and v may be
    column ranges of one stacked projection."""
    dev, dtype = k.get_device(), k.dtype
    if dev >= 0 and dev != _current_device():
        with torch.cuda.device(dev):
            return paged_append(k, v, kcache, vcache, page_table, positions, cos, sin, seq_ids=seq_ids, q=q, q_out=q_out, k_out=k_out)
    (ks, shape), (vs, v_shape) = _heads(k, "k", dtype, dev), _heads(v, "v", dtype, dev)
    if dtype not in _TYPE_IDS or v_shape != shape:
        raise ValueError("k and v must be f32, f16 or bf16 and of one shape")
    rows, kv, hd = shape
    (pages, ckv, page, chd), cache_type = _paged(kcache, vcache, dev)
    if ckv != kv or chd != hd:
        raise ValueError(f"the caches hold {ckv} heads of {chd}, k has {kv} of {hd}")
    seqs, width = _indices(page_table, "page_table", 2, dev)
    if (_indices(positions, "positions", 1, dev)[0] != rows
            or (seq_ids is not None and _indices(seq_ids, "seq_ids", 1, dev)[0] != rows)):
        raise ValueError("positions and seq_ids need one entry per row")
    table = cos.shape
    if len(table) != 2 or table[1] != hd or sin.shape != table:
        raise ValueError("cos and sin must be f32 tables of [positions, head_dim], of one shape")
    for t in cos, sin:
        if t.dtype is not _F32 or t.get_device() != dev or not t.is_contiguous():
            raise ValueError("cos and sin must be contiguous f32 tables on the device of the other operands")
    heads = qs = 0
    if q is not None:
        qs, q_shape = _heads(q, "q", dtype, dev)
        q_rows, heads, q_hd = q_shape
        if q_rows != rows or q_hd != hd:
            raise ValueError("q must have the rows and the head_dim of k")
        q_out = _result(q_out, q_shape, dtype, dev, "q_out")
    if k_out is not None:
        _result(k_out, shape, dtype, dev, "k_out")
    status = _L.fuelq_paged_append(_TYPE_IDS[dtype], cache_type, k.data_ptr(), ks, v.data_ptr(), vs,
                                   None if q is None else q.data_ptr(), qs, None if q is None else q_out.data_ptr(),
                                   None if k_out is None else k_out.data_ptr(), kcache.data_ptr(), vcache.data_ptr(),
                                   page_table.data_ptr(), None if seq_ids is None else seq_ids.data_ptr(), positions.data_ptr(),
                                   cos.data_ptr(), sin.data_ptr(), rows, seqs, heads, kv, hd, page, pages, width,
                                   table[0], _raw_stream(dev))
    if status:
        _lib.check(status, "fuelq_paged_append")
    return None if q is None else q_out


def paged_attn_workspace(n_seqs: int, n_heads: int, n_kv_heads: int, head_dim: int, device) -> torch.Tensor:
    """Scratch for paged_attn_decode; one serves every layer of a model, and every call on one stream."""
    nbytes = _L.fuelq_paged_attn_workspace_bytes(n_seqs, n_heads, n_kv_heads, head_dim)
    return torch.empty(max(nbytes, 16), dtype=torch.uint8, device=device)


def paged_attn_decode(q: torch.Tensor, kcache: torch.Tensor, vcache: torch.Tensor, page_table: torch.Tensor,
                      seq_lens: torch.Tensor, scale: float | None = None, out: torch.Tensor | None = None,
                      workspace: torch.Tensor | None = None) -> torch.Tensor:
    """Attention of one new token per sequence, q [sequences, heads, head_dim] already rotated, over the first seq_lens[s]
    positions of its pages. A length of zero, a free slot of the batch, gives zeros. Default scale: 1 / sqrt(head_dim)."""
    dev, dtype = q.get_device(), q.dtype
    if dev >= 0 and dev != _current_device():
        with torch.cuda.device(dev):
            return paged_attn_decode(q, kcache, vcache, page_table, seq_lens, scale, out, workspace)
    qs, shape = _heads(q, "q", dtype, dev)
    n, heads, hd = shape
    (pages, kv, page, chd), cache_type = _paged(kcache, vcache, dev)
    if dtype not in _TYPE_IDS or chd != hd:
        raise ValueError("q must be f32, f16 or bf16 with the head_dim of the caches")
    seqs, width = _indices(page_table, "page_table", 2, dev)
    if seqs != n or _indices(seq_lens, "seq_lens", 1, dev)[0] != n:
        raise ValueError("page_table and seq_lens need one row per sequence")
    out = _result(out, shape, dtype, dev, "out")
    workspace = _scratch(workspace, _L.fuelq_paged_attn_workspace_bytes(n, heads, kv, hd) if workspace is None else 0, q)
    status = _L.fuelq_paged_attn_decode(_TYPE_IDS[dtype], cache_type, q.data_ptr(), qs, kcache.data_ptr(),
                                        vcache.data_ptr(), out.data_ptr(), page_table.data_ptr(), seq_lens.data_ptr(), n, heads,
                                        kv, hd, page, pages, width, hd ** -0.5 if scale is None else scale,
                                        workspace.data_ptr(), workspace.nbytes, _raw_stream(dev))
    if status:
        _lib.check(status, "fuelq_paged_attn_decode")
    return out


def prompt_attn_workspace(q: torch.Tensor, k: torch.Tensor) -> torch.Tensor:
    """Scratch for prompt_attn on tensors of these shapes; calls on one stream may share it."""
    if q.dtype not in _TYPE_IDS:
        raise ValueError("q must be f32, f16 or bf16")
    nbytes = _L.fuelq_prompt_attn_workspace_bytes(_TYPE_IDS[q.dtype], q.shape[0], q.shape[1], k.shape[1], q.shape[2])
    return torch.empty(max(nbytes, 16), dtype=torch.uint8, device=q.device)


def prompt_attn(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, cu_seqlens: torch.Tensor, scale: float | None = None,
                out: torch.Tensor | None = None, workspace: torch.Tensor | None = None) -> torch.Tensor:
    """Causal attention inside packed prompts: rows cu_seqlens[s] .. cu_seqlens[s + 1] of q [rows, heads, head_dim] (rotated)
    and of k, v [rows, kv_heads, head_dim] are sequence s. Rows behind the last sequence are padding: not read, and left as
    they were in `out`. Default scale: 1 / sqrt(head_dim)."""
    dev, dtype = q.get_device(), q.dtype
    if dev >= 0 and dev != _current_device():
        with torch.cuda.device(dev):
            return prompt_attn(q, k, v, cu_seqlens, scale, out, workspace)
    (qs, shape), (ks, k_shape), (vs, v_shape) = _heads(q, "q", dtype, dev), _heads(k, "k", dtype, dev), _heads(v, "v", dtype, dev)
    rows, heads, hd = shape
    k_rows, kv, k_hd = k_shape
    if dtype not in _TYPE_IDS or k_shape != v_shape or k_rows != rows or k_hd != hd:
        raise ValueError("q, k and v must be f32, f16 or bf16 with the same rows and head_dim")
    seqs = _indices(cu_seqlens, "cu_seqlens", 1, dev)[0] - 1
    if seqs < 0:
        raise ValueError("cu_seqlens needs n_seqs + 1 entries")
    out = _result(out, shape, dtype, dev, "out")
    workspace = _scratch(workspace, 0 if workspace is not None else
                         _L.fuelq_prompt_attn_workspace_bytes(_TYPE_IDS[dtype], rows, heads, kv, hd), q)
    status = _L.fuelq_prompt_attn(_TYPE_IDS[dtype], q.data_ptr(), qs, k.data_ptr(), ks, v.data_ptr(), vs, out.data_ptr(),
                                  cu_seqlens.data_ptr(), seqs, rows, heads, kv, hd, hd ** -0.5 if scale is None else scale,
                                  workspace.data_ptr(), workspace.nbytes, _raw_stream(dev))
    if status:
        _lib.check(status, "fuelq_prompt_attn")
    return out


def device_error(clear: bool = True) -> int:
    import ctypes
    code = ctypes.c_int32(0)
    _lib.check(_L.fuelq_device_error(ctypes.byref(code), 1 if clear else 0), "fuelq_device_error")
    return code.value
