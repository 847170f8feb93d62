"""Reference-named operator wrappers over device tensors.

Each function mirrors one operator of the reference's compute seam and calls the
matching ``glacier_cuda_*`` entry point on torch CUDA tensors (torch is used only
for device memory and streams).  Shapes are validated by the library; errors
raise ``GlacierCudaError``.
"""
from __future__ import annotations

import torch

from ._lib import EINVAL, GlacierCudaError, call, lib


def _ptr(t):
    return None if t is None else t.data_ptr()


def _stream(stream=None):
    s = stream if stream is not None else torch.cuda.current_stream()
    return s.cuda_stream


def linear_int4_on_the_fly(x: torch.Tensor, packed: torch.Tensor, scales: torch.Tensor,
                           out_f: int, in_f: int, group: int, bias: torch.Tensor | None = None,
                           out: torch.Tensor | None = None, stream=None) -> torch.Tensor:
    """int4_matmul.zig:215 linearInt4OnTheFly: out[b] = x[b] * dequant(W)^T + bias.

    ``scales`` is float32 or float16 (the reference's f32 scales or its fp16
    mirror, int4_weights.zig:86-90)."""
    x = x.reshape(-1, in_f)
    assert x.dtype == torch.float32 and x.is_contiguous()
    if out is None:
        out = torch.empty((x.shape[0], out_f), dtype=torch.float32, device=x.device)
    call("glacier_cuda_int4_linear", x.data_ptr(), x.shape[0], packed.data_ptr(), scales.data_ptr(),
         int(scales.dtype == torch.float16), _ptr(bias), out.data_ptr(), out_f, in_f, group,
         _stream(stream))
    return out


def linear_int4_tensor_core(x: torch.Tensor, packed: torch.Tensor, scales_f16: torch.Tensor, out_f: int,
                            in_f: int, group: int, bias: torch.Tensor | None = None, out=None, stream=None):
    """Batched linearInt4OnTheFly on the tcgen05 dequant GEMM (int4_neon.c:1439 M4 GEMM role)."""
    x = x.reshape(-1, in_f)
    b = x.shape[0]
    out = torch.empty((b, out_f), dtype=torch.float32, device=x.device) if out is None else out
    ws_n = lib().glacier_cuda_int4_matmul_workspace(b, in_f, out_f)
    ws = torch.empty(ws_n, dtype=torch.uint8, device=x.device)
    call("glacier_cuda_int4_matmul_f16scale", x.data_ptr(), b, packed.data_ptr(), scales_f16.data_ptr(), _ptr(bias),
         out.data_ptr(), out_f, in_f, group, ws.data_ptr(), ws_n, _stream(stream))
    return out


def rms_norm_f32(x: torch.Tensor, weight: torch.Tensor, eps: float, out=None, stream=None):
    """kernels.zig:141 rmsNormF32 over rows of x [batch, dim]."""
    b, d = x.shape
    out = torch.empty_like(x) if out is None else out
    call("glacier_cuda_rmsnorm_f32", x.data_ptr(), weight.data_ptr(), eps, out.data_ptr(), b, d, _stream(stream))
    return out


def add_rms_norm_f32(a, b, weight, eps: float, residual=None, out=None, stream=None):
    """kernels.zig:322 addRmsNormF32: residual = a + b, out = rmsnorm(residual)."""
    residual = torch.empty_like(a) if residual is None else residual
    out = torch.empty_like(a) if out is None else out
    call("glacier_cuda_add_rmsnorm_f32", a.data_ptr(), b.data_ptr(), residual.data_ptr(), weight.data_ptr(), eps,
         out.data_ptr(), a.shape[0], a.shape[1], _stream(stream))
    return residual, out


def silu_mul_f32(gate, up, out=None, stream=None):
    """kernels.zig:465 siluMulF32 over rows: silu(gate) * up."""
    b, n = gate.shape
    out = torch.empty_like(gate) if out is None else out
    call("glacier_cuda_silu_mul_f32", gate.data_ptr(), up.data_ptr(), gate.stride(0), out.data_ptr(), out.stride(0),
         b, n, _stream(stream))
    return out


def load_embedding_rows(table_f16, tokens, stream=None):
    """generate.zig:3653 loadEmbeddingRow for a batch of tokens (fp16 table)."""
    vocab, dim = table_f16.shape
    out = torch.empty((tokens.numel(), dim), dtype=torch.float32, device=tokens.device)
    call("glacier_cuda_embedding_f16", table_f16.data_ptr(), vocab, dim, tokens.data_ptr(), tokens.numel(),
         out.data_ptr(), _stream(stream))
    return out


def qkv_rope_append(qkv, bias, cos, sin, pos, num_heads, num_kv_heads, head_dim, kv_pages, page_floats,
                    block_tables, layer, stream=None):
    """RopeTable.apply (generate.zig:816) on q and k + appendRowTxn (paged_kv_cache.zig:1074)."""
    b = qkv.shape[0]
    q_out = torch.empty((b, num_heads * head_dim), dtype=torch.float32, device=qkv.device)
    call("glacier_cuda_qkv_rope_append_f32", qkv.data_ptr(), qkv.stride(0), _ptr(bias), cos.data_ptr(),
         sin.data_ptr(), cos.shape[0], pos.data_ptr(), b, num_heads, num_kv_heads, head_dim, q_out.data_ptr(),
         q_out.stride(0), kv_pages.data_ptr(), page_floats, block_tables.data_ptr(), block_tables.shape[1], layer,
         _stream(stream))
    return q_out


def paged_attention_f32(q, kv_pages, page_floats, block_tables, ctx_lens, max_ctx, layer, num_heads, num_kv_heads,
                        head_dim, stream=None):
    """paged_attention.zig:108 attentionMultiHead, one query row per lane."""
    lanes = q.shape[0]
    ws_n = lib().glacier_cuda_paged_attention_workspace(lanes, num_heads, num_kv_heads, head_dim, max_ctx)
    ws = torch.empty(ws_n, dtype=torch.float32, device=q.device)
    out = torch.empty((lanes, num_heads * head_dim), dtype=torch.float32, device=q.device)
    call("glacier_cuda_paged_attention_f32", q.data_ptr(), kv_pages.data_ptr(), page_floats, block_tables.data_ptr(),
         block_tables.shape[1], ctx_lens.data_ptr(), max_ctx, lanes, layer, num_heads, num_kv_heads, head_dim,
         out.data_ptr(), ws.data_ptr(), ws_n, _stream(stream))
    return out


def argmax_eligible(logits, words=None, stream=None):
    """sampling.zig:55 argmaxEligible per row -> (tokens int32, status int32)."""
    b, n = logits.shape
    ws_n = lib().glacier_cuda_argmax_workspace(b, n)
    ws = torch.empty(ws_n, dtype=torch.uint8, device=logits.device)
    tokens = torch.empty(b, dtype=torch.int32, device=logits.device)
    status = torch.empty(b, dtype=torch.int32, device=logits.device)
    wc = 0 if words is None else words.shape[-1]
    call("glacier_cuda_argmax_eligible_f32", logits.data_ptr(), b, n, _ptr(words), wc, tokens.data_ptr(),
         status.data_ptr(), None, ws.data_ptr(), ws_n, _stream(stream))
    return tokens, status


# ---- the KV cache held in 4 bits ----
# These run on the device their tensors are on, whichever is current; what they allocate belongs
# to the stream they run on, and what they are given is kept until a stream= has done with it.  Tensors of
# another type, shape, layout or device are refused.
# A decode step makes them every layer, so the checks are plain comparisons (about 2 us a call) and
# only a refusal looks for the tensor to name.

_F32, _I32, _I64, _U8 = torch.float32, torch.int32, torch.int64, torch.uint8
# The bare forms of torch.cuda.current_device and current_stream (absent from a torch without CUDA).
_device, _raw_stream = (getattr(torch._C, n, None) for n in ("_cuda_getDevice", "_cuda_getCurrentRawStream"))


def _refuse(dev, **tensors):
    """Raises for the first (tensor, dtype, shape) that is not contiguous on `dev` with that type and shape."""
    for name, (t, dtype, shape) in tensors.items():
        if t is None:
            continue
        if t.dtype is not dtype or t.get_device() != dev or not t.is_contiguous() or tuple(t.shape) != tuple(shape):
            raise GlacierCudaError(EINVAL, f"{name}: {str(t.dtype)[6:]} {tuple(t.shape)} on {t.device}, expected a "
                                           f"contiguous {str(dtype)[6:]} {tuple(shape)} on the GPU of the first tensor")
    raise GlacierCudaError(EINVAL, "the 4-bit cache is on a GPU")


def _fits(t, dtype, shape, dev):
    return t.dtype is dtype and t.shape == shape and t.get_device() == dev and t.is_contiguous()


class _On:
    """Makes another device, or a given stream, current around a call; the call's tensors may be dropped behind it."""

    def __init__(self, dev, stream, *tensors):
        if dev < 0:
            _refuse(dev)
        if stream is not None and stream.device.index != dev:
            raise GlacierCudaError(EINVAL, f"a stream of {stream.device} for tensors on GPU {dev}")
        if stream is not None:
            for t in tensors:
                if t is not None and t.get_device() == dev:
                    t.record_stream(stream)
        self.ctx = torch.cuda.stream(stream if stream is not None else torch.cuda.current_stream(dev))

    def __enter__(self):
        self.ctx.__enter__()

    def __exit__(self, *exc):
        self.ctx.__exit__(*exc)


def kv_q4_page_bytes(num_layers: int, num_kv_heads: int, head_dim: int) -> int:
    """Bytes of one 16-position page of a 4-bit pool (all layers)."""
    return lib().glacier_cuda_kv_q4_page_bytes(num_layers, num_kv_heads, head_dim)


def qkv_rope_append_q4(qkv, bias, cos, sin, pos, slots, num_heads, num_kv_heads, head_dim, pages, num_layers, layer,
                       q_out=None, stream=None):
    """qkv_rope_append into a 4-bit pool: ``pages`` uint8 [num_pages, kv_q4_page_bytes], row b's K and V
    quantised into position ``slots[b]`` (int64: page * 16 + row; -1: a padding row).  Returns the rotated q
    [batch, num_heads * head_dim].  ``qkv`` may be a view with a row stride."""
    dev = qkv.get_device()
    if stream is not None or dev < 0 or dev != _device():
        with _On(dev, stream, qkv, bias, cos, sin, pos, slots, pages, q_out):
            return qkv_rope_append_q4(qkv, bias, cos, sin, pos, slots, num_heads, num_kv_heads, head_dim, pages,
                                      num_layers, layer, q_out)
    qd, kvd = num_heads * head_dim, num_kv_heads * head_dim
    width = qd + 2 * kvd
    if qkv.dtype is not _F32 or qkv.dim() != 2 or qkv.shape[1] != width or qkv.stride(1) != 1:
        raise GlacierCudaError(EINVAL, f"qkv: {qkv.dtype} {tuple(qkv.shape)}, expected float32 rows of {width}")
    b, positions, num_pages = qkv.shape[0], cos.shape[0], pages.shape[0]
    rows, table, page = (b,), (positions, head_dim // 2), (num_pages, 18 * num_layers * kvd)
    if not (_fits(cos, _F32, table, dev) and _fits(sin, _F32, table, dev) and _fits(pos, _I32, rows, dev)
            and _fits(slots, _I64, rows, dev) and _fits(pages, _U8, page, dev)
            and (bias is None or _fits(bias, _F32, (width,), dev))
            and (q_out is None or _fits(q_out, _F32, (b, qd), dev))):
        _refuse(dev, cos=(cos, _F32, table), sin=(sin, _F32, table), pos=(pos, _I32, rows), slots=(slots, _I64, rows),
                pages=(pages, _U8, page), bias=(bias, _F32, (width,)), q_out=(q_out, _F32, (b, qd)))
    if q_out is None:
        q_out = qkv.new_empty((b, qd))
    call("glacier_cuda_qkv_rope_append_q4", qkv.data_ptr(), qkv.stride(0) if b > 1 else width, _ptr(bias),
         cos.data_ptr(), sin.data_ptr(), positions, pos.data_ptr(), slots.data_ptr(), b, num_heads, num_kv_heads,
         head_dim, q_out.data_ptr(), qd, pages.data_ptr(), num_pages, num_layers, layer, _raw_stream(dev))
    return q_out


def kv_q4_read(pages, slots, num_layers, layer, num_kv_heads, head_dim, stream=None):
    """The K and V values held at ``slots``: two float32 [rows, num_kv_heads * head_dim] (zeros for slot -1)."""
    dev = pages.get_device()
    if stream is not None or dev < 0 or dev != _device():
        with _On(dev, stream, pages, slots):
            return kv_q4_read(pages, slots, num_layers, layer, num_kv_heads, head_dim)
    rows, num_pages, kvd = slots.numel(), pages.shape[0], num_kv_heads * head_dim
    page = (num_pages, 18 * num_layers * kvd)
    if not (_fits(slots, _I64, (rows,), dev) and _fits(pages, _U8, page, dev)):
        _refuse(dev, slots=(slots, _I64, (rows,)), pages=(pages, _U8, page))
    k = pages.new_empty((rows, kvd), dtype=_F32)
    v = torch.empty_like(k)
    call("glacier_cuda_kv_q4_read_f32", pages.data_ptr(), num_pages, num_layers, layer, num_kv_heads, head_dim,
         slots.data_ptr(), rows, k.data_ptr(), v.data_ptr(), _raw_stream(dev))
    return k, v


def paged_attention_q4_workspace(num_heads, num_kv_heads, head_dim, device=None):
    """Workspace of paged_attention_q4, for calls that do not run at the same time."""
    n = lib().glacier_cuda_paged_attention_q4_workspace(num_heads, num_kv_heads, head_dim)
    return torch.empty(n, dtype=_F32, device="cuda" if device is None else device)


def paged_attention_q4(q, pages, block_tables, ctx_lens, num_layers, layer, num_heads, num_kv_heads, head_dim,
                       out=None, workspace=None, stream=None):
    """paged_attention_f32 over a 4-bit pool, one query row per lane."""
    dev = q.get_device()
    if stream is not None or dev < 0 or dev != _device():
        with _On(dev, stream, q, pages, block_tables, ctx_lens, out, workspace):
            return paged_attention_q4(q, pages, block_tables, ctx_lens, num_layers, layer, num_heads, num_kv_heads,
                                      head_dim, out, workspace)
    lanes, num_pages, max_pages = q.shape[0], pages.shape[0], block_tables.shape[-1]
    rows, page = (lanes, num_heads * head_dim), (num_pages, 18 * num_layers * num_kv_heads * head_dim)
    floats = 0 if workspace is None else workspace.numel()
    if not (_fits(q, _F32, rows, dev) and _fits(pages, _U8, page, dev)
            and _fits(block_tables, _I32, (lanes, max_pages), dev) and _fits(ctx_lens, _I32, (lanes,), dev)
            and (out is None or _fits(out, _F32, rows, dev))
            and (workspace is None or _fits(workspace, _F32, (floats,), dev))):
        _refuse(dev, q=(q, _F32, rows), pages=(pages, _U8, page), block_tables=(block_tables, _I32, (lanes, max_pages)),
                ctx_lens=(ctx_lens, _I32, (lanes,)), out=(out, _F32, rows), workspace=(workspace, _F32, (floats,)))
    if workspace is None:
        workspace = paged_attention_q4_workspace(num_heads, num_kv_heads, head_dim, q.device)
        floats = workspace.numel()
    if out is None:
        out = torch.empty_like(q)
    call("glacier_cuda_paged_attention_q4", q.data_ptr(), pages.data_ptr(), num_pages, num_layers,
         block_tables.data_ptr(), max_pages, ctx_lens.data_ptr(), lanes, layer, num_heads, num_kv_heads, head_dim,
         out.data_ptr(), workspace.data_ptr(), floats, _raw_stream(dev))
    return out


def kv_resize(lens, targets, block_tables, free_pages, free_count, status, positions=None, row_lanes=None, slots=None,
              row_offsets=None, row_stride=0, stream=None):
    """Brings every lane from ``lens`` to ``targets`` positions in place: pages move between the
    ``block_tables`` and the ``free_pages`` stack of ``free_count`` entries, and the new positions are written
    as rows (positions, row_lanes int32, slots int64; packed, or row_stride rows per lane).  All int32 but slots;
    see glacier_cuda_kv_resize for the order in which lanes are served and the statuses."""
    dev = lens.get_device()
    if stream is not None or dev < 0 or dev != _device():
        with _On(dev, stream, lens, targets, block_tables, free_pages, free_count, status, positions, row_lanes, slots,
                 row_offsets):
            return kv_resize(lens, targets, block_tables, free_pages, free_count, status, positions, row_lanes, slots,
                             row_offsets, row_stride)
    n, max_pages, capacity = lens.shape[0], block_tables.shape[-1], free_pages.numel()
    lanes, rows = (n,), 0 if slots is None else slots.numel()
    if not (_fits(lens, _I32, lanes, dev) and _fits(targets, _I32, lanes, dev)
            and _fits(block_tables, _I32, (n, max_pages), dev) and _fits(free_pages, _I32, (capacity,), dev)
            and _fits(free_count, _I32, (1,), dev) and _fits(status, _I32, lanes, dev)
            and (row_offsets is None or _fits(row_offsets, _I32, (n + 1,), dev))):
        _refuse(dev, lens=(lens, _I32, lanes), targets=(targets, _I32, lanes),
                block_tables=(block_tables, _I32, (n, max_pages)), free_pages=(free_pages, _I32, (capacity,)),
                free_count=(free_count, _I32, (1,)), status=(status, _I32, lanes),
                row_offsets=(row_offsets, _I32, (n + 1,)))
    if slots is not None and positions is not None and row_lanes is not None:
        if not (_fits(slots, _I64, (rows,), dev) and _fits(positions, _I32, (rows,), dev)
                and _fits(row_lanes, _I32, (rows,), dev)):
            _refuse(dev, slots=(slots, _I64, (rows,)), positions=(positions, _I32, (rows,)),
                    row_lanes=(row_lanes, _I32, (rows,)))
    elif not (slots is positions is row_lanes is None):
        raise GlacierCudaError(EINVAL, "kv_resize: positions, row_lanes and slots go together")
    call("glacier_cuda_kv_resize", lens.data_ptr(), targets.data_ptr(), n, block_tables.data_ptr(), max_pages,
         free_pages.data_ptr(), capacity, free_count.data_ptr(), status.data_ptr(), row_stride, rows, _ptr(positions),
         _ptr(row_lanes), _ptr(slots), _ptr(row_offsets), _raw_stream(dev))
