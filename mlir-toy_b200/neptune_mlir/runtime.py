"""Run-time support for modules emitted by ``neptune_mlir.translators.b200``.

An emitted module contains one function per ``func.func`` of the HTile program; its body is a single
call into this module with the tensors the caller passed (in memref-argument order, outputs written
in place, as with the reference's emitted kernels -- tests/test_translators.py:184-194) and the
static facts read from the program (shapes, dtype, constants).  Each function here checks the
tensors against those facts, then passes raw device pointers and torch's current CUDA stream to the
nb200 C ABI.  Launches are asynchronous; the caller synchronises.  Nothing here computes: without
the kernel library every call raises.
"""

from __future__ import annotations

import threading

import torch

from . import native

_TORCH_DTYPES = {"f16": torch.float16, "bf16": torch.bfloat16, "f32": torch.float32}
_status_buffers: dict[int, torch.Tensor] = {}
_captured_words: dict[int, list[torch.Tensor]] = {}   # words of calls that were captured before the device had its own
_status_lock = threading.Lock()


def _check(name: str, t, shape, dtype: str | torch.dtype) -> None:
    if not isinstance(t, torch.Tensor):
        raise TypeError(f"{name}: expected a torch.Tensor, got {type(t).__name__}")
    if not t.is_cuda:
        raise ValueError(f"{name}: expected a CUDA tensor (the B200 target has no CPU path)")
    want = _TORCH_DTYPES[dtype] if isinstance(dtype, str) else dtype
    if t.dtype != want:
        raise TypeError(f"{name}: dtype {t.dtype}, the program says {want}")
    if tuple(t.shape) != tuple(shape):
        raise ValueError(f"{name}: shape {tuple(t.shape)}, the program says {tuple(shape)}")
    if not t.is_contiguous():
        raise ValueError(f"{name}: tensor must be contiguous row-major")


def _same_device(*tensors) -> torch.device:
    dev = tensors[0].device
    for t in tensors[1:]:
        if t.device != dev:
            raise ValueError("all tensors of one call must live on the same CUDA device")
    return dev


def _stream(dev: torch.device) -> int:
    return torch.cuda.current_stream(dev).cuda_stream


def _rows(name: str, t, shape, dtype: str) -> None:
    """Check a tensor whose rows (last dimension) are contiguous and whose other strides are free."""
    if not isinstance(t, torch.Tensor):
        raise TypeError(f"{name}: expected a torch.Tensor, got {type(t).__name__}")
    if not t.is_cuda:
        raise ValueError(f"{name}: expected a CUDA tensor (the B200 target has no CPU path)")
    if t.dtype != _TORCH_DTYPES[dtype]:
        raise TypeError(f"{name}: dtype {t.dtype}, the program says {_TORCH_DTYPES[dtype]}")
    if t.shape != shape:
        raise ValueError(f"{name}: shape {tuple(t.shape)}, the program says {tuple(shape)}")
    if t.stride(-1) != 1:
        raise ValueError(f"{name}: rows must be contiguous")


def _pools(k_pages, v_pages, Hkv: int, page_size: int, D: int, dtype: str) -> None:
    """Check the two page pools of a paged cache."""
    want = _TORCH_DTYPES[dtype]
    for name, pool in (("k_pages", k_pages), ("v_pages", v_pages)):
        if not (isinstance(pool, torch.Tensor) and pool.is_cuda and pool.is_contiguous() and pool.dim() == 4
                and pool.shape[1:] == (Hkv, page_size, D) and pool.dtype == want):
            raise ValueError(f"{name}: expected a contiguous CUDA [num_pages, {Hkv}, {page_size}, {D}] {dtype} tensor")
    if k_pages.shape[0] != v_pages.shape[0]:
        raise ValueError("k_pages and v_pages must hold the same number of pages")


def status_buffer(dev: torch.device) -> torch.Tensor:
    """Per-device int32[4] that kernels with bounded device-side waits report into.

    Made once per device, whichever threads ask first: the native binding keeps the address (_first_status_buffer), so
    there is one tensor and it stays.  The stream that clears it is waited for, because every stream of the device uses
    it from then on.  A graph capture cannot wait: words made inside one are that call's alone, cleared by each replay.
    """
    idx = dev.index if dev.index is not None else torch.cuda.current_device()
    buf = _status_buffers.get(idx)
    if buf is None:
        with _status_lock, torch.cuda.device(idx):
            buf = _status_buffers.get(idx)
            if buf is None:
                buf = torch.zeros(native.STATUS_WORDS, dtype=torch.int32, device=torch.device("cuda", idx))
                if torch.cuda.is_current_stream_capturing():
                    _captured_words.setdefault(idx, []).append(buf)
                    return buf
                torch.cuda.current_stream(idx).synchronize()
                _status_buffers[idx] = buf
    return buf


def check_status(device=None) -> None:
    """Synchronise and raise if a kernel reported an expired device-side wait on ``device``."""
    dev = torch.device("cuda", torch.cuda.current_device()) if device is None else torch.device(device)
    own = status_buffer(dev)
    for buf in (own, *_captured_words.get(own.device.index, ())):
        rc = native.lib().nb200_status_read(buf.data_ptr(), None, _stream(dev))
        if rc != 0:
            buf.zero_()
        native.check(rc, "nb200 status")


def attn_fwd(q, k, v, out, *, shape, kv_len, dtype, scale_log2, causal) -> None:
    """Fused attention forward; ``shape`` = (B, H, Sq, D) of q and out, k/v are (B, H, kv_len, D)."""
    B, H, Sq, D = shape
    _check("q", q, shape, dtype)
    _check("k", k, (B, H, kv_len, D), dtype)
    _check("v", v, (B, H, kv_len, D), dtype)
    _check("out", out, shape, dtype)
    dev = _same_device(q, k, v, out)
    with torch.cuda.device(dev):
        rc = native.lib().nb200_attn_fwd(
            q.data_ptr(), k.data_ptr(), v.data_ptr(), out.data_ptr(), B, H, Sq, kv_len, D,
            native.DTYPE_CODES[dtype], float(scale_log2), int(bool(causal)),
            status_buffer(dev).data_ptr(), _stream(dev))
    native.check(rc, "nb200_attn_fwd")


def decode_workspace_floats(B, Hq, D, n_splits) -> int:
    return native.lib().nb200_decode_workspace_bytes(B, Hq, D, n_splits) // 4


def decode_splitk(q, k, v, partials, out, *, B, Hq, Hkv, L, D, n_splits, dtype, scale_log2) -> None:
    """Split-K flash-decoding + LSE combine; ``partials`` is fp32 [B, Hq, n_splits, D + 2] scratch.

    ``n_splits = 0`` lets the library choose the count for the GPU it runs on (nb200_decode_auto_splits), bounded
    by the third extent of ``partials``, of which the first B*Hq*n*(D+2) floats are then used.
    """
    _check("q", q, (B, Hq, D), dtype)
    _check("k", k, (B, Hkv, L, D), dtype)
    _check("v", v, (B, Hkv, L, D), dtype)
    cap = n_splits if n_splits > 0 else (partials.shape[2] if isinstance(partials, torch.Tensor) and partials.dim() == 4 else 0)
    _check("partials", partials, (B, Hq, cap, D + 2), torch.float32)
    _check("out", out, (B, Hq, D), dtype)
    dev = _same_device(q, k, v, partials, out)
    lib = native.lib()
    with torch.cuda.device(dev):
        st = _stream(dev)
        if n_splits == 0:
            n_splits = lib.nb200_decode_auto_splits(B, Hkv, L, cap)
            if n_splits <= 0:
                raise native.NativeLibraryError("nb200_decode_auto_splits could not choose a split count")
        rc = lib.nb200_decode_splitk(q.data_ptr(), k.data_ptr(), v.data_ptr(), partials.data_ptr(), B, Hq, Hkv,
                                     L, D, n_splits, native.DTYPE_CODES[dtype], float(scale_log2),
                                     status_buffer(dev).data_ptr(), st)
        native.check(rc, "nb200_decode_splitk")
        rc = lib.nb200_decode_combine(partials.data_ptr(), out.data_ptr(), B * Hq, D, n_splits,
                                      n_splits * (D + 2), D + 2, native.DTYPE_CODES[dtype], st)
        native.check(rc, "nb200_decode_combine")


def decode_paged(q, k_pages, v_pages, block_table, seq_lens, partials, out, *, B, Hq, Hkv, max_pages, page_size, D,
                 n_splits, dtype, scale_log2) -> None:
    """Split-K decode over a paged KV cache + combine; pools are [num_pages, Hkv, page_size, D]."""
    _check("q", q, (B, Hq, D), dtype)
    for name, pool in (("k_pages", k_pages), ("v_pages", v_pages)):
        if not (isinstance(pool, torch.Tensor) and pool.is_cuda and pool.is_contiguous() and pool.dim() == 4
                and tuple(pool.shape[1:]) == (Hkv, page_size, D) and pool.dtype == _TORCH_DTYPES[dtype]):
            raise ValueError(f"{name}: expected a contiguous CUDA [num_pages, {Hkv}, {page_size}, {D}] {dtype} tensor")
    if k_pages.shape[0] != v_pages.shape[0]:
        raise ValueError("k_pages and v_pages must hold the same number of pages")
    _check("block_table", block_table, (B, max_pages), torch.int32)
    _check("seq_lens", seq_lens, (B,), torch.int32)
    _check("partials", partials, (B, Hq, n_splits, D + 2), torch.float32)
    _check("out", out, (B, Hq, D), dtype)
    dev = _same_device(q, k_pages, v_pages, block_table, seq_lens, partials, out)
    lib = native.lib()
    with torch.cuda.device(dev):
        st = _stream(dev)
        rc = lib.nb200_decode_paged_splitk(q.data_ptr(), k_pages.data_ptr(), v_pages.data_ptr(), block_table.data_ptr(),
                                           seq_lens.data_ptr(), partials.data_ptr(), B, Hq, Hkv, int(k_pages.shape[0]),
                                           max_pages, page_size, D, n_splits, native.DTYPE_CODES[dtype],
                                           float(scale_log2), status_buffer(dev).data_ptr(), st)
        native.check(rc, "nb200_decode_paged_splitk")
        rc = lib.nb200_decode_combine(partials.data_ptr(), out.data_ptr(), B * Hq, D, n_splits,
                                      n_splits * (D + 2), D + 2, native.DTYPE_CODES[dtype], st)
        native.check(rc, "nb200_decode_combine")


def decode_combine(partials, out, *, rows, D, n_splits, row_stride, split_stride, out_dtype) -> None:
    """LSE combine with explicit strides (in floats); out_dtype 'f32' writes a partial of D + 2 floats."""
    if not (partials.is_cuda and out.is_cuda and partials.dtype == torch.float32):
        raise ValueError("decode_combine: partials must be a CUDA fp32 tensor and out a CUDA tensor")
    if not (partials.is_contiguous() and out.is_contiguous()):
        raise ValueError("decode_combine: tensors must be contiguous")
    need = (rows - 1) * row_stride + (n_splits - 1) * split_stride + D + 2
    if partials.numel() < need:
        raise ValueError(f"decode_combine: partials has {partials.numel()} floats, the strides need {need}")
    out_elems = rows * (D + 2 if out_dtype == "f32" else D)
    if out.numel() != out_elems or out.dtype != _TORCH_DTYPES[out_dtype]:
        raise ValueError("decode_combine: out has the wrong size or dtype")
    dev = _same_device(partials, out)
    with torch.cuda.device(dev):
        rc = native.lib().nb200_decode_combine(partials.data_ptr(), out.data_ptr(), rows, D, n_splits,
                                               row_stride, split_stride, native.DTYPE_CODES[out_dtype],
                                               _stream(dev))
    native.check(rc, "nb200_decode_combine")


def decode_merge_nccl(local_partial, gathered, out, *, rows, D, world, out_dtype, comm) -> None:
    """All-gather per-rank partials over ``comm`` (a ``nccl_comm.Communicator``) and combine across ranks."""
    _check("local_partial", local_partial, (rows, D + 2), torch.float32)
    _check("gathered", gathered, (world, rows, D + 2), torch.float32)
    _check("out", out, (rows, D + 2 if out_dtype == "f32" else D), out_dtype)
    dev = _same_device(local_partial, gathered, out)
    with torch.cuda.device(dev):
        rc = native.lib().nb200_decode_merge_nccl(local_partial.data_ptr(), gathered.data_ptr(), out.data_ptr(),
                                                  rows, D, world, native.DTYPE_CODES[out_dtype], comm.handle,
                                                  _stream(dev))
    native.check(rc, "nb200_decode_merge_nccl")


# The operators of a decode step go through the native binding, which checks the tensors and launches in a few
# microseconds; it returns None if a tensor is not what the arguments say, and the checks here then say which.

def _refuse(what: str):
    raise ValueError(f"{what}: the tensors do not fit the arguments")   # the checks before this name the tensor


def _first_status_buffer(dev: torch.device) -> None:
    """Give the native binding the address of a device's status words, which are not made inside a graph capture: their
    memory would end with the graph."""
    if dev.index not in _status_buffers and torch.cuda.is_current_stream_capturing():
        raise RuntimeError("the first call on a device makes its status words: call once before capturing a graph")
    native.binding().set_status(dev.index, status_buffer(dev).data_ptr())


def _weight_checks(weights, D: int, dtype: str) -> list:
    """Check the norm weights that are there; return them."""
    there = [(name, w) for name, w in zip(("q_weight", "k_weight"), weights) if w is not None]
    for name, w in there:
        _check(name, w, (D,), dtype)
    return [w for _, w in there]


def qk_norm_rope(q, k, positions, inv_freq, q_out, k_out, q_weight=None, k_weight=None, *, B, S, Hq, Hkv, D, rot_dim,
                 interleaved, eps, dtype) -> None:
    """Norm of every query and key head (where it has weights) and position rotation, in one pass.

    q [B, S, Hq, D] and k [B, S, Hkv, D] are token-major, as a projection leaves them; q_out [B, Hq, S, D] and
    k_out [B, Hkv, S, D] head-major, as ``attn_fwd`` reads them.  Rows of D are contiguous, the other strides free
    multiples of 16 bytes (so an output may also be its input's ``transpose(1, 2)``, in place).  positions is int32
    [S] or [B, S], inv_freq fp32 [rot_dim / 2]; the weights are [D].
    """
    rc = native.binding().qk_norm_rope(q, k, positions, inv_freq, q_out, k_out, q_weight, k_weight, B, S, Hq, Hkv, D,
                                       rot_dim, interleaved, eps, native.DTYPE_CODES[dtype])
    if rc == 0:
        return
    if rc is None:
        _rows("q", q, (B, S, Hq, D), dtype)
        _rows("k", k, (B, S, Hkv, D), dtype)
        _rows("q_out", q_out, (B, Hq, S, D), dtype)
        _rows("k_out", k_out, (B, Hkv, S, D), dtype)
        one_row = isinstance(positions, torch.Tensor) and positions.dim() == 1
        _check("positions", positions, (S,) if one_row else (B, S), torch.int32)
        _check("inv_freq", inv_freq, (rot_dim // 2,), torch.float32)
        _same_device(q, k, positions, inv_freq, q_out, k_out, *_weight_checks((q_weight, k_weight), D, dtype))
        _refuse("qk_norm_rope")
    native.check(rc, "nb200_qk_norm_rope")


def _paged_checks(k_pages, v_pages, block_table, cu_seqlens, seq_lens, B, Hkv, max_pages, page_size, D, dtype) -> None:
    _pools(k_pages, v_pages, Hkv, page_size, D, dtype)
    _check("block_table", block_table, (B, max_pages), torch.int32)
    _check("cu_seqlens", cu_seqlens, (B + 1,), torch.int32)
    _check("seq_lens", seq_lens, (B,), torch.int32)


def rope_append(q, k, v, k_pages, v_pages, block_table, cu_seqlens, seq_lens, inv_freq, q_out, q_weight=None,
                k_weight=None, *, T, B, Hq, Hkv, max_pages, page_size, D, rot_dim, interleaved, eps, dtype) -> None:
    """Append a ragged batch of new tokens to the paged cache of ``decode_paged``, normed and rotated on the way.

    Rows cu_seqlens[b] .. cu_seqlens[b+1]-1 of k, v [T, Hkv, D] are the last tokens of sequence b, seq_lens[b] its
    length with them; q [T, Hq, D] is rotated into q_out the same way (both None with Hq = 0: keys and values only).
    Rows of D are contiguous, the other strides free multiples of 16 bytes; q_out may be q.  Positions or pages that
    the table or the pool does not have are reported by ``check_status``.
    """
    args = (q, k, v, k_pages, v_pages, block_table, cu_seqlens, seq_lens, inv_freq, q_out, q_weight, k_weight, T, B, Hq,
            Hkv, max_pages, page_size, D, rot_dim, interleaved, eps, native.DTYPE_CODES[dtype])
    rc = native.binding().rope_append(*args)
    if rc == 0:
        return
    if rc is None:
        if Hq == 0:
            if q is not None or q_out is not None:
                raise ValueError("rope_append: Hq = 0 goes with q = q_out = None")
        else:
            _rows("q", q, (T, Hq, D), dtype)
            _rows("q_out", q_out, (T, Hq, D), dtype)
        _rows("k", k, (T, Hkv, D), dtype)
        _rows("v", v, (T, Hkv, D), dtype)
        _paged_checks(k_pages, v_pages, block_table, cu_seqlens, seq_lens, B, Hkv, max_pages, page_size, D, dtype)
        _check("inv_freq", inv_freq, (rot_dim // 2,), torch.float32)
        dev = _same_device(k, v, k_pages, v_pages, block_table, cu_seqlens, seq_lens, inv_freq,
                           *_weight_checks((q_weight, k_weight), D, dtype), *((q, q_out) if Hq else ()))
        _first_status_buffer(dev)
        rc = native.binding().rope_append(*args)
        if rc is None:
            _refuse("rope_append")
    native.check(rc, "nb200_rope_append")


def attn_paged_workspace_bytes() -> int:
    """Scratch memory of one ``attn_paged`` call, whatever its sizes."""
    return native.lib().nb200_attn_paged_workspace_bytes()


def attn_paged(q, k_pages, v_pages, block_table, cu_seqlens, seq_lens, workspace, out, *, T, B, Hq, Hkv, max_pages,
               page_size, D, dtype, scale_log2) -> None:
    """Attention of a ragged batch of new tokens (see ``rope_append``) over the paged cache that holds them already.

    q, out [T, Hq, D] with contiguous rows and token and head strides that are multiples of 16 bytes; workspace is a
    uint8 tensor of attn_paged_workspace_bytes(), one for each call that can run at the same time.
    """
    args = (q, k_pages, v_pages, block_table, cu_seqlens, seq_lens, workspace, out, T, B, Hq, Hkv, max_pages, page_size, D,
            native.DTYPE_CODES[dtype], scale_log2)
    rc = native.binding().attn_paged(*args)
    if rc == 0:
        return
    if rc is None:
        _rows("q", q, (T, Hq, D), dtype)
        _rows("out", out, (T, Hq, D), dtype)
        _paged_checks(k_pages, v_pages, block_table, cu_seqlens, seq_lens, B, Hkv, max_pages, page_size, D, dtype)
        need = attn_paged_workspace_bytes()
        if not (isinstance(workspace, torch.Tensor) and workspace.is_cuda and workspace.is_contiguous()
                and workspace.numel() * workspace.element_size() >= need):
            raise ValueError(f"workspace: need a contiguous CUDA tensor of at least {need} bytes")
        _first_status_buffer(_same_device(q, k_pages, v_pages, block_table, cu_seqlens, seq_lens, workspace, out))
        rc = native.binding().attn_paged(*args)
        if rc is None:
            _refuse("attn_paged")
    native.check(rc, "nb200_attn_paged")


def selective_scan(u, delta, A, Bm, Cm, Dskip, z, out, *, B, Dm, L, N, dtype) -> None:
    """Mamba-1 selective scan forward (layouts in include/nb200.h)."""
    _check("u", u, (B, Dm, L), dtype)
    _check("delta", delta, (B, Dm, L), dtype)
    _check("A", A, (Dm, N), torch.float32)
    _check("Bm", Bm, (B, N, L), dtype)
    _check("Cm", Cm, (B, N, L), dtype)
    _check("Dskip", Dskip, (Dm,), torch.float32)
    _check("z", z, (B, Dm, L), dtype)
    _check("out", out, (B, Dm, L), dtype)
    dev = _same_device(u, delta, A, Bm, Cm, Dskip, z, out)
    with torch.cuda.device(dev):
        rc = native.lib().nb200_selective_scan_fwd(
            u.data_ptr(), delta.data_ptr(), A.data_ptr(), Bm.data_ptr(), Cm.data_ptr(), Dskip.data_ptr(),
            z.data_ptr(), out.data_ptr(), B, Dm, L, N, native.DTYPE_CODES[dtype], _stream(dev))
    native.check(rc, "nb200_selective_scan_fwd")


def check_workspace_status(workspace) -> None:
    """Synchronise and raise if the SSD kernel recorded an expired device-side wait in ``workspace``."""
    dev = workspace.device
    rc = native.lib().nb200_status_read(workspace.data_ptr(), None, _stream(dev))
    native.check(rc, "nb200 ssd status")


def ssd_workspace_bytes(B, L, H, P, N, G, chunk) -> int:
    return native.lib().nb200_ssd_workspace_bytes(B, L, H, P, N, G, chunk)


def ssd_launches(B, L, H, P, N, G, chunk) -> int:
    """Kernel launches one SSD call makes on the current device (2 when the sequences are cut into segments)."""
    return native.lib().nb200_ssd_launches(B, L, H, P, N, G, chunk)


def ssd_chunk_scan(x, dt, A, Bm, Cm, workspace, y, *, B, L, H, P, N, G, chunk, dtype) -> None:
    """Mamba-2 SSD chunked scan forward; ``workspace`` is a uint8 tensor of ssd_workspace_bytes(...)."""
    _check("x", x, (B, L, H, P), dtype)
    _check("dt", dt, (B, L, H), torch.float32)
    _check("A", A, (H,), torch.float32)
    _check("Bm", Bm, (B, L, G, N), dtype)
    _check("Cm", Cm, (B, L, G, N), dtype)
    _check("y", y, (B, L, H, P), dtype)
    need = ssd_workspace_bytes(B, L, H, P, N, G, chunk)
    if not (isinstance(workspace, torch.Tensor) and workspace.is_cuda and workspace.is_contiguous()
            and workspace.numel() * workspace.element_size() >= need):
        raise ValueError(f"workspace: need a contiguous CUDA tensor of at least {need} bytes")
    dev = _same_device(x, dt, A, Bm, Cm, workspace, y)
    with torch.cuda.device(dev):
        rc = native.lib().nb200_ssd_chunk_scan_fwd(
            x.data_ptr(), dt.data_ptr(), A.data_ptr(), Bm.data_ptr(), Cm.data_ptr(), y.data_ptr(),
            workspace.data_ptr(), B, L, H, P, N, G, chunk, native.DTYPE_CODES[dtype], _stream(dev))
    native.check(rc, "nb200_ssd_chunk_scan_fwd")
