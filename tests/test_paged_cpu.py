"""The paged-cache operators without a GPU: refusals of the C ABI and the runtime, declarations, the oracle."""

import ast
import ctypes
import math

import pytest
import torch

from neptune_mlir import native, programs, runtime
from neptune_mlir.translators import b200
from oracle import attention, paged


@pytest.fixture
def ptr():
    buf = ctypes.create_string_buffer(64)
    p = ctypes.addressof(buf)
    yield p + (-p) % 16, buf


def longs(*values):
    return (ctypes.c_longlong * len(values))(*values)


def test_norm_rope_rejects_bad_calls_without_a_gpu(native_lib, ptr):
    lib, p = native.load(str(native_lib)), ptr[0]
    plain = longs(*[1024, 128, 128] * 4, 0)

    def call(q=p, strides=plain, B=1, S=8, Hq=1, Hkv=1, D=128, rot=128, eps=1e-6, dtype=1, wq=None):
        return lib.nb200_qk_norm_rope(q, p, p, p, p, p, wq, None, strides, B, S, Hq, Hkv, D, rot, 0, eps, dtype, None)

    for kwargs, code, text in (
            (dict(q=None), -1, b"null pointer"), (dict(S=0), -1, b"non-positive"), (dict(dtype=5), -2, b"dtype 5"),
            (dict(D=120), -2, b"D = 120"), (dict(D=272), -2, b"D = 272"), (dict(rot=24), -2, b"rot_dim = 24"),
            (dict(rot=144), -2, b"rot_dim = 144"), (dict(rot=0), -2, b"rot_dim = 0"), (dict(eps=-1.0), -1, b"eps"),
            (dict(eps=math.nan), -1, b"eps"), (dict(q=p + 2), -1, b"q must be 16-byte aligned"),
            (dict(strides=longs(*[1024, 132, 128] * 4, 0)), -1, b"strides of q"), (dict(wq=p + 4), -1, b"weights"),
            (dict(B=1 << 16, S=1 << 16), -2, b"31 bits"), (dict(Hq=70000), -2, b"too many heads")):
        assert call(**kwargs) == code and text in lib.nb200_last_error(), kwargs


def test_rope_append_rejects_bad_calls_without_a_gpu(native_lib, ptr):
    lib, p = native.load(str(native_lib)), ptr[0]

    def call(q=p, k=p, strides=longs(*[128, 128] * 4), T=1, B=1, Hq=1, page=64, max_pages=4, D=128, rot=128, dtype=1, pool=p):
        return lib.nb200_rope_append(q, k, p, p, pool, p, p, p, p, p, None, None, strides, T, B, Hq, 1, 8, max_pages, page,
                                     D, rot, 0, 1e-6, dtype, None, None)

    for kwargs, code, text in (
            (dict(k=None), -1, b"null pointer"), (dict(q=None), -1, b"null pointer"), (dict(T=0), -1, b"non-positive"),
            (dict(B=0), -1, b"non-positive"), (dict(Hq=-1), -1, b"non-positive"), (dict(dtype=2), -2, b"f16 and bf16 only"),
            (dict(D=64), -2, b"only 128"), (dict(page=16), -2, b"only 64 rows per page"), (dict(rot=136), -2, b"rot_dim"),
            (dict(max_pages=1 << 25), -2, b"31 bits"), (dict(pool=p + 8), -1, b"page pools"),
            (dict(strides=longs(128, 128, 128, 4, 128, 128, 128, 128)), -1, b"strides of k")):
        assert call(**kwargs) == code and text in lib.nb200_last_error(), kwargs


def test_attn_paged_rejects_bad_calls_without_a_gpu(native_lib, ptr):
    lib, p = native.load(str(native_lib)), ptr[0]
    assert lib.nb200_attn_paged_workspace_bytes() % 16 == 0

    def call(q=p, work=p, strides=longs(1024, 128, 1024, 128), T=1, B=1, Hq=8, Hkv=2, pages=8, max_pages=4, page=64, D=128,
             dtype=1, scale=0.1):
        return lib.nb200_attn_paged(q, p, p, p, p, p, work, p, strides, T, B, Hq, Hkv, pages, max_pages, page, D, dtype, scale,
                                    None, None)

    for kwargs, code, text in (
            (dict(work=None), -1, b"null pointer"), (dict(T=0), -1, b"non-positive"), (dict(scale=0.0), -1, b"scale_log2"),
            (dict(scale=math.nan), -1, b"scale_log2"), (dict(dtype=2), -2, b"f16 and bf16 only"), (dict(D=64), -2, b"only 128"),
            (dict(page=32), -2, b"only 64 rows per page"), (dict(Hq=7), -2, b"Hq % Hkv"), (dict(Hq=258), -2, b"128 query heads"),
            (dict(q=p + 8), -1, b"16-byte aligned"), (dict(T=2, strides=longs(1020, 128, 1024, 128)), -1, b"strides"),
            (dict(T=2, strides=longs(-1024, 128, 1024, 128)), -1, b"strides"), (dict(strides=longs(1024, 128, 1024, 0)), -1, b"strides"),
            (dict(T=1 << 30), -2, b"30 bits"), (dict(max_pages=1 << 25), -2, b"30 bits"),
            (dict(pages=1 << 30), -2, b"num_pages * Hkv")):
        assert call(**kwargs) == code and text in lib.nb200_last_error(), kwargs


def test_outputs_whose_rows_lie_over_one_another_are_refused(native_lib, ptr):
    lib, p = native.load(str(native_lib)), ptr[0]

    def norm_rope(q_out, k_out=(2048, 256, 128), B=2, S=8):
        strides = longs(2048, 256, 128, 2048, 256, 128, *q_out, *k_out, 0)
        return lib.nb200_qk_norm_rope(p, p, p, p, p, p, None, None, strides, B, S, 2, 2, 128, 128, 0, 1e-6, 1, None)

    def append(q_out):
        return lib.nb200_rope_append(p, p, p, p, p, p, p, p, p, p, None, None, longs(256, 128, 256, 128, 256, 128, *q_out), 2, 1,
                                     2, 2, 8, 4, 64, 128, 128, 0, 1e-6, 1, None, None)

    for call, args, name in ((norm_rope, [(0, 256, 128)], b"q_out"), (norm_rope, [(2048, 0, 128)], b"q_out"),
                             (norm_rope, [(2048, 256, 64)], b"q_out"), (norm_rope, [(2048, 256, 128), (2048, 256, 0)], b"k_out"),
                             (append, [(0, 128)], b"q_out"), (append, [(256, 120)], b"q_out")):
        assert call(*args) == -1 and b"strides of " + name + b" must be at least a row" in lib.nb200_last_error(), args


def test_runtime_refuses_cpu_tensors(native_lib):
    x = torch.zeros((1, 4, 2, 128), dtype=torch.bfloat16)
    i = torch.zeros((4,), dtype=torch.int32)
    with pytest.raises(ValueError, match="CUDA tensor"):
        runtime.qk_norm_rope(x, x, i, torch.zeros(64), x, x, B=1, S=4, Hq=2, Hkv=2, D=128, rot_dim=128, interleaved=False,
                             eps=1e-6, dtype="bf16")
    facts = dict(T=4, B=1, Hkv=2, max_pages=1, page_size=64, D=128, dtype="bf16")
    with pytest.raises(ValueError, match="CUDA tensor"):
        runtime.rope_append(x[0], x[0], x[0], x, x, i, i, i, i, x[0], Hq=2, rot_dim=128, interleaved=False, eps=1e-6, **facts)
    with pytest.raises(ValueError, match="Hq = 0"):
        runtime.rope_append(x[0], x[0], x[0], x, x, i, i, i, i, None, Hq=0, rot_dim=128, interleaved=False, eps=1e-6, **facts)
    with pytest.raises(TypeError, match="torch.Tensor"):
        runtime.attn_paged(None, x, x, i, i, i, x, x[0], Hq=2, scale_log2=0.1, **facts)


def test_declarations(tmp_path, monkeypatch):
    cases = (
        (programs.qk_norm_rope_decl("f", 2, 9, 8, 4, 96, 32, norm=False, interleaved=True, dtype="f32"), "ptr_5, B=2, S=9, Hq=8, "
         "Hkv=4, D=96, rot_dim=32, interleaved=True, eps=", "memref<2x9xi32>", "memref<2x9xi64>", "positions"),
        (programs.rope_append_decl("f", 40, 3, 8, 2, 21, 5, 128, 64), "ptr_11, T=40, B=3, Hq=8, Hkv=2, max_pages=5, page_size=64, "
         "D=128, rot_dim=64, interleaved=False, eps=", "memref<4xi32>", "memref<3xi32>", "cu_seqlens"),
        (programs.attn_paged_decl("f", 40, 3, 8, 2, 21, 5, 128, 4096), "ptr_7, T=40, B=3, Hq=8, Hkv=2, max_pages=5, page_size=64, "
         "D=128, dtype='bf16', scale_log2=0.127517", "memref<4096xi8>", "memref<4096xf32>", "workspace"))
    path = tmp_path / "f.mlir"
    for text, part, old, new, why in cases:
        path.write_text(text)
        sources = []
        for front in ("native", "python"):
            monkeypatch.setenv("NEPTUNE_HTILE_FRONT", front)
            sources.append(ast.unparse(b200.translate_file(str(path))))
        assert sources[0] == sources[1] and part in sources[0], sources[0]
        assert old in text
        path.write_text(text.replace(old, new))
        with pytest.raises(NotImplementedError, match=why):
            b200.translate_file(str(path))


def test_the_oracle_agrees_with_the_dense_one():
    """Chunk attention over pages is causal attention over the sequence, row for row."""
    S, H, D = 150, 2, 128
    gen = torch.Generator().manual_seed(0)
    q, k, v = (torch.randn((1, H, S, D), generator=gen) for _ in range(3))
    ref = attention.attention_reference(q, k, v, causal=True)[0].transpose(0, 1)
    table = torch.tensor([[2, 0, 3]], dtype=torch.int32)
    pools = [torch.full((4, H, 64, D), float("nan")) for _ in range(2)]
    for x, pool in zip((k, v), pools):
        for p in range(3):
            rows = min(64, S - 64 * p)
            pool[table[0, p], :, :rows] = x[0, :, 64 * p:64 * p + rows]
    out, _, _ = paged.attn_paged(q[0, :, 100:].transpose(0, 1), *pools, table, [0, 50], [S], 1 / math.sqrt(D))
    torch.testing.assert_close(out.float(), ref[100:], rtol=1e-5, atol=1e-5)


def test_the_oracle_rotates_a_pair_by_its_angle():
    """Two halves or neighbours: a relative rotation depends on the distance of the positions alone."""
    x = torch.randn((2, 1, 32), generator=torch.Generator().manual_seed(1), dtype=torch.float64)
    freq = torch.tensor([1.0, 0.1, 0.01, 0.001] * 4)
    for interleaved in (False, True):
        dots = []
        for at in (0, 977):
            y, _ = paged.norm_rope(x, None, torch.tensor([at, at + 13]), freq, 0.0, interleaved)
            dots.append((y[0, 0] * y[1, 0]).sum())
        torch.testing.assert_close(dots[0], dots[1])
        y, _ = paged.norm_rope(x, torch.ones(32), torch.tensor([0, 0]), freq, 0.0, interleaved)
        torch.testing.assert_close(y.pow(2).mean(-1), torch.ones((2, 1), dtype=torch.float64))


def test_outputs_whose_rows_coincide_only_together_are_refused(native_lib, ptr):
    """Strides that are each a row or more, and of which two, or one and a multiple of another, are the same address."""
    lib, p = native.load(str(native_lib)), ptr[0]

    def norm_rope(q_out, B=2, S=8):
        strides = longs(2048, 256, 128, 2048, 256, 128, *q_out, 2048, 256, 128, 0)
        return lib.nb200_qk_norm_rope(p, p, p, p, p, p, None, None, strides, B, S, 2, 2, 128, 128, 0, 1e-6, 1, None)

    def append(q_out, Hq=2):
        strides = longs(128 * Hq, 128, 256, 128, 256, 128, *q_out)
        return lib.nb200_rope_append(p, p, p, p, p, p, p, p, p, p, None, None, strides, 2, 1, Hq, 2, 8, 4, 64, 128, 128, 0,
                                     1e-6, 1, None, None)

    def attend(out, T=2):
        return lib.nb200_attn_paged(p, p, p, p, p, p, p, p, longs(512, 128, *out), T, 1, 4, 2, 8, 4, 64, 128, 1, 0.1, None, None)

    for call, out, name in ((norm_rope, (128, 128, 128), b"q_out"), (norm_rope, (2048, 128, 128), b"q_out"),
                            (norm_rope, (256, 256, 128), b"q_out"), (norm_rope, (1024, 256, -128), b"q_out"),
                            (norm_rope, (2048, 256, 2048), b"q_out"), (norm_rope, (1024, 128, 896), b"q_out"),
                            (append, (128, 128), b"q_out"), (append, (256, 256), b"q_out"), (append, (200, 128), b"q_out"),
                            (attend, (128, 128), b"out"), (attend, (384, 128), b"out"), (attend, (136, 256), b"out")):
        assert call(out) == -1 and b"rows of " + name + b" must lie apart" in lib.nb200_last_error(), (call, out, lib.nb200_last_error())


def test_the_batch_or_token_stride_of_an_extent_of_one_is_not_looked_at(native_lib, ptr):
    """It is never taken, whatever a slice of a wider tensor left there.  (A check that comes later refuses these calls.)"""
    lib, p = native.load(str(native_lib)), ptr[0]
    for strides, extents in (((1001, 128, 128), (1, 8, 1)), ((1024, 3, 128), (2, 1, 1)), ((1, 1, 128), (1, 1, 2))):
        B, S, H = extents
        rc = lib.nb200_qk_norm_rope(p, p, p, p, p, p, p + 4, None, longs(*strides * 4, 0), B, S, H, H, 128, 128, 0, 1e-6, 1, None)
        assert rc == -1 and b"weights must be" in lib.nb200_last_error(), (strides, lib.nb200_last_error())
    for strides, T, H in (((77, 128), 1, 2), ((0, 128), 1, 1), ((-3, 256), 1, 4)):
        rc = lib.nb200_rope_append(p, p, p, p, p + 8, p, p, p, p, p, None, None, longs(*strides * 4), T, 1, H, H, 8, 4, 64, 128,
                                   128, 0, 1e-6, 1, None, None)
        assert rc == -1 and b"page pools" in lib.nb200_last_error(), (strides, lib.nb200_last_error())


def test_attention_in_place_is_refused(native_lib, ptr):
    """Several CTAs read a tile's queries after the first has written its part of the output."""
    lib, p = native.load(str(native_lib)), ptr[0]
    for strides in (longs(512, 128, 512, 128), longs(512, 128, 1024, 256)):
        rc = lib.nb200_attn_paged(p, p, p, p, p, p, p, p, strides, 2, 1, 4, 2, 8, 4, 64, 128, 1, 0.1, None, None)
        assert rc == -1 and b"out must not be q" in lib.nb200_last_error()
