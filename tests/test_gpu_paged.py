"""Norm and rotation, append to the paged cache and chunk attention over it, against 64-bit definitions on the CPU.

Bounds.  A rounding to the storage type is off by h = eps(dtype) / 2 relative to the value.

* Norm and rotation work in fp32 (u = 2^-24): the sum of D <= 256 squares by 8 sequential terms and 5 tree levels, the
  division, root and weight give at most 20 u relative, the angle (a fraction of a turn, at most a half, rounded to
  fp32: pi u) and the sine and cosine (2 ulp = 4 u) at most 8 u of |y1| + |y2|, two products and a sum 3 u more:
  |out - exact| <= h |exact| + 32 u (|y1| + |y2|), and the smallest subnormal of fp16.
* Attention: a weight is rounded to the storage type before the second product (h relative; in fp16 a weight below 2^-14
  by 2^-25 of the row's largest, whose weight is at least 1), a score sums 128 products in fp32 (at most
  128 * 2u * sum |q_i k_i|, a truncating accumulator included, and the same relative error in the weight), and the sums
  over the rows add len * 2u:  |out - exact| <= h |exact| + (h + 2 * 256 u * score + 2 len u) sum w |v| + len 2^-25 max|v|.
"""

import math

import pytest
import torch

from gpu_util import finish, translate_text
from oracle import paged

pytestmark = pytest.mark.gpu

LOG2E = 1.4426950408889634
U = 2.0 ** -24
PAGE, D = 64, 128
NAMES = {torch.float16: "f16", torch.bfloat16: "bf16", torch.float32: "f32"}


def randn(shape, seed, dtype):
    return torch.randn(shape, generator=torch.Generator().manual_seed(seed)).to(dtype)


def frequencies(rot):
    return 10000.0 ** (-torch.arange(0, rot, 2, dtype=torch.float32) / rot)


def close_to_rotation(got, exact, size, dtype):
    h = torch.finfo(dtype).eps / 2
    bound = h * exact.abs() + 32 * U * size + 2.0 ** -25 * (dtype == torch.float16)
    err = (got.double().cpu() - exact).abs()
    assert bool((err <= bound).all()), f"worst excess {(err - bound).max().item():.3e}"


def close_to_attention(got, exact, spread, score, length, vmax, dtype):
    h = torch.finfo(dtype).eps / 2
    bound = h * exact.abs() + (h + 512 * U * score + 2 * length * U) * spread + length * 2.0 ** -25 * vmax
    err = (got.double().cpu() - exact).abs()
    assert bool((err <= bound).all()), f"worst excess {(err - bound).max().item():.3e} over {bound.max().item():.3e}"


class Batch:
    """A ragged batch over a paged cache: pages dealt in random order, NaN wherever a sequence owns nothing."""

    def __init__(self, new, lens, Hkv, dtype, seed=0, pad=2, spare=3, max_pages=None):
        self.new, self.lens, self.Hkv, self.dtype = new, lens, Hkv, dtype
        self.cu = [0]
        for n in new:
            self.cu.append(self.cu[-1] + n)
        self.T = self.cu[-1] + pad
        self.max_pages = max_pages or max(1, max((n + PAGE - 1) // PAGE for n in lens))
        need = [min(self.max_pages, max(0, (n + PAGE - 1) // PAGE)) for n in lens]
        self.num_pages = sum(need) + spare
        perm = torch.randperm(self.num_pages, generator=torch.Generator().manual_seed(seed)).to(torch.int32)
        sentinel = int(perm[-1])                                  # belongs to no sequence
        self.table = torch.full((len(lens), self.max_pages), sentinel, dtype=torch.int32)
        self.k = torch.full((self.num_pages, Hkv, PAGE, D), float("nan"), dtype=dtype)
        self.v = self.k.clone()
        at = 0
        for b, count in enumerate(need):
            self.table[b, :count] = perm[at:at + count]
            at += count
            for p in range(count):
                rows = min(PAGE, lens[b] - p * PAGE)
                self.k[self.table[b, p], :, :rows] = randn((Hkv, rows, D), seed + 1000 * b + 2 * p + 1, dtype)
                self.v[self.table[b, p], :, :rows] = randn((Hkv, rows, D), seed + 1000 * b + 2 * p + 2, dtype)

    def device_args(self, dev):
        return (self.table.to(dev), torch.tensor(self.cu, dtype=torch.int32, device=dev),
                torch.tensor(self.lens, dtype=torch.int32, device=dev))

    def facts(self, Hq):
        return dict(T=self.T, B=len(self.lens), Hq=Hq, Hkv=self.Hkv, max_pages=self.max_pages, page_size=PAGE, D=D,
                    dtype=NAMES[self.dtype])


def scratch(dev):
    from neptune_mlir import runtime

    return torch.full((runtime.attn_paged_workspace_bytes(),), 0xFF, dtype=torch.uint8, device=dev)   # NaN, if read as fp32


def attend(batch, q, dev, out=None, **over):
    from neptune_mlir import runtime

    out = torch.full(q.shape, 7.0, dtype=batch.dtype, device=dev) if out is None else out
    runtime.attn_paged(q, batch.k.to(dev), batch.v.to(dev), *batch.device_args(dev), scratch(dev), out,
                       scale_log2=LOG2E / math.sqrt(D), **{**batch.facts(q.shape[1]), **over})
    return out


def check_attention(batch, q, out):
    exact, spread, score = paged.attn_paged(q, batch.k, batch.v, batch.table, batch.cu, batch.lens, 1 / math.sqrt(D))
    total = batch.cu[-1]
    vmax = batch.v[~batch.v.isnan()].abs().max().item() if bool((~batch.v.isnan()).any()) else 0.0
    close_to_attention(out[:total], exact[:total], spread[:total], score, max(batch.lens), vmax, batch.dtype)
    assert bool((out[total:].float() == 7.0).all()), "rows behind the last sequence were written"


# ---- norm and rotation -----------------------------------------------------------------------------------------------

@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16, torch.float32], ids=NAMES.get)
@pytest.mark.parametrize("interleaved", [False, True], ids=["halves", "neighbours"])
@pytest.mark.parametrize("B,S,Hq,Hkv,dim,rot,norm", [
    (1, 1, 1, 1, 16, 16, True), (2, 5, 4, 2, 32, 16, True), (1, 33, 3, 1, 64, 64, False), (2, 129, 8, 8, 128, 128, True),
    (1, 700, 33, 3, 128, 96, True), (3, 17, 5, 5, 96, 32, True), (1, 9, 2, 1, 256, 256, True), (2, 301, 12, 4, 208, 80, False),
])
def test_norm_and_rotation(cuda, native_lib, dtype, interleaved, B, S, Hq, Hkv, dim, rot, norm):
    """Views into a packed projection in, head-major tensors out; one row of positions or one per batch element."""
    from neptune_mlir import runtime

    x = randn((B, S, (Hq + 2 * Hkv) * dim), 1, dtype)
    positions = torch.randint(0, 5000, (B, S) if B > 1 else (S,), generator=torch.Generator().manual_seed(2)).to(torch.int32)
    freq = frequencies(rot)
    wq, wk = (randn((dim,), 3, dtype), randn((dim,), 4, dtype)) if norm else (None, None)
    xd = x.to(cuda)
    q, k = xd[..., :Hq * dim].view(B, S, Hq, dim), xd[..., Hq * dim:(Hq + Hkv) * dim].view(B, S, Hkv, dim)
    q_out = torch.full((B, Hq, S, dim), float("nan"), dtype=dtype, device=cuda)
    k_out = torch.full((B, Hkv, S, dim), float("nan"), dtype=dtype, device=cuda)
    on = [None if w is None else w.to(cuda) for w in (wq, wk)]
    runtime.qk_norm_rope(q, k, positions.to(cuda), freq.to(cuda), q_out, k_out, *on, B=B, S=S, Hq=Hq, Hkv=Hkv, D=dim,
                         rot_dim=rot, interleaved=interleaved, eps=1e-6, dtype=NAMES[dtype])
    finish()
    flat = positions.expand(B, S).reshape(-1)
    for view, w, out, heads in ((q, wq, q_out, Hq), (k, wk, k_out, Hkv)):
        exact, size = paged.norm_rope(view.cpu().reshape(B * S, heads, dim), w, flat, freq, 1e-6, interleaved)
        close_to_rotation(out.transpose(1, 2).reshape(B * S, heads, dim), exact, size, dtype)


def test_rotation_at_far_and_negative_positions(cuda, native_lib):
    """An angle of 2^31 - 1 radians still has its fraction of a turn: in fp64 it is off by 2e-7 turns, which the bound
    gets as 1.5e-6 * (|y1| + |y2|) on top."""
    from neptune_mlir import runtime

    positions = torch.tensor([0, 1, -1, 65535, 1000003, -1000003, 2 ** 31 - 1, -2 ** 31], dtype=torch.int32)
    S = len(positions)
    q, k, freq = randn((1, S, 2, D), 1, torch.float32), randn((1, S, 1, D), 2, torch.float32), frequencies(D)
    q_out, k_out = torch.empty((1, 2, S, D), device=cuda), torch.empty((1, 1, S, D), device=cuda)
    runtime.qk_norm_rope(q.to(cuda), k.to(cuda), positions.to(cuda), freq.to(cuda), q_out, k_out, B=1, S=S, Hq=2, Hkv=1,
                         D=D, rot_dim=D, interleaved=False, eps=1e-6, dtype="f32")
    finish()
    for x, out in ((q, q_out), (k, k_out)):
        exact, size = paged.norm_rope(x[0], None, positions, freq, 1e-6, False)
        err = (out[0].transpose(0, 1).double().cpu() - exact).abs()
        assert bool((err <= U * exact.abs() + (32 * U + 1.5e-6) * size).all())
        near = err[:6] <= U * exact[:6].abs() + 32 * U * size[:6]
        assert bool(near.all())


def test_norm_and_rotation_in_place_on_a_side_stream(cuda, native_lib):
    """The outputs are the inputs' own elements, seen head-major; a zero row stays zero."""
    from neptune_mlir import runtime

    B, S, H = 2, 70, 6
    x = randn((B, S, 3 * H * D), 5, torch.bfloat16)
    x[1, 3] = 0
    freq, w = frequencies(D), randn((D,), 6, torch.bfloat16)
    side = torch.cuda.Stream(device=cuda)
    with torch.cuda.stream(side):
        xd = x.to(cuda)
        q, k = (xd[..., i * H * D:(i + 1) * H * D].view(B, S, H, D) for i in (0, 1))
        runtime.qk_norm_rope(q, k, torch.arange(S, dtype=torch.int32, device=cuda), freq.to(cuda), q.transpose(1, 2),
                             k.transpose(1, 2), w.to(cuda), None, B=B, S=S, Hq=H, Hkv=H, D=D, rot_dim=D,
                             interleaved=True, eps=1e-5, dtype="bf16")
    side.synchronize()
    finish()
    pos = torch.arange(S).repeat(B)
    for i, weight in ((0, w), (1, None)):
        exact, size = paged.norm_rope(x[..., i * H * D:(i + 1) * H * D].reshape(B * S, H, D), weight, pos, freq, 1e-5, True)
        close_to_rotation(xd[..., i * H * D:(i + 1) * H * D].reshape(B * S, H, D), exact, size, torch.bfloat16)
    assert torch.equal(xd[..., 2 * H * D:].cpu(), x[..., 2 * H * D:])


# ---- append ----------------------------------------------------------------------------------------------------------

def append(batch, x, Hq, cuda, freq, wq=None, wk=None, interleaved=False, with_q=True, **over):
    """One rope_append from a packed projection x [T, (Hq + 2 Hkv) D]; returns (q_out, k_pages, v_pages)."""
    from neptune_mlir import runtime

    xd = x.to(cuda)
    q, k, v = xd.split((Hq * D, batch.Hkv * D, batch.Hkv * D), -1)
    q, k, v = (t.unflatten(-1, (-1, D)) for t in (q, k, v))
    kp, vp = batch.k.to(cuda), batch.v.to(cuda)
    q_out = torch.full((x.shape[0], Hq, D), 7.0, dtype=batch.dtype, device=cuda) if with_q else None
    on = [None if w is None else w.to(cuda) for w in (wq, wk)]
    runtime.rope_append(q if with_q else None, k, v, kp, vp, *batch.device_args(cuda), freq.to(cuda), q_out, *on,
                        rot_dim=2 * freq.shape[0], interleaved=interleaved, eps=1e-6,
                        **{**batch.facts(Hq if with_q else 0), **over})
    return q_out, kp, vp


def check_append(batch, x, Hq, got, freq, wq=None, wk=None, interleaved=False, skipped=()):
    q_out, kp, vp = got
    q, k, v = (t.unflatten(-1, (-1, D)) for t in x.split((Hq * D, batch.Hkv * D, batch.Hkv * D), -1))
    where = [r for r in paged.positions_of(batch.cu, batch.lens) if r[0] not in skipped]
    rows = torch.tensor([t for t, _, _ in where], dtype=torch.long)
    pos = torch.tensor([p for _, _, p in where], dtype=torch.long)
    if q_out is not None:
        exact, size = paged.norm_rope(q[rows], wq, pos, freq, 1e-6, interleaved)
        close_to_rotation(q_out.cpu()[rows], exact, size, batch.dtype)
        rest = torch.ones(x.shape[0], dtype=torch.bool)
        rest[rows] = False
        assert bool((q_out.cpu()[rest].float() == 7.0).all()), "rows of no sequence were written"
    page = torch.stack([batch.table[b, p // PAGE] for _, b, p in where]).long() if where else rows
    exact, size = paged.norm_rope(k[rows], wk, pos, freq, 1e-6, interleaved)
    close_to_rotation(kp.cpu()[page, :, pos % PAGE], exact, size, batch.dtype)
    kept_k, kept_v = batch.k.clone(), batch.v.clone()
    kept_v[page, :, pos % PAGE] = v[rows]
    kept_k[page, :, pos % PAGE] = kp.cpu()[page, :, pos % PAGE]
    assert torch.equal(kp.cpu().view(torch.int16), kept_k.view(torch.int16)), "cache rows of no new token were written"
    assert torch.equal(vp.cpu().view(torch.int16), kept_v.view(torch.int16))


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16], ids=NAMES.get)
@pytest.mark.parametrize("Hq,Hkv,new,lens,rot,interleaved,norm", [
    (1, 1, [1], [1], 128, False, True), (32, 8, [1, 1, 0, 1], [1, 64, 9, 65], 128, False, True),
    (8, 2, [5, 0, 130, 64, 1], [5, 0, 200, 64, 129], 64, True, True), (15, 3, [63, 65], [63, 1000], 16, False, False),
    (64, 8, [700], [765], 128, True, False), (0, 4, [3, 70], [67, 70], 128, False, True),
])
def test_append(cuda, native_lib, dtype, Hq, Hkv, new, lens, rot, interleaved, norm):
    """Chunks that start and end inside pages, sequences that bring nothing, one token each, no queries."""
    batch = Batch(new, lens, Hkv, dtype)
    x = randn((batch.T, (Hq + 2 * Hkv) * D), 11, dtype)
    wq, wk = (randn((D,), 12, dtype), randn((D,), 13, dtype)) if norm else (None, None)
    freq = frequencies(rot)
    got = append(batch, x, Hq, cuda, freq, wq if Hq else None, wk, interleaved, with_q=Hq > 0)
    finish()
    check_append(batch, x, Hq, got, freq, wq, wk, interleaved)


def test_append_of_many_sequences(cuda, native_lib):
    """More sequences than a block has threads."""
    new = [i % 3 for i in range(700)]
    batch = Batch(new, [n + (7 * i) % 80 for i, n in enumerate(new)], 1, torch.bfloat16)
    x = randn((batch.T, 4 * D), 14, torch.bfloat16)
    got = append(batch, x, 2, cuda, frequencies(D))
    finish()
    check_append(batch, x, 2, got, frequencies(D))


def test_append_keeps_values_bit_for_bit(cuda, native_lib):
    """Values are copied as they are: NaNs with their payload, infinities, negative zero."""
    batch = Batch([4], [70], 1, torch.float16, pad=0)
    x = randn((4, 3 * D), 15, torch.float16)
    x[0, 2 * D:2 * D + 5] = torch.tensor([0x7e01, 0x7c00, -0x8000, 0x0001, 0x7fff], dtype=torch.int16).view(torch.float16)
    _, _, vp = append(batch, x, 1, cuda, frequencies(D))
    finish()
    row = vp.cpu()[batch.table[0, 1].long(), 0, 2]
    assert torch.equal(row.view(torch.int16), x[0, 2 * D:].view(torch.int16))


def test_append_refuses_rows_without_a_place(cuda, native_lib):
    """A page outside the pool, a position before the sequence's start or beyond its row of the table: nothing of that
    row is written, the status names it, the other rows are appended."""
    from neptune_mlir import runtime

    freq = frequencies(D)
    for what, new, lens, skipped, match in (
            ("table", [2, 3], [66, 10], (0, 1), "block table entry 999 is outside the page pool"),
            ("before", [2, 3], [66, 1], (2, 3), "row 2 is at position -2|row 3 is at position -1"),
            ("beyond", [2, 3], [66, 129], (4,), "row 4 is at position 128")):
        batch = Batch(new, lens, 2, torch.bfloat16, max_pages=2)
        if what == "table":
            batch.table[0, 1] = 999
        x = randn((batch.T, 8 * D), 16, torch.bfloat16)
        finish()
        got = append(batch, x, 4, cuda, freq)
        torch.cuda.synchronize()
        with pytest.raises(ValueError, match=match):
            runtime.check_status(cuda)
        check_append(batch, x, 4, got, freq, skipped=skipped)


# ---- chunk attention -------------------------------------------------------------------------------------------------

@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16], ids=NAMES.get)
@pytest.mark.parametrize("Hq,Hkv,new,lens", [
    (1, 1, [1], [1]), (4, 1, [1], [64]), (32, 8, [1], [65]), (8, 8, [130], [130]), (8, 2, [33], [1000]), (6, 2, [128], [128]),
    (10, 2, [26, 0, 1, 25], [300, 5, 129, 25]), (16, 2, [17, 16, 15], [127, 128, 129]), (128, 1, [3, 2], [70, 2]),
    (7, 1, [200, 1, 1, 1, 1], [257, 0, 1, 63, 700]), (24, 3, [64, 65], [64, 1065]), (100, 1, [2], [191]), (2, 1, [513], [700]),
])
def test_chunk_attention(cuda, native_lib, dtype, Hq, Hkv, new, lens):
    """Groups that do and do not divide 128, lengths around pages and blocks, chunks of one token, an empty cache, rows
    of the cache behind a sequence's end that hold NaN."""
    batch = Batch(new, lens, Hkv, dtype)
    q = randn((batch.T, Hq, D), 21, dtype)
    out = attend(batch, q.to(cuda), cuda)
    finish()
    check_attention(batch, q, out)


def test_chunk_attention_rows_that_see_nothing_are_zero(cuda, native_lib):
    """More new rows than the sequence is long: the first rows are at negative positions."""
    batch = Batch([40, 3, 2], [10, 0, 200], 2, torch.bfloat16)
    q = randn((batch.T, 8, D), 22, torch.bfloat16)
    out = attend(batch, q.to(cuda), cuda)
    finish()
    assert bool((out[:30] == 0).all()) and bool((out[40:43] == 0).all())
    check_attention(batch, q, out)


def test_chunk_attention_over_a_long_cache(cuda, native_lib):
    """Few rows over many: the rows of one tile are split over many blocks and joined."""
    batch = Batch([3, 1], [9000, 4500], 2, torch.bfloat16)
    q = randn((batch.T, 8, D), 23, torch.bfloat16)
    out = attend(batch, q.to(cuda), cuda)
    finish()
    check_attention(batch, q, out)


def test_chunk_attention_with_growing_scores(cuda, native_lib):
    """Scores that rise along the cache by far more than 2^8, and whole blocks far below the maximum: the running maximum
    moves often, and weights of early blocks vanish."""
    batch = Batch([40], [1500], 1, torch.float16)
    for p in range(batch.max_pages):
        rows = min(PAGE, 1500 - p * PAGE)
        batch.k[batch.table[0, p], :, :rows] = (batch.k[batch.table[0, p], :, :rows].float() * (0.2 + p)).half()
    q = randn((batch.T, 4, D), 24, torch.float16)
    out = attend(batch, q.to(cuda), cuda)
    finish()
    check_attention(batch, q, out)


def test_chunk_attention_of_many_sequences(cuda, native_lib):
    """More sequences than a block has threads, a quarter of them without new tokens."""
    new = [i % 4 for i in range(1100)]
    batch = Batch(new, [n + (13 * i) % 150 for i, n in enumerate(new)], 1, torch.bfloat16)
    q = randn((batch.T, 2, D), 25, torch.bfloat16)
    out = attend(batch, q.to(cuda), cuda)
    finish()
    check_attention(batch, q, out)


def test_chunk_attention_over_shared_pages(cuda, native_lib):
    """Sequences that begin with the same pages, and one that holds a page twice."""
    batch = Batch([5, 70, 1], [300, 250, 200], 2, torch.bfloat16)
    batch.table[1, :2] = batch.table[0, :2]
    batch.table[2, :2] = batch.table[0, 0]
    q = randn((batch.T, 6, D), 28, torch.bfloat16)
    out = attend(batch, q.to(cuda), cuda)
    finish()
    check_attention(batch, q, out)


def test_chunk_attention_with_strided_queries_and_output(cuda, native_lib):
    """Queries inside a packed projection, the output inside a wider buffer and head-major."""
    batch = Batch([50, 9], [90, 400], 2, torch.bfloat16)
    x = randn((batch.T, 12 * D), 26, torch.bfloat16)
    wide = torch.full((8, batch.T, 2 * D), 7.0, dtype=torch.bfloat16, device=cuda)
    out = attend(batch, x.to(cuda)[:, 2 * D:10 * D].unflatten(-1, (8, D)), cuda, out=wide.transpose(0, 1)[..., D:])
    finish()
    check_attention(batch, x[:, 2 * D:10 * D].unflatten(-1, (8, D)), out)
    assert bool((wide[..., :D] == 7.0).all())
    heads = x[:, 2 * D:10 * D].unflatten(-1, (8, D)).transpose(0, 1).contiguous().to(cuda)   # head-major queries
    out = attend(batch, heads.transpose(0, 1), cuda)
    finish()
    check_attention(batch, x[:, 2 * D:10 * D].unflatten(-1, (8, D)), out)


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16], ids=NAMES.get)
def test_chunk_attention_keeps_non_finite_rows_to_those_that_see_them(cuda, native_lib, dtype):
    """A value of one new token is infinite, another's is NaN, a key of a third is NaN: rows before them are as if they
    were not there, rows that see them are not finite in that column (value) or at all (key)."""
    new, lens = [150, 4], [700, 300]
    batch = Batch(new, lens, 2, dtype)
    q = randn((batch.T, 8, D), 31, dtype)

    def place(b, j):
        return batch.table[b, j // PAGE].long(), j % PAGE

    page, row = place(0, 550 + 37)
    batch.v[page, 0, row, 77] = float("inf")
    page, row = place(0, 550 + 90)
    batch.v[page, 1, row, 3] = float("nan")
    page, row = place(1, 298)
    batch.k[page, 1, row, 5] = float("nan")
    out = attend(batch, q.to(cuda), cuda).cpu()
    finish()
    hidden = [(0, 77, range(37)), (1, 3, range(90))]
    batch.k = batch.k.nan_to_num(0.0)
    batch.v = batch.v.nan_to_num(0.0, posinf=0.0)
    exact, spread, score = paged.attn_paged(q, batch.k, batch.v, batch.table, batch.cu, batch.lens, 1 / math.sqrt(D))
    for h, col, _ in hidden:
        seen = out[:150, 4 * h:4 * h + 4, col]
        assert bool(seen[(37, 90)[h]:].isfinite().logical_not().all()) and bool(seen[:(37, 90)[h]].isfinite().all())
        rows = slice((37, 90)[h], 150)
        out[rows, 4 * h:4 * h + 4, col] = exact[rows, 4 * h:4 * h + 4, col].to(dtype)
    assert bool(out[152:154, 4:].isnan().all())
    out[152:154, 4:] = exact[152:154, 4:].to(dtype)
    close_to_attention(out[:154], exact[:154], spread[:154], score, 700, 6.0, dtype)


def test_chunk_attention_refuses_a_table_entry_outside_the_pool(cuda, native_lib):
    from neptune_mlir import runtime

    batch = Batch([5, 20, 5], [500, 700, 129], 2, torch.bfloat16)
    q = randn((batch.T, 8, D), 27, torch.bfloat16)
    for entry in (batch.num_pages, -1):
        good = batch.table[1, 6].clone()
        batch.table[1, 6] = entry
        finish()
        out = attend(batch, q.to(cuda), cuda)
        torch.cuda.synchronize()
        with pytest.raises(ValueError, match=f"block table entry {entry} is outside the page pool"):
            runtime.check_status(cuda)
        batch.table[1, 6] = good
        assert bool(out[5:25].isnan().all())
        exact, spread, score = paged.attn_paged(q, batch.k, batch.v, batch.table, batch.cu, batch.lens, 1 / math.sqrt(D))
        for part in (slice(0, 5), slice(25, 30)):
            close_to_attention(out[part], exact[part], spread[part], score, 700, 6.0, torch.bfloat16)


def test_chunk_attention_cuts_a_length_to_the_table(cuda, native_lib):
    batch = Batch([4], [4 * PAGE + 2], 1, torch.bfloat16, max_pages=4)
    q = randn((batch.T, 4, D), 28, torch.bfloat16)
    out = attend(batch, q.to(cuda), cuda)
    finish()
    check_attention(batch, q, out)


def test_chunk_attention_with_offsets_beyond_31_bits(cuda, native_lib):
    """A pool of more than 2^31 elements, used at its end."""
    from neptune_mlir import runtime

    batch = Batch([3], [200], 8, torch.bfloat16)
    pages = 2 ** 31 // (8 * PAGE * D) + 8
    big_k = torch.zeros((pages, 8, PAGE, D), dtype=torch.bfloat16, device=cuda)
    big_v = torch.zeros_like(big_k)
    big_k[-batch.num_pages:], big_v[-batch.num_pages:] = batch.k.to(cuda), batch.v.to(cuda)
    table, cu, lens = batch.device_args(cuda)
    x = randn((batch.T, 24 * D), 29, torch.bfloat16).to(cuda)
    q, k, v = (t.unflatten(-1, (8, D)) for t in x.split(8 * D, -1))
    table += pages - batch.num_pages
    q_out = torch.empty_like(q)
    facts = batch.facts(8)
    runtime.rope_append(q, k, v, big_k, big_v, table, cu, lens, frequencies(D).to(cuda), q_out, rot_dim=D, interleaved=False,
                        eps=1e-6, **facts)
    out = torch.full(q.shape, 7.0, dtype=torch.bfloat16, device=cuda)
    runtime.attn_paged(q_out, big_k, big_v, table, cu, lens, scratch(cuda), out, scale_log2=LOG2E / math.sqrt(D), **facts)
    finish()
    batch.k, batch.v = big_k[-batch.num_pages:].cpu(), big_v[-batch.num_pages:].cpu()
    check_attention(batch, q_out.cpu(), out)


@pytest.mark.parametrize("dtype,Hq,Hkv,new,lens", [
    (torch.bfloat16, 40, 8, [(5 * i) % 8 for i in range(32)], [1 + (1237 * i) % 16001 for i in range(32)]),
    (torch.float16, 32, 8, [499] + [1] * 15, [4299] + [1 + (1811 * i) % 7600 for i in range(15)]),
    (torch.bfloat16, 16, 1, [300, 200, 5, 1], [6000, 200, 20000, 333]),
    (torch.bfloat16, 32, 8, [700], [17001]),                      # a cache beyond half the L2: tiles dealt out in waves
    (torch.float16, 16, 16, [1300], [9003]),
    (torch.bfloat16, 24, 8, [1536], [16512]),                     # tiles of 126 rows, no remainder behind the waves but one
], ids=["drafts", "mixed", "wide", "document", "heads", "thirds"])
def test_chunk_attention_streams_many_long_sequences(cuda, native_lib, dtype, Hq, Hkv, new, lens):
    """A cache larger than the L2: blocks arrive late and in bursts, while every CTA goes through parts of many tiles.
    The definition in 64 bits is evaluated on the device."""
    lens = [max(n, length) for n, length in zip(new, lens)]
    batch = Batch(new, lens, Hkv, dtype)
    q = randn((batch.T, Hq, D), 32, dtype).to(cuda)
    batch.k, batch.v, batch.table = batch.k.to(cuda), batch.v.to(cuda), batch.table.to(cuda)
    exact, spread, score = paged.attn_paged(q, batch.k, batch.v, batch.table, batch.cu, lens, 1 / math.sqrt(D))
    total, vmax = batch.cu[-1], batch.v.nan_to_num(0.0).abs().max().item()
    for _ in range(3):
        out = attend(batch, q, cuda)
        close_to_attention(out[:total], exact[:total].cpu(), spread[:total].cpu(), score, max(lens), vmax, dtype)
        assert bool((out[total:].float() == 7.0).all())
    finish()


def test_chunk_attention_is_the_same_twice(cuda, native_lib):
    batch = Batch([300, 1, 9], [4000, 2500, 9], 2, torch.bfloat16)
    q = randn((batch.T, 8, D), 30, torch.bfloat16).to(cuda)
    assert torch.equal(attend(batch, q, cuda), attend(batch, q, cuda))
    finish()


# ---- together --------------------------------------------------------------------------------------------------------

def test_a_layer_run_dense_and_paged(cuda, native_lib):
    """One attention layer over the same tokens twice: dense (norm and rotation, then causal attention), and served (a
    first chunk, a ragged second one beside another sequence, then single tokens by chunk attention and by split-K
    decode).  Both evaluate the same formula on the same rounded keys, so they differ by two attention bounds at most."""
    from neptune_mlir import runtime

    S, H, dtype = 333, 4, torch.bfloat16
    facts = dict(Hq=H, Hkv=H, D=D, dtype="bf16")
    x = randn((2, S, 3 * H * D), 41, dtype).to(cuda)
    freq, wq, wk = frequencies(D).to(cuda), randn((D,), 42, dtype).to(cuda), randn((D,), 43, dtype).to(cuda)
    q, k, v = (t.unflatten(-1, (H, D)) for t in x.split(H * D, -1))
    qr, kr, dense = (torch.empty((2, H, S, D), dtype=dtype, device=cuda) for _ in range(3))
    runtime.qk_norm_rope(q, k, torch.arange(S, dtype=torch.int32, device=cuda), freq, qr, kr, wq, wk, B=2, S=S, rot_dim=D,
                         interleaved=False, eps=1e-6, **facts)
    vh = v.transpose(1, 2).contiguous()
    runtime.attn_fwd(qr, kr, vh, dense, shape=(2, H, S, D), kv_len=S, dtype="bf16", scale_log2=LOG2E / math.sqrt(D), causal=True)

    max_pages = (S + PAGE - 1) // PAGE
    table = torch.randperm(2 * max_pages, generator=torch.Generator().manual_seed(1)).to(torch.int32).view(2, max_pages).to(cuda)
    kp = torch.full((2 * max_pages, H, PAGE, D), float("nan"), dtype=dtype, device=cuda)
    vp = kp.clone()
    work, served = scratch(cuda), torch.full((2, S, H, D), float("nan"), dtype=dtype, device=cuda)
    done = [0, 0]
    for step in ((200, 0), (100, 257), (1, 1), (32, 75)):
        rows = torch.cat([x[b, done[b]:done[b] + n] for b, n in enumerate(step)])
        T = rows.shape[0]
        qs, ks, vs = (t.unflatten(-1, (H, D)) for t in rows.split(H * D, -1))
        done = [d + n for d, n in zip(done, step)]
        cu = torch.tensor([0, step[0], T], dtype=torch.int32, device=cuda)
        lens = torch.tensor(done, dtype=torch.int32, device=cuda)
        q_out, out = torch.empty((T, H, D), dtype=dtype, device=cuda), torch.empty((T, H, D), dtype=dtype, device=cuda)
        more = dict(T=T, B=2, max_pages=max_pages, page_size=PAGE, **facts)
        runtime.rope_append(qs, ks, vs, kp, vp, table, cu, lens, freq, q_out, wq, wk, rot_dim=D, interleaved=False, eps=1e-6, **more)
        runtime.attn_paged(q_out, kp, vp, table, cu, lens, work, out, scale_log2=LOG2E / math.sqrt(D), **more)
        for b, part in ((0, out[:step[0]]), (1, out[step[0]:])):
            served[b, done[b] - step[b]:done[b]] = part
        if step == (1, 1):
            partials, single = torch.empty((2, H, 2, D + 2), device=cuda), torch.empty((2, H, D), dtype=dtype, device=cuda)
            runtime.decode_paged(q_out, kp, vp, table, lens, partials, single, B=2, max_pages=max_pages, page_size=PAGE,
                                 n_splits=2, scale_log2=LOG2E / math.sqrt(D), **facts)
            torch.testing.assert_close(single.float(), out.float(), rtol=2 ** -7, atol=2e-2)
    finish()
    assert done == [S, S]
    # the rotated queries and keys are the same bits
    for b in range(2):
        cached = kp[table[b].long()].transpose(1, 2).reshape(-1, H, D)[:S].transpose(0, 1)
        assert torch.equal(cached, kr[b])
    h = 2.0 ** -8
    weights = torch.softmax((qr.float() @ kr.float().transpose(-1, -2) / math.sqrt(D)).masked_fill(
        torch.ones(S, S, dtype=torch.bool, device=cuda).triu(1), float("-inf")), -1)
    spread = weights @ vh.float().abs()
    bound = 2 * (h * dense.float().abs() + (h + 512 * U * 12 + 2 * S * U) * spread)
    assert bool(((served.transpose(1, 2).float() - dense.float()).abs() <= bound).all())


def test_the_paged_step_through_emitted_modules_and_custom_ops(cuda, native_lib):
    """The declared operators and the torch.library ops make the same calls."""
    from neptune_mlir import programs, runtime, torch_ops  # noqa: F401

    batch = Batch([5, 70], [69, 70], 2, torch.bfloat16, pad=0)
    T, Hq = batch.T, 4
    x = randn((T, 8 * D), 51, torch.bfloat16).to(cuda)
    q, k, v = (t.unflatten(-1, (-1, D)).contiguous() for t in x.split((4 * D, 2 * D, 2 * D), -1))
    freq, wq, wk = frequencies(D).to(cuda), randn((D,), 52, torch.bfloat16).to(cuda), randn((D,), 53, torch.bfloat16).to(cuda)
    table, cu, lens = batch.device_args(cuda)
    sizes = dict(T=T, B=2, Hq=Hq, Hkv=2, num_pages=batch.num_pages, max_pages=batch.max_pages, D=D)
    text = programs.rope_append_decl("app", rot_dim=D, **sizes)
    mod = translate_text(text, "paged_append")
    att = translate_text(programs.attn_paged_decl("att", workspace_bytes=runtime.attn_paged_workspace_bytes(), **sizes), "paged_att")
    got = []
    for way in ("emitted", "op"):
        kp, vp, q_out, out = batch.k.to(cuda), batch.v.to(cuda), torch.empty_like(q), torch.empty_like(q)
        if way == "emitted":
            mod.app(q, k, v, kp, vp, table, cu, lens, freq, q_out, wq, wk)
            att.att(q_out, kp, vp, table, cu, lens, scratch(cuda).view(torch.int8), out)
        else:
            torch.ops.nb200.rope_append(q, k, v, kp, vp, table, cu, lens, freq, q_out, wq, wk, 1e-6, False)
            torch.ops.nb200.attn_paged(q_out, kp, vp, table, cu, lens, scratch(cuda), out, 1 / math.sqrt(D))
        got.append((q_out, kp.view(torch.int16), vp.view(torch.int16), out))
    finish()
    for a, b in zip(*got):
        torch.testing.assert_close(a.float(), b.float(), rtol=2 ** -7, atol=1e-6)   # the scale constant differs in its last bit
    rot = translate_text(programs.qk_norm_rope_decl("rot", 1, T, Hq, 2, D, D, norm=False), "paged_rot")
    outs = [torch.empty((1, h, T, D), dtype=torch.bfloat16, device=cuda) for h in (4, 2, 4, 2)]
    pos = torch.arange(T, dtype=torch.int32, device=cuda)
    rot.rot(q[None], k[None], pos[None], freq, *outs[:2])
    torch.ops.nb200.qk_norm_rope(q[None], k[None], pos, freq, *outs[2:], None, None, 1e-6, False)
    finish()
    assert torch.equal(outs[0], outs[2]) and torch.equal(outs[1], outs[3])


def test_the_paged_step_replays_from_two_cuda_graphs(cuda, native_lib):
    """Lengths, tables and chunk borders are read on the device: graphs captured for one step serve others.  Two graphs
    with a workspace each run at the same time on two streams."""
    from neptune_mlir import runtime

    new, lens = [9, 1, 30], [100, 700, 30]
    graphs = []
    for seed in (1, 2):
        batch = Batch(new, [3000, 3000, 3000], 2, torch.bfloat16, seed=seed)
        kp, vp = batch.k.to(cuda), batch.v.to(cuda)
        table, cu, lens_d = batch.device_args(cuda)
        lens_d.copy_(torch.tensor(lens))
        x = randn((batch.T, 12 * D), 60 + seed, torch.bfloat16).to(cuda)
        q, k, v = (t.unflatten(-1, (-1, D)) for t in x.split((8 * D, 2 * D, 2 * D), -1))
        q_out, out = torch.empty((batch.T, 8, D), dtype=torch.bfloat16, device=cuda), torch.full((batch.T, 8, D), 7.0, dtype=torch.bfloat16, device=cuda)
        freq, work = frequencies(D).to(cuda), scratch(cuda)

        def step():
            runtime.rope_append(q, k, v, kp, vp, table, cu, lens_d, freq, q_out, rot_dim=D, interleaved=False, eps=1e-6, **batch.facts(8))
            runtime.attn_paged(q_out, kp, vp, table, cu, lens_d, work, out, scale_log2=LOG2E / math.sqrt(D), **batch.facts(8))

        side = torch.cuda.Stream(device=cuda)
        side.wait_stream(torch.cuda.current_stream(cuda))
        with torch.cuda.stream(side):
            step()
        torch.cuda.current_stream(cuda).wait_stream(side)
        finish()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            step()
        graphs.append((batch, graph, kp, vp, cu, lens_d, q_out, out, (x, work, freq, table)))   # a graph keeps pointers, not tensors
    for new2, lens2 in (([9, 1, 30], [100, 700, 30]), ([0, 39, 1], [5, 2600, 129]), ([40, 0, 0], [40, 0, 0])):
        streams = [torch.cuda.Stream(device=cuda) for _ in graphs]
        for (batch, _, _, _, cu, lens_d, _, out, _) in graphs:
            batch.new, batch.lens = new2, lens2
            batch.cu = [0, new2[0], new2[0] + new2[1], sum(new2)]
            cu.copy_(torch.tensor(batch.cu))
            lens_d.copy_(torch.tensor(lens2))
            out.fill_(7.0)
        torch.cuda.synchronize()
        for entry, stream in zip(graphs, streams):
            with torch.cuda.stream(stream):
                entry[1].replay()
        finish()
        for (batch, _, kp, vp, _, _, q_out, out, _) in graphs:
            batch.k, batch.v = kp.cpu(), vp.cpu()
            check_attention(batch, q_out.cpu(), out)
