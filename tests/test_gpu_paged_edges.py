"""Chunk attention and append over the paged cache where rows, values and weights are at their limits.

Bounds are those of the module with the operators' tests: a rounding to the storage type is off by half a step.
"""

import math

import pytest
import torch

from gpu_util import finish
from oracle import paged
from test_gpu_paged import D, NAMES, PAGE, Batch, attend, close_to_attention, close_to_rotation, randn

pytestmark = pytest.mark.gpu

SCALE = 1 / math.sqrt(D)


def cache_row(batch, b, j):
    """Pool page and row of position j of sequence b."""
    return batch.table[b, j // PAGE].long(), j % PAGE


def definition(batch, q):
    """The 64-bit definition; its score bound without the keys that are not finite."""
    exact, spread, _ = paged.attn_paged(q, batch.k, batch.v, batch.table, batch.cu, batch.lens, SCALE)
    tame = batch.k.clone()
    tame[~tame.isfinite()] = 0
    _, _, score = paged.attn_paged(q, tame, batch.v, batch.table, batch.cu, batch.lens, SCALE)
    return exact, spread, score


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16], ids=NAMES.get)
@pytest.mark.parametrize("Hq,Hkv,new,lens", [(4, 1, [3, 2], [3, 40]), (8, 2, [130, 1], [130, 300]), (4, 2, [140], [200])])
def test_rows_whose_visible_scores_are_all_minus_infinity_are_nan(cuda, native_lib, dtype, Hq, Hkv, new, lens):
    """The first sequence's first keys score -inf with every query: the rows that see no others are NaN, as the softmax of
    such a row is and unlike rows that see nothing; the rows after them are as if those keys were not there."""
    batch = Batch(new, lens, Hkv, dtype)
    q = randn((batch.T, Hq, D), 61, dtype)
    q[..., 7] = 1.0
    blind = lens[0] - new[0] + 2                              # the first two new rows see such keys alone
    for j in range(blind):
        page, row = cache_row(batch, 0, j)
        batch.k[page, :, row, 7] = float("-inf")
    out = attend(batch, q.to(cuda), cuda)
    finish()
    out = out.cpu()
    exact, spread, score = definition(batch, q)
    assert bool(exact[:2].isnan().all()) and bool(exact[2:batch.cu[-1]].isfinite().all())
    assert bool(out[:2].isnan().all())
    part = slice(2, batch.cu[-1])
    close_to_attention(out[part], exact[part], spread[part], score, max(lens), 6.0, dtype)


def test_a_row_of_minus_infinities_over_a_long_cache_is_nan(cuda, native_lib):
    """The same where a row's blocks are split over many CTAs and joined: in one sequence every key, in another all but
    the keys of one page."""
    lens = [9000, 9000, 5000]
    batch = Batch([1, 1, 2], lens, 2, torch.bfloat16)
    q = randn((batch.T, 8, D), 62, torch.bfloat16)
    q[..., 7] = 1.0
    for b, kept in ((0, None), (1, 70)):
        for p in range((lens[b] + PAGE - 1) // PAGE):
            if p != kept:
                batch.k[batch.table[b, p], :, :min(PAGE, lens[b] - p * PAGE), 7] = float("-inf")
    out = attend(batch, q.to(cuda), cuda)
    finish()
    out = out.cpu()
    exact, spread, score = definition(batch, q)
    assert bool(exact[0].isnan().all()) and bool(out[0].isnan().all())
    close_to_attention(out[1:4], exact[1:4], spread[1:4], score, 9000, 6.0, torch.bfloat16)


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16], ids=NAMES.get)
@pytest.mark.parametrize("Hq,Hkv,new,lens", [(8, 2, [150, 4], [700, 300]), (4, 2, [6, 1], [9000, 50]), (24, 3, [16, 16], [131, 700])])
def test_values_that_are_not_finite_are_added_wherever_they_stand(cuda, native_lib, dtype, Hq, Hkv, new, lens):
    """Infinities of either sign and NaN, in blocks that every row of a tile sees and in those that only some do: a row
    that sees them gets their sum, a row that does not is as if they were not there."""
    batch = Batch(new, lens, Hkv, dtype)
    q = randn((batch.T, Hq, D), 63, dtype)
    start = lens[0] - new[0]
    inf, nan, late = float("inf"), float("nan"), start + new[0] // 2
    placed = [(0, 5, inf), (late, 6, inf), (late, 7, -inf), (1, 8, -inf), (late, 8, -inf), (1, 9, inf), (late, 9, -inf),
              (late, 10, nan), (0, 11, nan), (late, 12, -inf), (lens[0] - 1, 12, inf), (lens[0] - 1, 127, -inf)]
    exact_values = batch.v.clone()
    for j, col, value in placed:
        page, row = cache_row(batch, 0, j)
        batch.v[page, 1, row, col] = value
        exact_values[page, 1, row, col] = 0
    out = attend(batch, q.to(cuda), cuda)
    finish()
    out, total = out.cpu(), batch.cu[-1]
    exact, spread, score = paged.attn_paged(q, batch.k, exact_values, batch.table, batch.cu, batch.lens, SCALE)
    group = Hq // Hkv
    added = torch.zeros(exact.shape)
    for j, col, value in placed:
        added[max(0, j - start):new[0], group:2 * group, col] += value
    seen = added[:total] != 0
    assert int(seen.sum()) > 0
    want = added[:total][seen]
    assert torch.equal(out[:total][seen].float().nan_to_num(nan=1.0, posinf=2.0, neginf=3.0), want.nan_to_num(nan=1.0, posinf=2.0, neginf=3.0))
    out = torch.where(added != 0, exact.to(dtype), out)
    close_to_attention(out[:total], exact[:total], spread[:total], score, max(lens), 6.0, dtype)


def test_odd_strides_of_extents_of_one(cuda, native_lib):
    """A batch of one and a step of one token, cut out of tensors whose other rows begin anywhere."""
    from neptune_mlir import runtime

    S, H, dtype = 9, 3, torch.bfloat16
    freq = (10000.0 ** (-torch.arange(0, D, 2, dtype=torch.float32) / D)).to(cuda)
    x = randn((1, S, H, D), 71, dtype)
    at = torch.arange(5, 5 + S, dtype=torch.int32)

    def cut(t):                                               # the same elements, the stride of extent 1 odd
        return t.contiguous().as_strided(t.shape, [7 if n == 1 else s for n, s in zip(t.shape, t.contiguous().stride())])

    xd = cut(x.to(cuda))
    q_out, k_out = (cut(torch.full((1, H, S, D), 7.0, dtype=dtype, device=cuda)) for _ in range(2))
    runtime.qk_norm_rope(xd, xd, at.to(cuda), freq, q_out, k_out, B=1, S=S, Hq=H, Hkv=H, D=D, rot_dim=D, interleaved=False,
                         eps=1e-6, dtype="bf16")
    batch = Batch([1], [70], H, dtype, pad=0)
    kp, vp = batch.k.to(cuda), batch.v.to(cuda)
    one, one_out = cut(x[0, :1].to(cuda)), cut(torch.full((1, H, D), 7.0, dtype=dtype, device=cuda))
    runtime.rope_append(one, one, one, kp, vp, *batch.device_args(cuda), freq, one_out, rot_dim=D, interleaved=False, eps=1e-6,
                        **batch.facts(H))
    finish()
    exact, size = paged.norm_rope(x[0], None, at, freq.cpu(), 1e-6, False)
    for out in (q_out, k_out):
        close_to_rotation(out[0].transpose(0, 1), exact, size, dtype)
    exact, size = paged.norm_rope(x[0, :1], None, torch.tensor([69]), freq.cpu(), 1e-6, False)
    page, row = cache_row(batch, 0, 69)
    close_to_rotation(one_out, exact, size, dtype)
    close_to_rotation(kp.cpu()[page, :, row][None], exact, size, dtype)
    assert torch.equal(vp.cpu()[page, :, row], x[0, 0])


def test_a_tile_that_takes_longer_than_a_wait_lasts(cuda, native_lib):
    """2^29 cached rows of one sequence, its pages all the same one, a kv head to every SM: each tile takes some seconds,
    more than the two of a bounded wait.  Every score is 0 and one value row in 64 is 1, so that sums are whole numbers
    below 2^24 (values) and multiples of 128 below 2^31 (weights): the output is 1/64 exactly."""
    from neptune_mlir import runtime

    heads = torch.cuda.get_device_properties(cuda).multi_processor_count
    rows = 2 ** 29
    k = torch.zeros((1, heads, PAGE, D), dtype=torch.bfloat16, device=cuda)
    v = torch.zeros_like(k)
    v[:, :, 5] = 1.0
    table = torch.zeros((1, rows // PAGE), dtype=torch.int32, device=cuda)
    cu, lens = (torch.tensor(x, dtype=torch.int32, device=cuda) for x in ([0, 1], [rows]))
    q = torch.zeros((1, heads, D), dtype=torch.bfloat16, device=cuda)
    out = torch.full_like(q, 7.0)
    work = torch.empty(runtime.attn_paged_workspace_bytes(), dtype=torch.uint8, device=cuda)
    finish()
    runtime.attn_paged(q, k, v, table, cu, lens, work, out, T=1, B=1, Hq=heads, Hkv=heads, max_pages=rows // PAGE, page_size=PAGE,
                       D=D, dtype="bf16", scale_log2=SCALE * math.log2(math.e))
    finish()
    assert bool((out == 1 / 64).all())


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16], ids=NAMES.get)
def test_many_small_weights_beside_a_large_one(cuda, native_lib, dtype):
    """One key of weight 1 whose value is 0 and 2^16 - 1 keys of weight 2^-26 whose value is 1: a thousandth, all
    of it from weights that are below half of fp16's least.  The rows of a head are not split (a kv head to every SM).
    Weights of fp16 are held times 2^7, so that one is off by 2^-25 / 2^7 at most."""
    from neptune_mlir import runtime

    heads = torch.cuda.get_device_properties(cuda).multi_processor_count
    rows = 2 ** 16
    k = torch.zeros((2, heads, PAGE, D), dtype=dtype)
    v = torch.ones_like(k)
    k[0, :, 3, 0] = 26 / (16 * SCALE * math.log2(math.e))     # rounded to the type, as the definition takes it
    v[0, :, 3] = 0
    table = torch.ones((1, rows // PAGE), dtype=torch.int32)
    table[0, 100] = 0
    q = torch.zeros((1, heads, D), dtype=dtype)
    q[..., 0] = 16
    out = torch.full_like(q, 7.0).to(cuda)
    work = torch.empty(runtime.attn_paged_workspace_bytes(), dtype=torch.uint8, device=cuda)
    cu, lens = (torch.tensor(x, dtype=torch.int32, device=cuda) for x in ([0, 1], [rows]))
    runtime.attn_paged(q.to(cuda), k.to(cuda), v.to(cuda), table.to(cuda), cu, lens, work, out, T=1, B=1, Hq=heads, Hkv=heads,
                       max_pages=rows // PAGE, page_size=PAGE, D=D, dtype=NAMES[dtype], scale_log2=SCALE * math.log2(math.e))
    finish()
    exact, spread, score = paged.attn_paged(q[:, :1], k[:, :1], v[:, :1], table, [0, 1], [rows], SCALE)
    assert 7e-4 < exact[0, 0, 0].item() < 1.3e-3
    h, u = torch.finfo(dtype).eps / 2, 2.0 ** -24
    bound = h * exact.abs() + (h + 512 * u * score + 2 * rows * u) * spread + rows * 2.0 ** -32 * (dtype == torch.float16)
    assert bool(((out.double().cpu() - exact).abs() <= bound).all()), (out[0, 0, 0].item(), exact[0, 0, 0].item(), bound.max().item())


@pytest.mark.parametrize("B,prompt,cached,dtype", [(17, 5000, 300, torch.bfloat16), (40, 3001, 0, torch.float16),
                                                   (300, 4096, 1000, torch.bfloat16), (512, 2500, 129, torch.float16)])
def test_a_long_prompt_among_many_sequences(cuda, native_lib, B, prompt, cached, dtype):
    """More sequences than a block has warps, one of them with a prompt of several thousand tokens: its place among the
    others varies."""
    at = (7 * B) % B if B % 2 else B // 2
    new = [prompt if b == at else b % 2 for b in range(B)]
    lens = [prompt + cached if b == at else new[b] + (37 * b) % 400 for b in range(B)]
    batch = Batch(new, lens, 2, dtype)
    q = randn((batch.T, 8, D), 64, dtype).to(cuda)
    batch.k, batch.v, batch.table = batch.k.to(cuda), batch.v.to(cuda), batch.table.to(cuda)
    exact, spread, score = paged.attn_paged(q, batch.k, batch.v, batch.table, batch.cu, lens, SCALE)
    out = attend(batch, q, cuda)
    finish()
    total = batch.cu[-1]
    close_to_attention(out[:total], exact[:total].cpu(), spread[:total].cpu(), score, max(lens), 6.0, dtype)
    assert bool((out[total:].float() == 7.0).all())


def test_a_batch_in_which_no_sequence_brings_anything(cuda, native_lib):
    """A padded step whose ranges are all empty, by attention and by append: nothing is written."""
    from neptune_mlir import runtime

    batch = Batch([0, 0, 0], [5, 0, 200], 2, torch.bfloat16, pad=4)
    q = randn((4, 8, D), 65, torch.bfloat16).to(cuda)
    kv = randn((4, 2, D), 66, torch.bfloat16).to(cuda)
    out = attend(batch, q, cuda)
    kp, vp, q_out = batch.k.to(cuda), batch.v.to(cuda), torch.full_like(q, 7.0)
    runtime.rope_append(q, kv, kv, kp, vp, *batch.device_args(cuda), torch.ones(64, device=cuda), q_out, rot_dim=D,
                        interleaved=False, eps=1e-6, **batch.facts(8))
    finish()
    assert bool((out == 7.0).all()) and bool((q_out == 7.0).all())
    assert torch.equal(kp.cpu().view(torch.int16), batch.k.view(torch.int16))
    assert torch.equal(vp.cpu().view(torch.int16), batch.v.view(torch.int16))


def test_rows_in_front_of_the_first_sequence_are_left_alone(cuda, native_lib):
    """cu_seqlens that begins behind row 0, by attention and by append."""
    from neptune_mlir import runtime

    front = 5
    batch = Batch([33, 1], [90, 300], 2, torch.bfloat16)
    q = randn((batch.T, 8, D), 67, torch.bfloat16)
    kv = randn((front + batch.T, 2, D), 68, torch.bfloat16).to(cuda)
    wide = torch.cat([torch.full((front, 8, D), float("nan"), dtype=q.dtype), q]).to(cuda)
    table, cu, lens = batch.device_args(cuda)
    out, q_out = torch.full_like(wide, 7.0), torch.full_like(wide, 7.0)
    facts = {**batch.facts(8), "T": front + batch.T}
    work = torch.empty(runtime.attn_paged_workspace_bytes(), dtype=torch.uint8, device=cuda)
    runtime.attn_paged(wide, batch.k.to(cuda), batch.v.to(cuda), table, cu + front, lens, work, out,
                       scale_log2=SCALE * math.log2(math.e), **facts)
    freq = 10000.0 ** (-torch.arange(0, D, 2, dtype=torch.float32) / D)
    kp, vp = batch.k.to(cuda), batch.v.to(cuda)
    runtime.rope_append(wide, kv, kv, kp, vp, table, cu + front, lens, freq.to(cuda), q_out, rot_dim=D, interleaved=False,
                        eps=1e-6, **facts)
    finish()
    assert bool((out[:front] == 7.0).all()) and bool((q_out[:front] == 7.0).all())
    exact, spread, score = paged.attn_paged(q, batch.k, batch.v, batch.table, batch.cu, batch.lens, SCALE)
    total = batch.cu[-1]
    close_to_attention(out[front:front + total], exact[:total], spread[:total], score, 300, 6.0, torch.bfloat16)
    where = paged.positions_of(batch.cu, batch.lens)
    exact, size = paged.norm_rope(q[:total], None, torch.tensor([p for _, _, p in where]), freq, 1e-6, False)
    close_to_rotation(q_out[front:front + total], exact, size, torch.bfloat16)
    for t, b, p in where:
        page, row = cache_row(batch, b, p)
        assert torch.equal(vp[page, :, row], kv[front + t])


def test_append_without_queries_through_the_custom_op(cuda, native_lib):
    """q and q_out absent: keys and values alone, the same bits as beside queries."""
    from neptune_mlir import torch_ops  # noqa: F401

    batch = Batch([5, 70], [69, 70], 2, torch.bfloat16, pad=0)
    q, k, v = (randn((batch.T, h, D), 69 + i, torch.bfloat16).to(cuda) for i, h in enumerate((4, 2, 2)))
    freq = torch.linspace(0.1, 1.0, 64).to(cuda)
    got = []
    for queries in (q, None):
        kp, vp = batch.k.to(cuda), batch.v.to(cuda)
        q_out = None if queries is None else torch.empty_like(q)
        torch.ops.nb200.rope_append(queries, k, v, kp, vp, *batch.device_args(cuda), freq, q_out, None, None, 1e-6, False)
        got.append((kp.view(torch.int16), vp.view(torch.int16)))
    finish()
    assert torch.equal(got[0][0], got[1][0]) and torch.equal(got[0][1], got[1][1])
    assert not torch.equal(got[0][0].cpu(), batch.k.view(torch.int16))


def test_two_threads_attend_at_the_same_time(cuda, native_lib):
    """A stream, a workspace and a batch each: neither waits for the other, neither reads the other's parts."""
    import threading

    from neptune_mlir import runtime

    jobs = []
    for seed, (new, lens) in enumerate((([3, 40], [5000, 300]), ([200], [2500]))):
        batch = Batch(new, lens, 2, torch.bfloat16, seed=seed)
        q = randn((batch.T, 8, D), 80 + seed, torch.bfloat16)
        want = attend(batch, q.to(cuda), cuda)
        on = (q.to(cuda), batch.k.to(cuda), batch.v.to(cuda), *batch.device_args(cuda))
        outs = [torch.full((batch.T, 8, D), 7.0, dtype=torch.bfloat16, device=cuda) for _ in range(20)]
        jobs.append((batch, on, torch.empty(runtime.attn_paged_workspace_bytes(), dtype=torch.uint8, device=cuda), outs, want))
    torch.cuda.synchronize()
    together, failed = threading.Barrier(2), []

    def work(batch, on, scratch, outs, want):
        try:
            with torch.cuda.stream(torch.cuda.Stream(device=cuda)):
                together.wait()
                for out in outs:
                    runtime.attn_paged(*on, scratch, out, scale_log2=SCALE * math.log2(math.e), **batch.facts(8))
                torch.cuda.current_stream().synchronize()
        except Exception as exc:
            failed.append(exc)

    threads = [threading.Thread(target=work, args=job) for job in jobs]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    finish()
    assert not failed
    for _, _, _, outs, want in jobs:
        for out in outs:
            assert torch.equal(out, want)
