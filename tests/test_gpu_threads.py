"""Calls from threads that have not used the GPU before."""

import math
import threading

import pytest
import torch

from gpu_util import finish
from oracle import attention, inputs

pytestmark = pytest.mark.gpu


def in_a_new_thread(call):
    """Run it as a thread's first use of the GPU; hand on what it raises."""
    failed = []

    def work():
        try:
            call()
        except Exception as exc:
            failed.append(exc)

    thread = threading.Thread(target=work)
    thread.start()
    thread.join()
    if failed:
        raise failed[0]


def test_dense_attention_as_a_threads_first_call(cuda, native_lib):
    from neptune_mlir import runtime

    q, k, v = (t.to(cuda) for t in inputs.attention_inputs(1, 2, 256, 128, torch.bfloat16, config=2))
    out = torch.full_like(q, 7.0)
    runtime.check_status(cuda)
    torch.cuda.synchronize()
    in_a_new_thread(lambda: runtime.attn_fwd(q, k, v, out, shape=(1, 2, 256, 128), kv_len=256, dtype="bf16",
                                             scale_log2=attention.scale_log2(128), causal=True))
    finish()
    ref = attention.attention_reference(q.cpu(), k.cpu(), v.cpu(), causal=True)
    assert (out.float().cpu() - ref).abs().max().item() <= 2e-2


def test_a_paged_step_as_a_threads_first_calls(cuda, native_lib):
    """Norm and rotation, append, and attention, each in a thread of its own; the same bits as in this one."""
    from neptune_mlir import runtime

    T, H, D = 70, 4, 128
    gen = torch.Generator().manual_seed(5)
    x = torch.randn((T, H, D), generator=gen).bfloat16().to(cuda)
    freq = torch.linspace(0.01, 1.0, 64).to(cuda)
    table, cu, lens = (torch.tensor(t, dtype=torch.int32, device=cuda) for t in ([[1, 0]], [0, T], [T]))
    at = torch.arange(T, dtype=torch.int32, device=cuda)
    facts = dict(Hq=H, Hkv=H, D=D, dtype="bf16")
    paged = dict(T=T, B=1, max_pages=2, page_size=64, **facts)
    got = []
    for how in (lambda call: call(), in_a_new_thread):
        kp, vp = (torch.zeros((2, H, 64, D), dtype=torch.bfloat16, device=cuda) for _ in range(2))
        q_out, out, dense_q, dense_k = (torch.full(s, 7.0, dtype=torch.bfloat16, device=cuda)
                                        for s in ((T, H, D), (T, H, D), (1, H, T, D), (1, H, T, D)))
        work = torch.empty(runtime.attn_paged_workspace_bytes(), dtype=torch.uint8, device=cuda)
        torch.cuda.synchronize()
        how(lambda: runtime.qk_norm_rope(x[None], x[None], at, freq, dense_q, dense_k, B=1, S=T, rot_dim=D, interleaved=False,
                                         eps=1e-6, **facts))
        how(lambda: runtime.rope_append(x, x, x, kp, vp, table, cu, lens, freq, q_out, rot_dim=D, interleaved=False, eps=1e-6,
                                        **paged))
        how(lambda: runtime.attn_paged(q_out, kp, vp, table, cu, lens, work, out, scale_log2=math.log2(math.e) / math.sqrt(D),
                                       **paged))
        finish()
        got.append((dense_q, dense_k, kp, vp, q_out, out))
    for a, b in zip(*got):
        assert torch.equal(a, b) and not bool((b == 7.0).all())


def test_ssd_as_a_threads_first_call(cuda, native_lib):
    from neptune_mlir import runtime
    from oracle import ssd

    B, L, H, P, N, G, chunk = 1, 256, 4, 64, 128, 1, 128
    args = inputs.ssd_inputs(B=B, L=L, H=H, P=P, N=N, G=G)
    on = [a.to(cuda) for a in args]
    ws = torch.zeros(max(16, runtime.ssd_workspace_bytes(B, L, H, P, N, G, chunk)), dtype=torch.uint8, device=cuda)
    y = torch.full((B, L, H, P), float("nan"), dtype=torch.bfloat16, device=cuda)
    torch.cuda.synchronize()
    in_a_new_thread(lambda: runtime.ssd_chunk_scan(*on, ws, y, B=B, L=L, H=H, P=P, N=N, G=G, chunk=chunk, dtype="bf16"))
    torch.cuda.synchronize()
    runtime.check_workspace_status(ws)
    ref = ssd.ssd_reference(*args)
    assert (y.float().cpu() - ref).pow(2).mean().sqrt().item() <= 2.0 ** -8 * ref.pow(2).mean().sqrt().item()
