"""The per-device status words as the operators share them, on the GPU.  No test makes a kernel wait or fail."""

import ctypes

import pytest
import torch

from gpu_util import finish
from oracle import attention, inputs

pytestmark = pytest.mark.gpu


@pytest.fixture
def no_words_yet(cuda, native_lib, monkeypatch):
    """The state before any call on the device; afterwards the operators have the process's own words again."""
    from neptune_mlir import native, runtime

    finish()
    with monkeypatch.context() as m:
        m.setattr(runtime, "_status_buffers", {})
        m.setattr(runtime, "_captured_words", {})
        yield
        torch.cuda.synchronize()
    native.binding().set_status(cuda.index, runtime.status_buffer(cuda).data_ptr())


def test_the_first_call_on_a_busy_stream_leaves_clear_words_for_every_other(cuda, no_words_yet):
    """The words are made on a stream with work in front of them, in memory that held something else; another stream
    reads them at once."""
    from neptune_mlir import runtime

    busy, other = torch.cuda.Stream(device=cuda), torch.cuda.Stream(device=cuda)
    with torch.cuda.stream(busy):
        stale = torch.full((128,), 41, dtype=torch.int32, device=cuda)
        torch.cuda.synchronize()
        del stale                                             # the next small tensor on this stream is in its place
        torch.cuda._sleep(200_000_000)                        # some 0.1 s
        words = runtime.status_buffer(cuda)
    with torch.cuda.stream(other):
        seen = words.clone()
    torch.cuda.synchronize()
    assert seen.tolist() == [0, 0, 0, 0]


def test_attention_captured_before_any_other_call(cuda, no_words_yet):
    """A first call inside a graph capture cannot wait for its words to be cleared: the graph clears its own."""
    from neptune_mlir import runtime

    q, k, v = (t.to(cuda) for t in inputs.attention_inputs(1, 2, 256, 128, torch.bfloat16, config=2))
    out = torch.full_like(q, 7.0)

    def call():
        runtime.attn_fwd(q, k, v, out, shape=(1, 2, 256, 128), kv_len=256, dtype="bf16",
                         scale_log2=attention.scale_log2(128), causal=True)

    call()                                                    # the kernel itself is loaded
    torch.cuda.synchronize()
    before = dict(runtime._status_buffers)                    # the binding still has their address
    runtime._status_buffers.clear()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        call()
    assert runtime._status_buffers == {}
    out.fill_(7.0)
    graph.replay()
    runtime.check_status(cuda)
    ref = attention.attention_reference(q.cpu(), k.cpu(), v.cpu(), causal=True)
    assert (out.float().cpu() - ref).abs().max().item() <= 2e-2
    del graph, before


def _dense(cuda, status):
    """One causal attention call through the C ABI with these status words; returns (output, reference)."""
    from neptune_mlir import native

    q, k, v = (t.to(cuda) for t in inputs.attention_inputs(1, 2, 256, 128, torch.bfloat16, config=2))
    out = torch.full_like(q, 7.0)
    native.check(native.lib().nb200_attn_fwd(q.data_ptr(), k.data_ptr(), v.data_ptr(), out.data_ptr(), 1, 2, 256, 256, 128, 1,
                                             attention.scale_log2(128), 1, status.data_ptr(),
                                             torch.cuda.current_stream(cuda).cuda_stream), "attn_fwd")
    torch.cuda.synchronize()
    return out, attention.attention_reference(q.cpu(), k.cpu(), v.cpu(), causal=True)


def _paged(cuda, status):
    """One chunk-attention call of 70 tokens of one sequence; returns (output, reference)."""
    from neptune_mlir import native

    lib = native.lib()
    q, k, v = inputs.attention_inputs(1, 2, 128, 128, torch.bfloat16, config=3)
    pools = [x.view(2, 2, 64, 128).transpose(0, 1).contiguous().to(cuda) for x in (k, v)]
    rows = q[0, :, 58:].transpose(0, 1).contiguous().to(cuda)
    out = torch.full_like(rows, 7.0)
    table, cu, lens = (torch.tensor(x, dtype=torch.int32, device=cuda) for x in ([0, 1], [0, 70], [128]))
    work = torch.empty(lib.nb200_attn_paged_workspace_bytes(), dtype=torch.uint8, device=cuda)
    strides = (ctypes.c_longlong * 4)(256, 128, 256, 128)
    native.check(lib.nb200_attn_paged(rows.data_ptr(), pools[0].data_ptr(), pools[1].data_ptr(), table.data_ptr(), cu.data_ptr(),
                                      lens.data_ptr(), work.data_ptr(), out.data_ptr(), strides, 70, 1, 2, 2, 2, 2, 64, 128, 1,
                                      attention.scale_log2(128), status.data_ptr(),
                                      torch.cuda.current_stream(cuda).cuda_stream), "attn_paged")
    torch.cuda.synchronize()
    ref = attention.attention_reference(q, k, v, causal=True)[0, :, 58:].transpose(0, 1)
    return out, ref


@pytest.mark.parametrize("call", [_dense, _paged], ids=["dense", "paged"])
@pytest.mark.parametrize("record,computes", [([22, 3, 999, 0], True), ([23, 3, 4, 128], True), ([41, 3, 0, 0], False),
                                             ([3, 17, 5, 96], False), ([31, 0, 1, 1], False)])
def test_refused_data_stops_nobody_else_and_an_expired_wait_stops_every_attention(cuda, native_lib, call, record, computes):
    status = torch.tensor(record, dtype=torch.int32, device=cuda)
    out, ref = call(cuda, status)
    assert status.tolist() == record                          # whoever recorded it reads it
    if computes:
        assert (out.float().cpu() - ref).abs().max().item() <= 2e-2
    else:
        assert bool((out == 7.0).all())


def test_a_row_without_a_place_does_not_stop_the_dense_attention_of_others(cuda, native_lib):
    """An append row whose position its table does not reach, then a dense call of the same process."""
    from neptune_mlir import runtime

    finish()
    pool = torch.zeros((1, 1, 64, 128), dtype=torch.bfloat16, device=cuda)
    rows = torch.ones((1, 1, 128), dtype=torch.bfloat16, device=cuda)
    ints = [torch.tensor(x, dtype=torch.int32, device=cuda) for x in ([[0]], [0, 1], [65])]
    runtime.rope_append(None, rows, rows, pool, pool.clone(), *ints, torch.ones(64, device=cuda), None, T=1, B=1, Hq=0, Hkv=1,
                        max_pages=1, page_size=64, D=128, rot_dim=128, interleaved=False, eps=1e-6, dtype="bf16")
    q, k, v = (t.to(cuda) for t in inputs.attention_inputs(1, 2, 256, 128, torch.bfloat16, config=2))
    out = torch.full_like(q, 7.0)
    runtime.attn_fwd(q, k, v, out, shape=(1, 2, 256, 128), kv_len=256, dtype="bf16", scale_log2=attention.scale_log2(128),
                     causal=True)
    torch.cuda.synchronize()
    with pytest.raises(ValueError, match="row 0 is at position 64"):
        runtime.check_status(cuda)
    ref = attention.attention_reference(q.cpu(), k.cpu(), v.cpu(), causal=True)
    assert (out.float().cpu() - ref).abs().max().item() <= 2e-2


@pytest.mark.parametrize("found,left", [([22, 3, 999, 0], [31, 0, 1, 1]), ([23, 3, 4, 128], [31, 0, 1, 1]),
                                        ([3, 17, 5, 96], [3, 17, 5, 96]), ([0, 0, 0, 0], [31, 0, 1, 1])])
def test_an_expired_wait_takes_the_place_of_refused_data(cuda, native_lib, found, left):
    """The merge waits 20 ms for a rank that nobody plays.  Its record replaces one of refused data, which stops nobody,
    but not that of another wait."""
    from neptune_mlir import native

    lib = native.load(str(native_lib))
    rows = 4
    size = lib.nb200_decode_merge_peer_workspace_bytes(rows, 128, 2)
    bufs = [torch.zeros(size // 4, device=cuda) for _ in range(2)]
    status = torch.tensor(found, dtype=torch.int32, device=cuda)
    part, out = torch.ones((rows, 130), device=cuda), torch.full((rows, 128), 5.0, dtype=torch.bfloat16, device=cuda)
    peers = (ctypes.c_void_p * 2)(*[b.data_ptr() for b in bufs])
    native.check(lib.nb200_decode_merge_peer(part.data_ptr(), peers, out.data_ptr(), rows, 128, 2, 0, 1, 1, 20_000_000,
                                             status.data_ptr(), torch.cuda.current_stream(cuda).cuda_stream), "merge_peer")
    torch.cuda.synchronize()
    got = status.tolist()
    assert [got[0], *got[2:]] == [left[0], *left[2:]]          # the second word is the block that recorded it
    assert bool((out == 5.0).all())
