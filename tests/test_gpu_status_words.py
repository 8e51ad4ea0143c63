"""The per-device status words as the operators share them, on the GPU.  No test makes a kernel wait or fail."""

import math

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
