"""The per-device status words without a GPU: host memory stands in for the device's, a fake for the native binding."""

import contextlib
import threading
import time

import pytest
import torch

from neptune_mlir import native, runtime

DEVICE = torch.device("cuda", 0)


class FakeBinding:
    """Keeps the address that was published last, as the native binding does."""

    def __init__(self, delays=()):
        self.delays, self.published = list(delays), {}

    def set_status(self, device, address):
        time.sleep(self.delays.pop(0) if self.delays else 0.0)
        self.published[device] = address


@pytest.fixture
def words(monkeypatch):
    """Host tensors in the place of device ones, no capture running; returns a function that starts over."""
    host_zeros = torch.zeros
    waited = []

    class Stream:
        def synchronize(self):
            waited.append(dict(runtime._status_buffers))      # what could be seen before the words were clear

    def start(make_delays=(), publish_delays=()):
        delays, binding = list(make_delays), FakeBinding(publish_delays)
        binding.waited = waited

        def zeros(*args, device=None, **kwargs):
            time.sleep(delays.pop(0) if delays else 0.0)
            return host_zeros(*args, **kwargs)

        monkeypatch.setattr(torch, "zeros", zeros)
        monkeypatch.setattr(native, "binding", lambda: binding)
        monkeypatch.setattr(runtime, "_status_buffers", {})
        monkeypatch.setattr(runtime, "_captured_words", {}, raising=False)
        waited.clear()
        return binding

    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: False)
    monkeypatch.setattr(torch.cuda, "current_stream", lambda device=None: Stream())
    monkeypatch.setattr(torch.cuda, "device", lambda device: contextlib.nullcontext())
    return start


@pytest.mark.parametrize("make,publish", [((0.05, 0.15), (0.25, 0.0)), ((0.0, 0.0), (0.1, 0.0)), ((0.0,) * 2, (0.0,) * 2)])
def test_first_calls_of_two_threads_publish_the_words_that_stay(words, make, publish):
    """Whichever thread is first at each step, the binding ends with the address of the tensor that is kept."""
    binding = words(make, publish)
    together, got = threading.Barrier(2), []

    def first_call():
        together.wait()
        runtime._first_status_buffer(DEVICE)
        got.append(runtime.status_buffer(DEVICE).data_ptr())

    threads = [threading.Thread(target=first_call) for _ in range(2)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    kept = runtime._status_buffers[0].data_ptr()
    assert got == [kept, kept]
    assert binding.published == {0: kept}


def test_the_words_are_clear_before_other_streams_can_use_them(words):
    """The fill is asynchronous: its stream is waited for once, before anything of the words can be seen."""
    binding = words()
    runtime._first_status_buffer(DEVICE)
    runtime.status_buffer(DEVICE)
    assert binding.waited == [{}] and 0 in runtime._status_buffers


def test_words_made_inside_a_capture_are_for_that_graph_alone(words, monkeypatch):
    """Their fill is part of the graph, so no call outside it may take them for clear."""
    binding = words()
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: True)
    captured = runtime.status_buffer(DEVICE)
    assert binding.waited == [] and binding.published == {} and runtime._status_buffers == {}
    with pytest.raises(RuntimeError, match="before capturing"):
        runtime._first_status_buffer(DEVICE)
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: False)
    runtime._first_status_buffer(DEVICE)
    kept = runtime.status_buffer(DEVICE)
    assert kept.data_ptr() != captured.data_ptr() and binding.published == {0: kept.data_ptr()}
    assert [w.data_ptr() for w in runtime._captured_words[0]] == [captured.data_ptr()]   # as long as the graph may run


def test_operators_outside_the_binding_do_not_need_it(words, monkeypatch):
    """Dense attention, decode, the peer merge and check_status take the words' address themselves."""
    words()

    def missing():
        raise native.NativeLibraryError("the torch binding (nb200_torch.so) was not found")

    monkeypatch.setattr(native, "binding", missing)
    for _ in range(2):
        assert runtime.status_buffer(DEVICE).tolist() == [0, 0, 0, 0]
    with pytest.raises(native.NativeLibraryError, match="torch binding"):
        runtime._first_status_buffer(DEVICE)


def test_the_binding_hears_of_words_that_an_earlier_operator_made(words):
    binding = words()
    kept = runtime.status_buffer(DEVICE)
    assert binding.published == {}
    runtime._first_status_buffer(DEVICE)
    assert binding.published == {0: kept.data_ptr()} and runtime.status_buffer(DEVICE) is kept


def test_the_binding_is_found_beside_the_library_that_was_loaded(native_lib, tmp_path, monkeypatch):
    """A library that the environment names, and its binding, can be anywhere."""
    from neptune_mlir import plugin

    monkeypatch.setattr(plugin, "_candidate_dirs", lambda: [tmp_path / "elsewhere"])
    library = tmp_path / "libnb200.so"
    library.write_bytes(b"")
    monkeypatch.setenv(plugin.DEFAULT_LIBRARY_ENV, str(library))
    assert plugin.find_library_path() == library.resolve()
    assert plugin.find_binding_path(plugin.find_library_path()) is None
    beside = tmp_path / "nb200_torch.so"
    beside.write_bytes(b"")
    assert plugin.find_binding_path(plugin.find_library_path()) == beside.resolve()
    assert plugin.find_binding_path() is None
