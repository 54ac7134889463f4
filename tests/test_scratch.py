"""The operators' default device scratch: who may share a buffer and who may not."""
import threading

import pytest
import torch

CPU = torch.device("cpu", 0)  # the bookkeeping is the same on any device


@pytest.fixture
def capturing(monkeypatch):
    """A switch for "the current stream is being captured"; device 0 is current."""
    state = {"on": False}
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: state["on"])
    monkeypatch.setattr(torch.cuda, "current_device", lambda: 0)
    return state


def test_calls_on_one_stream_share_a_buffer(capturing):
    from nsn_b200 import _lib as L
    a = L.scratch(1 << 10, CPU, 901)
    assert L.scratch(1 << 12, CPU, 901).data_ptr() == a.data_ptr()
    assert L.scratch(1 << 12, CPU, 902).data_ptr() != a.data_ptr()
    b = L.scratch(1 << 21, CPU, 901)
    assert b.numel() >= 1 << 21 and L.scratch(16, CPU, 901).data_ptr() == b.data_ptr()


def test_a_captured_call_never_gets_an_eager_buffer(capturing):
    """A graph keeps the addresses it was captured with, so its buffer must be its own: an eager
    buffer is replaced (and freed) when it grows, and is written by eager calls during a replay."""
    from nsn_b200 import _lib as L
    eager = L.scratch(1 << 10, CPU, 903)
    capturing["on"] = True
    graph = L.scratch(1 << 10, CPU, 903)
    assert graph.data_ptr() != eager.data_ptr()
    capturing["on"] = False
    assert L.scratch(1 << 10, CPU, 903).data_ptr() == eager.data_ptr()


def test_host_threads_on_one_stream_do_not_share(capturing):
    """An operator enqueues two kernels; another thread's may come between them."""
    from nsn_b200 import _lib as L
    mine, other = L.scratch(1 << 10, CPU, 904), []
    t = threading.Thread(target=lambda: other.append(L.scratch(1 << 10, CPU, 904)))
    t.start()
    t.join()
    assert other[0].data_ptr() != mine.data_ptr()


def test_decode_attention_in_a_graph(capturing, monkeypatch):
    """The decode kernels' default workspace keeps the same rules."""
    from types import SimpleNamespace
    from nsn_b200 import kernel
    monkeypatch.setattr(torch.cuda, "current_stream", lambda device=None: SimpleNamespace(cuda_stream=905))
    eager = kernel.workspace(1 << 10, CPU)
    assert kernel.workspace(1 << 9, CPU).data_ptr() == eager.data_ptr()
    capturing["on"] = True
    assert kernel.workspace(1 << 10, CPU).data_ptr() != eager.data_ptr()


def test_a_status_word_is_where_the_kernel_can_write_it():
    """An address of another device's memory is refused on the host, not met by the kernel."""
    from nsn_b200 import ContractError
    from nsn_b200.primitives import status_ptr
    ok = torch.zeros(1, dtype=torch.int32)
    assert status_ptr(None, ok.device) is None and status_ptr(ok, ok.device) == ok.data_ptr()
    for bad in (ok.to(torch.int64), ok.float(), ok[:0]):
        with pytest.raises(ContractError):
            status_ptr(bad, ok.device)
    with pytest.raises(ContractError):
        status_ptr(ok, torch.device("cuda", 0))


def test_a_workspace_is_where_the_kernel_can_write_it():
    from nsn_b200 import ContractError
    from nsn_b200.primitives import require_workspace
    ok = torch.empty(64, dtype=torch.uint8)
    require_workspace(ok, ok.device)
    for bad, device in ((ok.float(), ok.device), (ok[::2], ok.device), (ok, torch.device("cuda", 0))):
        with pytest.raises(ContractError):
            require_workspace(bad, device)
