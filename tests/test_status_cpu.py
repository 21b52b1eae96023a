"""CPU: what the status monitor does with reports of the kernels, on words that no kernel wrote."""
import pytest
import torch

from flex_block_attn_b200 import interface


@pytest.fixture
def monitor(monkeypatch):
    """A monitor without a device; ``monitor.capturing`` says whether the stream is being captured."""
    mon = interface._StatusMonitor.__new__(interface._StatusMonitor)
    mon.device, mon.pending, mon.capturing = torch.device("cpu"), False, False
    mon.buf, mon.host, mon.mapped = (torch.zeros(8, dtype=torch.int32) for _ in range(3))
    mon._mapped_np = mon.mapped.numpy()
    mon.event = type("Done", (), {"query": lambda self: True})()
    monkeypatch.setattr(interface, "_capturing", lambda: mon.capturing)
    monkeypatch.setattr(torch.cuda, "synchronize", lambda device=None: None)
    return mon


PAGE = [2, 0, 0, 3, 0, 0, 77, 0]
WAIT = [1, 2, 13, 5, 6, 7, 100, 0]


def put(words, values):
    words.copy_(torch.tensor(values, dtype=torch.int32))


def test_a_report_is_raised_once(monitor):
    monitor.poll_mapped()
    put(monitor.mapped, PAGE)
    with pytest.raises(RuntimeError, match="page number 77 for sequence 3"):
        monitor.poll_mapped()
    monitor.poll_mapped()


def test_a_report_waits_for_the_end_of_a_capture(monitor):
    """Nothing is raised, cleared or read while it may still be incomplete, and nothing recorded into the graph."""
    put(monitor.mapped, PAGE)
    monitor.capturing = True
    monitor.poll_mapped()
    assert monitor.mapped.tolist() == PAGE
    monitor.capturing = False
    with pytest.raises(RuntimeError, match="page number 77"):
        monitor.poll_mapped()


def test_a_report_in_one_set_of_words_does_not_clear_the_other(monitor):
    """The block operator's (device words and their mirror) and those in host memory."""
    put(monitor.mapped, PAGE)
    put(monitor.buf, WAIT)
    with pytest.raises(RuntimeError, match="page number 77"):
        monitor.poll_mapped()
    assert monitor.buf.tolist() == WAIT and not monitor.mapped.any()
    put(monitor.host, WAIT)
    put(monitor.mapped, PAGE)
    monitor.pending = True
    with pytest.raises(RuntimeError, match=r"wait timed out.*block=\(5,6\)"):
        monitor.poll()
    assert not monitor.buf.any() and not monitor.host.any() and monitor.mapped.tolist() == PAGE
    with pytest.raises(RuntimeError, match="page number 77"):
        monitor.poll_mapped()


def test_a_timeout_in_the_words_in_host_memory(monitor):
    """The window kernels report there."""
    put(monitor.mapped, WAIT)
    with pytest.raises(RuntimeError, match="kernel=2 role=13"):
        monitor.poll_mapped()
    assert not monitor.mapped.any()


def test_threads_that_call_first_share_one_monitor(monkeypatch):
    """Words that nobody looks at again would lose what kernels report there."""
    import threading

    both = threading.Barrier(2, timeout=10)

    class Slow:
        def __init__(self, device):
            both.wait()

    monkeypatch.setattr(interface, "_StatusMonitor", Slow)
    monkeypatch.setattr(interface, "_monitors", {})
    monkeypatch.setattr(interface, "_capturing", lambda: False)
    got = []
    threads = [threading.Thread(target=lambda: got.append(interface._monitor(torch.device("cuda", 0)))) for _ in range(2)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert len(got) == 2 and got[0] is got[1] is interface._monitors[0]
