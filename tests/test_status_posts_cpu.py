"""When the copies of the kernels' status words are queued, with events and streams that are stood in for."""
import pytest
import torch


class Event:
    def __init__(self, landed=True):
        self.landed = landed

    def query(self):
        return self.landed

    def record(self, stream=None):
        pass


@pytest.fixture
def ops(monkeypatch):
    from moddit_b200 import ops as _ops
    monkeypatch.setattr(_ops, "_POSTED", {})
    monkeypatch.setattr(_ops, "_LAST_POST", {})
    monkeypatch.setattr(_ops, "_STATUS", {0: torch.zeros(4, dtype=torch.int32)})
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: False)
    monkeypatch.setattr(torch.cuda, "current_stream", lambda device=None: None)
    monkeypatch.setattr(torch.cuda, "Event", Event)
    return _ops


def test_a_copy_that_was_not_queued_holds_up_none(ops):
    """A call that finds the last copy still on its way queues none: the next call's spacing does not count from it."""
    dev = torch.device("cuda", 0)
    slot = [torch.zeros(4, dtype=torch.int32), Event(landed=False)]
    ops._POSTED[0] = slot
    ops.post_status(dev, spacing=60.0)
    ops._STATUS[0][:] = torch.tensor([3, 1, 2, 0])
    slot[1].landed = True
    ops.post_status(dev, spacing=60.0)
    assert slot[0].tolist() == [3, 1, 2, 0]
    with pytest.raises(Exception, match="bounded wait expired"):
        ops.check_posted_status(dev)


def test_spacing_counts_from_the_last_copy(ops):
    dev = torch.device("cuda", 0)
    slot = [torch.zeros(4, dtype=torch.int32), Event()]
    ops._POSTED[0] = slot
    ops.post_status(dev, spacing=60.0)
    ops._STATUS[0][0] = 5
    ops.post_status(dev, spacing=60.0)
    assert slot[0][0] == 0
    ops.post_status(dev)
    assert slot[0][0] == 5
