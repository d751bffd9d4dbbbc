"""The scratch memory of the front end's calls, eager and under capture (no GPU)."""
import torch


def test_a_captured_call_has_scratch_of_its_own(pkg, monkeypatch):
    """A graph replays on the address it was captured with: it must not be the shared buffer, which a later,
    larger call gives back to the allocator."""
    from llm_serving_b200 import paged_ops
    ws = paged_ops.Workspace()
    dev = torch.device("cpu")
    monkeypatch.setattr(paged_ops, "_capturing", lambda device: False, raising=False)
    shared = ws.get(dev, 1000, 7)
    assert ws.get(dev, 500, 7) is shared
    monkeypatch.setattr(paged_ops, "_capturing", lambda device: True, raising=False)
    a, b = ws.get(dev, 500, 7), ws.get(dev, 5000, 7)
    assert a.numel() >= 500 and b.numel() >= 5000
    assert len({t.data_ptr() for t in (shared, a, b)}) == 3
    monkeypatch.setattr(paged_ops, "_capturing", lambda device: False, raising=False)
    assert ws.get(dev, 1000, 7) is shared  # neither took its place
