"""perf/operators.py without a GPU."""
import types


def test_contexts_by_device_and_stream(monkeypatch):
    import torch
    import computelibrary_b200 as cl
    from perf import operators

    at = [0, 0]
    monkeypatch.setattr(torch.cuda, "current_device", lambda: at[0])
    monkeypatch.setattr(torch.cuda, "current_stream", lambda: types.SimpleNamespace(cuda_stream=at[1]))
    monkeypatch.setattr(cl, "Context", lambda device, stream: (device, stream))
    monkeypatch.setattr(operators, "_kept", {})
    seen = []
    for at[:] in ((0, 0), (1, 0), (0, 5), (1, 5), (0, 0)):
        seen.append(operators._context())
    assert seen == [(0, 0), (1, 0), (0, 5), (1, 5), (0, 0)] and len(operators._kept) == 4
