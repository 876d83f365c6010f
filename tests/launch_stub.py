"""keypoints_amd.lowp / norm on CPU tensors with every launch noted instead of made: what a call would launch, and what autograd makes of it."""
import contextlib


def stub(monkeypatch):
    """-> the list of (entry, arguments) that calls append to.  Pointers are the tensors' own, strides and sizes as they would be handed over."""
    import torch
    from keypoints_amd import lowp, norm
    from keypoints_amd.models import functional
    made = []
    for module in (lowp, norm, functional):
        monkeypatch.setattr(module, 'call', lambda name, *args: made.append((name, args)))
        monkeypatch.setattr(module, 'require_device', lambda *tensors: None)
        monkeypatch.setattr(module, 'stream_ptr', lambda: 0)
    for module in (lowp, norm):
        monkeypatch.setattr(module, 'device_of', lambda t: contextlib.nullcontext())
    return made
