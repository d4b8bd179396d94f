"""Every decoder operator is launched on its tensors' device, whichever is current (without a GPU: the devices, the tensors
and the library are stand-ins)."""
import contextlib

import pytest
import torch

from tdgs_amd import core, decoder


class OnDevice(torch.Tensor):
    """A tensor that says it is on GPU 1."""
    is_cuda = True
    device = torch.device("cuda", 1)

    def get_device(self):
        return 1


@pytest.mark.parametrize("current", [0, 1])
@pytest.mark.parametrize("name", ["attention", "attention_grad", "norm", "norm_grad", "lookup", "embedding_grad"])
def test_launched_on_the_tensors_device(monkeypatch, name, current):
    now, seen = [current], []

    @contextlib.contextmanager
    def device(d):
        before, now[0] = now[0], d
        yield
        now[0] = before

    class Library:
        def __getattr__(self, entry):
            return lambda *args: 64 if entry.endswith("temp_bytes") else seen.append((entry, now[0])) or 0

    monkeypatch.setattr(torch._C, "_cuda_getDevice", lambda: now[0], raising=False)
    monkeypatch.setattr(torch.cuda, "device", device)
    monkeypatch.setattr(torch._C, "_cuda_getCurrentRawStream", lambda d: 0, raising=False)
    monkeypatch.setattr(decoder, "lib", Library)
    monkeypatch.setattr(core, "context", lambda d: None)

    def t(*shape, dtype=torch.float32):
        return torch.zeros(shape, dtype=dtype).as_subclass(OnDevice)

    x, img, w, rows = t(1, 3, 2, 8), t(1, 4, 8), t(8), t(3, 8)
    stats, lse, tokens, temp = t(1, 2, 2), t(1, 2, 3), t(3, dtype=torch.int32), t(64, dtype=torch.uint8)
    {
        "attention": lambda: decoder.cross_attention_(x, x, x, x, temp=temp),
        "attention_grad": lambda: decoder.cross_attention_grad_(x, x, x, x, x, lse, x, x, x, temp=temp),
        "norm": lambda: decoder.group_norm_(img, img, 2, w, w, temp=temp),
        "norm_grad": lambda: decoder.group_norm_grad_(img, w, w, img, img, stats, 2, w, w, temp=temp),
        "lookup": lambda: decoder.embedding_lookup_(rows, rows, tokens),
        "embedding_grad": lambda: decoder.embedding_grad_(rows, rows, tokens, temp=temp),
    }[name]()
    assert len(seen) == 1 and seen[0][1] == 1 and now == [current]
