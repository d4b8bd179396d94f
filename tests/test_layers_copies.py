"""A rotation passes the address of the frequencies that it holds, whatever was copied from what (without a GPU: the device
and the library are stand-ins)."""
import copy
import io
import pickle

import pytest
import torch

from tdgs_amd import abi, decoder


class OnDevice(torch.Tensor):
    """A tensor that says it is on GPU 0."""
    is_cuda = True
    device = torch.device("cuda", 0)

    def get_device(self):
        return 0


def t(*shape, dtype=torch.float32):
    return torch.zeros(shape, dtype=dtype).as_subclass(OnDevice)


@pytest.fixture
def rotary(monkeypatch):
    monkeypatch.setattr(decoder, "_dev", lambda device: torch.device("cpu"))
    r = decoder.Rotary((3, 1))
    r.turns = r.turns.as_subclass(OnDevice)
    return r


@pytest.fixture
def seen(monkeypatch):
    """The frequencies' addresses of the calls."""
    addresses = []

    class Library:
        def __getattr__(self, entry):
            def call(*args):
                if entry == "tdgs_head_norm_forward":
                    addresses.append(abi.HeadNormC.from_buffer_copy(args[1]).turns)
                return 0
            return call

    monkeypatch.setattr(torch._C, "_cuda_getDevice", lambda: 0, raising=False)
    monkeypatch.setattr(torch._C, "_cuda_getCurrentRawStream", lambda d: 0, raising=False)
    monkeypatch.setattr(decoder, "lib", Library)
    return addresses


def as_on_device(r):
    r.turns = r.turns.as_subclass(OnDevice)
    return r


def saved(r):
    file = io.BytesIO()
    torch.save(r, file)
    file.seek(0)
    return torch.load(file, weights_only=False)


def moved(r):
    """Frequencies put elsewhere by the program."""
    other = copy.copy(r)
    other.turns = r.turns.clone()
    return other


@pytest.mark.parametrize("how", ["copied", "pickled", "saved", "moved"])
def test_addresses_of_copies(rotary, seen, how):
    rotary.turns = rotary.turns.as_subclass(torch.Tensor)   # (the stand-in cannot be copied)
    other = {"copied": copy.deepcopy, "moved": moved, "saved": saved,
             "pickled": lambda r: pickle.loads(pickle.dumps(r))}[how](rotary)
    as_on_device(rotary), as_on_device(other)
    assert other.turns.data_ptr() != rotary.turns.data_ptr() and torch.equal(other.turns, rotary.turns)
    q, places = t(1, 2, 3, 8), t(2, 2, dtype=torch.int32)
    for r in (rotary, other):
        decoder.head_norm_(t(1, 2, 3, 8), None, q, rotary=r, positions=places)
        decoder.rotate_(t(1, 2, 3, 8), None, q, None, r, places)
    assert seen == [rotary.turns.data_ptr()] * 2 + [other.turns.data_ptr()] * 2


def test_the_frequencies_device_is_looked_at(rotary, seen):
    """Also of frequencies that have moved since the rotation was made."""
    rotary.turns = rotary.turns.as_subclass(torch.Tensor)
    with pytest.raises(ValueError, match="rotary"):
        decoder.rotate_(t(1, 2, 3, 8), None, t(1, 2, 3, 8), None, rotary, t(2, 2, dtype=torch.int32))
    assert not seen
