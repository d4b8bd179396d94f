"""Head norms and rotations of which not all gradients are wanted: those that are, are the full call's, and what is frozen is no
part of the gradient call."""
import itertools

import pytest
import torch

from tdgs_amd import decoder

pytestmark = pytest.mark.gpu


def rand(*shape, seed=0):
    return torch.randn(shape, generator=torch.Generator().manual_seed(seed)).cuda()


@pytest.fixture
def calls(monkeypatch):
    """(queries or keys, keys) heads of each gradient call."""
    seen = []

    def record(name, at):
        f = getattr(decoder, name)

        def call(*args, **kw):
            seen.append(tuple(0 if t is None else t.shape[2] for t in args[at:at + 2]))
            return f(*args, **kw)
        monkeypatch.setattr(decoder, name, call)

    record("head_norm_grad_", 0)
    record("rotate_", 0)
    return seen


@pytest.mark.parametrize("wanted", list(itertools.product([False, True], repeat=4))[1:], ids=str)
def test_head_norm(gpu, calls, wanted):
    rotary, places = decoder.Rotary((4,)), torch.arange(5, device="cuda")[:, None]
    tensors = (rand(2, 5, 4, 8), rand(2, 5, 2, 8, seed=1), 1 + rand(8, seed=2) / 4, 1 + rand(8, seed=3) / 4)
    coef = rand(2, 5, 4, 8, seed=4), rand(2, 5, 2, 8, seed=5)

    def grads(wants):
        leaves = [t.clone().requires_grad_(w) for t, w in zip(tensors, wants)]
        q, k = decoder.head_norm(*leaves, rotary=rotary, positions=places)
        ((q * coef[0]).sum() + (k * coef[1]).sum()).backward()
        return [leaf.grad for leaf in leaves]

    want, got = grads((True,) * 4), grads(wanted)
    for g, h, w in zip(got, want, wanted):
        assert g is None if not w else torch.equal(g, h)
    q, k = wanted[0] or wanted[2], wanted[1] or wanted[3]
    assert calls[1:] == [(4, 2) if q and k else (4, 0) if q else (2, 0)]


@pytest.mark.parametrize("wanted", [(True, False), (False, True), (True, True)], ids=str)
def test_rotate(gpu, calls, wanted):
    rotary, places = decoder.Rotary((4,)), torch.arange(5, device="cuda")[:, None]
    leaves = [rand(2, 5, n, 8, seed=n).requires_grad_(w) for n, w in zip((4, 2), wanted)]
    outs = decoder.rotate(*leaves, rotary, places)
    coef = [rand(2, 5, n, 8, seed=10 + n) for n in (4, 2)]
    del calls[:]
    sum((o * c).sum() for o, c in zip(outs, coef)).backward()
    back = decoder.rotate(*coef, rotary, places, inverse=True)
    for leaf, w, b in zip(leaves, wanted, back):
        assert leaf.grad is None if not w else torch.equal(leaf.grad, b)
    assert calls[0] == {(True, False): (4, 0), (False, True): (2, 0), (True, True): (4, 2)}[wanted]


def test_one_sided_calls(gpu):
    """Without keys, with a weight alone wanted."""
    q, w = rand(2, 5, 4, 8), (1 + rand(8, seed=2) / 4).requires_grad_(True)
    full, fw = q.clone().requires_grad_(True), w.detach().clone().requires_grad_(True)
    decoder.head_norm(q, None, w).square().sum().backward()
    decoder.head_norm(full, None, fw).square().sum().backward()
    assert torch.equal(w.grad, fw.grad)


def test_weight_of_no_keys(gpu):
    """Its gradient is zero, alone and with q's."""
    for wants_q in (False, True):
        q, w = rand(2, 5, 4, 8).requires_grad_(wants_q), (1 + rand(8, seed=2) / 4).requires_grad_(True)
        torch.full((8,), 5.0, device="cuda")   # (what a gradient left unwritten would likely hold)
        (decoder.head_norm(q, None, None, w).sum() + 0 * w.sum()).backward()
        assert w.grad is not None and not w.grad.any() and (q.grad is not None) == wants_q
