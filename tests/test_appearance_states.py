"""An encoder's states and their positions: in training as in serving, and refused where nothing would look at them."""
import copy

import pytest
import torch

from tdgs_amd import appearance


def step_without_gpu(monkeypatch, *args, **kw):
    seen = {}

    def dec(rgb, image, states=None, **options):
        seen.update(states=states, **options)
        return rgb * 2

    monkeypatch.setattr(appearance, "loss_grad_", lambda out, photograph, grad, *rest: grad.fill_(1.0))
    loss = object.__new__(appearance.AppearanceLoss)
    loss.dssim_weight, loss.sums, loss.temp = 0.2, torch.zeros(2), None
    optimizer = torch.optim.SGD([torch.zeros(1, requires_grad=True)], 0.1)
    loss.step_(dec, optimizer, torch.zeros(2, 2, 3), 0, torch.zeros(2, 2, 3), *args, **kw)
    return seen


def test_training_hands_positions_on(monkeypatch):
    states, places = torch.ones(5, 4), torch.ones(5, 2)
    assert step_without_gpu(monkeypatch, states, places) == {"states": states, "states_positions": places}
    assert step_without_gpu(monkeypatch, states, states_positions=places)["states_positions"] is places
    assert step_without_gpu(monkeypatch, states) == {"states": states}
    assert step_without_gpu(monkeypatch) == {"states": None}


@pytest.mark.parametrize("rotary,states,places,text", [
    (None, (5, 4), (5, 2), "without rotary"), (object(), None, (5, 2), "without states"), (object(), (5, 4), (4, 2), "shape"),
    (object(), (5, 4), (1, 2), "shape"), (object(), (5, 4), (5, 3), "shape"), (object(), (0, 4), (1, 2), "shape")])
def test_refusals(rotary, states, places, text):
    dec = object.__new__(appearance.AppearanceDecoder)   # (refused before anything of it is used)
    dec.nb_images, dec.rotary = 2, rotary
    with pytest.raises(ValueError, match=text):
        dec(torch.zeros(8, 8, 3), 0, None if states is None else torch.zeros(states), states_positions=torch.zeros(places))


@pytest.mark.gpu
def test_training_at_the_states_positions(gpu):
    """A step's parameters are those that the same gradient, taken by hand, leads to; without positions they are others."""
    gen = torch.Generator().manual_seed(0)
    rgb, photograph = (torch.rand((20, 12, 3), generator=gen).cuda() for _ in range(2))
    states, places = torch.randn((7, 6), generator=gen).cuda(), torch.randint(1, 5, (7, 2), generator=gen).cuda()
    dec = appearance.AppearanceDecoder(2, channels=32, heads=2, groups=4, states_dim=6, rotary=True, seed=3)
    loss = appearance.AppearanceLoss(20, 12)
    results = []
    for at in (places, places.float(), None):
        d = copy.deepcopy(dec)
        loss.step_(d, torch.optim.SGD(d.parameters.values(), 0.1), rgb, 1, photograph, states, at)
        results.append(d.parameters)
    x = rgb.clone().requires_grad_(True)
    out = dec(x, 1, states, states_positions=places).contiguous()
    grad = torch.empty_like(out)
    appearance.loss_grad_(out.detach(), photograph, grad, loss.dssim_weight, loss.sums, loss.temp)
    out.backward(grad)
    for name, p in dec.parameters.items():
        assert torch.equal(results[0][name], results[1][name]), name
        want = p.detach() - 0.1 * p.grad
        # (the update's product and sum, rounded once or twice)
        assert ((results[0][name] - want).abs() <= 2.0 ** -23 * (want.abs() + p.grad.abs())).all(), name
    assert not torch.equal(results[2]["key"], results[0]["key"])
