"""The differentiable decoder operators without a GPU: the calls that reach the kernels are replaced by the formulas in
torch, so that what is tested is what stands between them and torch's differentiation."""
import pytest
import torch

from tdgs_amd import decoder


def _attention(q, k, v, scale=None):
    scale = q.shape[3] ** -0.5 if scale is None else scale
    k, v = (x.repeat_interleave(q.shape[2] // k.shape[2], dim=2) for x in (k, v))
    s = scale * (q.transpose(1, 2) @ k.permute(0, 2, 3, 1))
    return (torch.softmax(s, dim=3) @ v.transpose(1, 2)).transpose(1, 2)


def _norm(x, groups, weight, bias):
    y = x.reshape(x.shape[0], -1, groups, x.shape[-1] // groups)
    y = (y - y.mean(dim=(1, 3), keepdim=True)) / torch.sqrt(y.var(dim=(1, 3), unbiased=False, keepdim=True) + 1e-5)
    return torch.nn.functional.silu(y.reshape(x.shape) * weight + bias)


@pytest.fixture
def stand_ins(monkeypatch):
    def gradients(outs, f, leaves, dout):
        with torch.enable_grad():
            leaves = [t.detach().requires_grad_(True) for t in leaves]
            for out, g in zip(outs, torch.autograd.grad(f(*leaves), leaves, dout)):
                if out is not None:
                    out.copy_(g)

    def attention_(out, q, k, v, *, scale=None, kv_lengths=None, kv_mask=None, lse=None, temp=None):
        out.copy_(_attention(q, k, v, scale))

    def attention_grad_(dq, dk, dv, dout, out, lse, q, k, v, *, scale=None, kv_lengths=None, kv_mask=None, temp=None):
        gradients((dq, dk, dv), lambda *t: _attention(*t, scale), (q, k, v), dout)

    def norm_(out, x, groups, weight=None, bias=None, *, eps=1e-5, activation="silu", stats=None, temp=None):
        out.copy_(_norm(x, groups, weight, bias))

    def norm_grad_(dx, dweight, dbias, dout, x, stats, groups, weight=None, bias=None, *, activation="silu", temp=None):
        gradients((dx, dweight, dbias), lambda *t: _norm(t[0], groups, *t[1:]), (x, weight, bias), dout)

    def lookup_(out, table, tokens, *, scale=1.0, ctx=None):
        out.copy_(scale * table[tokens].reshape(out.shape))

    def lookup_grad_(dtable, dout, tokens, *, scale=1.0, padding=None, temp=None, ctx=None):
        dtable.zero_().index_add_(0, tokens.reshape(-1).long(), scale * dout)

    for name, f in (("cross_attention_", attention_), ("cross_attention_grad_", attention_grad_), ("group_norm_", norm_),
                    ("group_norm_grad_", norm_grad_), ("embedding_lookup_", lookup_), ("embedding_grad_", lookup_grad_)):
        monkeypatch.setattr(decoder, name, f)


def _calls():
    gen = torch.Generator().manual_seed(0)

    def leaf(*shape):
        return torch.randn(shape, generator=gen, dtype=torch.float64).requires_grad_(True)

    q, k, v = leaf(1, 5, 2, 4), leaf(1, 3, 2, 4), leaf(1, 3, 2, 4)
    x, w, b, table = leaf(1, 6, 4), leaf(4), leaf(4), leaf(7, 3)
    tokens = torch.tensor([1, 5, 5, 0])
    return {"attention": (lambda: decoder.cross_attention(q, k, v), q), "norm": (lambda: decoder.group_norm(x, 2, w, b), x),
            "embedding": (lambda: decoder.embedding(table, tokens) ** 2, table)}


@pytest.mark.parametrize("name", ["attention", "norm", "embedding"])
def test_first_derivative(stand_ins, name):
    f, leaf = _calls()[name]
    g, = torch.autograd.grad((f() ** 2).sum(), leaf)
    d = torch.randn(leaf.shape, generator=torch.Generator().manual_seed(1), dtype=torch.float64)
    value, sums = leaf.data.clone(), []
    for sign in (1, -1):
        leaf.data.copy_(value + sign * 2.0 ** -13 * d)
        sums.append((f().detach() ** 2).sum())
    # central differences: step^2 of the third derivative and 2^-52 of the value over the step
    assert abs((g * d).sum() - (sums[0] - sums[1]) * 2.0 ** 12) <= 1e-4 * g.norm() * d.norm()


@pytest.mark.parametrize("name", ["attention", "norm", "embedding"])
def test_second_derivative_raises(stand_ins, name):
    """The gradients are no function of their operands for torch: a gradient of them has to be refused, not to lack a part
    in silence where the loss has another path to the leaf."""
    f, leaf = _calls()[name]
    for loss in (lambda: f().sum(), lambda: (f() ** 2).sum()):   # the operator's dout: constant, and not
        g, = torch.autograd.grad(loss() + (leaf ** 3).sum(), leaf, create_graph=True)
        with pytest.raises(RuntimeError, match="differentiated again"):
            torch.autograd.grad((g ** 2).sum(), leaf, retain_graph=True)
        with pytest.raises(RuntimeError, match="differentiated again"):
            (g ** 2).sum().backward()


def test_gradients_that_nothing_needs(stand_ins, monkeypatch):
    """Frozen states and parameters: their gradients are not asked for, the others are the same."""
    asked = {}

    def record(name, n):
        f = getattr(decoder, name)
        monkeypatch.setattr(decoder, name, lambda *a, **kw: (asked.update({name: [t is not None for t in a[:n]]}), f(*a, **kw))[1])

    record("cross_attention_grad_", 3)
    record("group_norm_grad_", 3)
    gen = torch.Generator().manual_seed(4)
    q, k, v, x = (torch.randn(s, generator=gen, dtype=torch.float64) for s in ((1, 5, 2, 4), (1, 3, 2, 4), (1, 3, 2, 4), (1, 6, 4)))
    w, b = torch.ones(4, dtype=torch.float64), torch.zeros(4, dtype=torch.float64)

    def grads(f, *leaves):
        for t in (q, k, v, x, w, b):
            t.requires_grad_(any(t is u for u in leaves))
        return torch.autograd.grad((f() ** 2).sum(), leaves)

    attention, norm = lambda: decoder.cross_attention(q, k, v), lambda: decoder.group_norm(x, 2, w, b)   # noqa: E731
    every = grads(attention, q, k, v) + grads(norm, x, w, b)
    assert asked == {"cross_attention_grad_": [True, True, True], "group_norm_grad_": [True, True, True]}
    some = grads(attention, q) + grads(norm, x, b)
    assert asked == {"cross_attention_grad_": [True, False, False], "group_norm_grad_": [True, False, True]}
    for a, g in zip(some, (every[0], every[3], every[5])):
        assert torch.equal(a, g)
