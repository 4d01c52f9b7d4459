"""Which derivatives the language-model operators have, and that asking for
another one raises instead of giving zeros or nothing."""

from __future__ import annotations

import pytest
import torch
from torch.autograd import forward_ad
from torch.func import grad as func_grad
from torch.func import jvp, vmap

from churten_amd import kernels as K

DEVICES = ["cpu", pytest.param("cuda", marks=pytest.mark.gpu)]
pytestmark = pytest.mark.parametrize("device", DEVICES)


def table(device, replicas=True):
    """A table of small whole numbers, whose sums and products are exact, and tokens."""
    g = torch.Generator().manual_seed(1)
    lead = (2,) if replicas else ()
    weight = torch.randint(-3, 4, (*lead, 7, 5), generator=g).float()
    return weight.to(device), torch.randint(0, 7, (*lead, 9), generator=g).to(device)


def lookups(tokens):
    """The operator and plain indexing, scaled by 2."""
    at = (tokens,) if tokens.dim() == 1 else (torch.arange(2, device=tokens.device)[:, None],
                                              tokens)
    return lambda w: K.embedding(w, tokens, 2.0), lambda w: w[at] * 2.0


def heads(device):
    g = torch.Generator().manual_seed(2)
    q, k = torch.randn(2, 3, 4, 8, generator=g), torch.randn(2, 3, 2, 8, generator=g)
    w, angle = torch.randn(2, 8, generator=g), torch.randn(6, 4, generator=g)
    positions = torch.randint(0, 6, (2, 3), generator=g)
    return [t.to(device) for t in (q, k, w, w + 1, angle.cos(), angle.sin(), positions)]


def rows(device):
    g = torch.Generator().manual_seed(3)
    row = [torch.randn(2, 3, 11, generator=g), torch.randn(2, 3, 4, generator=g),
           torch.randint(0, 11, (2, 3, 4), generator=g), torch.tensor([1.0, 2.0])]
    return [t.to(device) for t in row]


def once_differentiable(device):
    """(function of one tensor, that tensor) for each operator without a second derivative."""
    _, *rest = heads(device)
    _, *teacher = rows(device)
    return [(lambda q: (K.qk_norm_rope(q, *rest)[0] ** 3).sum(), heads(device)[0]),
            (lambda w: (K.qk_norm_rope(*heads(device)[:2], w, *rest[2:])[0] ** 3).sum(), rest[1]),
            (lambda x: K.distill_loss(x, *teacher).sum(), rows(device)[0])]


@pytest.mark.parametrize("replicas", [False, True])
def test_embedding_is_differentiable_more_than_once(device, replicas):
    weight, tokens = table(device, replicas)
    ours, plain = lookups(tokens)

    def penalty(lookup):  # every derivative up to the third is of use
        def loss(w):
            return (lookup(w) ** 4).sum()

        leaf = weight.clone().requires_grad_()
        first, = torch.autograd.grad(loss(leaf), leaf, create_graph=True)
        second, = torch.autograd.grad((first ** 2).sum(), leaf, create_graph=True)
        third, = torch.autograd.grad((loss(leaf) + second.sum()), leaf)
        nested = func_grad(lambda w: (func_grad(loss)(w) ** 2).sum())(weight)
        return first, second, third, nested

    for got, want in zip(penalty(ours), penalty(plain)):
        assert want.any() and torch.equal(got, want)


def test_second_derivatives_of_embedding_under_vmap(device):
    weight, tokens = table(device)

    def curvature(w, ids):
        return func_grad(lambda w: (func_grad(
            lambda w: (K.embedding(w, ids, 2.0) ** 3).sum())(w) ** 2).sum())(w)

    each = torch.stack([curvature(w, ids) for w, ids in zip(weight, tokens)])
    assert each.any() and torch.equal(vmap(curvature)(weight, tokens), each)


def test_a_second_derivative_that_is_not_there_raises(device):
    for f, x in once_differentiable(device):
        leaf = x.clone().requires_grad_()
        first, = torch.autograd.grad(f(leaf), leaf, create_graph=True)
        torch.testing.assert_close(first, func_grad(f)(x))  # the first is there
        with pytest.raises(RuntimeError, match="not implemented"):
            (f(leaf) + (first ** 2).sum()).backward()
        with pytest.raises(RuntimeError, match="not implemented"):
            func_grad(lambda x: (func_grad(f)(x) ** 2).sum())(x)


def test_a_derivative_of_a_gradient_operator_raises(device):
    row = rows(device)
    row[0].requires_grad_()
    q, k, *rest = heads(device)
    q.requires_grad_()
    for out in (K.distill_loss_grad(*row)[0],
                K.qk_norm_rope_grad(torch.ones_like(q), torch.ones_like(k), q, k, *rest)[2]):
        with pytest.raises(RuntimeError, match="not implemented"):
            out.sum().backward()


def test_the_embedding_gradient_is_differentiable(device):
    _, tokens = table(device)
    grad = torch.ones(2, 9, 5, device=device, requires_grad=True)
    up = torch.arange(70.0, device=device).view(2, 7, 5)
    (K.embedding_grad(grad, tokens, 7, 2.0) * up).sum().backward()
    assert torch.equal(grad.grad, K.embedding(up, tokens, 2.0))


def test_forward_mode_raises(device):
    """A tangent that no derivative carries on is not dropped."""
    weight, tokens = table(device)
    row = rows(device)
    q, k, *rest = heads(device)
    calls = [(lambda w: K.embedding(w, tokens, 2.0), weight),
             (lambda q: K.qk_norm_rope(q, k, *rest)[0], q),
             (lambda w: K.qk_norm_rope(q, k, rest[0], w, *rest[2:])[1], rest[1]),
             (lambda x: K.distill_loss(x, *row[1:]), row[0]),
             (lambda t: K.distill_loss(*row[:3], t), row[3]),
             (lambda g: K.embedding_grad(g, tokens, 7), weight[:, [0, 1, 2, 3, 4, 5, 6, 0, 1]]),
             (lambda x: K.distill_loss_grad(x, *row[1:]), row[0])]
    for call, x in calls:
        with forward_ad.dual_level():
            with pytest.raises((RuntimeError, NotImplementedError), match="jvp|forward AD"):
                call(forward_ad.make_dual(x, torch.ones_like(x)))
        with pytest.raises((RuntimeError, NotImplementedError), match="jvp|forward AD"):
            jvp(call, (x,), (torch.ones_like(x),))
        with forward_ad.dual_level():
            call(x)  # no tangent: as ever


def test_the_gradient_in_place_is_seen_by_autograd(device):
    """As torch's own operators in place: the version counter rises, a saved tensor
    that is overwritten is noticed, a leaf that requires gradients is refused."""
    _, tokens = table(device)
    grad = torch.ones(2, 9, 5, device=device)
    flat = torch.zeros(2, 40, device=device)
    out = flat[:, 1:36].view(2, 7, 5)
    K.embedding_grad_(out, grad, tokens)
    assert out._version == 1 and flat._version == 1
    K.embedding_grad_(out, grad, tokens, 2.0, accumulate=True)
    assert out._version == 2
    leaf = torch.ones(2, 7, 5, device=device, requires_grad=True)
    product = leaf * out
    K.embedding_grad_(out, grad, tokens)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        product.sum().backward()
    with pytest.raises(RuntimeError, match="leaf Variable that requires grad"):
        K.embedding_grad_(leaf, grad, tokens)
    assert (leaf == 1).all()
    with torch.no_grad():
        K.embedding_grad_(leaf, grad, tokens)  # as an optimizer writes to its parameters
    assert torch.equal(leaf.detach(), K.embedding_grad(grad, tokens, 7))
    # A target that gradients would go through: they would have to go through this.
    target = leaf * 1
    K.embedding_grad_(target, grad, tokens, accumulate=True)
    with pytest.raises(RuntimeError, match="not implemented"):
        target.sum().backward()
    with forward_ad.dual_level():
        with pytest.raises((RuntimeError, NotImplementedError), match="forward AD"):
            K.embedding_grad_(out, forward_ad.make_dual(grad, grad), tokens)


def test_an_input_without_a_derivative_does_not_lose_its_gradient_silently(device):
    x, z, index, t = rows(device)
    weight, share = torch.rand(2, 3, device=device), torch.rand(2, device=device)
    labels = torch.randint(0, 11, (2, 3)).to(device)
    q, k, qw, kw, cos, sin, positions = heads(device)
    calls = [(lambda x, t: K.distill_loss(x, z, index, t), x, t),
             (lambda x, w: K.distill_loss(x, z, index, t, w), x, weight),
             (lambda x, h: K.distill_loss(x, z, index, t, weight, labels, h), x, share),
             (lambda q, c: K.qk_norm_rope(q, k, qw, kw, c, sin, positions)[0], q, cos),
             (lambda q, s: K.qk_norm_rope(q, k, qw, kw, cos, s, positions)[0], q, sin)]
    for call, main, other in calls:
        want, = torch.autograd.grad(call(leaf := main.clone().requires_grad_(), other).sum(), leaf)
        for with_main in (False, True):
            leaf = main.clone().requires_grad_(with_main)
            learned = other.clone().requires_grad_()
            out = call(leaf, learned)
            with pytest.raises(RuntimeError, match="not implemented"):
                out.sum().backward()
            with pytest.raises(RuntimeError, match="not implemented"):
                func_grad(lambda o: call(leaf.detach(), o).sum())(other)
        # Where it is not asked for, the other gradient is there.
        got, = torch.autograd.grad(call(leaf, learned).sum(), leaf)
        assert torch.equal(got, want)
        assert torch.equal(func_grad(lambda m: call(m, learned.detach()).sum())(main), want)
        with torch.no_grad():
            assert torch.equal(call(leaf, learned), call(main, other))
        # A derivative in the one around a derivative in the other.
        with pytest.raises(RuntimeError, match="not implemented"):
            func_grad(lambda o: func_grad(lambda m: call(m, o).sum())(main).sum())(other)
        each = vmap(func_grad(lambda m: call(m, learned.detach()).sum()))(torch.stack([main] * 2))
        torch.testing.assert_close(each[1], want)


def test_no_gradient_flows_to_the_teacher(device):
    x, z, index, t = rows(device)
    taught = z.clone().requires_grad_()
    assert not K.distill_loss(x, taught, index, t).requires_grad
    leaf = x.clone().requires_grad_()
    K.distill_loss(leaf, taught, index, t).sum().backward()
    assert taught.grad is None
    assert torch.equal(leaf.grad, K.distill_loss_grad(x, z, index, t)[1])
    both = func_grad(lambda x, z: K.distill_loss(x, z, index, t).sum(), argnums=(0, 1))(x, z)
    assert torch.equal(both[0], leaf.grad) and not both[1].any()


def test_embedding_in_inference_mode_and_traced_with_symbols(device):
    weight, tokens = table(device)
    grad = torch.ones(2, 9, 5, device=device)
    want = K.embedding_grad(grad, tokens, 7)
    with torch.inference_mode():
        made = torch.zeros(2, 7, 5, device=device)
        assert torch.equal(K.embedding(weight, tokens, 2.0), lookups(tokens)[1](weight))
    K.embedding_grad_(made, grad, tokens)
    assert torch.equal(made, want)
    with torch.inference_mode():
        K.embedding_grad_(made, grad, tokens, accumulate=True)
    assert torch.equal(made, 2 * want)

    def loss(w, ids):
        return (K.embedding(w, ids, 2.0) ** 2).sum()

    compiled = torch.compile(loss, backend="aot_eager", dynamic=True, fullgraph=True)
    for V, B in ((7, 9), (6, 5), (4, 8)):
        leaf, ids = weight[:, :V].clone().requires_grad_(), tokens[:, :B] % V
        got, = torch.autograd.grad(compiled(leaf, ids), leaf)
        assert torch.equal(got, torch.autograd.grad(loss(leaf, ids), leaf)[0])
