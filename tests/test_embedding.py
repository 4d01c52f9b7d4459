"""``embedding`` and its gradient against plain forms: types, odd widths,
strides, tokens outside the table, one token to many tiles of the sorted list,
runs that end in and cross its chunks, writing into and adding to a buffer."""

from __future__ import annotations

import pytest
import torch
from torch.func import grad as func_grad
from torch.func import vmap

from churten_amd import kernels as K
from churten_amd.state import State
from lm_reference import assert_within, embedding_grad

DEVICES = ["cpu", pytest.param("cuda", marks=pytest.mark.gpu)]
DTYPES = [torch.float32, torch.float16, torch.bfloat16]
pytestmark = pytest.mark.parametrize("device", DEVICES)


def gen(seed):
    return torch.Generator().manual_seed(seed)


def make_tokens(kind, N, B, V, g):
    if kind == "zipf":  # words: frequency falls as 1/rank
        return ((V + 1.0) ** torch.rand(N, B, generator=g, dtype=torch.float64) - 1).long() \
            .clamp_(0, V - 1)
    if kind == "one":  # padding: a single token throughout
        return torch.full((N, B), V // 2)
    if kind == "outside":  # a third of them outside the table
        return torch.randint(-V, 2 * V, (N, B), generator=g)
    if kind == "none":
        return torch.full((N, B), -1)
    if kind == "runs":  # runs of 63, 64 and 65: either side of a chunk
        length = torch.tensor([63, 64, 65, 1, 128, 2])
        ids = torch.arange(6).repeat_interleave(length).repeat(-(-B // 323))[:B] % V
        return ids.expand(N, B).clone()
    return torch.randint(0, V, (N, B), generator=g)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("N,B,V,D", [(1, 1, 1, 1), (3, 1, 50, 8), (2, 7, 11, 33), (4, 130, 40, 64),
                                     (2, 65, 9, 520), (1, 1000, 300, 1030)])
def test_lookup_is_the_scaled_row(device, dtype, N, B, V, D):
    g = gen(1)
    weight = torch.randn(N, V, D, generator=g).to(dtype)
    tokens = make_tokens("outside", N, B, V, g)
    inside = (tokens >= 0) & (tokens < V)
    rows = weight[torch.arange(N)[:, None], tokens.clamp(0, V - 1)].float() * 0.37
    want = torch.where(inside[..., None], rows, 0.0).to(dtype)
    got = K.embedding(weight.to(device), tokens.to(device), 0.37).cpu()
    # One product, rounded to float32 and once more to the type.
    assert torch.equal(got, want)


def test_lookup_reads_views_shared_and_narrow_tokens(device):
    g = gen(2)
    N, B, V, D = 3, 19, 23, 12
    flat = torch.randn(N, 7 + V * D + 5, generator=g).to(device)
    weight = flat[:, 7:7 + V * D].view(N, V, D)
    tokens = torch.randint(0, V, (B,), generator=g).to(device)
    want = torch.stack([weight[n][tokens] * 2.0 for n in range(N)])
    assert torch.equal(K.embedding(weight, tokens, 2.0), want)
    assert torch.equal(K.embedding(weight, tokens.int(), 2.0), want)
    assert torch.equal(K.embedding(weight, tokens.expand(N, B), 2.0), want)
    wide = torch.stack([tokens, tokens], 1).reshape(-1)[::2]  # a stride of 2
    assert torch.equal(K.embedding(weight, wide, 2.0), want)
    # A table whose columns are strided.
    assert torch.equal(K.embedding(weight.mT.contiguous().mT, tokens, 2.0), want)
    # One replica's call.
    assert torch.equal(K.embedding(weight[1], tokens, 2.0), want[1])


def test_lookup_keeps_special_values(device):
    weight = torch.tensor([[[float("nan"), float("inf"), -float("inf"), -0.0]]], device=device)
    got = K.embedding(weight, torch.zeros(1, 1, dtype=torch.long, device=device), 1.0)
    assert torch.equal(got.view(torch.int32), weight.view(torch.int32))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("kind", ["zipf", "one", "outside", "none", "runs", "even"])
@pytest.mark.parametrize("N,B,V,D", [(1, 1, 1, 1), (2, 3, 100, 8), (3, 64, 17, 33), (2, 65, 33, 64),
                                     (2, 1000, 300, 36), (1, 4096, 90, 16), (2, 4097, 700, 40),
                                     (1, 300, 40, 1100)])
def test_gradient_sums_each_tokens_rows(device, dtype, kind, N, B, V, D):
    g = gen(3)
    grad = torch.randn(N, B, D, generator=g).to(dtype)
    tokens = make_tokens(kind, N, B, V, g)
    want, bound = embedding_grad(grad, tokens, V, 0.6)
    got = K.embedding_grad(grad.to(device), tokens.to(device), V, 0.6)
    assert_within(got, want, bound)


@pytest.mark.parametrize("B", [16 * 4096 + 5, 17 * 4096])
def test_gradient_of_a_list_that_takes_two_merges(device, B):
    g = gen(4)
    V, D = 3000, 4
    grad = torch.randn(1, B, D, generator=g)
    tokens = make_tokens("zipf", 1, B, V, g)
    want, bound = embedding_grad(grad, tokens, V, 1.0)
    assert_within(K.embedding_grad(grad.to(device), tokens.to(device), V), want, bound)


def test_gradient_of_shared_tokens_and_strided_gradients(device):
    g = gen(5)
    N, B, V, D = 4, 500, 60, 24
    tokens = make_tokens("zipf", 1, B, V, g)[0]
    wide = torch.randn(N, B, 2 * D, generator=g)
    want, bound = embedding_grad(wide[..., :D], tokens.expand(N, B), V, 1.0)
    for grad in (wide.to(device)[..., :D], wide.to(device)[..., :D].mT.contiguous().mT):
        assert_within(K.embedding_grad(grad, tokens.to(device), V), want, bound)
        assert_within(K.embedding_grad(grad, tokens.int().to(device), V), want, bound)
    # An incoming gradient that is one number, expanded.
    one = torch.ones(1, device=device).expand(N, B, D)
    count = torch.bincount(tokens, minlength=V).float()
    assert torch.equal(K.embedding_grad(one, tokens.to(device), V).cpu(),
                       count[None, :, None].expand(N, V, D))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("B", [0, 1, 130, 5000])
def test_gradient_into_a_replicas_slice_writes_only_it(device, dtype, B):
    g = gen(6)
    N, V, D = 3, 37, 20
    flat = torch.randn(N, 9 + V * D + 6, generator=g).to(dtype)
    grad = torch.randn(N, B, D, generator=g).to(dtype)
    tokens = make_tokens("outside", N, B, V, g)
    buffer = flat.to(device)
    view = buffer[:, 9:9 + V * D].view(N, V, D)
    want, bound = embedding_grad(grad, tokens, V, 3.0)
    assert K.embedding_grad_(view, grad.to(device), tokens.to(device), 3.0) is None
    assert_within(view, want, bound)
    after = buffer.cpu()
    assert torch.equal(after[:, :9], flat[:, :9])
    assert torch.equal(after[:, 9 + V * D:], flat[:, 9 + V * D:])
    # Again, added: the rows that no token names keep their bits.
    before = view.cpu().clone()
    K.embedding_grad_(view, grad.to(device), tokens.to(device), 3.0, accumulate=True)
    total = before.double() + want
    assert_within(view, total, bound + 2 ** -23 * total.abs()
                  + (2 ** -8 if dtype == torch.bfloat16 else 2 ** -11) * total.abs())
    ok = (tokens >= 0) & (tokens < V)
    for n in range(N):
        unnamed = torch.ones(V, dtype=torch.bool)
        unnamed[tokens[n][ok[n]]] = False
        assert torch.equal(view[n].cpu()[unnamed], before[n][unnamed])


def test_gradient_is_the_same_on_every_run(device):
    g = gen(7)
    grad = torch.randn(2, 9000, 48, generator=g).to(device)
    tokens = make_tokens("zipf", 2, 9000, 50, g).to(device)
    first = K.embedding_grad(grad, tokens, 50)
    for _ in range(3):
        assert torch.equal(K.embedding_grad(grad, tokens, 50), first)


def test_nan_and_infinity_stay_in_their_rows(device):
    g = gen(8)
    B, V, D = 200, 30, 8
    grad = torch.randn(1, B, D, generator=g)
    tokens = torch.randint(0, V, (1, B), generator=g)
    tokens[0, 5] = -1
    grad[0, 5] = float("nan")  # takes no part
    tokens[0, 6], tokens[0, 7] = 3, 4
    grad[0, 6], grad[0, 7] = float("nan"), float("inf")
    want, bound = embedding_grad(grad, tokens, V, 1.0)
    got = K.embedding_grad(grad.to(device), tokens.to(device), V).cpu()
    assert got[0, 3].isnan().all() and (got[0, 4] == float("inf")).all()
    rest = torch.ones(V, dtype=torch.bool)
    rest[[3, 4]] = False
    assert_within(got[:, rest], want[:, rest], bound[:, rest])


def test_autograd_and_vmap(device):
    g = gen(9)
    N, B, V, D = 3, 40, 25, 6
    weight = torch.randn(N, V, D, generator=g).to(device).requires_grad_()
    tokens = torch.randint(0, V, (N, B), generator=g).to(device)

    def loss(w, ids):
        return (K.embedding(w, ids, 0.5) ** 2).sum()

    loss(weight, tokens).backward()
    plain = weight.detach().clone().requires_grad_()
    rows = plain[torch.arange(N, device=device)[:, None], tokens] * 0.5
    (rows ** 2).sum().backward()
    torch.testing.assert_close(weight.grad, plain.grad)
    each = vmap(func_grad(loss))(weight.detach(), tokens)
    assert torch.equal(each, weight.grad)
    shared = vmap(func_grad(loss), in_dims=(0, None))(weight.detach(), tokens[0])
    assert torch.equal(shared, torch.stack(
        [func_grad(loss)(w, tokens[0]) for w in weight.detach()]))
    # A batch dimension that is not the first, over calls with replicas.
    moved = weight.detach().movedim(0, 2).unsqueeze(0)
    out = vmap(lambda w: K.embedding(w, tokens[:1], 0.5), in_dims=3)(moved)
    assert torch.equal(out[:, 0], K.embedding(weight.detach(), tokens[0], 0.5))


def test_gradient_reaches_a_states_buffer(device):
    models = [torch.nn.Sequential(torch.nn.Embedding(21, 6), torch.nn.Linear(6, 3))
              for _ in range(4)]
    state = State.from_models([m.to(device) for m in models])
    g = gen(10)
    tokens = torch.randint(0, 21, (4, 30), generator=g).to(device)
    grad = torch.randn(4, 30, 6, generator=g).to(device)
    table = state._consolidated_grads["0.weight"]
    K.embedding_grad_(table, grad, tokens)
    assert torch.equal(state.grads[:, :126].view(4, 21, 6), K.embedding_grad(grad, tokens, 21))
    assert not state.grads[:, 126:].any()


def test_empty_sizes(device):
    def long(*shape):
        return torch.zeros(*shape, dtype=torch.long, device=device)

    def real(*shape):
        return torch.ones(*shape, device=device)

    assert K.embedding(real(2, 5, 4), long(2, 0)).shape == (2, 0, 4)
    assert K.embedding(real(0, 5, 4), long(0, 3)).shape == (0, 3, 4)
    assert K.embedding(real(2, 5, 0), long(2, 3)).shape == (2, 3, 0)
    assert torch.equal(K.embedding(real(2, 0, 4), long(2, 3)), real(2, 3, 4) * 0)
    assert torch.equal(K.embedding_grad(real(2, 0, 4), long(2, 0), 5), real(2, 5, 4) * 0)
    assert K.embedding_grad(real(2, 3, 4), long(2, 3), 0).shape == (2, 0, 4)
    assert K.embedding_grad(real(2, 3, 0), long(2, 3), 5).shape == (2, 5, 0)


def test_refusals(device):
    w = torch.zeros(2, 5, 4, device=device)
    ids = torch.zeros(2, 3, dtype=torch.long, device=device)
    g = torch.zeros(2, 3, 4, device=device)

    def refused(match, fn, *args, **kw):
        with pytest.raises(RuntimeError, match=match):
            fn(*args, **kw)

    refused("unsupported dtype", K.embedding, w.double(), ids)
    refused("must be int64 or int32", K.embedding, w, ids.float())
    refused("weight must be", K.embedding, w[0, 0], ids)
    refused("tokens must have", K.embedding, w, ids[None])
    refused("must have 2 replicas", K.embedding, w, torch.cat([ids, ids[:1]]))
    refused("beside a weight without replicas", K.embedding, w[0], ids)
    refused("the lookup's shape", K.embedding_grad, g[:, :2], ids, 5)
    refused("must not be negative", K.embedding_grad, g, ids, -1)
    refused("must have dtype", K.embedding_grad_, w, g.half(), ids)
    refused("the lookup's shape", K.embedding_grad_, w, g[..., :3], ids)
    refused("rows must be contiguous", K.embedding_grad_, w.mT.contiguous().mT, g, ids)
    refused("must not share memory", K.embedding_grad_, w[:1].expand(2, 5, 4), g, ids)
    refused("got \\[5, 4\\] and", K.embedding_grad_, w[0], g, ids)


@pytest.mark.gpu
def test_other_devices_tensors_are_refused(device):
    if device == "cpu":
        pytest.skip("needs two devices")
    w = torch.zeros(2, 5, 4, device=device)
    with pytest.raises(RuntimeError, match="must be on"):
        K.embedding(w, torch.zeros(2, 3, dtype=torch.long))
    with pytest.raises(RuntimeError, match="must be on"):
        K.embedding_grad_(w, torch.zeros(2, 3, 4), torch.zeros(2, 3, dtype=torch.long,
                                                               device=device))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("kind", ["zipf", "one", "outside"])
@pytest.mark.parametrize("B,V,D", [(255, 70, 3), (256, 70, 9), (257, 70, 3), (1024, 500, 10),
                                   (1025, 500, 7), (2049, 40, 12)])
def test_gradient_at_the_edges_of_its_ways(device, dtype, kind, B, V, D):
    """One launch up to 256 tokens, a sorted word per thread up to 1024, four
    beyond; rows narrower than a pack and rows whose last pack overlaps the one before."""
    g = gen(11)
    grad = torch.randn(2, B, D, generator=g).to(dtype)
    tokens = make_tokens(kind, 2, B, V, g)
    want, bound = embedding_grad(grad, tokens, V, -1.5)
    assert_within(K.embedding_grad(grad.to(device), tokens.to(device), V, -1.5), want, bound)


@pytest.mark.parametrize("V", [2 ** 22 - 2, 2 ** 22 - 1, 2 ** 22 + 5])
@pytest.mark.parametrize("B", [200, 900, 9000])
def test_gradient_of_very_large_vocabularies(device, V, B):
    """Tables of more rows than a sorted word of 32 bits has room for."""
    g = gen(13)
    grad = torch.randn(1, B, 2, generator=g)
    tokens = make_tokens("zipf", 1, B, V, g)
    tokens[0, :8] = torch.tensor([V - 1, V, V + 1, 2 ** 31 - 1, 2 ** 40, -1, 0, V - 2])
    want, bound = embedding_grad(grad, tokens, V, 1.0)
    assert_within(K.embedding_grad(grad.to(device), tokens.to(device), V), want, bound)


@pytest.mark.parametrize("V", [1, 2, 255, 256, 2 ** 16 - 1, 2 ** 16, 2 ** 20 - 1, 2 ** 20])
@pytest.mark.parametrize("B", [257, 1024, 1025, 4096, 4097])
def test_gradient_at_the_edges_of_the_tokens_digits(device, V, B):
    """Tokens of 1 to 21 bits: one to three digits, words of 32 and of 64 bits,
    tiles that are full and tiles that hold one token."""
    g = gen(14)
    grad = torch.randn(2, B, 2, generator=g)
    tokens = make_tokens("even", 2, B, V, g)
    tokens[0, 3:7] = torch.tensor([V - 1, V, V - 1, 0])
    tokens[1, -3:] = torch.tensor([V, -1, V - 1])
    want, bound = embedding_grad(grad, tokens, V, 1.0)
    assert_within(K.embedding_grad(grad.to(device), tokens.to(device), V), want, bound)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("B", [100, 700, 3000])
@pytest.mark.parametrize("D", [3, 259, 1030])
def test_adding_counts_every_element_once(device, dtype, B, D):
    """Where packs overlap, at a row's end and between a row's wavefronts."""
    g = gen(12)
    N, V = 2, 19
    grad = torch.randn(N, B, D, generator=g).to(dtype)
    tokens = make_tokens("zipf", N, B, V, g)
    before = torch.randn(N, V, D, generator=g).to(dtype)
    want, bound = embedding_grad(grad, tokens, V, 1.0)
    total = before.double() + want
    got = before.to(device)
    K.embedding_grad_(got, grad.to(device), tokens.to(device), 1.0, accumulate=True)
    half = 2.0 ** -8 if dtype == torch.bfloat16 else 2.0 ** -23
    assert_within(got, total, bound + half * total.abs() + 2.0 ** -23 * want.abs())


@pytest.mark.gpu
def test_tables_of_more_than_2_to_the_31_elements(device):
    if device == "cpu":
        pytest.skip("GPU memory")
    V, D = 66000, 33000
    tokens = torch.tensor([[V - 1, 0, 65535, V - 1]], device=device)
    weight = torch.zeros(1, V, D, device=device, dtype=torch.bfloat16)
    weight[0, -1] = torch.arange(D, device=device) % 250
    weight[0, 65535] = 3
    out = K.embedding(weight, tokens, 2.0)
    assert torch.equal(out[0, 0], weight[0, -1] * 2) and torch.equal(out[0, 3], out[0, 0])
    assert (out[0, 2] == 6).all() and not out[0, 1].any()
    for B in (4, 400):  # one launch, and sorted
        ids = tokens.repeat(1, B // 4)
        grad = torch.ones(1, B, D, device=device, dtype=torch.bfloat16)
        weight.fill_(float("nan"))
        K.embedding_grad_(weight, grad, ids)
        assert (weight[0, -1] == B // 2).all() and (weight[0, 65535] == B // 4).all()
        assert (weight[0, 0] == B // 4).all() and not weight[0, 1:65535].any()
        assert not weight[0, 65536:-1].any()


def test_gradient_in_place_under_vmap(device):
    """Over one replica's code, over calls with replicas, and along a dimension that
    is not the first; what the replicas share is shared."""
    g = gen(15)
    S, N, B, V, D = 4, 3, 70, 11, 6
    grad = torch.randn(S, N, B, D, generator=g).to(device)
    tokens = torch.randint(-1, V, (S, N, B), generator=g).to(device)
    before = torch.randn(S, N, V, D, generator=g).to(device)
    want = torch.stack([K.embedding_grad(grad[s], tokens[s], V, 0.5) for s in range(S)])

    def write(out, grad, tokens, scale=0.5, accumulate=False):
        K.embedding_grad_(out, grad, tokens, scale, accumulate=accumulate)
        return out

    flat = torch.zeros(N, 3 + V * D, device=device)
    view = flat[:, 3:].view(N, V, D)
    vmap(write)(view, grad[0], tokens[0])
    assert torch.equal(view, want[0]) and not flat[:, :3].any()
    out = before.clone()
    vmap(lambda o, g, t: write(o, g, t, accumulate=True))(out, grad, tokens)
    each = before.clone()
    for s in range(S):
        K.embedding_grad_(each[s], grad[s], tokens[s], 0.5, accumulate=True)
    assert torch.equal(out, each)
    # Rows of all of them that no one view holds: (N, S, V, D) of a wider buffer.
    wide = torch.zeros(N, S, V, 2 * D, device=device)
    vmap(write, in_dims=(1, 0, 0))(wide[..., :D], grad, tokens)
    assert torch.equal(wide[..., :D].transpose(0, 1), want) and not wide[..., D:].any()
    # Twice, with shared tokens and a shared gradient.
    out = torch.zeros(S, N, V, D, device=device)
    vmap(vmap(lambda o: write(o, grad[0, 0], tokens[0, 0], 1.0)))(out)
    assert torch.equal(out, K.embedding_grad(grad[0, 0], tokens[0, 0], V).expand(S, N, V, D))
    out = torch.zeros(S, N, V, D, device=device)
    vmap(lambda o, g: write(o, g, tokens[0], 1.0))(out, grad)
    assert torch.equal(out[2], K.embedding_grad(grad[2], tokens[0], V))
    with pytest.raises(RuntimeError, match="written in place"):
        vmap(lambda g: write(out[0], g, tokens[0]))(grad)


def test_a_table_that_vmap_is_not_over_is_not_repeated(device):
    from torch.utils._python_dispatch import TorchDispatchMode

    class Largest(TorchDispatchMode):
        bytes = 0

        def __torch_dispatch__(self, func, types, args=(), kwargs=None):
            out = func(*args, **(kwargs or {}))
            for t in out if isinstance(out, (tuple, list)) else (out,):
                if isinstance(t, torch.Tensor) and t.untyped_storage().data_ptr() not in known:
                    self.bytes = max(self.bytes, t.untyped_storage().nbytes())
            return out

    g = gen(16)
    S, N, B, V, D = 5, 3, 4, 2000, 8
    weight = torch.randn(N, V, D, generator=g).to(device)
    tokens = torch.randint(-1, V + 1, (S, N, B), generator=g).to(device)
    known = {weight.untyped_storage().data_ptr()}
    want = torch.stack([K.embedding(weight, ids, 0.5) for ids in tokens])
    for w, ids, dim, expected in ((weight, tokens, 0, want),
                                  (weight, tokens.movedim(0, 2), 2, want),
                                  (weight, tokens[:, 0], 0, torch.stack(
                                      [K.embedding(weight, ids, 0.5) for ids in tokens[:, 0]])),
                                  (weight[0], tokens[:, 0], 0, want[:, 0])):
        with Largest() as largest:
            got = vmap(lambda t: K.embedding(w, t, 0.5), in_dims=dim)(ids)
        assert torch.equal(got, expected)
        assert largest.bytes < N * V * D * 4
    # Its gradient adds up over the batch.
    up = torch.randint(-3, 4, (S, N, B, D), generator=g).float().to(device)
    got = func_grad(lambda w: (vmap(lambda t: K.embedding(w, t, 2.0))(tokens) * up).sum())(weight)
    assert torch.equal(got, sum(K.embedding_grad(u, t, V, 2.0) for u, t in zip(up, tokens)))


@pytest.mark.parametrize("shared", [False, True])
@pytest.mark.parametrize("kind", ["zipf", "one", "outside", "even"])
@pytest.mark.parametrize("B", [12289, 16384, 16385, 20000, 32768, 32769, 65536])
def test_gradient_of_lists_of_four_to_sixteen_tiles(device, B, kind, shared):
    """One merge of up to four, eight and sixteen runs, the last of them whole or short."""
    g = gen(17)
    V, D = 5000, 4
    grad = torch.randn(2, B, D, generator=g)
    tokens = make_tokens(kind, 1 if shared else 2, B, V, g)
    want, bound = embedding_grad(grad, tokens.expand(2, B), V, 0.7)
    given = tokens[0] if shared else tokens
    assert_within(K.embedding_grad(grad.to(device), given.to(device), V, 0.7), want, bound)


@pytest.mark.parametrize("B", [20000, 40000])
def test_gradient_of_many_tiles_of_a_very_large_vocabulary(device, B):
    """Sorted words of 64 bits, merged."""
    g = gen(18)
    V, D = 2 ** 21, 2
    grad = torch.randn(1, B, D, generator=g)
    tokens = make_tokens("zipf", 1, B, V, g)
    want, bound = embedding_grad(grad, tokens, V, 1.0)
    assert_within(K.embedding_grad(grad.to(device), tokens.to(device), V), want, bound)
