"""``qk_norm_rope`` and its backward pass against plain forms in 64 bits: types,
head widths (packs of 16 and 8 bytes, single elements), partial and neighbouring
pairs, strides, grouped heads, positions outside the tables."""

from __future__ import annotations

import pytest
import torch
from torch.func import grad as func_grad
from torch.func import vmap

from churten_amd import kernels as K
from lm_reference import assert_within, qk_side, qk_side_grad

DEVICES = ["cpu", pytest.param("cuda", marks=pytest.mark.gpu)]
DTYPES = [torch.float32, torch.float16, torch.bfloat16]
pytestmark = pytest.mark.parametrize("device", DEVICES)

EPS = 1e-6
# D, rot: vectors of 16 bytes (64, 128, 96 of 48, 512), of 8 (80 of 40 and 48 of
# 24 across pairs), odd packs, single elements, no rotation, more than 64 units.
WIDTHS = [(64, 64), (128, 128), (96, 48), (80, 40), (48, 24), (512, 512), (12, 4), (33, 32),
          (33, 0), (1, 0), (2, 2), (7, 6), (510, 254), (257, 128), (256, 0), (129, 2)]
SHAPES = [(1, 1, 1, 1), (2, 5, 4, 2), (3, 37, 6, 3), (1, 130, 7, 1)]


def inputs(N, M, Hq, Hk, D, rot, dtype, seed, P=50, fused=False):
    g = torch.Generator().manual_seed(seed)
    if fused:
        x = torch.randn(N, M, Hq + 2 * Hk, D, generator=g).to(dtype)
        q, k = x[:, :, :Hq], x[:, :, Hq:Hq + Hk]
    else:
        q = torch.randn(N, M, Hq, D, generator=g).to(dtype)
        k = (3 * torch.randn(N, M, Hk, D, generator=g)).to(dtype)
    qw = (1 + 0.2 * torch.randn(N, D, generator=g)).to(dtype)
    kw = (1 + 0.2 * torch.randn(N, D, generator=g)).to(dtype)
    angle = torch.randn(P, rot // 2, generator=g, dtype=torch.float64) * 3
    positions = torch.randint(-2, P + 2, (N, M), generator=g)
    dq = torch.randn(N, M, Hq, D, generator=g).to(dtype)
    dk = torch.randn(N, M, Hk, D, generator=g).to(dtype)
    return q, k, qw, kw, angle.cos().float(), angle.sin().float(), positions, dq, dk


def check(device, args, dq, dk, interleaved):
    q, k, qw, kw, cos, sin, positions = args
    on = [t.to(device) for t in args]
    outs = K.qk_norm_rope(*on, EPS, interleaved)
    for x, w, out, name in ((q, qw, outs[0], "q"), (k, kw, outs[1], "k")):
        assert_within(out, *qk_side(x, w, cos, sin, positions, EPS, interleaved), name)
    grads = K.qk_norm_rope_grad(dq.to(device), dk.to(device), *on, EPS, interleaved)
    for dy, x, w, dx, dw, name in ((dq, q, qw, grads[0], grads[2], "q"),
                                   (dk, k, kw, grads[1], grads[3], "k")):
        want = qk_side_grad(dy, x, w, cos, sin, positions, EPS, interleaved)
        assert_within(dx, *want[:2], "d" + name)
        assert_within(dw, *want[2:], "d" + name + "_weight")
    return outs, grads


@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("D,rot", WIDTHS)
def test_widths(device, D, rot, dtype, interleaved):
    *args, dq, dk = inputs(2, 21, 4, 2, D, rot, dtype, 1)
    check(device, args, dq, dk, interleaved)


@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("D,rot", [(8, 8), (16, 16), (16, 0), (24, 16), (24, 8), (32, 32), (32, 16),
                                   (40, 16), (56, 32), (72, 48)])
def test_heads_of_few_packs(device, D, rot, dtype, interleaved):
    """Fewer packs than lanes, an odd number of them, heads left over."""
    *args, dq, dk = inputs(2, 133, 5, 1, D, rot, dtype, 12)
    check(device, args, dq, dk, interleaved)


@pytest.mark.parametrize("fused", [False, True])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("shape", SHAPES)
def test_shapes(device, shape, dtype, fused):
    *args, dq, dk = inputs(*shape, 64, 32, dtype, 2, fused=fused)
    check(device, args, dq, dk, False)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_many_tokens(device, dtype):
    """More tokens than one round of workgroups, so the weights' gradient is
    joined from many."""
    *args, dq, dk = inputs(2, 3001, 5, 3, 32, 32, dtype, 3)
    outs, grads = check(device, args, dq, dk, False)
    on = [t.to(device) for t in args]
    again = K.qk_norm_rope_grad(dq.to(device), dk.to(device), *on, EPS, False)
    assert all(torch.equal(a, b) for a, b in zip(grads, again))


def test_strides_shared_positions_and_table_views(device):
    q, k, qw, kw, cos, sin, positions, dq, dk = inputs(3, 11, 4, 2, 16, 8, torch.float32, 4)
    positions = positions[0]
    base = (q, k, qw, kw, cos, sin, positions.expand(3, 11))
    want = K.qk_norm_rope(*[t.to(device) for t in base], EPS, False)
    grads = K.qk_norm_rope_grad(dq.to(device), dk.to(device), *[t.to(device) for t in base], EPS,
                                False)

    def heads_first(t):  # (N, H, M, D) storage
        return t.to(device).transpose(1, 2).contiguous().transpose(1, 2)

    def columns(t):  # an innermost stride of 2
        return torch.stack([t, t], -1).flatten(-2).to(device)[..., ::2]

    both = torch.cat([cos, sin], 1).to(device)
    for move in (heads_first, columns):
        args = (move(q), move(k), columns(qw), columns(kw), both[:, :4], both[:, 4:],
                positions.to(device).int())
        for a, b in zip(K.qk_norm_rope(*args, EPS, False), want):
            assert torch.equal(a, b)
        for a, b in zip(K.qk_norm_rope_grad(move(dq), move(dk), *args, EPS, False), grads):
            assert torch.equal(a, b)
    # One replica's call, and cos and sin with rows of different strides.
    one = [t.to(device) for t in (q[1], k[1], qw[1], kw[1], cos, sin, positions)]
    one[5] = both[:, 4:]
    for a, b in zip(K.qk_norm_rope(*one, EPS, False), want):
        assert torch.equal(a, b[1])
    # A gradient that is one number, expanded.
    flat = torch.ones(1, device=device)
    got = K.qk_norm_rope_grad(flat.expand(q.shape), flat.expand(k.shape),
                              *[t.to(device) for t in base], EPS, False)
    full = K.qk_norm_rope_grad(flat.expand(q.shape).contiguous(),
                               flat.expand(k.shape).contiguous(),
                               *[t.to(device) for t in base], EPS, False)
    assert all(torch.equal(a, b) for a, b in zip(got, full))


def test_zero_heads_and_special_values(device):
    q, k, qw, kw, cos, sin, positions, dq, dk = inputs(1, 4, 2, 1, 8, 8, torch.float32, 5)
    q[0, 0] = 0
    q[0, 1, 0, 0] = float("nan")
    on = [t.to(device) for t in (q, k, qw, kw, cos, sin, positions)]
    out = K.qk_norm_rope(*on, EPS, False)
    assert not out[0][0, 0].any() and out[0][0, 1, 0].isnan().all()
    assert out[0][0, 1, 1].isfinite().all() and out[1].isfinite().all()
    grads = K.qk_norm_rope_grad(dq.to(device), dk.to(device), *on, EPS, False)
    want = qk_side_grad(dq[:, :1], q[:, :1], qw, cos, sin, positions[:, :1], EPS, False)
    assert_within(grads[0][:, :1], *want[:2])
    assert grads[1].isfinite().all() and grads[3].isfinite().all()


def test_gradient_against_differences(device):
    """The backward pass against differences of the forward one, in float32 on
    values where a step of 2^-7 leaves the truncation near its rounding."""
    q, k, qw, kw, cos, sin, positions, dq, dk = inputs(1, 2, 2, 1, 6, 4, torch.float32, 6)
    args = [t.to(device) for t in (q, k, qw, kw, cos, sin, positions)]
    dq, dk = dq.to(device), dk.to(device)
    grads = K.qk_norm_rope_grad(dq, dk, *args, EPS, True)

    def value(changed):
        a, b = K.qk_norm_rope(*changed, EPS, True)
        return (a.double() * dq).sum() + (b.double() * dk).sum()

    step = 2.0 ** -7
    for i in range(4):
        for j in range(0, args[i].numel(), 3):
            sides = []
            for sign in (1, -1):
                moved = [t.clone() for t in args]
                moved[i].view(-1)[j] += sign * step
                sides.append(value(moved))
            slope = (sides[0] - sides[1]) / (2 * step)
            # Truncation: step^2 / 6 of a third derivative, below 1e3 here;
            # rounding: 2^-24 of sums below 32, over the step.
            assert abs(slope - grads[i].view(-1)[j].double()) < 1e3 * step ** 2 / 6 + 1e-3


def test_autograd_and_vmap(device):
    q, k, qw, kw, cos, sin, positions, _, _ = inputs(3, 9, 4, 2, 16, 8, torch.float32, 7)
    cos, sin, positions = cos.to(device), sin.to(device), positions[0].to(device)
    args = [t.to(device) for t in (q, k, qw, kw)]

    def loss(q, k, qw, kw):
        a, b = K.qk_norm_rope(q, k, qw, kw, cos, sin, positions, EPS)
        return (a ** 2).sum() * 0.3 + (b ** 3).sum()

    leaves = [t.clone().requires_grad_() for t in args]
    loss(*leaves).backward()
    out = K.qk_norm_rope(*args, cos, sin, positions, EPS)
    want = K.qk_norm_rope_grad(out[0] * 0.6, 3 * out[1] ** 2, *args, cos, sin, positions, EPS)
    for leaf, w in zip(leaves, want):
        torch.testing.assert_close(leaf.grad, w)
    each = vmap(func_grad(loss, argnums=(0, 1, 2, 3)))(*args)
    for a, leaf in zip(each, leaves):
        torch.testing.assert_close(a, leaf.grad)
    # Only one of the results used.
    leaves = [t.clone().requires_grad_() for t in args]
    K.qk_norm_rope(*leaves, cos, sin, positions, EPS)[1].sum().backward()
    assert not leaves[0].grad.any() and leaves[1].grad.any()
    # A batch dimension over calls with replicas.
    stacked = [torch.stack([t, 2 * t]) for t in args[:2]]
    got = vmap(lambda q, k: K.qk_norm_rope(q, k, args[2], args[3], cos, sin, positions, EPS))(
        *stacked)
    assert torch.equal(got[0][0], out[0])
    with pytest.raises(RuntimeError, match="every replica shares"):
        vmap(lambda c: K.qk_norm_rope(*args, c, sin, positions, EPS))(torch.stack([cos, cos]))


def test_empty_sizes(device):
    q, k, qw, kw, cos, sin, positions, dq, dk = inputs(2, 0, 3, 1, 8, 4, torch.float32, 8)
    args = [t.to(device) for t in (q, k, qw, kw, cos, sin, positions)]
    assert K.qk_norm_rope(*args)[0].shape == (2, 0, 3, 8)
    grads = K.qk_norm_rope_grad(dq.to(device), dk.to(device), *args)
    assert torch.equal(grads[2].cpu(), torch.zeros(2, 8))
    assert torch.equal(grads[3].cpu(), torch.zeros(2, 8))
    none = [t[:0] for t in args[:4]] + args[4:6] + [args[6][:0]]
    assert K.qk_norm_rope(*none)[1].shape == (0, 0, 1, 8)
    # Tables without rows: nothing rotates.
    q, k, qw, kw, cos, sin, positions, dq, dk = inputs(2, 3, 3, 1, 8, 4, torch.float32, 9)
    args = [t.to(device) for t in (q, k, qw, kw, cos[:0], sin[:0], positions)]
    assert_within(K.qk_norm_rope(*args)[0],
                  *qk_side(q, qw, cos[:0], sin[:0], positions, 1e-6, False))


def test_refusals(device):
    q, k, qw, kw, cos, sin, positions, dq, dk = [
        t.to(device) for t in inputs(2, 5, 4, 2, 16, 8, torch.float32, 10)]

    def refused(match, *args):
        with pytest.raises(RuntimeError, match=match):
            K.qk_norm_rope(*args)

    refused("unsupported dtype", q.double(), k.double(), qw, kw, cos, sin, positions)
    refused("k must have dtype", q, k.half(), qw, kw, cos, sin, positions)
    refused("q_weight must have dtype", q, k, qw.half(), kw, cos, sin, positions)
    refused("q_weight must be", q, k, qw[:1], kw, cos, sin, positions)
    refused("k_weight must be", q, k, qw, kw[:, :8], cos, sin, positions)
    refused("agree but in the number of heads", q, k[:, :3], qw, kw, cos, sin, positions)
    refused("must be \\(M, H, D\\)", q, k[0], qw, kw, cos, sin, positions)
    refused("float32", q, k, qw, kw, cos.double(), sin, positions)
    refused("one shape", q, k, qw, kw, cos[:, :2], sin, positions)
    wide = torch.zeros(50, 9, device=device)
    refused("9 rotated pairs", q, k, qw, kw, wide, wide, positions)
    refused("M = 5", q, k, qw, kw, cos, sin, positions[:, :4])
    refused("int64 or int32", q, k, qw, kw, cos, sin, positions.float())
    refused("beside heads without replicas", q[0], k[0], qw[0], kw[0], cos, sin, positions)
    big = torch.zeros(1, 1, 1, 513, device=device)
    refused("1 to 512 wide", big, big, big[0, 0], big[0, 0], cos, sin, positions[:1, :1])
    refused("1 to 65535 heads", q, k[:, :, :0], qw, kw, cos, sin, positions)
    with pytest.raises(RuntimeError, match="grad_k must have the shape"):
        K.qk_norm_rope_grad(dq, dk[:, :, :1], q, k, qw, kw, cos, sin, positions)
    with pytest.raises(RuntimeError, match="grad_q must have dtype"):
        K.qk_norm_rope_grad(dq.half(), dk, q, k, qw, kw, cos, sin, positions)


@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("D,rot", [(64, 64), (64, 32), (128, 128), (96, 48), (80, 40), (48, 24),
                                   (33, 16), (33, 0), (257, 128), (24, 8)])
def test_infinities_stay_with_their_pair(device, D, rot, dtype, interleaved):
    """An infinite element makes its head's norm infinite: it becomes NaN and the
    head's other elements 0. NaN reaches another element by a rotation alone, not
    beyond ``rot`` nor at a position outside the tables."""
    N, M, H, P = 1, 2 * D, 3, 8
    g = torch.Generator().manual_seed(13)
    x = torch.randn(N, M, H, D, generator=g)
    at = torch.arange(M) % D
    x[0, torch.arange(M), 1, at] = torch.inf  # in one of the token's heads
    positions = torch.where(torch.arange(M) < D, 3, P)  # the second half: outside
    w = 1 + torch.rand(N, D, generator=g)
    angle = 0.5 + torch.rand(P, rot // 2, generator=g)
    args = [t.to(device) for t in (x.to(dtype), x[:, :, 1:].to(dtype).contiguous(), w.to(dtype),
                                   w.to(dtype), angle.cos(), angle.sin(), positions)]
    odd = torch.zeros(M, D, dtype=torch.bool)
    odd[torch.arange(M), at] = True
    partner = at ^ 1 if interleaved else (at + rot // 2) % max(rot, 1)
    turned = (at < rot) & (positions < P)
    odd[torch.arange(M)[turned], partner[turned]] = True
    for out, head in zip(K.qk_norm_rope(*args, EPS, interleaved), (1, 0)):
        out = out.float().cpu()[0, :, head]
        assert torch.equal(out.isnan(), odd) and not out[~odd].any()
    dy = torch.randn(N, M, H, D, generator=g)
    for m in range(0, M, max(1, M // 8)):  # one token at a time: one infinity
        one = [t[:, m:m + 1] for t in args[:2]] + args[2:6] + [args[6][m:m + 1]]
        dq = dy[:, m:m + 1].to(dtype).to(device)
        grads = K.qk_norm_rope_grad(dq, dq[:, :, 1:].contiguous(), *one, EPS, interleaved)
        alone = torch.arange(D) == at[m]
        for dw in grads[2:]:
            assert torch.equal(dw.cpu()[0].isnan(), alone)
        # An infinite incoming gradient: the weights' gradient of its pair.
        finite = [one[0][:, :, :1].contiguous(), one[1][:, :, 1:].contiguous(), *one[2:]]
        dq[0, 0, 0, at[m]] = torch.inf
        dq = dq[:, :, :1].contiguous()
        grads = K.qk_norm_rope_grad(dq, dq, *finite, EPS, interleaved)
        for dw in grads[2:]:
            assert torch.equal(~dw.cpu()[0].isfinite(), odd[m])
