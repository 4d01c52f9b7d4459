"""What the language-model operators share: the C ABI's exports and refusals,
schemas and fake kernels, graph capture, other streams, torch.compile, offsets
past 32 bits, and the example that runs them together."""

from __future__ import annotations

import ctypes
import importlib.util
import re
from pathlib import Path

import pytest
import torch

from churten_amd import kernels as K
from lm_reference import assert_within, distill, qk_side

ROOT = Path(__file__).resolve().parents[1]
HEADER = ROOT / "include" / "churten_lm.h"
DEVICES = ["cpu", pytest.param("cuda", marks=pytest.mark.gpu)]


def declared():
    return sorted(set(re.findall(r"^(?:int|size_t)\s+(ts_\w+)\s*\(", HEADER.read_text(),
                                 flags=re.M)))


def library():
    lib = ctypes.CDLL(str(ROOT / "churten_amd" / "lib" / "libchurten_optim.so"))
    for name in declared():
        if name.endswith("_workspace"):
            getattr(lib, name).restype = ctypes.c_size_t
    return lib


class Rows(ctypes.Structure):
    _fields_ = [("data", ctypes.c_void_p), ("stride_n", ctypes.c_int64),
                ("stride_b", ctypes.c_int64)]


class Index(ctypes.Structure):
    _fields_ = [("data", ctypes.c_void_p), ("stride_n", ctypes.c_int64),
                ("stride_b", ctypes.c_int64), ("bits", ctypes.c_int)]


class Heads(ctypes.Structure):
    _fields_ = [("data", ctypes.c_void_p), ("stride_n", ctypes.c_int64),
                ("stride_m", ctypes.c_int64), ("stride_h", ctypes.c_int64)]


class QkShape(ctypes.Structure):
    _fields_ = [(n, ctypes.c_int64) for n in ("N", "M", "Hq", "Hk", "D", "rot", "P")] + [
        ("cos", ctypes.c_void_p), ("sin", ctypes.c_void_p), ("table_stride", ctypes.c_int64),
        ("positions", Index), ("eps", ctypes.c_float), ("flags", ctypes.c_uint32)]


class Distill(ctypes.Structure):
    _fields_ = [(n, ctypes.c_int64) for n in ("N", "B", "V", "K")] + [
        ("logits", Rows), ("teacher", Rows), ("index", Index), ("temperature", ctypes.c_void_p),
        ("hard", ctypes.c_void_p), ("labels", Index), ("weight", ctypes.c_void_p),
        ("weight_stride_n", ctypes.c_int64), ("weight_stride_b", ctypes.c_int64),
        ("loss", ctypes.c_void_p), ("grad", Rows)]


P = 4096  # an address that is never read: every call here is refused on the host
I64 = ctypes.c_int64


def test_the_library_exports_every_declared_entry_point():
    lib = library()
    assert declared() == sorted([
        "ts_embedding", "ts_embedding_grad", "ts_embedding_grad_workspace", "ts_qk_norm_rope",
        "ts_qk_norm_rope_grad", "ts_qk_norm_rope_grad_workspace", "ts_distill",
        "ts_distill_workspace"])
    for name in declared():
        assert hasattr(lib, name), name


def test_embedding_refuses_bad_arguments_before_any_launch():
    lib = library()
    rows, index = Rows(P, 1, 1), Index(P, 1, 1, 64)

    def lookup(weight=rows, tokens=index, out=rows, dtype=0, N=1, B=1, V=1, D=1):
        return lib.ts_embedding(weight, tokens, out, dtype, I64(N), I64(B), I64(V), I64(D),
                                ctypes.c_float(1), None)

    none = Rows(None, 1, 1)
    assert lookup(dtype=1) == 1 and lookup(dtype=9) == 1
    assert lookup(N=-1) == 1 and lookup(N=65536) == 1 and lookup(B=-1) == 1
    assert lookup(V=2 ** 31) == 1 and lookup(D=2 ** 31) == 1 and lookup(B=2 ** 31) == 1
    assert lookup(weight=none) == 1 and lookup(out=none) == 1
    assert lookup(tokens=Index(P, 1, 1, 16)) == 1 and lookup(tokens=Index(None, 1, 1, 64)) == 1
    assert lookup(weight=none, B=0) == 0 and lookup(weight=none, N=0) == 0

    size = lib.ts_embedding_grad_workspace(0, I64(2), I64(5000), I64(100), I64(8), 0)
    assert size > 0
    assert lib.ts_embedding_grad_workspace(0, I64(2), I64(5000), I64(100), I64(8), 1) < size
    assert lib.ts_embedding_grad_workspace(0, I64(2), I64(-1), I64(100), I64(8), 0) == 0

    def grad(ws=P, given=size, flags=0, dtype=0, out=rows, g=rows, tokens=index, B=5000):
        return lib.ts_embedding_grad(out, g, tokens, dtype, I64(2), I64(B), I64(100), I64(8),
                                     ctypes.c_float(1), flags, ws, ctypes.c_size_t(given), None)

    assert grad(ws=None) == 1 and grad(given=size - 1) == 1 and grad(ws=P + 8) == 1
    assert grad(flags=2) == 1 and grad(dtype=1) == 1 and grad(B=-1) == 1
    assert grad(out=none) == 1 and grad(g=none) == 1 and grad(tokens=Index(P, 1, 1, 8)) == 1
    assert grad(flags=1, B=0, out=none) == 0


def test_qk_norm_rope_refuses_bad_arguments_before_any_launch():
    lib = library()

    def shape(**kw):
        base = dict(N=2, M=4000, Hq=4, Hk=2, D=64, rot=64, P=10, cos=P, sin=P, table_stride=32,
                    positions=Index(P, 1, 1, 64), eps=1e-6, flags=0)
        return QkShape(**{**base, **kw})

    heads, none = Heads(P, 1, 1, 1), Heads(None, 1, 1, 1)

    def forward(s, q=heads, w=P, dtype=0):
        return lib.ts_qk_norm_rope(ctypes.byref(s), dtype, q, heads, w, I64(64), P, I64(64),
                                   heads, heads, None)

    for bad in (dict(N=-1), dict(N=65536), dict(M=-1), dict(M=2 ** 31), dict(Hq=0), dict(Hk=0),
                dict(Hq=65536), dict(D=0), dict(D=513), dict(rot=65), dict(rot=63), dict(rot=-2),
                dict(P=-1), dict(flags=1), dict(cos=None), dict(positions=Index(P, 1, 1, 0)),
                dict(positions=Index(None, 1, 1, 64))):
        assert forward(shape(**bad)) == 1, bad
        assert lib.ts_qk_norm_rope_grad_workspace(ctypes.byref(shape(**bad)), 0) == 0, bad
    assert lib.ts_qk_norm_rope(None, 0, heads, heads, P, I64(1), P, I64(1), heads, heads,
                               None) == 1
    assert forward(shape(), dtype=1) == 1 and forward(shape(), q=none) == 1
    assert forward(shape(), w=None) == 1
    assert forward(shape(M=0), q=none) == 0 and forward(shape(N=0)) == 0

    s = shape()
    size = lib.ts_qk_norm_rope_grad_workspace(ctypes.byref(s), 0)
    assert size > 0

    def backward(ws=P, given=size, dq=heads, wg=P):
        return lib.ts_qk_norm_rope_grad(ctypes.byref(s), 0, dq, heads, heads, heads, P, I64(64),
                                        P, I64(64), heads, heads, wg, P, ws,
                                        ctypes.c_size_t(given), None)

    assert backward(ws=None) == 1 and backward(given=size - 1) == 1 and backward(ws=P + 4) == 1
    assert backward(dq=none) == 1 and backward(wg=None) == 1


def test_distill_refuses_bad_arguments_before_any_launch():
    lib = library()
    rows, index = Rows(P, 1, 1), Index(P, 1, 1, 64)

    def call(dtype=0, ws=P, given=1 << 30, **kw):
        base = dict(N=1, B=2, V=100000, K=4, logits=rows, teacher=rows, index=index,
                    temperature=P, hard=None, labels=Index(None, 0, 0, 0), weight=None, loss=P,
                    grad=rows)
        a = Distill(**{**base, **kw})
        return lib.ts_distill(ctypes.byref(a), dtype, ws, ctypes.c_size_t(given), None)

    none = Rows(None, 1, 1)
    for bad in (dict(N=-1), dict(N=65536), dict(B=-1), dict(V=-1), dict(V=2 ** 31), dict(K=-1),
                dict(K=1025), dict(logits=none), dict(teacher=none), dict(loss=None),
                dict(index=Index(P, 1, 1, 3)), dict(temperature=None), dict(hard=P),
                dict(labels=index), dict(hard=P, labels=Index(P, 1, 1, 5)), dict(dtype=1),
                dict(ws=None), dict(given=16), dict(ws=P + 4)):
        assert call(**bad) == 1, bad
    assert lib.ts_distill(None, 0, P, ctypes.c_size_t(0), None) == 1
    assert call(N=0, loss=None) == 0 and call(B=0, logits=none) == 0


def small_calls(device):
    """One small call of each operator: (operator, arguments)."""
    g = torch.Generator().manual_seed(3)

    def real(*shape):
        return torch.randn(*shape, generator=g).to(device)

    def whole(high, *shape):
        return torch.randint(0, high, shape, generator=g).to(device)

    ops = torch.ops.churten
    q, k, cos, sin = real(2, 5, 4, 8), real(2, 5, 2, 8), real(9, 3), real(9, 3)
    positions = whole(9, 2, 5)
    rest = (real(2, 8), real(2, 8), cos, sin, positions, 1e-6, False)
    row = (real(2, 6, 50), real(2, 6, 4), whole(50, 2, 6, 4), torch.tensor([1.0, 2.0]).to(device),
           torch.rand(2, 6, generator=g).to(device), whole(50, 2, 6),
           torch.tensor([0.2, 0.4]).to(device))
    return [(ops.embedding, (real(2, 11, 6), whole(11, 2, 7), 2.0)),
            (ops.embedding_grad, (real(2, 7, 6), whole(11, 2, 7), 11, 2.0)),
            (ops.embedding_grad_, (real(2, 11, 6), real(2, 7, 6), whole(11, 2, 7), 2.0, True)),
            (ops.qk_norm_rope, (q, k, *rest)),
            (ops.qk_norm_rope_grad, (real(2, 5, 4, 8), real(2, 5, 2, 8), q, k, *rest)),
            (ops.distill_loss, row), (ops.distill_loss_grad, row)]


@pytest.mark.parametrize("device", DEVICES)
def test_schemas_and_fake_kernels(device):
    for op, args in small_calls(device):
        torch.library.opcheck(op, args, test_utils=("test_schema", "test_faketensor"))


@pytest.mark.parametrize("device", DEVICES)
def test_compiled_calls(device):
    calls = dict(zip("lookup lg lgi qk qkg loss lossg".split(), small_calls(device)))
    weight, tokens, scale = calls["lookup"][1]
    args = calls["qk"][1]
    row = calls["loss"][1]

    def step(weight, q, logits):
        a = K.embedding(weight, tokens, scale)
        q, k = K.qk_norm_rope(q, *args[1:])
        return a.square().sum() + q.sum() + k.square().sum() + K.distill_loss(
            logits, *row[1:]).sum()

    leaves = [t.clone().requires_grad_() for t in (weight, args[0], row[0])]
    step(*leaves).backward()
    compiled = torch.compile(step, backend="aot_eager", fullgraph=True)
    again = [t.clone().requires_grad_() for t in (weight, args[0], row[0])]
    compiled(*again).backward()
    for a, b in zip(leaves, again):
        torch.testing.assert_close(a.grad, b.grad)


def captured_calls():
    """Calls of every launch sequence, on inputs that a test refills."""
    g = torch.Generator(device="cuda").manual_seed(5)

    def real(*shape, dtype=torch.float32):
        return torch.randn(*shape, generator=g, device="cuda", dtype=dtype)

    def whole(high, *shape):
        return torch.randint(0, high, shape, generator=g, device="cuda")

    few, tile, many = whole(70, 2, 90), whole(70, 2, 900), whole(700, 2, 20000)
    cos, sin, positions = real(64, 16), real(64, 16), whole(64, 2, 700)
    rest = (real(2, 32), real(2, 32), cos, sin, positions, 1e-6, False)
    t = torch.tensor([1.0, 2.0], device="cuda")

    def rows(B, V, dtype):
        return real(2, B, V, dtype=dtype), real(2, B, 8), whole(V, 2, B, 8), t

    return [(K.embedding, [real(2, 70, 24), tile]),
            (K.embedding_grad, [real(2, 90, 24), few, 70]),
            (K.embedding_grad, [real(2, 900, 24), tile, 70]),
            (K.embedding_grad, [real(2, 20000, 24), many, 700]),
            (K.qk_norm_rope, [real(2, 700, 4, 32), real(2, 700, 2, 32), *rest]),
            (K.qk_norm_rope_grad, [real(2, 700, 4, 32), real(2, 700, 2, 32),
                                   real(2, 700, 4, 32), real(2, 700, 2, 32), *rest]),
            (K.distill_loss, list(rows(40, 3000, torch.float32))),
            (K.distill_loss_grad, list(rows(40, 3000, torch.bfloat16))),
            (K.distill_loss_grad, list(rows(3, 40000, torch.float32)))]


def outputs(result):
    return [result] if isinstance(result, torch.Tensor) else list(result)


@pytest.mark.gpu
def test_graph_replays_equal_the_eager_calls():
    calls = captured_calls()
    for call, args in calls:
        call(*args)  # the allocator's and the library's first calls
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = [outputs(call(*args)) for call, args in calls]
    for turn in range(4):
        for call, args in calls:  # other inputs, in place
            args[0].normal_()
        eager = [[t.clone() for t in outputs(call(*args))] for call, args in calls]
        graph.replay()
        torch.cuda.synchronize()
        for want, got in zip(eager, held):
            for a, b in zip(want, got):
                assert torch.equal(a, b), turn


@pytest.mark.gpu
def test_calls_run_on_the_current_stream():
    calls = captured_calls()
    want = [[t.clone() for t in outputs(call(*args))] for call, args in calls]
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        for (call, args), expected in zip(calls, want):
            copy = [a.clone() if isinstance(a, torch.Tensor) else a for a in args]
            for a, b in zip(outputs(call(*copy)), expected):
                assert torch.equal(a, b)
    side.synchronize()


@pytest.mark.gpu
def test_offsets_past_32_bits():
    V = 131072
    logits = torch.zeros(1, 16500, V, device="cuda", dtype=torch.bfloat16)
    g = torch.Generator(device="cuda").manual_seed(6)
    logits[0, -2:] = torch.randn(2, V, generator=g, device="cuda")
    z = torch.randn(1, 16500, 4, generator=g, device="cuda")
    index = torch.randint(0, V, (1, 16500, 4), generator=g, device="cuda")
    t = torch.tensor([1.5], device="cuda")
    loss, grad = K.distill_loss_grad(logits, z, index, t)
    for at in (slice(0, 2), slice(16498, 16500)):
        want = distill(logits[:, at].cpu(), z[:, at].cpu(), index[:, at].cpu(), t.cpu())
        assert_within(loss[:, at], want[0], want[1])
        assert_within(grad[:, at], want[2], want[3])
    assert torch.equal(K.distill_loss(logits, z, index, t)[0, :16498],
                       K.distill_loss(logits[:, :16498], z[:, :16498], index[:, :16498], t)[0])
    del logits, grad
    x = torch.zeros(1, 140000, 128, 128, device="cuda", dtype=torch.bfloat16)
    x[0, -1] = torch.randn(128, 128, generator=g, device="cuda")
    w = torch.ones(1, 128, device="cuda", dtype=torch.bfloat16)
    angle = torch.randn(20, 64, generator=g, device="cuda")
    positions = torch.full((140000,), 7, device="cuda")
    q, _ = K.qk_norm_rope(x, x[:, :, :1], w, w, angle.cos(), angle.sin(), positions)
    want = qk_side(x[:, -1:].cpu(), w.cpu(), angle.cos().cpu(), angle.sin().cpu(),
                   positions[None, -1:].cpu(), 1e-6, False)
    assert_within(q[:, -1:], *want)
    assert not q[:, :-1].any()


@pytest.mark.parametrize("device", DEVICES)
def test_the_example_trains_an_ensemble(device):
    spec = importlib.util.spec_from_file_location("ensemble_lm",
                                                  ROOT / "examples" / "ensemble_lm.py")
    example = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(example)
    state, losses = example.train(steps=12, device=device, replicas=3, vocabulary=40, width=32,
                                  heads=2, kv_heads=1, layers=1, count=4, length=16, top=8)
    assert losses.shape == (12, 3) and losses.isfinite().all()
    assert (losses[10:, :2].mean(0) < 0.8 * losses[0, :2]).all()
    assert not losses[6:, 2].any()  # frozen: no row has weight
    assert state.optimizer_state["state_steps"].tolist() == [12, 12, 6]


@pytest.mark.parametrize("device", DEVICES)
def test_the_examples_gradients_are_those_of_plain_operations(device):
    spec = importlib.util.spec_from_file_location("ensemble_lm",
                                                  ROOT / "examples" / "ensemble_lm.py")
    example = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(example)
    torch.manual_seed(1)
    model = example.Decoder(30, 16, 2, 1, 1).to(device)
    cos, sin = example.rotation(6, 8, device)
    tokens = torch.randint(0, 30, (2, 6)).to(device)
    z, index = torch.randn(12, 5).to(device), torch.randint(0, 30, (12, 5)).to(device)
    t = torch.tensor([1.5], device=device)

    def plain_qk(q, k, q_weight, k_weight, cos, sin, positions, eps=1e-6):
        def one(x, w):
            y = x * (x.square().mean(-1, keepdim=True) + eps).rsqrt() * w
            a, b = y.chunk(2, -1)
            c, s = cos[positions][:, None], sin[positions][:, None]
            return torch.cat([a * c - b * s, b * c + a * s], -1)

        return one(q, q_weight), one(k, k_weight)

    def plain_distill(x, z, index, t):
        p, log_p = (z / t).softmax(-1), (z / t).log_softmax(-1)
        log_q = (x / t).log_softmax(-1).gather(-1, index)
        return t * t * (p * (log_p - log_q)).sum(-1)

    K.distill_loss(model(tokens, cos, sin), z, index, t).sum().backward()
    got = {name: p.grad.clone() for name, p in model.named_parameters()}
    model.zero_grad()
    kernels, example.K = example.K, type("Plain", (), {
        "embedding": staticmethod(lambda w, ids, scale: w[ids] * scale),
        "qk_norm_rope": staticmethod(plain_qk)})
    try:
        plain_distill(model(tokens, cos, sin), z, index, t).sum().backward()
    finally:
        example.K = kernels
    for name, p in model.named_parameters():
        # float32 both ways; a dozen layers of operations on values near 1.
        torch.testing.assert_close(got[name], p.grad, rtol=2e-4, atol=2e-5)


def test_a_gradient_too_large_for_its_launches_is_refused_before_any():
    """No launch has 2^24 workgroups or more, and none is made of a call of which a
    later one would: nothing is written, and without a GPU nothing else fails."""
    lib = library()
    most = 2 ** 31 - 2
    rows = Rows(P, 1, 1)

    def call(N, B, V, D, shared, flags=0):
        size = lib.ts_embedding_grad_workspace(0, I64(N), I64(B), I64(V), I64(D), shared)
        assert size > 0
        index = Index(P, 0 if shared else B, 1, 64)
        return lib.ts_embedding_grad(rows, rows, index, 0, I64(N), I64(B), I64(V), I64(D),
                                     ctypes.c_float(1), flags, P, ctypes.c_size_t(size), None)

    assert call(1, most, 100, 8, False) == 1  # joining its chunks
    assert call(1, most, 100, 8, False, 1) == 1
    assert call(16, 2 ** 29, 100, 8, False) == 1  # merging its lists
    assert call(64, 300, most, 1, True) == 1  # zeroing its rows, without a merge
    assert call(64, 9000, most, 1, True) == 1  # and beside one


@pytest.mark.gpu
def test_graph_replays_follow_the_tokens():
    """Every launch sequence of the embedding, with other tokens, tables and
    incoming gradients at each replay."""
    g = torch.Generator(device="cuda").manual_seed(7)
    V = 3000
    calls = []
    for B in (90, 900, 5000, 20000, 40000, 70000):
        for lead in ((2,), ()):  # a list for each replica, and one for both
            tokens = torch.randint(-1, V + 1, (*lead, B), generator=g, device="cuda")
            grad = torch.randn(2, B, 6, generator=g, device="cuda")
            into = torch.zeros(2, V, 6, device="cuda")
            calls.append((K.embedding_grad, [grad, tokens, V]))
            calls.append((lambda o, g, t: K.embedding_grad_(o, g, t) or o, [into, grad, tokens]))
    calls.append((K.embedding, [torch.randn(2, V, 6, device="cuda"), tokens]))
    for call, args in calls:
        call(*args)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = [call(*args) for call, args in calls]
    for turn in range(4):
        for call, args in calls:
            for t in args:
                if isinstance(t, torch.Tensor) and t.is_floating_point():
                    t.normal_()
                elif isinstance(t, torch.Tensor):
                    t.random_(-1, (V, 20, V + 5, 1)[turn])
        eager = [call(*args).clone() for call, args in calls]
        for _, args in calls:
            if len(args) == 3 and isinstance(args[2], torch.Tensor):
                args[0].fill_(float("nan"))
        graph.replay()
        torch.cuda.synchronize()
        for want, got in zip(eager, held):
            assert torch.equal(want, got), turn
