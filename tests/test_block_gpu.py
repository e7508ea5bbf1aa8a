"""The boundary between two blocks against its definition in float64 (GPU).

A value rounded once to bf16 is off by at most half a step, 2^-8 of itself; over many
values the errors' norm is 2^-7 / sqrt(12) = 1.16 * 2^-9 of theirs where all significands
are near 1, and less where they spread. The
float32 sums before it (of at most 8192 values, statistics and the products of
the gradients) add less than 2^-15. Gradients of the update come through a
bf16 t: the same t as the definition's here, since the tests take it from the
call, so nothing else is added.
"""

from __future__ import annotations

import pytest
import torch
import torch.nn.functional as F

import representax_amd as rx
from oracle import dropout as odrop
from representax_amd import norms, ops
from tests.helpers import kernel_names

pytestmark = pytest.mark.gpu
DEV, BF16, F32, F64 = "cuda:0", torch.bfloat16, torch.float32, torch.float64
# relative to the norm of what is compared: one rounding (2^-9), or float32 sums
BOUND = {BF16: 1.25 * 2.0 ** -9, F32: 2.0 ** -17}


def _close(got, want, dtype, what):
    assert got.dtype == dtype, what
    err = (got.to(F64) - want).norm() / want.norm().clamp_min(1e-30)
    assert err <= BOUND[dtype], (what, float(err))


def _module(kind, size, dtype, seed):
    if kind is None:
        return None
    g = torch.Generator().manual_seed(seed)
    norm = (rx.LayerNorm if kind == "layer" else rx.RMSNorm)(size, 1e-6, DEV)
    for name, p in list(norm.named_parameters()):
        v = (name == "weight") + 0.3 * torch.randn(size, generator=g)
        setattr(norm, name, torch.nn.Parameter(v.to(DEV, dtype)))
    return norm


def _norm64(norm, v, dtype):
    if isinstance(norm, rx.LayerNorm):
        return F.layer_norm(v, v.shape[-1:], norm.weight.to(dtype).to(F64),
                            norm.bias.to(dtype).to(F64), norm.eps)
    return v * torch.rsqrt(v.square().mean(-1, keepdim=True) + norm.eps) * norm.weight.to(F64)


def _factor(shape, rate, key, site):
    below = odrop.threshold(rate)
    keep = odrop.kept(torch.Size(shape).numel(), *key.tolist(), site, below)
    return torch.from_numpy(keep).to(DEV, F64).view(shape) * (65536 / below)


def _check(shape, dtype, norm, post, gate, rate, scale=0.75, site=2, dt=True, dh=True,
           weight_dtype=None, seed=0):
    size = shape[-1]
    wdt = dtype if weight_dtype is None else weight_dtype
    g = torch.Generator().manual_seed(seed + size)
    draw = lambda s, m=1.0: (m * torch.randn(s, generator=g)).to(DEV, dtype)
    x, u, gt, gh = (draw(shape) for _ in range(4))
    norm, post = _module(norm, size, wdt, seed + 1), _module(post, size, wdt, seed + 2)
    gate = None if gate is None else (1 + draw(gate, 0.5)).requires_grad_(True)
    x.requires_grad_(True), u.requires_grad_(True)
    key = torch.tensor([991, 5], device=DEV)
    leaves = [x, u, *([] if gate is None else [gate])]
    for m in (norm, post):
        leaves += [] if m is None else list(m.parameters())
    t, h = rx.block_norm(norm, x, u, post=post, gate=gate, scale=scale, rate=rate, key=key,
                         site=site)
    assert type(t.grad_fn).__name__ == "BlockNormFnBackward"
    wide = {id(v): v.detach().to(F64).requires_grad_(True) for v in leaves}
    p = wide[id(u)]
    saved = {}
    for m in (norm, post):  # the modules' weights in 64 bits, as leaves
        if m is not None:
            for name, v in list(m._parameters.items()):
                saved[m, name] = v
                m._parameters[name] = None
                del m._parameters[name]
                object.__setattr__(m, name, wide[id(v)])
    if post is not None:
        p = _norm64(post, p, F64)
    if gate is not None:
        p = p * wide[id(gate)]
    if rate:
        p = p * _factor(shape, rate, key, site)
    want_t = wide[id(x)] + scale * p
    _close(t.detach(), want_t.detach(), dtype, "t")
    # h is the norm of t as it is stored
    stored = want_t + (t.detach().to(F64) - want_t.detach())
    outs, grads, outs64 = [], [], []
    if dt:
        outs, grads, outs64 = [t], [gt], [want_t]
    if norm is not None:
        want_h = _norm64(norm, stored, F64)
        _close(h.detach(), want_h.detach(), dtype, "h")
        if dh:
            outs, grads, outs64 = outs + [h], grads + [gh], outs64 + [want_h]
    else:
        assert h is None
    got = torch.autograd.grad(outs, leaves, grads, allow_unused=True)
    want = torch.autograd.grad(outs64, [wide[id(v)] for v in leaves], [v.to(F64) for v in grads],
                               allow_unused=True)
    for i, (a, b, leaf) in enumerate(zip(got, want, leaves)):
        if b is None:
            assert a is None or not a.any()
        else:
            _close(a, b, leaf.dtype, ("gradient", i))
    return x, got


# rows about the ends of each layout of lanes, odd sizes among them
@pytest.mark.parametrize("size", [1, 8, 33, 128, 129, 512, 513, 1000, 1024, 1032, 2047, 2048, 2056,
                                  4096, 4100, 8192])
@pytest.mark.parametrize("dtype", [BF16, F32])
def test_sizes(size, dtype):
    # of one value a LayerNorm keeps nothing and an RMSNorm its sign: no gradient to
    # compare behind either
    kind, post = ("rms", None) if size < 8 else ("layer", "rms")
    _check((3, 5, size), dtype, kind, post, (3, 1, size), 0.2)


@pytest.mark.parametrize("norm", ["layer", "rms", None])
@pytest.mark.parametrize("post", ["layer", "rms", None])
@pytest.mark.parametrize("gate", [None, "vector", "group", "each"])
def test_parts(norm, post, gate):
    shape = (4, 9, 264)
    gate = {None: None, "vector": (264,), "group": (4, 1, 264), "each": shape}[gate]
    _check(shape, BF16, norm, post, gate, 0.0)
    _check(shape, BF16, norm, post, gate, 0.4)


# one row, rows of one gate over several workers, many gates a worker, many rows
@pytest.mark.parametrize("shape,gate", [((1, 768), (768,)), ((1, 1, 768), (1, 1, 768)),
                                        ((2, 301, 768), (2, 1, 768)), ((37, 3, 96), (37, 1, 96)),
                                        ((613, 1, 2048), (613, 1, 2048)), ((5003, 256), (256,)),
                                        ((3, 1700, 520), (3, 1, 520)), ((9000, 104), None)])
def test_rows_and_groups(shape, gate):
    _check(shape, BF16, "layer", "layer", gate, 0.1)


def test_masters_in_float32_keep_float32_gradients():
    _check((7, 31, 320), BF16, "rms", "rms", (320,), 0.0, weight_dtype=F32)


def test_a_layer_norm_takes_its_masters_in_the_values_type():
    x, u = (torch.randn(9, 264, device=DEV).to(BF16) for _ in range(2))
    masters, views = (_module("layer", 264, F32, 3) for _ in range(2))
    with torch.no_grad():
        for p in views.parameters():
            p.copy_(p.to(BF16))
    x.requires_grad_(True)
    got, want = (rx.block_norm(m, x, u, post=m) for m in (masters, views))
    for a, b in zip(got, want):
        assert torch.equal(a, b)
    grads = [torch.autograd.grad(out, [x, *m.parameters()], (u, u))
             for out, m in ((got, masters), (want, views))]
    for a, b in zip(*grads):
        assert torch.equal(a, b) and a.dtype in (BF16, F32)


@pytest.mark.parametrize("dt,dh", [(True, False), (False, True)])
def test_one_output_used(dt, dh):
    _check((6, 40, 136), BF16, "layer", "rms", (6, 1, 136), 0.3, dt=dt, dh=dh)


def test_frozen_parts_get_no_gradient_and_no_second_launch():
    x = torch.randn(64, 768, device=DEV).to(BF16).requires_grad_(True)
    u = torch.randn_like(x)
    norm = _module("rms", 768, F32, 0).requires_grad_(False)
    t, h = rx.block_norm(norm, x, u)
    (dx,), names = kernel_names(lambda: torch.autograd.grad((t, h), x, (u, u)))
    assert any("k_block_bwd" in n for n in names) and not any("k_block_join" in n for n in names)
    (want,) = torch.autograd.grad(rx.add_norm(norm, x, u), x, (u, u))
    _close(dx, want.to(F64), BF16, "dx")
    with torch.no_grad():
        out, names = kernel_names(lambda: rx.block_norm(norm, x, u))
    assert sum("k_block_fwd" in n for n in names) == 1
    assert torch.equal(out[0], t) and torch.equal(out[1], h)


def test_the_fused_call_has_the_bits_of_its_steps():
    """Sums, gates of one and dropout alone: the same roundings as separate calls."""

    x, u = (torch.randn(17, 333, device=DEV).to(BF16) for _ in range(2))
    key = torch.tensor([5, 6], device=DEV)
    t, _ = rx.block_norm(None, x, u, rate=0.35, key=key, site=8)
    factor = _factor(x.shape, 0.35, key, 8).float()
    assert torch.equal(t, (x.float() + u.float() * factor).to(BF16))


def test_the_same_bits_every_time():
    shape = (4, 700, 768)
    args = (shape, BF16, "layer", "layer", (4, 1, 768), 0.1)
    first, second = _check(*args)[1], _check(*args)[1]
    assert all(torch.equal(a, b) for a, b in zip(first, second))


def test_rows_of_nan_stay_in_their_row():
    x, u = (torch.randn(40, 512, device=DEV).to(BF16) for _ in range(2))
    norm = _module("layer", 512, BF16, 3)
    x[7, 3], u[9, 100] = float("nan"), float("inf")
    x.requires_grad_(True)
    t, h = rx.block_norm(norm, x, u, post=_module("rms", 512, BF16, 4))
    (dx,) = torch.autograd.grad((t, h), x, (u.nan_to_num(0, 0, 0),) * 2)
    rest = [i for i in range(40) if i not in (7, 9)]
    for v in (t, h, dx):
        assert torch.isfinite(v[rest]).all()
    assert torch.isnan(h[7]).all() and torch.isnan(h[9]).all()


def test_views_and_offsets():
    base = torch.randn(4, 6, 1003, device=DEV).to(BF16)
    x, u = base[:, 1:4, 1:1001], base.flip(0)[:, 2:5, 2:1002]
    norm = _module("rms", 1000, BF16, 0)
    flat = torch.randn(1001, device=DEV).to(BF16)
    norm.weight = torch.nn.Parameter(flat[1:])  # two bytes past an aligned address
    t, h = rx.block_norm(norm, x, u, gate=flat[:1000])
    want = x.to(F64) + u.to(F64) * flat[:1000].to(F64)
    _close(t.detach(), want, BF16, "t")
    _close(h.detach(), _norm64(norm, t.detach().to(F64), BF16), BF16, "h")


def test_calls_that_take_the_expressions():
    norm = _module("rms", 16, F32, 0)
    x = torch.randn(3, 16, device=DEV)
    for value in (x.half(), x.double()):
        t, _ = rx.block_norm(norm, value, value)
        assert t.dtype == value.dtype
    wide = torch.randn(2, 8200, device=DEV)
    t, h = rx.block_norm(_module("rms", 8200, F32, 0), wide, wide)
    _close(t.detach(), 2 * wide.to(F64), F32, "t")
    t, h = rx.block_norm(norm, x[:0], x[:0])
    assert t.shape == (0, 16)
    gate = torch.randn(3, 16, device=DEV)
    value = torch.randn(2, 3, 16, device=DEV)
    t, _ = rx.block_norm(norm, value, value, gate=gate)
    _close(t.detach(), (value + value * gate).to(F64), F32, "t")


def test_second_derivatives():
    norm = _module("rms", 24, F32, 1)
    x, u = (torch.randn(5, 24, device=DEV, requires_grad=True) for _ in range(2))
    key = torch.tensor([1, 2], device=DEV)

    def loss(xx, uu, n, dtype):
        t, h = rx.block_norm(n, xx, uu, post=n, rate=0.2, key=key)
        return (h ** 3).sum() + (t ** 2).sum()

    grads = torch.autograd.grad(loss(x, u, norm, F32), (x, u), create_graph=True)
    got = torch.autograd.grad(sum((v ** 2).sum() for v in grads), (x, u))
    x64, u64 = x.detach().double().requires_grad_(True), u.detach().double().requires_grad_(True)
    n64 = _module("rms", 24, F64, 1)
    with torch.no_grad():
        n64.weight.copy_(norm.weight)
    grads = torch.autograd.grad(loss(x64, u64, n64, F64), (x64, u64), create_graph=True)
    want = torch.autograd.grad(sum((v ** 2).sum() for v in grads), (x64, u64))
    for a, b in zip(got, want):
        assert (a.to(F64) - b).norm() / b.norm() < 1e-4


def test_captured_and_replayed_on_another_stream():
    shape = (2, 150, 768)
    norm, post = _module("layer", 768, BF16, 1), _module("rms", 768, BF16, 2)
    x, u, dt, dh = (torch.randn(shape, device=DEV).to(BF16) for _ in range(4))
    gate = torch.randn(2, 1, 768, device=DEV).to(BF16).requires_grad_(True)
    x.requires_grad_(True), u.requires_grad_(True)
    leaves = [x, u, gate, *norm.parameters(), *post.parameters()]
    keys = rx.DropoutKeys(5, DEV)

    def step():
        key = keys.next()
        t, h = rx.block_norm(norm, x, u, post=post, gate=gate, rate=0.1, key=key, site=1)
        grads = torch.autograd.grad((t, h), leaves, (dt, dh))
        return key, [t.detach(), h.detach(), *grads]

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        key, outs = step()
    for _ in range(3):
        with torch.no_grad():
            x.add_(0.125)
        graph.replay()
        torch.cuda.synchronize()
        t, h = rx.block_norm(norm, x, u, post=post, gate=gate, rate=0.1, key=key.clone(), site=1)
        want = [t.detach(), h.detach(), *torch.autograd.grad((t, h), leaves, (dt, dh))]
        for a, b in zip(outs, want):
            assert torch.equal(a, b)


def test_a_changed_key_or_update_is_noticed():
    x, u = (torch.randn(4, 64, device=DEV, requires_grad=True) for _ in range(2))
    key = torch.tensor([1, 2], device=DEV)
    t, _ = rx.block_norm(_module("rms", 64, F32, 1), x, u, rate=0.5, key=key)
    key.add_(1)
    with pytest.raises(RuntimeError, match="modified by an inplace"):
        t.sum().backward()


def test_workspaces_are_released():
    _check((2, 64, 768), BF16, "layer", None, None, 0.0)
    ops.release_workspaces()
    assert norms.block_norm is rx.block_norm
