"""Adapters of many requests against their definition in float64 (GPU).

One rounding to bf16 is off by at most 2^-8 of a value; over many values of spread
significands x in [1, 2) its norm is 2^-7 / sqrt(12) against sqrt(mean x^2) = sqrt(7 / 3),
2^-9.4 of theirs: STEP = 2^-9 a rounding. y, dx: one rounding of float32 sums, on top of
the rounding of h (dh) to bf16, whose independent errors of 2^-9 each enter the
adapter's term, a part of y, as a norm does: together at most 2^-9 (1 + 1) where the
adapter's term is as large as y (the tests' scalings make it about that). The calls that add the term to a base product already rounded (or
round that base first) add one rounding of each: 2^-9 (1 + 1 + 1) in all. dA, dB: sums
of products with h or dh: 2^-9 (1 + 1) with bf16 gradients, 2^-9 with float32 ones.
"""

from __future__ import annotations

import threading

import pytest
import torch

import representax_amd as rx
from oracle import dropout as odrop
from representax_amd import _native as nat
from representax_amd import bank, ops
from representax_amd.bank import AdapterPlan
from representax_amd.trainstep import BertConfig, build_int4lora_encoder
from tests.helpers import kernel_names

pytestmark = pytest.mark.gpu
DEV, BF16, F32, F64 = "cuda:0", torch.bfloat16, torch.float32, torch.float64
STEP = 2.0 ** -9


def _err(got, want):
    return float((got.to(F64) - want).norm() / want.norm().clamp_min(1e-30))


def _weight(n, k, group, g):
    packed = torch.randint(0, 256, (n, (k + 1) // 2), generator=g, dtype=torch.int32)
    if k % 2:
        packed[:, -1] &= 15
    scales = (0.01 + 0.02 * torch.rand((n, k // group if group else 1), generator=g)).to(BF16)
    low, high = packed & 15, packed >> 4
    q = torch.stack((low, high), 2).view(n, -1)[:, :k]
    q = (q - 16 * (q > 7)).to(F64)
    w = (q.view(n, scales.shape[1], -1) * scales.to(F64)[..., None]).view(n, k)
    bits = scales.view(torch.int16).view(torch.uint16).to(DEV)
    return packed.to(torch.uint8).to(DEV), bits, w.to(BF16).to(DEV, F64)


class Case:
    def __init__(self, m, k, n, rank, adapters, index, *, group=None, bias=False, rate=0.0,
                 master=BF16, seed=0):
        g = torch.Generator().manual_seed(seed + m + k + n)
        self.packed, self.scales, self.w = _weight(n, k, group, g)
        draw = lambda *s: torch.randn(s, generator=g)
        self.x = draw(m, k).to(DEV, BF16)
        self.dy = draw(m, n).to(DEV, BF16)
        self.a = (draw(adapters, rank, k) * k ** -0.5).to(DEV, master)
        self.b = (draw(adapters, n, rank) * (0.1 * k / rank) ** 0.5).to(DEV, master)
        self.s = (0.5 + torch.rand(adapters, generator=g)).to(DEV)
        self.bias = draw(n).to(DEV, BF16) if bias else None
        if index == "rows":
            self.index = torch.randint(-1, adapters, (m,), generator=g, dtype=torch.int32)
        elif index == "runs":
            ends = torch.randint(0, m, (max(1, m // 40),), generator=g)
            self.index = torch.randint(-1, adapters, (m + 1,), generator=g, dtype=torch.int32)[
                torch.bucketize(torch.arange(m), ends.sort().values)]
        else:
            self.index = torch.full((m,), int(index), dtype=torch.int32)
        self.index = self.index.to(DEV)
        self.plan = rx.adapter_plan(self.index, adapters)
        self.key = torch.tensor([123456789, 17], device=DEV)
        self.group, self.rate, self.adapters = group, rate, adapters

    def call(self, x=None, a=None, b=None, plan=None):
        return rx.bank_linear(self.x if x is None else x, self.packed, self.scales,
                              self.a if a is None else a, self.b if b is None else b, self.s,
                              plan or self.plan, group_size=self.group, bias=self.bias,
                              rate=self.rate, key=self.key, site=6)

    def train(self):
        leaves = [t.detach().clone().requires_grad_(True) for t in (self.x, self.a, self.b)]
        y = self.call(*leaves)
        return [y.detach(), *torch.autograd.grad(y, leaves, self.dy)]

    def want(self):
        """y, dx, dA and dB in float64."""

        x, dy = self.x.to(F64), self.dy.to(F64)
        a, b = self.a.to(BF16).to(F64), self.b.to(BF16).to(F64)
        factor = torch.ones_like(x)
        if self.rate:
            below = odrop.threshold(self.rate)
            keep = odrop.kept(x.numel(), *self.key.tolist(), 6, below)
            factor = torch.from_numpy(keep).to(DEV, F64).view(x.shape) * (65536 / below)
        xd = x * factor
        y = x @ self.w.t()
        if self.bias is not None:
            y = y + self.bias.to(F64)
        dx, da, db = dy @ self.w, torch.zeros_like(a), torch.zeros_like(b)
        for e in range(self.adapters):
            at = (self.index == e).nonzero().view(-1)
            s, h = float(self.s[e]), xd[at] @ a[e].t()
            dh = dy[at] @ b[e]
            y[at] += s * (h @ b[e].t())
            dx[at] += s * (dh @ a[e]) * factor[at]
            da[e], db[e] = s * (dh.t() @ xd[at]), s * (dy[at].t() @ h)
        return y, dx, da, db

    def check(self):
        y, dx, da, db = self.want()
        assert _err(self.call(), y) <= 3 * STEP
        got = self.train()
        assert _err(got[0], y) <= 3 * STEP and _err(got[1], dx) <= 3 * STEP
        for t, want, leaf in ((got[2], da, self.a), (got[3], db, self.b)):
            assert t.dtype == leaf.dtype
            assert _err(t, want) <= 2 * STEP
        empty = [e for e in range(self.adapters) if not (self.index == e).any()]
        assert not got[2][empty].any() and not got[3][empty].any()


# rows about the ends of the tiles and of the few-row kernels
@pytest.mark.parametrize("m", [1, 2, 4, 5, 16, 17, 33, 64, 65, 130, 333, 1024, 1025])
@pytest.mark.parametrize("index", ["rows", "runs"])
def test_rows(m, index):
    Case(m, 256, 192, 16, 5, index, group=64, bias=m % 2 == 0).check()


@pytest.mark.parametrize("m", [3, 40, 200, 1100])
@pytest.mark.parametrize("rank", [1, 4, 8, 12, 16, 24, 32, 33, 48, 64])
def test_ranks(m, rank):
    Case(m, 128, 136, rank, 3, "rows").check()


# whole and ragged slices of K, columns that end inside a tile, odd sizes
@pytest.mark.parametrize("m", [2, 100])
@pytest.mark.parametrize("k,n,group", [(64, 8, None), (192, 1000, 32), (2048, 72, 64),
                                       (96, 200, 32), (100, 33, None), (77, 41, None),
                                       (320, 17, 20), (1088, 264, 64)])
def test_shapes(m, k, n, group):
    Case(m, k, n, 8, 4, "rows", group=group, bias=True).check()


@pytest.mark.parametrize("m,rank", [(300, 8), (1100, 8), (1100, 40)])
def test_more_groups_than_a_tile_keeps(m, rank):
    """1024 scales a row."""

    Case(m, 32768, 72, rank, 3, "rows", group=32, bias=True).check()


# the ends of slices, stages and columns of up to 1024 rows
@pytest.mark.parametrize("m", [16, 17, 64, 65, 321])
@pytest.mark.parametrize("k,n,group", [(32, 33, None), (160, 131, 32), (288, 3, None),
                                       (2080, 129, None), (4128, 257, None)])
def test_few_rows_of_odd_columns(m, k, n, group):
    Case(m, k, n, 12, 4, "rows", group=group, bias=True, rate=0.2).check()


# one tile a CU of 64 and of 128 rows, and more
@pytest.mark.parametrize("m", [257, 700, 1300, 1500])
def test_tiles_of_a_few_hundred_rows(m):
    Case(m, 1024, 2056, 16, 5, "runs", group=32).check()


@pytest.mark.parametrize("m,k,n", [(1, 256, 64), (50, 256, 72), (300, 256, 64), (90, 77, 30),
                                   (4500, 256, 128)])
def test_dropout(m, k, n):
    Case(m, k, n, 16, 3, "runs", rate=0.3).check()


def test_many_rows_and_adapters():
    Case(5000, 256, 320, 16, 3, "runs", group=64).check()
    Case(4097, 128, 128, 32, 700, "rows").check()
    Case(700, 128, 64, 8, 1024, "rows").check()


@pytest.mark.parametrize("tile", [0, 18, 19])
@pytest.mark.parametrize("rank", [5, 8, 16, 24, 32])
@pytest.mark.parametrize("index", ["rows", "runs"])
def test_dropout_in_every_product(tile, rank, index):
    """The planners' tiles for these sizes, and both of the large products'."""

    case = Case(1100, 512, 456, rank, 5, index, rate=0.3)
    with ops.tuning(int4_tile=tile, bf16_tile=tile):
        case.check()


def test_the_large_products():
    """Sizes that take the products over a bf16 copy of the weight."""

    Case(4500, 2048, 2048, 16, 4, "runs", group=64).check()


def test_more_rows_than_a_grid_axis_and_32_bits_reach():
    """2^24 rows are 65536 chunks of the gradients' sums; y has over 2^32 bytes."""

    m, k, n, rank, adapters = (1 << 24) + 300, 64, 136, 4, 3
    g = torch.Generator().manual_seed(8)
    packed, scales, w = _weight(n, k, None, g)
    x, dy = (torch.randn((m, c), device=DEV, dtype=BF16) for c in (k, n))
    a = torch.randn((adapters, rank, k), device=DEV).to(BF16) / 8
    b = torch.randn((adapters, n, rank), device=DEV).to(BF16)
    s = torch.ones(adapters, device=DEV)
    index = torch.arange(m, device=DEV, dtype=torch.int32) * 7 % (adapters + 1) - 1
    leaves = [t.requires_grad_(True) for t in (x, a, b)]
    y = rx.bank_linear(x, packed, scales, a, b, s, rx.adapter_plan(index, adapters))
    dx, da, db = torch.autograd.grad(y, leaves, dy)
    x, a, b, y = x.detach(), a.detach().to(F64), b.detach().to(F64), y.detach()
    rows = torch.cat([torch.randint(0, m, (2000,), generator=g), torch.arange(m - 300, m)]).to(DEV)
    e = index[rows].long().clamp_min(0)
    on = (index[rows] >= 0).to(F64)[:, None]
    xr, gr = x[rows].to(F64), dy[rows].to(F64)
    h, dh = (xr[:, None] * a[e]).sum(2), (gr[..., None] * b[e]).sum(1)
    assert _err(y[rows], xr @ w.t() + on * (h[:, None] * b[e]).sum(2)) <= 3 * STEP
    assert _err(dx[rows], gr @ w + on * (dh[..., None] * a[e]).sum(1)) <= 3 * STEP
    want_a, want_b = torch.zeros_like(a), torch.zeros_like(b)
    for part in torch.arange(m, device=DEV).split(1 << 21):
        for i in range(adapters):
            at = part[index[part] == i]
            xs, gs = x[at].to(F64), dy[at].to(F64)
            want_a[i] += (gs @ b[i]).t() @ xs
            want_b[i] += gs.t() @ (xs @ a[i].t())
    # sums of 4 million terms of either sign: those of the rounded h and dh differ by their
    # roundings' random walk, as the terms themselves do
    assert _err(da, want_a) <= 2 * STEP and _err(db, want_b) <= 2 * STEP


@pytest.mark.parametrize("m", [3, 40, 500])
def test_float32_masters(m):
    case = Case(m, 256, 128, 16, 3, "rows", master=F32)
    case.check()


@pytest.mark.parametrize("m", [1, 60, 300])
@pytest.mark.parametrize("index", [-1, 2])
def test_no_adapter_and_one(m, index):
    case = Case(m, 256, 128, 16, 4, index, bias=True)
    case.check()
    if index < 0:
        got = case.train()
        assert not got[2].any() and not got[3].any()


@pytest.mark.parametrize("m", [1, 2, 13, 40, 333, 4500])
def test_rows_of_h_without_an_adapter_are_left(m):
    case = Case(m, 128, 64, 4, 2, "rows")
    case.index[m // 2] = -1
    plan = rx.adapter_plan(case.index, 2)
    y = torch.empty((m, 64), dtype=BF16, device=DEV)
    h = torch.full((m, 8), 77.0, dtype=BF16, device=DEV)
    cfg = {"group": 0, "site": 0, "threshold": 65536}
    fields = bank._bank_fields(case.x, case.packed, case.scales, None, case.a, case.b, case.s,
                               plan.buffer, None, cfg)
    need = nat.bank_call("forward_workspace", fields, 1)
    ws = torch.empty(max(need, 16), dtype=torch.uint8, device=DEV)
    nat.bank_call("forward", fields, y.data_ptr(), h.data_ptr(), ws.data_ptr(), need,
                  torch.cuda.current_stream().cuda_stream)
    none = case.index < 0
    assert (h[none] == 77).all() and not h[~none][:, 4:].any()
    e = case.index.long().clamp_min(0)
    want = (case.x.to(F64)[:, None] * case.a.to(F64)[e]).sum(2)
    # one rounding
    assert bool(none.all()) or _err(h[~none][:, :4], want[~none]) <= STEP * 2


def test_no_rows():
    case = Case(1, 64, 32, 8, 2, 0)
    case.plan = rx.adapter_plan(torch.empty(0, dtype=torch.int32, device=DEV), 2)
    case.x, case.dy = case.x[:0], case.dy[:0]
    y, dx, da, db = case.train()
    assert y.shape == (0, 32) and dx.shape == (0, 64) and not da.any() and not db.any()
    assert case.call().shape == (0, 32)


@pytest.mark.parametrize("m", [4, 60, 600, 1200])
def test_adapters_do_not_reach_each_others_rows(m):
    """Infinities and NaN of one adapter (and of its rows) stay with its rows, and
    their gradients with it."""

    case = Case(m, 256, 128, 16, 3, "rows", bias=True)
    case.index[:3] = torch.tensor([0, 1, 2], dtype=torch.int32)
    case.plan = rx.adapter_plan(case.index, 3)
    clean = case.train()
    case.a[1, 3, 5], case.b[1, 7] = float("inf"), float("nan")
    case.x[case.index == 1] = float("nan")
    got = case.train()
    others = case.index != 1
    for i in (0, 1):
        assert torch.equal(got[i][others], clean[i][others])
    assert torch.isnan(got[0][~others]).any()
    for i in (2, 3):
        assert torch.equal(got[i][[0, 2]], clean[i][[0, 2]])


@pytest.mark.parametrize("m,rate", [(10, 0.1), (40, 0.0), (700, 0.2), (1300, 0.2)])
def test_the_same_bits_every_time_and_in_every_order(m, rate):
    case = Case(m, 256, 128, 16, 4, "rows")
    case.rate = rate
    first, second = case.train(), case.train()
    assert all(torch.equal(a, b) for a, b in zip(first, second))
    if not rate:
        # rows in another order give the same rows
        at = torch.randperm(m, device=DEV)
        moved = case.call(x=case.x[at].contiguous(),
                          plan=rx.adapter_plan(case.index[at], case.adapters))
        assert torch.equal(moved, case.call()[at])


def test_plans_of_either_type_and_place_are_one():
    index = torch.randint(-1, 9, (3, 411), dtype=torch.int64)
    plans = [rx.adapter_plan(i, 9) for i in (index, index.to(DEV), index.to(DEV, torch.int32),
                                             index.view(-1).tolist(), index.to(DEV).t().t())]
    assert all(p.rows == 1233 for p in plans)
    first = plans[0].buffer
    # what a plan's words say: compare the ones in use (rows, order, offsets)
    words = first.view(torch.int32)
    assert torch.equal(words[:1233].cpu(), index.view(-1).int())
    used = int((index >= 0).sum())
    order = words[1236:1236 + used].cpu().long()
    flat = index.view(-1)[order]
    assert (flat[1:] >= flat[:-1]).all()
    same = flat[1:] == flat[:-1]
    assert (order[1:][same] > order[:-1][same]).all()  # within one, the rows' own order
    for p in plans[1:]:
        assert torch.equal(p.buffer.view(torch.int32)[1236:1236 + used], words[1236:1236 + used])


def test_an_index_outside_the_bank_is_reported():
    case = Case(9, 64, 32, 8, 2, 0)
    bad = case.index.clone()
    bad[4], bad[6] = 2, -7
    plan = rx.adapter_plan(bad, 2)
    y = case.call(plan=plan)
    with pytest.raises(nat.DeviceError, match="outside the bank"):
        ops.check_device_errors()
    assert ops.check_device_errors() == 0
    case.index = torch.where((bad == 2) | (bad == -7), -1, bad)
    assert torch.equal(y, case.call(plan=rx.adapter_plan(case.index, 2)))


def test_views_and_leading_axes():
    case = Case(24, 128, 64, 8, 3, "rows")
    base = torch.randn(4, 7, 130, device=DEV).to(BF16)
    x = base[:, 1:, 1:129]
    assert x.data_ptr() % 16
    y = case.call(x=x)
    assert y.shape == (4, 6, 64)
    assert torch.equal(y.view(24, 64), case.call(x=x.reshape(24, 128).contiguous()))
    a = torch.randn(128, 8, 3, device=DEV).to(BF16).permute(2, 1, 0)
    assert torch.equal(case.call(x=x, a=a), case.call(x=x, a=a.contiguous()))


@pytest.mark.parametrize("m", [4, 300])
def test_only_what_is_wanted(m):
    case = Case(m, 128, 64, 8, 3, "rows")
    full = case.train()
    for i in range(3):
        leaves = [t.detach().clone() for t in (case.x, case.a, case.b)]
        leaves[i].requires_grad_(True)
        (g,) = torch.autograd.grad(case.call(*leaves), leaves[i], case.dy)
        assert torch.equal(g, full[1 + i])


def test_few_rows_take_few_launches():
    case = Case(1, 2048, 512, 16, 4, 1)
    _, names = kernel_names(case.call)
    assert sum("k_bank" in n for n in names) == 1, names
    case = Case(13, 2048, 512, 16, 4, "rows")
    _, names = kernel_names(case.call)
    assert sum("k_bank" in n for n in names) == 2, names


@pytest.mark.parametrize("m", [4, 40, 500])
def test_captured_with_its_plan(m):
    """A step captured whole, plan included: replays read new inputs and indexes."""

    case = Case(m, 256, 128, 16, 4, "rows")
    case.rate = 0.1
    leaves = [t.requires_grad_(True) for t in (case.x, case.a, case.b)]

    def step():
        plan = rx.adapter_plan(case.index, 4)
        y = case.call(plan=plan)
        return [y.detach(), *torch.autograd.grad(y, leaves, case.dy)]

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        outs = step()
    for i in range(3):
        case.index.copy_(torch.randint(-1, 4, (m,), device=DEV))
        case.key[1] += 1
        with torch.no_grad():
            case.x.normal_()
        graph.replay()
        torch.cuda.synchronize()
        for a, b in zip(outs, step()):
            assert torch.equal(a, b), i


def test_two_streams():
    cases = [Case(m, 512, 256, 16, 4, "rows", seed=m) for m in (13, 300)]
    want = [c.train() for c in cases]
    streams = [torch.cuda.Stream() for _ in cases]
    torch.cuda.synchronize()
    for _ in range(5):
        got = []
        for c, s in zip(cases, streams):
            with torch.cuda.stream(s):
                got.append(c.train())
        torch.cuda.synchronize()
        for a, b in zip(got, want):
            assert all(torch.equal(u, v) for u, v in zip(a, b))


def test_threads_on_streams_of_their_own():
    cases = [Case(m, 256, 192, 16, 4, "rows", group=64, seed=m) for m in (2, 13, 100, 1100)]
    want = [case.train() for case in cases]
    torch.cuda.synchronize()
    wrong = []

    def work(case, expected):
        with torch.cuda.stream(torch.cuda.Stream()):
            for _ in range(5):
                got = case.train()
                torch.cuda.current_stream().synchronize()
                if not all(torch.equal(a, b) for a, b in zip(got, expected)):
                    wrong.append(case.x.shape)

    threads = [threading.Thread(target=work, args=pair) for pair in zip(cases, want)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not wrong


def test_gradients_of_constants_are_refused():
    case = Case(9, 64, 32, 8, 2, "rows", bias=True)
    case.s.requires_grad_(True)
    with pytest.raises(ValueError, match="constants"):
        case.call()
    with torch.no_grad():
        case.call()


def test_a_second_derivative_is_refused():
    case = Case(9, 64, 32, 8, 2, "rows")
    x = case.x.requires_grad_(True)
    (g,) = torch.autograd.grad(case.call(), x, case.dy, create_graph=True)
    with pytest.raises(RuntimeError):
        g.sum().backward()


CONFIG = dict(vocab_size=64, hidden_size=128, num_hidden_layers=2, num_attention_heads=2,
              intermediate_size=256, max_position_embeddings=32)


def _models(count):
    models = []
    for i in range(count):
        model = build_int4lora_encoder(BertConfig(**CONFIG), rank=8, alpha=16.0, seed=0,
                                       device=DEV)
        g = torch.Generator().manual_seed(i)
        with torch.no_grad():
            for p in rx.lora_parameters(model):
                p.copy_(torch.randn(p.shape, generator=g) * 0.05)
        models.append(model)
    return models


@pytest.mark.parametrize("remat", ["none", "full"])
def test_an_encoder_with_banks_is_its_models(remat):
    """Sequences of three tasks through one encoder with banks: each as through its
    own model, and the adapters' gradients as theirs."""

    models = _models(3)
    banked = rx.bank_quantized_lora(models)
    banked.remat = remat
    ids = torch.randint(0, 64, (6, 20), device=DEV)
    tasks = torch.tensor([0, 2, 1, 1, 0, 2])
    plan = rx.adapter_plan(tasks.repeat_interleave(20), 3)
    policy = rx.resolve_precision_policy(rx.PrecisionConfig.bfloat16_mixed())
    weight = torch.randn(6, 128, device=DEV)
    with rx.precision_context(policy), rx.adapter_rows(plan):
        out = banked.encode(ids)
    (out * weight).sum().backward()
    for task, model in enumerate(models):
        at = (tasks == task).nonzero().view(-1).to(DEV)
        with rx.precision_context(policy):
            alone = model.encode(ids[at])
        # two layers of bf16 products, rounded at other places: a few steps of 2^-8
        assert _err(out[at], alone.to(F64)) <= 8 * 2.0 ** -8
        (alone * weight[at]).sum().backward()
        grads = dict(banked.named_parameters())
        for name, p in model.named_parameters():
            if rx.lora_parameter_filter(model)[name]:
                assert _err(grads[name].grad[task], p.grad.to(F64)) <= 16 * 2.0 ** -8, name


def test_a_serving_run():
    """Requests of different lengths and adapters, then single tokens, as a server
    would call a bank: every row has what its own adapter's linear gives it."""

    model = _models(4)
    layers = [m.layers[0].mlp.input for m in model]
    bank = rx.QuantizedLoRABank.from_adapters(layers).eval()
    policy = rx.resolve_precision_policy(rx.PrecisionConfig.bfloat16_mixed())
    with torch.no_grad(), rx.precision_context(policy):
        for lengths, which in (([3, 17, 40, 90], [0, 1, 2, 3]), ([1] * 7, [3, 3, 0, 1, 2, 0, 1]),
                               ([1], [2])):
            index = torch.tensor(which).repeat_interleave(torch.tensor(lengths))
            x = torch.randn(len(index), 128, device=DEV).to(BF16)
            with rx.adapter_rows(rx.adapter_plan(index, 4)):
                y = bank(x)
            for e, layer in enumerate(layers):
                at = (index == e).nonzero().view(-1).to(DEV)
                if len(at):
                    # the linear rounds base, term and bias sum one by one
                    assert _err(y[at], layer(x[at]).to(F64)) <= 5 * STEP


def test_a_plan_of_another_batch_is_refused():
    case = Case(9, 64, 32, 8, 2, "rows")
    with pytest.raises(ValueError, match="plan"):
        case.call(x=case.x[:8])
    with pytest.raises(ValueError, match="plan"):
        case.call(plan=AdapterPlan(case.plan.buffer[:64], 9, 3))
    with pytest.raises(ValueError, match="smaller"):
        case.call(plan=AdapterPlan(case.plan.buffer[:64], 9, 2))
