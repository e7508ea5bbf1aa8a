"""Adapters of many requests, dropout and the boundaries of blocks: what their
speed is measured on.

* ``serve``    a packed INT4 projection shared by many requests, each row with
  the low-rank adapter of its request (``index[i] = -1``: none):
  ``y[i] = x[i] W^T + b + s_e (x[i] A_e^T) B_e^T``, ``e = index[i]``;
* ``adapt``    the same in training, several adapters in one batch, with the
  gradients of x, A and B, and with dropout on the adapters' input;
* ``dropout``  dropout and its gradient, the mask made from a counter and never
  stored;
* ``block``    the boundary between two blocks, no gradients: the norm after the
  first one, its gate, dropout, the scaled residual sum, and the norm before the
  second one;
* ``block_train``  the same with the gradients of everything.

The weight is ``W[n, k] = bf16(q s)``: q signed 4-bit, two to a byte (column 2 j
in the low half of byte j), s one bfloat16 scale a row or for every 64 columns.

A dropout's bits: element i of a tensor (in its dense order) has 16 of the 128
bits that Philox4x32-10 (Salmon et al., "Parallel random numbers: as easy as 1,
2, 3", 2011) gives for the counter (i / 8, its high word, site, step) and the
key seed; it is kept where they are below T = round(65536 (1 - rate)), times
65536 / T. ``key`` holds seed and step on the device.

The boundary: t = x + c drop(gate * post(u)) rounded to the type of x, and
h = norm(t) of that t.

Sizes are those of this repository's encoders (hidden 768 and 2048, 6144 in the
feed-forward block) and ragged ones.
"""

from __future__ import annotations

import math

import numpy
import torch

own = False

SITE = 5  # which of a step's dropouts this is


# ---------------------------------------------------------------------------
# the cases
# ---------------------------------------------------------------------------
def _serve(m, k, n, rank, adapters, group, runs, bias, **more):
    return {"kind": "serve", "m": m, "k": k, "n": n, "rank": rank, "adapters": adapters,
            "group": group, "runs": runs, "bias": bias, "rate": 0.0, **more}


def _block(kind, groups, rows, size, norm, post, gate, rate, dtype, **more):
    return {"kind": kind, "groups": groups, "rows": rows, "size": size, "norm": norm,
            "post": post, "gate": gate, "rate": rate, "dtype": dtype, **more}


def listed():
    return [
        # a query's single token through a feed-forward projection: latency
        _serve(1, 2048, 6144, 16, 32, 64, False, False, name="serve_m1_2048x6144"),
        # one token each of 13 requests, every one with its own adapter
        _serve(13, 6144, 2048, 16, 64, 0, False, True, name="serve_m13_6144x2048"),
        # short queries of ragged lengths from many tenants
        _serve(333, 2048, 6144, 8, 24, 64, True, False, name="serve_m333_2048x6144"),
        # documents indexed under eight task adapters
        _serve(16384, 6144, 2048, 32, 8, 64, True, False, name="serve_m16384_6144x2048"),
        # three tasks trained in one small ragged batch
        _serve(1001, 768, 768, 8, 3, 0, True, True, name="adapt_1001_768x768") | {
            "kind": "adapt"},
        # four tasks, 16384 tokens, dropout on the adapters' input
        _serve(16384, 2048, 6144, 16, 4, 64, True, False, name="adapt_16384_2048x6144") | {
            "kind": "adapt", "rate": 0.05},
        # a float32 tensor of odd sizes
        {"name": "dropout_f32_1001x777", "kind": "dropout", "m": 1001, "k": 777, "rate": 0.1,
         "dtype": "float32"},
        # the hidden states of 32 sequences of 512 tokens
        {"name": "dropout_16384x2048", "kind": "dropout", "m": 16384, "k": 2048, "rate": 0.1,
         "dtype": "bfloat16"},
        # one token between two blocks, a learned scale on the first one: latency
        _block("block", 1, 1, 2048, "rms", True, "vector", 0.0, "bfloat16", name="block_1x2048"),
        # a post-norm encoder's sum and norm with hidden dropout, a ragged batch
        _block("block_train", 1, 5003, 768, "layer", False, "none", 0.1, "bfloat16",
               name="block_train_5003x768"),
        # float32 and an odd size: nine sequences of 37 tokens, a gate for each
        _block("block_train", 9, 37, 1001, "layer", True, "group", 0.1, "float32",
               name="block_train_f32_333x1001"),
        # norms on both sides of a block, a gate a sequence: 32 sequences of 512
        _block("block_train", 32, 512, 2048, "rms", True, "group", 0.0, "bfloat16",
               name="block_train_16384x2048"),
    ]


def _spread(rng, low, high):
    """A size between the two, spread over its logarithm."""

    return max(low, min(high, int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))))


def draw(rng):
    kind = rng.choice(["serve", "serve", "adapt", "dropout", "block", "block_train",
                       "block_train"])
    if kind in ("serve", "adapt"):
        k, n = rng.choice([(768, 768), (2048, 2048), (2048, 6144), (6144, 2048), (0, 0)])
        if k == 0:
            k, n = 64 * _spread(rng, 4, 64), 8 * _spread(rng, 30, 512)
        m = _spread(rng, 1 if kind == "serve" else 30, 16384)
        return _serve(m, k, n, rng.choice([4, 8, 16, 32]), rng.randint(1, 48),
                      rng.choice([0, 64]), rng.random() < 0.7, rng.random() < 0.3) | {
            "kind": kind, "rate": rng.choice([0.0, 0.05, 0.1]) if kind == "adapt" else 0.0}
    dtype = rng.choice(["bfloat16", "bfloat16", "float32"])
    rate = rng.choice([0.1, 0.3, round(rng.uniform(0.01, 0.9), 3)])
    size = rng.choice([768, 2048, _spread(rng, 64, 4096), 8 * _spread(rng, 8, 512)])
    if dtype == "float32":
        size = min(size, 2048)
    if kind == "dropout":
        return {"kind": kind, "m": _spread(rng, 1, 16384 * 2048 // (size + 2048)), "k": size,
                "rate": rate, "dtype": dtype}
    groups = rng.randint(1, 32)
    limit = 16384 * 2048 // (2 * (size + 1024)) // groups
    return _block(kind, groups, _spread(rng, 1, limit), size, rng.choice(["rms", "layer"]),
                  rng.random() < 0.6, rng.choice(["none", "vector", "group"]),
                  rng.choice([0.0, rate]), dtype)


def work(case):
    kind = case["kind"]
    if kind in ("serve", "adapt"):
        m, k, n, r = case["m"], case["k"], case["n"], case["rank"]
        used = min(case["adapters"], m)
        weight = n * k // 2 + 2 * n * (k // case["group"] if case["group"] else 1)
        weight += 2 * n if case["bias"] else 0
        low = 2 * used * r * (k + n)
        if kind == "serve":
            return {"bytes": 2 * m * (k + n) + weight + low + 4 * m,
                    "flops": 2 * m * n * k + 2 * m * r * (k + n)}
        # x, dy, W, A, B and the index read; y, dx, dA and dB written
        return {"bytes": 4 * m * (k + n) + weight + 2 * low + 4 * m,
                "flops": 4 * m * n * k + 6 * m * r * (k + n)}
    size = 4 if case["dtype"] == "float32" else 2
    if kind == "dropout":
        return {"bytes": 4 * size * case["m"] * case["k"], "flops": 0}
    count = case["groups"] * case["rows"] * case["size"]
    # x and u read, t and h written; in training also dt, dh read and dx, du written
    # (the backward cannot keep t and u on the chip)
    return {"bytes": size * count * (4 if kind == "block" else 10), "flops": 0}


# ---------------------------------------------------------------------------
# inputs
# ---------------------------------------------------------------------------
def _activations(g, m, k, dtype):
    """Hidden states: a few strong channels, tokens of different norms."""

    x = torch.randn((m, k), generator=g, device="cuda")
    x *= torch.exp(0.7 * torch.randn((1, k), generator=g, device="cuda"))
    x *= torch.exp(0.3 * torch.randn((m, 1), generator=g, device="cuda"))
    return x.to(dtype)


def _packed(g, n, k, group):
    """A projection's weight packed to 4 bits: codes uint8 [n, k / 2] and the bits
    of its bfloat16 scales, [n] or [n, k / group]."""

    w = 0.02 * torch.randn((n, k), generator=g, device="cuda")
    w = w.view(n, -1, group or k)
    s = (w.abs().amax(-1, keepdim=True) / 7).to(torch.bfloat16)
    q = torch.round(w / s.float()).clamp_(-7, 7).to(torch.int8).view(n, k)
    codes = (q[:, 0::2] & 15) | (q[:, 1::2] << 4)
    s = s.view(torch.int16).view(torch.uint16)
    return codes.view(torch.uint8), s.view(n, -1) if group else s.view(n)


def _index(g, m, adapters, runs):
    """Each row's adapter, int32: requests of ragged lengths one after another
    (``runs``) or rows in any order; about one request in twelve has none."""

    def pick(count):
        e = torch.randint(0, adapters, (count,), generator=g, device="cuda", dtype=torch.int32)
        none = torch.rand((count,), generator=g, device="cuda") < 1 / 12
        return e.masked_fill_(none, -1)

    if not runs:
        return pick(m)
    # each request begins at a row of its own choice: request 0 at the first row,
    # request i at the i-th of the sorted others
    starts = (torch.rand((m // 150,), generator=g, device="cuda") * m).sort().values
    rows = torch.arange(m, device="cuda", dtype=torch.float32)
    return pick(m // 150 + 1)[torch.searchsorted(starts, rows, right=True)]


def prepare(case, seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(int(seed) * 6121 + 29)
    kind = case["kind"]
    s = {"case": case, "kind": kind}
    s["key"] = torch.tensor([(seed * 0x9E3779B97F4A7C15 + 12345) % 2 ** 62, seed % 1000],
                            dtype=torch.int64, device="cuda")
    if kind in ("serve", "adapt"):
        m, k, n, r, e = (case[name] for name in ("m", "k", "n", "rank", "adapters"))
        bf16 = torch.bfloat16
        s["x"] = _activations(g, m, k, bf16)
        s["packed"], s["scales"] = _packed(g, n, k, case["group"])
        s["a"] = (torch.randn((e, r, k), generator=g, device="cuda") * k ** -0.5).to(bf16)
        s["b"] = (torch.randn((e, n, r), generator=g, device="cuda") * 0.05).to(bf16)
        s["s"] = 2.0 * torch.rand((e,), generator=g, device="cuda") + 0.5
        s["bias"] = None
        if case["bias"]:
            s["bias"] = torch.randn((n,), generator=g, device="cuda").to(bf16)
        s["index"] = _index(g, m, e, case["runs"])
        if kind == "adapt":
            s["dy"] = 1e-3 * torch.randn((m, n), generator=g, device="cuda")
            s["dy"] = s["dy"].to(bf16)
            for name in ("x", "a", "b"):
                s[name].requires_grad_()
        if own:
            import representax_amd as rx

            # made once a batch, for every projection of the model
            s["plan"] = rx.adapter_plan(s["index"], e)
        return s
    dtype = getattr(torch, case["dtype"])
    if kind == "dropout":
        s["x"] = _activations(g, case["m"], case["k"], dtype).requires_grad_()
        s["dy"] = (1e-3 * torch.randn((case["m"], case["k"]), generator=g, device="cuda")).to(dtype)
        return s
    b, rows, size = case["groups"], case["rows"], case["size"]

    def values(scale):
        return (scale * _activations(g, b * rows, size, torch.float32)).to(dtype).view(b, rows, size)

    def weight(mean):
        # the compute views of the norms' masters
        return (mean + 0.2 * torch.randn((size,), generator=g, device="cuda")).to(dtype)

    s["x"], s["u"] = values(1.0), values(0.3)
    s["weight"], s["bias"] = weight(1.0), weight(0.0) if case["norm"] == "layer" else None
    s["post_weight"] = weight(1.0) if case["post"] else None
    s["post_bias"] = weight(0.0) if case["post"] and case["norm"] == "layer" else None
    s["gate"] = None
    if case["gate"] != "none":
        shape = (size,) if case["gate"] == "vector" else (b, 1, size)
        s["gate"] = (1 + 0.5 * torch.randn(shape, generator=g, device="cuda")).to(dtype)
    if kind == "block_train":
        s["dt"] = (1e-3 * torch.randn((b, rows, size), generator=g, device="cuda")).to(dtype)
        s["dh"] = (1e-3 * torch.randn((b, rows, size), generator=g, device="cuda")).to(dtype)
        for t in _leaves(s):
            t.requires_grad_()
    return s


def _leaves(s):
    """What a boundary's gradients are of, in the order of the outputs."""

    names = ("x", "u", "gate", "weight", "bias", "post_weight", "post_bias")
    return [s[name] for name in names if s[name] is not None]


SCALE = 0.75  # of the update in the residual sum
EPS = {"layer": 1e-12, "rms": 1e-6}


# ---------------------------------------------------------------------------
# the plain forms
# ---------------------------------------------------------------------------
def _mask(count, key, rate):
    """65536 / T or 0 for each of ``count`` elements, float32."""

    low = 0xFFFFFFFF
    vec = torch.arange(-(-count // 8), device="cuda")
    c0, c1 = vec & low, vec >> 32
    c2, c3 = torch.full_like(vec, SITE), (key[1] & low).expand_as(vec)
    k0, k1 = key[0] & low, (key[0] >> 32) & low
    for _ in range(10):
        p0, p1 = c0 * 0xD2511F53, c2 * 0xCD9E8D57
        c0, c1, c2, c3 = (((p1 >> 32) & low) ^ c1 ^ k0, p1 & low,
                          ((p0 >> 32) & low) ^ c3 ^ k1, p0 & low)
        k0, k1 = (k0 + 0x9E3779B9) & low, (k1 + 0xBB67AE85) & low
    words = torch.stack((c0, c1, c2, c3), 1)
    bits = torch.stack((words & 0xFFFF, words >> 16), 2).view(-1)[:count]
    kept = min(65536, max(1, round(65536 * (1 - rate))))
    return (bits < kept).float() * (65536 / kept)


def _dropped(t, s):
    """t float32, through the case's dropout."""

    rate = s["case"]["rate"]
    return t if rate == 0 else t * _mask(t.numel(), s["key"], rate).view(t.shape)


def _weight(s):
    codes, n = s["packed"], s["packed"].shape[0]
    q = torch.stack((codes & 15, codes >> 4), 2).view(n, -1).to(torch.int32)
    q = (q - 16 * (q >= 8).to(torch.int32)).float()
    scale = s["scales"].view(torch.int16).view(torch.bfloat16).float().view(n, -1, 1)
    return (q.view(n, scale.shape[1], -1) * scale).to(torch.bfloat16).float().view(n, -1)


def _plain_bank(s):
    x, a, b = (s[name].detach().float() for name in ("x", "a", "b"))
    w, scale, adapters = _weight(s), s["s"], s["case"]["adapters"]
    rows = [(s["index"] == e)[:, None] for e in range(adapters)]
    zero = torch.zeros((), device="cuda")
    xd = _dropped(x, s)
    h = torch.zeros((x.shape[0], a.shape[1]), device="cuda")
    for e in range(adapters):
        h = torch.where(rows[e], torch.matmul(xd, a[e].t()), h)
    y = torch.matmul(x, w.t())
    for e in range(adapters):
        y += torch.where(rows[e], torch.matmul(h, b[e].t()) * scale[e], zero)
    if s["bias"] is not None:
        y += s["bias"].float()
    y = y.to(torch.bfloat16)
    if s["kind"] == "serve":
        return [y]
    dy = s["dy"].float()
    dx, low = torch.matmul(dy, w), torch.zeros_like(x)
    da, db = torch.zeros_like(a), torch.zeros_like(b)
    for e in range(adapters):
        g = torch.where(rows[e], dy * scale[e], zero)
        dh = torch.matmul(g, b[e])
        low += torch.matmul(dh, a[e])
        da[e] = torch.matmul(dh.t(), xd)
        db[e] = torch.matmul(g.t(), h)
    dx += _dropped(low, s)
    return [y] + [t.to(torch.bfloat16) for t in (dx, da, db)]


def _plain_norm(v, kind):
    """(the normalised rows of v, 1 / their deviation), float32."""

    if kind == "layer":
        v = v - v.mean(-1, keepdim=True)
    rstd = torch.rsqrt((v * v).mean(-1, keepdim=True) + EPS[kind])
    return v * rstd, rstd


def _plain_norm_gradient(g, v, rstd, kind):
    """The gradient of v's row for the gradient g of the normalised row v."""

    mean = g.mean(-1, keepdim=True) if kind == "layer" else 0
    return rstd * (g - mean - v * (g * v).mean(-1, keepdim=True))


def _plain_block(s):
    kind, dtype = s["case"]["norm"], s["x"].dtype

    def wide(t):
        return t.detach().float()

    x, u = s["x"].detach().float(), s["u"].detach().float()
    p = u
    if s["post_weight"] is not None:
        v, v_rstd = _plain_norm(u, kind)
        p = v * wide(s["post_weight"])
        if s["post_bias"] is not None:
            p = p + wide(s["post_bias"])
    gate = None if s["gate"] is None else s["gate"].detach().float()
    t = (x + SCALE * _dropped(p if gate is None else gate * p, s)).to(dtype)
    n, n_rstd = _plain_norm(t.float(), kind)
    h = n * wide(s["weight"])
    if s["bias"] is not None:
        h = h + wide(s["bias"])
    h = h.to(dtype)
    if s["kind"] == "block":
        return [t, h]
    dh = s["dh"].float()
    d = s["dt"].float() + _plain_norm_gradient(dh * wide(s["weight"]), n, n_rstd, kind)
    out = [t, h, d.to(dtype)]
    db = SCALE * _dropped(d, s)
    dp = db if gate is None else db * gate
    du = dp
    if s["post_weight"] is not None:
        du = _plain_norm_gradient(dp * wide(s["post_weight"]), v, v_rstd, kind)
    out.append(du.to(dtype))
    if gate is not None:
        dgate = (db * p).sum(1, keepdim=True)
        out.append((dgate.sum(0).view(-1) if s["gate"].dim() == 1 else dgate).to(dtype))
    out.append((dh * n).sum((0, 1)).to(dtype))
    if s["bias"] is not None:
        out.append(dh.sum((0, 1)).to(dtype))
    if s["post_weight"] is not None:
        out.append((dp * v).sum((0, 1)).to(dtype))
        if s["post_bias"] is not None:
            out.append(dp.sum((0, 1)).to(dtype))
    return out


def _plain(s):
    if s["kind"] in ("serve", "adapt"):
        return _plain_bank(s)
    if s["kind"] == "dropout":
        mask = _mask(s["x"].numel(), s["key"], s["case"]["rate"]).view(s["x"].shape)
        return [(t.detach().float() * mask).to(t.dtype) for t in (s["x"], s["dy"])]
    return _plain_block(s)


# ---------------------------------------------------------------------------
# the framework's operators
# ---------------------------------------------------------------------------
def _modules(s, norms):
    """The norms of a boundary as its program keeps them."""

    if "norm" not in s:
        kind, size = s["case"]["norm"], s["case"]["size"]

        def module(weight, bias):
            if weight is None:
                return None
            cls = norms.LayerNorm if kind == "layer" else norms.RMSNorm
            norm = cls(size, EPS[kind], device="cuda")
            norm.weight = torch.nn.Parameter(weight.detach(), weight.requires_grad)
            if bias is not None:
                norm.bias = torch.nn.Parameter(bias.detach(), bias.requires_grad)
            return norm

        s["norm"] = module(s["weight"], s["bias"])
        s["post"] = module(s["post_weight"], s["post_bias"])
    return s["norm"], s["post"]


def _framework(s):
    import representax_amd as rx
    from representax_amd import norms

    kind, case = s["kind"], s["case"]
    if kind in ("serve", "adapt"):
        plan = s.get("plan") or rx.adapter_plan(s["index"], case["adapters"])
        y = rx.bank_linear(s["x"], s["packed"], s["scales"], s["a"], s["b"], s["s"], plan,
                           group_size=case["group"] or None, bias=s["bias"], rate=case["rate"],
                           key=s["key"], site=SITE)
        if kind == "serve":
            return [y]
        return [y.detach(), *torch.autograd.grad(y, (s["x"], s["a"], s["b"]), s["dy"])]
    if kind == "dropout":
        y = rx.dropout(s["x"], case["rate"], s["key"], site=SITE)
        return [y.detach(), *torch.autograd.grad(y, s["x"], s["dy"])]
    norm, post = _modules(s, norms)
    t, h = rx.block_norm(norm, s["x"], s["u"], post=post, gate=s["gate"], scale=SCALE,
                         rate=case["rate"], key=s["key"], site=SITE)
    if kind == "block":
        return [t, h]
    leaves = [s["x"], s["u"]] + ([] if s["gate"] is None else [s["gate"]])
    leaves += [*norm.parameters(), *(() if post is None else post.parameters())]
    return [t.detach(), h.detach(), *torch.autograd.grad((t, h), leaves, (s["dt"], s["dh"]))]


def run(state):
    return _framework(state) if own else _plain(state)


# ---------------------------------------------------------------------------
# the definitions in 64 bits
# ---------------------------------------------------------------------------
def _exact_factor(shape, key, rate):
    """The dropout's factors from the generator's definition, in unsigned 64 bits."""

    seed, step = (int(v) for v in key.cpu())
    count = math.prod(shape)
    word = numpy.uint64(0xFFFFFFFF)
    shift = numpy.uint64(32)
    block = numpy.arange((count + 7) // 8, dtype=numpy.uint64)
    x = [block & word, block >> shift, numpy.full_like(block, SITE),
         numpy.full_like(block, step & 0xFFFFFFFF)]
    keys = [seed & 0xFFFFFFFF, (seed >> 32) & 0xFFFFFFFF]
    for r in range(10):
        bump = [numpy.uint64((keys[0] + r * 0x9E3779B9) & 0xFFFFFFFF),
                numpy.uint64((keys[1] + r * 0xBB67AE85) & 0xFFFFFFFF)]
        first = x[0] * numpy.uint64(0xD2511F53)
        second = x[2] * numpy.uint64(0xCD9E8D57)
        x = [(second >> shift) ^ x[1] ^ bump[0], second & word,
             (first >> shift) ^ x[3] ^ bump[1], first & word]
    bits = numpy.empty((block.size, 8), dtype=numpy.uint16)
    for j in range(8):
        bits[:, j] = (x[j // 2] >> numpy.uint64(16 * (j % 2))).astype(numpy.uint16)
    threshold = min(65536, max(1, int(round((1.0 - rate) * 65536))))
    kept = bits.reshape(-1)[:count].astype(numpy.int32) < threshold
    return torch.from_numpy(kept).cuda().double().view(shape) * (65536.0 / threshold)


def _exact_bank(s):
    case = s["case"]
    x, a, b = s["x"].detach().double(), s["a"].detach().double(), s["b"].detach().double()
    byte = s["packed"].to(torch.int64)
    q = torch.empty((byte.shape[0], 2 * byte.shape[1]), dtype=torch.int64, device="cuda")
    q[:, ::2], q[:, 1::2] = (byte % 16 + 8) % 16 - 8, (byte // 16 + 8) % 16 - 8
    scale = s["scales"].view(torch.int16).view(torch.bfloat16).double()
    scale = scale.view(byte.shape[0], -1).repeat_interleave(case["group"] or case["k"], 1)
    w = (q.double() * scale).to(torch.bfloat16).double()
    d = x
    if case["rate"] > 0:
        factor = _exact_factor(x.shape, s["key"], case["rate"])
        d = x * factor
    index = s["index"].long()
    y = x @ w.t()
    if s["bias"] is not None:
        y = y + s["bias"].double()
    train = case["kind"] == "adapt"
    if train:
        dy = s["dy"].double()
        dx, da, db = dy @ w, torch.zeros_like(a), torch.zeros_like(b)
    for e in range(case["adapters"]):
        at = torch.nonzero(index == e).view(-1)
        if at.numel() == 0:
            continue
        se = float(s["s"][e])
        h = d[at] @ a[e].t()
        y[at] += se * (h @ b[e].t())
        if train:
            dh = se * (dy[at] @ b[e])
            back = dh @ a[e]
            dx[at] += back if case["rate"] == 0 else back * factor[at]
            da[e], db[e] = dh.t() @ d[at], se * (dy[at].t() @ h)
    return [y, dx, da, db] if train else [y]


def _exact_block(s):
    case = s["case"]
    dtype = s["x"].dtype

    def norm(v, weight, bias):
        if case["norm"] == "layer":
            return torch.nn.functional.layer_norm(v, v.shape[-1:], weight, bias, EPS["layer"])
        return v / torch.sqrt(torch.mean(v ** 2, -1, keepdim=True) + EPS["rms"]) * weight

    leaves = {}
    for name in ("x", "u", "gate", "weight", "bias", "post_weight", "post_bias"):
        if s[name] is not None:
            leaves[name] = s[name].detach().double().requires_grad_(case["kind"] == "block_train")
    update = leaves["u"]
    if "post_weight" in leaves:
        update = norm(update, leaves["post_weight"], leaves.get("post_bias"))
    if "gate" in leaves:
        update = update * leaves["gate"]
    if case["rate"] > 0:
        update = update * _exact_factor(update.shape, s["key"], case["rate"])
    t = leaves["x"] + SCALE * update
    # h is the norm of t as stored; the gradient of that rounding is one
    stored = t + (t.detach().to(dtype).double() - t.detach())
    h = norm(stored, leaves["weight"], leaves.get("bias"))
    out = [t.detach(), h.detach()]
    if case["kind"] == "block_train":
        out += torch.autograd.grad((t, h), list(leaves.values()),
                                   (s["dt"].double(), s["dh"].double()))
    return out


def exact(case, seed):
    s = prepare(case, seed)
    if case["kind"] in ("serve", "adapt"):
        return _exact_bank(s)
    if case["kind"] == "dropout":
        factor = _exact_factor(s["x"].shape, s["key"], case["rate"])
        return [s["x"].detach().double() * factor, s["dy"].double() * factor]
    return _exact_block(s)
