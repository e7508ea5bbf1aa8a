"""The microscaled 4-bit operators: what their speed is measured on.

A matrix held in MXFP4 has, for each row, blocks of 32 consecutive columns. A
block has one power-of-two scale 2^e, e = floor(log2(max |v|)) - 2 (at least
-127), and each value is the 4-bit number (sign, 0, 0.5, 1, 1.5, 2, 3, 4 or 6)
nearest to v / 2^e, ties to the even code, at most 6 in magnitude. A block that
holds an infinity or a NaN stands for NaN throughout. Every product contracts
the columns of two such matrices: out[i, j] = sum_c A[i, c] B[j, c], summed in
32 bits and rounded once to the output's type.

As stored: ``codes`` uint8 [rows, C / 2] with C the columns rounded up to 256
(column 2 j in the low half of byte j, codes of columns past the end zero) and
``scales`` uint8 [C / 256, R, 8] with R the rows rounded up to 32: the scale of
block b of row i is 2^(scales[b // 8, i, b % 8] - 127), 255 for NaN.

Kinds of case:

* ``encode``  one matrix to MXFP4 along its rows and along its columns (a weight
  for its forward and its input-gradient product), and back to the values that
  the codes stand for;
* ``serve``   x W^T with a weight that the program keeps in MXFP4, x encoded
  within the call (a query's single token, short queries, batches of documents);
* ``train``   y = x W^T with its gradients: dx = dy W, dW = dy^T x, each of the
  three products over operands encoded along the axis that it contracts;
* ``gated``   silu(x G^T) * (x U^T) over two kept weights, the first half of a
  gated feed-forward block;
* ``gated_train``  the same with its gradients. The two projections are rounded
  to bfloat16 before the activation, as separate linears would leave them, and
  the gradients of the projections are encoded before their two products, over
  both projections at once: dx = [dg | du] [G; U], [dG; dU] = [dg | du]^T x.

Sizes are those of this repository's encoders (hidden 768 with 3072, 2048 with
6144) and ragged ones between.
"""

from __future__ import annotations

import math

import torch

own = False

BLOCK = 32
SLICE = 256
ROW_PAD = 32


# ---------------------------------------------------------------------------
# the cases
# ---------------------------------------------------------------------------
def listed():
    return [
        # a text tower's feed-forward weight, for both of its products
        {"name": "encode_6144x2048", "kind": "encode", "m": 6144, "k": 2048, "n": 0,
         "dtype": "bfloat16"},
        # a float32 master of odd sizes
        {"name": "encode_f32_1001x777", "kind": "encode", "m": 1001, "k": 777, "n": 0,
         "dtype": "float32"},
        # one query's single token through a feed-forward projection: latency
        {"name": "serve_m1_2048x6144", "kind": "serve", "m": 1, "k": 2048, "n": 6144,
         "dtype": "bfloat16"},
        # a short query's 13 tokens back to the hidden size
        {"name": "serve_m13_6144x2048", "kind": "serve", "m": 13, "k": 6144, "n": 2048,
         "dtype": "bfloat16"},
        # a few short documents, a ragged number of tokens
        {"name": "serve_m333_2048x6144", "kind": "serve", "m": 333, "k": 2048, "n": 6144,
         "dtype": "bfloat16"},
        # a batch of documents when an index is built
        {"name": "serve_m16384_6144x2048", "kind": "serve", "m": 16384, "k": 6144, "n": 2048,
         "dtype": "bfloat16"},
        # the training step of a BERT-base feed-forward projection, 256 sequences of 32
        {"name": "train_8192_768x3072", "kind": "train", "m": 8192, "k": 768, "n": 3072,
         "dtype": "bfloat16"},
        # its other projection over sequences of 500 tokens: the tokens, which the
        # weight gradient contracts, are no multiple of a block
        {"name": "train_3500_3072x768", "kind": "train", "m": 3500, "k": 3072, "n": 768,
         "dtype": "bfloat16"},
        # the gated block for one query's single token
        {"name": "gated_m1_2048x6144", "kind": "gated", "m": 1, "k": 2048, "n": 6144,
         "dtype": "bfloat16"},
        # and for a ragged batch of documents
        {"name": "gated_m5003_2048x6144", "kind": "gated", "m": 5003, "k": 2048, "n": 6144,
         "dtype": "bfloat16"},
        # a training step at odd sizes: every axis ends within a block
        {"name": "gated_train_1001_500x1300", "kind": "gated_train", "m": 1001, "k": 500,
         "n": 1300, "dtype": "bfloat16"},
        # the training step of a text tower's gated block, 16384 tokens
        {"name": "gated_train_16384_2048x6144", "kind": "gated_train", "m": 16384, "k": 2048,
         "n": 6144, "dtype": "bfloat16"},
    ]


def _spread(rng, low, high):
    """A size between the two, spread over its logarithm; half of them multiples of 64."""

    size = int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))
    if size >= 64 and rng.random() < 0.5:
        size -= size % 64
    return max(low, min(high, size))


def draw(rng):
    kind = rng.choice(["encode", "serve", "serve", "train", "gated", "gated_train"])
    dtype = "float32" if kind in ("encode", "serve") and rng.random() < 0.25 else "bfloat16"
    if kind == "encode":
        return {"kind": kind, "m": _spread(rng, 64, 8192), "k": _spread(rng, 64, 6144), "n": 0,
                "dtype": dtype}
    # the feed-forward sizes of the encoders or ragged ones between them
    k, n = rng.choice([(768, 3072), (3072, 768), (2048, 6144), (6144, 2048), (0, 0), (0, 0)])
    if k == 0:
        k, n = _spread(rng, 200, 4096), _spread(rng, 200, 6144)
    if kind.startswith("gated") and k > n:
        k, n = n, k
    low = 1 if kind in ("serve", "gated") else 32
    m = min(_spread(rng, low, 16384), 16384 * 2048 * 6144 // (k * n))  # the largest listed
    return {"kind": kind, "m": m, "k": k, "n": n, "dtype": dtype}


def work(case):
    m, k, n = case["m"], case["k"], case["n"]
    size = 4 if case["dtype"] == "float32" else 2
    if case["kind"] == "encode":
        # read once; the values of both encodings, in bfloat16, written once
        return {"bytes": m * k * (size + 4), "flops": 0}
    weight = n * k // 2 + n * -(-k // BLOCK)  # one kept weight: codes and scales
    if case["kind"] == "serve":
        return {"bytes": size * (m * k + m * n) + weight, "flops": 2 * m * n * k}
    if case["kind"] == "gated":
        return {"bytes": size * (m * k + m * n) + 2 * weight, "flops": 4 * m * n * k}
    if case["kind"] == "train":
        # x, W and dy read; y, dx and dW written
        return {"bytes": 2 * (2 * m * k + 2 * n * k + 2 * m * n), "flops": 6 * m * n * k}
    # x, G, U and dh read; h, dx, dG and dU written
    return {"bytes": 2 * (2 * m * k + 4 * n * k + 2 * m * n), "flops": 12 * m * n * k}


# ---------------------------------------------------------------------------
# inputs
# ---------------------------------------------------------------------------
def _generator(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(int(seed) * 7919 + 17)
    return g


def _normal(g, rows, columns, scale, dtype):
    return torch.randn((rows, columns), generator=g, device="cuda").mul_(scale).to(dtype)


def _activations(g, m, k, dtype):
    """Hidden states: a few strong channels, tokens of different norms, and (from
    eight tokens on) rows of padding that are zero throughout."""

    x = torch.randn((m, k), generator=g, device="cuda")
    x *= torch.exp(0.7 * torch.randn((1, k), generator=g, device="cuda"))
    x *= torch.exp(0.3 * torch.randn((m, 1), generator=g, device="cuda"))
    if m >= 8:
        x[m // 2::8] = 0
    return x.to(dtype)


def _exponents(amax):
    """floor(log2(amax)) - 2, at least -127, as int32; -127 where amax is zero."""

    return torch.where(amax > 0, torch.frexp(amax).exponent - 3, -127).clamp_(min=-127)


def _blocks(t):
    """t [rows, columns] as float32 blocks [rows, blocks, 32], zeros past the end."""

    rows, columns = t.shape
    nblocks = -(-columns // BLOCK)
    wide = torch.zeros((rows, nblocks * BLOCK), dtype=torch.float32, device=t.device)
    wide[:, :columns] = t
    return wide.view(rows, nblocks, BLOCK)


def _nearest(a):
    """The 4-bit magnitude nearest to a >= 0, ties to the even code (the codes of
    0, 0.5, 1, 1.5, 2, 3, 4 and 6 in order), at most 6."""

    step = torch.where(a < 2, 0.5, torch.where(a < 4, 1.0, 2.0))
    return (torch.round(a / step) * step).clamp_(max=6.0)


def _encode(t):
    """(values / 2^e, e) of t's blocks: [rows, blocks, 32] and [rows, blocks]."""

    v = _blocks(t)
    e = _exponents(v.abs().amax(dim=-1))
    a = torch.ldexp(v, -e[..., None])
    return torch.copysign(_nearest(a.abs()), a), e


def _stored(t):
    """The codes and scales of t as a program keeps them (see the top)."""

    rows, columns = t.shape
    v, e = _encode(t)
    levels = torch.tensor([0, 0.5, 1, 1.5, 2, 3, 4, 6], device=t.device)
    code = torch.bucketize(v.abs(), levels).to(torch.uint8)
    code |= (torch.signbit(v).to(torch.uint8) << 3)
    slices = -(-columns // SLICE)
    wide = torch.zeros((rows, slices * SLICE), dtype=torch.uint8, device=t.device)
    wide[:, :code.shape[1] * BLOCK] = code.view(rows, -1)
    codes = wide[:, 0::2] | (wide[:, 1::2] << 4)
    scales = torch.zeros((-(-rows // ROW_PAD) * ROW_PAD, slices * 8), dtype=torch.uint8,
                         device=t.device)
    scales[:rows, :e.shape[1]] = (e + 127).to(torch.uint8)
    return codes, scales.view(-1, slices, 8).permute(1, 0, 2).contiguous()


def prepare(case, seed):
    g = _generator(seed)
    m, k, n = case["m"], case["k"], case["n"]
    dtype = getattr(torch, case["dtype"])
    state = {"kind": case["kind"], "m": m, "k": k, "n": n, "dtype": dtype}
    if case["kind"] == "encode":
        state["w"] = _normal(g, m, k, 0.02, dtype)
        return state
    state["x"] = _activations(g, m, k, dtype)
    if case["kind"] == "serve":
        state["w"] = _stored(_normal(g, n, k, 0.02, torch.float32))
    elif case["kind"] == "gated":
        state["gate"] = _stored(_normal(g, n, k, 0.02, torch.float32))
        state["up"] = _stored(_normal(g, n, k, 0.02, torch.float32))
    else:
        state["dy"] = _normal(g, m, n, 1e-3, dtype)
        for name in ("w",) if case["kind"] == "train" else ("gate", "up"):
            state[name] = _normal(g, n, k, 0.02, dtype).requires_grad_()
        state["x"].requires_grad_()
    return state


# ---------------------------------------------------------------------------
# the plain forms
# ---------------------------------------------------------------------------
def _values(t):
    """What t's encoding along its columns stands for, in float32."""

    v, e = _encode(t)
    return torch.ldexp(v, e[..., None]).view(t.shape[0], -1)[:, :t.shape[1]]


def _kept_values(kept, columns):
    """What stored codes and scales stand for, in float32 [rows, columns]."""

    codes, scales = kept
    rows = codes.shape[0]
    code = torch.stack((codes & 15, codes >> 4), dim=-1).view(rows, -1).to(torch.int64)
    levels = torch.tensor([0, 0.5, 1, 1.5, 2, 3, 4, 6, -0.0, -0.5, -1, -1.5, -2, -3, -4, -6],
                          device=codes.device)
    e = scales.permute(1, 0, 2).reshape(scales.shape[1], -1)[:rows].to(torch.int32) - 127
    v = torch.ldexp(levels[code].view(rows, -1, BLOCK), e[..., None])
    return v.view(rows, -1)[:, :columns]


def _plain(s):
    kind, dtype = s["kind"], s["dtype"]
    if kind == "encode":
        bf16 = torch.bfloat16
        return [_values(s["w"]).to(bf16), _values(s["w"].t()).to(bf16)]
    if kind == "serve":
        return [torch.matmul(_values(s["x"]), _kept_values(s["w"], s["k"]).t()).to(dtype)]
    if kind == "gated":
        x = _values(s["x"])
        g = torch.matmul(x, _kept_values(s["gate"], s["k"]).t()).to(dtype).float()
        u = torch.matmul(x, _kept_values(s["up"], s["k"]).t()).to(dtype).float()
        return [(g / (1 + torch.exp(-g)) * u).to(dtype)]
    x, dy = s["x"].detach(), s["dy"]
    if kind == "train":
        w = s["w"].detach()
        y = torch.matmul(_values(x), _values(w).t())
        dx = torch.matmul(_values(dy), _values(w.t()).t())
        dw = torch.matmul(_values(dy.t()), _values(x.t()).t())
        return [t.to(dtype) for t in (y, dx, dw)]
    gate, up = s["gate"].detach(), s["up"].detach()
    xv = _values(x)
    g = torch.matmul(xv, _values(gate).t()).to(dtype).float()
    u = torch.matmul(xv, _values(up).t()).to(dtype).float()
    sig = 1 / (1 + torch.exp(-g))
    h = g * sig * u
    dh = dy.float()
    dg = dh * u * sig * (1 + g * (1 - sig))
    du = dh * g * sig
    dx = torch.matmul(_values(dg), _values(gate.t()).t())
    dx = dx + torch.matmul(_values(du), _values(up.t()).t())
    xt = _values(x.t()).t()
    return [t.to(dtype) for t in (h, dx, torch.matmul(_values(dg.t()), xt),
                                  torch.matmul(_values(du.t()), xt))]


# ---------------------------------------------------------------------------
# the framework's operators
# ---------------------------------------------------------------------------
_POLICY = []


def _policy(rx):
    if not _POLICY:
        _POLICY.append(rx.resolve_precision_policy(rx.PrecisionConfig.mxfp4_mixed()))
    return _POLICY[0]


def _framework(s):
    import representax_amd as rx

    kind = s["kind"]
    if kind == "encode":
        along_rows, along_columns = rx.mxfp4_quantize_both(s["w"])
        return [along_rows.dequantize(), along_columns.dequantize()]
    if kind == "serve":
        return [rx.mxfp4_linear(s["x"], rx.MXFP4Matrix(*s["w"], s["k"]))]
    if kind == "gated":
        return [rx.mxfp4_gated(s["x"], rx.MXFP4Matrix(*s["gate"], s["k"]),
                               rx.MXFP4Matrix(*s["up"], s["k"]))]
    with rx.precision_context(_policy(rx)):
        if kind == "train":
            leaves = (s["x"], s["w"])
            y = rx.linear_matmul(s["x"], s["w"].t())
        else:
            leaves = (s["x"], s["gate"], s["up"])
            y = rx.gated_matmul(s["x"], s["gate"].t(), s["up"].t())
    return [y.detach(), *torch.autograd.grad(y, leaves, s["dy"])]


def run(state):
    return _framework(state) if own else _plain(state)


# ---------------------------------------------------------------------------
# the definition in 64 bits
# ---------------------------------------------------------------------------
def _exact_values(t):
    t = t.detach().double()
    rows, columns = t.shape
    short = -columns % BLOCK
    v = torch.nn.functional.pad(t, (0, short)).unflatten(1, (-1, BLOCK))
    top = v.abs().amax(-1, keepdim=True)
    power = torch.floor(torch.log2(top.clamp(min=2.0 ** -149))) - 2
    scale = torch.exp2(power.clamp(min=-127.0))
    a = v.abs() / scale
    q = 0.5 * ((a > 0.25).double() + (a >= 0.75) + (a > 1.25) + (a >= 1.75))
    q = q + (a > 2.5).double() + (a >= 3.5).double() + 2 * (a > 5).double()
    return (torch.sign(v) * q * scale).flatten(1)[:, :columns]


def _exact_kept(kept, columns):
    codes, scales = kept
    byte = codes.double()
    high = torch.floor(byte / 16)
    code = torch.stack((byte - 16 * high, high), -1).flatten(1)
    sign = 1 - 2 * (code >= 8).double()
    code = code - 8 * (code >= 8)
    value = torch.where(code < 4, code / 2, torch.where(code < 6, code - 2, 2 * code - 8))
    power = torch.cat([scales[i] for i in range(scales.shape[0])], 1)[:codes.shape[0]].double() - 127
    return ((sign * value) * torch.exp2(power).repeat_interleave(BLOCK, 1))[:, :columns]


def _rounded(t):
    """To bfloat16 and back, where the definition rounds a projection."""

    return t.to(torch.float32).to(torch.bfloat16).double()


def exact(case, seed):
    s = prepare(case, seed)
    kind = s["kind"]
    if kind == "encode":
        return [_exact_values(s["w"]), _exact_values(s["w"].t())]
    x = _exact_values(s["x"])
    if kind == "serve":
        return [x @ _exact_kept(s["w"], s["k"]).t()]
    if kind == "gated":
        g = _rounded(x @ _exact_kept(s["gate"], s["k"]).t())
        u = _rounded(x @ _exact_kept(s["up"], s["k"]).t())
        return [g * torch.special.expit(g) * u]
    dy = s["dy"].double()
    xt = _exact_values(s["x"].t())
    if kind == "train":
        return [x @ _exact_values(s["w"]).t(), _exact_values(dy) @ _exact_values(s["w"].t()).t(),
                _exact_values(dy.t()) @ xt.t()]
    g = _rounded(x @ _exact_values(s["gate"]).t())
    u = _rounded(x @ _exact_values(s["up"]).t())
    sig = torch.special.expit(g)
    h = g * sig * u
    dg = dy * u * (sig + g * sig * torch.special.expit(-g))
    du = dy * (g * sig)
    dx = torch.cat([_exact_values(dg), _exact_values(du)], 1) @ torch.cat(
        [_exact_values(s["gate"].t()), _exact_values(s["up"].t())], 1).t()
    return [h, dx, _exact_values(dg.t()) @ xt.t(), _exact_values(du.t()) @ xt.t()]
