"""Banks at the ends of what they accept (GPU)."""

from __future__ import annotations

import pytest
import torch

import representax_amd as rx
from representax_amd import _native as nat
from representax_amd import bank

pytestmark = pytest.mark.gpu
DEV, BF16, F64 = "cuda:0", torch.bfloat16, torch.float64


@pytest.mark.parametrize("wanted", ["both", "a", "b"])
def test_gradients_of_a_large_bank_end_where_their_tensors_do(wanted):
    """Adapters whose gradients take more than 2^21 workgroups to join, launched as a
    grid of two rows with workgroups to spare: what lies behind the gradients stays."""

    m, adapters, rank = 3, 1024, 64
    # workgroups an adapter: k / 4 + n / 4, or one of the two
    k, n = (4160, 4096) if wanted == "both" else (8256, 64) if wanted == "a" else (64, 8256)
    assert adapters * ((k if wanted != "b" else 0) + (n if wanted != "a" else 0)) // 4 > 1 << 21
    g = torch.Generator().manual_seed(3)
    used = [0, 700, adapters - 1]
    a = torch.zeros((adapters, rank, k), dtype=BF16, device=DEV)
    b = torch.zeros((adapters, n, rank), dtype=BF16, device=DEV)
    for e in used:
        a[e] = (torch.randn((rank, k), generator=g) * k ** -0.5).to(DEV, BF16)
        b[e] = torch.randn((n, rank), generator=g).to(DEV, BF16)
    x = torch.randn((m, k), generator=g).to(DEV, BF16)
    dy = torch.randn((m, n), generator=g).to(DEV, BF16)
    packed = torch.zeros((n, k // 2), dtype=torch.uint8, device=DEV)
    scales = torch.zeros((n,), dtype=torch.uint16, device=DEV)
    scalings = torch.ones(adapters, device=DEV)
    plan = rx.adapter_plan(torch.tensor(used, dtype=torch.int32), adapters, DEV)
    cfg = {"group": 0, "site": 0, "threshold": 65536}
    fields = bank._bank_fields(x, packed, scales, None, a, b, scalings, plan.buffer, None, cfg)
    h = (x.to(F64) @ a[used].to(F64).transpose(1, 2))[range(m), range(m)].to(BF16)
    behind = 1 << 26
    bits = torch.full((a.numel() + behind,), 77.0, dtype=BF16, device=DEV)
    bits_b = torch.full((b.numel() + behind,), 77.0, dtype=BF16, device=DEV)
    need_a, need_b = wanted != "b", wanted != "a"
    need = nat.bank_call("backward_workspace", fields, 0, int(need_a), int(need_b))
    ws = torch.empty(need, dtype=torch.uint8, device=DEV)
    nat.bank_call("backward", fields, dy.data_ptr(), h.data_ptr(), None,
                  bits.data_ptr() if need_a else None, nat.DTYPE_BF16,
                  bits_b.data_ptr() if need_b else None, nat.DTYPE_BF16, ws.data_ptr(), need,
                  torch.cuda.current_stream().cuda_stream)
    assert (bits[a.numel():] == 77).all() and (bits_b[b.numel():] == 77).all()
    for i, e in enumerate(used):
        xi, gi, ae, be = (t.to(F64) for t in (x[i], dy[i], a[e], b[e]))
        # one row: roundings of dh (or h) to bf16 and of the product, 2^-8 each at most
        for got, want, on in ((bits[:a.numel()].view(a.shape)[e], torch.outer(gi @ be, xi), need_a),
                              (bits_b[:b.numel()].view(b.shape)[e], torch.outer(gi, ae @ xi), need_b)):
            assert not on or ((got.to(F64) - want).abs() <= 2.01 * 2.0 ** -8 * want.abs()
                              + 2.0 ** -14 * want.abs().max()).all()
    rest = torch.ones(adapters, dtype=torch.bool, device=DEV)
    rest[used] = False
    if need_a:
        assert not bits[:a.numel()].view(a.shape)[rest].any()
    if need_b:
        assert not bits_b[:b.numel()].view(b.shape)[rest].any()
