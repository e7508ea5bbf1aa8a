"""Buffer sizes through the MXFP4 fast binding (CPU only, nothing launched)."""

from __future__ import annotations

import pytest

from representax_amd import _native as nat

P = 16  # never dereferenced: the sizes are refused first
BF16 = nat.DTYPE_BF16
BIG = 1 << 30
CALLS = {
    "linear": ([P, BF16, 65, 64, 64, P, P, 64, P, P, BIG, None], (10,)),
    "gated": ([P, BF16, 65, 64, 64, P, P, P, P, 64, P, P, BIG, None], (12,)),
    "linear_forward": ([P, BF16, 40, 64, 64, P, BF16, 48, 1, 64, P, BF16, P, BIG, 1, 1, P, BIG,
                        None], (13, 17)),
    "linear_backward": ([P, BF16, 40, 48, 48, P, BIG, 64, 1, 1, P, BF16, P, BF16, P, BIG, None],
                        (6, 15)),
    "gated_forward": ([P, BF16, 40, 64, 64, P, BF16, 1, 64, P, BF16, 1, 64, 48, P, P, P, BF16, P,
                       BIG, 1, 1, P, BIG, None], (19, 23)),
    "gated_backward_products": ([P, P, P, BF16, 40, 48, P, BIG, 64, 1, 1, P, BF16, P, BF16, P, BIG,
                                 None], (7, 16)),
}


@pytest.mark.parametrize("name,at", [(n, i) for n, (_, sizes) in CALLS.items() for i in sizes])
def test_negative_buffer_sizes_are_refused(name, at):
    """As sizes they would be near 2^64, and pass for room enough."""

    args = list(CALLS[name][0])
    args[at] = -1
    with pytest.raises(ValueError, match="non-negative"):
        getattr(nat.fast(), "mxfp4_" + name)(*args)
