"""Buffer sizes through the fast binding of banks and block boundaries (CPU only,
nothing launched)."""

from __future__ import annotations

import pytest

from representax_amd import _native as nat

P = 1 << 20  # never dereferenced: the sizes are refused first
BANK = [P, 5, 64, P, P, 24, 0, None, P, P, P, 3, 8, P, 1 << 20, None, 0, 65536]
BLOCK = [P, P, None, 0, None, None, 0, 0, 1e-6, P, None, 0, 1, 1e-6, None, 0, 65536, 4, 64, P, P,
         0, 0, 1.0]
CALLS = {
    "bank_forward_workspace": (BANK + [0], (14,)),
    "bank_forward": (BANK + [P, P, P, 1 << 20, None], (14, 21)),
    "bank_backward_workspace": (BANK + [1, 1, 1], (14,)),
    "bank_backward": (BANK + [P, P, P, P, 0, P, 0, P, 1 << 20, None], (14, 26)),
    "block_backward": (BLOCK + [P, P, P, P, None, None, None, None, None, P, 1 << 20, None], (34,)),
}


@pytest.mark.parametrize("name,at", [(n, i) for n, (_, sizes) in CALLS.items() for i in sizes])
def test_negative_buffer_sizes_are_refused(name, at):
    """As sizes they would be near 2^64, and pass for room enough."""

    args = list(CALLS[name][0])
    args[at] = -1
    with pytest.raises(ValueError, match="non-negative"):
        getattr(nat.fast(), name)(*args)


@pytest.mark.parametrize("name", CALLS)
def test_calls_take_their_number_of_arguments(name):
    args = list(CALLS[name][0])
    for wrong in (args[:-1], args + [None]):
        with pytest.raises(TypeError):
            getattr(nat.fast(), name)(*wrong)
