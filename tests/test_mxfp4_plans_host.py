"""Which MXFP4 products are split over their sums: those that ask for scratch (CPU only)."""

from __future__ import annotations

import pytest

from representax_amd import _native as nat


# few small tiles over a long sum; 144 tiles over a very long one
@pytest.mark.parametrize("m,n,k", [(96, 160, 16384), (256, 256, 12288), (768, 768, 12288),
                                   (768, 768, 32768), (1024, 1024, 16384), (1024, 2048, 16384),
                                   (768, 3072, 32768), (1536, 1536, 65536)])
def test_split(m, n, k):
    assert nat.query("rpx_mxfp4_gemm_workspace", m, n, k) > 0


# tiles that fill the card, where the partial sums cost more than they save; short sums
@pytest.mark.parametrize("m,n,k", [(768, 3072, 12288), (768, 3072, 16384), (3072, 768, 28672),
                                   (2048, 2048, 16384), (2048, 2048, 65536), (6144, 2048, 16384),
                                   (2048, 6144, 16384), (4096, 4096, 65536), (768, 768, 8192),
                                   (96, 160, 6144)])
def test_whole(m, n, k):
    assert nat.query("rpx_mxfp4_gemm_workspace", m, n, k) == 0
