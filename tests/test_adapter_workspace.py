"""Workspace sizes of the adapters (runs without a GPU): partial sums are reserved where sums are
split, and not for every adapter there is."""

from __future__ import annotations

import pytest

from mmfp4 import _lib

MIB = 1 << 20


def records(T, r, L):
    """What two records of every tile of 64 tokens take: hi and lo of 16 bits, in two orders, the
    ranks in chunks of 16, 32 or 64."""
    rp = 16 if r <= 16 else 32 if r <= 32 else 64
    return 2 * (T // 64 + min(L, T)) * 64 * -(-r // rp) * rp * 8


@pytest.mark.parametrize("T,K,N,r,L", [
    (4000, 4096, 4096, 16, 1000), (1000, 14336, 4096, 64, 64), (4000, 4096, 14336, 64, 1000),
    (8192, 14336, 14336, 128, 1024), (100, 4096, 4096, 16, 1024), (300000, 4096, 4096, 8, 64)])
def test_many_adapters(T, K, N, r, L):
    """Nothing of the size of all adapters' gradients (L r (K + N) fp32): the records, lists of
    tokens and tiles, and the partial sums of at most 512 blocks of 64 x 64 twice."""
    need = _lib.load().mm_lora_workspace_bytes(T, K, N, r, L, 1)
    lists = 4 * 64 * (T // 64 + L + 1) + 16 * (T // 64 + 2 * L + 2)
    assert records(T, r, L) <= need <= records(T, r, L) + lists + 2 * 512 * 64 * 64 * 4 + MIB


def test_split_sums_have_their_place():
    size = _lib.load().mm_lora_workspace_bytes
    one = records(4096, 16, 1)
    # 4096 tokens of one adapter: both weight gradients in two parts
    assert size(4096, 4096, 14336, 16, 1, 1) >= one + 2 * 16 * 4 * (4096 + 14336)
    # 1111 tokens, the forward's 14336 columns cut in several
    assert size(1111, 14336, 4096, 64, 4, 0) >= 2 * (17 + 4) * 64 * 64 * 4
