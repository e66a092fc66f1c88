"""The error word that a call hands to its kernels: anything but int32 with an
element on the call's device is refused before a kernel could write to it."""

from __future__ import annotations

import pytest
import torch

from bpdecode_amd import ops
from bpdecode_amd.kv import PagedKV4, block_bytes

DEVICES = ["cpu", pytest.param("cuda", marks=pytest.mark.gpu)]


def wrong_words(device) -> list[torch.Tensor]:
    other = torch.zeros(1, dtype=torch.int32, device="cpu" if device == "cuda" else "meta")
    return [other, torch.zeros(1, device=device), torch.zeros(1, dtype=torch.int64, device=device),
            torch.zeros(0, dtype=torch.int32, device=device)]


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("which", range(4))
def test_verification_refuses_a_wrong_error_word(which, device):
    z, x = torch.zeros(2, 3, 8, device=device), torch.zeros(2, 2, dtype=torch.int32, device=device)
    u = torch.zeros(2, 3, device=device)
    with pytest.raises(RuntimeError, match="err must be int32"):
        ops.dense_verify(z, x, u, err=wrong_words(device)[which])
    good = torch.zeros(1, dtype=torch.int32, device=device)
    ops.dense_verify(z, x, u, err=good)
    assert not int(good)
    ops.dense_verify(z.fill_(float("nan")), x, u, err=good)
    assert int(good)


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("which", range(4))
def test_the_cache_refuses_a_wrong_error_word(which, device):
    pages = torch.zeros(2, 1, block_bytes(16, 64), dtype=torch.uint8, device=device)
    with pytest.raises(RuntimeError, match="err must be int32"):
        PagedKV4(pages, 16, 64, torch.bfloat16, wrong_words(device)[which])
