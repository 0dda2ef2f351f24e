"""Calls of the 8-bit key/value cache at the edges of what they take: which of them run, by which way, and what is refused."""
import pytest
import torch

from easyllm_b200.ops import infer as iops
from test_kv8 import (BF16, DEVICES, F32, _device, _no_kernel_gave_up, check_attention, filled, ints, near, plain_attention, rand,  # noqa: F401
                      step)


class NoKernel:
    """In the place of the launchers: a call of any of them is a failure."""

    def __getattr__(self, name):
        raise AssertionError(f"{name} was called")


# ---- borders without a sequence ---------------------------------------------------------------------
@pytest.mark.parametrize("max_len,max_q", [(64, 1), (64, 3), (5000, 3), (5000, 300)])
def test_rows_without_a_sequence_reach_no_kernel(monkeypatch, max_len, max_q):
    cache = iops.kv8_empty(64, 2, 32, 16, 16)
    monkeypatch.setattr(iops, "_kern", lambda x: True)
    monkeypatch.setattr(iops, "_cu", NoKernel)
    q, places = torch.ones(5, 4, 32, dtype=BF16), ints([999] * 5)
    got = iops.attention_kv8(q, cache, places, places, max_len, 1.0, cu_seqlens=ints([0]), max_q=max_q)
    assert got.shape == (5, 4, 16) and got.dtype == BF16 and not bool(got.any())


def test_the_entry_refuses_borders_without_a_sequence():
    """Before it looks at anything on the device, so this needs none."""
    import ctypes
    from easyllm_b200.ops import cuda, cuda_infer
    at = 1 << 20                                                  # an address that nobody looks at
    words = (at, at, at, at, 2, 32, 16, 16, 64)
    for n_seq in (0, -1):
        call = cuda_infer._KV8_CALLS["ell_attn_kv8"](*words, at, at, 0, 0, at, at, 0, 0, at, 5, n_seq, 1, 4, 128, 64, 0, 1, at, 1.0)
        assert cuda.lib().ell_attn_kv8(ctypes.c_char_p(call), ctypes.c_void_p(0)) == -2


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("max_len,max_q,H", [(64, 1, 4), (64, 3, 4), (5000, 3, 4), (5000, 300, 4), (5000, 2, 512)])
def test_rows_without_a_sequence_are_zero(device, dtype, max_len, max_q, H):
    dev = _device(device)
    cache, _ = filled(64, 2, 32, 32, 16, dev)
    places = ints([0, 999, -1, 1 << 30, 16], dev)
    got = iops.attention_kv8(torch.ones(5, H, 32, dtype=dtype, device=dev), cache, places, places, max_len, 1.0, cu_seqlens=ints([0], dev), max_q=max_q)
    assert got.shape == (5, H, 32) and got.dtype == dtype and not bool(got.any())
