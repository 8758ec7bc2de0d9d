"""What the paged operators refuse or report, without a GPU."""

import ctypes as C

import pytest

from light_b200 import _lib, ops


@pytest.mark.parametrize("device", [63, 64, -1])
def test_status_of_a_device_that_is_not_there_is_an_error_and_no_bits(device):
    """CUDA's error codes are positive: 100, as bits, would say that a slot was outside the cache."""
    assert _lib.lib().light_b200_paged_status(device) < 0
    with pytest.raises(_lib.Light200Error, match="light_b200"):
        ops.paged_status(device)
    assert _lib.lib().light_b200_paged_status_clear(device) < 0
    with pytest.raises(_lib.Light200Error, match="light_b200"):
        ops.paged_status(device, clear=True)


@pytest.mark.parametrize("scale,softcap", [(1e19, 1e-20), (-1e19, 1e-20), (3e38, 0.0), (float("inf"), 0.0), (float("nan"), 0.0), (float("nan"), 1.0), (2e38, 30.0)])
def test_attention_entry_refuses_scales_that_overflow(scale, softcap):
    """What scores are multiplied by is an f32: infinite, it would make NaN of a score of 0, whose weight is finite."""
    rows = dict(q_stride=(256, 64), k_stride=(8192, 1024, 64), v_stride=(8192, 1024, 64))
    a = _lib.PagedAttnArgs(q=256, k=256, v=256, block_table=256, lens=256, out=256, table_stride=4, pages=5, dtype=0, B=2, NH=4, KH=2, D=64, page_size=16, W=4, window=0, scale=scale,
                           softcap=softcap, **{n: (C.c_int64 * len(v))(*v) for n, v in rows.items()})
    assert _lib.lib().light_b200_paged_attn_scratch_bytes(C.byref(a), 0) == 0
    assert _lib.lib().light_b200_paged_decode_attn(C.byref(a), 0, None) == -2
    assert "scale" in _lib.last_error()


@pytest.mark.parametrize("beta", [dict(beta_fast=0.0), dict(beta_slow=0.0), dict(beta_fast=1.0, beta_slow=32.0), dict(beta_fast=2.0, beta_slow=2.0), dict(beta_fast=float("nan"))])
def test_yarn_refuses_turns_in_no_order(beta):
    with pytest.raises(ValueError, match="RoPEFrequencies"):
        ops.RoPEFrequencies(16, 10000.0, "yarn", 4.0, original=4096, device="cpu", **beta)
