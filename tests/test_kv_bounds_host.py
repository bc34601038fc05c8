"""CPU: counts and sizes that the 32-bit fields of include/dmx_kv.h do not hold
are refused by drinkme_amd.kv_ops before anything is made of them, and a scale
that fp32 does not hold times log2(e) by the C ABI."""

import ctypes as ct
import os

import pytest
import torch

from drinkme_amd import _native, kv_ops

CPU = torch.device("cpu")
OVER = [2 ** 30, 2 ** 31 + 2, 2 ** 32 + 2, 2 ** 64 + 2]


def seqs(total=2, table=None, lengths=None, cu=None, max_tokens=None):
    one = torch.zeros(1, dtype=torch.int32)
    return kv_ops._seqs_of(one.expand(2, 3) if table is None else table, one.expand(2) if lengths is None else lengths, cu,
                           total, max_tokens, CPU, "test")[0]


@pytest.mark.parametrize("total", OVER + [-2])
def test_tokens_of_a_call(total):
    with pytest.raises(ValueError, match=f"test: {total} tokens"):
        seqs(total)
    assert seqs(2 ** 30 - 2).total == 2 ** 30 - 2


@pytest.mark.parametrize("over", OVER)
def test_bounds_on_new_tokens(over):
    """A bound past the call's tokens is the call's tokens."""
    cu = torch.tensor([0, 1, 5], dtype=torch.int32)
    assert seqs(5, cu=cu, max_tokens=over).max_tokens == 5 and seqs(5, cu=cu, max_tokens=4).max_tokens == 4


@pytest.mark.parametrize("over", OVER[:3])
def test_sequences_and_columns(over):
    one = torch.zeros(1, dtype=torch.int32)  # (views of one element: nothing is made of them)
    with pytest.raises(ValueError, match="block_table"):
        seqs(table=one.expand(2, over))
    with pytest.raises(ValueError, match="block_table"):
        seqs(table=one.expand(over, 3), lengths=one.expand(over), cu=one.expand(over + 1))


@pytest.mark.parametrize("over", OVER[:3])
def test_positions_of_a_table(over):
    with pytest.raises(ValueError, match="positions"):
        kv_ops._rotary_of(torch.zeros(1).expand(over, 32, 2), "half", 64, CPU, "test")


@pytest.mark.skipif(os.path.exists("/dev/kfd"), reason="stand-in device pointers: CPU only")
@pytest.mark.parametrize("scale", [2.0 ** 127 * 1.5, 3.4e38, float("inf"), 0.0, float("nan")])
def test_a_scale_whose_product_overflows(scale):
    """Infinity times a score of 0 is NaN."""
    fake = 0x10000  # never dereferenced: the call is refused first
    cache = _native.KvCache(fake, fake, fake, fake, 4, 2, 64, 128)
    s, q = _native.KvSeqs(fake, fake, None, 2, 3, 4, 2), _native.KvRows(None, 1024, 128, 4)
    err = _native.error_buffer()
    st = _native.lib().dmx_kv_attention(ct.byref(cache), ct.byref(s), ct.byref(q), 0, scale, 1, 0, 0, fake, None, None, 0,
                                        None, err, len(err))
    assert st == 1 and b"scale" in err.value
