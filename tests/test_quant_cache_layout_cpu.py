"""Layouts that the quantised cache's wrappers are given, without a GPU: rows that need a copy, buffers that are refused."""
import pytest
import torch

from utmist_bigger_bird_b200 import QuantKV
from utmist_bigger_bird_b200.quant_cache import _rows


def flat(n):
    """Elements on a 16-byte boundary."""
    return torch.arange(n + 16, dtype=torch.float32).to(torch.bfloat16)[:n].clone()


@pytest.mark.parametrize("x", [
    flat(2 * 3 * 64 + 1)[1:].view(2, 3, 64),                        # contiguous, at an address of 2 mod 16
    flat(3 * 64).as_strided((1, 3, 64), (1, 64, 1)),                # one head at an odd stride
    flat(2 * 64).as_strided((2, 1, 64), (64, 3, 1)),                # one row at an odd stride
    flat(2 * 3 * 64).as_strided((1, 1, 64), (5, 7, 1)),
    flat(2 * 3 * 131)[: 2 * 3 * 131].view(2, 3, 131)[..., 1:65],    # rows at odd addresses
    flat(2 * 64 * 3).view(2, 64, 3).transpose(1, 2),                # dimensions three elements apart
    flat(2 * 3 * 64).view(2, 3, 64),
    flat(2 * 3 * 64).view(3, 2, 64).transpose(0, 1),
    flat(64)[None, None].expand(2, 3, 64),
])
def test_rows_come_back_as_the_kernels_read_them(x):
    y, p, sh, st = _rows(x)
    es = x.element_size()
    assert p == y.data_ptr() and p % 16 == 0 and sh * es % 16 == 0 and st * es % 16 == 0 and y.stride(-1) == 1
    # what a kernel finds at p + h sh + t st
    assert torch.equal(torch.as_strided(y, x.shape, (sh, st, 1)), x)


def test_rows_that_need_no_copy_are_not_copied():
    for x in (flat(2 * 3 * 64).view(2, 3, 64), flat(2 * 3 * 64).view(3, 2, 64).transpose(0, 1),
              flat(2 * 3 * 136).view(2, 3, 136)[..., 8:72]):
        assert _rows(x)[1] == x.data_ptr()


@pytest.mark.parametrize("which", [1, 3])
def test_pairs_at_an_odd_head_stride_are_refused(which):
    """(step, low) pairs are addressed as 32-bit words: heads an odd number of elements apart cannot be."""
    def buffers(stride, hk=2):
        b = [torch.zeros(hk, 10, 32, dtype=torch.uint8), torch.zeros(hk, 10, 1, 2, dtype=torch.bfloat16),
             torch.zeros(hk, 10, 32, dtype=torch.uint8), torch.zeros(hk, 10, 1, 2, dtype=torch.bfloat16)]
        b[which] = torch.zeros(64, dtype=torch.bfloat16).as_strided((hk, 10, 1, 2), (stride, 2, 2, 1))
        return b
    with pytest.raises(ValueError, match="pairs"):
        QuantKV.from_buffers(*buffers(21), bits=4)
    for kv in (QuantKV.from_buffers(*buffers(22), bits=4), QuantKV.from_buffers(*buffers(21, 1), bits=4)):
        assert kv.group == 64
    assert QuantKV.from_buffers(*buffers(22), bits=4)._struct.k_meta_h in (10, 11)
