"""Paged attention, append and adjusted logits where their kernels change form: rows that are not finite, pages that are not there, strides beyond 32 bits, sizes behind
which a launch is made another way."""
import pytest
import torch

from paged_cases import BF16, attention64, batch, within
from tensor_parallel_b200.ops import functional as OF

pytestmark = pytest.mark.gpu


def native():
    from tensor_parallel_b200.ops import native

    return native


def status_of(device="cuda"):
    word = native().device_state(torch.device(device)).status
    code = int(word[0])
    word.zero_()
    return code


def cache_of(b):
    return OF.PagedCache(b["keys"], b["values"], b["table"])


def attend(b, **kw):
    before = native().launch_count
    out = OF.paged_attention(b["q"], cache_of(b), b["starts"], b["past"], **kw)
    assert native().launch_count > before
    return out


@pytest.mark.parametrize("dim", [64, 128])
def test_values_that_a_row_does_not_see_yet(dim):
    """The largest numbers of the type in the values of later tokens of the same sequence."""
    b = batch([200], [40], 4, 2, dim, 16, device="cuda")
    want, tol = attention64(b)
    low = torch.finfo(BF16).min
    for at in range(100, 240):  # (tokens 60 and up see them)
        b["values"][b["table"][0, at // 16].long(), :, at % 16] = low
    within(attend(b)[:60], want[:60], tol[:60])
    want, tol = attention64(b, window=30)
    within(attend(b, window=30)[:60], want[:60], tol[:60])
