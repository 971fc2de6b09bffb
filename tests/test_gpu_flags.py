"""The flag words by which CTAs of one launch hand partial sums to one another (the cut tiles of the layer
products).  A launch in a CUDA graph is replayed with the same token and the same words, so a word must come
out of every launch clean: also when the taker's bounded wait ran out and the giver came after that."""

import pytest
import torch

pytestmark = pytest.mark.gpu

TOKEN = 0x9E3779B97F4A7C15


@pytest.mark.parametrize("before", [0, 1, -1, 0x7FC0000000000000])  # whatever the scratch held
@pytest.mark.parametrize("late", [0, 1])
def test_a_word_is_clean_after_giver_and_taker(late, before):
    from kvstreams import _native as N

    word = torch.full((1,), before, dtype=torch.long, device="cuda")
    out = torch.full((3,), -1, dtype=torch.int32, device="cuda")
    rc = N.lib().kvs_selftest_flag(late, 64, TOKEN, word.data_ptr(), out.data_ptr(), N.stream_ptr(out.device))
    assert rc == 0
    seen, clean, stale = out.tolist()
    assert seen == 1 - late
    assert clean == 1
    assert stale == 0  # the next replay does not take the earlier launch's flag for its own


def test_refusals():
    from kvstreams import _native as N

    t = torch.zeros(4, dtype=torch.long, device="cuda")
    p, s = t.data_ptr(), N.stream_ptr(t.device)
    for late, polls, token, flag, out in ((2, 1, 5, p, p + 8), (-1, 1, 5, p, p + 8), (0, 0, 5, p, p + 8),
                                          (0, 1, 0, p, p + 8), (0, 1, 2**64 - 1, p, p + 8), (0, 1, 5, None, p + 8),
                                          (0, 1, 5, p, None)):
        assert N.lib().kvs_selftest_flag(late, polls, token, flag, out, s) == -1
