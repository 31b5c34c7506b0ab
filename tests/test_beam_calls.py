"""Sizes of beam search and batched chunks that no launch can hold, refused by the C calls
before any GPU work: a launch has fewer than 2^32 threads."""
import pytest

from tests.test_beam_host import chunks, refused, select

BIG = dict(wb=1 << 60)


@pytest.mark.parametrize("call,status,needle", [
    # 2^24 rows of one workgroup of 256 threads, by groups and by the vocabulary
    (select(G=1 << 18, W=64, V=100, **BIG), 1, "logits too large"),
    (select(G=1 << 18, W=32, V=4097, **BIG), 1, "logits too large"),
    # few rows alone (256 threads), both kinds (pairs of them behind the tiles' 512)
    (chunks(B=1024, N=1 << 17, Hq=2049, Hkv=2049, gqa=1, new=128), 1, "grid too large"),
    (chunks(B=1024, N=300 * 1024, Hq=1171, Hkv=1171, gqa=1, new=300), 1, "grid too large"),
    (chunks(B=1, N=(1 << 22) - 1, Hq=255, Hkv=255, gqa=1, new=(1 << 22) - 1, D=512), 1, "grid too large"),
])
def test_grids_that_cannot_be_launched(call, status, needle):
    refused(*call, status, needle)
