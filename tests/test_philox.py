"""The oracle's generator against the published known answers of Philox4x32-10
(Random123's kat_vectors: zeros, ones and the digits of pi)."""
import pytest

from tests import attention_oracle as oracle


def rounds(counter, key):
    """Philox4x32-10 word by word, from Salmon et al., SC 2011."""
    c, k = list(counter), list(key)
    for _ in range(10):
        a, b = c[0] * 0xD2511F53, c[2] * 0xCD9E8D57
        c = [b >> 32 ^ c[1] ^ k[0], b & 0xffffffff, a >> 32 ^ c[3] ^ k[1], a & 0xffffffff]
        k = [(k[0] + 0x9E3779B9) & 0xffffffff, (k[1] + 0xBB67AE85) & 0xffffffff]
    return c


@pytest.mark.parametrize('counter,key,want', [
    ((0,) * 4, (0,) * 2, (0x6627e8d5, 0xe169c58d, 0xbc57ac4c, 0x9b00dbd8)),
    ((0xffffffff,) * 4, (0xffffffff,) * 2, (0x408f276d, 0x41c83b0e, 0xa20bc7c6, 0x6d5451fd)),
    ((0x243f6a88, 0x85a308d3, 0x13198a2e, 0x03707344), (0xa4093822, 0x299f31d0),
     (0xd16cfe09, 0x94fdcceb, 0x5001e420, 0x24126ea1))])
def test_published_answers(counter, key, want):
    assert tuple(rounds(counter, key)) == want


@pytest.mark.parametrize('key,offset', [(0x299f31d0a4093822, 0x0370734413198a2e), (-7, 1), (1, -(1 << 40)),
                                        (123456789, 0xffffffff)])
def test_oracle_takes_its_words_in_their_places(key, offset):
    """Keys and offsets whose halves differ: low words first, the counter's low half counts blocks of four."""
    low = 0xffffffff
    want = [w for block in range(5)
            for w in rounds((block, 0, offset & low, offset >> 32 & low), (key & low, key >> 32 & low))]
    assert [int(w) for w in oracle.philox(18, key, offset)] == want[:18]
