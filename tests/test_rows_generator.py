"""The generator behind dropout against its authors' published test vectors, with counter and key word by word."""

import random

import pytest
import torch

import rows_reference as ref


def words(counter, key):
    """Ten rounds of four 32-bit words, by the definition: products of 32-bit words, high halves crossed with the other pair, key words
    raised every round."""
    c, k = list(counter), list(key)
    for _ in range(10):
        a, b = 0xD2511F53 * c[0], 0xCD9E8D57 * c[2]
        c = [(b >> 32) ^ c[1] ^ k[0], b % 2 ** 32, (a >> 32) ^ c[3] ^ k[1], a % 2 ** 32]
        k = [(k[0] + 0x9E3779B9) % 2 ** 32, (k[1] + 0xBB67AE85) % 2 ** 32]
    return c


@pytest.mark.parametrize("counter,key,want", [
    ((0, 0, 0, 0), (0, 0), (0x6627E8D5, 0xE169C58D, 0xBC57AC4C, 0x9B00DBD8)),
    ((0xFFFFFFFF,) * 4, (0xFFFFFFFF,) * 2, (0x408F276D, 0x41C83B0E, 0xA20BC7C6, 0x6D5451FD)),
    ((0x243F6A88, 0x85A308D3, 0x13198A2E, 0x03707344), (0xA4093822, 0x299F31D0), (0xD16CFE09, 0x94FDCCEB, 0x5001E420, 0x24126EA1)),
])
def test_published(counter, key, want):
    assert tuple(words(counter, key)) == want


def test_where_the_numbers_stand():
    """The seed is the key and the offset the counter's second half, low words first; a word is two numbers, low half first."""
    rng = random.Random(1)
    for _ in range(20):
        seed, offset = rng.getrandbits(64), rng.getrandbits(64)
        bits = ref.bits16(seed, offset, 8 * 3)
        for block in range(3):
            got = words((block, 0, offset % 2 ** 32, offset >> 32), (seed % 2 ** 32, seed >> 32))
            assert torch.equal(bits[8 * block:8 * block + 8], torch.tensor([half for w in got for half in (w & 0xFFFF, w >> 16)]))
