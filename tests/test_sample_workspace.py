"""navi_sample_workspace: what suffices for a server's largest step suffices for its smaller ones."""
import numpy as np
import pytest
import torch

from navi_amd import abi


def test_it_does_not_fall_with_the_rows():
    """Across each change of the chunks' size: 26 rows of 151936 tokens are in smaller chunks than 27, 128 of 32000 than 129."""
    for vocab in (16385, 20000, 32000, 65536, 65537, 151936, 262144, 262145, 1 << 20):
        sizes = [abi.sample_workspace(rows, vocab) for rows in range(1, 260)]
        assert sizes == sorted(sizes) and sizes[0] > 0, vocab


def test_it_does_not_fall_with_the_vocabulary():
    vocabs = list(range(1000, 300000, 997)) + [262144, 262145, 1 << 19, 1 << 20]
    for rows in (1, 2, 15, 16, 17, 26, 27, 100, 204, 205, 1000):
        sizes = [abi.sample_workspace(rows, v) for v in sorted(vocabs)]
        assert sizes == sorted(sizes), rows


@pytest.mark.gpu
def test_one_buffer_for_fewer_rows_and_shorter_ones():
    from sample_util import Call
    most = abi.sample_workspace(40, 151936)
    g = torch.Generator().manual_seed(1)
    for rows, vocab in ((40, 151936), (26, 151936), (27, 151936), (1, 151936), (36, 110000), (40, 100000), (40, 16385), (40, 1000)):
        c = Call(torch.randn(rows, vocab, generator=g) * 3, [(0.9, 40, 0.95, 0.01, 1)], np.linspace(0, 0.99, rows))
        c.ws = torch.full((most,), 0xFF, dtype=torch.uint8, device="cuda")
        c.check()
