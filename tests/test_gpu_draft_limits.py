"""Drafted tokens and scores where numbers lie at the ends of their ranges: a NaN at the first token, paths that are none, tokens outside the
vocabulary, scores of texts of all lengths."""
import math

import pytest

from test_gpu_draft import _check_logprobs, dev, ints, trees

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
@pytest.mark.parametrize("rows,vocab,shift", [(12, 4, 0), (12, 20, 0), (12, 32, 1), (12, 33, 3), (12, 700, 1), (600, 700, 1), (12, 9001, 0), (600, 2500, 1), (12, 130001, 3), (200, 40000, 0)])
def test_a_nan_at_the_first_token(ctx, dtype, rows, vocab, shift):
    """It is the first alternative: alone, among others, in rows of nothing else. In rows of a warp, of a block and of a cluster; in a vector of loads and in front of the first."""
    import torch
    g = torch.Generator(device="cuda").manual_seed(vocab)
    x = torch.randn(rows, vocab + shift, generator=g, device="cuda")[:, shift:]
    x[::6, 0] = math.nan
    x[1::6] = math.nan
    x[2::6, :3] = math.nan
    x[3::6, 0], x[3::6, 1] = math.nan, math.inf
    x[4::6, 1:], x[4::6, 0] = -math.inf, math.nan
    x[5::6, vocab - 1] = math.nan
    wide = torch.empty(rows, vocab + shift, dtype=getattr(torch, dtype), device="cuda")
    wide[:, shift:] = x
    x = wide[:, shift:]
    tokens = torch.tensor([[0, vocab - 1]], dtype=torch.int32, device="cuda").expand(rows, 2).contiguous()
    for top in {1, min(vocab, 5), min(vocab, 32)}:
        _check_logprobs(x, tokens, top)
