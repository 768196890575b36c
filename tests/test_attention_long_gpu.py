"""Pieces of work that take longer than a wait's limit: what waits for them goes on as long as they do."""
import math

import pytest
import torch

from conftest import ROOT  # noqa: F401

pytestmark = pytest.mark.gpu


def test_a_piece_of_seconds():
    """150 million keys in one piece (many requests, so that the keys are not split): warps that wait for all of it wait for
    over a second.  A wait that runs out gives NaN to the rows of both requests.  The sum of equal weights is a multiple of 64
    below 2^30 in each thread, so exact; that of the values, in the tensor cores, drops bits over so many keys."""
    import vesper_db_b200 as V
    n, d, lens = 150_000_000, 8, [200] + [0] * 90 + [3]
    k = torch.zeros(n + 4, 1, d, dtype=torch.float16, device="cuda")
    v = torch.zeros(n + 4, 1, d, dtype=torch.float16, device="cuda")
    v[1:n:2] = 1
    v[n:] = 5
    q = torch.randn(sum(lens), 1, d, device="cuda").half()
    ints = lambda x: torch.tensor(x, dtype=torch.int32, device="cuda")  # noqa: E731
    starts = ints([0, 200] + [200] * 90 + [203])
    starts_k = ints([0, n] + [n] * 90 + [n + 4])
    out, lse = V.prompt_attention(q, k, v, starts, starts_k, causal=False, stats=True)
    assert torch.isfinite(out).all() and (out[200:] == 5).all()
    assert (lse[:200].double() - math.log(n)).abs().max() <= 2.0 ** -18 and (lse[200:] - math.log(4)).abs().max() <= 2.0 ** -20
    del k, v
    torch.cuda.empty_cache()
