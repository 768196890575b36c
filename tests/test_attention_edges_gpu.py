"""The attention operators where sizes, argument kinds and non-finite values meet the edges of what they take."""
import math
import os
import subprocess
import sys

import pytest
import torch

from conftest import ROOT

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def V():
    import vesper_db_b200
    return vesper_db_b200


def rand(*shape, dtype=torch.bfloat16, seed=0, scale=1.0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return (torch.randn(shape, generator=g, device="cuda") * scale).to(dtype)


def ints(x, dtype=torch.int32):
    return torch.tensor(x, dtype=dtype, device="cuda")


# ------------------------------------------------------------------------------------------ page_tables
MANY_REQUESTS = """
import sys
import torch
import vesper_db_b200 as V
page, width = 16, 3
for n in map(int, sys.argv[1:]):
    i = torch.arange(n)
    cached, fresh = (i * 7) % 20, (i * 5) % 9
    had, need = (cached + page - 1) // page, (cached + fresh + page - 1) // page
    table = torch.where(torch.arange(width)[None] < had[:, None], i[:, None] * width + torch.arange(width)[None], -1)
    free = 100000 + torch.arange(int((need - had).sum()))
    starts = torch.cat([torch.zeros(1, dtype=torch.long), fresh.cumsum(0)])
    total = int(starts[-1])
    want = table.clone()
    fill = (torch.arange(width)[None] >= had[:, None]) & (torch.arange(width)[None] < need[:, None])
    want[fill] = free  # row by row: request order
    row = torch.repeat_interleave(i, fresh)
    at = cached[row] + torch.arange(total) - starts[row]
    slots = want[row, at // page] * page + at % page
    dev = lambda x: x.to(torch.int32).cuda()
    got = V.page_tables(dev(cached), dev(fresh), dev(free), dev(table), page, total, base=3)
    for name, a, b in zip(got._fields, got, (want, cached + fresh, starts, at + 3, slots, (need - had).sum()[None])):
        assert torch.equal(a.cpu().long(), b), (n, name)
print("as expected")
"""


@pytest.mark.parametrize("sizes", [[4073, 4074, 4095, 4096, 16384, 4090], [4095], [16384, 4074, 16384]])
def test_tables_request_counts_around_the_shared_memory_limit(V, sizes):
    """In a process of its own: what an earlier call opted in to must not matter."""
    r = subprocess.run([sys.executable, "-c", MANY_REQUESTS, *map(str, sizes)], cwd=ROOT, capture_output=True, text=True,
                       env={**os.environ, "PYTHONPATH": ROOT}, timeout=300)
    assert r.returncode == 0 and "as expected" in r.stdout, r.stderr[-2000:]


# ------------------------------------------------------------------------------------------ arguments
def refused(says, call):
    from vesper_db_b200 import VesperError
    with pytest.raises(VesperError, match=says):
        call()


def some_inputs():
    q, k, v = rand(5, 8, 64, seed=1), rand(5, 2, 64, seed=2), rand(5, 2, 64, seed=3)
    kc, vc = rand(4, 16, 2, 64, seed=4), rand(4, 16, 2, 64, seed=5)
    return q, k, v, kc, vc, ints([[0, 1]] * 5), ints([3] * 5), ints([2]), torch.zeros(9, 64, device="cuda")


def test_truth_values_that_have_none_are_refused(V):
    q, k, v, kc, vc, table, lens, pages, turns = some_inputs()
    two, starts, pos = torch.tensor([True, False]), ints([0, 5]), ints([0] * 5)
    refused("causal must be", lambda: V.prompt_attention(q, k, v, starts, causal=two))
    refused("stats must be", lambda: V.prompt_attention(q, k, v, starts, stats=two))
    refused("stats must be", lambda: V.shared_prefix_attention(q, kc, vc, pages, 9, table, lens, stats=two))
    refused("pairs must be", lambda: V.norm_rotate(q, k, v, pos, turns, pairs=two))
    refused("keep_k must be", lambda: V.norm_rotate(q, k, v, pos, turns, keep_k=two))


def test_inputs_that_require_a_gradient_are_refused(V):
    """There is no backward pass: a result that silently stands outside the graph would train on wrong gradients."""
    q, k, v, kc, vc, table, lens, pages, turns = some_inputs()
    starts, pos, slots = ints([0, 5]), ints([0] * 5), ints([0, 1, 2, 3, 4], torch.int64)
    w = torch.ones(64, dtype=torch.bfloat16, device="cuda")
    grad = lambda x: x.clone().requires_grad_()  # noqa: E731
    calls = [lambda g: V.prompt_attention(g(q), k, v, starts), lambda g: V.prompt_attention(q, g(k), v, starts),
             lambda g: V.prompt_attention(q, k, g(v), starts),
             lambda g: V.shared_prefix_attention(g(q), kc, vc, pages, 9, table, lens),
             lambda g: V.shared_prefix_attention(q, g(kc), vc, pages, 9, table, lens),
             lambda g: V.shared_prefix_attention(q, kc, g(vc), pages, 9, table, lens),
             lambda g: V.norm_rotate(g(q), k, v, pos, turns), lambda g: V.norm_rotate(q, g(k), v, pos, turns),
             lambda g: V.norm_rotate(q, k, g(v), pos, turns, slots=slots, k_cache=kc, v_cache=vc),
             lambda g: V.norm_rotate(q, k, v, pos, g(turns)), lambda g: V.norm_rotate(q, k, v, pos, turns, q_weight=g(w)),
             lambda g: V.norm_rotate(q, k, v, pos, turns, k_weight=g(w)),
             lambda g: V.norm_rotate(q, k, v, pos, turns, slots=slots, k_cache=g(kc), v_cache=vc),
             lambda g: V.norm_rotate(q, k, v, pos, turns, slots=slots, k_cache=kc, v_cache=g(vc))]
    for call in calls:
        refused("requires a gradient", lambda: call(grad))
        with torch.no_grad():
            call(grad)
        call(lambda x: grad(x).detach())


def test_tensors_written_in_place_count_the_write(V):
    q, k, v, kc, vc, table, lens, pages, turns = some_inputs()
    before = [t._version for t in (table, kc, vc)]
    V.page_tables(lens, lens, pages, table, 16, 15)
    V.norm_rotate(q, k, v, ints([0] * 5), turns, slots=ints([0, 1, 2, 3, 4], torch.int64), k_cache=kc, v_cache=vc)
    assert [t._version for t in (table, kc, vc)] == [n + 1 for n in before]
    both = rand(4, 2, 16, 2, 64)
    old = both._version
    V.norm_rotate(q, k, v, ints([0] * 5), turns, slots=ints([0] * 5, torch.int64), k_cache=both[:, 0], v_cache=both[:, 1])
    assert both._version > old
    with torch.inference_mode():  # such tensors have no version
        table, kc, vc = table.clone(), kc.clone(), vc.clone()
        V.page_tables(lens, lens, pages, table, 16, 15)
    V.norm_rotate(q, k, v, ints([0] * 5), turns, slots=ints([0] * 5, torch.int64), k_cache=kc, v_cache=vc)


# ------------------------------------------------------------------------------------------ values that are seen
@pytest.mark.parametrize("bad", [math.nan, math.inf])
def test_seen_values_reach_the_row_however_small_their_weight(V, bad):
    """Parts of a row's keys are computed apart and joined: a value that is not finite shows wherever it stands, also where
    its part's weight is zero in 32 bits (the definition gives it a weight above zero)."""
    d, heads = 64, 4
    # keys of the first part score -200, those of the second +200
    q = torch.ones(3, heads, d, dtype=torch.bfloat16, device="cuda")
    kc, vc = rand(8, 16, 2, d, seed=1), rand(8, 16, 2, d, seed=2)
    kc[:4], kc[4:] = -25, 25  # times 64 ones, scaled by 1 / 8
    pages, table = ints([0, 1, 2, 3]), ints([[4], [5], [6]])
    vc[2, 3, :, 7] = bad
    out = V.shared_prefix_attention(q, kc, vc, pages, 64, table, ints([16, 1, 9]))
    assert not torch.isfinite(out[..., 7]).any() and torch.isfinite(out[..., :7]).all()
    # a few queries over many packed keys: split over the keys, then joined
    n = 20000
    k, v = rand(n, 2, d, seed=3), rand(n, 2, d, seed=4)
    k[:n // 2], k[n // 2:] = -25, 25
    v[100, :, 9] = bad
    out = V.prompt_attention(q, k, v, ints([0, 3]), ints([0, n]), causal=False)
    assert not torch.isfinite(out[..., 9]).any() and torch.isfinite(out[..., :9]).all()
