"""Keys and values that are not finite: they reach the rows that see them, and no other row, wherever they stand."""
import math

import pytest
import torch

from conftest import ROOT  # noqa: F401
from test_attention_gpu import assert_near, rand, row_reference, starts_of

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def V():
    import vesper_db_b200
    return vesper_db_b200


def poisoned_call(V, *args, **kw):
    """The call with outputs and workspaces in memory that holds NaN: what is not written shows."""
    sizes = [t.numel() * t.element_size() for t in V.prompt_attention(*args, stats=True, **kw)]
    held = [torch.full((n // 4 + 1,), math.nan, device="cuda") for n in (*sizes, *sizes, 1 << 20)]
    del held
    return V.prompt_attention(*args, stats=True, **kw)


def check(V, q, k, v, lens, lens_k, causal=True, rows=None):
    """Every column of the rows (of each request: `rows`, or all) against the formula in 64 bits: where a row sees values
    that are not finite, their sum; elsewhere the finite ones', which the others must not have touched."""
    heads, kv, d = q.shape[1], k.shape[1], q.shape[2]
    out, lse = poisoned_call(V, q, k, v, starts_of(lens), None if lens_k is None else starts_of(lens_k), causal=causal)
    a = b = 0
    for n, m in zip(lens, lens if lens_k is None else lens_k):
        for r0 in range(0, n, 512):
            r1 = min(n, r0 + 512)
            if rows is not None and not any(r0 <= r < r1 for r in rows):
                continue
            row, col = torch.arange(r0, r1, device="cuda")[:, None], torch.arange(m, device="cuda")[None]
            seen = (col <= row + m - n) if causal else (col < m).expand(r1 - r0, m)
            vals = v[b:b + m].double()
            finite = torch.isfinite(vals)
            o, l, err, lse_err = row_reference(q[a + r0:a + r1], k[b:b + m], torch.where(finite, vals, 0.0).to(v.dtype), seen,
                                               d ** -0.5, q.dtype)
            count = lambda x: torch.einsum("qk,khd->qhd", seen.double(), x.double()).repeat_interleave(heads // kv, 1)  # noqa: E731
            up, down, nan = (count(vals == math.inf) > 0, count(vals == -math.inf) > 0, count(vals.isnan()) > 0)
            got = out[a + r0:a + r1]
            assert_near(torch.where(up | down | nan, 0.0, got), torch.where(up | down | nan, 0.0, o), err, f"rows {r0}..{r1}")
            assert got[nan | (up & down)].isnan().all()
            assert (got[up & ~down & ~nan] == math.inf).all() and (got[down & ~up & ~nan] == -math.inf).all()
            assert_near(lse[a + r0:a + r1], l, lse_err, f"lse of rows {r0}..{r1}")
        a, b = a + n, b + m


def inputs(nq, nk, heads, kv, d, dtype=torch.bfloat16, seed=0):
    return (rand(nq, heads, d, dtype=dtype, seed=seed), rand(nk, kv, d, dtype=dtype, seed=seed + 1),
            rand(nk, kv, d, dtype=dtype, seed=seed + 2))


@pytest.mark.parametrize("heads,kv,d", [(4, 4, 64), (2, 2, 128), (8, 2, 128), (6, 2, 64)])
def test_one_query_tile_done_before_the_other(V, heads, kv, d):
    """The two query tiles of a piece end at different key tiles: values that only the later one sees, in every piece, while
    the earlier one's results are written.  Each row comes whole, again and again."""
    lens = [700, 1, 1300, 515]
    q, k, v = inputs(sum(lens), sum(lens), heads, kv, d, seed=heads)
    for t in range(40, sum(lens), 90):
        v[t, :, (t * 7) % d] = (math.nan, math.inf, -math.inf)[t % 3]
    check(V, q, k, v, lens, None)
    first, first_lse = poisoned_call(V, q, k, v, starts_of(lens))
    for _ in range(20):
        again, lse = poisoned_call(V, q, k, v, starts_of(lens))
        assert torch.equal(again.view(torch.int16), first.view(torch.int16)) and torch.equal(lse, first_lse)


@pytest.mark.parametrize("heads,kv", [(2, 2), (8, 2)])
def test_unseen_values_where_the_keys_are_split(V, heads, kv):
    """Few queries after many keys: the parts that the splits leave, joined."""
    lens, lens_k = [300], [9000]
    q, k, v = inputs(300, 9000, heads, kv, 64, torch.float16, seed=5)
    v[8790, :, 3], v[8950, :, 40], v[8951, 0, 40] = math.nan, math.inf, -math.inf
    check(V, q, k, v, lens, lens_k)


@pytest.mark.parametrize("heads,kv,d", [(8, 8, 128), (16, 4, 64)])
def test_unseen_values_at_the_end_of_a_long_prompt(V, heads, kv, d):
    """More pieces than blocks, and one that holds an unseen value after 16,000 keys: neither its rows nor those of the
    pieces that its block takes next are touched."""
    lens = [16384, 900]
    q, k, v = inputs(sum(lens), sum(lens), heads, kv, d, seed=1)
    v[16200, :, 5], v[16384 + 800, :, 9] = math.nan, math.inf
    out, lse = poisoned_call(V, q, k, v, starts_of(lens))
    assert torch.isfinite(lse).all()
    unseen = torch.ones_like(out, dtype=torch.bool)
    unseen[16200:16384, :, 5] = unseen[16384 + 800:, :, 9] = False
    assert torch.isfinite(out[unseen]).all() and not torch.isfinite(out[~unseen]).any()
    check(V, q, k, v, lens, None, rows=(0, 600, 850, 16199, 16200, 16300))


def test_unseen_values_in_every_piece_of_a_long_prompt(V):
    """A column of values that is not finite in every thirtieth token: the other columns are right."""
    lens, heads, kv, d = [16384], 8, 4, 128
    q, k, v = inputs(16384, 16384, heads, kv, d, seed=2)
    v[::30, :, 77] = math.nan
    v[29::30, :, 3] = -math.inf
    out, lse = poisoned_call(V, q, k, v, starts_of(lens))
    assert torch.isfinite(lse).all()
    others = torch.arange(d, device="cuda")
    assert torch.isfinite(out[..., (others != 77) & (others != 3)]).all()
    assert out[..., 77].isnan().all() and torch.isfinite(out[:29, :, 3]).all() and (out[29:, :, 3] == -math.inf).all()
    check(V, q, k, v, lens, None, rows=(0, 129, 5000, 16383))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("heads,kv,d", [(7, 1, 128), (6, 2, 96), (2, 1, 40), (3, 3, 8), (24, 1, 72), (128, 1, 128)])
def test_unseen_values_in_every_head_layout(V, dtype, heads, kv, d):
    """Prompts on the tensor-memory tiles, and continued ones with fewer and with more keys than queries."""
    for lens, lens_k in (([700, 1, 333, 1300], None), ([600, 500], [900, 300])):
        nk = sum(lens if lens_k is None else lens_k)
        q, k, v = inputs(sum(lens), nk, heads, kv, d, dtype, seed=d)
        for t in range(5, nk, 61):
            v[t, :, (t * 5) % d] = (math.nan, math.inf, -math.inf)[t % 3]
        check(V, q, k, v, lens, lens_k)


# ------------------------------------------------------------------------------------------ short prompts, small blocks
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("heads,kv,d", [(8, 2, 128), (4, 4, 64), (7, 1, 128), (6, 2, 96), (2, 1, 40), (3, 3, 8), (64, 1, 64)])
def test_unseen_values_in_short_prompts(V, dtype, heads, kv, d):
    for lens, lens_k in (([1, 33, 0, 130, 97, 2], None), ([5, 64, 0, 70], [30, 64, 9, 41])):
        nk = sum(lens if lens_k is None else lens_k)
        q, k, v = inputs(sum(lens), nk, heads, kv, d, dtype, seed=d + 1)
        for t in range(3, nk, 13):
            v[t, :, (t * 5) % d] = (math.nan, math.inf, -math.inf)[t % 3]
        check(V, q, k, v, lens, lens_k)


def test_unseen_values_in_a_long_prompt_among_short_ones(V):
    """By their mean these go to the small blocks, the long one too."""
    lens = [3] * 400 + [6000] + [20] * 100
    q, k, v = inputs(sum(lens), sum(lens), 4, 2, 64, seed=3)
    v[7::31, 0, 11] = math.nan
    check(V, q, k, v, lens, None)


def test_unseen_values_cost_no_more_than_looking_for_them(V):
    """200 prompts of 100 tokens with one such value in thirty tokens: ten times the time without is far more than one more
    look at the values takes, and far less than computing rows again."""
    n, lens = 20000, starts_of([100] * 200)
    q, k, v = inputs(n, n, 12, 12, 64)

    def time():
        for _ in range(3):
            V.prompt_attention(q, k, v, lens)
        a, b = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
        a.record()
        for _ in range(10):
            V.prompt_attention(q, k, v, lens)
        b.record()
        torch.cuda.synchronize()
        return a.elapsed_time(b)
    clean = time()
    v[::30, :, 3] = math.nan
    assert time() < 10 * clean
