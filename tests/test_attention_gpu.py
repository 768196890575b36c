"""Attention over retrieved passages: every operator against its definition in 64 bits.

Tolerances are bounds, not fits: the 64-bit value, moved by the error that 32-bit arithmetic may make, and then rounded
to the 16-bit type, must enclose the result.  With u the largest relative rounding error of the type (2^-8 bf16: eight
bits of precision; 2^-11 f16), n keys, P_j the softmax, A = sum_j P_j |v_j|, S = scale * max_j sum_i |q_i k_ji|:
  * each probability is rounded once (u A);
  * a score is a sum of head_dim products in 32 bits: off by at most head_dim 2^-24 S, its exponential by that much
    relative, both in the numerator and the sum; the exponential itself by at most 2^-18 relative;
  * the sums over keys run in 32 bits: n 2^-24 A; an f16 probability below 2^-14 is off by 2^-25 absolute.
"""
import math

import pytest
import torch

from conftest import ROOT  # noqa: F401

pytestmark = pytest.mark.gpu

U = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}
TYPES = [torch.bfloat16, torch.float16]


@pytest.fixture(scope="module")
def V():
    import vesper_db_b200
    return vesper_db_b200


def rand(*shape, dtype=torch.bfloat16, seed=0, scale=1.0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return (torch.randn(shape, generator=g, device="cuda") * scale).to(dtype)


def ints(x, dtype=torch.int32):
    return torch.tensor(x, dtype=dtype, device="cuda")


def starts_of(lens):
    return ints([0] + list(torch.tensor(lens, dtype=torch.int64).cumsum(0).tolist()) if len(lens) else [0])


def row_reference(q, k, v, seen, scale, dtype):
    """64-bit attention of q [lq, heads, d] over k, v [lk, kv, d] with the boolean mask seen [lq, lk]: out, lse, and the
    error bounds of both."""
    lq, heads, d = q.shape
    lk, kv = k.shape[:2]
    if lk == 0:
        z = torch.zeros(lq, heads, d, dtype=torch.float64, device="cuda")
        inf = torch.full((lq, heads), -math.inf, dtype=torch.float64, device="cuda")
        return z, inf, torch.zeros_like(z), torch.zeros_like(inf)
    q, k, v = q.double(), k.double().repeat_interleave(heads // kv, 1), v.double().repeat_interleave(heads // kv, 1)
    x = torch.einsum("qhd,khd->hqk", q, k) * scale
    x = torch.where(seen[None], x, -math.inf)
    mag = torch.einsum("qhd,khd->hqk", q.abs(), torch.where(seen.any(0)[:, None, None], k, 0.0).abs()) * scale
    mag = torch.where(seen[None], mag, 0.0).amax(-1).T  # [lq, heads]
    some = seen.any(1)
    top = torch.where(some, x.amax(-1), 0.0)
    p = torch.exp(x - top[..., None])
    total = p.sum(-1)
    lse = (top + total.log()).T
    p = torch.where(some[:, None], p / total[..., None], 0.0)
    vz = torch.where(seen.any(0)[:, None, None], v, 0.0)

    def mean(values):  # masked keys take no part, whatever they hold
        return torch.einsum("hqk,khd->qhd", p, values)
    out, a = mean(vz), mean(vz.abs())
    n, u = seen.sum(1)[:, None], U[dtype]
    delta = (d + 1) * 2.0 ** -24 * mag + 2.0 ** -18 + n * 2.0 ** -24
    err = (u + 2 * delta)[..., None] * a + (n * 2.0 ** -25)[..., None] * vz.abs().amax((0, 2), keepdim=True) + 1e-30
    return out, lse, err, delta + 2.0 ** -22 * lse.abs().nan_to_num(posinf=0.0)


def assert_near(got, want, err, what):
    """got, of its type, lies between the roundings of want - err and want + err to that type."""
    low, high = (want - err).to(got.dtype), (want + err).to(got.dtype)
    bad = ~((low <= got) & (got <= high))
    off = (got.double() - want).abs()
    assert not bad.any(), f"{what}: {int(bad.sum())} of {bad.numel()} off, worst {(off / err).nan_to_num(posinf=9e9).max():.3g} bounds"


def check_prompt(V, lens, lens_k, heads, kv, d, dtype, causal, seed=0, scale=None, mul=2.0, tail=0, edit=None):
    starts = starts_of(lens)
    starts_k = None if lens_k is None else starts_of(lens_k)
    lk = lens if lens_k is None else lens_k
    nq, nk = sum(lens) + tail, sum(lk) + (tail if lens_k is None else 0)
    q = rand(nq, heads, d, dtype=dtype, seed=seed, scale=mul)
    fused = rand(nk, 2 * kv, d, dtype=dtype, seed=seed + 1)
    k, v = fused[:, :kv], fused[:, kv:]
    if edit:
        edit(q, k, v)
    out, lse = V.prompt_attention(q, k, v, starts, starts_k, causal=causal, scale=scale, stats=True)
    alone = V.prompt_attention(q, k, v, starts, starts_k, causal=causal, scale=scale)
    assert torch.equal(out.view(torch.int16), alone.view(torch.int16)), "stats change the result"
    s = d ** -0.5 if scale is None else scale
    a = b = 0
    for i, (n, m) in enumerate(zip(lens, lk)):
        for r0 in range(0, n, 1024):
            r1 = min(n, r0 + 1024)
            row = torch.arange(r0, r1, device="cuda")[:, None]
            col = torch.arange(m, device="cuda")[None]
            seen = (col <= row + m - n) if causal else (col < m).expand(r1 - r0, m)
            o, l, e, el = row_reference(q[a + r0:a + r1], k[b:b + m], v[b:b + m], seen, s, dtype)
            assert_near(out[a + r0:a + r1], o, e, f"request {i} rows {r0}..{r1}")
            assert_near(lse[a + r0:a + r1], l, el, f"lse of request {i} rows {r0}..{r1}")
        a, b = a + n, b + m
    assert not out[a:].any() and bool(torch.isneginf(lse[a:]).all())
    return out, lse


# ------------------------------------------------------------------------------------------ prompt_attention
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("heads,kv,d", [(8, 2, 128), (4, 4, 64), (7, 1, 128), (6, 2, 96), (2, 1, 40), (3, 3, 8),
                                        (16, 1, 64), (24, 1, 72)])
def test_prompt_heads_and_types(V, dtype, causal, heads, kv, d):
    check_prompt(V, [1, 33, 0, 130, 257], None, heads, kv, d, dtype, causal, seed=heads)


@pytest.mark.parametrize("lens", [[1], [2, 1, 1], [127], [128], [129], [255, 256, 257], [0, 0, 5, 0], [1023, 1, 640],
                                  list(range(1, 70)), [3000]])
@pytest.mark.parametrize("causal", [True, False])
def test_prompt_lengths(V, lens, causal):
    check_prompt(V, lens, None, 8, 2, 128, torch.bfloat16, causal, seed=len(lens))


@pytest.mark.parametrize("lens,lens_k", [([1, 5, 64], [400, 5, 1000]), ([64], [8000]), ([3, 200, 40, 9], [0, 70, 40, 128]),
                                         ([300], [129]), ([1, 1], [1, 20000])])
@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("d", [64, 128])
def test_prompt_continued_and_rows_without_keys(V, lens, lens_k, causal, d):
    """Keys before the queries, and fewer keys than queries: the first rows then see none."""
    check_prompt(V, lens, lens_k, 8, 2, d, torch.bfloat16, causal, seed=11)


def test_prompt_padding_rows(V):
    check_prompt(V, [40, 200], None, 4, 1, 128, torch.float16, True, tail=37)


def test_prompt_no_requests(V):
    q, k = rand(5, 4, 64), rand(5, 2, 64)
    out, lse = V.prompt_attention(q, k, k, ints([0]), stats=True)
    assert not out.any() and bool(torch.isneginf(lse).all())
    assert V.prompt_attention(q[:0], k[:0], k[:0], ints([0])).shape == (0, 4, 64)
    out = V.prompt_attention(q, k[:0], k[:0], ints([0, 5]), ints([0, 0]))
    assert not out.any()


@pytest.mark.parametrize("mul,scale", [(40.0, None), (1.0, 3.0), (1.0, 1e-3), (0.0, None)])
def test_prompt_score_ranges(V, mul, scale):
    """Peaked and flat rows, and a maximum that grows along the keys (every block has to rescale)."""
    def rising(q, k, v):
        k *= torch.linspace(0.05, 1, k.shape[0], device="cuda")[:, None, None].to(k.dtype)
    check_prompt(V, [700], None, 4, 2, 128, torch.bfloat16, True, mul=mul, scale=scale, edit=rising)


def test_prompt_very_low_then_high_scores(V):
    """The first blocks' scores are far below the later ones (and below zero), then the other way round."""
    def edit(q, k, v):
        q[:], sign = 1, torch.where(torch.arange(k.shape[0], device="cuda") < k.shape[0] // 2, -6.0, 4.0)
        k[:] = sign[:, None, None].to(k.dtype)
    check_prompt(V, [900], None, 4, 2, 128, torch.bfloat16, False, edit=edit)
    check_prompt(V, [900], None, 4, 2, 128, torch.bfloat16, True, edit=edit)
    check_prompt(V, [900], None, 4, 2, 128, torch.bfloat16, False, edit=lambda q, k, v: (edit(q, k, v), k.neg_()))


@pytest.mark.parametrize("bad", [math.nan, math.inf, -math.inf])
@pytest.mark.parametrize("d", [64, 128])
def test_prompt_unseen_keys_and_values_do_not_leak(V, bad, d):
    """Later tokens of the same prompt, and neighbouring prompts, hold NaN or infinity: rows that do not see them stay
    right, bit for bit."""
    lens = [130, 70, 260]
    n, heads, kv = sum(lens), 8, 2
    q, k, v = rand(n, heads, d, seed=1), rand(n, kv, d, seed=2), rand(n, kv, d, seed=3)
    clean, clean_lse = V.prompt_attention(q, k, v, starts_of(lens), stats=True)
    k2, v2 = k.clone(), v.clone()
    hit = [100, 130 + 69, 200 + 37, 200 + 38]  # tokens 100, 69, 37, 38 of the three prompts
    for t in hit:
        k2[t, 0], v2[t, 1] = bad, bad
    out, lse = V.prompt_attention(q, k2, v2, starts_of(lens), stats=True)
    for a, e, first in ((0, 130, 100), (130, 200, 199), (200, 460, 237)):
        got, want = out[a:first].double(), clean[a:first].double()
        assert torch.isfinite(got).all()
        assert (got - want).abs().max() <= 2.0 ** -7 * want.abs().max()
        # head 0 of the keys hits its scores, head 1 its values: from the first hit on the values are not finite
        assert not torch.isfinite(out[first:e, 4:]).any()
        assert torch.equal(lse[a:e, 4:], clean_lse[a:e, 4:])
    # a prompt that only neighbours the bad tokens
    only = V.prompt_attention(q, k2, v2, starts_of(lens), causal=False)
    assert not torch.isfinite(only[:, 4:]).any()
    v3 = v.clone()
    v3[130:200] = bad
    k3 = k.clone()
    k3[130:200] = bad
    for causal in (True, False):
        want = V.prompt_attention(q, k, v, starts_of(lens), causal=causal)
        got = V.prompt_attention(q, k3, v3, starts_of(lens), causal=causal)
        assert torch.equal(got[:130], want[:130]) and torch.equal(got[200:], want[200:])


def test_prompt_bad_starts_stay_in_bounds(V):
    """Starts that leave the tensors, or run backwards, are bounded: nothing outside is read or written."""
    q, k = rand(50, 4, 64), rand(50, 2, 64)
    out = V.prompt_attention(q, k, k, ints([0, 20, 90]), causal=True)
    good = V.prompt_attention(q, k, k, ints([0, 20, 50]), causal=True)
    assert torch.equal(out, good)
    V.prompt_attention(q, k, k, ints([-3, 20, 10, 2 ** 31 - 1]), causal=False)
    torch.cuda.synchronize()


def test_prompt_strides(V):
    """Slices of a projection's output, heads before tokens, one token, and a stream that is not the default one."""
    x = rand(300, 12, 128, seed=5)
    q, k, v = x[:, :8], x[:, 8:10], x[:, 10:]
    want = V.prompt_attention(q.contiguous(), k.contiguous(), v.contiguous(), ints([0, 300]))
    assert torch.equal(V.prompt_attention(q, k, v, ints([0, 300])), want)
    qt, kt, vt = (t.transpose(0, 1).contiguous().transpose(0, 1) for t in (q, k, v))
    assert torch.equal(V.prompt_attention(qt, kt, vt, ints([0, 300])), want)
    assert torch.equal(V.prompt_attention(q[::2], k[::2], v[::2], ints([0, 150])),
                       V.prompt_attention(q[::2].contiguous(), k[::2].contiguous(), v[::2].contiguous(), ints([0, 150])))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = V.prompt_attention(q, k, v, ints([0, 300]))
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(got, want)


def test_prompt_repeats_bit_for_bit(V):
    q, k, v = rand(700, 8, 128, seed=1), rand(9000, 2, 128, seed=2), rand(9000, 2, 128, seed=3)
    args = (q, k, v, ints([0, 3, 700]), ints([0, 8000, 9000]))
    first = V.prompt_attention(*args)
    for _ in range(3):
        assert torch.equal(V.prompt_attention(*args), first)


# ------------------------------------------------------------------------------------------ shared prefix
def make_cache(pages, page, kv, d, dtype, seed, layout="plain"):
    if layout == "joined":  # keys and values of a page side by side
        both = rand(pages, 2, page, kv, d, dtype=dtype, seed=seed)
        return both[:, 0], both[:, 1]
    if layout == "heads":  # [pages, kv_heads, page_size, head_dim]
        k, v = rand(pages, kv, page, d, dtype=dtype, seed=seed), rand(pages, kv, page, d, dtype=dtype, seed=seed + 1)
        return k.transpose(1, 2), v.transpose(1, 2)
    return rand(pages, page, kv, d, dtype=dtype, seed=seed), rand(pages, page, kv, d, dtype=dtype, seed=seed + 1)


def check_shared(V, lens, prefix, heads, kv, d, dtype, page, seed=0, layout="plain", scale=None, mul=2.0, spoil=None):
    b, shared = len(lens), -(-prefix // page)
    need = [-(-n // page) for n in lens]
    total = shared + sum(need) + 2
    g = torch.Generator().manual_seed(seed)
    order = torch.randperm(total, generator=g).to(torch.int32)
    table = torch.full((b, max(need, default=0) + 2), -1, dtype=torch.int32)
    at = shared
    for i, n in enumerate(need):
        table[i, :n] = order[at:at + n]
        at += n
    kc, vc = make_cache(total, page, kv, d, dtype, seed + 7, layout)
    k_rows, v_rows = kc.clone(), vc.clone()
    if spoil is not None:  # everything that no request may see
        used = torch.zeros(total, page, dtype=torch.bool)
        for pages, n in [(order[:shared], prefix)] + [(table[i, :need[i]], n) for i, n in enumerate(lens)]:
            for j, p in enumerate(pages.tolist()):
                used[p, :min(page, n - j * page)] = True
        kc[~used.cuda()] = spoil
        vc[~used.cuda()] = spoil
    q = rand(b, heads, d, dtype=dtype, seed=seed + 3, scale=mul)
    prefix_pages, table_d = order[:shared].cuda(), table.cuda()
    out, lse = V.shared_prefix_attention(q, kc, vc, prefix_pages, prefix, table_d, ints(lens), scale=scale, stats=True)
    assert torch.equal(V.shared_prefix_attention(q, kc, vc, prefix_pages, prefix, table_d, ints(lens), scale=scale), out)
    s = d ** -0.5 if scale is None else scale
    for i, n in enumerate(lens):
        k, v = (torch.cat([x[order[:shared].long().cuda()].reshape(-1, kv, d)[:prefix],
                           x[table[i, :need[i]].long().cuda()].reshape(-1, kv, d)[:n]]) for x in (k_rows, v_rows))
        seen = torch.ones(1, k.shape[0], dtype=torch.bool, device="cuda")
        o, l, e, el = row_reference(q[i:i + 1], k, v, seen, s, dtype)
        # two parts joined: one more product with a weight in 32 bits each
        assert_near(out[i:i + 1], o, e * (1 + 2.0 ** -20), f"request {i}")
        assert_near(lse[i:i + 1], l, el + 2.0 ** -22, f"lse of request {i}")
    return out


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("heads,kv,d", [(8, 2, 128), (4, 4, 64), (7, 1, 128), (28, 4, 128), (6, 2, 96), (2, 1, 40),
                                        (3, 3, 8), (32, 1, 64), (48, 2, 128), (100, 1, 64)])
def test_shared_heads_and_types(V, dtype, heads, kv, d):
    check_shared(V, [1, 0, 77, 160, 33], 300, heads, kv, d, dtype, 16, seed=heads)


@pytest.mark.parametrize("page", [16, 32, 64, 128, 256])
@pytest.mark.parametrize("layout", ["plain", "joined", "heads"])
def test_shared_pages_and_layouts(V, page, layout):
    check_shared(V, [5, 300, 128], 515, 8, 2, 128, torch.bfloat16, page, seed=page, layout=layout)


@pytest.mark.parametrize("prefix", [0, 1, 15, 16, 127, 128, 129, 1000, 5003])
@pytest.mark.parametrize("lens", [[0], [1], [0, 0, 3], [513, 2]])
def test_shared_lengths(V, prefix, lens):
    check_shared(V, lens, prefix, 8, 2, 128, torch.bfloat16, 32, seed=prefix)


@pytest.mark.parametrize("b", [1, 31, 32, 33, 65, 150])
def test_shared_batches(V, b):
    check_shared(V, [(7 * i) % 91 for i in range(b)], 700, 8, 2, 128, torch.bfloat16, 16, seed=b)


def test_shared_long(V):
    check_shared(V, [9000, 1, 2500], 12345, 16, 2, 128, torch.bfloat16, 64, seed=5)
    check_shared(V, [20000], 0, 4, 1, 64, torch.float16, 128, seed=6)


@pytest.mark.parametrize("mul,scale", [(40.0, None), (1.0, 3.0), (0.0, None)])
def test_shared_score_ranges(V, mul, scale):
    check_shared(V, [200, 30], 400, 8, 2, 128, torch.bfloat16, 16, mul=mul, scale=scale)


@pytest.mark.parametrize("spoil", [math.nan, math.inf])
@pytest.mark.parametrize("page", [16, 64])
def test_shared_unused_slots_do_not_leak(V, spoil, page):
    check_shared(V, [1, 0, 77, 160, 33], 300, 8, 2, 128, torch.bfloat16, page, seed=9, spoil=spoil)
    check_shared(V, [1, 0, 77], 0, 8, 2, 64, torch.float16, page, seed=9, spoil=spoil)


def test_shared_bad_pages_and_lengths_stay_in_bounds(V):
    """Page numbers outside the cache read as zero keys and values; lengths are cut to the table."""
    kc, vc = rand(4, 16, 2, 64, seed=1), rand(4, 16, 2, 64, seed=2)
    q = rand(2, 4, 64, seed=3)
    table = ints([[3, 900], [-7, 2]])
    pages = ints([0, 77])
    got = V.shared_prefix_attention(q, kc, vc, pages, 30, table, ints([32, 999]))
    zero = torch.zeros(1, 16, 2, 64, dtype=kc.dtype, device="cuda")
    kz, vz = torch.cat([kc, zero]), torch.cat([vc, zero])
    want = V.shared_prefix_attention(q, kz, vz, ints([0, 4]), 30, ints([[3, 4], [4, 2]]), ints([32, 32]))
    assert torch.equal(got, want)
    got = V.shared_prefix_attention(q, kc, vc, pages, 30, table, ints([-5, 0]))
    want = V.shared_prefix_attention(q, kz, vz, ints([0, 4]), 30, table, ints([0, 0]))
    assert torch.equal(got, want)


def test_shared_cache_past_32_bit_offsets(V):
    """A cache of over 2^31 elements: pages at its end."""
    page, kv, d = 256, 8, 128
    pages = 2 ** 31 // (page * kv * d) + 40
    kc = torch.zeros(pages, page, kv, d, dtype=torch.bfloat16, device="cuda")
    vc = torch.zeros_like(kc)
    small_k, small_v = rand(8, page, kv, d, seed=1), rand(8, page, kv, d, seed=2)
    kc[-8:], vc[-8:] = small_k, small_v
    q = rand(3, 16, d, seed=3)
    last = pages - 8
    got = V.shared_prefix_attention(q, kc, vc, ints([last, last + 1]), 400, ints([[last + 2, last + 7]] * 3), ints([500, 3, 0]))
    want = V.shared_prefix_attention(q, small_k, small_v, ints([0, 1]), 400, ints([[2, 7]] * 3), ints([500, 3, 0]))
    assert torch.equal(got, want)
    slots = ints([(pages - 1) * page + 5, last * page], torch.int64)
    x = rand(2, 16 + 2 * kv, d, seed=4)
    turns = torch.ones(4, d, device="cuda")
    _, k = V.norm_rotate(x[:, :16], x[:, 16:16 + kv], x[:, 16 + kv:], ints([1, 2]), turns, slots=slots, k_cache=kc, v_cache=vc)
    assert torch.equal(kc[pages - 1, 5], k[0]) and torch.equal(vc[last, 0], x[1, 16 + kv:])
    del kc, vc
    torch.cuda.empty_cache()


def test_shared_matches_prompt_attention(V):
    """The same keys, packed and in pages, through both operators."""
    page, kv, d, heads = 32, 2, 128, 8
    kc, vc = rand(40, page, kv, d, seed=1), rand(40, page, kv, d, seed=2)
    q = rand(3, heads, d, seed=3)
    lens, prefix = [50, 9, 400], 333
    table = torch.arange(11, 37, dtype=torch.int32, device="cuda")[:26].view(2, 13)
    table = torch.cat([table, table[:1]])
    got, lse = V.shared_prefix_attention(q, kc, vc, torch.arange(11, dtype=torch.int32, device="cuda"), prefix, table,
                                         ints(lens), stats=True)
    k, v = (torch.cat([torch.cat([x[:11].reshape(-1, kv, d)[:prefix], x[table[i].long()].reshape(-1, kv, d)[:n]])
                       for i, n in enumerate(lens)]) for x in (kc, vc))
    want, want_lse = V.prompt_attention(q, k, v, ints([0, 1, 2, 3]), starts_of([prefix + n for n in lens]), stats=True)
    assert (got.double() - want.double()).abs().max() <= 2.0 ** -7 * want.double().abs().max()
    assert (lse - want_lse).abs().max() <= 1e-4


# ------------------------------------------------------------------------------------------ norm and rotation
def rotate_reference(x, w, turns, pos, eps, pairs):
    x = x.double()
    if w is not None:
        x = x / torch.sqrt(x.square().mean(-1, keepdim=True) + eps) * w.double()
    r = turns.shape[1]
    size = x.abs().clone()
    if r:
        i = torch.arange(r, device="cuda")
        ang, mate = (i // 2, i ^ 1) if pairs else (i % (r // 2), (i + r // 2) % r)
        low = (i % 2 == 0) if pairs else (i < r // 2)
        cos, sin = (turns[pos.long()][:, None, o + ang].double() for o in (0, r // 2))
        a = x[..., :r]
        b = a[..., mate]
        size[..., :r] = a.abs() + b.abs()
        x = torch.cat([a * cos + torch.where(low, -1.0, 1.0) * b * sin, x[..., r:]], -1)
    return x, size


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("heads,kv,d,turned", [(32, 8, 128, 128), (4, 4, 64, 32), (7, 1, 256, 256), (6, 2, 96, 96),
                                               (5, 5, 40, 16), (3, 1, 8, 0), (2, 2, 192, 64)])
@pytest.mark.parametrize("pairs", [False, True])
@pytest.mark.parametrize("norm", [True, False])
def test_norm_rotate(V, dtype, heads, kv, d, turned, pairs, norm):
    t, page, pages = 37, 16, 5
    x = rand(t, heads + 2 * kv, d, dtype=dtype, seed=d, scale=3.0)
    q, k, v = x[:, :heads], x[:, heads:heads + kv], x[:, heads + kv:]
    turns = torch.randn(50, turned, device="cuda").clamp(-1, 1)
    pos = torch.randint(0, 50, (t,), device="cuda", dtype=torch.int32)
    wq = (1 + rand(d, dtype=dtype, seed=1) / 4) if norm else None
    wk = (1 + rand(d, dtype=dtype, seed=2) / 4) if norm else None
    slots = torch.randperm(pages * page, device="cuda")[:t]
    slots[5], slots[9] = -1, pages * page  # skipped, and past the cache
    kc, vc = rand(pages, page, kv, d, dtype=dtype, seed=3), rand(pages, page, kv, d, dtype=dtype, seed=4)
    kept = torch.ones(t, dtype=torch.bool, device="cuda")
    kept[[5, 9]] = False
    k_want, v_want = kc.clone(), vc.clone()
    gq, gk = V.norm_rotate(q, k, v, pos, turns, q_weight=wq, k_weight=wk, eps=1e-5, pairs=pairs, slots=slots, k_cache=kc,
                           v_cache=vc)
    for got, src, w in ((gq, q, wq), (gk, k, wk)):
        want, size = rotate_reference(src, w, turns, pos, 1e-5, pairs)
        # in 32 bits: the mean of d squares (d + 4 roundings, halved by the root), the root, three products a term
        assert_near(got, want, (d + 16) * 2.0 ** -24 * size, "rotated")
    k_want.view(-1, kv, d)[slots[kept]] = gk[kept]
    v_want.view(-1, kv, d)[slots[kept]] = v[kept]
    assert torch.equal(kc, k_want) and torch.equal(vc, v_want)
    # without k, without a cache, and with strided caches: the same values
    q2, none = V.norm_rotate(q, k, None, pos, turns, q_weight=wq, k_weight=wk, eps=1e-5, pairs=pairs, keep_k=False)
    assert none is None and torch.equal(q2, gq)
    both = torch.zeros(pages, 2, page, kv, d, dtype=dtype, device="cuda")
    V.norm_rotate(q, k, v, pos, turns, q_weight=wq, k_weight=wk, eps=1e-5, pairs=pairs, slots=slots,
                  k_cache=both[:, 0], v_cache=both[:, 1], keep_k=False)
    assert torch.equal(both[:, 0].reshape(-1, kv, d)[slots[kept]], gk[kept])
    assert torch.equal(both[:, 1].reshape(-1, kv, d)[slots[kept]], v[kept])


def test_norm_rotate_sizes_and_extremes(V):
    turns = torch.cat([torch.ones(9, 32), torch.zeros(9, 32)], 1).cuda()
    for t in (0, 1, 2, 999):
        x = rand(t, 12, 64, seed=t)
        q, k = V.norm_rotate(x[:, :8], x[:, 8:10], None, torch.zeros(t, dtype=torch.int32, device="cuda"), turns)
        assert torch.equal(q, x[:, :8]) and torch.equal(k, x[:, 8:10])  # angle 0, no norm: a copy
    x = torch.zeros(2, 3, 64, dtype=torch.bfloat16, device="cuda")
    w = torch.ones(64, dtype=torch.bfloat16, device="cuda")
    q, k = V.norm_rotate(x[:, :2], x[:, 2:], None, ints([0, 1]), turns, q_weight=w, k_weight=w, eps=1e-6)
    assert not q.any() and not k.any()
    big = torch.full((1, 3, 64), 1e15, dtype=torch.bfloat16, device="cuda")  # squares of 1e30: within 32 bits
    q, _ = V.norm_rotate(big[:, :2], big[:, 2:], None, ints([3]), turns, q_weight=w, k_weight=w)
    assert (q.float() - 1).abs().max() <= 2.0 ** -8
    q, _ = V.norm_rotate(big[:, :2], big[:, 2:], None, ints([9]), turns)  # a position past the table
    assert q[..., :64].isnan().all()
    q, _ = V.norm_rotate(big[:, :2], big[:, 2:], None, ints([-1]), turns)
    assert q.isnan().all()


# ------------------------------------------------------------------------------------------ page tables
def tables_reference(cached, fresh, free, table, page, total, base):
    table, at, t = [list(r) for r in table], 0, 0
    starts, positions, slots = [0], [0] * total, [-1] * total
    for b, (c, f) in enumerate(zip(cached, fresh)):
        for col in range(-(-c // page), -(-(c + f) // page)):
            if col < len(table[b]):
                table[b][col] = free[at] if at < len(free) else -1
            at += 1
        for n in range(c, c + f):
            if t < total:
                p = table[b][n // page] if n // page < len(table[b]) else -1
                positions[t], slots[t] = base + n, (p * page + n % page if p >= 0 else -1)
            t += 1
        starts.append(t)
    return table, [c + f for c, f in zip(cached, fresh)], starts, positions, slots, [at]


def check_tables(V, cached, fresh, page, width, spare=0, short=0, base=0, seed=0):
    g = torch.Generator().manual_seed(seed)
    n = len(cached)
    order = torch.randperm(200000, generator=g).tolist()
    table = [[order.pop() if c < -(-cached[b] // page) else -1 for c in range(width)] for b in range(n)]
    need = sum(-(-(c + f) // page) - -(-c // page) for c, f in zip(cached, fresh))
    free = [order.pop() for _ in range(max(0, need + 3 - short))]
    total = max(0, sum(fresh) + spare)
    want = tables_reference(cached, fresh, free, table, page, total, base)
    t = torch.tensor(table, dtype=torch.int32).reshape(n, width).cuda()
    for _ in range(2):  # the call may be repeated
        got = V.page_tables(ints(cached), ints(fresh), ints(free), t, page, total, base=base)
        assert got.table is t
        for name, a, b in zip(got._fields, got, want):
            assert a.cpu().tolist() == b, name


@pytest.mark.parametrize("page", [16, 64, 256])
def test_tables_small(V, page):
    check_tables(V, [0, 5, 16, 31, 0, 64], [1, 1, 1, 1, 0, 1], page, 8)
    check_tables(V, [0, 5, 16, 31, 0, 700], [17, 300, 0, 1, 64, 1], page, 70, spare=9, base=12345)
    check_tables(V, [7], [0], page, 3, spare=2)
    check_tables(V, [], [], page, 4, spare=3)


def test_tables_large(V):
    g = torch.Generator().manual_seed(1)
    for n in (513, 1500):
        cached = torch.randint(0, 400, (n,), generator=g).tolist()
        fresh = torch.randint(0, 90, (n,), generator=g).tolist()
        check_tables(V, cached, fresh, 16, 40, spare=100, seed=n)
    check_tables(V, [3], [100000], 16, 7000)


def test_tables_short_of_pages_and_columns(V):
    check_tables(V, [0, 5, 16], [40, 300, 20], 16, 30, short=8)
    check_tables(V, [0, 5, 16], [40, 300, 20], 16, 30, short=1000)
    check_tables(V, [0, 5, 100], [40, 300, 20], 16, 4)
    check_tables(V, [0, 5, 100], [40, 300, 20], 16, 30, spare=-50)  # fewer rows than new tokens


def test_tables_negative_counts(V):
    t = torch.full((2, 3), -1, dtype=torch.int32, device="cuda")
    got = V.page_tables(ints([-4, 0]), ints([5, -9]), ints([8, 9]), t, 16, 6)
    assert got.lengths.tolist() == [5, 0] and got.starts.tolist() == [0, 5, 5] and got.used.tolist() == [1]
    assert got.slots.tolist() == [128, 129, 130, 131, 132, -1] and t[0, 0] == 8


# ------------------------------------------------------------------------------------------ together
def test_operators_in_a_graph_and_on_a_side_stream(V):
    """One step of answering captured in a CUDA graph: replays follow the buffers they were given."""
    heads, kv, d, page, b, prefix = 8, 2, 64, 16, 5, 100
    kc, vc = rand(60, page, kv, d, seed=1), rand(60, page, kv, d, seed=2)
    x = rand(b, heads + 2 * kv, d, seed=3)
    turns = torch.randn(500, d, device="cuda").clamp(-1, 1)
    cached, fresh = ints([3, 16, 40, 0, 31]), ints([1] * b)
    table = torch.arange(10, 10 + 5 * b, dtype=torch.int32, device="cuda").view(b, 5)
    free, shared = torch.arange(40, 60, dtype=torch.int32, device="cuda"), torch.arange(7, dtype=torch.int32, device="cuda")

    def step():
        pt = V.page_tables(cached, fresh, free, table, page, b, base=prefix)
        q, _ = V.norm_rotate(x[:, :heads], x[:, heads:heads + kv], x[:, heads + kv:], pt.positions, turns, slots=pt.slots,
                             k_cache=kc, v_cache=vc, keep_k=False)
        return V.shared_prefix_attention(q, kc, vc, shared, prefix, pt.table, pt.lengths)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    for seed in (8, 9):
        x.copy_(rand(b, heads + 2 * kv, d, seed=seed))
        graph.replay()
        replayed = out.clone()
        assert torch.equal(replayed, step())


# Prompts whose mean is above what goes to the small blocks: every head layout on the tensor-memory tiles too.
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("heads,kv,d", [(8, 2, 128), (4, 4, 64), (7, 1, 128), (6, 2, 96), (2, 1, 40), (3, 3, 8),
                                        (16, 1, 64), (24, 1, 72), (100, 1, 64), (128, 1, 128)])
def test_prompt_heads_and_types_long(V, dtype, causal, heads, kv, d):
    check_prompt(V, [700, 1, 333, 0, 1300], None, heads, kv, d, dtype, causal, seed=heads)


@pytest.mark.parametrize("bad", [math.nan, math.inf])
@pytest.mark.parametrize("heads,kv,d", [(8, 2, 128), (2, 2, 64)])
def test_prompt_unseen_values_do_not_leak_long(V, bad, heads, kv, d):
    """One non-finite value row in the middle of a long prompt, and one neighbouring prompt full of them."""
    lens = [900, 300, 1100]
    n = sum(lens)
    q, k, v = rand(n, heads, d, seed=1), rand(n, kv, d, seed=2), rand(n, kv, d, seed=3)
    clean = V.prompt_attention(q, k, v, starts_of(lens))
    v2, k2 = v.clone(), k.clone()
    v2[500, :, d // 2] = bad
    v2[900:1200], k2[900:1200] = bad, bad
    out = V.prompt_attention(q, k2, v2, starts_of(lens))
    err = (out.double() - clean.double()).abs()
    keep = torch.ones(n, dtype=torch.bool, device="cuda")
    keep[500:1200] = False
    assert err[keep].max() <= 2.0 ** -7 * clean.double().abs().max()
    assert torch.isfinite(out[500:900, :, :d // 2]).all() and not torch.isfinite(out[500:900, :, d // 2]).any()


def test_prompt_many_requests(V):
    """More requests than one step of the search for a block's request looks at, empty ones among them."""
    lens = [(i * 7919) % 23 if i % 5 else 0 for i in range(1500)] + [2000]
    check_prompt(V, lens, None, 2, 1, 64, torch.bfloat16, True, seed=3)
    lens = [1] * 40 + [0] * 40 + [9000]
    check_prompt(V, lens, None, 2, 1, 64, torch.bfloat16, False, seed=4)


# ------------------------------------------------------------------------------------------ refusals on tensors
def refused(says, call):
    from vesper_db_b200 import VesperError
    with pytest.raises(VesperError, match=says):
        call()


def test_refusals_of_tensors(V):
    q, k = rand(5, 8, 64), rand(5, 2, 64)
    st, pos, slots = ints([0, 5]), ints([0] * 5), ints([0] * 5, torch.int64)
    turns = torch.zeros(9, 64, device="cuda")
    kc = rand(4, 16, 2, 64)
    table, lens, pages = ints([[0, 1]] * 5), ints([3] * 5), ints([2])
    P, R, S, T = V.prompt_attention, V.norm_rotate, V.shared_prefix_attention, V.page_tables
    refused("bf16 or f16", lambda: P(q.float(), k.float(), k.float(), st))
    refused("k is Half", lambda: P(q, k.half(), k, st))
    refused("CUDA", lambda: P(q.cpu(), k, k, st))
    refused("k is on cpu", lambda: P(q, k.cpu(), k, st))
    refused("k has shape", lambda: P(q, k[..., :32], k, st))
    refused("v has shape", lambda: P(q, k, k[:4], st))
    refused("multiple of kv_heads", lambda: P(q[:, :7], k, k, st))
    refused("starts is Long", lambda: P(q, k, k, st.long()))
    refused("starts_k must be", lambda: P(q, k, k, st, ints([0, 1, 5])))
    refused("d_starts_k", lambda: P(q, rand(9, 2, 64), rand(9, 2, 64), st))
    refused("scale", lambda: P(q, k, k, st, scale=0.0))
    refused("scale must be a number", lambda: P(q, k, k, st, scale="x"))
    refused("last dimension", lambda: P(rand(5, 64, 8).transpose(1, 2), k, k, st))
    refused("head_dim", lambda: P(rand(5, 8, 136), rand(5, 2, 136), rand(5, 2, 136), st))
    refused("strides", lambda: P(rand(5, 8, 68)[..., :64], k, k, st))
    refused("aligned", lambda: P(rand(5 * 8 * 64 + 4)[4:].view(5, 8, 64), k, k, st))
    refused("turned", lambda: R(q, k, None, pos, turns[:, :24].contiguous()))
    refused("turns is", lambda: R(q, k, None, pos, turns.half()))
    refused("slots need", lambda: R(q, k, None, pos, turns, slots=slots))
    refused("slots is Int", lambda: R(q, k, k, pos, turns, slots=pos, k_cache=kc, v_cache=kc))
    refused("k_cache", lambda: R(q, k, k, pos, turns, slots=slots, k_cache=kc[:, :, :1], v_cache=kc))
    refused("q_weight", lambda: R(q, k, None, pos, turns, q_weight=q[0, 0, :32]))
    refused("eps", lambda: R(q, k, None, pos, turns, eps=-1.0))
    refused("positions", lambda: R(q, k, None, pos[:4], turns))
    refused("prefix_pages do not hold", lambda: S(q, kc, kc, pages, 17, table, lens))
    refused("prefix_len", lambda: S(q, kc, kc, pages, -1, table, lens))
    refused("table must be", lambda: S(q, kc, kc, pages, 9, table[:4], lens))
    refused("lengths must be", lambda: S(q, kc, kc, pages, 9, table, lens[:4]))
    refused("page_size", lambda: S(q, kc[:, :8], kc[:, :8], pages, 4, table, lens))
    refused("fresh must be", lambda: T(lens, lens[:2], pages, table, 16, 9))
    refused("page_size", lambda: T(lens, lens, pages, table, 17, 9))
    refused("total must not be negative", lambda: T(lens, lens, pages, table, 16, -1))
    refused("base", lambda: T(lens, lens, pages, table, 16, 9, base=-1))
    refused("contiguous rows", lambda: T(lens[:2], lens[:2], pages, table.T, 16, 9))


def test_calls_with_addresses(V):
    """The C entry points with device addresses give what the tensors' calls give."""
    from vesper_db_b200 import attention as A
    q, k, v = rand(70, 4, 64, seed=1), rand(70, 2, 64, seed=2), rand(70, 2, 64, seed=3)
    st, out = ints([0, 30, 70]), torch.empty(70, 4, 64, dtype=torch.bfloat16, device="cuda")
    A.call_device("prompt_attention", [0, 2, 70, 70, 4, 2, 64, 1, 0.125, q.data_ptr(), 256, 64, k.data_ptr(), 128, 64,
                                       v.data_ptr(), 128, 64, st.data_ptr(), 0, out.data_ptr(), 0, 0, 0],
                  torch.cuda.current_stream().cuda_stream)
    assert torch.equal(out, V.prompt_attention(q, k, v, st))
    refused("scale", lambda: A.call_device("prompt_attention", [0, 2, 70, 70, 4, 2, 64, 1, -1.0] + [0] * 15))


def test_expanded_tensors_are_refused(V):
    q, k = rand(5, 8, 64), rand(5, 1, 64).expand(5, 2, 64)
    refused("strides", lambda: V.prompt_attention(q, k, k, ints([0, 5])))
    refused("strides", lambda: V.norm_rotate(q, k, None, ints([0] * 5), torch.zeros(9, 64, device="cuda")))
    one = rand(1, 8, 64).expand(1, 8, 64)  # a single element's stride does not matter
    assert V.prompt_attention(one, one[:, :2], one[:, :2], ints([0, 1])).shape == (1, 8, 64)
