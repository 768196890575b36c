"""Answering steps captured in CUDA graphs where the prefix is on the tensor-core tiles and the own pages run beside it."""
import pytest
import torch

from conftest import ROOT  # noqa: F401
from test_attention_gpu import assert_near, row_reference

pytestmark = pytest.mark.gpu


def ints(x, dtype=torch.int32):
    return torch.tensor(x, dtype=dtype, device="cuda")


@pytest.mark.parametrize("b,longest", [(64, 0), (64, 1), (61, 10), (256, 10), (40, 300)])
@pytest.mark.parametrize("dtype,heads,kv,d", [(torch.bfloat16, 32, 8, 128), (torch.float16, 28, 4, 128),
                                              (torch.bfloat16, 8, 2, 64)])
def test_prefix_tiles_in_a_graph(b, longest, dtype, heads, kv, d):
    """The own pages are over long before the prefix is: what joins both parts must come after the later one.  Replays on
    changing queries against the direct call, and against the formula with the prefix in 64 bits."""
    import vesper_db_b200 as V
    page, prefix = 64, 20001
    shared, width = -(-prefix // page), max(1, -(-longest // page))
    g = torch.Generator(device="cuda").manual_seed(b + longest)
    normal = lambda *s: torch.randn(s, generator=g, device="cuda").to(dtype)  # noqa: E731
    kc, vc = normal(shared + b * width, page, kv, d), normal(shared + b * width, page, kv, d)
    pages = torch.arange(shared, dtype=torch.int32, device="cuda")
    table = (shared + torch.arange(b * width, dtype=torch.int32, device="cuda")).view(b, width)
    lens = ints([(7 * i) % (longest + 1) for i in range(b)])
    q, out, lse = normal(b, heads, d), None, None

    def step():
        return V.shared_prefix_attention(q, kc, vc, pages, prefix, table, lens, stats=True)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        for _ in range(3):  # one behind the other: the next call's tiles reuse the workspace of the last
            out, lse = step()
    for seed in range(6):
        q.copy_(normal(b, heads, d))
        graph.replay()
        got, got_lse = out.clone(), lse.clone()
        want, want_lse = step()
        assert torch.equal(got, want) and torch.equal(got_lse, want_lse)
    for i in (0, b // 2, b - 1):
        n = int(lens[i])
        k, v = (torch.cat([x[:shared].reshape(-1, kv, d)[:prefix], x[table[i].long()].reshape(-1, kv, d)[:n]])
                for x in (kc, vc))
        seen = torch.ones(1, prefix + n, dtype=torch.bool, device="cuda")
        o, l, err, lse_err = row_reference(q[i:i + 1], k, v, seen, d ** -0.5, dtype)
        # two parts joined: one more product with a weight in 32 bits each
        assert_near(got[i:i + 1], o, err * (1 + 2.0 ** -20), f"request {i}")
        assert_near(got_lse[i:i + 1], l, lse_err + 2.0 ** -22, f"lse of request {i}")
