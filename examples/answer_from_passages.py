"""Answering from retrieved passages: a search, one shared prompt, many questions.

    python examples/answer_from_passages.py

A flat top-k search finds the passages nearest to a topic; their tokens become one prompt that every question shares.
A small decoder (random weights: there is nothing to download) reads the prompt once with prompt_attention, its keys
and values going to the pages of a cache, and then answers all questions together, one token a step, with
shared_prefix_attention over the prompt's pages and each question's own.  page_tables finds the pages, norm_rotate
norms and rotates queries and keys and fills the cache.
"""
import os
import sys

import torch

sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))
import vesper_db_b200 as vesper  # noqa: E402


class Decoder:
    """A plain pre-norm decoder: grouped heads, normed and rotated queries and keys, a gated feed-forward layer."""

    def __init__(self, vocab=2000, width=512, layers=2, heads=8, kv_heads=2, head_dim=64, longest=4096, seed=0,
                 dtype=torch.bfloat16):
        g = torch.Generator(device="cuda").manual_seed(seed)
        self.heads, self.kv, self.dim, self.layers = heads, kv_heads, head_dim, []

        def weight(n, m):
            return (torch.randn(n, m, generator=g, device="cuda") * n ** -0.5).to(dtype)
        self.embed = (torch.randn(vocab, width, generator=g, device="cuda")).to(dtype)
        self.read_out = weight(width, vocab)
        for _ in range(layers):
            self.layers.append({
                "qkv": weight(width, (heads + 2 * kv_heads) * head_dim), "out": weight(heads * head_dim, width),
                "up": weight(width, 4 * width), "gate": weight(width, 4 * width), "down": weight(4 * width, width),
                "q_norm": torch.ones(head_dim, dtype=dtype, device="cuda"),
                "k_norm": torch.ones(head_dim, dtype=dtype, device="cuda")})
        angle = torch.arange(longest, device="cuda")[:, None] * 10000.0 ** (
            -torch.arange(0, head_dim, 2, device="cuda") / head_dim)
        self.turns = torch.cat([angle.cos(), angle.sin()], 1).float()

    @staticmethod
    def _norm(x):
        return torch.nn.functional.rms_norm(x, (x.shape[-1],))

    def forward(self, tokens, positions, attend):
        """Logits of every token; attend(layer, q, k, v, weights, positions) gives a layer's attention."""
        x = self.embed[tokens]
        for i, w in enumerate(self.layers):
            qkv = (self._norm(x) @ w["qkv"]).view(-1, self.heads + 2 * self.kv, self.dim)
            q, k, v = qkv.split((self.heads, self.kv, self.kv), 1)
            x = x + attend(i, q, k, v, w, positions).flatten(1) @ w["out"]
            y = self._norm(x)
            x = x + (torch.nn.functional.silu(y @ w["gate"]) * (y @ w["up"])) @ w["down"]
        return self._norm(x) @ self.read_out


class Cache:
    """Paged keys and values of all layers, and the pages that are still free."""

    def __init__(self, model, pages, page_size=16):
        shape = (pages, page_size, model.kv, model.dim)
        self.k = [torch.zeros(shape, dtype=model.embed.dtype, device="cuda") for _ in model.layers]
        self.v = [torch.zeros_like(k) for k in self.k]
        self.page_size = page_size
        self.free = torch.randperm(pages, device="cuda").to(torch.int32)

    def take(self, n):
        """The first n free pages."""
        taken, self.free = self.free[:n], self.free[n:]
        return taken


def ints(values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


def read_prompt(model, cache, tokens):
    """Reads the shared prompt once: (pages that hold it, logits)."""
    n = tokens.shape[0]
    pages = -(-n // cache.page_size)
    table = torch.full((1, pages), -1, dtype=torch.int32, device="cuda")
    pt = vesper.page_tables(ints([0]), ints([n]), cache.free, table, cache.page_size, n)
    cache.take(pages)

    def attend(i, q, k, v, w, positions):
        q, k = vesper.norm_rotate(q, k, v, positions, model.turns, q_weight=w["q_norm"], k_weight=w["k_norm"],
                                  slots=pt.slots, k_cache=cache.k[i], v_cache=cache.v[i])
        return vesper.prompt_attention(q, k, v, pt.starts)
    return table[0], model.forward(tokens, pt.positions, attend)


def answer(model, cache, shared, prompt_len, questions, steps):
    """Feeds the questions' tokens, then `steps` greedy tokens more, all requests together: (tokens, logits of each
    step).  questions: [requests, length]."""
    b, length = questions.shape
    width = -(-(length + steps) // cache.page_size)
    table = torch.full((b, width), -1, dtype=torch.int32, device="cuda")
    held, one = ints([0] * b), ints([1] * b)
    tokens, out, logits = questions[:, 0], [], []
    for step in range(length + steps - 1):
        pt = vesper.page_tables(held, one, cache.free, table, cache.page_size, b, base=prompt_len)
        if step % cache.page_size == 0:  # every request has just taken a page
            cache.take(b)

        def attend(i, q, k, v, w, positions):
            q, _ = vesper.norm_rotate(q, k, v, positions, model.turns, q_weight=w["q_norm"], k_weight=w["k_norm"],
                                      slots=pt.slots, k_cache=cache.k[i], v_cache=cache.v[i], keep_k=False)
            return vesper.shared_prefix_attention(q, cache.k[i], cache.v[i], shared, prompt_len, pt.table, pt.lengths)
        logits.append(model.forward(tokens, pt.positions, attend))
        held = pt.lengths
        tokens = questions[:, step + 1] if step + 1 < length else logits[-1].argmax(-1)
        out.append(tokens)
    return torch.stack(out[length - 1:], 1), torch.stack(logits, 1)


def retrieve(topic, passages, k):
    """Indices of the k passages nearest to the topic (flat top-k search on the device)."""
    index = torch.empty(1, k, dtype=torch.int32, device="cuda")
    score = torch.empty(1, k, dtype=torch.float32, device="cuda")
    torch.cuda.synchronize()
    vesper.flat_topk_device("l2", topic.data_ptr(), 1, passages.data_ptr(), passages.shape[0], passages.shape[1], k,
                            index.data_ptr(), score.data_ptr())
    return index[0].long()


def main():
    torch.manual_seed(0)
    model = Decoder()
    passages = torch.randn(20000, 128, device="cuda")  # embeddings, and 40 tokens of text each
    text = torch.randint(0, 2000, (20000, 40), device="cuda")
    topic = passages[123:124] + 0.1 * torch.randn(1, 128, device="cuda")
    found = retrieve(topic, passages, 25)
    prompt = text[found].flatten()
    cache = Cache(model, pages=400)
    shared, _ = read_prompt(model, cache, prompt)
    questions = torch.randint(0, 2000, (12, 7), device="cuda")
    tokens, _ = answer(model, cache, shared, prompt.shape[0], questions, steps=20)
    print(f"{prompt.shape[0]} tokens of {found.shape[0]} passages read once; {tokens.shape[0]} answers of "
          f"{tokens.shape[1]} tokens:")
    for row in tokens.tolist():
        print("  ", *row)


if __name__ == "__main__":
    main()
