"""Serving several continuations of one prompt: windowed and full attention layers over one paged cache, and sampling.

A toy decoder whose layers take turns: even ones see a sliding window and the first tokens, odd ones everything. The prompt goes
through once (`gqa_fwd_window_prefill`), its pages are shared by all continuations. Each step then runs, per layer,
`gqa_fwd_window_decode` on the prompt's pages followed by the sequence's own, or `gqa_fwd_shared_prefix_decode`, which reads the prompt once
for the whole batch, and draws the next tokens with `sample_tokens`. Random weights; the last step's logits are checked against one pass
over every whole sequence.

    python examples/shared_prompt_serving.py            # on a GPU if there is one
"""
import os
import sys

import torch

sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))

import triton_distributed_b200 as tdist  # noqa: E402


class ToyDecoder:
    """Embedding, attention layers with residuals, logits."""

    def __init__(self, device, dtype, vocab=1000, hidden=256, heads=8, kv_heads=2, head_dim=64, layers=4, window=48, sinks=4, page=16, pages=256, seed=0):
        g = torch.Generator(device="cpu").manual_seed(seed)
        new = lambda *shape, scale: (torch.randn(*shape, generator=g) * scale).to(device, dtype)   # noqa: E731
        self.heads, self.kv_heads, self.head_dim, self.window, self.sinks, self.page = heads, kv_heads, head_dim, window, sinks, page
        self.embed, self.head = new(vocab, hidden, scale=1.0), new(hidden, vocab, scale=3.0 * hidden ** -0.5)
        self.qkv = [new(hidden, (heads + 2 * kv_heads) * head_dim, scale=hidden ** -0.5) for _ in range(layers)]
        self.out = [new(heads * head_dim, hidden, scale=(heads * head_dim) ** -0.5) for _ in range(layers)]
        # one pool of pages, keys and values of all layers
        self.cache = [tuple(torch.zeros(pages, page, kv_heads, head_dim, device=device, dtype=dtype) for _ in "kv") for _ in range(layers)]

    def forward(self, tokens, slots, attend):
        """``tokens [n]`` whose keys and values go to the cache rows ``slots [n]``; ``attend(layer, q, k_cache, v_cache)``."""
        x = self.embed[tokens.long()]
        for i, (wqkv, wout) in enumerate(zip(self.qkv, self.out)):
            qkv = (torch.nn.functional.rms_norm(x, x.shape[-1:]) @ wqkv).view(-1, self.heads + 2 * self.kv_heads, self.head_dim)
            k, v = self.cache[i]
            k.view(-1, self.kv_heads, self.head_dim)[slots] = qkv[:, self.heads:self.heads + self.kv_heads]
            v.view(-1, self.kv_heads, self.head_dim)[slots] = qkv[:, self.heads + self.kv_heads:]
            x = x + attend(i, qkv[:, :self.heads], k, v).reshape(x.shape[0], -1) @ wout
        return torch.nn.functional.rms_norm(x, x.shape[-1:]) @ self.head


def run(device, batch=6, prompt=96, steps=20, seed=0):
    dtype = torch.bfloat16 if device.type == "cuda" else torch.float32
    model = ToyDecoder(device, dtype, seed=seed)
    page, window, sinks = model.page, model.window, model.sinks
    g = torch.Generator(device="cpu").manual_seed(seed + 1)
    int32 = dict(dtype=torch.int32, device=device)
    # pages in no order: the prompt's, then every sequence's own
    order = torch.randperm(256, generator=g).to(**int32)
    per_seq = -(-steps // page)
    prompt_pages, own_pages = order[:prompt // page], order[prompt // page:prompt // page + batch * per_seq].view(batch, per_seq)
    both = torch.cat([prompt_pages.expand(batch, -1), own_pages], 1).contiguous()   # the prompt fills its pages
    text = torch.randint(0, 1000, (prompt,), generator=g).to(device)

    def slot(pages, position):
        return pages[..., position // page].long() * page + position % page

    # ---- the prompt, once
    at = torch.arange(prompt, device=device)
    starts, lens = torch.tensor([0, prompt], **int32), torch.tensor([prompt], **int32)
    logits = model.forward(text, slot(prompt_pages, at), lambda i, q, k, v: tdist.gqa_fwd_window_prefill(
        q, k, v, starts, lens, prompt_pages.view(1, -1), window=window if i % 2 == 0 else None, sinks=sinks if i % 2 == 0 else 0))
    logits = logits[-1:].expand(batch, -1)

    # ---- the continuations, one token each per step
    drawn = []
    prompt_len = torch.tensor([prompt], **int32)
    for step in range(steps):
        u = torch.rand(batch, generator=g).to(device)
        tokens = tdist.sample_tokens(logits, u, temperature=0.9, top_k=50, top_p=0.95, min_p=0.01).tokens
        drawn.append(tokens)
        own_lens = torch.full((batch,), step + 1, **int32)

        def attend(i, q, k, v):
            if i % 2 == 0:
                return tdist.gqa_fwd_window_decode(q.contiguous(), k, v, own_lens + prompt, both, window=window, sinks=sinks)
            return tdist.gqa_fwd_shared_prefix_decode(q.contiguous(), k, v, prompt_len, prompt_pages, own_lens, own_pages)

        logits = model.forward(tokens, slot(own_pages, step), attend)
    drawn = torch.stack(drawn, 1)

    # ---- every whole sequence in one ragged batch, on a cache of its own: the same logits for its last token
    check = ToyDecoder(device, dtype, seed=seed)
    n = prompt + steps
    pages = torch.arange(batch * -(-n // page), **int32).view(batch, -1)
    at = torch.arange(n, device=device)
    slots = torch.cat([slot(pages[b], at) for b in range(batch)])
    starts, lens = torch.arange(batch + 1, **int32) * n, torch.full((batch,), n, **int32)
    whole = torch.cat([torch.cat([text, drawn[b].to(text.dtype)]) for b in range(batch)])
    ref = check.forward(whole, slots, lambda i, q, k, v: tdist.gqa_fwd_window_prefill(
        q, k, v, starts, lens, pages, window=window if i % 2 == 0 else None, sinks=sinks if i % 2 == 0 else 0))
    ref = ref.view(batch, n, -1)[:, -1]
    tol = 0.15 if dtype == torch.bfloat16 else 1e-3
    torch.testing.assert_close(logits.float(), ref.float(), atol=tol, rtol=tol)
    return drawn


if __name__ == "__main__":
    dev = torch.device("cuda", 0) if torch.cuda.is_available() else torch.device("cpu")
    for row in run(dev).tolist():
        print(" ".join(str(t) for t in row))
