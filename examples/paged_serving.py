"""A serving loop on the paged 8-bit KV cache: requests of different lengths prefill in chunks, decode side by side, end,
give their pages back, and new ones take them.

    python examples/paged_serving.py [--requests 64] [--prompt 400] [--new 64] [--cache e4m3|int8]

The model is a small random decoder; what is shown is the step: pages for the new tokens, their K and V into the cache,
attention over it, the next tokens -- four calls on one stream, with one read by the host per step (the tokens, which a
server sends to its users anyway).
"""

from __future__ import annotations

import argparse
import sys
import time
from pathlib import Path

import torch

sys.path.insert(0, str(Path(__file__).resolve().parents[1]))

from pto_wsp_b200 import serving  # noqa: E402


class Decoder:
    """A decoder of random weights with a paged 8-bit cache per layer."""

    def __init__(self, pages, *, page_size=16, layers=2, heads=16, kv_heads=4, dim=128, vocab=8192, cache="e4m3", seed=0):
        self.page_size, self.heads, self.kv_heads, self.dim = page_size, heads, kv_heads, dim
        gen = torch.Generator(device="cuda").manual_seed(seed)
        width = heads * dim
        weight = lambda *s: (torch.randn(s, generator=gen, device="cuda") * s[0] ** -0.5).half()  # noqa: E731
        self.embedding, self.position = weight(vocab, width) * vocab ** 0.5, weight(4096, width) * 8
        self.qkv = [weight(width, (heads + 2 * kv_heads) * dim) for _ in range(layers)]
        self.out = [weight(width, width) for _ in range(layers)]
        self.head = weight(width, vocab)
        codes = torch.float8_e4m3fn if cache == "e4m3" else torch.int8
        # the tokens of one head of a page stand together in memory: [pages, heads, page, dim] seen as [pages, page, ...]
        make = lambda: torch.zeros(pages, kv_heads, page_size, dim, dtype=torch.int8, device="cuda").view(codes).transpose(1, 2)  # noqa: E731
        self.k, self.v = ([make() for _ in range(layers)] for _ in range(2))
        self.k_scale, self.v_scale = ([torch.ones(pages, kv_heads, device="cuda") for _ in range(layers)] for _ in range(2))

    def logits(self, tokens, step: serving.PageStep, table, max_q: int, status):
        """The next-token logits of each request's last new token; `tokens`: the new tokens, request after request."""
        x = self.embedding[tokens] + self.position[step.positions.clamp(min=0).long() % 4096]
        for i in range(len(self.qkv)):
            qkv = (torch.nn.functional.layer_norm(x, x.shape[-1:]) @ self.qkv[i]).view(len(x), -1, self.dim)
            q, k, v = qkv.split((self.heads, self.kv_heads, self.kv_heads), 1)
            cache = self.k[i], self.v[i], self.k_scale[i], self.v_scale[i]
            serving.append_kv8(k, v, step.slots, *cache, status=status)
            a = serving.attend_kv8(q, *cache, table, step.kv_len, q_start=step.q_start, max_q=max_q, status=status)
            x = x + a.reshape(len(x), -1) @ self.out[i]
        last = x[(step.q_start[1:] - 1).clamp(min=0).long()]
        return torch.nn.functional.layer_norm(last, last.shape[-1:]) @ self.head


class Server:
    """Slots for requests, their block table, and the ring of free pages."""

    def __init__(self, model: Decoder, slots: int, pages: int, max_pages: int, chunk: int = 512):
        self.model, self.chunk = model, chunk
        self.table = torch.zeros(slots, max_pages, dtype=torch.int32, device="cuda")
        self.length = torch.zeros(slots, dtype=torch.int32, device="cuda")
        self.ring = torch.arange(pages, dtype=torch.int32, device="cuda")
        self.free = torch.tensor([0, pages], device="cuda")
        self.status = torch.zeros(1, dtype=torch.int32, device="cuda")
        self.waiting: list[list[int]] = [[] for _ in range(slots)]  # tokens that are not in the cache yet
        self.left = [0] * slots                                      # tokens still to generate; -1: ended, 0: empty
        self.texts: list[list[int]] = [[] for _ in range(slots)]

    def admit(self, slot: int, prompt: list[int], new: int) -> None:
        self.waiting[slot], self.left[slot], self.texts[slot] = list(prompt), new, []

    def step(self, temperature, top_p, generator=None):
        """One step of every request: a chunk of its prompt or its next token.  Returns the logits, for who wants them."""
        take = [-1 if n < 0 else min(len(w), self.chunk) for w, n in zip(self.waiting, self.left)]
        tokens = [t for w, n in zip(self.waiting, take) for t in w[:max(n, 0)]]
        counts = torch.tensor(take, dtype=torch.int32).pin_memory().cuda(non_blocking=True)
        new = torch.tensor(tokens, dtype=torch.int64).pin_memory().cuda(non_blocking=True)
        self.plan = serving.reserve_pages(self.table, self.length, counts, self.ring, self.free,
                                          page_size=self.model.page_size, max_tokens=len(tokens), status=self.status)
        self.length, self.free = self.plan.kv_len, self.plan.free_state
        self.left = [0 if n < 0 else left for n, left in zip(take, self.left)]
        if not tokens:  # requests ended, and that was all
            return None
        logits = self.model.logits(new, self.plan, self.table, max(max(take), 1), self.status)
        u = torch.rand(len(take), device="cuda", generator=generator)
        token, _ = serving.sample_tokens(logits, u, temperature=temperature, top_p=top_p)
        for slot, (n, t) in enumerate(zip(take, token.tolist())):
            if n > 0:
                self.waiting[slot] = self.waiting[slot][n:]
                if not self.waiting[slot]:  # the prompt is in: the token counts
                    self.texts[slot].append(t)
                    self.left[slot] -= 1
                    if self.left[slot]:
                        self.waiting[slot] = [t]
                    else:
                        self.left[slot] = -1
        return logits

    def busy(self) -> bool:
        return any(n != 0 for n in self.left)


def main() -> None:
    ap = argparse.ArgumentParser(description=__doc__, formatter_class=argparse.RawDescriptionHelpFormatter)
    ap.add_argument("--requests", type=int, default=64)
    ap.add_argument("--slots", type=int, default=32)
    ap.add_argument("--prompt", type=int, default=400, help="longest prompt")
    ap.add_argument("--new", type=int, default=64, help="tokens to generate per request")
    ap.add_argument("--cache", choices=("e4m3", "int8"), default="e4m3")
    a = ap.parse_args()
    max_pages = -(-(a.prompt + a.new) // 16)
    pages = a.slots * max_pages
    server = Server(Decoder(pages, cache=a.cache), a.slots, pages, max_pages)
    gen = torch.Generator().manual_seed(0)
    queue = [torch.randint(8192, (int(torch.randint(1, a.prompt + 1, (1,), generator=gen)),), generator=gen).tolist()
             for _ in range(a.requests)]
    temperature = torch.full((a.slots,), 0.8, device="cuda")
    top_p = torch.full((a.slots,), 0.95, device="cuda")
    done, steps, start = 0, 0, time.perf_counter()
    while queue or server.busy():
        for slot in range(a.slots):
            if server.left[slot] == 0 and queue:
                server.admit(slot, queue.pop(), a.new)
        server.step(temperature, top_p)
        done += sum(n == -1 for n in server.left)
        steps += 1
    torch.cuda.synchronize()
    spent = time.perf_counter() - start
    serving.check_status(server.status)
    head, tail = server.free.tolist()
    print(f"{done} requests, {done * a.new} tokens in {steps} steps, {done * a.new / spent:.0f} tokens/s; "
          f"{tail - head} of {pages} pages free again")


if __name__ == "__main__":
    main()
