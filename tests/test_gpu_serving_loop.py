"""The serving loop of examples/paged_serving.py (-m gpu): its logits against a plain recompute, its pages, its end."""

import importlib.util
from pathlib import Path

import pytest

torch = pytest.importorskip("torch")

from pto_wsp_b200 import serving  # noqa: E402

pytestmark = pytest.mark.gpu


def example():
    path = Path(__file__).resolve().parents[1] / "examples" / "paged_serving.py"
    spec = importlib.util.spec_from_file_location("paged_serving", path)
    module = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(module)
    return module


def plain_logits(model, texts):
    """The model over whole texts with unquantised K and V, in f64: the last token's logits of each."""
    got = []
    for text in texts:
        x = (model.embedding[torch.tensor(text, device="cuda")] + model.position[:len(text)]).double()
        for qkv, out in zip(model.qkv, model.out):
            y = (torch.nn.functional.layer_norm(x, x.shape[-1:]) @ qkv.double()).view(len(text), -1, model.dim)
            q, k, v = y.split((model.heads, model.kv_heads, model.kv_heads), 1)
            k, v = (t.repeat_interleave(model.heads // model.kv_heads, 1) for t in (k, v))
            s = torch.einsum("qhd,khd->hqk", q, k) * model.dim ** -0.5
            s = s.masked_fill(torch.ones_like(s[0]).triu(1).bool(), float("-inf"))
            x = x + torch.einsum("hqk,khd->qhd", torch.softmax(s, -1), v).reshape(len(text), -1) @ out.double()
        got.append(torch.nn.functional.layer_norm(x[-1], x.shape[-1:]) @ model.head.double())
    return torch.stack(got)


@pytest.mark.parametrize("cache", ["e4m3", "int8"])
def test_serving_loop(cache, require_cuda):
    ex = example()
    slots, max_pages = 5, 12
    pages = 30  # fewer than the slots could fill: pages have to come back
    model = ex.Decoder(pages, heads=8, kv_heads=2, dim=64, vocab=512, cache=cache)
    server = ex.Server(model, slots, pages, max_pages, chunk=50)
    gen = torch.Generator().manual_seed(1)
    prompts = [torch.randint(512, (n,), generator=gen).tolist() for n in (1, 15, 16, 90, 47, 33, 64, 2, 77)]
    waiting, texts = list(prompts), {}
    greedy, all_p = torch.zeros(slots, device="cuda"), torch.ones(slots, device="cuda")
    worst = 0.0
    for _ in range(100):
        for slot in range(slots):
            if server.left[slot] == 0 and waiting and len([n for n in server.left if n > 0]) < 3:
                texts[slot] = waiting.pop(0)
                server.admit(slot, texts[slot], 6)
        if not server.busy():
            break
        active = [s for s in range(slots) if server.left[s] > 0]
        before = {s: len(server.texts[s]) for s in active}
        logits = server.step(greedy, all_p)
        assert server.plan.granted[active].all()
        fresh = [s for s in active if len(server.texts[s]) > before[s]]  # those whose logits count
        if fresh:
            want = plain_logits(model, [texts[s] + server.texts[s][:-1] for s in fresh])
            off = (logits[fresh].double() - want).norm(dim=-1) / want.norm(dim=-1)
            worst = max(worst, float(off.max()))
            assert [server.texts[s][-1] for s in fresh] == logits[fresh].float().argmax(-1).tolist()
    # The 8-bit cache leaves each K and V element off by at most 1/16 (e4m3) or 1/254 of its page's largest (int8).  The
    # attention's part of a layer's output averages these over tokens and heads; an eighth of the norm bounds both.
    assert worst < 0.125
    assert not waiting and not server.busy()
    serving.check_status(server.status)
    head, tail = server.free.tolist()
    assert tail - head == pages  # every page came back
    at = torch.arange(head, tail) % pages
    assert sorted(server.ring.cpu()[at].tolist()) == list(range(pages))


def dequantised_logits(ex, model, server, slot, text):
    """The model over a whole text in f64, each layer's attention over the K and V that the server's cache holds for it."""
    pages = server.table[slot, :-(-len(text) // model.page_size)].long()
    x = (model.embedding[torch.tensor(text, device="cuda")] + model.position[:len(text)]).double()
    for i, (qkv, out) in enumerate(zip(model.qkv, model.out)):
        y = (torch.nn.functional.layer_norm(x, x.shape[-1:]) @ qkv.double()).view(len(text), -1, model.dim)
        k, v = ((c[i][pages].double() * s[i][pages].double()[:, None, :, None]).reshape(-1, model.kv_heads, model.dim)
                [:len(text)].repeat_interleave(model.heads // model.kv_heads, 1)
                for c, s in ((model.k, model.k_scale), (model.v, model.v_scale)))
        s = torch.einsum("qhd,khd->hqk", y[:, :model.heads], k) * model.dim ** -0.5
        s = s.masked_fill(torch.ones_like(s[0]).triu(1).bool(), float("-inf"))
        x = x + torch.einsum("hqk,khd->qhd", torch.softmax(s, -1), v).reshape(len(text), -1) @ out.double()
    return torch.nn.functional.layer_norm(x[-1], x.shape[-1:]) @ model.head.double()


@pytest.mark.parametrize("cache", ["e4m3", "int8"])
def test_serving_loop_logits_follow_from_the_cache(cache, require_cuda):
    # One token per step into short texts, so that every page's scale counts.  What is left between the two is rounding to
    # f16 (2^-11) in some six places per layer, none of which a layer norm enlarges: 2^-7 of the logits' norm.  A layer's own
    # row is written from f16 activations, which the recompute has in f64; that is among the six.
    ex = example()
    model = ex.Decoder(12, heads=8, kv_heads=2, dim=64, vocab=512, cache=cache)
    server = ex.Server(model, 3, 12, 4, chunk=1)
    prompts = [[5, 9, 300], [17], [400, 2, 2, 511, 30]]
    for slot, prompt in enumerate(prompts):
        server.admit(slot, prompt, 30)
    texts = [[] for _ in prompts]
    for _ in range(30):
        fed = [list(w[:1]) for w in server.waiting]
        logits = server.step(torch.zeros(3, device="cuda"), torch.ones(3, device="cuda"))
        for slot, new in enumerate(fed):
            texts[slot] += new
            if not new:
                continue
            want = dequantised_logits(ex, model, server, slot, texts[slot])
            assert float((logits[slot].double() - want).norm() / want.norm()) < 2.0 ** -7, (slot, len(texts[slot]))
    serving.check_status(server.status)
