"""The serving operators against plain implementations (-m gpu).

Whole numbers (slots, tables, codes, tokens) are compared exactly.  The attention's tolerance follows from its
roundings, per row: weights (of the V codes c_t, the scales s_t folded in) enter the second product as f16 with the
largest at 2^7 or above, so each is off by 2^-11 of itself or, below f16's normal numbers, by 2^-25, which is 2^-32 of
the largest; a score is off by at most (D + 8) 2^-24 sum_d |q_d k_d| scale from the f32 sums plus 2^-20 of the
exponent's size from its f32 form; and the result is rounded to its type (unit roundoff 2^-8 for the 8 significant bits
of bf16, 2^-11 for f16).  So

    |out - exact| <= ulp |exact| + (2^-11 + 2 e + 2^-18) sum_t w_t |v_t| + 2^-32 max_t (w_t s_t) sum_t |c_t|
    |lse - exact| <= e + 2^-18

with sum_t w_t = 1 and e the largest error of a visible score."""

import math

import numpy as np
import pytest

torch = pytest.importorskip("torch")

from pto_wsp_b200 import serving  # noqa: E402
from pto_wsp_b200.runtime import PtoWspCudaError  # noqa: E402

pytestmark = pytest.mark.gpu
FORMATS = {"e4m3": torch.float8_e4m3fn, "int8": torch.int8}


@pytest.fixture(autouse=True)
def _cuda(require_cuda):
    torch.manual_seed(0)


def dev(x, dtype):
    return torch.tensor(np.asarray(x), dtype=dtype, device="cuda")


# ---------------------------------------------------------------------------
# reserve_pages
# ---------------------------------------------------------------------------


def reserve_reference(table, lens, new, ring, free, page, max_tokens):
    """The definition, request after request."""
    table, ring, cap = table.copy(), ring.copy(), len(ring)
    before, (head, tail) = ring.copy(), free
    slots, positions, start, out, granted = [], [], [0], [], []
    taken = asked = 0
    for r, (n, x) in enumerate(zip(lens, new)):
        want, have = max(0, x), -(-n // page)
        after, first = -(-(n + want) // page), start[-1]
        start.append(first + want)
        fits = x >= 0 and after <= table.shape[1] and start[-1] <= max_tokens
        need = after - have if fits else 0
        asked += need
        ok = fits and (need == 0 or asked <= tail - head)
        granted.append(ok)
        if ok:
            for j in range(have, after):
                table[r, j] = before[(head + taken) % cap]
                taken += 1
        for i in range(want):
            slots.append(table[r, (n + i) // page] * page + (n + i) % page if ok else -1)
            positions.append(n + i if ok else -1)
        out.append(0 if x < 0 else n + (want if ok else 0))
    back = tail
    for r, x in enumerate(new):
        if x < 0:
            for j in range(-(-lens[r] // page)):
                ring[back % cap] = table[r, j]
                back += 1
    slots, positions = (np.array((v + [-1] * max_tokens)[:max_tokens], np.int64) for v in (slots, positions))
    return slots, positions, start, out, [head + taken, back], granted, table, ring


def reserve_case(rng, requests, page, max_len, new, max_pages, spare, head=0, max_tokens=None):
    lens = rng.integers(0, max_len + 1, requests)
    used = int(sum(-(-n // page) for n in lens))
    cap = used + spare
    perm = rng.permutation(cap).astype(np.int32)
    table = np.full((requests, max_pages), -1, np.int32)
    at = 0
    for r, n in enumerate(lens):
        k = -(-int(n) // page)
        table[r, :k] = perm[at:at + k]
        at += k
    ring = np.full(cap, -7, np.int32)
    for i in range(spare):
        ring[(head + i) % cap] = perm[used + i]
    new = np.asarray(new(rng, requests))
    total = int(np.maximum(new, 0).sum()) if max_tokens is None else max_tokens
    return table, lens, new, ring, [head, head + spare], page, total


@pytest.mark.parametrize("requests,page,max_len,new,max_pages,spare,head,max_tokens", [
    (1, 16, 0, lambda g, n: [1], 1, 1, 0, None),                              # the first token of the first request
    (1, 16, 16, lambda g, n: [0], 2, 0, 0, None),                             # nothing to do
    (7, 16, 100, lambda g, n: np.ones(n, int), 8, 7, 5, None),
    (33, 32, 300, lambda g, n: g.integers(0, 70, n), 13, 200, 11, None),
    (33, 32, 300, lambda g, n: g.integers(0, 70, n), 13, 20, 11, None),       # the ring runs dry
    (33, 32, 300, lambda g, n: g.integers(0, 70, n), 11, 200, 11, None),      # some pass the table
    (33, 32, 300, lambda g, n: g.integers(0, 70, n), 13, 200, 11, 500),       # some pass the token list
    (33, 32, 300, lambda g, n: g.integers(0, 70, n), 13, 200, 11, 4000),      # the list has room behind
    (60, 16, 90, lambda g, n: g.integers(-1, 3, n), 8, 30, 250, None),        # a third ends
    (2500, 16, 60, lambda g, n: g.integers(-1, 9, n), 5, 4000, 3, None),      # several rounds of the block scan
    (40, 1, 30, lambda g, n: g.integers(0, 9, n), 64, 300, 0, None),          # pages of one token
])
def test_reserve_against_the_definition(requests, page, max_len, new, max_pages, spare, head, max_tokens):
    rng = np.random.default_rng(requests * 7 + spare)
    table, lens, new, ring, free, page, total = reserve_case(rng, requests, page, max_len, new, max_pages, spare, head,
                                                             max_tokens)
    want = reserve_reference(table, lens.tolist(), new.tolist(), ring, free, page, total)
    wide = torch.full((requests, max_pages + 3), 99, dtype=torch.int32, device="cuda")  # rows of a wider table
    wide[:, :max_pages] = dev(table, torch.int32)
    t, ring_d = wide[:, :max_pages], dev(ring, torch.int32)
    status = torch.zeros(1, dtype=torch.int32, device="cuda")
    for _ in range(2):  # the call can be repeated on the same inputs
        step = serving.reserve_pages(t, dev(lens, torch.int32), dev(new, torch.int32), ring_d, dev(free, torch.int64),
                                     page_size=page, max_tokens=total, status=status)
        got = (step.slots, step.positions, step.q_start, step.kv_len, step.free_state, step.granted, t, ring_d)
        for g, w in zip(got, want):
            np.testing.assert_array_equal(g.cpu().numpy(), np.asarray(w).astype(g.cpu().numpy().dtype))
        assert (wide[:, max_pages:] == 99).all()
        refused = any(not ok and x >= 0 for ok, x in zip(want[5], new))
        assert int(status) == (serving.REFUSED if refused else 0)
        status.zero_()


@pytest.mark.parametrize("order", [[6016, 6017, 6112, 6144, 6145, 16384, 6145], [16384, 7000, 16384, 1]])
def test_reserve_of_many_requests(order):
    # more than some 6100 requests take more shared memory than a kernel has unasked; a smaller call may not lower the limit
    rng = np.random.default_rng(1)
    for requests in order:
        table, lens, new, ring, free, page, total = reserve_case(rng, requests, 16, 40, lambda g, n: g.integers(-1, 4, n),
                                                                 4, 9000, 5)
        want = reserve_reference(table, lens.tolist(), new.tolist(), ring, free, page, total)
        t, ring_d = dev(table, torch.int32), dev(ring, torch.int32)
        step = serving.reserve_pages(t, dev(lens, torch.int32), dev(new, torch.int32), ring_d, dev(free, torch.int64),
                                     page_size=page, max_tokens=total)
        got = (step.slots, step.positions, step.q_start, step.kv_len, step.free_state, step.granted, t, ring_d)
        for g, w in zip(got, want):
            np.testing.assert_array_equal(g.cpu().numpy(), np.asarray(w).astype(g.cpu().numpy().dtype))


def test_reserve_of_many_requests_from_several_threads():
    from concurrent.futures import ThreadPoolExecutor

    def work(requests):
        zeros, ones = (torch.full((requests,), x, dtype=torch.int32, device="cuda") for x in (0, 1))
        ring, free = torch.arange(requests, dtype=torch.int32, device="cuda"), dev([0, requests], torch.int64)
        table = torch.zeros(requests, 1, dtype=torch.int32, device="cuda")
        for _ in range(200):
            step = serving.reserve_pages(table, zeros, ones, ring, free, page_size=16, max_tokens=requests)
        return bool((step.slots == 16 * torch.arange(requests, device="cuda")).all())

    with ThreadPoolExecutor(4) as pool:
        assert all(pool.map(work, (6145, 16384, 9000, 16384)))


def test_reserve_reports_a_broken_ring_and_bad_lengths():
    def run(lens, new, state, cap=4):
        status = torch.zeros(1, dtype=torch.int32, device="cuda")
        step = serving.reserve_pages(torch.zeros(len(lens), 4, dtype=torch.int32, device="cuda"), dev(lens, torch.int32),
                                     dev(new, torch.int32), torch.arange(cap, dtype=torch.int32, device="cuda"),
                                     dev(state, torch.int64), page_size=16, max_tokens=8, status=status)
        return step, status

    step, status = run([3], [1], [5, 2])  # tail before head: nothing is given, a token in a page at hand still is
    assert int(status) == serving.RING and step.granted.tolist() == [True]
    step, status = run([16], [1], [0, 9])  # more free pages than places
    assert int(status) == serving.RING | serving.REFUSED and step.slots.tolist() == [-1] * 8
    step, status = run([64, 1], [-1, 1], [0, 3])  # four pages back, one place
    assert int(status) == serving.RING and step.free_state.tolist() == [0, 3]
    step, status = run([-5, 1000, 1], [1, 1, 1], [0, 4])
    assert int(status) & serving.LENGTH and step.granted.tolist() == [False, False, True]
    with pytest.raises(PtoWspCudaError, match="length"):
        serving.check_status(status)
    assert int(status) == 0
    serving.check_status(status)


@pytest.mark.parametrize("state", [[0, -3], [-5, -3], [-2, 1], [5, 2], [0, 9], [-(2 ** 63), 0], [0, 2 ** 63 - 1],
                                   [2 ** 63 - 3, 2 ** 63 - 2]])
def test_reserve_leaves_a_broken_ring_alone(state):
    wide = torch.arange(100, 112, dtype=torch.int32, device="cuda")
    ring, before = wide[4:8], wide.clone()  # words on both sides that nothing may touch
    table = torch.tensor([[50, 51, 0, 0], [60, 0, 0, 0], [70, 0, 0, 0]], dtype=torch.int32, device="cuda")
    status = torch.zeros(1, dtype=torch.int32, device="cuda")
    step = serving.reserve_pages(table.clone(), dev([20, 16, 3], torch.int32), dev([-1, 1, 1], torch.int32), ring,
                                 torch.tensor(state, device="cuda"), page_size=16, max_tokens=8, status=status)
    assert int(status) == serving.RING | serving.REFUSED  # no page for request 1; request 2 has room in its own
    assert torch.equal(wide, before) and step.free_state.tolist() == state
    assert step.granted.tolist() == [False, False, True] and step.kv_len.tolist() == [0, 16, 4]
    assert step.slots.tolist() == [-1, 70 * 16 + 3] + [-1] * 6


def test_reserve_without_requests():
    e = torch.empty(0, dtype=torch.int32, device="cuda")
    step = serving.reserve_pages(e.reshape(0, 4), e, e, torch.arange(3, dtype=torch.int32, device="cuda"),
                                 dev([1, 3], torch.int64), page_size=16, max_tokens=2)
    assert step.q_start.tolist() == [0] and step.free_state.tolist() == [1, 3] and step.slots.tolist() == [-1, -1]


# ---------------------------------------------------------------------------
# append_kv8
# ---------------------------------------------------------------------------


def new_cache(fmt, pages, page, heads, dim, layout):
    dtype = FORMATS[fmt]
    if layout == "hnd":
        return torch.zeros(pages, heads, page, dim, dtype=torch.int8, device="cuda").view(dtype).transpose(1, 2)
    if layout == "nhd":
        return torch.zeros(pages, page, heads, dim, dtype=torch.int8, device="cuda").view(dtype)
    # a padded one: K and V of a page interleaved in one buffer
    return torch.zeros(pages, 2, page, heads, dim, dtype=torch.int8, device="cuda").view(dtype)[:, 1]


def e4m3(x):
    """The nearest e4m3 value, ties to even, in 64 bits."""
    x = np.clip(x, -448, 448)
    a = np.maximum(np.abs(x), 2.0 ** -6)
    step = 2.0 ** (np.floor(np.log2(a)) - 3)
    return np.round(x / step) * step


def append_reference(x, slots, codes, scale, fmt):
    """The definition, page after page and head after head, in 64 bits but for the int8 scale, which is f32."""
    codes, scale = codes.astype(np.float64), scale.astype(np.float32).copy()
    page = codes.shape[1]
    touched = {}
    for i, s in enumerate(slots):
        if s >= 0:
            touched.setdefault(int(s) // page, []).append((i, int(s) % page))
    rounded = e4m3 if fmt == "e4m3" else (lambda v: np.clip(np.round(v), -127, 127))
    for p, items in touched.items():
        for h in range(codes.shape[2]):
            rows = np.array([x[i, h] for i, _ in items], np.float64)
            a = np.abs(rows[np.isfinite(rows)]).max(initial=0.0)
            if fmt == "int8":
                need = np.clip(np.float32(a) * (np.float32(1) / np.float32(127)), np.float32(2.0 ** -60), np.float32(2.0 ** 60))
            else:
                need = np.float32(2.0 ** np.clip(np.ceil(np.log2(a / 448)), -60, 60)) if a > 0 else np.float32(2.0 ** -60)
            old = scale[p, h]
            fresh = any(off == 0 for _, off in items)
            new = need if fresh else max(old, need)
            if not fresh and new > old:
                f32 = np.float32  # the product and the quotient are f32
                codes[p, :, h] = rounded((codes[p, :, h].astype(f32) * old / new).astype(np.float64))
            scale[p, h] = new
            for (i, off), row in zip(items, rows):
                row = np.where(np.isnan(row), 0.0, row).astype(np.float32)
                with np.errstate(over="ignore"):
                    codes[p, off, h] = rounded((row / new).astype(np.float64))
    return codes, scale


@pytest.mark.parametrize("fmt", ["e4m3", "int8"])
@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
@pytest.mark.parametrize("heads,dim,page,layout,runs", [
    (1, 64, 16, "hnd", [(0, 1)]),
    (2, 128, 16, "nhd", [(15, 1), (3, 14), (0, 40), (7, 1), (5, 11)]),
    (3, 64, 32, "split", [(31, 2), (1, 95), (0, 32), (0, 31)]),
    (8, 128, 64, "hnd", [(60, 200), (0, 1), (63, 1)]),
    (1, 128, 128, "nhd", [(100, 128), (0, 128), (1, 5)]),
])
def test_append_against_the_definition(fmt, dtype, heads, dim, page, layout, runs):
    rng = np.random.default_rng(dim + page)
    spans = [-(-(s + n) // page) for s, n in runs]
    pages = sum(spans) + 2
    perm, slots, at = rng.permutation(pages), [], 0
    for (s, n), k in zip(runs, spans):
        slots += [int(perm[at + (s + i) // page]) * page + (s + i) % page for i in range(n)]
        slots += [-1]  # a token without a slot between the runs
        at += k
    n = len(slots)
    caches, refs, xs = [], [], []
    fused = torch.randn(n, 2 * heads + 1, dim, device="cuda").to(dtype)  # k and v as views of one projection
    fused *= torch.exp(torch.randn(n, 2 * heads + 1, 1, device="cuda")).to(dtype)
    fused[:, :, 3] = -0.0
    for side in range(2):
        x = fused[:, side * heads:(side + 1) * heads]
        c = new_cache(fmt, pages, page, heads, dim, layout)
        start = torch.randn(c.shape, device="cuda") * 60
        c.copy_(start.clamp(-127, 127).round() if fmt == "int8" else start)
        scale = torch.exp2(torch.randint(-9, -5, (pages, heads), device="cuda").float())
        if fmt == "int8":
            scale *= torch.rand_like(scale) + 0.5
        refs.append(append_reference(x.float().cpu().numpy(), slots, c.float().cpu().numpy(), scale.cpu().numpy(), fmt))
        caches.append((c, scale))
        xs.append(x)
    (kc, ks), (vc, vs) = caches
    status = torch.zeros(1, dtype=torch.int32, device="cuda")
    for _ in range(2):  # writing the same tokens again changes nothing
        serving.append_kv8(*xs, dev(slots, torch.int64), kc, vc, ks, vs, status=status)
        for (c, scale), (codes, want) in zip(caches, refs):
            np.testing.assert_array_equal(scale.cpu().numpy(), want)
            np.testing.assert_array_equal(c.float().cpu().numpy(), codes)
    assert int(status) == 0


@pytest.mark.parametrize("fmt", ["e4m3", "int8"])
def test_append_of_zeros_infinities_and_nan(fmt):
    page, top = 16, 448.0 if fmt == "e4m3" else 127.0
    kc, vc = (new_cache(fmt, 4, page, 1, 64, "hnd") for _ in range(2))
    ks, vs = (torch.ones(4, 1, device="cuda") for _ in range(2))
    k = torch.zeros(3, 1, 64, device="cuda")
    k[1, 0, :4] = torch.tensor([math.inf, -math.inf, math.nan, 2.0])
    k[2] = 1e30
    serving.append_kv8(k, -k, dev([0, 16, 32], torch.int64), kc, vc, ks, vs)
    assert float(ks[0]) == 2.0 ** -60 and not kc[0].float().any()           # a page of zeros: the smallest scale
    assert kc[1, 0, 0, :3].float().tolist() == [top, -top, 0.0]             # infinities clamp, NaN is zero
    assert vc[1, 0, 0, :2].float().tolist() == [-top, top]
    assert abs(float(kc[1, 0, 0, 3].float() * ks[1]) - 2.0) < 2e-2          # and neither sets the scale
    assert float(ks[2]) == 2.0 ** 60 and float(kc[2, 0, 0, 0].float()) == top  # beyond the largest scale: clamped


def test_append_reports_slots_outside_the_cache():
    kc, vc = (new_cache("e4m3", 2, 16, 1, 64, "nhd") for _ in range(2))
    ks, vs = (torch.ones(2, 1, device="cuda") for _ in range(2))
    status = torch.zeros(1, dtype=torch.int32, device="cuda")
    x = torch.ones(4, 1, 64, device="cuda")
    serving.append_kv8(x, x, dev([32, -2, 31, 1 << 40], torch.int64), kc, vc, ks, vs, status=status)
    assert int(status) == serving.PAGE
    assert kc.float().count_nonzero() == 64 and float(kc[1, 15].float().min()) > 0


# ---------------------------------------------------------------------------
# attend_kv8
# ---------------------------------------------------------------------------


def paged(fmt, lens, page, heads, dim, layout, gen, spread=0.5, extra_pages=2):
    """A cache and a table for the lengths, and the real K, V and V scales of each request's tokens; what no request owns is NaN or the
    largest code, table entries behind a request's pages are out of range."""
    have = [-(-n // page) for n in lens]
    pages = sum(have) + extra_pages
    perm = torch.randperm(pages, generator=gen, device="cuda")
    table = torch.full((len(lens), max(have + [1]) + 1), 1 << 30, dtype=torch.int32, device="cuda")
    sides, at = [], 0
    for _ in range(2):
        c = new_cache(fmt, pages, page, heads, dim, layout)
        x = torch.randn(c.shape, generator=gen, device="cuda") * (96 if fmt == "e4m3" else 40)
        c.copy_(x.clamp(-448, 448) if fmt == "e4m3" else x.round().clamp(-127, 127))
        size = torch.exp(spread * torch.randn(pages, heads, generator=gen, device="cuda"))
        scale = torch.exp2(torch.round(torch.log2(size / 96))) if fmt == "e4m3" else size / 40
        sides.append([c, scale])
    owned = torch.zeros(pages, page, dtype=torch.bool, device="cuda")
    real = []
    for r, (n, k) in enumerate(zip(lens, have)):
        ids = perm[at:at + k]
        table[r, :k] = ids.int()
        at += k
        real.append([(c[ids].double() * s[ids].double()[:, None, :, None]).reshape(-1, heads, dim)[:n] for c, s in sides])
        real[-1].append(sides[1][1][ids].double()[:, None].expand(-1, page, -1).reshape(-1, heads)[:n])
        owned[ids] = (torch.arange(k * page, device="cuda") < n).reshape(k, page)
    for c, _ in sides:
        c.view(torch.int8).masked_fill_(~owned[:, :, None, None], 127)  # e4m3: NaN
    return sides, table, real


def attention_reference(q, real, lens, qs, window, scale):
    """In 64 bits, request after request: (out, lse, sum w|v|, largest error of a visible score, max(w s) sum |c|)."""
    outs, at = [], 0
    heads = real[0][0].shape[1] if real else 1
    group, dim = q.shape[1] // heads, q.shape[2]
    for (k, v, s), n, m in zip(real, lens, qs):
        x = q[at:at + m].double().reshape(m, heads, group, dim)
        z = torch.einsum("jhgd,thd->jhgt", x, k) * scale
        err = torch.einsum("jhgd,thd->jhgt", x.abs(), k.abs()) * abs(scale) * (dim + 8) * 2.0 ** -24 + z.abs() * 2.0 ** -20
        last = torch.arange(n - m, n, device="cuda")[:, None]
        t = torch.arange(n, device="cuda")[None]
        hidden = t > last
        if window:
            hidden = hidden | (t <= last - window)
        z = z.masked_fill(hidden[:, None, None], -math.inf)
        err = err.masked_fill(hidden[:, None, None], 0.0)
        if n == 0:
            z = torch.full((m, heads, group, 1), -math.inf, device="cuda", dtype=torch.float64)
            err, v = torch.zeros_like(z), torch.zeros(1, heads, dim, device="cuda", dtype=torch.float64)
            s = torch.ones(1, heads, device="cuda", dtype=torch.float64)
        lse = torch.logsumexp(z, -1)
        w = torch.exp(z - torch.where(torch.isinf(lse), 0.0, lse)[..., None])
        outs.append((torch.einsum("jhgt,thd->jhgd", w, v).reshape(m, heads * group, dim), lse.reshape(m, heads * group),
                     torch.einsum("jhgt,thd->jhgd", w, v.abs()).reshape(m, heads * group, dim),
                     err.amax(-1).reshape(m, heads * group),
                     ((w * s.T[:, None]).amax(-1)[..., None] * torch.einsum(
                         "jhgt,thd->jhgd", (w > 0).double(), v.abs() / s[..., None])).reshape(m, heads * group, dim)))
        at += m
    return [torch.cat(c) for c in zip(*outs)]


def check_attention(out, lse, want, dtype):
    ref, ref_lse, mass, e, floor = want
    assert not torch.isnan(out.float()).any()
    ulp = 2.0 ** -8 if dtype == torch.bfloat16 else 2.0 ** -11
    tol = ulp * ref.abs() + (2.0 ** -11 + 2 * e[..., None] + 2.0 ** -18) * mass + 2.0 ** -32 * floor + (6e-8 if dtype == torch.float16 else 0)
    off = (out.double() - ref).abs() - tol
    assert float(off.max()) <= 0, f"off by {float(off.max()):.3g} more than the tolerance"
    empty = torch.isinf(ref_lse)
    assert torch.equal(torch.isinf(lse) & (lse < 0), empty) and not out[empty].any()
    assert float(((lse.double() - ref_lse).abs() - e - 2.0 ** -18).masked_fill(empty, -1.0).max()) <= 0


def attend_case(fmt, dtype, heads, group, dim, page, lens, qs=None, window=0, layout="hnd", seed=0, spread=0.5,
                q_size=1.5, scale=None):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    (k, ks), (v, vs) = (sides := paged(fmt, lens, page, heads, dim, layout, gen, spread))[0]
    table, real = sides[1], sides[2]
    qs = qs or [1] * len(lens)
    q = (q_size * torch.randn(sum(qs), heads * group, dim, generator=gen, device="cuda")).to(dtype)
    start = None
    if max(qs) > 1 or min(qs) == 0:
        start = dev(np.cumsum([0] + list(qs)), torch.int32)
    status = torch.zeros(1, dtype=torch.int32, device="cuda")
    out, lse = serving.attend_kv8(q, k, v, ks, vs, table, dev(lens, torch.int32), q_start=start, max_q=max(qs),
                                  window=window, return_lse=True, status=status, scale=scale)
    want = attention_reference(q, real, lens, qs, window, dim ** -0.5 if scale is None else scale)
    check_attention(out, lse, want, dtype)
    assert int(status) == 0
    return out, lse


EDGES = [0, 1, 15, 16, 17, 31, 32, 33, 127, 128, 129, 255, 257, 500]


@pytest.mark.parametrize("fmt", ["e4m3", "int8"])
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("heads,group,dim,page,layout", [
    (2, 4, 128, 16, "hnd"), (1, 1, 64, 16, "nhd"), (3, 8, 128, 32, "split"), (2, 6, 64, 64, "hnd"),
    (1, 16, 128, 128, "nhd"), (2, 20, 64, 32, "hnd"), (1, 40, 128, 16, "nhd"),
])
def test_attend_one_token(fmt, dtype, heads, group, dim, page, layout):
    attend_case(fmt, dtype, heads, group, dim, page, EDGES, layout=layout)


@pytest.mark.parametrize("fmt", ["e4m3", "int8"])
@pytest.mark.parametrize("dim,group,page", [(128, 4, 16), (64, 2, 32), (128, 1, 64), (64, 8, 128)])
@pytest.mark.parametrize("window", [0, 1, 20, 130])
def test_attend_several_tokens(fmt, dim, group, page, window):
    lens = [1, 2, 7, 40, 128, 129, 131, 300, 17, 64, 5]
    qs = [1, 2, 7, 3, 1, 5, 8, 6, 0, 4, 8]  # the last one asks for more rows than it has tokens: three see nothing
    attend_case(fmt, torch.float16, 2, group, dim, page, lens, qs, window)


@pytest.mark.parametrize("fmt", ["e4m3", "int8"])
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("dim,heads,group,page,layout", [
    (128, 2, 4, 16, "hnd"), (64, 1, 2, 32, "nhd"), (128, 1, 1, 64, "split"), (64, 2, 6, 128, "hnd"),
    (128, 1, 16, 16, "nhd"),
])
@pytest.mark.parametrize("window", [0, 100])
def test_attend_prefill(fmt, dtype, dim, heads, group, page, layout, window):
    lens = [1, 130, 300, 64, 700, 257, 129, 20]
    qs = [1, 130, 37, 64, 1, 256, 0, 33]
    attend_case(fmt, dtype, heads, group, dim, page, lens, qs, window, layout)


@pytest.mark.parametrize("lens,qs", [([4000], [1]), ([9000, 3], [1, 1]), ([6000, 100], [3, 1]), ([5000, 2000], [400, 1])])
@pytest.mark.parametrize("heads,group", [(1, 1), (2, 4), (1, 12)])
def test_attend_long_histories_split_and_joined(lens, qs, heads, group):
    attend_case("e4m3", torch.float16, heads, group, 128, 16, lens, qs)


def test_attend_many_requests():
    rng = np.random.default_rng(3)
    attend_case("int8", torch.bfloat16, 2, 2, 64, 16, rng.integers(0, 200, 700).tolist())


@pytest.mark.parametrize("fmt", ["e4m3", "int8"])
@pytest.mark.parametrize("qs", [[1, 1], [60, 90]])
def test_attend_pages_of_very_different_size(fmt, qs):
    # V scales from 2^-12 to 2^12 of each other: the small pages' values must not drown in the large ones' rounding,
    # nor the weights overflow; K scales as wide give peaked rows
    attend_case(fmt, torch.bfloat16, 1, 4, 128, 16, [500, 333], qs, spread=2.5, q_size=0.5)


@pytest.mark.parametrize("qs", [[1, 1, 1], [5, 2, 8], [150, 40, 200]])
def test_attend_large_and_tiny_queries(qs):
    for size in (1e-30, 1e-6, 30.0):
        attend_case("e4m3", torch.bfloat16, 1, 2, 64, 16, [300, 40, 257], qs, q_size=size)
    attend_case("int8", torch.float16, 1, 2, 64, 16, [300, 40, 257], qs, q_size=1e-6)
    attend_case("int8", torch.float16, 1, 2, 64, 16, [300, 40, 257], qs, scale=-0.5)
    attend_case("int8", torch.float16, 1, 2, 64, 16, [300, 40, 257], qs, scale=0.0)


def test_attend_pages_freed_behind_the_window():
    gen = torch.Generator(device="cuda").manual_seed(1)
    lens, qs, window = [400, 333], [2, 40], 100
    (k, ks), (v, vs) = (made := paged("e4m3", lens, 16, 2, 128, "hnd", gen))[0]
    table, real = made[1], made[2]
    for r, (n, m) in enumerate(zip(lens, qs)):
        table[r, :(n - m + 1 - window) // 16] = -1  # given back: no row sees them
    q = torch.randn(sum(qs), 8, 128, device="cuda").half()
    status = torch.zeros(1, dtype=torch.int32, device="cuda")
    out, lse = serving.attend_kv8(q, k, v, ks, vs, table, dev(lens, torch.int32), q_start=dev([0, 2, 42], torch.int32),
                                  max_q=40, window=window, return_lse=True, status=status)
    check_attention(out, lse, attention_reference(q, real, lens, qs, window, 128 ** -0.5), q.dtype)
    assert int(status) == 0


@pytest.mark.parametrize("qs", [[1, 1, 1], [40, 3, 70]])
def test_attend_hides_bad_pages_and_reports_them(qs):
    gen = torch.Generator(device="cuda").manual_seed(2)
    lens = [300, 200, 180]
    (k, ks), (v, vs) = (made := paged("int8", lens, 16, 1, 64, "nhd", gen))[0]
    table, real = made[1], made[2]
    table[1, 3], table[1, 4] = -1, k.shape[0]
    x, y, z = real[1]
    keep = torch.ones(200, dtype=torch.bool, device="cuda")
    keep[48:80] = False
    q = torch.randn(sum(qs), 2, 64, device="cuda").bfloat16()
    status = torch.zeros(1, dtype=torch.int32, device="cuda")
    start = dev(np.cumsum([0] + qs), torch.int32)
    out, lse = serving.attend_kv8(q, k, v, ks, vs, table, dev(lens, torch.int32), q_start=start, max_q=max(qs),
                                  return_lse=True, status=status)
    assert int(status) == serving.PAGE
    real[1] = [x[keep], y[keep], z[keep]]  # the hidden tokens are all before the new ones
    check_attention(out, lse, attention_reference(q, real, [300, 168, 180], qs, 0, 0.125), q.dtype)
    # a length beyond the table is cut to it
    status.zero_()
    short = table[:, :3].contiguous()
    out, lse = serving.attend_kv8(q, k, v, ks, vs, short, dev(lens, torch.int32), q_start=start, max_q=max(qs),
                                  return_lse=True, status=status)
    assert int(status) & serving.LENGTH
    assert not torch.isnan(out.float()).any()


@pytest.mark.parametrize("qs", [[1, 1], [3, 5], [70, 40]])
def test_attend_strided_rows_other_stream_and_repeat(qs):
    gen = torch.Generator(device="cuda").manual_seed(5)
    lens = [500, 90]
    (k, ks), (v, vs) = (made := paged("e4m3", lens, 16, 2, 128, "nhd", gen))[0]
    fused = torch.randn(sum(qs), 3, 8, 128, generator=gen, device="cuda").half()  # q as a view of one projection
    q = fused[:, 1]
    want = attention_reference(q, made[2], lens, qs, 0, 128 ** -0.5)
    args = (k, v, ks, vs, made[1], dev(lens, torch.int32))
    more = {"q_start": dev(np.cumsum([0] + qs), torch.int32), "max_q": max(qs), "return_lse": True}
    first, lse = serving.attend_kv8(q, *args, **more)
    check_attention(first, lse, want, q.dtype)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        wide = torch.full((sum(qs), 8, 256), 7.0, dtype=q.dtype, device="cuda")
        serving.attend_kv8(q, *args, out=wide[:, :, 128:], **more)
    side.synchronize()
    assert torch.equal(wide[:, :, 128:], first) and (wide[:, :, :128] == 7).all()  # the same bits, and nothing beside
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        again, _ = serving.attend_kv8(q, *args, **more)
    again.zero_()
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(again, first)


@pytest.mark.parametrize("fmt,group,qs", [("int8", 8, [1200, 900, 1500, 700]), ("e4m3", 4, [1900, 1800, 2100]),
                                          ("int8", 8, [1, 2, 1, 3] * 40)])
def test_attend_gives_the_same_bits_every_time(fmt, group, qs):
    # Many short tasks per CTA: the copy of a coming tile may not pass the reads of the present one, which stand in a queue
    # behind the stores of the task before.
    gen = torch.Generator(device="cuda").manual_seed(11)
    lens = [n + 300 * (i % 3) for i, n in enumerate(qs)]
    (k, ks), (v, vs) = (made := paged(fmt, lens, 16, 1, 128, "hnd", gen))[0]
    q = (1.5 * torch.randn(sum(qs), group, 128, generator=gen, device="cuda")).half()
    args = (q, k, v, ks, vs, made[1], dev(lens, torch.int32))
    more = {"q_start": dev(np.cumsum([0] + qs), torch.int32), "max_q": max(qs), "window": 1100, "return_lse": True}
    first, first_lse = serving.attend_kv8(*args, **more)
    check_attention(first, first_lse, attention_reference(q, made[2], lens, qs, 1100, 128 ** -0.5), q.dtype)
    runs = [serving.attend_kv8(*args, **more) for _ in range(150)]
    assert all(torch.equal(o, first) and torch.equal(l, first_lse) for o, l in runs)


@pytest.mark.parametrize("fmt,heads,group,dim", [("e4m3", 2, 2, 128), ("int8", 1, 4, 64)])
def test_attend_full_tiles_after_short_ones(fmt, heads, group, dim):
    # 256 and then 24 to 104 rows per request and head: one of the two row tiles sits the second part out, whose number of
    # steps varies, and comes back where the pages' scales are others, up to 2^15 apart.
    gen = torch.Generator(device="cuda").manual_seed(12)
    qs = [(256 + 24 + 16 * (i % 6)) // group for i in range(150)]
    lens = [m + 37 * (i % 23) for i, m in enumerate(qs)]
    (k, ks), (v, vs) = (made := paged(fmt, lens, 16, heads, dim, "hnd", gen, spread=2.0))[0]
    q = (0.5 * torch.randn(sum(qs), heads * group, dim, generator=gen, device="cuda")).half()
    args = (q, k, v, ks, vs, made[1], dev(lens, torch.int32))
    more = {"q_start": dev(np.cumsum([0] + qs), torch.int32), "max_q": max(qs), "return_lse": True}
    first, first_lse = serving.attend_kv8(*args, **more)
    check_attention(first, first_lse, attention_reference(q, made[2], lens, qs, 0, dim ** -0.5), q.dtype)
    runs = [serving.attend_kv8(*args, **more) for _ in range(50)]
    assert all(torch.equal(o, first) and torch.equal(l, first_lse) for o, l in runs)


@pytest.mark.parametrize("qs,max_q", [([1, 5, 2, 0, 3], 3), ([1, 40, 2, 70, 3], 64), ([2, 4, 1, 3, 1], 1)])
@pytest.mark.parametrize("front,back", [(0, 0), (3, 0), (0, 50), (2, 700)])
def test_attend_rows_without_a_request(qs, max_q, front, back):
    # rows before the first request's and behind the last one's, and requests of more rows than max_q: zeros, lse -inf
    gen = torch.Generator(device="cuda").manual_seed(8)
    lens = [100, 90, 33, 12, 400]
    (k, ks), (v, vs) = (made := paged("e4m3", lens, 16, 2, 64, "hnd", gen))[0]
    rows = front + sum(qs) + back
    q = torch.randn(rows, 8, 64, generator=gen, device="cuda").half()
    start = np.cumsum([front] + qs)
    status = torch.zeros(1, dtype=torch.int32, device="cuda")
    wide = torch.full((rows, 8, 96), math.nan, dtype=q.dtype, device="cuda")
    out = wide[:, :, 16:80]
    del_me = torch.full((rows, 8), math.nan, device="cuda")  # where lse will probably stand
    del del_me
    _, lse = serving.attend_kv8(q, k, v, ks, vs, made[1], dev(lens, torch.int32), q_start=dev(start, torch.int32),
                                max_q=max_q, return_lse=True, status=status, out=out)
    want = attention_reference(q[front:front + sum(qs)], made[2], lens, qs, 0, 0.125)
    taken = torch.zeros(rows, dtype=torch.bool, device="cuda")
    for a, m in zip(start, qs):
        if m <= max_q:
            taken[a:a + m] = True
    inner = taken[front:front + sum(qs)]
    check_attention(out[taken], lse[taken], [c[inner] for c in want], q.dtype)
    assert not out[~taken].any() and bool((lse[~taken] == -math.inf).all())
    assert bool(torch.isnan(wide[:, :, :16]).all()) and bool(torch.isnan(wide[:, :, 80:]).all())
    assert int(status) == (serving.LENGTH if max(qs) > max_q else 0)


@pytest.mark.parametrize("qs", [[1, 1, 1], [3, 1, 4], [60, 1, 40]])
def test_attend_without_max_q(qs):
    gen = torch.Generator(device="cuda").manual_seed(9)
    lens = [100, 90, 300]
    (k, ks), (v, vs) = (made := paged("int8", lens, 16, 2, 128, "nhd", gen))[0]
    q = torch.randn(sum(qs), 8, 128, generator=gen, device="cuda").bfloat16()
    out, lse = serving.attend_kv8(q, k, v, ks, vs, made[1], dev(lens, torch.int32), return_lse=True,
                                  q_start=dev(np.cumsum([0] + qs), torch.int32))
    check_attention(out, lse, attention_reference(q, made[2], lens, qs, 0, 128 ** -0.5), q.dtype)


def test_attend_rows_without_any_request():
    gen = torch.Generator(device="cuda").manual_seed(10)
    (k, ks), (v, vs) = (made := paged("int8", [20], 16, 2, 64, "nhd", gen))[0]
    none = torch.empty(0, dtype=torch.int32, device="cuda")
    for rows in (1, 100):
        q = torch.randn(rows, 4, 64, device="cuda").half()
        out, lse = serving.attend_kv8(q, k, v, ks, vs, made[1][:0], none, q_start=dev([0], torch.int32), return_lse=True,
                                      out=torch.full_like(q, math.nan))
        assert not out.any() and bool((lse == -math.inf).all())
        with pytest.raises(PtoWspCudaError):  # a row per request, but there is none
            serving.attend_kv8(q, k, v, ks, vs, made[1][:0], none)


@pytest.mark.parametrize("window", [2 ** 31 - 1, 2 ** 31 - 5, 2 ** 30, 600])
@pytest.mark.parametrize("lens,qs", [([300, 20, 130, 1], [40, 37, 138, 5]), ([5, 60, 2], [8, 3, 5])])
def test_attend_windows_longer_than_the_history(window, lens, qs):
    # with requests of more rows than tokens, whose first rows see nothing
    out, lse = attend_case("e4m3", torch.float16, 1, 2, 128, 16, lens, qs, window)
    plain, plain_lse = attend_case("e4m3", torch.float16, 1, 2, 128, 16, lens, qs)
    assert torch.equal(out, plain) and torch.equal(lse, plain_lse)


def test_strides_of_dimensions_of_one_element():
    # one page, one head, one token: nothing steps by their strides, whatever they are
    gen = torch.Generator(device="cuda").manual_seed(13)
    fill = lambda *size: torch.randn(size, generator=gen, device="cuda")  # noqa: E731
    odd = lambda t: torch.as_strided(t, (1, *t.shape), (1027, *t.stride()))  # noqa: E731
    for dtype in (torch.float16, torch.float32):
        kc, vc = (torch.zeros(16, 128, dtype=torch.int8, device="cuda") for _ in range(2))
        kc, vc = (torch.as_strided(c, (1, 16, 1, 128), (5, 128, 3, 1)) for c in (kc, vc))
        ks, vs = (torch.ones(1, 1, device="cuda") for _ in range(2))
        k, v = fill(2, 1, 1, 128).to(dtype)
        k, v = (torch.as_strided(x, (1, 1, 128), (7, 5, 1)) for x in (k, v))
        serving.append_kv8(k, v, dev([0], torch.int64), kc, vc, ks, vs)
        assert torch.allclose(kc[0, 0].float() * ks, k[0].float(), atol=0.02)
        assert torch.allclose(vc[0, 0].float() * vs, v[0].float(), atol=0.02)
        for group in (1, 4):
            q, out = (odd(fill(group, 128).half()) for _ in range(2))
            if group == 1:
                q, out = (torch.as_strided(x, (1, 1, 128), (3, 5, 1)) for x in (q, out))
            got = serving.attend_kv8(q, kc, vc, ks, vs, dev([[0]], torch.int32), dev([1], torch.int32), out=out)
            assert torch.allclose(got.float(), (vc[0, 0].float() * vs).expand(1, group, 128), atol=1e-2)


def test_attend_offsets_beyond_32_bits():
    pages, page, heads, dim = 140_000, 16, 8, 128  # 2.3e9 codes
    gen = torch.Generator(device="cuda").manual_seed(6)
    k = torch.empty(pages, page, heads, dim, dtype=torch.int8, device="cuda")
    v = torch.empty_like(k)
    ks, vs = (torch.full((pages, heads), 1 / 40, device="cuda") for _ in range(2))
    n = 200
    ids = torch.arange(pages - 13, pages, device="cuda")
    slots = (ids.repeat_interleave(page) * page + torch.arange(page, device="cuda").repeat(13))[:n]
    x = torch.randn(2, n, heads, dim, generator=gen, device="cuda").half()
    serving.append_kv8(x[0], x[1], slots, k, v, ks, vs)
    real = [(c[ids].double() * s[ids].double()[:, None, :, None]).reshape(-1, heads, dim)[:n] for c, s in ((k, ks), (v, vs))]
    real.append(vs[ids].double()[:, None].expand(-1, page, -1).reshape(-1, heads)[:n])
    assert float((real[0] - x[0].double()).abs().max()) < 0.03
    for m in (1, 40):
        q = torch.randn(m, heads * 2, dim, generator=gen, device="cuda").half()
        out, lse = serving.attend_kv8(q, k, v, ks, vs, ids[None].int(), dev([n], torch.int32),
                                      q_start=dev([0, m], torch.int32), max_q=m, return_lse=True)
        check_attention(out, lse, attention_reference(q, [real], [n], [m], 0, dim ** -0.5), q.dtype)


def test_attend_refusals():
    gen = torch.Generator(device="cuda").manual_seed(7)
    (k, ks), (v, vs) = (made := paged("int8", [20], 16, 2, 64, "nhd", gen))[0]
    q, n = torch.randn(1, 4, 64, device="cuda").half(), dev([20], torch.int32)
    table = made[1]
    for args, error in (((q.float(), k, v, ks, vs, table, n), TypeError), ((q, k.half(), v, ks, vs, table, n), TypeError),
                        ((q, k, v.half(), ks, vs, table, n), TypeError), ((q, k, v, ks.double(), vs, table, n), TypeError),
                        ((q, k, v, ks[:, :1], vs, table, n), ValueError), ((q, k, v, ks, vs, table.long(), n), TypeError),
                        ((q, k, v, ks, vs, table, n.long()), TypeError), ((q[:, :3], k, v, ks, vs, table, n), PtoWspCudaError),
                        ((q[..., :32], k, v, ks, vs, table, n), ValueError), ((q, k, v, ks, vs, table.cpu(), n), ValueError),
                        ((q, k[:, :8], v[:, :8], ks, vs, table, n), PtoWspCudaError),
                        ((torch.cat([q, q]), k, v, ks, vs, table, n), PtoWspCudaError)):
        with pytest.raises(error):
            serving.attend_kv8(*args)
    with pytest.raises(ValueError):
        serving.attend_kv8(q, k, v, ks, vs, table, n, out=torch.empty(2, 4, 64, device="cuda").half())


def test_inputs_that_require_a_gradient():
    gen = torch.Generator(device="cuda").manual_seed(7)
    (k, ks), (v, vs) = (made := paged("int8", [20], 16, 2, 64, "nhd", gen))[0]
    q, x, n, u = torch.randn(1, 4, 64).half(), torch.randn(1, 2, 64), dev([20], torch.int32), torch.rand(1, device="cuda")
    q, x, logits = (t.cuda().requires_grad_() for t in (q, x, torch.randn(1, 50)))
    calls = (lambda: serving.attend_kv8(q, k, v, ks, vs, made[1], n), lambda: serving.sample_tokens(logits, u),
             lambda: serving.append_kv8(x, x.detach(), dev([0], torch.int64), k, v, ks, vs),
             lambda: serving.append_kv8(x.detach(), x, dev([0], torch.int64), k, v, ks, vs))
    for call in calls:
        with pytest.raises(ValueError, match="gradient"):
            call()
        with torch.no_grad():
            call()
        with torch.inference_mode():
            call()


# ---------------------------------------------------------------------------
# sample_tokens
# ---------------------------------------------------------------------------


def check_sample(x, u, token, logprob, temperature=None, top_k=None, top_p=None, min_p=None):
    """The token against the definition in 64 bits: it is a candidate, and the running sum passes u at it; both up to
    2^-18 of the sum (V 2^-40 from the whole-number weights, 2^-23 per weight from f32)."""
    tol = 2.0 ** -18
    for r in range(x.shape[0]):
        row, i = np.where(np.isnan(x[r]), -np.inf, x[r].astype(np.float64)), int(token[r])
        t = 1.0 if temperature is None else float(temperature[r])
        if row.max() == -np.inf:
            assert i == -1 and logprob[r] == -np.inf
            continue
        if not t > 0:
            assert i == int(row.argmax()) and logprob[r] == 0
            continue
        order = np.argsort(-row, kind="stable")
        rank = np.empty_like(order)
        rank[order] = np.arange(row.size)
        with np.errstate(invalid="ignore"):
            w = np.where(row == row.max(), 1.0, np.exp((row - row.max()) / t))
        kept = np.ones(row.size, bool)
        if top_k is not None and top_k[r] > 0:
            kept &= rank < top_k[r]
        m = 0.0 if min_p is None else min(1.0, float(min_p[r]))
        assert kept[i] and w[i] >= m * (1 - tol) and w[i] > 0
        kept &= w >= m
        total = (w * kept).sum()
        p = 1.0 if top_p is None else float(top_p[r])
        before = np.cumsum((w * kept)[order])[rank] - w  # the mass of what comes first
        if p < 1:
            assert rank[i] == 0 or before[i] < p * total + tol * total
            kept &= (before < p * total) | (rank == 0)
            total = (w * kept).sum()
            # the candidate at the edge may be in or out by rounding
            slack = tol * total + (w[kept].min() if abs(before[kept].max() - p * (w * (w >= m)).sum()) < tol * total else 0)
        else:
            slack = tol * total
        end = np.cumsum(w * kept)[i]
        assert end - w[i] - slack <= float(u[r]) * total <= end + slack, (r, i, end, w[i], float(u[r]) * total)
        assert abs(logprob[r] - math.log(w[i] / total)) < 1e-5 * max(1.0, abs(logprob[r])) + slack / total


def run_sample(x, u, **settings):
    token, logprob = serving.sample_tokens(x, u, **settings)
    host = {k: None if s is None else s.cpu().numpy() for k, s in settings.items()}
    check_sample(x.float().cpu().numpy(), u.cpu().numpy(), token.cpu().numpy(), logprob.cpu().numpy(), **host)
    return token, logprob


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
@pytest.mark.parametrize("rows,vocab", [(1, 1), (3, 2), (5, 31), (4, 1000), (7, 1025), (3, 4097), (16, 32000), (2, 131072),
                                        (3, 100003), (300, 517), (1, 262145)])
@pytest.mark.parametrize("filters", ["", "k", "p", "m", "kp", "kpm"])
def test_sample_against_the_definition(dtype, rows, vocab, filters):
    x = (3 * torch.randn(rows, vocab, device="cuda")).to(dtype)
    rand = lambda: torch.rand(rows, device="cuda")  # noqa: E731
    t = 0.3 + rand()
    t[::4] = 0.0
    run_sample(x, rand(), temperature=t,
               top_k=torch.randint(0, max(2, min(vocab + 2, 300)), (rows,), device="cuda", dtype=torch.int32) if "k" in filters else None,
               top_p=rand() if "p" in filters else None, min_p=0.3 * rand() if "m" in filters else None)


@pytest.mark.parametrize("vocab", [5, 1024, 40_000])
def test_sample_ties_go_to_the_lowest_index(vocab):
    rows = 64
    u = torch.arange(rows, device="cuda").float() / rows
    x = torch.zeros(rows, vocab, device="cuda")
    x[:, ::2] = -0.0  # the same value
    k = torch.full((rows,), 4, dtype=torch.int32, device="cuda")
    token, logprob = serving.sample_tokens(x, u, top_k=k)
    assert token.tolist() == [int(4 * i / rows) for i in range(rows)]  # the first four, evenly
    assert torch.allclose(logprob, torch.full_like(logprob, math.log(0.25)))
    p = torch.full((rows,), 0.5, device="cuda")
    token, _ = serving.sample_tokens(x, u, top_p=p)
    half = -(-vocab // 2)
    assert token.tolist() == [min(half - 1, int(half * i / rows)) for i in range(rows)]
    token, logprob = serving.sample_tokens(x, u, temperature=torch.zeros(rows, device="cuda"))
    assert not token.any() and not logprob.any()


def test_sample_masked_and_broken_rows():
    inf, nan = math.inf, math.nan
    x = torch.tensor([[-inf] * 6, [nan] * 6, [nan, -inf, 1, -inf, nan, 1], [-inf, -inf, -inf, -1e38, -inf, -inf],
                      [0, inf, 3, inf, nan, -inf], [3e38, -3e38, 0, 0, 0, 0], [-3.4028235e38] * 5 + [-3.4e38]], device="cuda")
    u = torch.full((7,), 0.7, device="cuda")
    for settings in ({}, {"top_p": torch.full((7,), 0.9, device="cuda")},
                     {"top_k": torch.full((7,), 2, dtype=torch.int32, device="cuda")},
                     {"temperature": torch.full((7,), 0.1, device="cuda")}):
        token, logprob = serving.sample_tokens(x, u, **settings)
        assert token.tolist()[:6] == [-1, -1, 5, 3, 3, 0], settings
        assert logprob.tolist()[:2] == [-inf, -inf] and logprob.tolist()[3] == 0
    assert serving.sample_tokens(x[6:], u[6:])[0].tolist() == [5]


def test_sample_edges_of_the_settings():
    rows, vocab = 9, 3000
    x = torch.randn(rows, vocab, device="cuda")
    big = x.argmax(-1).int()
    u = torch.tensor([0.0, 0.5, 0.99999994] * 3, device="cuda")
    full = lambda v, d=torch.float32: torch.full((rows,), v, dtype=d, device="cuda")  # noqa: E731
    for settings in ({"top_k": full(1, torch.int32)}, {"top_p": full(0.0)}, {"top_p": full(-1.0)}, {"min_p": full(1.0)},
                     {"min_p": full(7.0)}, {"temperature": full(-2.0)}, {"temperature": full(math.nan)},
                     {"temperature": full(1e-30)}):
        assert torch.equal(serving.sample_tokens(x, u, **settings)[0], big), settings
    plain = serving.sample_tokens(x, u)[0]
    for settings in ({"top_k": full(0, torch.int32)}, {"top_k": full(vocab, torch.int32)}, {"top_k": full(-3, torch.int32)},
                     {"top_p": full(1.0)}, {"top_p": full(2.0)}, {"min_p": full(0.0)}, {"temperature": full(1.0)}):
        assert torch.equal(serving.sample_tokens(x, u, **settings)[0], plain), settings
    assert torch.equal(serving.sample_tokens(x, full(-1.0))[0], serving.sample_tokens(x, full(0.0))[0])
    assert torch.equal(serving.sample_tokens(x, full(5.0))[0], serving.sample_tokens(x, full(1.0))[0])
    even = serving.sample_tokens(x, u, temperature=full(math.inf))[0]  # every token alike
    assert (even - (u * vocab).int()).abs().max() <= 1


def test_sample_rows_of_a_wider_tensor_and_refusals():
    x = torch.randn(5, 3001, device="cuda").bfloat16()
    u = torch.rand(5, device="cuda")
    run_sample(x[:, 1:], u, top_p=torch.full((5,), 0.8, device="cuda"))  # rows begin at odd addresses
    run_sample(x[::2, 7:2000], u[::2].contiguous())
    with pytest.raises(TypeError):
        serving.sample_tokens(x.double(), u)
    with pytest.raises(ValueError):
        serving.sample_tokens(x.T, u)
    with pytest.raises(ValueError):
        serving.sample_tokens(x, u[:4])
    with pytest.raises(TypeError):
        serving.sample_tokens(x, u, top_k=torch.ones(5, device="cuda"))
    with pytest.raises(ValueError):
        serving.sample_tokens(x, u.cpu())


def test_sample_shares_follow_the_distribution():
    # a grid of u over one row gives every candidate its share to within one
    rows, vocab = 4096, 50
    x = torch.randn(1, vocab, device="cuda").expand(rows, vocab)  # rows that share memory
    u = (torch.arange(rows, device="cuda").float() + 0.5) / rows
    token, _ = serving.sample_tokens(x, u)
    share = torch.bincount(token.long(), minlength=vocab).double()
    assert float((share - torch.softmax(x[0].double(), 0) * rows).abs().max()) <= 1.001


def test_a_whole_step_in_a_graph():
    # reserve, append, attend and sample captured once and replayed, the state in place, against the same calls one by one
    requests, heads, group, dim, vocab, page, steps = 5, 2, 4, 64, 700, 16, 40
    gen = torch.Generator(device="cuda").manual_seed(14)
    most = 12  # rows of a step: fewer are used, the rest is padding
    x = torch.randn(steps, 3, most, heads * group, dim, generator=gen, device="cuda").half()
    u = torch.rand(steps, requests, generator=gen, device="cuda")
    new = torch.randint(0, 3, (steps, requests), generator=gen, device="cuda", dtype=torch.int32)
    new[17, 2] = new[23, 0] = -1
    weight = torch.randn(heads * group * dim, vocab, generator=gen, device="cuda").half()
    top_p = torch.full((requests,), 0.9, device="cuda")

    def state():
        cache = [torch.zeros(60, heads, page, dim, dtype=torch.int8, device="cuda").transpose(1, 2) for _ in range(2)]
        return cache + [torch.ones(60, heads, device="cuda") for _ in range(2)], {
            "table": torch.zeros(requests, 8, dtype=torch.int32, device="cuda"), "ring": torch.arange(60, device="cuda").int(),
            "len": torch.zeros(requests, dtype=torch.int32, device="cuda"), "free": dev([0, 60], torch.int64),
            "status": torch.zeros(1, dtype=torch.int32, device="cuda")}

    def step(cache, s, x, new, u):
        plan = serving.reserve_pages(s["table"], s["len"], new, s["ring"], s["free"], page_size=page, max_tokens=most,
                                     status=s["status"])
        serving.append_kv8(x[1][:, :heads], x[2][:, :heads], plan.slots, *cache, status=s["status"])
        a, lse = serving.attend_kv8(x[0], *cache, s["table"], plan.kv_len, q_start=plan.q_start, max_q=2, return_lse=True,
                                    status=s["status"])
        rows = (plan.q_start[1:] - 1).clamp(min=0).long()
        token, logprob = serving.sample_tokens(a.reshape(most, -1)[rows] @ weight, u, top_p=top_p)
        s["len"].copy_(plan.kv_len)
        s["free"].copy_(plan.free_state)
        return a, lse, token, logprob

    one, other = state(), state()
    want = [[t.clone() for t in step(*one, x[i], new[i], u[i])] for i in range(steps)]
    ins = [x[0].clone(), torch.zeros_like(new[0]), u[0].clone()]
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):  # the calls before have loaded the code
        got = step(*other, *ins)
    for i in range(steps):
        for to, t in zip(ins, (x, new, u)):
            to.copy_(t[i])
        graph.replay()
        for name, w, g in zip(("out", "lse", "token", "logprob"), want[i], got):
            assert torch.equal(w, g), (i, name)
        pad = int(new[i].clamp(min=0).sum())
        assert not got[0][pad:].any()
    for a, b in zip([*one[0], *one[1].values()], [*other[0], *other[1].values()]):
        assert torch.equal(a, b)
    serving.check_status(other[1]["status"])


def test_attend_from_several_threads():
    from concurrent.futures import ThreadPoolExecutor

    gen = torch.Generator(device="cuda").manual_seed(15)
    cases = []
    for lens, qs in (([700, 20], [1, 1]), ([500, 300], [70, 1]), ([90, 4000], [3, 5]), ([260, 300], [200, 256])):
        (k, ks), (v, vs) = (made := paged("e4m3", lens, 16, 2, 128, "hnd", gen))[0]
        q = torch.randn(sum(qs), 8, 128, generator=gen, device="cuda").half()
        more = {"q_start": dev(np.cumsum([0] + qs), torch.int32), "max_q": max(qs)}
        args = (q, k, v, ks, vs, made[1], dev(lens, torch.int32))
        cases.append((args, more, serving.attend_kv8(*args, **more)))
    torch.cuda.synchronize()

    def work(case):
        args, more, want = case
        with torch.cuda.stream(torch.cuda.Stream()):
            got = [serving.attend_kv8(*args, **more) for _ in range(50)]
            torch.cuda.current_stream().synchronize()
            return all(torch.equal(g, want) for g in got)

    with ThreadPoolExecutor(4) as pool:
        assert all(pool.map(work, cases))
