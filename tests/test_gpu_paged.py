"""The paged-cache operators against their definitions in 64 bits.

Pools hold pages in no order, with NaN scales in every row that no sequence holds: a row read by
mistake shows. Tolerances (derived here, before any run):

* queries out of append: f32 arithmetic, a few roundings of 2^-24 each, then one rounding to the row type;
* codes: value rows, and key rows without norm and with the identity rotation, equal the quantizer's bytes
  (its arithmetic is the reference's); normed and rotated keys lie within half a step of the exact
  value, plus 1e-3 step for the f32 arithmetic before it;
* attention: the queries' f16 parts and the f32 sums move a score by less than 2^-21 |q| |k| / sqrt(d)
  (two parts), and weights by that plus 2^-22; below, |q| |k| / sqrt(d) < 40, so 4e-5 of the largest
  |v|. 16-bit rows: the query is exact in one part, a weight rounds by 2^-11, and the output once to its type.
"""

import threading

import numpy as np
import pytest
import torch

from qwenscriber_b200 import paged, quant
from qwenscriber_b200 import runtime as rt

pytestmark = pytest.mark.gpu

TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
UNIT = {"f32": 2.0 ** -23, "f16": 2.0 ** -11, "bf16": 2.0 ** -8}


class World:
    """A pool, a batch and their contents on the host."""

    def __init__(self, query, context, page, kv_heads, dim, seed=0, extra_pages=3):
        r = np.random.default_rng(seed)
        self.query, self.context = np.asarray(query), np.asarray(context)
        self.page, self.kv_heads, self.dim = page, kv_heads, dim
        need = -(-self.context // page)
        self.pages = int(need.sum()) + extra_pages
        order = r.permutation(self.pages)
        self.table = np.full((len(query), max(1, int(need.max()))), -1, np.int32)
        at = 0
        for s, n in enumerate(need):
            self.table[s, :n] = order[at:at + n]
            at += n
        width = kv_heads * dim
        rows = self.pages * page
        self.scales, self.codes = {}, {}
        held = np.zeros(rows, bool)
        for s, c in enumerate(self.context):
            held[self.rows(s, np.arange(c))] = True
        for n, size in (("k", 1.0), ("v", 0.7)):
            sc, co = quant.quantize(quant.Q8, (r.standard_normal((rows, width)) * size).astype(np.float32))
            sc = sc.reshape(rows, -1).copy()
            sc[~held] = 0x7E00  # NaN
            co[~held] = 255
            self.scales[n], self.codes[n] = sc.view(np.float16), co
        self.starts = np.concatenate([[0], np.cumsum(self.query)]).astype(np.int32)
        self.tokens = int(self.starts[-1])
        self.held = held

    def rows(self, s, pos):
        return self.table[s, pos // self.page].astype(np.int64) * self.page + pos % self.page

    def device(self, dev):
        put = lambda a: torch.from_numpy(np.ascontiguousarray(a)).to(dev)  # noqa: E731
        self.cache = paged.PagedCache(put(self.scales["k"]), put(self.codes["k"]), put(self.scales["v"]),
                                      put(self.codes["v"]), page_size=self.page, kv_heads=self.kv_heads, head_dim=self.dim)
        self.batch = paged.PagedBatch(put(self.starts), put(self.context.astype(np.int32)), put(self.table),
                                      tokens=self.tokens, max_query=int(self.query.max(initial=0)),
                                      max_context=int(self.context.max(initial=0)))
        return self.cache, self.batch

    def values(self, name, rows):
        s = self.scales[name][rows].astype(np.float64).repeat(64, axis=1)
        return ((self.codes[name][rows].astype(np.float64) - 128) * s).reshape(len(rows), self.kv_heads, self.dim)

    def attention(self, q):
        """softmax(q k / sqrt(d)) v over the positions that each token sees, in 64 bits."""
        heads = q.shape[1]
        out = np.zeros((self.tokens, heads, self.dim))
        for s in range(len(self.query)):
            n, c = int(self.query[s]), int(self.context[s])
            pos = np.arange(c)
            ok = (self.table[s, pos // self.page] >= 0) & (self.table[s, pos // self.page] < self.pages)
            pos = pos[ok]
            rows = self.rows(s, pos)
            k, v = self.values("k", rows), self.values("v", rows)
            for i in range(n):
                seen = pos <= c - n + i
                if not seen.any():
                    continue
                for h in range(heads):
                    g = h // (heads // self.kv_heads)
                    z = k[seen, g] @ q[self.starts[s] + i, h] / np.sqrt(self.dim)
                    w = np.exp(z - z.max())
                    out[self.starts[s] + i, h] = w @ v[seen, g] / w.sum()
        return out


def check_attention(world, kind, heads, gpu, seed=1, strided=False, size=1.0):
    cache, batch = world.device(gpu)
    g = torch.Generator().manual_seed(seed)
    wide = torch.randn(max(1, world.tokens), heads + (3 if strided else 0), world.dim, generator=g) * size
    wide = wide.to(TYPES[kind]).to(gpu)
    q = wide[:world.tokens, :heads]
    out = None
    if strided:
        out = torch.full((world.tokens, heads + 1, world.dim), 7.0, dtype=TYPES[kind], device=gpu)
    got = paged.attention(cache, batch, q, None if out is None else out[:, :heads])
    torch.cuda.synchronize()
    ref = world.attention(q.double().cpu().numpy())
    vmax = max([np.abs(world.values("v", np.flatnonzero(world.held))).max()] if world.held.any() else [1.0])
    tol = 4e-5 * vmax * size if kind == "f32" else (4e-5 * size + 2.0 ** -10) * vmax + UNIT[kind] * np.abs(ref)
    assert got.shape == ref.shape
    diff = np.abs(got.double().cpu().numpy() - ref)
    assert np.all(diff <= tol), (float(diff.max()), vmax)
    if strided:
        assert torch.all(out[:, heads:] == 7.0)
    again = paged.attention(cache, batch, q)
    assert torch.equal(again, got)  # the same bits whatever the order of the work
    return got


@pytest.mark.parametrize("kind", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("heads,kv_heads,dim", [(16, 8, 128), (4, 4, 64), (14, 2, 64), (3, 1, 128), (32, 1, 128)])
def test_attention_of_single_tokens(gpu, cuda_lib, kind, heads, kv_heads, dim):
    world = World([1, 1, 1, 1, 1, 0, 1], [1, 2, 63, 64, 301, 40, 65], 16, kv_heads, dim, seed=heads)
    check_attention(world, kind, heads, gpu)


@pytest.mark.parametrize("page", [1, 7, 16, 24, 64, 100, 256])
def test_attention_of_ragged_chunks_over_any_page_size(gpu, cuda_lib, page):
    world = World([5, 1, 64, 17, 33], [5, 130, 200, 77, 33], page, 2, 128, seed=page)
    check_attention(world, "f32", 4, gpu, seed=page)


@pytest.mark.parametrize("kind", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("query", [2, 3, 4, 5, 7, 8, 9, 15, 16, 31, 63, 64, 65, 127, 129, 200])
def test_attention_of_chunks(gpu, cuda_lib, kind, query):
    world = World([query, 1, query], [query, 90, query + 190], 16, 1, 128, seed=query)
    check_attention(world, kind, 2, gpu, seed=query)


@pytest.mark.parametrize("kind", ["f32", "bf16"])
@pytest.mark.parametrize("query,context", [(1, 4096), (6, 3000), (150, 2500), (1, 8192)])
def test_attention_over_long_contexts(gpu, cuda_lib, kind, query, context):
    world = World([query, 1], [context, context - 77], 64, 2, 64, seed=context)
    check_attention(world, kind, 4, gpu)


@pytest.mark.parametrize("kind,sequences,most", [("f32", 1000, 2), ("bf16", 600, 20), ("f32", 600, 20)])
def test_attention_of_more_sequences_than_a_block_has_threads(gpu, cuda_lib, kind, sequences, most):
    r = np.random.default_rng(sequences + most)
    query = r.integers(0, most + 1, sequences)
    world = World(query, query + r.integers(0, 100, sequences), 16, 1, 64, seed=sequences)
    check_attention(world, kind, 2, gpu, seed=most)


def test_attention_of_odd_head_shares(gpu, cuda_lib):
    for heads, kv_heads, dim in ((5, 5, 64), (9, 3, 128), (7, 1, 64), (40, 8, 128)):
        check_attention(World([3, 50, 1], [70, 50, 9], 16, kv_heads, dim, seed=heads), "f32", heads, gpu)


def test_attention_with_strides_and_large_scores(gpu, cuda_lib):
    world = World([1, 40, 9], [300, 301, 9], 16, 2, 128, seed=5)
    for kind in TYPES:
        check_attention(world, kind, 4, gpu, strided=True)
    check_attention(world, "f32", 4, gpu, size=8.0)  # near one-hot rows


def test_attention_rows_that_see_nothing_are_zero(gpu, cuda_lib):
    # A context shorter than its tokens: the first tokens lie before position 0. An empty context.
    world = World([4, 3, 70], [2, 0, 69], 16, 2, 64, seed=6)
    got = check_attention(world, "f32", 4, gpu)
    assert torch.all(got[:2] == 0) and torch.all(got[4:7] == 0) and torch.all(got[7] == 0)
    assert not torch.any(got[2:4] == 0)


def test_attention_skips_pages_outside_the_pool(gpu, cuda_lib):
    world = World([1, 20, 1], [100, 100, 3], 16, 2, 128, seed=7)
    world.table[0, 2], world.table[1, 0], world.table[1, 4] = -1, world.pages, 2 ** 30
    world.table[2, 0] = -5  # nothing left to see
    got = check_attention(world, "f32", 4, gpu)
    assert torch.all(got[21] == 0)


@pytest.mark.parametrize("kind", ["f32", "bf16"])
def test_attention_of_values_of_every_size(gpu, cuda_lib, kind):
    # Value scales from the smallest f16 to large ones: the weights must keep their bits.
    for query in (1, 40):
        for power in (-20, -9, 6, 14):
            world = World([query], [200], 16, 1, 128, seed=power + 100)
            live = world.scales["v"].astype(np.float32)
            world.scales["v"] = np.where(np.isnan(live), live, np.maximum(live * 2.0 ** power, 2.0 ** -24)).astype(np.float16)
            check_attention(world, kind, 2, gpu)


def test_attention_of_queries_of_every_size(gpu, cuda_lib):
    # f32 queries far outside the f16 range, against keys that bring the scores back.
    world = World([1, 30], [64, 90], 16, 1, 128, seed=8)
    live = world.scales["k"].astype(np.float32)
    world.scales["k"] = np.where(np.isnan(live), live, np.maximum(live * 2.0 ** -10, 2.0 ** -24)).astype(np.float16)
    cache, batch = world.device(gpu)
    q = torch.randn(31, 2, 128, generator=torch.Generator().manual_seed(3)).to(gpu) * 1024.0
    q[:, 1] *= 2.0 ** 10
    q[:, 0, 5] = 1e-30
    got = paged.attention(cache, batch, q).double().cpu().numpy()
    ref = world.attention(q.double().cpu().numpy())
    vmax = np.abs(world.values("v", np.flatnonzero(world.held))).max()
    assert np.abs(got[:, 0] - ref[:, 0]).max() <= 4e-5 * vmax
    # Head 1's scores reach thousands: their f32 spacing alone is 2^-12, times a weight's slope.
    assert np.abs(got[:, 1] - ref[:, 1]).max() <= 4e-5 * 1024 * vmax


def test_attention_nan_stays_in_its_row(gpu, cuda_lib):
    for query in (2, 40):
        world = World([query, query], [100, 100], 16, 1, 128, seed=9)
        cache, batch = world.device(gpu)
        q = torch.randn(2 * query, 2, 128, device=gpu)
        clean = paged.attention(cache, batch, q)
        q[1, 0, 3] = float("nan")
        q[query, 1, 0] = float("inf")
        got = paged.attention(cache, batch, q)
        assert torch.all(torch.isnan(got[1, 0])) and torch.all(torch.isnan(got[query, 1]))
        same = torch.ones(2 * query, 2, dtype=torch.bool, device=gpu)
        same[1, 0] = same[query, 1] = False
        assert torch.equal(got[same], clean[same])


def test_attention_on_another_stream(gpu, cuda_lib):
    world = World([1, 40], [500, 300], 16, 2, 128, seed=10)
    cache, batch = world.device(gpu)
    q = torch.randn(41, 4, 128, device=gpu)
    want = paged.attention(cache, batch, q)
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(3)]
    got = []
    for st in streams:
        with torch.cuda.stream(st):
            q2 = torch.zeros_like(q)
            q2.copy_(q)
            got.append([paged.attention(cache, batch, q2) for _ in range(4)])
    torch.cuda.synchronize()
    for outs in got:
        assert all(torch.equal(o, want) for o in outs)


@pytest.mark.parametrize("query", [1, 40])
def test_attention_in_a_graph(gpu, cuda_lib, query):
    world = World([query, query], [500, 300], 16, 2, 128, seed=12)
    cache, batch = world.device(gpu)
    q = torch.randn(2 * query, 4, 128, device=gpu)
    want = paged.attention(cache, batch, q)
    side = torch.cuda.Stream()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        got = paged.attention(cache, batch, q)
    with torch.cuda.stream(side):  # before the first replay: nothing that the capture made is used
        early = paged.attention(cache, batch, q)
    torch.cuda.synchronize()
    assert torch.equal(early, want)
    other = torch.cuda.Stream()
    for _ in range(3):
        got.zero_()
        torch.cuda.synchronize()
        with torch.cuda.stream(other):
            graph.replay()
        beside = paged.attention(cache, batch, q)
        torch.cuda.synchronize()
        assert torch.equal(got, want) and torch.equal(beside, want)


@pytest.mark.parametrize("query", [1, 40])
def test_attention_with_a_workspace_of_the_callers(gpu, cuda_lib, query):
    world = World([query, query], [500, 300], 16, 2, 128, seed=13)
    cache, batch = world.device(gpu)
    q = torch.randn(2 * query, 4, 128, device=gpu)
    want = paged.attention(cache, batch, q)
    work = paged.workspace(cache, batch, 4)
    work[rt.PAGED_WORKSPACE_HEAD:] = 255  # only the head has to be zero
    for _ in range(3):
        assert torch.equal(paged.attention(cache, batch, q, workspace=work), want)
    assert not work[:rt.PAGED_WORKSPACE_HEAD].any()
    paged.check_waits(work)
    paged.check_waits()
    work[0] = 3
    with pytest.raises(rt.QwcError) as e:
        paged.check_waits(work)
    assert e.value.name == "invalid_state"
    paged.check_waits(work)
    for bad, name in ((work[:-16], "limit_exceeded"), (work[1:], "invalid_argument"), (work.view(torch.int32), "invalid_argument"),
                      (work.cpu(), "invalid_argument"), (torch.zeros(2 * work.numel(), dtype=torch.uint8, device=gpu)[::2], "invalid_argument")):
        with pytest.raises(rt.QwcError) as e:
            paged.attention(cache, batch, q, workspace=bad)
        assert e.value.name == name


def test_lengths_that_change_on_the_device(gpu, cuda_lib):
    # The bounds stay, the lengths do not: one batch object serves many steps, and replays in a graph.
    world = World([1, 1, 1], [300, 200, 100], 16, 2, 128, seed=11)
    cache, batch = world.device(gpu)
    q = torch.randn(3, 4, 128, device=gpu)
    paged.attention(cache, batch, q)
    graph, out = torch.cuda.CUDAGraph(), torch.empty_like(q)
    with torch.cuda.graph(graph):
        paged.attention(cache, batch, q, out)
    for lens in ([300, 200, 100], [17, 1, 64], [0, 299, 5]):
        batch.context_lens.copy_(torch.tensor(lens, dtype=torch.int32))
        graph.replay()
        world.context = np.asarray(lens)
        full = World([1, 1, 1], [300, 200, 100], 16, 2, 128, seed=11)
        world.table, world.scales, world.codes = full.table, full.scales, full.codes
        lens_ok = np.minimum(lens, [300, 200, 100])
        if np.any(lens_ok != lens):
            batch.context_lens.copy_(torch.tensor(lens_ok, dtype=torch.int32))
            graph.replay()
            world.context = lens_ok
        torch.cuda.synchronize()
        ref = world.attention(q.double().cpu().numpy())
        assert np.abs(out.double().cpu().numpy() - ref).max() <= 4e-5 * 4


# ---- append and read ----


def identity_tables(n, dim, dev):
    return torch.ones(n, dim // 2, device=dev), torch.zeros(n, dim // 2, device=dev)


def angles(n, dim, dev):
    c, s = rt.rope_tables(1000000.0, dim, n)
    return (torch.from_numpy(a.reshape(n, dim // 2)).to(dev) for a in (c, s))


@pytest.mark.parametrize("kind", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("heads,kv_heads,dim,page", [(16, 8, 128, 64), (4, 4, 64, 16), (14, 2, 64, 7), (3, 1, 128, 1)])
def test_append_is_the_quantizer_bit_for_bit(gpu, cuda_lib, kind, heads, kv_heads, dim, page):
    world = World([1, 0, 9, 30], [20, 8, 9, 77], page, kv_heads, dim, seed=heads)
    cache, batch = world.device(gpu)
    g = torch.Generator().manual_seed(4)
    rows = torch.randn(world.tokens, (heads + 2 * kv_heads) * dim, generator=g)
    rows *= torch.tensor([1e-4, 0.03, 1.0, 77.0])[torch.arange(world.tokens) % 4][:, None]
    rows[3, heads * dim: heads * dim + 64] = 0.0  # a group of zeros
    rows[4, heads * dim: heads * dim + 64] = torch.arange(64) - 31.5  # halves land on ties
    rows = rows.to(TYPES[kind]).to(gpu)
    q, k, v = (t.unflatten(1, (-1, dim)) for t in rows.split([heads * dim, kv_heads * dim, kv_heads * dim], 1))
    before = {n: (cache.__dict__[n + "_scales"].clone(), cache.__dict__[n + "_codes"].clone()) for n in "kv"}
    q_out = paged.append(cache, batch, q, k, v, *identity_tables(100, dim, gpu))
    assert torch.equal(q_out, q)
    written = np.concatenate([world.rows(s, np.arange(c - n, c)) for s, (n, c) in enumerate(zip(world.query, world.context))])
    for n, x in (("k", k), ("v", v)):
        es, ec = quant.quantize(quant.Q8, x.float().cpu().numpy().reshape(world.tokens, -1))
        gs, gc = cache.__dict__[n + "_scales"].cpu().numpy(), cache.__dict__[n + "_codes"].cpu().numpy()
        assert np.array_equal(gs[written].view(np.uint16), es.view(np.uint16).reshape(len(written), -1))
        assert np.array_equal(gc[written], ec)
        others = np.setdiff1d(np.arange(world.pages * page), written)
        assert np.array_equal(gs[others].view(np.uint16), before[n][0].cpu().numpy()[others].view(np.uint16))
        assert np.array_equal(gc[others], before[n][1].cpu().numpy()[others])
    for out_type in TYPES.values():
        rk, rv = paged.read(cache, batch, out_type)
        for n, got in (("k", rk), ("v", rv)):
            s = torch.from_numpy(cache.__dict__[n + "_scales"].cpu().numpy()[written]).float().repeat_interleave(64, 1)
            c = torch.from_numpy(cache.__dict__[n + "_codes"].cpu().numpy()[written]).float() - 128
            assert torch.equal(got.cpu().flatten(1), (c * s).to(out_type))


@pytest.mark.parametrize("kind", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("heads,kv_heads,dim", [(16, 8, 128), (4, 2, 64)])
def test_append_norms_and_rotates(gpu, cuda_lib, kind, heads, kv_heads, dim):
    world = World([1, 40], [300, 41], 16, kv_heads, dim, seed=heads)
    cache, batch = world.device(gpu)
    g = torch.Generator().manual_seed(5)
    q, k, v = (torch.randn(world.tokens, n, dim, generator=g).to(TYPES[kind]).to(gpu) for n in (heads, kv_heads, kv_heads))
    qn, kn = (1 + 0.3 * torch.randn(dim, generator=g).to(gpu) for _ in range(2))
    cos, sin = angles(400, dim, gpu)
    pos = np.concatenate([np.arange(c - n, c) for n, c in zip(world.query, world.context)])

    def turned(x, w):
        x = x.double().cpu()
        x = x / (x.square().mean(-1, keepdim=True) + 1e-6).sqrt() * w.double().cpu()
        c, s = cos.double().cpu()[pos][:, None], sin.double().cpu()[pos][:, None]
        lo, hi = x.chunk(2, -1)
        return torch.cat([lo * c - hi * s, hi * c + lo * s], -1)

    q_in = q.clone()
    q_out = paged.append(cache, batch, q, k, v, cos, sin, q_norm=qn, k_norm=kn, eps=1e-6)
    assert torch.equal(q, q_in)
    want = turned(q, qn)
    assert torch.all((q_out.double().cpu() - want).abs() <= UNIT[kind] * want.abs() + 2e-6)
    got, _ = paged.read(cache, batch, torch.float32)
    want = turned(k, kn).flatten(1).unflatten(1, (-1, 64))
    amax = want.abs().amax(-1, keepdim=True)
    step = amax / 128
    # The top code is 127: the largest value of a group may lie one step out; the stored scale rounds by 2^-11.
    err = (got.double().cpu().flatten(1).unflatten(1, (-1, 64)) - want).abs()
    top = want >= amax * (126.4 / 128)
    assert torch.all(err <= torch.where(top, 1.1, 0.501 + 0.0) * step + 2.0 ** -11 * amax)
    # In place, and with a view of wider rows as the output.
    inplace = paged.append(cache, batch, q, k, v, cos, sin, q_norm=qn, k_norm=kn, eps=1e-6, q_out=q)
    assert inplace is q and torch.equal(q, q_out)


def test_append_and_read_of_positions_that_are_not_cached(gpu, cuda_lib):
    world = World([4, 3], [2, 3], 16, 2, 64, seed=12)  # two tokens before position 0
    world.table[1, 0] = world.pages  # a page that the pool lacks
    cache, batch = world.device(gpu)
    before = [t.clone() for t in (cache.k_scales, cache.k_codes, cache.v_scales, cache.v_codes)]
    q, k, v = (torch.randn(7, n, 64, device=gpu) for n in (4, 2, 2))
    q_out = paged.append(cache, batch, q, k, v, *identity_tables(2, 64, gpu))
    assert torch.all(q_out[:2] == 0) and torch.equal(q_out[2:4], q[2:4]) and torch.all(q_out[4:] == 0)
    changed = world.rows(0, np.arange(2))
    for old, new in zip(before, (cache.k_scales, cache.k_codes, cache.v_scales, cache.v_codes)):
        keep = np.setdiff1d(np.arange(old.shape[0]), changed)
        as_bytes = lambda t: t[keep].contiguous().view(torch.uint8)  # noqa: E731
        assert torch.equal(as_bytes(old), as_bytes(new))
    rk, rv = paged.read(cache, batch)
    assert torch.all(rk[:2] == 0) and torch.all(rv[4:] == 0) and not torch.any(torch.isnan(rk[2:4]))
    # A rotation table that ends too early: position 1 has no row in it.
    q_out = paged.append(cache, batch, q, k, v, *identity_tables(1, 64, gpu))
    assert torch.equal(q_out[2], q[2]) and torch.all(q_out[3] == 0)


def test_nothing_to_do(gpu, cuda_lib):
    world = World([0, 0], [5, 0], 16, 2, 64)
    cache, batch = world.device(gpu)
    q, kv = torch.zeros(0, 4, 64, device=gpu), torch.zeros(0, 2, 64, device=gpu)
    assert paged.attention(cache, batch, torch.zeros(0, 4, 64, device=gpu)).shape == (0, 4, 64)
    assert paged.append(cache, batch, q, kv, kv, *identity_tables(8, 64, gpu)).shape == (0, 4, 64)
    assert paged.read(cache, batch)[0].shape == (0, 2, 64)


def test_rows_past_32_bit_offsets(gpu, cuda_lib):
    # 4.5 GB of codes in each plane: the last pages' rows start past 2^32.
    page, kv_heads, dim = 256, 8, 128
    pages = (1 << 32) // (page * 1024) + 200
    cache = paged.PagedCache.zeros(pages, page, kv_heads, dim, gpu)
    put = lambda a: torch.tensor(a, dtype=torch.int32, device=gpu)  # noqa: E731
    for query in (5, 100):
        context = 600
        batch = paged.PagedBatch(put([0, query]), put([context]), put([[pages - 1, 3, pages - 7]]), tokens=query,
                                 max_query=query, max_context=context)
        small = paged.PagedCache.zeros(3, page, kv_heads, dim, gpu)
        near = paged.PagedBatch(put([0, query]), put([context]), put([[2, 0, 1]]), tokens=query, max_query=query, max_context=context)
        full = [paged.PagedBatch(put([0, context]), put([context]), b.page_table, tokens=context, max_query=context,
                                 max_context=context) for b in (batch, near)]
        q, k, v = (torch.randn(context, n, dim, device=gpu) for n in (16, kv_heads, kv_heads))
        tables = identity_tables(context, dim, gpu)
        for c, b in ((cache, full[0]), (small, full[1])):
            paged.append(c, b, q, k, v, *tables)
        assert all(torch.equal(x, y) for x, y in zip(paged.read(cache, full[0]), paged.read(small, full[1])))
        assert torch.equal(paged.attention(cache, batch, q[:query].contiguous()), paged.attention(small, near, q[:query].contiguous()))
    del cache
    torch.cuda.empty_cache()


def test_refusals(gpu, cuda_lib):
    world = World([1, 3], [20, 9], 16, 2, 64)
    cache, batch = world.device(gpu)
    q = torch.zeros(4, 4, 64, device=gpu)
    kv = torch.zeros(4, 2, 64, device=gpu)
    tables = identity_tables(32, 64, gpu)

    def refused(name, f, *a, **k):
        with pytest.raises(rt.QwcError) as e:
            f(*a, **k)
        assert e.value.name == name

    refused("unsupported", paged.attention, cache, batch, q.double())
    refused("shape_mismatch", paged.attention, cache, batch, q[:3])
    refused("shape_mismatch", paged.attention, cache, batch, q[:, :3].contiguous())  # 3 heads over 2
    refused("invalid_argument", paged.attention, cache, batch, q.transpose(0, 1).contiguous().transpose(0, 1))
    refused("invalid_argument", paged.attention, cache, batch, q, q.half())
    refused("invalid_argument", paged.attention, cache, batch, torch.zeros(4 * 256 + 1, device=gpu)[1:].view(4, 4, 64))
    refused("invalid_argument", paged.append, cache, batch, q, kv.half(), kv, *tables)
    refused("shape_mismatch", paged.append, cache, batch, q, kv[:, :1], kv, *tables)
    refused("shape_mismatch", paged.append, cache, batch, q, kv, kv, *tables, q_norm=torch.ones(32, device=gpu))
    refused("invalid_argument", paged.append, cache, batch, q, kv, kv, *tables, k_norm=torch.ones(64, device=gpu).half())
    refused("unsupported", paged.read, cache, batch, torch.float64)
    refused("shape_mismatch", paged.PagedBatch, batch.query_starts, batch.context_lens, batch.page_table[:1], tokens=4,
            max_query=3, max_context=20)
    refused("invalid_argument", paged.PagedBatch, batch.query_starts.long(), batch.context_lens, batch.page_table,
            tokens=4, max_query=3, max_context=20)
    refused("shape_mismatch", paged.PagedCache, cache.k_scales, cache.k_codes, cache.v_scales, cache.v_codes,
            page_size=7, kv_heads=2, head_dim=64)
    wrong = paged.PagedCache(cache.k_scales, cache.k_codes, cache.v_scales, cache.v_codes, page_size=16, kv_heads=4, head_dim=32)
    refused("unsupported", paged.attention, wrong, batch, torch.zeros(4, 4, 32, device=gpu))
    long = paged.PagedBatch(batch.query_starts, batch.context_lens, batch.page_table, tokens=4, max_query=3, max_context=16 * 50)
    refused("shape_mismatch", paged.attention, cache, long, q)


def test_append_of_heads_whose_squares_overflow(gpu, cuda_lib):
    # 128 squares of 1e19 and more pass f32: the norm's factor is 0 then, and so are the head's values, as in f32
    # arithmetic throughout (x * (1 / sqrt(inf)) = 0). The other heads of the token keep theirs.
    world = World([3], [3], 16, 2, 128, seed=14)
    cache, batch = world.device(gpu)
    g = torch.Generator().manual_seed(9)
    q, k, v = (torch.randn(3, n, 128, generator=g).to(gpu) for n in (4, 2, 2))
    norms = dict(q_norm=torch.ones(128, device=gpu), k_norm=torch.ones(128, device=gpu))
    tables = identity_tables(3, 128, gpu)
    clean = paged.append(cache, batch, q, k, v, *tables, **norms)
    clean_k = paged.read(cache, batch)[0]
    q[1, 2] *= 1e20
    k[2, 0, 5] = -3e19
    got = paged.append(cache, batch, q, k, v, *tables, **norms)
    got_k = paged.read(cache, batch)[0]
    assert torch.all(got[1, 2] == 0) and torch.all(got_k[2, 0] == 0)
    clean[1, 2], clean_k[2, 0] = 0, 0
    assert torch.equal(got, clean) and torch.equal(got_k, clean_k)


def test_append_with_rotation_tables_of_no_rows(gpu, cuda_lib):
    # rope_rows of 0 in the C call: every token lies past the tables, which are not read (the rows here are NaN).
    world = World([2, 1], [20, 5], 16, 2, 64, seed=15)
    cache, batch = world.device(gpu)
    before = [t.clone() for t in (cache.k_scales, cache.k_codes, cache.v_scales, cache.v_codes)]
    q, k, v = (torch.randn(3, n, 64, device=gpu) for n in (4, 2, 2))
    out, nan = torch.full_like(q, 7.0), torch.full((1, 32), float("nan"), device=gpu)
    st = rt.lib().qwc_op_paged_append(
        cache._ref, batch._ref, rt.FORMAT_F32, q.data_ptr(), 256, k.data_ptr(), 128, v.data_ptr(), 128, 4, None, None, 1e-6,
        nan.data_ptr(), nan.data_ptr(), 0, out.data_ptr(), 256, paged.current_stream(gpu))
    torch.cuda.synchronize()
    assert st == 0 and torch.all(out == 0)
    for old, new in zip(before, (cache.k_scales, cache.k_codes, cache.v_scales, cache.v_codes)):
        assert torch.equal(old.view(torch.uint8), new.view(torch.uint8))


@pytest.mark.parametrize("query", [1, 30])
def test_tables_that_are_views(gpu, cuda_lib, query):
    # Columns of a wider table, and one row for all sequences (a prefix that they share).
    world = World([query, query, 2], [100, 70, 90], 16, 2, 128, seed=16)
    world.table[1:] = world.table[0]
    cache, batch = world.device(gpu)
    q = torch.randn(world.tokens, 4, 128, device=gpu)
    want, want_k = paged.attention(cache, batch, q), paged.read(cache, batch)[0]
    wide = torch.full((3, 40), 2 ** 30, dtype=torch.int32, device=gpu)
    wide[:, 11:11 + world.table.shape[1]] = batch.page_table
    for table in (wide[:, 11:11 + world.table.shape[1]], batch.page_table[:1].expand(3, -1)):
        b = paged.PagedBatch(batch.query_starts, batch.context_lens, table, tokens=world.tokens, max_query=max(query, 2), max_context=100)
        assert torch.equal(paged.attention(cache, b, q), want) and torch.equal(paged.read(cache, b)[0], want_k)


def test_threads_on_one_stream_with_growing_workspaces(gpu, cuda_lib):
    worlds = [World([query] * n, [300] * n, 16, 2, 128, seed=20 + n) for query, n in ((1, 1), (40, 1), (1, 40), (40, 6))]
    made = [(*w.device(gpu), torch.randn(w.tokens, 4, 128, device=gpu)) for w in worlds]
    want = [paged.attention(*m) for m in made]
    torch.cuda.synchronize()
    key = (gpu.index, paged.current_stream(gpu))
    wrong, start = [], threading.Barrier(4)

    def work(i):
        start.wait()
        for n in range(60):
            if i == 0:
                paged._workspaces.pop(key, None)  # the next calls grow it again, from nothing
            j = (n + i) % len(made)
            if not torch.equal(paged.attention(*made[j]), want[j]):
                wrong.append((i, n))

    threads = [threading.Thread(target=work, args=(i,)) for i in range(4)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not wrong
    paged.check_waits()


def close_where_finite(got, ref, tol):
    got = got.double().cpu().numpy()
    numbers = np.isfinite(ref)
    assert np.array_equal(np.isfinite(got), numbers), (np.argwhere(np.isfinite(got) != numbers)[:5], numbers.mean())
    assert np.all(np.abs(got - ref)[numbers] <= tol[numbers]), float(np.abs(got - ref)[numbers].max())


@pytest.mark.parametrize("kind", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("query", [1, 2, 4, 8, 40, 300])
@pytest.mark.parametrize("bad", [np.inf, np.nan])
def test_attention_of_values_that_are_no_numbers(gpu, cuda_lib, kind, query, bad):
    # Value scales of two positions: one among the new tokens, which the earlier of them do not see, and one in the middle of
    # another sequence's context. The heads' rows that see one are no numbers, and nothing else is.
    world = World([query, query], [query + 70, query + 70], 16, 2, 128, seed=17 + query)
    vmax = np.abs(world.values("v", np.flatnonzero(world.held))).max()
    for s, p, group in ((0, 70 + query // 2, 1), (1, 33, 2)):
        world.scales["v"][world.rows(s, np.array([p])), group] = bad
    cache, batch = world.device(gpu)
    q = torch.randn(world.tokens, 4, 128, generator=torch.Generator().manual_seed(query)).to(TYPES[kind]).to(gpu)
    with np.errstate(invalid="ignore"):
        ref = world.attention(q.double().cpu().numpy())
    assert not np.isfinite(ref[:, :2, 64:][query // 2:query]).any() and np.isfinite(ref[:query // 2]).all() and np.isfinite(ref[:query, 2:]).all()
    ref[~np.isfinite(ref).all(-1)] = np.nan
    tol = np.full(ref.shape, 4e-5 * vmax) if kind == "f32" else (4e-5 + 2.0 ** -10) * vmax + UNIT[kind] * np.abs(ref)
    close_where_finite(paged.attention(cache, batch, q), ref, tol)


@pytest.mark.parametrize("kind", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("query", [2, 8, 40, 300])
@pytest.mark.parametrize("bad", [np.inf, np.nan])
def test_attention_beside_keys_that_are_no_numbers(gpu, cuda_lib, kind, query, bad):
    # A key scale among the new tokens: the tokens before it keep their results.
    world = World([query], [query + 70], 16, 2, 128, seed=18 + query)
    vmax = np.abs(world.values("v", np.flatnonzero(world.held))).max()
    p = 70 + query // 2
    world.scales["k"][world.rows(0, np.array([p])), 1] = bad
    cache, batch = world.device(gpu)
    q = torch.randn(world.tokens, 4, 128, generator=torch.Generator().manual_seed(query)).to(TYPES[kind]).to(gpu)
    with np.errstate(invalid="ignore"):
        ref = world.attention(q.double().cpu().numpy())
    got = paged.attention(cache, batch, q).double().cpu().numpy()
    tol = np.full(ref.shape, 4e-5 * vmax) if kind == "f32" else (4e-5 + 2.0 ** -10) * vmax + UNIT[kind] * np.abs(ref)
    free = np.zeros(ref.shape, bool)
    free[:query // 2] = free[:, 2:] = True  # does not see it, or is another kv head's
    assert np.all(np.abs(got - ref)[free] <= tol[free]), float(np.abs(got - ref)[free].max())


@pytest.mark.parametrize("kind", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("query", [2, 8, 40, 300])
@pytest.mark.parametrize("plane", ["k", "v"])
def test_attention_beside_a_position_of_another_size(gpu, cuda_lib, kind, query, plane):
    # One position's keys or values are a thousand times the others', and a token before it does not see it: what it may cost
    # them. A weight times a scale is off by 2^-31 of the largest value scale (times 128 codes); bf16 rows in tiles have keys
    # and values off by 2^-17 of the largest scale (a score by that times the sum of its |q| / sqrt(d), a weight by e to it).
    world = World([query], [query + 70], 16, 2, 128, seed=19 + query)
    p, large = 70 + query // 2, 32.0
    seen = np.abs(world.values("v", world.rows(0, np.arange(p)))).max()
    world.scales[plane][world.rows(0, np.array([p]))] = large
    cache, batch = world.device(gpu)
    q = torch.randn(world.tokens, 4, 128, generator=torch.Generator().manual_seed(query)).to(TYPES[kind]).to(gpu)
    ref = world.attention(q.double().cpu().numpy())[:query // 2]
    got = paged.attention(cache, batch, q).double().cpu().numpy()[:query // 2]
    tiles = kind == "bf16" and query * 2 > 16
    if plane == "v":
        rest = 2.0 ** -17 * large if tiles else 2.0 ** -24 * large
    else:
        rest = 2 * 2.0 ** -17 * large * float(q.abs().sum(-1).max()) / 128 ** 0.5 * seen if tiles else 0.0
    tol = rest + (4e-5 * seen if kind == "f32" else (4e-5 + 2.0 ** -10) * seen + UNIT[kind] * np.abs(ref))
    assert np.all(np.abs(got - ref) <= tol), (float(np.abs(got - ref).max()), seen)
