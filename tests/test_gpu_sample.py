"""qwc_op_sample against its definition in 64 bits.

The operator's weights are f32 exponentials (relative error below 1e-6 for the arguments that matter)
and its sums are exact; a token may differ from the 64-bit answer only where the given number, or top_p, lies
within 1e-5 of a boundary of the cumulative distribution. The reference below returns every token
that such a nudge can give. Log-probabilities: 1e-5 absolute, plus 1e-6 of their size.
"""

import numpy as np
import pytest
import torch

from qwenscriber_b200 import runtime as rt
from qwenscriber_b200 import sampling

pytestmark = pytest.mark.gpu

TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}


def allowed(x, heat, k, p, least, u):
    """(tokens that the definition gives for numbers within 1e-5 of these, log-probabilities of all tokens)."""
    x = np.where(np.isnan(x), -np.inf, x.astype(np.float64))
    best = x.max()
    if best == -np.inf:
        return {0}, np.full(len(x), -np.inf)
    greedy = not heat > 0
    with np.errstate(invalid="ignore"):
        z = np.where(x == best, 0.0, np.where(x == -np.inf, -np.inf, (x - best) / (1.0 if greedy else heat)))
    w = np.exp(z)
    logp = z - np.log(w.sum())
    if greedy:
        return {int(np.argmax(x))}, logp
    order = np.lexsort((np.arange(len(x)), -x))
    if 0 < k < len(x):
        order = order[:k]
    found = set()
    wo = w[order]
    before = np.concatenate([[0.0], np.cumsum(wo)[:-1]])
    for p2 in {p, max(p - 1e-5, 0.0), min(p + 1e-5, 1.0)} if p < 1 else {1.0}:
        for least2 in {least, least * (1 - 1e-5), least * (1 + 1e-5)}:
            keep = (before < p2 * wo.sum()) | (p2 >= 1)
            keep &= wo >= min(least2, 1.0)
            keep[0] = True
            chosen = np.sort(order[keep])
            mass = np.cumsum(w[chosen])
            for u2 in (u - 1e-5, u, u + 1e-5):
                goal = min(max(u2, 0.0), 1.0) * mass[-1]
                found.add(int(chosen[min(np.searchsorted(mass, goal, side="right"), len(chosen) - 1)]))
    return found, logp


def check(x, kind, heat, k, p, least, u, gpu, given=("temperature", "top_k", "top_p", "min_p")):
    x = torch.as_tensor(x).to(TYPES[kind])
    rows = x.shape[0]
    cols = {"temperature": (heat, np.float32), "top_k": (k, np.int32), "top_p": (p, np.float32), "min_p": (least, np.float32)}
    host = {n: np.broadcast_to(np.asarray(v, t), (rows,)).copy() for n, (v, t) in cols.items()}
    u = np.broadcast_to(np.asarray(u, np.float32), (rows,)).copy()
    token, logprob = sampling.sample(x.to(gpu), torch.from_numpy(u).to(gpu), **{n: torch.from_numpy(host[n]).to(gpu) for n in given})
    token, logprob, xs = token.cpu().numpy(), logprob.cpu().numpy(), x.float().numpy()
    for r in range(rows):
        tokens, logp = allowed(xs[r], *(float(host[n][r]) if n != "top_k" else int(host[n][r]) for n in cols), float(u[r]))
        assert int(token[r]) in tokens, (r, int(token[r]), tokens)
        want = logp[token[r]]
        assert logprob[r] == want or abs(logprob[r] - want) <= 1e-5 + 1e-6 * abs(want), (r, logprob[r], want)
    return token


@pytest.mark.parametrize("kind", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("vocab", [1, 2, 31, 1000, 4097, 32003, 151936, 400001])
def test_settings_of_every_kind(gpu, cuda_lib, kind, vocab):
    r = np.random.default_rng(vocab)
    rows = 40 if vocab < 100000 else 12
    x = r.standard_normal((rows, vocab)) * 2.5
    x[np.arange(rows), r.integers(0, vocab, rows)] += 9
    check(x, kind, r.choice([0.0, 0.2, 0.7, 1.0, 1.9], rows), r.choice([0, 1, 2, 40, 900, vocab, vocab + 5], rows),
          r.choice([0.0, 1e-3, 0.3, 0.9, 0.99, 1.0, 2.0], rows), r.choice([0.0, 0.0, 0.02, 0.3, 1.0, 3.0], rows), r.random(rows), gpu)


@pytest.mark.parametrize("missing", ["temperature", "top_k", "top_p", "min_p"])
def test_settings_left_out(gpu, cuda_lib, missing):
    r = np.random.default_rng(1)
    off = {"temperature": 1.0, "top_k": 0, "top_p": 1.0, "min_p": 0.0}
    on = {"temperature": 0.8, "top_k": 30, "top_p": 0.9, "min_p": 0.01}
    v = {n: off[n] if n == missing else on[n] for n in on}
    check(r.standard_normal((16, 5000)) * 3, "f32", v["temperature"], v["top_k"], v["top_p"], v["min_p"], r.random(16), gpu,
          given=tuple(n for n in on if n != missing))


def test_flat_rows_keep_the_lowest_indices(gpu, cuda_lib):
    # Every logit ties: the cuts keep the first tokens, and u walks them in order.
    n = 3000
    x = np.full((64, n), 1.25)
    u = (np.arange(64) + 0.5) / 64
    assert np.array_equal(check(x, "f32", 1.0, 64, 1.0, 0.0, u, gpu), np.arange(64))
    assert np.array_equal(check(x, "bf16", 1.0, 0, 63.5 / n, 0.0, u, gpu), np.arange(64))
    assert np.array_equal(check(x, "f32", 1.0, 0, 1.0, 0.0, u, gpu), (u * n).astype(int))
    check(x, "f32", 0.0, 0, 1.0, 0.0, u, gpu)


@pytest.mark.parametrize("kind", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("vocab", [2500, 32003, 151936, 400001])
@pytest.mark.parametrize("p", [0.05, 0.5, 0.9, 0.999, 0.9999999])
def test_large_nuclei(gpu, cuda_lib, kind, vocab, p):
    # Flat distributions: the kept set is a good part of the row, in f16 and bf16 with many ties at its end.
    r = np.random.default_rng(vocab + int(1000 * p))
    x = r.standard_normal((6, vocab)) * np.array([0.05, 0.5, 1.0, 1.0, 2.0, 3.0])[:, None]
    check(x, kind, [1.0, 1.0, 0.8, 3.0, 1.0, 2.0], 0, p, [0.0, 0.0, 0.0, 0.01, 0.0, 0.001], r.random(6), gpu)


@pytest.mark.parametrize("few", [1, 700, 1500])
def test_two_values(gpu, cuda_lib, few):
    # Two heaps of ties, the cut in either; numbers at both ends.
    n = 20000
    x = np.full((8, n), -1.0)
    at = np.random.default_rng(few).permutation(n)[:few]
    x[:, at] = 2.0
    mass = few * np.exp(3.0)
    ps = np.array([0.5 * mass, 0.999 * mass, mass + 0.5 * (n - few), mass + n - few - 1.5]) / (mass + n - few)
    check(x, "f32", 1.0, 0, np.repeat(ps, 2), 0.0, np.tile([0.0, 0.99999], 4), gpu)


def test_temperatures_without_bounds(gpu, cuda_lib):
    x = np.random.default_rng(4).standard_normal((4, 3000))
    x[:, ::3] = -np.inf
    token = check(x, "f32", [1e38, 3e38, np.inf, np.inf], 0, [1.0, 0.5, 1.0, 0.5], 0.0, [0.3, 0.6, 0.9, 0.999], gpu)
    assert np.all(token % 3 != 0)


def test_zeros_of_both_signs_tie(gpu, cuda_lib):
    x = np.full((2, 100), -50.0)
    x[:, 7], x[:, 3], x[:, 90] = 0.0, -0.0, 0.0
    assert list(check(x, "f32", 1.0, 1, 1.0, 0.0, 0.99, gpu)) == [3, 3]
    assert list(check(x, "f32", 0.0, 0, 1.0, 0.0, 0.99, gpu)) == [3, 3]
    assert list(check(x, "f32", 1.0, 2, 1.0, 0.0, [0.2, 0.8], gpu)) == [3, 7]


def test_masked_rows(gpu, cuda_lib):
    x = np.random.default_rng(2).standard_normal((9, 700))
    x[0] = -np.inf
    x[1] = np.nan
    x[2, ::2] = -np.inf
    x[3, :] = -np.inf
    x[3, 451] = -3.0
    x[4, 0] = np.nan
    x[5, [10, 20, 30]] = np.inf
    x[6] = np.finfo(np.float32).min
    x[7, :] = np.finfo(np.float32).min
    x[7, 699] = 5.0
    x[8, 1:] = -np.inf
    for kind in ("f32", "bf16"):
        for k, p in ((0, 1.0), (5, 1.0), (0, 0.9), (5, 0.5), (1, 0.0)):
            for u in (0.0, 0.4, 0.99999994):
                token = check(x, kind, 0.8, k, p, 0.0, u, gpu)
                assert token[0] == token[1] == 0 and token[3] == 451 and token[7] == 699 and token[8] == 0
                assert token[2] % 2 == 1 and token[4] != 0 and token[5] in (10, 20, 30)
    assert list(check(x, "f32", 0.0, 0, 1.0, 0.0, 0.5, gpu))[5] == 10
    assert list(check(x, "f32", np.nan, 0, 1.0, 0.0, 0.5, gpu))[5] == 10  # no temperature: the largest


def test_numbers_at_the_ends_and_outside(gpu, cuda_lib):
    x = np.array([[0.0, 1.0, 2.0, -np.inf]] * 6)
    u = np.array([0.0, 1.0, 0.99999994, -1.0, 2.0, np.nan], np.float32)
    token, _ = sampling.sample(torch.tensor(x, dtype=torch.float32, device=gpu), torch.from_numpy(u).to(gpu))
    assert token.tolist()[:5] == [0, 2, 2, 0, 2] and 0 <= token[5] < 3


def test_rows_of_a_wider_tensor(gpu, cuda_lib):
    r = np.random.default_rng(3)
    for kind in ("f32", "bf16"):
        wide = torch.from_numpy(r.standard_normal((8, 1111))).to(TYPES[kind]).to(gpu)
        u = torch.from_numpy(r.random(8).astype(np.float32)).to(gpu)
        for a, b in ((0, 1000), (1, 1000), (3, 1110), (5, 6)):
            got = sampling.sample(wide[:, a:b], u, top_p=torch.full((8,), 0.9, device=gpu))
            want = sampling.sample(wide[:, a:b].contiguous(), u, top_p=torch.full((8,), 0.9, device=gpu))
            assert all(torch.equal(x, y) for x, y in zip(got, want))


def test_frequencies(gpu, cuda_lib):
    # An even grid of numbers gives each token its share, to one grid step for each boundary.
    x = torch.randn(1, 50, generator=torch.Generator().manual_seed(6))
    n = 4096
    u = (torch.arange(n) + 0.5) / n
    token, _ = sampling.sample(x.expand(n, 50).contiguous().to(gpu), u.to(gpu), top_k=torch.full((n,), 20, dtype=torch.int32, device=gpu))
    share = torch.bincount(token.cpu().long(), minlength=50).double() / n
    p = x[0].double().exp()
    p[x[0].argsort(descending=True)[20:]] = 0
    assert torch.all((share - p / p.sum()).abs() <= 2.0 / n)


def test_refusals(gpu, cuda_lib):
    x, u = torch.zeros(2, 10, device=gpu), torch.zeros(2, device=gpu)

    def refused(name, *a, **k):
        with pytest.raises(rt.QwcError) as e:
            sampling.sample(*a, **k)
        assert e.value.name == name

    refused("unsupported", x.double(), u)
    refused("invalid_argument", x[0], u)
    refused("invalid_argument", x.t().contiguous().t(), u)
    refused("shape_mismatch", x, u[:1])
    refused("invalid_argument", x, u.half())
    refused("invalid_argument", x, u, top_k=torch.zeros(2, device=gpu))
    refused("invalid_argument", x[:, :0], u)
    refused("limit_exceeded", torch.zeros(1, rt.SAMPLE_MAX_VOCAB + 1, device=gpu), u[:1])


def check_counts_and_masses(x, kind, heat, k, p, least, gpu):
    """One row of logits with several numbers, so that most of the kept set is walked."""
    u = (np.arange(12) + 0.5) / 12
    check(np.broadcast_to(x, (12, len(x))).copy(), kind, heat, k, p, least, u, gpu)


def test_a_count_above_a_thousand_and_a_mass(gpu, cuda_lib):
    # top_k's cut lies in a bin of few tokens or many, top_p's likewise: the two searches follow one another.
    r = np.random.default_rng(21)
    check_counts_and_masses(r.uniform(0, 0.055, 2100), "f32", 1.0, 2000, 0.5, 0.0, gpu)
    check_counts_and_masses(r.standard_normal(5000), "f32", 20.0, 4900, 0.6, 0.0, gpu)
    check_counts_and_masses(2.2 * r.standard_normal(151936), "f32", 10.0, 151000, 0.3, 0.0, gpu)
    x = np.concatenate([r.uniform(0.032, 0.060, 1200), r.uniform(0, 0.028, 900)])
    check_counts_and_masses(r.permutation(x), "f32", 1.0, 1900, 0.45, 0.0, gpu)
    x = np.concatenate([[1.0], np.full(2000, 0.975), r.uniform(0.3685, 0.3965, 900), np.full(4000, -9.0)])
    check_counts_and_masses(r.permutation(x), "f32", 1.0, 2500, 0.6, 0.0, gpu)


@pytest.mark.parametrize("kind", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("at_mass", [300, 3000])
@pytest.mark.parametrize("at_count", [300, 3000])
@pytest.mark.parametrize("least", [0.0, 0.2])
def test_ties_at_both_cuts(gpu, cuda_lib, kind, at_mass, at_count, least):
    # Heaps of ties, small and large, the mass's cut inside the upper one and the count's inside the lower one.
    r = np.random.default_rng(at_mass + 7 * at_count)
    x = np.concatenate([2.0 + np.arange(1200) / 1200, np.full(at_mass, 1.5), 1.0 + np.arange(600) / 2400, np.full(at_count, 0.5),
                        r.uniform(-4, -3, 5000)])
    x = torch.as_tensor(x).to(TYPES[kind]).double().numpy()
    k = 1200 + at_mass + 600 + at_count // 2
    w = np.exp(x)
    p = (w[:1200].sum() + w[1200:1200 + at_mass].sum() / 2) / w[:k].sum()
    check_counts_and_masses(r.permutation(x), kind, 1.0, k, p, least, gpu)


@pytest.mark.parametrize("kind", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("vocab", [1100, 2100, 32003, 151936, 400001])
def test_large_counts_with_masses(gpu, cuda_lib, kind, vocab):
    r = np.random.default_rng(vocab)
    rows = 16
    x = r.standard_normal((rows, vocab)) * r.choice([0.02, 0.3, 1.0, 2.2], rows)[:, None]
    k = np.exp(r.uniform(np.log(1025), np.log(vocab - 1), rows)).astype(int)
    check(x, kind, r.choice([0.7, 1.0, 5.0, 20.0], rows), k, r.choice([0.05, 0.3, 0.6, 0.9, 0.999, 1.0], rows),
          r.choice([0.0, 0.0, 0.001, 0.5], rows), r.random(rows), gpu)


@pytest.mark.parametrize("gap", [9.0, 14.0, 18.0, 20.0])
@pytest.mark.parametrize("heat", [0.0, 0.7, 1.0])
def test_log_probabilities_near_zero(gpu, cuda_lib, gap, heat):
    # A token that is all but certain: its log-probability is -log1p of the others' weight. Each weight is off by the
    # exponential's 2^-22 and by three roundings of its exponent (below 30: 30 * 3 * 2^-24), and by 2^-43 as an integer.
    n = 40
    r = np.random.default_rng(int(gap))
    x = np.full((6, n), -np.inf)
    x[:, 3] = 11.0
    x[:, 7:7 + 6] = 11.0 - gap * (heat or 1.0) - np.arange(6) / 5 - r.random((6, 1))
    x = torch.as_tensor(x).float()
    temperature = torch.full((6,), heat, device=gpu)
    token, logprob = sampling.sample(x.to(gpu), torch.full((6,), 0.5, device=gpu), temperature=temperature)
    assert torch.all(token == 3)
    z = (x.double() - x.double()[:, 3:4]) / (float(temperature[0]) or 1.0)
    z[:, 3] = -np.inf
    tail = z.exp().sum(-1)
    want = -torch.log1p(tail)
    bound = (2.0 ** -22 + 30 * 3 * 2.0 ** -24 + 2.0 ** -22) * want.abs() + 6 * 2.0 ** -43
    assert torch.all((logprob.double().cpu() - want).abs() <= bound), (logprob, want)
