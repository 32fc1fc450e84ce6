"""The filtered sampler against its definition, written out row by row in 64 bits.

Tokens have to be equal.  The kernel's weights are exact to about 2^-45 of the largest, and the reference's sums to
about 1e-13 of theirs, so the two can only differ where a border (top-p's limit, the draw) lies within that of a partial
sum: for the numbers of rows and entries below, at odds of under one in a million for the whole file.  Probabilities are
one rounding to fp32 (2^-24 relative) of a quotient that is exact to V * 2^-46 of the sum at worst: V <= 2^18 gives
2^-28, so 2^-23 in all."""
import math

import numpy as np
import pytest

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def eng(qm):
    e = qm.TalkerAttention(layers=1, num_pages=1, max_positions=8)
    yield e
    e.close()


def want(z, u, heat=1.0, k=0, p=1.0, low=0.0):
    """(token, probability) of one row of float64 scores."""
    z = np.where(np.isnan(z), -np.inf, z)
    if not (z > -np.inf).any():
        return -1, 0.0
    order = np.lexsort((np.arange(len(z)), -z))
    if not heat > 0:
        return int(order[0]), 1.0
    with np.errstate(invalid="ignore", over="ignore"):
        w = np.where(z == z.max(), 1.0, np.exp((z - z.max()) / heat))
    w = np.where(np.isnan(w), 0.0, w)
    if k > 0:
        order = order[:k]
    if p < 1:
        ahead = np.concatenate([[0.0], np.cumsum(w[order])])
        order = order[:max(1, int((ahead[:-1] < p * ahead[-1]).sum()))]
    if low > 0:
        order = order[(w[order] >= low) | (z[order] == z.max())]
    kept = np.sort(order)
    c = np.cumsum(w[kept])
    at = min(int(np.searchsorted(c, min(max(u, 0.0), 1.0) * c[-1], side="right")), int(np.nonzero(w[kept])[0][-1]))
    return int(kept[at]), float(w[kept[at]] / c[-1])


def check(eng, z, u, heat=None, k=None, p=None, low=None):
    import torch

    def dev(v, dtype=torch.float32):
        return None if v is None else torch.tensor(v, dtype=dtype, device="cuda")

    t, q = eng.sample_filtered(z, dev(u), dev(heat), dev(k, torch.int32), dev(p), dev(low))
    rows = z.double().cpu().numpy()
    f32 = lambda v, i, off: off if v is None else float(np.float32(v[i]))      # noqa: E731
    for i in range(z.shape[0]):
        token, chance = want(rows[i], f32(u, i, 0), f32(heat, i, 1.0), 0 if k is None else k[i], f32(p, i, 1.0), f32(low, i, 0.0))
        assert int(t[i]) == token, (i, int(t[i]), token, float(q[i]), chance)
        assert abs(float(q[i]) - chance) <= 2.0 ** -23 * chance + 1e-45, (i, float(q[i]), chance)
    return t


def scores(seed, batch, vocab, spread=2.5, dtype="float32"):
    import torch

    g = torch.Generator(device="cuda").manual_seed(seed)
    return (torch.randn((batch, vocab), generator=g, device="cuda") * spread).to(getattr(torch, dtype))


def uniform(seed, batch):
    return [float(v) for v in np.random.default_rng(seed).random(batch, dtype=np.float32)]


KINDS = {
    "open": dict(),
    "warm": dict(heat=[0.3, 0.7, 1.0, 1.5, 4.0]),
    "top_k": dict(k=[1, 2, 50, 1000, 5]),
    "top_p": dict(p=[0.1, 0.5, 0.9, 0.99, 0.999]),
    "min_p": dict(low=[0.5, 0.1, 0.01, 1e-6, 1.0]),
    "all": dict(heat=[0.8, 1.2, 0.0, 1.0, 2.0], k=[50, 0, 7, 300, 3], p=[0.9, 0.95, 0.5, 1.0, 0.3], low=[0.0, 0.05, 0.0, 0.2, 0.01]),
}


@pytest.mark.parametrize("kind", sorted(KINDS))
@pytest.mark.parametrize("vocab,dtype", [(1, "float32"), (2, "bfloat16"), (33, "float32"), (2048, "bfloat16"), (4097, "float32"),
                                         (8192, "float32"), (8193, "bfloat16"), (50257, "float32"), (100003, "bfloat16"),
                                         (262144, "float32")])
def test_filters(eng, kind, vocab, dtype):
    for seed in range(2):
        check(eng, scores(seed + vocab, 5, vocab, dtype=dtype), uniform(seed, 5), **KINDS[kind])


@pytest.mark.parametrize("vocab", [64, 5000, 40000, 262144])
def test_many_equal_scores(eng, vocab):
    """All equal, two values, whole numbers: bins with far more entries than the list holds."""
    import torch

    flat = torch.full((1, vocab), -3.5, device="cuda")
    two = torch.where(torch.arange(vocab, device="cuda")[None, :] % 3 == 0, 1.0, -1.0)
    steps = torch.round(scores(3, 1, vocab, 3.0))
    near = 5.0 + scores(4, 1, vocab) * 1e-6                      # a handful of neighbouring fp32 numbers
    z = torch.cat([flat, two, steps, near] * 4)
    n = z.shape[0]
    big = max(1, vocab // 2)
    check(eng, z, uniform(1, n), k=[big] * 4 + [1] * 4 + [0] * 4 + [big + 1] * 4, p=[1.0] * 8 + [0.5] * 4 + [0.73] * 4)
    check(eng, z.bfloat16(), uniform(2, n), heat=[2.0] * n, p=[0.3] * 8 + [0.999] * 8, low=[0.0, 0.1, 0.01, 0.0] * 4)


def test_masked_rows(eng):
    """-inf, the type's lowest value, NaN, +inf; rows with nothing, or with one entry, left."""
    import torch

    for vocab in (100, 30000):
        z = scores(5, 10, vocab)
        z[0] = -torch.inf
        z[1] = torch.nan
        z[2] = -torch.inf
        z[2, vocab - 1] = -7.0
        z[3, ::2] = torch.finfo(torch.float32).min
        z[4] = torch.finfo(torch.float32).min
        z[5, 1::3] = -torch.inf
        z[6, 5:9] = torch.inf
        z[7, :50] = torch.nan
        z[8, 3] = torch.finfo(torch.float32).max
        z[9, 4] = -torch.inf
        u = uniform(vocab, 10)
        t = check(eng, z, u)
        assert t[0] == -1 and t[1] == -1 and t[2] == vocab - 1
        check(eng, z, u, k=[3] * 10, p=[0.8] * 10)
        check(eng, z, u, k=[vocab] * 10, p=[0.99] * 10, low=[0.3] * 10)
        check(eng, z, u, heat=[0.0] * 10)


def test_the_ends_of_the_parameters(eng):
    import torch

    z = scores(6, 12, 9000)
    z[:, 17] = z[:, 4000] = z.amax(1) + 0.25                     # two largest scores
    u = [0.0, -1.0, 0.5, 1.0, 2.0, float("nan"), 1 - 2.0 ** -24, 2.0 ** -30, 0.5, 0.5, 0.5, 0.999]
    nan_as_zero = [0.0 if v != v else v for v in u]
    for given in (dict(), dict(k=[2] * 12), dict(p=[0.9] * 12)):
        a, _ = eng.sample_filtered(z, torch.tensor(u, device="cuda"),
                                   **{"top_" + n: torch.tensor(v, device="cuda", dtype=torch.int32 if n == "k" else torch.float32)
                                      for n, v in given.items()})
        assert torch.equal(a, check(eng, z, nan_as_zero, **given))
    check(eng, z, u[:2] * 6, p=[0.0, -1.0, 1e-30, 1.0, 1.5, 0.0] * 2, k=[0, -5, 1, 2**31 - 1, 9000, 8999] * 2)
    check(eng, z, uniform(1, 12), heat=[1e-30, 1e-6, 1e30, 3e38, -1.0, 0.0] * 2, p=[0.9] * 6 + [1.0] * 6)
    check(eng, z, uniform(1, 12), heat=[0.01, 100.0, 1e4, 1e8, 1.0, 2.0] * 2, k=[40] * 12, low=[0.0, 0.5, 1.0, 2.0, 0.999, 1e-9] * 2)
    nan = torch.full((12,), torch.nan, device="cuda")
    t, _ = eng.sample_filtered(z, torch.tensor(uniform(1, 12), device="cuda"), top_p=nan, min_p=nan)
    assert torch.equal(t, check(eng, z, uniform(1, 12)))
    t, _ = eng.sample_filtered(z, torch.tensor(uniform(1, 12), device="cuda"), temperature=nan)
    assert bool((t == 17).all()), "a NaN temperature is greedy, the lower of two equal scores wins"


@pytest.mark.parametrize("vocab", [300, 2048, 40000, 262144])
@pytest.mark.parametrize("share", [1.0, 0.6])
def test_top_k_of_every_size(eng, vocab, share):
    """Around the sizes at which the entries that can stay are sorted as one list, or no longer; the last index among them."""
    ks = [1, 2, 31, 32, 33, 63, 64, 65, 127, 128, 129, 200, 255, 256, 257, 400, 480, 500, 511, 512, 513, 600, 1000]
    n = len(ks)
    z = scores(41, n, vocab)
    z[:, vocab - 1] = z.amax(1) - 0.1
    z[::2, 0] = z[::2].amax(1)
    for seed in range(3):
        u = uniform(seed, n) if seed < 2 else [0.99999] * n
        check(eng, z, u, k=ks, p=[share] * n, low=[0.0, 0.01, 0.2][seed:seed + 1] * n, heat=[1.0, 3.0, 0.5][seed:seed + 1] * n)
    check(eng, z.round(), uniform(7, n), k=ks, p=[share] * n)


@pytest.mark.parametrize("offset", [0.0, 3.0e4, -1.0e5, 1.0e30, -1.0e-30])
@pytest.mark.parametrize("vocab", [700, 20000])
def test_scores_far_from_zero(eng, offset, vocab):
    """Scores whose spacing is near a bin's width, a temperature's, or min-p's border, with a min-p at either side of 1e-6."""
    import torch

    z = offset + scores(31, 12, vocab, 3.0) * max(1.0, abs(offset) * 2.0 ** -20)
    if abs(offset) < 1e-20:
        z = z * 1e-30
    size = float(z.amax() - z.amin())
    for seed, share in enumerate((1e-6, 1e-3, 0.1, 1.0, 100.0)):
        heat = [max(size * share * f, 1e-38) for f in (0.3, 0.7, 1.0)] * 4
        u = uniform(seed, 12)
        check(eng, z, u, heat=heat, low=[1.0, 0.5, 0.1, 1e-3, 1.0001e-6, 0.999e-6, 1e-9, 1e-20, 0.9999999, 3.0, 0.25, 0.0])
        check(eng, z, u, heat=heat, p=[0.2, 0.9, 0.999, 0.6] * 3, k=[0, 100, 500, 7] * 3)
    flat = torch.full((2, vocab), offset, device="cuda")
    check(eng, flat, [0.3, 0.9], p=[0.4, 1.0], low=[1.0, 0.5])


def test_strides_offsets_and_types(eng):
    import torch

    wide = scores(7, 6, 5000 + 77)
    for view in (wide[:, :5000], wide[:, 1:5001], wide[:, 77:], wide.bfloat16()[:, 3:5002], wide[::2, 5:900]):
        n = view.shape[0]
        check(eng, view, uniform(2, n), k=[60] * n, p=[0.9] * n)
        check(eng, view, uniform(3, n))


def test_frequencies(eng):
    """Evenly spread uniforms give every token its share of them, to within one."""
    import torch

    n = 4096
    z = scores(8, 1, 37, 1.0)
    t, _ = eng.sample_filtered(z.expand(n, 37), (torch.arange(n, device="cuda") + 0.5) / n, top_k=torch.full((n,), 20, dtype=torch.int32, device="cuda"))
    w = torch.exp(z[0].double())
    w[z[0].argsort(descending=True)[20:]] = 0
    counts = torch.bincount(t.long(), minlength=37)
    assert bool(((counts.double() - n * w / w.sum()).abs() <= 1 + 1e-6).all())


def test_the_same_inputs_give_the_same_tokens_anywhere(eng):
    import torch

    z, u = scores(9, 64, 70000), torch.tensor(uniform(9, 64), device="cuda")
    p, k = torch.full((64,), 0.95, device="cuda"), torch.full((64,), 500, dtype=torch.int32, device="cuda")
    first = eng.sample_filtered(z, u, top_k=k, top_p=p)
    torch.cuda.synchronize()
    for _ in range(20):
        assert all(torch.equal(a, b) for a, b in zip(first, eng.sample_filtered(z, u, top_k=k, top_p=p)))
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        again = eng.sample_filtered(z, u, top_k=k, top_p=p)
    other = eng.sample_filtered(z, u, top_k=k, top_p=p)          # both streams at once: the call keeps nothing
    torch.cuda.synchronize()
    assert torch.equal(again[0], first[0]) and torch.equal(other[0], first[0])
    graph = torch.cuda.CUDAGraph()
    whole = torch.full((66,), 5, dtype=torch.int32, device="cuda")
    tokens, probs = whole[:64], torch.zeros(64, device="cuda")
    with torch.cuda.graph(graph):
        eng.sample_filtered(z, u, top_k=k, top_p=p, tokens=tokens, probs=probs)
    u.copy_(1 - u)
    graph.replay()
    torch.cuda.synchronize()
    now = eng.sample_filtered(z, u, top_k=k, top_p=p)
    assert torch.equal(tokens, now[0]) and torch.equal(probs, now[1]) and whole[64:].tolist() == [5, 5]


def test_processed_scores_feed_it(eng, qm):
    """The chain of a decode step: penalty and suppression by the final head, the draw by this call."""
    import torch

    vocab, batch = 2048, 6
    logits = scores(10, batch, vocab, 3.0, "bfloat16")
    history = torch.randint(0, vocab - 1024, (batch, 64), dtype=torch.int32, device="cuda")
    index = torch.full((batch,), 40, dtype=torch.int32, device="cuda")
    processed = torch.empty((batch, vocab), device="cuda")
    eng.final_head_sample(logits, index, history, qm.QM_SAMPLE_REPETITION | qm.QM_SAMPLE_SUPPRESS, eos_token=1000,
                          reserved_begin=vocab - 1024, processed=processed)
    t = check(eng, processed, uniform(4, batch), k=[50] * batch, p=[0.9] * batch)
    assert bool((t < vocab - 1024).all())


def test_the_python_call_checks_its_tensors(eng):
    import torch

    z, u = scores(1, 4, 64), torch.zeros(4, device="cuda")
    for bad in (lambda: eng.sample_filtered(z.half(), u), lambda: eng.sample_filtered(z[:, ::2], u),
                lambda: eng.sample_filtered(z, u[:3]), lambda: eng.sample_filtered(z, u.double()),
                lambda: eng.sample_filtered(z, u, top_k=torch.zeros(4, dtype=torch.int64, device="cuda")),
                lambda: eng.sample_filtered(z, u, top_p=torch.zeros(5, device="cuda"))):
        with pytest.raises(ValueError):
            bad()
    assert math.isfinite(float(eng.sample_filtered(z, u)[1].sum()))
