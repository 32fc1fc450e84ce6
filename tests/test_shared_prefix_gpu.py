"""Decode attention over shared prefixes against its definition in 64 bits.

Bound per element, with h = torch.finfo(bfloat16).eps / 2 = 2^-8: the result is rounded once, h |out|; every softmax weight
of the shared keys is rounded to bf16 for the product with V, which moves the result by at most
h sum_j p_j |v_j| (p the true weights); fp32 scores of 128 terms are off by at most 128 * 2^-24 * sum |q k| / sqrt(128)
<= 2^-11 for the |q|, |k| <= 6 here, which changes weights by that factor, 2^-11 sum_j p_j |v_j| twice (numerator and
sum); the exponentials' and folds' own fp32 errors are below 2^-18 of the same sum.  In all
h |out| + (h + 2^-9) sum_j p_j |v_j|."""
import math

import numpy as np
import pytest

pytestmark = pytest.mark.gpu
H = 2.0 ** -8
PAGE, D = 64, 128


class Case:
    """Groups of (streams, shared pages); own tokens of every stream behind them (negative: the stream is that much
    shorter than the shared part; None: idle)."""

    def __init__(self, qm, groups, own, kv_heads=8, layers=1, seed=0, loose_front=0, loose_back=0, spare=3):
        import torch

        self.qm, self.kv_heads = qm, kv_heads
        rng = np.random.default_rng(seed)
        counts = [n for n, _ in groups]
        batch = loose_front + sum(counts) + loose_back
        shared_of = [0] * loose_front + [p for n, p in groups for _ in range(n)] + [0] * loose_back
        group_of = [-1] * loose_front + [g for g, (n, _) in enumerate(groups) for _ in range(n)] + [-1] * loose_back
        own = [own[i % len(own)] for i in range(batch)]
        self.lens = [0 if o is None else max(0, shared_of[i] * PAGE + o) for i, o in enumerate(own)]
        need = [max(1, (n + PAGE - 1) // PAGE) for n in self.lens]
        max_pages = max(max(need), max([p for _, p in groups], default=1)) + 1
        first, total = [], 0
        for _, p in groups:
            first.append(total)
            total += p
        table = np.full((batch, max_pages), 10 ** 6, dtype=np.int64)      # not a page: nobody may look there
        for s in range(batch):
            for i in range(need[s]):
                if i < shared_of[s] and self.lens[s] >= shared_of[s] * PAGE:
                    table[s, i] = first[group_of[s]] + i
                else:
                    table[s, i] = total
                    total += 1
        names = rng.permutation(total + spare)
        self.table = torch.tensor(np.where(table < 10 ** 6, names[np.minimum(table, total - 1)], 10 ** 6), dtype=torch.int32, device="cuda")
        self.eng = qm.TalkerAttention(layers=layers, num_pages=total + spare, q_heads=2 * kv_heads, kv_heads=kv_heads, max_positions=8)
        gen = torch.Generator(device="cuda").manual_seed(seed)
        self.layer = layers - 1
        self.k, self.v = self.eng.pool_view(self.layer)
        for t in (self.k, self.v):
            t.copy_(torch.randn(t.shape, generator=gen, device="cuda").clamp(-6, 6))
        self.q = torch.randn((batch, 2 * kv_heads, D), generator=gen, device="cuda").clamp(-6, 6).to(torch.bfloat16)
        self.starts = torch.tensor(np.cumsum([loose_front] + counts), dtype=torch.int32, device="cuda")
        self.pages = torch.tensor([p for _, p in groups], dtype=torch.int32, device="cuda")
        self.most = max([p for _, p in groups], default=0)
        self.seq = torch.tensor(self.lens, dtype=torch.int32, device="cuda")

    def run(self, out=None, **change):
        a = dict(layer=self.layer, q_rot=self.q, seq_lens=self.seq, page_table=self.table, group_starts=self.starts, shared_pages=self.pages,
                 max_shared_pages=self.most, out=out)
        return self.eng.launch_attention_shared(**{**a, **change})

    def check(self, out, lens=None, q=None):
        import torch

        q = self.q if q is None else q
        for s, n in enumerate(self.lens if lens is None else lens):
            if n == 0:
                assert not out[s].any(), s
                continue
            at = torch.arange(n, device="cuda")
            page = self.table[s].long()[at // PAGE]
            k = self.k[page, :, at % PAGE].double().transpose(0, 1)           # [heads][n][D]
            v = self.v[page, :, at % PAGE].double().transpose(0, 1)
            p = torch.softmax(q[s].double().reshape(self.kv_heads, 2, D) @ k.transpose(1, 2) / math.sqrt(D), 2)
            want, size = (p @ v).reshape(-1, D), (p @ v.abs()).reshape(-1, D)
            off = (out[s].double() - want).abs()
            assert bool((off <= H * want.abs() + (H + 2.0 ** -9) * size).all()), (s, n, float((off - H * want.abs()).div(size).max()))

    def done(self):
        assert self.eng.status() == 0
        self.eng.close()


CASES = {
    "one stream, one page, no own keys": dict(groups=[(1, 1)], own=[0]),
    "one stream, one own key": dict(groups=[(1, 1)], own=[1]),
    "two streams": dict(groups=[(2, 3)], own=[5, 64]),
    "odd heads": dict(groups=[(5, 7)], own=[1, 63, 64, 65, 200], kv_heads=3),
    "one head": dict(groups=[(3, 40)], own=[10, 0, 130], kv_heads=1),
    "a full tile": dict(groups=[(64, 9)], own=[1, 70, 0, 129]),
    "a tile and one stream": dict(groups=[(65, 9)], own=[1, 70, 0, 129]),
    "three tiles": dict(groups=[(150, 5)], own=[1, 30, 90], kv_heads=2),
    "the largest batch": dict(groups=[(256, 4)], own=[1, 2, 3], kv_heads=2),
    "a long prefix": dict(groups=[(3, 700)], own=[7, 0, 64]),
    "a long prefix, one head": dict(groups=[(2, 1500)], own=[7, 900], kv_heads=1),
    "ragged groups": dict(groups=[(4, 12), (1, 33), (7, 2), (70, 5), (2, 0)], own=[1, 64, 100, 0, 333], kv_heads=4),
    "an empty group": dict(groups=[(3, 4), (0, 9), (2, 6)], own=[12]),
    "idle streams": dict(groups=[(6, 10)], own=[None, 3, None, 0, 77, None]),
    "nobody at all": dict(groups=[(4, 3)], own=[None]),
    "streams shorter than the prefix": dict(groups=[(6, 10), (2, 5)], own=[-1, 50, -64, -639, -640, 0]),
    "the first stream is idle": dict(groups=[(5, 20)], own=[None, 40, 1, 2, -30]),
    "streams outside the groups": dict(groups=[(4, 8), (3, 2)], own=[300, 20, 1], loose_front=3, loose_back=2),
    "more tiles and heads than CTAs": dict(groups=[(2, i % 3 + 1) for i in range(40)], own=[9, 100, 0], kv_heads=16),
    "pieces go round, nothing of their own": dict(groups=[(1, 1 + i % 4) for i in range(50)], own=[0], kv_heads=9),
    "every stream a group": dict(groups=[(1, i % 5) for i in range(40)], own=[9, 100, 0], kv_heads=2),
}


@pytest.mark.parametrize("name", list(CASES))
def test_against_the_definition(qm, name):
    import torch

    c = Case(qm, seed=len(name), **CASES[name])
    whole = torch.full((c.q.shape[0] + 2, 2 * c.kv_heads, D), 3.0, dtype=torch.bfloat16, device="cuda")
    out = c.run(out=whole[:-2])
    c.check(out)
    assert bool((whole[-2:] == 3).all()), "rows behind the last stream stay as they were"
    first = out.clone()
    for _ in range(3):
        assert torch.equal(c.run(), first), "the same call gives the same bits"
    c.done()


def test_agrees_with_the_plain_call(qm):
    """The same tables without groups: the two entry points differ by bf16 steps only, and share a workspace in turn."""
    import torch

    c = Case(qm, [(20, 30), (9, 4)], [1, 500, 64, 0], seed=5)
    got, plain = c.run(), c.eng.launch_attention(0, c.q, c.seq, c.table)
    c.check(got)
    c.check(plain)
    assert torch.equal(c.run(max_shared_pages=0), plain)
    none = torch.zeros((0,), dtype=torch.int32, device="cuda")
    assert torch.equal(c.run(group_starts=torch.zeros(1, dtype=torch.int32, device="cuda"), shared_pages=none), plain)
    assert torch.equal(c.run(), got)
    c.check(c.run(max_shared_pages=3))        # longer entries are cut
    c.done()


def test_group_arrays_out_of_order_are_forced_into_it(qm):
    import torch

    c = Case(qm, [(4, 6), (4, 6)], [5, 70], seed=6)
    for starts, pages in (([4, 0, 8], [6, 6]), ([-3, 4, 100], [6, 6]), ([8, 8, 0], [6, 6])):
        out = c.run(group_starts=torch.tensor(starts, dtype=torch.int32, device="cuda"), shared_pages=torch.tensor(pages, dtype=torch.int32, device="cuda"))
        torch.cuda.synchronize()
        assert c.eng.status() == qm.DEVSTAT_BAD_POS
        c.check(out)
    c.check(c.run(shared_pages=torch.tensor([-5, 6], dtype=torch.int32, device="cuda")))
    c.done()


def test_bad_pages_and_lengths_are_reported(qm):
    import torch

    c = Case(qm, [(3, 4)], [10], seed=7)
    c.table[0, 1] = c.eng.num_pages
    c.run()
    assert c.eng.status() == qm.DEVSTAT_BAD_PAGE
    c.table[0, 1] = -1
    c.run()
    assert c.eng.status() == qm.DEVSTAT_BAD_PAGE
    c.table[0, 1] = 0
    c.run(seq_lens=torch.full_like(c.seq, 10 ** 6))
    assert c.eng.status() & qm.DEVSTAT_BAD_POS
    c.eng.close()


def test_nothing_behind_a_streams_end_is_seen(qm):
    """NaN in every slot that no stream attends, infinities behind the shorter streams."""
    import torch

    c = Case(qm, [(5, 6)], [10, 0, 64, -20, None], seed=8)
    want = c.run().clone()
    seen = torch.zeros(c.k.shape[0] * PAGE, dtype=torch.bool, device="cuda")
    for s, n in enumerate(c.lens):
        at = torch.arange(n, device="cuda")
        seen[c.table[s].long()[at // PAGE] * PAGE + at % PAGE] = True
    hidden = ~seen.reshape(-1, 1, PAGE, 1).expand(c.k.shape)
    c.k[hidden] = torch.nan
    c.v[hidden] = torch.inf
    assert torch.equal(c.run(), want)
    c.done()


def test_large_scores(qm):
    """Scores far apart and growing along the prefix: the running maximum moves again and again."""
    import torch

    c = Case(qm, [(7, 30)], [100, 0], seed=9, kv_heads=2)
    ramp = torch.linspace(0.05, 40, c.k.shape[0], device="cuda")[torch.argsort(torch.argsort(c.table[0, :30].long()))]
    for i in range(30):
        c.k[c.table[0, i].long()] = (c.k[c.table[0, i].long()].float() * ramp[i]).to(torch.bfloat16)
    out = c.run()
    for s, n in enumerate(c.lens):       # scores up to a few hundred: their fp32 error is 128 * 2^-24 * sum |q k| / sqrt(128)
        at = torch.arange(n, device="cuda")
        page = c.table[s].long()[at // PAGE]
        k, v = (t[page, :, at % PAGE].double().transpose(0, 1) for t in (c.k, c.v))
        q = c.q[s].double().reshape(2, 2, D)
        score, size = q @ k.transpose(1, 2) / math.sqrt(D), q.abs() @ k.abs().transpose(1, 2) / math.sqrt(D)
        p = torch.softmax(score, 2)
        off = 128 * 2.0 ** -24 * size.amax(2, keepdim=True)
        assert float(off.max()) < 0.02
        bound = H * (p @ v).abs() + (H + 3 * off + 2.0 ** -12) * (p @ v.abs())
        assert bool(((out[s].double().reshape(2, 2, D) - p @ v).abs() <= bound).all()), s
    c.done()


def test_inputs_written_by_the_launch_just_before(qm):
    """The second launch starts before the first has ended: lengths, tables, queries, K and V that the kernel in front of
    both writes have to be the ones it sees."""
    import torch

    c = Case(qm, [(8, 5)], [200, 30, 1, 65], seed=10)
    q, k = c.q.clone(), c.k.clone()
    want = c.run().clone()
    ones = torch.ones(D, dtype=torch.bfloat16, device="cuda")
    normed = c.eng.launch_rmsnorm(c.q.reshape(-1, D), ones).reshape(c.q.shape).clone()
    want_normed = c.run(q_rot=normed).clone()
    assert not torch.equal(want, want_normed)
    buffer = torch.zeros_like(c.q)
    for _ in range(30):
        buffer.zero_()
        c.eng.launch_rmsnorm(q.reshape(-1, D), ones, out=buffer.view(-1, D))        # a launch that lets the next one go early
        assert torch.equal(c.run(q_rot=buffer), want_normed)
        c.seq.zero_()
        c.k.zero_()
        c.k.copy_(k)
        c.seq.copy_(torch.tensor(c.lens, dtype=torch.int32))
        assert torch.equal(c.run(), want)
    c.done()


def test_captured_and_on_another_stream(qm):
    import torch

    c = Case(qm, [(10, 11), (6, 3)], [33, 500, 0], seed=11)
    want = c.run().clone()
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        got = c.run()
    side.synchronize()
    assert torch.equal(got, want)
    between, out = torch.zeros_like(c.q), torch.zeros_like(c.q)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        c.run(out=between)
        c.run(q_rot=between, out=out)
    other = c.q.flip(0).contiguous()
    want_other = c.run(q_rot=c.run(q_rot=other).clone()).clone()
    c.q.copy_(other)
    for _ in range(3):
        graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(out, want_other)
    c.done()


def test_a_captured_graph_keeps_its_workspace(qm, monkeypatch):
    """A larger batch between the capture of a graph and its replay, and a smaller one after it."""
    import torch

    c = Case(qm, [(12, 11), (60, 3)], [33, 500, 0, 90], seed=21)
    few = dict(q_rot=c.q[:5], seq_lens=c.seq[:5], page_table=c.table[:5], group_starts=torch.tensor([0, 5], dtype=torch.int32, device="cuda"),
               shared_pages=c.pages[:1])
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: True)
    with pytest.raises(RuntimeError):
        c.run(**few)
    monkeypatch.undo()
    small = c.run(**few).clone()
    out = torch.zeros_like(small)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        c.run(**few, out=out)
    want = c.run().clone()
    taken = [torch.full((1 << 20,), 77, dtype=torch.uint8, device="cuda") for _ in range(40)]      # what a freed workspace would go to
    graph.replay()
    again = c.run()
    torch.cuda.synchronize()
    assert torch.equal(out, small) and torch.equal(again, want)
    assert all(bool((t == 77).all()) for t in taken)
    c.check(again)
    c.done()


def test_page_offsets_past_32_bits(qm):
    """Pages far into a pool of more than 2^32 elements."""
    import torch

    c = Case(qm, [(3, 6)], [70, 5], seed=12, kv_heads=8, spare=66000)
    assert c.k.numel() > 2 ** 32
    high = torch.arange(c.eng.num_pages - 20, c.eng.num_pages, dtype=torch.int32, device="cuda")
    used = torch.unique(c.table[c.table < 10 ** 6])
    assert len(used) <= 20
    moved = high[: len(used)]
    for t in (c.k, c.v):
        t[moved.long()] = t[used.long()].clone()
    lookup = torch.full((10 ** 6 + 1,), 10 ** 6, dtype=torch.int32, device="cuda")
    lookup[used.long()] = moved
    want = c.run().clone()
    c.table = lookup[c.table.long()]
    assert torch.equal(c.run(), want)
    c.check(want)
    c.done()


def test_the_python_call_checks_its_tensors(qm):
    c = Case(qm, [(3, 2)], [10], seed=13)
    for bad in (dict(q_rot=c.q.float()), dict(seq_lens=c.seq.long()), dict(seq_lens=c.seq[:2]), dict(group_starts=c.starts[:1]),
                dict(page_table=c.table[:, ::2]), dict(q_rot=c.q[:, :4])):
        with pytest.raises(ValueError):
            c.run(**bad)
    c.done()


NOBODY = {
    "as many pieces as CTAs": dict(groups=[(6, 74)]),                        # 8 heads x 37 pieces of two pages: 2 x 148 SMs
    "as many pieces as CTAs, longer": dict(groups=[(6, 148)]),
    "pieces go round": dict(groups=[(1, 1 + i % 4) for i in range(50)], kv_heads=9),
    "few pieces": dict(groups=[(5, 3), (2, 9)], kv_heads=2),
}


@pytest.mark.parametrize("name", list(NOBODY))
def test_nobody_has_keys_of_its_own_after_a_call_where_everybody_had(qm, name):
    """Lengths that end with the shared part, or at nothing: what an earlier call left in the workspace is not folded in."""
    import torch

    c = Case(qm, own=[70, 5], seed=30 + len(name), **NOBODY[name])
    before = c.run().clone()
    c.check(before)
    shared = [p * PAGE for n, p in NOBODY[name]["groups"] for _ in range(n)]
    for idle in (10 ** 6, 3):
        lens = [0 if i % idle == 1 else n for i, n in enumerate(shared)]
        seq = torch.tensor(lens, dtype=torch.int32, device="cuda")
        first = c.run(seq_lens=seq).clone()
        c.check(first, lens=lens)
        assert torch.equal(c.run(), before)
        assert torch.equal(c.run(seq_lens=seq), first)
    c.done()


@pytest.mark.parametrize("pages", [74, 75])
def test_a_length_past_the_table_is_reported_whichever_ctas_run(qm, pages):
    """Tables that end with the shared part: a longer stream is cut to it, and nobody has keys of its own."""
    import torch

    c = Case(qm, [(6, pages)], [0], seed=31)
    table = c.table[:, :pages].contiguous()
    want = c.run(page_table=table).clone()
    assert c.eng.status() == 0
    c.check(want)
    over = c.seq.clone()
    over[2] += 1
    assert torch.equal(c.run(page_table=table, seq_lens=over), want)
    assert c.eng.status() == qm.DEVSTAT_BAD_POS
    assert torch.equal(c.run(page_table=table, seq_lens=torch.full_like(c.seq, 2 ** 31 - 1)), want)
    assert c.eng.status() == qm.DEVSTAT_BAD_POS
    c.done()
