"""8-bit integer projections and the row quantiser against their definitions in 64 bits.

Bounds, with u = 2^-24 (half a step of fp32) and h = torch.finfo(bfloat16).eps / 2 = 2^-8 (half a step of bf16):

  quantiser, no norm   127 x and the largest |x| are bf16 numbers times 127, and a quotient of two of them is either a
                       half step exactly or at least 2^-16 (relative) away from one, far above u: q equals the
                       rounding of the true quotient.  The scale is one division: u.
  quantiser, norm      q is the rounding of the fp32 quotient, at most half a step plus 127 u from the true one.  The
                       scale: products and largest are exact; the sum of squares has at most dim / 256 + 16 additions
                       of positive terms one after another, each u, and the root halves them; rsqrtf 4 u; mean,
                       epsilon, two products and the division by 127, 5 u.
  linear               the integer sum is exact; its conversion, two products and two additions are u each, of the
                       largest quantity in sight; then one rounding to bf16, h of the result.
  gated                the gate's own error is 3 u |g| in the exponent's argument; the exponential (2 + 1.16 |g|) * 2 u;
                       the rest at most 8 u; then h.
"""
import numpy as np
import pytest

pytestmark = pytest.mark.gpu
U, H = 2.0 ** -24, 2.0 ** -8


@pytest.fixture(scope="module")
def eng(qm):
    e = qm.TalkerAttention(layers=1, num_pages=1, max_positions=8)
    yield e
    assert e.status() == 0
    e.close()


def numbers(seed, *shape, scale=1.0, dtype=None):
    import torch

    g = torch.Generator(device="cuda").manual_seed(seed)
    return (torch.randn(shape, generator=g, device="cuda") * scale).to(dtype or torch.bfloat16)


def levels(seed, *shape):
    import torch

    g = torch.Generator(device="cuda").manual_seed(seed)
    return torch.randint(-128, 128, shape, generator=g, device="cuda", dtype=torch.int8)


def scales(seed, n, of):
    import torch

    g = torch.Generator(device="cuda").manual_seed(seed)
    return torch.rand((n,), generator=g, device="cuda") * of + of / 10


def padded(rows, cols, dtype):
    """An output with three rows behind the last one, and what they hold."""
    import torch

    whole = torch.full((rows + 3, cols), 7, dtype=dtype, device="cuda")
    return whole, whole[:rows]


# ---- quantiser

@pytest.mark.parametrize("rows,dim", [(1, 2048), (3, 1), (5, 7), (2, 16), (33, 1000), (4, 24576), (2, 24575), (700, 2048)])
def test_quantised_rows(eng, rows, dim):
    import torch

    x = numbers(11 + dim, rows, dim, scale=3.0)
    whole, q = padded(rows, dim, torch.int8)
    q, scale = eng.quantize_rows_int8(x, q=q)
    wide = x.double().cpu().numpy()
    big = np.abs(wide).max(1, keepdims=True)
    assert np.array_equal(q.cpu().numpy(), np.rint(127 * wide / big))
    assert np.all(np.abs(scale.double().cpu().numpy() - big[:, 0] / 127) <= U * big[:, 0] / 127)
    assert bool((whole[rows:] == 7).all())


def test_half_steps_go_to_even(eng):
    import torch

    # largest 127: every half is a tie; largest 254: so is every odd number
    row = np.arange(-127, 127.5, 0.5)
    x = torch.tensor(np.stack([row, 2 * row]), dtype=torch.float32, device="cuda").to(torch.bfloat16)
    assert np.array_equal(x.double().cpu().numpy(), np.stack([row, 2 * row])), "the values are bf16 numbers"
    q, scale = eng.quantize_rows_int8(x)
    assert np.array_equal(q.cpu().numpy(), np.stack([np.rint(row), np.rint(row)]))
    assert scale.tolist() == [1.0, 2.0]
    # half of any largest value is the tie 63.5
    big = numbers(3, 500, 1).abs() + 1
    q, _ = eng.quantize_rows_int8(torch.cat([big, big / 2, -big / 2], 1).contiguous())
    assert q.cpu().tolist() == [[127, 64, -64]] * 500


@pytest.mark.parametrize("rows,dim", [(1, 2048), (2, 1), (5, 1001), (300, 1024), (2, 24576)])
def test_quantised_norm(eng, rows, dim):
    x, w = numbers(21 + dim, rows, dim, scale=2.0), numbers(22 + dim, dim) + 1
    q, scale = eng.quantize_rows_int8(x, w)
    xw, ww = x.double().cpu().numpy(), w.double().cpu().numpy()
    v = xw * ww
    big = np.abs(v).max(1, keepdims=True)
    assert np.all(np.abs(127 * v / big - q.cpu().numpy()) <= 0.5 + 127 * U)
    want = big[:, 0] / 127 / np.sqrt((xw ** 2).mean(1) + eng.epsilon)
    assert np.all(np.abs(scale.double().cpu().numpy() - want) <= ((dim / 256 + 16) / 2 + 9) * U * want)


def test_rows_without_a_scale_and_at_the_ends_of_the_range(eng):
    import torch

    x = torch.zeros((8, 40), dtype=torch.bfloat16, device="cuda")
    x[1, 3] = torch.inf
    x[2, 5] = torch.nan
    x[3] = torch.linspace(-3e38, 3e38, 40)       # the difference of the ends is infinite: this row holds NaN
    x[4] = torch.linspace(-1e-38, 1e-38, 40)
    x[5, 39] = 2.0 ** -133                       # the smallest bf16 number above zero
    x[6, 0] = -torch.inf
    x[7] = torch.linspace(-1, 1, 40) * 3e38
    fine = torch.isfinite(x).all(1)
    assert fine.tolist() == [True, False, False, False, True, True, False, True]
    for source in (x, torch.cat([x.new_zeros(1), x.reshape(-1)])[1:].view(8, 40)):      # the second is not 16-byte aligned
        q, scale = eng.quantize_rows_int8(source)
        assert torch.isnan(scale[~fine]).all() and scale[0] == 0 and torch.isfinite(scale[fine]).all()
        assert not q[~fine].any() and not q[0].any()
        wide = x[[4, 5, 7]].double().cpu().numpy()
        assert np.array_equal(q[[4, 5, 7]].cpu().numpy(), np.rint(127 * wide / np.abs(wide).max(1, keepdims=True)))


def test_a_row_of_zeros_without_an_epsilon(eng, monkeypatch):
    """The root mean square is zero and its inverse infinite; the scale is 0 all the same."""
    import torch

    monkeypatch.setattr(eng, "epsilon", 0.0)
    for rows, dim in ((3, 64), (3, 7), (5000, 64)):
        x, w = numbers(1, rows, dim), numbers(2, dim) + 1
        x[1] = 0
        q, scale = eng.quantize_rows_int8(x, w)
        assert scale[1] == 0 and not q[1].any() and torch.isfinite(scale).all() and bool((scale[2:] > 0).all())


# ---- products

def check_linear(got, xq, xs, wq, ws, bias=None, residual=None):
    product = (xq.double() @ wq.double().t()) * xs.double()[:, None] * ws.double()[None, :]      # sums below 2^53: exact
    want, seen = product.clone(), product.abs()
    for extra in (bias, residual):
        if extra is not None:
            want, seen = want + extra.double(), seen + extra.double().abs()
    off = (got.double() - want).abs()
    assert bool((off <= H * want.abs() + (1 + H) * 5 * U * seen).all()), float((off / (want.abs() + 1e-30)).max())


@pytest.mark.parametrize("rows", [1, 16, 17, 33, 64, 65, 129, 700])
@pytest.mark.parametrize("inner,outer", [(16, 1), (48, 7), (128, 64), (144, 100), (2048, 129), (6144, 256)])
def test_linear(eng, rows, inner, outer):
    import torch

    xq, wq = levels(rows, rows, inner), levels(inner + outer, outer, inner)
    xs, ws = scales(5, rows, 0.02), scales(6, outer, 0.01)
    bias, residual = numbers(7, outer), numbers(8, rows, outer, scale=4.0)
    whole, out = padded(rows, outer, torch.bfloat16)
    check_linear(eng.linear_int8(xq, xs, wq, ws, out=out), xq, xs, wq, ws)
    check_linear(eng.linear_int8(xq, xs, wq, ws, bias, residual, out=out), xq, xs, wq, ws, bias, residual)
    assert bool((whole[rows:] == 7).all())
    first = out.clone()
    assert torch.equal(eng.linear_int8(xq, xs, wq, ws, bias, residual), first), "the same call gives the same bits"


@pytest.mark.parametrize("rows", [1, 40, 64, 65, 1000])
@pytest.mark.parametrize("outer", [2048, 100, 37])
def test_the_residual_may_be_the_output(eng, rows, outer):
    import torch

    xq, wq = levels(rows, rows, 512), levels(outer, outer, 512)
    xs, ws, residual = scales(5, rows, 0.02), scales(6, outer, 0.01), numbers(8, rows, outer, scale=4.0)
    want = eng.linear_int8(xq, xs, wq, ws, residual=residual)
    assert eng.linear_int8(xq, xs, wq, ws, residual=residual, out=residual) is residual
    assert torch.equal(residual, want)


def test_the_largest_sums_are_exact(eng):
    import torch

    for rows in (2, 70):
        xq = torch.full((rows, 65536), -128, dtype=torch.int8, device="cuda")
        wq = torch.full((40, 65536), -128, dtype=torch.int8, device="cuda")
        wq[1:] = 127
        one = torch.ones((rows,), device="cuda"), torch.ones((40,), device="cuda")
        got = eng.linear_int8(xq, one[0], wq, one[1])
        assert got[0, 0] == 2.0 ** 30 and got[-1, 1] == torch.tensor(-128.0 * 127 * 65536).to(torch.bfloat16)


@pytest.mark.parametrize("rows", [3, 64, 200])
def test_many_tiles_of_every_width(eng, rows):
    """Outputs wide enough for 256-, 128- and 64-column tiles, and rows of several tiles."""
    for rows_here, outer in ((rows, 2048), (rows * 11, 2184), (rows * 40, 6144)):
        xq, wq = levels(rows_here, rows_here, 256), levels(outer, outer, 256)
        xs, ws = scales(15, rows_here, 0.02), scales(16, outer, 0.01)
        check_linear(eng.linear_int8(xq, xs, wq, ws), xq, xs, wq, ws)


@pytest.mark.parametrize("rows,inner,outer", [(2305, 16, 2049), (2432, 1040, 2041), (5000, 112, 1000), (18945, 144, 7), (130, 2048, 19200)])
def test_the_widest_tiles_at_their_edges(eng, rows, inner, outer):
    """Enough rows and columns for the widest tiles: last tiles of one row or one column, K of less than a chunk and of more
    than the ring, several tiles to an SM."""
    import torch

    xq, wq = levels(rows, rows, inner), levels(outer, outer, inner)
    xs, ws = scales(15, rows, 0.02), scales(16, outer, 0.01)
    bias, residual = numbers(7, outer), numbers(8, rows, outer, scale=4.0)
    whole, out = padded(rows, outer, torch.bfloat16)
    check_linear(eng.linear_int8(xq, xs, wq, ws, out=out), xq, xs, wq, ws)
    check_linear(eng.linear_int8(xq, xs, wq, ws, bias, residual, out=out), xq, xs, wq, ws, bias, residual)
    assert bool((whole[rows:] == 7).all())
    for _ in range(3):
        assert torch.equal(eng.linear_int8(xq, xs, wq, ws, bias, residual), out)
    other = slice(0, 70)                                   # the same rows in a small call
    assert torch.equal(eng.linear_int8(xq[other], xs[other], wq, ws, bias, residual[other]), out[other])
    if outer < 64:
        return
    of = 3.0 / (0.011 * 74 * 74 * inner ** 0.5)
    gs, us, up = scales(4, outer, of), scales(5, outer, of), levels(3, outer, inner)
    gated = eng.gate_up_swiglu_int8(xq, xs, wq, gs, up, us)
    assert torch.equal(eng.gate_up_swiglu_int8(xq[other], xs[other], wq, gs, up, us), gated[other])
    assert torch.equal(eng.gate_up_swiglu_int8(xq[-70:], xs[-70:], wq, gs, up, us), gated[-70:])


def test_qkv_of_tiles_of_several_kinds(eng):
    """Queries wide enough for the widest tiles, keys and values for narrow ones."""
    import torch

    xq, xs = levels(1, 2100, 272), scales(1, 2100, 0.02)
    mats = [(levels(30 + i, n, 272), scales(40 + i, n, 0.01)) for i, n in enumerate((2304, 300, 300))]
    got = eng.qkv_linear_int8(xq, xs, mats[0][0], mats[0][1], mats[1][0], mats[1][1], mats[2][0], mats[2][1])
    for out, (w, s) in zip(got, mats):
        check_linear(out, xq, xs, w, s)


@pytest.mark.parametrize("rows", [1, 31, 64, 65, 300])
@pytest.mark.parametrize("inner,q_dim,kv_dim", [(1024, 2048, 1024), (80, 24, 9)])
def test_qkv_equals_three_linears(eng, rows, inner, q_dim, kv_dim):
    import torch

    xq, xs = levels(rows, rows, inner), scales(1, rows, 0.02)
    mats = [(levels(30 + i, n, inner), scales(40 + i, n, 0.01), numbers(50 + i, n)) for i, n in enumerate((q_dim, kv_dim, kv_dim))]
    got = eng.qkv_linear_int8(xq, xs, mats[0][0], mats[0][1], mats[1][0], mats[1][1], mats[2][0], mats[2][1],
                              mats[0][2], None, mats[2][2])
    for i, (w, s, b) in enumerate(mats):
        b = None if i == 1 else b
        check_linear(got[i], xq, xs, w, s, b)
        assert torch.equal(got[i], eng.linear_int8(xq, xs, w, s, b))


@pytest.mark.parametrize("rows", [1, 16, 61, 64, 65, 500])
@pytest.mark.parametrize("inner,outer", [(2048, 6144), (48, 1), (272, 77), (1024, 200)])
def test_gated(eng, rows, inner, outer):
    import torch

    xq, xs = levels(rows, rows, inner), scales(1, rows, 0.02)
    gate, up = levels(2, outer, inner), levels(3, outer, inner)
    of = 3.0 / (0.011 * 74 * 74 * inner ** 0.5)               # gates of a few units
    gs, us = scales(4, outer, of), scales(5, outer, of)
    whole, out = padded(rows, outer, torch.bfloat16)
    eng.gate_up_swiglu_int8(xq, xs, gate, gs, up, us, out=out)
    g = (xq.double() @ gate.double().t()) * xs.double()[:, None] * gs.double()
    u = (xq.double() @ up.double().t()) * xs.double()[:, None] * us.double()
    assert float(g.abs().max()) < 80
    want = g / (1 + torch.exp(-g)) * u
    bound = want.abs() * (H + (1 + H) * (3 * g.abs() + 2 * (2 + 1.16 * g.abs()) + 8) * U)
    assert bool(((out.double() - want).abs() <= bound).all())
    assert bool((whole[rows:] == 7).all())


def test_a_row_without_a_scale_stays_its_own(eng):
    """NaN and infinity in one row reach that row's outputs alone; a row of zeros gives the bias."""
    import torch

    for rows in (6, 70):
        x = numbers(1, rows, 64)
        x[1, 0], x[2, 3], x[3] = torch.nan, torch.inf, 0
        wq, ws, bias = levels(2, 40, 64), scales(3, 40, 0.01), numbers(4, 40)
        out = eng.linear_int8(*eng.quantize_rows_int8(x), wq, ws, bias)
        assert torch.isnan(out[1:3]).all() and torch.isfinite(out[[0] + list(range(3, rows))]).all()
        assert torch.equal(out[3], bias)


def test_weights_quantised_by_the_launch_just_before(eng):
    """A weight matrix may come from the launch in front of the projection, in either order of the two operands."""
    import torch

    for rows in (4, 64, 300):
        x, w = numbers(rows, rows, 2048), numbers(rows + 1, 2048, 2048)
        want = eng.linear_int8(*[t.clone() for t in eng.quantize_rows_int8(x)], *[t.clone() for t in eng.quantize_rows_int8(w)])
        torch.cuda.synchronize()
        xq, xs = eng.quantize_rows_int8(x)
        wq, ws = torch.zeros((2048, 2048), dtype=torch.int8, device="cuda"), torch.zeros(2048, device="cuda")
        for _ in range(20):
            wq.zero_()
            ws.zero_()
            eng.quantize_rows_int8(w, q=wq, scale=ws)
            assert torch.equal(eng.linear_int8(xq, xs, wq, ws), want)
            xq.zero_()
            eng.quantize_rows_int8(x, q=xq, scale=xs)
            assert torch.equal(eng.linear_int8(xq, xs, wq, ws), want)


def test_on_another_stream_and_captured(eng):
    import torch

    x, wq, ws = numbers(1, 40, 512), levels(2, 300, 512), scales(3, 300, 0.01)
    xq, xs = eng.quantize_rows_int8(x)
    want = eng.linear_int8(xq, xs, wq, ws)
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        got = eng.linear_int8(*eng.quantize_rows_int8(x), wq, ws)
    side.synchronize()
    assert torch.equal(got, want)
    out = torch.zeros_like(want)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        eng.quantize_rows_int8(x, q=xq, scale=xs)
        eng.linear_int8(xq, xs, wq, ws, out=out)
    x.copy_(numbers(9, 40, 512))
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(out, eng.linear_int8(*eng.quantize_rows_int8(x), wq, ws))


def test_the_python_calls_check_their_tensors(eng):
    import torch

    x, (wq, ws) = numbers(1, 4, 64), (levels(2, 32, 64), scales(3, 32, 0.01))
    xq, xs = eng.quantize_rows_int8(x)
    for bad in (lambda: eng.quantize_rows_int8(x.float()), lambda: eng.quantize_rows_int8(x[:, ::2]),
                lambda: eng.quantize_rows_int8(x, numbers(1, 63)), lambda: eng.linear_int8(xq, xs[:3], wq, ws),
                lambda: eng.linear_int8(xq, xs, wq[:, :32], ws), lambda: eng.linear_int8(xq, xs, wq, ws[:5].contiguous()),
                lambda: eng.linear_int8(xq, xs, wq, ws, bias=numbers(1, 31)),
                lambda: eng.gate_up_swiglu_int8(xq, xs, wq, ws, wq[:16].contiguous(), ws),
                lambda: eng.linear_int8(xq.cpu(), xs, wq, ws), lambda: eng.quantize_rows_int8(x.cpu())):
        with pytest.raises(ValueError):
            bad()


def test_tensors_of_another_device_are_refused(eng, monkeypatch):
    """The launch goes to the current device: here that is made to look like another one than the tensors'."""
    import torch

    x, (wq, ws) = numbers(1, 4, 64), (levels(2, 32, 64), scales(3, 32, 0.01))
    xq, xs = eng.quantize_rows_int8(x)
    monkeypatch.setattr(torch.cuda, "current_device", lambda: 1)
    for bad in (lambda: eng.quantize_rows_int8(x), lambda: eng.linear_int8(xq, xs, wq, ws), lambda: eng.gate_up_swiglu_int8(xq, xs, wq, ws, wq, ws),
                lambda: eng.qkv_linear_int8(xq, xs, wq, ws, wq, ws, wq, ws), lambda: eng.sample_filtered(x.float(), xs)):
        with pytest.raises(ValueError):
            bad()
