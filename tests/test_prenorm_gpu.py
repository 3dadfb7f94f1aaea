"""GPU tests of the pre-norm block's operators against plain 64-bit forms (prenorm_oracle.py, which also derives the bounds)."""
import numpy as np
import pytest
import torch

import prenorm_oracle as P

pytestmark = pytest.mark.gpu
TORCH = {"f16": torch.float16, "bf16": torch.bfloat16, "f32": torch.float32}
SEED, STEP = 0x9abcdef012345678, (5 << 32) + 77


@pytest.fixture(scope="module")
def ops():
    from cgpt_b200 import ops as m
    return m


@pytest.fixture(scope="module")
def state(ops):
    return ops.make_dropout_state(SEED, STEP)


def rng(seed):
    return np.random.default_rng(seed)


def dev(a, dt):
    return torch.from_numpy(np.ascontiguousarray(a, dtype=np.float32)).cuda().to(TORCH[dt])


def host(t):
    return t.detach().double().cpu().numpy()


class Guarded:
    """An output between two margins of a known value: what an operator writes outside its output shows. `shift` elements off
    the 16-byte grid. The output starts as NaN: what it leaves out shows too."""
    def __init__(self, shape, dt, shift=0):
        n = int(np.prod(shape))
        self.flat = torch.full((n + 128 + shift,), 7.0, device="cuda", dtype=TORCH[dt])
        self.lo, self.hi = 64 + shift, 64 + shift + n
        self.t = self.flat[self.lo:self.hi].view(shape)
        self.t.fill_(float("nan"))

    def check(self):
        assert bool((self.flat[:self.lo] == 7).all()) and bool((self.flat[self.hi:] == 7).all()), "wrote outside its output"
        return host(self.t)


def shifted(a, dt, shift):
    t = torch.zeros(a.size + 64 + shift, device="cuda", dtype=TORCH[dt])
    t[64 + shift:] = dev(a, dt).reshape(-1)
    return t[64 + shift:].view(a.shape)


def close(got, want, bound, what):
    assert np.all(np.isfinite(got)), f"{what}: not finite"
    over = np.abs(got - want) - bound
    assert over.max() <= 0, f"{what}: off by {np.abs(got - want).reshape(-1)[over.argmax()]:.3e}, bound {(np.zeros_like(got) + bound).reshape(-1)[over.argmax()]:.3e} at {over.argmax()}"


# ------------------------------------------------------------------------------------------------------------ dropout
@pytest.mark.parametrize("dt", ["f16", "bf16", "f32"])
@pytest.mark.parametrize("count", [1, 7, 8, 9, 255, 2048, 2049, 100003])
@pytest.mark.parametrize("shift", [0, 1])
def test_dropout(ops, state, dt, count, shift):
    r = rng(count)
    x, res = shifted(r.standard_normal(count), dt, shift), shifted(r.standard_normal(count), dt, shift)
    for p, site in ((0.1, 0), (0.5, 1), (0.999, 0xffffffff)):
        o = ops.DropoutOptions(p, site)
        want = P.drop(host(x), p, SEED, STEP, site)
        out, summed, grad = Guarded((count,), dt, shift), Guarded((count,), dt, shift), Guarded((count,), dt, shift)
        ops.dropout_forward(out.t, x, state, options=o)
        ops.dropout_forward(summed.t, x, state, options=o, residual=res)
        ops.dropout_backward(grad.t, x, state, options=o)
        # one product by a rounded scale, one addition
        close(out.check(), want, P.rounding(want, TORCH[dt]) + 3 * P.U * np.abs(want), "out")
        assert np.array_equal(grad.check(), host(out.t))
        both = want + host(res)
        close(summed.check(), both, P.rounding(both, TORCH[dt]) + 4 * P.U * (np.abs(want) + np.abs(both)), "residual")


def test_dropout_in_place_and_accumulating(ops, state):
    r = rng(1)
    a, b, o = dev(r.standard_normal(5000), "bf16"), dev(r.standard_normal(5000), "bf16"), ops.DropoutOptions(0.3, 4)
    out, summed = torch.empty_like(a), torch.empty_like(a)
    ops.dropout_forward(out, a, state, options=o)
    ops.dropout_forward(summed, a, state, options=o, residual=b)
    x = a.clone()
    ops.dropout_forward(x, x, state, options=o)
    assert torch.equal(x, out)
    x, y = a.clone(), b.clone()
    ops.dropout_forward(x, x, state, options=o, residual=y)
    ops.dropout_forward(y, a, state, options=o, residual=y)
    assert torch.equal(x, summed) and torch.equal(y, summed)
    y = b.clone()
    ops.dropout_backward(y, a, state, options=o, accumulate_input=True)
    assert torch.equal(y, summed)


@pytest.mark.parametrize("bad", [float("inf"), float("-inf"), float("nan")])
def test_dropped_places_are_zero_whatever_they_held(ops, state, bad):
    x = torch.full((4096,), bad, device="cuda", dtype=torch.float16)
    out = torch.empty_like(x)
    ops.dropout_forward(out, x, state, options=ops.DropoutOptions(0.5, 2))
    kept = torch.from_numpy(P.keep(4096, 0.5, SEED, STEP, 2)).cuda()
    assert bool((out[~kept] == 0).all()) and torch.equal(out[kept].isnan(), x[kept].isnan()) and not bool(out[kept].isfinite().any())


def test_dropout_share_sites_and_steps(ops):
    """The kept share of n independent decisions is within six standard deviations of its mean; two sites, or two steps, agree in
    half of the places the same way."""
    n, p = 1 << 20, 0.5
    x = torch.ones(n, device="cuda")
    masks = []
    state = ops.make_dropout_state(3, 10)
    for site in (0, 1):
        out = torch.empty_like(x)
        ops.dropout_forward(out, x, state, options=ops.DropoutOptions(p, site))
        masks.append(out != 0)
    ops.dropout_advance(state)
    assert state.tolist() == [3, 11]
    ops.dropout_forward(x, x, state, options=ops.DropoutOptions(p, 0))
    masks.append(x != 0)
    for share in [m.double().mean().item() for m in masks] + [(masks[0] == m).double().mean().item() for m in masks[1:]]:
        assert abs(share - 0.5) < 6 * (0.25 / n) ** 0.5


def test_dropout_without_probability_is_the_identity(ops):
    x = dev(rng(0).standard_normal(1001), "f16")
    out = torch.empty_like(x)
    ops.dropout_forward(out, x, None)
    assert torch.equal(out, x)


def test_dropout_beyond_32_bit_offsets(ops, state):
    n = (1 << 32) + 1003
    x = torch.ones(n, device="cuda", dtype=torch.bfloat16)
    ops.dropout_forward(x, x, state, options=ops.DropoutOptions(0.5, 9))
    for first in (0, (1 << 31) - 500, (1 << 32) - 500, n - 1000):
        assert np.array_equal(host(x[first:first + 1000]) != 0, P.keep(1000, 0.5, SEED, STEP, 9, first))


# --------------------------------------------------------------------------------------------------------- layer norm
# rows of one element, below a vector, at and around every change of layout, and beyond what registers hold
SHAPES = [(1, 1), (5, 2), (3, 7), (1, 8), (2, 64), (9, 100), (33, 250), (64, 256), (7, 257), (130, 512), (65, 688), (31, 1000), (17, 1001),
          (37, 712), (40, 1024), (12, 1032), (9, 1537), (11, 2048), (300, 2056), (6, 4096), (7, 4099), (5, 5000), (6, 6008), (4, 8191), (4, 8192), (3, 8200), (2, 12008),
          (3, 14016), (3, 16384), (3, 16385), (2, 33000), (2, 70001)]


def norm_inputs(rows, hidden, dt, seed=0):
    r = rng(rows * 131 + hidden + seed)
    x = r.standard_normal((rows, hidden)) * (0.2 + r.random((rows, 1))) + r.standard_normal((rows, 1))
    x[:, :: max(1, hidden // 5)] *= 6
    vec = lambda c: dev(c + 0.3 * r.standard_normal(hidden), dt)
    return dev(x, dt), vec(1), vec(0), dev(r.standard_normal((rows, hidden)), dt), dev(r.standard_normal((rows, hidden)), dt)


@pytest.mark.parametrize("dt", ["f16", "bf16", "f32"])
@pytest.mark.parametrize("rows,hidden", SHAPES)
def test_layernorm(ops, dt, rows, hidden):
    x, w, b, dy, res = norm_inputs(rows, hidden, dt)
    X, W, B, DY, RES = map(host, (x, w, b, dy, res))
    y, plain = Guarded(x.shape, dt), Guarded(x.shape, dt)
    ops.layernorm_forward(y.t, x, w, b, 1e-5)
    ops.layernorm_forward(plain.t, x, w, None, 1e-5)
    for got, bias in ((y, B), (plain, None)):
        want = P.layernorm(X, W, bias, 1e-5)
        close(got.check(), want, P.rounding(want, TORCH[dt]) + 2 * P.layernorm_error(X, W, bias, 1e-5), "y")
    dx, dw, db = Guarded(x.shape, dt), Guarded(w.shape, dt), Guarded(w.shape, dt)
    ops.layernorm_backward(dx.t, dw.t, db.t, dy, x, w, 1e-5)
    want, err = P.layernorm_backward(DY, X, W, 1e-5), P.layernorm_backward_error(DY, X, W, 1e-5)
    for got, v, e, what in zip((dx, dw, db), want, err, ("dx", "dw", "db")):
        close(got.check(), v, P.rounding(v, TORCH[dt]) + 2 * e, what)
    again, dw2 = Guarded(x.shape, dt), Guarded(w.shape, dt)
    ops.layernorm_backward(again.t, dw2.t, None, dy, x, w, 1e-5, residual=res)
    v = want[0] + RES
    close(again.check(), v, P.rounding(v, TORCH[dt]) + 2 * err[0] + 2 * P.U * (np.abs(RES) + np.abs(v)), "dx + residual")
    assert np.array_equal(dw2.check(), host(dw.t)), "dw depends on what else is asked for"
    in_place = res.clone()
    ops.layernorm_backward(in_place, dw2.t, db.t, dy, x, w, 1e-5, residual=in_place)
    assert torch.equal(in_place, again.t)


@pytest.mark.parametrize("rows,hidden", [(5, 1024), (3, 520), (4, 2048), (4, 99), (2, 40000)])
def test_layernorm_misaligned_tensors(ops, rows, hidden):
    dt = "bf16"
    arrays = [host(t) for t in norm_inputs(rows, hidden, dt)]
    x, w, b, dy, res = (shifted(a, dt, k) for a, k in zip(arrays, (1, 2, 3, 5, 6)))
    X, W, B, DY, RES = arrays
    y, dx, dw, db = (Guarded(s, dt, 1) for s in (x.shape, x.shape, w.shape, w.shape))
    ops.layernorm_forward(y.t, x, w, b, 1e-5)
    ops.layernorm_backward(dx.t, dw.t, db.t, dy, x, w, 1e-5, residual=res)
    want = P.layernorm(X, W, B, 1e-5)
    close(y.check(), want, P.rounding(want, torch.bfloat16) + 2 * P.layernorm_error(X, W, B, 1e-5), "y")
    want, err = P.layernorm_backward(DY, X, W, 1e-5), P.layernorm_backward_error(DY, X, W, 1e-5)
    v = want[0] + RES
    close(dx.check(), v, P.rounding(v, torch.bfloat16) + 2 * err[0] + 2 * P.U * (np.abs(RES) + np.abs(v)), "dx")
    for got, v, e, what in ((dw, want[1], err[1], "dw"), (db, want[2], err[2], "db")):
        close(got.check(), v, P.rounding(v, torch.bfloat16) + 2 * e, what)


@pytest.mark.parametrize("rows,hidden", [(3000, 256), (2500, 1024), (1500, 2048), (700, 4096), (400, 8192), (600, 1001), (900, 2303), (300, 7001), (5000, 130), (5000, 61), (9001, 3), (3000, 24), (1, 4096), (20000, 8)])
@pytest.mark.parametrize("dt", ["bf16", "f32"])
def test_layernorm_many_rows_repeat_bit_for_bit(ops, dt, rows, hidden):
    x, w, _, dy, _ = norm_inputs(rows, hidden, dt)
    want, err = P.layernorm_backward(host(dy), host(x), host(w), 1e-5), P.layernorm_backward_error(host(dy), host(x), host(w), 1e-5)
    outs = []
    for _ in range(2):
        dx, dw, db = Guarded(x.shape, dt), Guarded(w.shape, dt), Guarded(w.shape, dt)
        ops.layernorm_backward(dx.t, dw.t, db.t, dy, x, w, 1e-5)
        for got, v, e, what in zip((dx, dw, db), want, err, ("dx", "dw", "db")):
            close(got.check(), v, P.rounding(v, TORCH[dt]) + 2 * e, what)
        outs.append((dx.t, dw.t, db.t))
    assert all(torch.equal(a, b) for a, b in zip(*outs))


@pytest.mark.parametrize("hidden", [64, 1000, 1024, 4096, 30000])
def test_layernorm_large_offsets_and_constant_rows(ops, hidden):
    """Offsets a thousand times the spread: the variance is taken around the mean. The mean's error, chain * U * 1000, is a shift
    of every element that the second pass sees too. A constant row has no spread: what is left is the mean's error through
    1 / sqrt(eps), within the same bound."""
    r = rng(hidden)
    x = dev(1000 + r.standard_normal((6, hidden)), "f32")
    x[3] = 3.0
    w, b = dev(np.ones(hidden), "f32"), dev(np.zeros(hidden), "f32")
    y = torch.empty_like(x)
    ops.layernorm_forward(y, x, w, b, 1e-5)
    want = P.layernorm(host(x), host(w), host(b), 1e-5)
    close(host(y), want, P.rounding(want, torch.float32) + 2 * P.layernorm_error(host(x), host(w), host(b), 1e-5), "y")
    assert np.abs(host(y)[3]).max() < 1e-2


def test_layernorm_non_finite_rows_stay_in_their_rows(ops):
    x, w, b, dy, _ = norm_inputs(9, 512, "f16")
    clean, dirty = torch.empty_like(x), torch.empty_like(x)
    ops.layernorm_forward(clean, x, w, b, 1e-5)
    x[4, 17] = float("inf")
    x[6, 100] = float("nan")
    ops.layernorm_forward(dirty, x, w, b, 1e-5)
    good = [0, 1, 2, 3, 5, 7, 8]
    assert torch.equal(clean[good], dirty[good]) and bool(dirty[6].isnan().all()) and bool(dirty[4].isnan().any())


def test_layernorm_gradient_against_differences(ops):
    """The kernel's fp32 gradient against central differences of the 64-bit forward (their error is below 1e-7)."""
    x, w, b, dy, _ = norm_inputs(6, 96, "f32")
    dx, dw, db = torch.empty_like(x), torch.empty_like(w), torch.empty_like(w)
    ops.layernorm_backward(dx, dw, db, dy, x, w, 1e-5)
    X, W, B, DY = map(host, (x, w, b, dy))
    err = P.layernorm_backward_error(DY, X, W, 1e-5)
    loss = lambda X, W, B: float((DY * P.layernorm(X, W, B, 1e-5)).sum())
    r, h = rng(3), 1e-5
    for _ in range(4):
        vx, vw, vb = r.standard_normal(X.shape), r.standard_normal(W.shape), r.standard_normal(W.shape)
        num = (loss(X + h * vx, W + h * vw, B + h * vb) - loss(X - h * vx, W - h * vw, B - h * vb)) / (2 * h)
        got = (host(dx) * vx).sum() + (host(dw) * vw).sum() + (host(db) * vb).sum()
        bound = sum(((2 * e + P.U * np.abs(g)) * np.abs(v)).sum() for e, g, v in zip(err, (host(dx), host(dw), host(db)), (vx, vw, vb)))
        assert abs(num - got) < bound + 1e-6


def test_layernorm_beyond_32_bit_offsets(ops):
    rows, hidden = (1 << 21) + 5, 1032
    x = torch.empty(rows, hidden, device="cuda", dtype=torch.bfloat16)
    x.normal_(generator=torch.Generator(device="cuda").manual_seed(0))
    w, b = dev(1 + 0.1 * rng(0).standard_normal(hidden), "bf16"), dev(rng(1).standard_normal(hidden), "bf16")
    y = torch.empty_like(x)
    ops.layernorm_forward(y, x, w, b, 1e-5)
    dx, dw = torch.empty_like(x), torch.empty_like(w)
    ops.layernorm_backward(dx, dw, None, y, x, w, 1e-5)
    for part in (slice(0, 4), slice(rows - 9, rows)):
        X, W, B = host(x[part]), host(w), host(b)
        want = P.layernorm(X, W, B, 1e-5)
        close(host(y[part]), want, P.rounding(want, torch.bfloat16) + 2 * P.layernorm_error(X, W, B, 1e-5), "y")
        DY = host(y[part])
        want, err = P.layernorm_backward(DY, X, W, 1e-5)[0], P.layernorm_backward_error(DY, X, W, 1e-5)[0]
        close(host(dx[part]), want, P.rounding(want, torch.bfloat16) + 2 * err, "dx")


# -------------------------------------------------------------------------------------------- dropout + add + layer norm
@pytest.mark.parametrize("dt", ["f16", "bf16", "f32"])
@pytest.mark.parametrize("rows,hidden", SHAPES)
def test_fused_equals_its_parts(ops, state, dt, rows, hidden):
    """Forward: bit for bit the two calls. Backward: d = dsum + dx is the layer norm's backward with dsum as its residual, bit
    for bit; its dropout map is taken before the rounding, so it is compared with the 64-bit form."""
    x, w, b, dy, res = norm_inputs(rows, hidden, dt)
    dsum = norm_inputs(rows, hidden, dt, seed=1)[4]
    o = ops.DropoutOptions(0.2, 6)
    y, total = Guarded(x.shape, dt), Guarded(x.shape, dt)
    ops.dropout_add_layernorm_forward(y.t, total.t, x, res, w, b, 1e-5, state, options=o)
    want_sum, want_y = torch.empty_like(x), torch.empty_like(x)
    ops.dropout_forward(want_sum, x, state, options=o, residual=res)
    ops.layernorm_forward(want_y, want_sum, w, b, 1e-5)
    y.check(), total.check()
    assert torch.equal(total.t, want_sum) and torch.equal(y.t, want_y)
    for gs in (dsum, None):
        dx, dr, dw, db = (Guarded(s, dt) for s in (x.shape, x.shape, w.shape, w.shape))
        ops.dropout_add_layernorm_backward(dx.t, dr.t, dw.t, db.t, dy, gs, total.t, w, 1e-5, state, options=o)
        want = [torch.empty_like(t) for t in (x, w, w)]
        ops.layernorm_backward(*want, dy, total.t, w, 1e-5, residual=gs)
        assert all(torch.equal(a.t, v) for a, v in zip((dr, dw, db), want))
        dx.check(), dr.check(), dw.check(), db.check()
        S, W, DY = map(host, (total.t, w, dy))
        d = P.layernorm_backward(DY, S, W, 1e-5)[0] + (0 if gs is None else host(gs))
        err = 2 * P.layernorm_backward_error(DY, S, W, 1e-5)[0] + (0 if gs is None else 2 * P.U * (np.abs(host(gs)) + np.abs(d)))
        v = P.drop(d, 0.2, SEED, STEP, 6)
        close(host(dx.t), v, P.rounding(v, TORCH[dt]) + 1.3 * err + 3 * P.U * np.abs(v), "dx")
        if gs is not None:
            buffer = gs.clone()
            ops.dropout_add_layernorm_backward(dx.t, buffer, dw.t, db.t, dy, buffer, total.t, w, 1e-5, state, options=o)
            assert torch.equal(buffer, dr.t)


def fused_against_its_parts_and_64_bits(ops, state, rows, hidden, dt):
    """Both directions of the fused operator: the bits of the two operators it joins, and the 64-bit forms."""
    x, w, b, dy, res = norm_inputs(rows, hidden, dt)
    dsum, o = torch.flip(res, (0,)).contiguous(), ops.DropoutOptions(0.2, 6)
    y, total = Guarded(x.shape, dt), Guarded(x.shape, dt)
    ops.dropout_add_layernorm_forward(y.t, total.t, x, res, w, b, 1e-5, state, options=o)
    want_sum, want_y = torch.empty_like(x), torch.empty_like(x)
    ops.dropout_forward(want_sum, x, state, options=o, residual=res)
    ops.layernorm_forward(want_y, want_sum, w, b, 1e-5)
    Y, S, W, B, DY = y.check(), total.check(), host(w), host(b), host(dy)
    assert torch.equal(total.t, want_sum) and torch.equal(y.t, want_y)
    dropped = P.drop(host(x), 0.2, SEED, STEP, 6)
    v = dropped + host(res)
    close(S, v, P.rounding(v, TORCH[dt]) + 4 * P.U * (np.abs(dropped) + np.abs(v)), "sum")
    v = P.layernorm(S, W, B, 1e-5)
    close(Y, v, P.rounding(v, TORCH[dt]) + 2 * P.layernorm_error(S, W, B, 1e-5), "y")
    dx, dr, dw, db = (Guarded(s, dt) for s in (x.shape, x.shape, w.shape, w.shape))
    ops.dropout_add_layernorm_backward(dx.t, dr.t, dw.t, db.t, dy, dsum, total.t, w, 1e-5, state, options=o)
    want = [torch.empty_like(t) for t in (x, w, w)]
    ops.layernorm_backward(*want, dy, total.t, w, 1e-5, residual=dsum)
    got = [t.check() for t in (dx, dr, dw, db)]
    assert all(torch.equal(a.t, v) for a, v in zip((dr, dw, db), want))
    (d, *sums), (err, *sum_err) = P.layernorm_backward(DY, S, W, 1e-5), P.layernorm_backward_error(DY, S, W, 1e-5)
    d, size = d + host(dsum), np.abs(host(dsum))
    err = 2 * err + 2 * P.U * (size + np.abs(d))
    close(got[1], d, P.rounding(d, TORCH[dt]) + err, "dresidual")
    v = P.drop(d, 0.2, SEED, STEP, 6)
    close(got[0], v, P.rounding(v, TORCH[dt]) + 1.3 * err + 3 * P.U * np.abs(v), "dx")
    for a, v, e, what in zip(got[2:], sums, sum_err, ("dw", "db")):
        close(a, v, P.rounding(v, TORCH[dt]) + 2 * e, what)


@pytest.mark.parametrize("rows,hidden,dt", [(12000, 1001, "bf16"), (20000, 511, "f16"), (5000, 1001, "f32"), (2000, 4099, "bf16")])
def test_fused_odd_rows_through_refilled_stages(ops, state, rows, hidden, dt):
    """Enough rows that every stage of a ring is filled again after its sums were written over what it held; one warp per row and
    several, more than one row a stage."""
    fused_against_its_parts_and_64_bits(ops, state, rows, hidden, dt)


@pytest.mark.parametrize("rows,hidden,dt", [(120000, 64, "bf16"), (20000, 512, "f16"), (10000, 1024, "bf16"), (4000, 2056, "f16"), (700, 8192, "bf16"), (500, 12008, "f16"),
                                            (6000, 1024, "f32"), (500, 8192, "f32")])
def test_fused_whole_vector_rows_through_refilled_stages(ops, state, rows, hidden, dt):
    """Every stage of the rings of both directions is filled again and used again: one, two and four vectors a lane, several rows a
    warp, several warps a row."""
    fused_against_its_parts_and_64_bits(ops, state, rows, hidden, dt)


@pytest.mark.parametrize("rows,hidden,dt", [(20000, 1001, "bf16"), (56000, 250, "f16"), (11000, 1024, "bf16"), (8000, 4099, "f16"), (10000, 1001, "f32"), (2000, 8191, "bf16")])
def test_layernorm_rows_do_not_depend_on_how_many_there_are(ops, rows, hidden, dt):
    """A call whose rings go round more than their stages against calls of 136 rows each (a multiple of 8: every part starts on the
    16-byte grid), which use each stage once: y has the same bits, and dx where rows are whole vectors (of other rows, the tile's
    height says how many warps share one)."""
    g = torch.Generator(device="cuda").manual_seed(rows)
    x, dy = (torch.randn(rows, hidden, device="cuda", generator=g).to(TORCH[dt]) for _ in range(2))
    w, b = dev(1 + 0.2 * rng(0).standard_normal(hidden), dt), dev(rng(1).standard_normal(hidden), dt)
    y, dx, dw, some = Guarded(x.shape, dt), Guarded(x.shape, dt), torch.empty_like(w), torch.empty(136, hidden, device="cuda", dtype=TORCH[dt])
    ops.layernorm_forward(y.t, x, w, b, 1e-5)
    ops.layernorm_backward(dx.t, dw, None, dy, x, w, 1e-5)
    y.check(), dx.check()
    for first in range(0, rows, 136):
        part = slice(first, min(rows, first + 136))
        out = some[:part.stop - first]
        ops.layernorm_forward(out, x[part], w, b, 1e-5)
        assert torch.equal(out, y.t[part])
        if hidden % 8 == 0:
            ops.layernorm_backward(out, dw, None, dy[part], x[part], w, 1e-5)
            assert torch.equal(out, dx.t[part])


@pytest.mark.parametrize("rows,hidden,dt", [(5, 1024, "bf16"), (300, 2048, "f16"), (3, 520, "bf16"), (700, 256, "f32"), (4, 99, "bf16"), (2, 40000, "f16")])
def test_fused_misaligned_tensors(ops, state, rows, hidden, dt):
    """All tensors off the 16-byte grid, each by its own: the bits of the parts, and the 64-bit forms. Then only x, or only the
    residual: sum is the same; y and the gradients are right, if not to the bit (rows are added in another order)."""
    inputs = norm_inputs(rows, hidden, dt)
    o, (X, W, B, DY, RES) = ops.DropoutOptions(0.2, 6), map(host, inputs)
    x, w, b, dy, res = (shifted(a, dt, k) for a, k in zip((X, W, B, DY, RES), (1, 2, 3, 5, 6)))
    dropped = P.drop(X, 0.2, SEED, STEP, 6)
    S = dropped + RES

    def forward(x, res, w, b, shift):
        y, total = Guarded((rows, hidden), dt, shift), Guarded((rows, hidden), dt, shift)
        ops.dropout_add_layernorm_forward(y.t, total.t, x, res, w, b, 1e-5, state, options=o)
        close(total.check(), S, P.rounding(S, TORCH[dt]) + 4 * P.U * (np.abs(dropped) + np.abs(S)), "sum")
        v = P.layernorm(host(total.t), W, B, 1e-5)
        close(y.check(), v, P.rounding(v, TORCH[dt]) + 2 * P.layernorm_error(host(total.t), W, B, 1e-5), "y")
        return y.t, total.t

    y, total = forward(x, res, w, b, 1)
    want_sum, want_y = Guarded(x.shape, dt, 1), Guarded(x.shape, dt, 1)
    ops.dropout_forward(want_sum.t, x, state, options=o, residual=res)
    ops.layernorm_forward(want_y.t, want_sum.t, w, b, 1e-5)
    assert torch.equal(total, want_sum.t) and torch.equal(y, want_y.t)
    for mixed in ((x, inputs[4]), (inputs[0], res)):
        assert torch.equal(forward(*mixed, inputs[1], inputs[2], 0)[1], total)

    T = host(total)
    d, err = P.layernorm_backward(DY, T, W, 1e-5), P.layernorm_backward_error(DY, T, W, 1e-5)
    v, e = d[0] + RES, 2 * err[0] + 2 * P.U * (np.abs(RES) + np.abs(d[0] + RES))
    dropped = P.drop(v, 0.2, SEED, STEP, 6)
    aligned = total.clone()
    for shift, dy_, dsum, total_, w_ in ((1, dy, res, total, w), (0, inputs[3], res, aligned, inputs[1]), (0, dy, inputs[4], aligned, inputs[1])):
        dx, dr, dw, db = (Guarded(s, dt, shift) for s in (x.shape, x.shape, w.shape, w.shape))
        ops.dropout_add_layernorm_backward(dx.t, dr.t, dw.t, db.t, dy_, dsum, total_, w_, 1e-5, state, options=o)
        close(dr.check(), v, P.rounding(v, TORCH[dt]) + e, "dresidual")
        close(dx.check(), dropped, P.rounding(dropped, TORCH[dt]) + 1.3 * e + 3 * P.U * np.abs(dropped), "dx")
        for got, want, bound, what in zip((dw, db), d[1:], err[1:], ("dw", "db")):
            close(got.check(), want, P.rounding(want, TORCH[dt]) + 2 * bound, what)


@pytest.mark.parametrize("hidden", [512, 511, 3000, 2999, 20000])
def test_fused_in_place_sum_and_no_dropout(ops, state, hidden):
    x, w, b, _, res = norm_inputs(1200, hidden, "f16")
    o = ops.DropoutOptions(0.4, 1)
    y, total = torch.empty_like(x), torch.empty_like(x)
    ops.dropout_add_layernorm_forward(y, total, x, res, w, b, 1e-5, state, options=o)
    for target in (x.clone(), res.clone()):
        y2 = torch.empty_like(x)
        a, r = (target, res) if torch.equal(target, x) else (x, target)
        ops.dropout_add_layernorm_forward(y2, target, a, r, w, b, 1e-5, state, options=o)
        assert torch.equal(target, total) and torch.equal(y2, y)
    ops.dropout_add_layernorm_forward(y, total, x, res, w, None, 1e-5, None)
    want = torch.empty_like(x)
    ops.add_tensors(want, x, res)
    assert torch.equal(total, want)


# ---------------------------------------------------------------------------------------------------------- embedding
def ids_dev(a):
    return torch.from_numpy(np.ascontiguousarray(a, dtype=np.uint32).view(np.int32)).cuda()


@pytest.mark.parametrize("dt", ["f16", "bf16", "f32"])
@pytest.mark.parametrize("tokens,vocab,hidden", [(1, 1, 1), (3, 5, 7), (17, 9, 8), (100, 1000, 64), (65, 33, 250), (33, 50, 1024), (9, 4, 1001), (5, 3, 5000)])
def test_scaled_embedding_forward(ops, state, dt, tokens, vocab, hidden):
    r = rng(tokens)
    ids = r.integers(0, vocab, tokens).astype(np.uint32)
    ids[tokens // 2] = vocab
    ids[tokens // 3] = 0xffffffff
    w = dev(r.standard_normal((vocab, hidden)), dt)
    for p in (0.0, 0.3):
        out = Guarded((tokens, hidden), dt)
        ops.scaled_embedding_forward(out.t, ids_dev(ids), tokens, w, state, options=ops.ScaledEmbeddingOptions(2.5, dropout=ops.DropoutOptions(p, 8)))
        want = P.drop(P.embedding(ids, host(w), 2.5), p, SEED, STEP, 8)
        close(out.check(), want, P.rounding(want, TORCH[dt]) + 4 * P.U * np.abs(want), "out")


@pytest.mark.parametrize("hidden", [8, 40, 1024])
@pytest.mark.parametrize("dt", ["bf16", "f32"])
def test_scaled_embedding_forward_of_unaligned_tensors(ops, state, hidden, dt):
    """Rows of whole vectors whose table, output or both start off the 16-byte grid: the bits of the aligned call."""
    r = rng(hidden)
    ids, table = r.integers(0, 60, 333).astype(np.uint32), r.standard_normal((50, hidden))
    for p in (0.0, 0.3):
        o, got = ops.ScaledEmbeddingOptions(2.5, dropout=ops.DropoutOptions(p, 8)), []
        for table_shift, out_shift in ((0, 0), (1, 0), (0, 1), (3, 1)):
            out = Guarded((333, hidden), dt, out_shift)
            ops.scaled_embedding_forward(out.t, ids_dev(ids), 333, shifted(table, dt, table_shift), state, options=o)
            got.append(out.check())
        assert all(np.array_equal(got[0], g) for g in got[1:])
        want = P.drop(P.embedding(ids, host(dev(table, dt)), 2.5), p, SEED, STEP, 8)
        close(got[0], want, P.rounding(want, TORCH[dt]) + 4 * P.U * np.abs(want), "out")


def backward_case(kind, tokens, vocab, r):
    if kind == "uniform":
        return r.integers(0, vocab, tokens)
    if kind == "same":
        return np.full(tokens, vocab // 2)
    if kind == "skewed":
        return np.minimum(vocab - 1, (np.exp(r.random(tokens) * np.log(vocab + 1)) - 1).astype(np.int64))
    if kind == "sorted":
        return np.sort(r.integers(0, vocab, tokens))
    if kind == "outside":
        return np.where(r.random(tokens) < 0.5, r.integers(0, vocab, tokens), vocab + r.integers(0, 1 << 20, tokens))
    return np.full(tokens, 0xffffffff)     # "none": no token points into the table


@pytest.mark.parametrize("kind", ["uniform", "same", "skewed", "sorted", "outside", "none"])
@pytest.mark.parametrize("tokens,vocab,hidden,dt", [(1, 1, 1, "f32"), (2, 3, 8, "bf16"), (31, 7, 64, "f16"), (32, 1, 40, "f32"), (33, 2, 250, "f32"),
                                                   (64, 600, 16, "bf16"), (777, 1000, 72, "f32"), (2048, 100, 8, "f32"), (2049, 511, 24, "f16"),
                                                   (5000, 40000, 4, "f32"), (10007, 300000, 8, "bf16"), (3000, 77, 1001, "bf16"), (1000, 5, 5000, "bf16"),
                                                   (1024, 1500, 1032, "bf16"), (1023, 3, 2100, "f32"), (900, 70000, 33, "f16"),
                                                   (1025, 40, 96, "bf16"), (512, 1500, 1032, "bf16"), (511, 3, 2100, "f32"),
                                                   (513, 300, 1000, "f16"), (9001, 700, 1024, "f16"), (30011, 90, 64, "bf16"), (5003, 2000, 512, "f32")])
def test_scaled_embedding_backward(ops, state, kind, tokens, vocab, hidden, dt):
    r = rng(tokens + vocab)
    ids = backward_case(kind, tokens, vocab, r).astype(np.uint32)
    grad, before = dev(r.standard_normal((tokens, hidden)), dt), dev(r.standard_normal((vocab, hidden)), dt)
    for p, padding, accumulate in ((0.0, None, False), (0.3, int(ids[0]) if ids[0] < vocab else 0, False), (0.3, None, True)):
        o = ops.ScaledEmbeddingOptions(1.75, padding, ops.DropoutOptions(p, 8), accumulate)
        table, size, count = P.embedding_backward(ids, P.drop(host(grad), p, SEED, STEP, 8), vocab, 1.75, padding)
        got = []
        for _ in range(2):
            out = Guarded((vocab, hidden), dt)
            if accumulate:
                out.t.copy_(before)
            ops.scaled_embedding_backward(out.t, grad, ids_dev(ids), tokens, state, options=o)
            want = table + (host(before) if accumulate else 0)
            # a row's sum has at most its token count of terms; the dropout scale, the scale and the old value round once each
            err = P.U * ((count[:, None] + 8) * size + 2 * np.abs(want))
            close(out.check(), want, P.rounding(want, TORCH[dt]) + err, "grad_weight")
            got.append(out.t)
        assert torch.equal(*got)
        if accumulate:
            untouched = torch.from_numpy(count == 0).cuda()
            assert torch.equal(got[0][untouched], before[untouched])


@pytest.mark.parametrize("kind", ["uniform", "same", "skewed", "outside", "none"])
@pytest.mark.parametrize("tokens,vocab,hidden,dt,shift", [(65537, 500, 8, "f32", 0), (70001, 511, 5, "bf16", 0), (70003, 40000, 8, "bf16", 0), (66000, 3000, 24, "f16", 1),
                                                         (100003, 300000, 4, "f32", 0), (68000, 262144, 3, "f16", 1)])
def test_scaled_embedding_backward_of_many_tokens(ops, state, kind, tokens, vocab, hidden, dt, shift):
    """More tokens than one cluster sorts: count, prefix and scatter launches, one, two and three passes of them, the table cleared
    by itself; ids outside the table, a padding id, accumulation, dropout, tensors off the 16-byte grid."""
    r = rng(tokens)
    ids = backward_case(kind, tokens, vocab, r).astype(np.uint32)
    grad, before = shifted(r.standard_normal((tokens, hidden)), dt, shift), dev(r.standard_normal((vocab, hidden)), dt)
    for p, padding, accumulate in ((0.0, None, False), (0.3, int(ids[0]) if ids[0] < vocab else 0, False), (0.3, None, True)):
        o = ops.ScaledEmbeddingOptions(1.75, padding, ops.DropoutOptions(p, 8), accumulate)
        table, size, count = P.embedding_backward(ids, P.drop(host(grad), p, SEED, STEP, 8), vocab, 1.75, padding)
        got = []
        for _ in range(2):
            out = Guarded((vocab, hidden), dt, shift)
            if accumulate:
                out.t.copy_(before)
            ops.scaled_embedding_backward(out.t, grad, ids_dev(ids), tokens, state, options=o)
            want = table + (host(before) if accumulate else 0)
            close(out.check(), want, P.rounding(want, TORCH[dt]) + P.U * ((count[:, None] + 8) * size + 2 * np.abs(want)), "grad_weight")
            got.append(out.t)
        assert torch.equal(*got)
        if accumulate:
            untouched = torch.from_numpy(count == 0).cuda()
            assert torch.equal(got[0][untouched], before[untouched])


@pytest.mark.parametrize("vocab", [400, 50000, 400000])
def test_both_sorts_keep_the_tokens_in_order(ops, state, vocab):
    """The same tokens through the cluster sort, and, with 64 skipped ones behind them, through the launches per digit. Both counts
    are summed in chunks of equal length, so the bits are the same exactly if the sorted tokens are."""
    tokens, hidden, more = 65536, 8, 64
    r = rng(vocab)
    ids, grad = backward_case("skewed", tokens, vocab, r), r.standard_normal((tokens + more, hidden))
    o, g = ops.ScaledEmbeddingOptions(1.5, dropout=ops.DropoutOptions(0.2, 4)), dev(grad, "f32")
    a, b = (torch.empty(vocab, hidden, device="cuda") for _ in range(2))
    ops.scaled_embedding_backward(a, g[:tokens], ids_dev(ids), tokens, state, options=o)
    ops.scaled_embedding_backward(b, g, ids_dev(np.concatenate([ids, vocab + np.arange(more)])), tokens + more, state, options=o)
    assert torch.equal(a, b)


def test_scaled_embedding_backward_of_unaligned_tensors(ops):
    r = rng(5)
    ids = r.integers(0, 40, 500).astype(np.uint32)
    g = r.standard_normal((500, 64))
    a, b = Guarded((40, 64), "bf16"), Guarded((40, 64), "bf16", 1)
    ops.scaled_embedding_backward(a.t, dev(g, "bf16"), ids_dev(ids), 500)
    ops.scaled_embedding_backward(b.t, shifted(g, "bf16", 1), ids_dev(ids), 500)
    assert np.array_equal(a.check(), b.check())


def test_scaled_embedding_large_table_and_many_tokens(ops):
    """A table of more than 2^31 elements, and more tokens than one pass of any small path takes."""
    vocab, hidden, tokens = (1 << 21) + 3, 1032, 3000
    ids = np.concatenate([[0, vocab - 1, vocab - 1], rng(0).integers(0, vocab, tokens - 3)]).astype(np.uint32)
    grad = torch.ones(tokens, hidden, device="cuda", dtype=torch.bfloat16)
    dw = torch.full((vocab, hidden), float("nan"), device="cuda", dtype=torch.bfloat16)
    ops.scaled_embedding_backward(dw, grad, ids_dev(ids), tokens)
    count = torch.from_numpy(np.bincount(ids, minlength=vocab)).cuda()
    assert torch.equal(dw[:, 0].long(), count) and torch.equal(dw[:, -1].long(), count)
    out = torch.empty(tokens, hidden, device="cuda", dtype=torch.bfloat16)
    ops.scaled_embedding_forward(out, ids_dev(ids), tokens, dw)
    assert torch.equal(out[:, 0], dw[torch.from_numpy(ids.astype(np.int64)).cuda(), 0])
    del dw
    tokens, vocab, hidden = 400_003, 1000, 8
    ids = rng(1).integers(0, vocab, tokens).astype(np.uint32)
    dw = torch.empty(vocab, hidden, device="cuda")
    ops.scaled_embedding_backward(dw, torch.ones(tokens, hidden, device="cuda"), ids_dev(ids), tokens)
    assert np.array_equal(host(dw)[:, 3], np.bincount(ids, minlength=vocab))


# ------------------------------------------------------------------------------- streams, graphs, workspaces, refusals
def test_refusals(ops, state):
    x, w, ids = torch.zeros(4, 8, device="cuda"), torch.zeros(8, device="cuda"), torch.zeros(4, device="cuda", dtype=torch.int32)
    y, table = torch.empty_like(x), torch.zeros(10, 8, device="cuda")
    bad = [
        lambda: ops.dropout_forward(y, x.half(), state),
        lambda: ops.dropout_forward(y, x, None, options=ops.DropoutOptions(0.5)),
        lambda: ops.dropout_forward(y, x, state.float(), options=ops.DropoutOptions(0.5)),
        lambda: ops.dropout_forward(y, x, state, options=ops.DropoutOptions(1.0)),
        lambda: ops.dropout_forward(y, x, state, options=ops.DropoutOptions(0.5, -1)),
        lambda: ops.dropout_forward(y[:, :4], x[:, :4], state),
        lambda: ops.dropout_forward(y, x, state, residual=x.view(-1)),
        lambda: ops.dropout_backward(x, x, state, options=ops.DropoutOptions(0.5), accumulate_input=True),
        lambda: ops.dropout_forward(torch.empty(0, device="cuda"), torch.empty(0, device="cuda"), state),
        lambda: ops.layernorm_forward(y, x, w[:4], None, 1e-5),
        lambda: ops.layernorm_forward(x, x, w, None, 1e-5),
        lambda: ops.layernorm_forward(y, x, w, None, 0.0),
        lambda: ops.layernorm_forward(y[:0], x[:0], w, None, 1e-5),
        lambda: ops.layernorm_forward(y.view(2, 2, 8), x.view(2, 2, 8), w, None, 1e-5),
        lambda: ops.layernorm_backward(y, w, w.clone(), x, x, w, 1e-5, workspace=torch.empty(4, device="cuda")),
        lambda: ops.layernorm_backward(x, w, w.clone(), x, y, w, 1e-5),
        lambda: ops.dropout_add_layernorm_forward(y, y, x, x.clone(), w, w, 1e-5, state),
        lambda: ops.dropout_add_layernorm_backward(y, y, w, w, x, None, x.clone(), w, 1e-5, state),
        lambda: ops.scaled_embedding_forward(y, ids.long(), 4, table),
        lambda: ops.scaled_embedding_forward(y, ids, 5, table),
        lambda: ops.scaled_embedding_forward(y, ids, 0, table),
        lambda: ops.scaled_embedding_backward(table, x, ids, 4, options=ops.ScaledEmbeddingOptions(padding_id=10)),
        lambda: ops.scaled_embedding_backward(table, x, ids, 4, workspace=torch.empty(4, device="cuda")),
    ]
    for i, call in enumerate(bad):
        with pytest.raises(ValueError):
            call()
            pytest.fail(f"call {i} was accepted")


def block_step(ops, t, o):
    """One forward and backward through embedding, branch, boundary, with the buffers of `t`."""
    s = t["state"]
    ops.scaled_embedding_forward(t["h0"], t["ids"], t["n"], t["table"], s, options=o["embed"])
    ops.layernorm_forward(t["y0"], t["h0"], t["w0"], t["b0"], 1e-5)
    ops.linear_forward(t["z"], t["y0"], t["proj"])
    ops.dropout_add_layernorm_forward(t["y1"], t["h1"], t["z"], t["h0"], t["w1"], t["b1"], 1e-5, s, options=o["branch"])
    ops.dropout_forward(t["out"], t["y1"], s, options=o["last"])
    ops.dropout_backward(t["dy1"], t["dout"], s, options=o["last"])
    ops.dropout_add_layernorm_backward(t["dz"], t["dh"], t["dw1"], t["db1"], t["dy1"], None, t["h1"], t["w1"], 1e-5, s, options=o["branch"])
    ops.linear_backward(t["dy0"], t["dproj"], None, t["dz"], t["y0"], t["proj"])
    ops.layernorm_backward(t["dh"], t["dw0"], t["db0"], t["dy0"], t["h0"], t["w0"], 1e-5, residual=t["dh"])
    ops.scaled_embedding_backward(t["dtable"], t["dh"], t["ids"], t["n"], s, options=o["embed"])
    ops.dropout_advance(s)


def block_tensors(ops, n, vocab, d, seed, dt="f32"):
    r = rng(seed)
    g = lambda *s, c=0.0, k=1.0: dev(c + k * r.standard_normal(s), dt)
    t = dict(n=n, ids=ids_dev(r.integers(0, vocab, n)), table=g(vocab, d, k=0.3), w0=g(d, c=1, k=0.2), b0=g(d, k=0.2), w1=g(d, c=1, k=0.2),
             b1=g(d, k=0.2), proj=g(d, d, k=d ** -0.5), dout=g(n, d), state=ops.make_dropout_state(seed, 3))
    for name in ("h0", "y0", "z", "y1", "h1", "out", "dy1", "dz", "dh", "dy0"):
        t[name] = torch.full((n, d), float("nan"), device="cuda", dtype=TORCH[dt])
    for name in ("dw0", "db0", "dw1", "db1"):
        t[name] = torch.full((d,), float("nan"), device="cuda", dtype=TORCH[dt])
    t["dtable"], t["dproj"] = torch.full_like(t["table"], float("nan")), torch.full_like(t["proj"], float("nan"))
    return t


def block_options(ops, d):
    return dict(embed=ops.ScaledEmbeddingOptions(d ** 0.5, dropout=ops.DropoutOptions(0.1, 0)), branch=ops.DropoutOptions(0.2, 1), last=ops.DropoutOptions(0.3, 2))


RESULTS = ("out", "h1", "dtable", "dw0", "db0", "dw1", "db1", "dproj")


@pytest.mark.parametrize("n,vocab,d", [(50, 20, 64), (33, 9, 100)])
def test_a_step_of_a_block(ops, n, vocab, d):
    """fp32 throughout, against the 64-bit composition. Each of the seven operators on the longest path (two of them products of
    d terms) is off by less than 2 chain(d) U of the size of its output, and every one passes an error on by a factor below
    ten (1 / keep, rstd and weights are all of order one): 1e-4 of the tensors' largest value is a hundred times their sum."""
    t = block_tensors(ops, n, vocab, d, 1)
    o = block_options(ops, d)
    block_step(ops, t, o)
    h = {k: host(v) for k, v in t.items() if isinstance(v, torch.Tensor) and v.is_floating_point()}
    ids = host(t["ids"]).astype(np.int64)
    mask = lambda x, p, site: P.drop(x, p, 1, 3, site)
    h0 = mask(P.embedding(ids, h["table"], d ** 0.5), 0.1, 0)
    y0 = P.layernorm(h0, h["w0"], h["b0"], 1e-5)
    h1 = h0 + mask(y0 @ h["proj"].T, 0.2, 1)
    out = mask(P.layernorm(h1, h["w1"], h["b1"], 1e-5), 0.3, 2)
    dy1 = mask(h["dout"], 0.3, 2)
    dh, dw1, db1 = P.layernorm_backward(dy1, h1, h["w1"], 1e-5)
    dz = mask(dh, 0.2, 1)
    dx0, dw0, db0 = P.layernorm_backward(dz @ h["proj"], h0, h["w0"], 1e-5)
    dtable = P.embedding_backward(ids, mask(dh + dx0, 0.1, 0), vocab, d ** 0.5)[0]
    want = dict(out=out, h1=h1, dtable=dtable, dw0=dw0, db0=db0, dw1=dw1, db1=db1, dproj=dz.T @ y0)
    for name in RESULTS:
        close(h[name], want[name], 1e-4 * np.abs(want[name]).max(), name)
    assert t["state"].tolist() == [1, 4]


def test_graph_replays_draw_new_masks_and_eager_calls_between_them_do_not_disturb(ops):
    n, vocab, d = 400, 50, 256
    o = block_options(ops, d)
    t, other, eager = (block_tensors(ops, n, vocab, d, s, "bf16") for s in (1, 2, 1))
    block_step(ops, other, o)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        block_step(ops, t, o)
    seen = []
    for step in range(3):
        graph.replay()
        block_step(ops, other, o)
        block_step(ops, eager, o)
        torch.cuda.synchronize()
        assert t["state"].tolist() == eager["state"].tolist() == [1, 4 + step]
        assert all(torch.equal(t[k], eager[k]) for k in RESULTS)
        seen.append(t["out"].clone())
    assert not torch.equal(seen[0], seen[1]) and not torch.equal(seen[1], seen[2])


def test_two_graphs_and_two_streams_at_once(ops):
    """Two captured steps replayed on two streams at the same time, and two eager ones: no workspace is shared."""
    n, vocab, d = 3000, 700, 512
    o = block_options(ops, d)
    alone, graphs, streams = [], [], [torch.cuda.Stream(), torch.cuda.Stream()]
    for seed in (1, 2):
        t = block_tensors(ops, n, vocab, d, seed, "bf16")
        block_step(ops, t, o)
        alone.append(t)
    together = [block_tensors(ops, n, vocab, d, seed, "bf16") for seed in (1, 2)]
    torch.cuda.synchronize()
    prenorm = lambda t: [f() for f in (
        lambda: ops.scaled_embedding_forward(t["h0"], t["ids"], n, t["table"], t["state"], options=o["embed"]),
        lambda: ops.dropout_add_layernorm_forward(t["y1"], t["h1"], alone[t["k"]]["z"], t["h0"], t["w1"], t["b1"], 1e-5, t["state"], options=o["branch"]),
        lambda: ops.dropout_backward(t["dy1"], t["dout"], t["state"], options=o["last"]),
        lambda: ops.dropout_add_layernorm_backward(t["dz"], t["dh"], t["dw1"], t["db1"], t["dy1"], None, t["h1"], t["w1"], 1e-5, t["state"], options=o["branch"]),
        lambda: ops.layernorm_backward(t["dh"], t["dw0"], t["db0"], alone[t["k"]]["dy0"], t["h0"], t["w0"], 1e-5, residual=t["dh"]),
        lambda: ops.scaled_embedding_backward(t["dtable"], t["dh"], t["ids"], n, t["state"], options=o["embed"]))]
    for k, t in enumerate(together):
        t["k"] = k
        graphs.append(torch.cuda.CUDAGraph())
        with torch.cuda.graph(graphs[-1]):
            prenorm(t)
    names = ("h1", "dz", "dtable", "dw0", "db0", "dw1", "db1")

    def run_and_compare(launch):
        for t in together:
            for k in names:
                t[k].fill_(float("nan"))
        torch.cuda.synchronize()
        for _ in range(4):
            for k in (0, 1):
                with torch.cuda.stream(streams[k]):
                    launch(k)
        torch.cuda.synchronize()
        for t, want in zip(together, alone):
            assert all(torch.equal(t[k], want[k]) for k in names)

    run_and_compare(lambda k: graphs[k].replay())
    run_and_compare(lambda k: prenorm(together[k]))


def test_explicit_stream_and_caller_workspace(ops, state):
    x, w, b, dy, _ = norm_inputs(200, 512, "bf16")
    want = [torch.empty_like(t) for t in (x, w, w)]
    ops.layernorm_backward(*want, dy, x, w, 1e-5)
    got = [torch.full_like(t, float("nan")) for t in (x, w, w)]
    workspace = torch.empty(ops.layernorm_backward_workspace_bytes(200, 512), device="cuda", dtype=torch.uint8)
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    ops.layernorm_backward(*got, dy, x, w, 1e-5, stream=stream, workspace=workspace)
    stream.synchronize()
    assert all(torch.equal(a, v) for a, v in zip(got, want))
    ops.layernorm_backward(*got, dy, x, w, 1e-5, stream=stream)
    stream.synchronize()
    assert all(torch.equal(a, v) for a, v in zip(got, want))


@pytest.mark.parametrize("hidden", [256, 1001, 1024])
def test_one_workspace_for_the_largest_batch(ops, state, hidden):
    """A workspace for the most rows serves all smaller calls: the bits are those of a call with its own."""
    most = 1300
    x, w, _, dy, _ = norm_inputs(most, hidden, "bf16")
    ids, o = ids_dev(rng(2).integers(0, 3000, most).astype(np.uint32)), ops.ScaledEmbeddingOptions(2.0, dropout=ops.DropoutOptions(0.1, 3))
    for_norm = torch.empty(ops.layernorm_backward_workspace_bytes(most, hidden), device="cuda", dtype=torch.uint8)
    for_table = torch.empty(ops.scaled_embedding_backward_workspace_bytes(most, hidden), device="cuda", dtype=torch.uint8)
    for n in (1, 2, 147, 296, 297, 591, 593, 1183, 1184, 1185, most):
        want, got = ([torch.full_like(t, float("nan")) for t in (x[:n], w, w)] for _ in range(2))
        ops.layernorm_backward(*want, dy[:n], x[:n], w, 1e-5)
        ops.layernorm_backward(*got, dy[:n], x[:n], w, 1e-5, workspace=for_norm)
        assert all(torch.equal(a, v) for a, v in zip(got, want))
        want, got = (torch.full((3000, hidden), float("nan"), device="cuda", dtype=x.dtype) for _ in range(2))
        ops.scaled_embedding_backward(want, dy[:n], ids, n, state, options=o)
        ops.scaled_embedding_backward(got, dy[:n], ids, n, state, options=o, workspace=for_table)
        assert torch.equal(got, want)


def test_the_callers_last_error_is_left_alone(ops):
    """A gradient through the sort between a refused runtime call and the caller's look at its error. (Not the first in its process:
    the runtime itself clears the error where it sets a kernel's attributes, once per device.)"""
    from cgpt_b200 import _lib
    runtime, ids, grad = _lib.lib, torch.zeros(2000, dtype=torch.int32, device="cuda"), torch.ones(2000, 64, device="cuda")
    table, size = torch.empty(50000, 64, device="cuda"), ops.scaled_embedding_backward_workspace_bytes(2000, 64)
    workspace, stream = torch.empty(size, dtype=torch.uint8, device="cuda"), torch.cuda.current_stream().cuda_stream
    call = lambda: _lib.lib.cgpt_scaled_embedding_backward(table.data_ptr(), grad.data_ptr(), ids.data_ptr(), workspace.data_ptr(), size, 2000,
                                                           50000, 64, 1.0, 0xffffffff, 0.0, None, 0, 0, _lib.F32, stream)
    assert call() == 0
    refused = runtime.cudaSetDevice(-1)
    rc, seen = call(), runtime.cudaGetLastError()
    assert rc == 0 and refused != 0 and seen == refused
    assert bool((table[0] == 2000).all()) and not bool(table[1:].any())
