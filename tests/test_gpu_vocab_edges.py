"""The row operations over the vocabulary where their numbers or their arguments are at an end of what is allowed, and rows of a call that
holds a bad one.  Tolerances: those of test_gpu_vocab_rows.py, whose derivation covers every case here."""
import numpy as np
import pytest

import rust_trainer_b200 as rt
import vocab_reference as R
from rust_trainer_b200 import ops
from test_gpu_vocab_rows import DT, U, Rows, _before, _check_distill, _check_prob, _check_top, _check_verify, _dev, _distill, _drafts, _empty, _lists, _logits, _sync, _top, _verify

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("k", [1, 5, 130])
def test_clusters_that_take_several_rows_and_find_all_in_one_place(ctx, k):
    """The largest elements of a row lie in one CTA's units, so that it waits for nobody's; the cluster goes on to the next row."""
    rng = np.random.default_rng(k)
    for rows, vocab in ((37, 50021), (19, 100003), (74, 20011), (146, 9001)):
        v = _logits(rng, rows, vocab)
        for r in range(rows):
            at = rng.integers(0, vocab - k)
            v[r, at:at + k] += 100.0
        z = Rows(v, "f32")
        want = _top(ctx, z, k, 1.0)
        _check_top(want, z, k, 1.0)
        for _ in range(10):
            got = _top(ctx, z, k, 1.0)
            assert all(np.array_equal(a, b) for a, b in zip(got, want))


@pytest.mark.parametrize("rows,vocab", [(1200, 640), (500, 9001), (40, 50021)])
def test_every_row_has_the_gradients_of_its_own_list(ctx, rows, vocab):
    """Long lists with indices that come twice, another one for each of many rows that follow one another: all listed gradients of all rows."""
    rng = np.random.default_rng(rows)
    k = 256
    z = Rows(_logits(rng, rows, vocab), "f32")
    index = rng.integers(0, vocab, (rows, k)).astype(np.int32)
    index[::2] = np.argsort(rng.random((rows, vocab)), axis=1)[::2, :k]  # every second list without repetition
    t = np.log(rng.dirichlet(np.ones(k), rows) * rng.uniform(0.3, 1.0, (rows, 1)))
    for mode in ("tail", "renorm"):
        got = _distill(ctx, z, index, t, 1.0, mode, None, "f32")
        _check_distill(got, z, index, t, 1.0, mode, None, "f32")
        for _ in range(5):
            again = _distill(ctx, z, index, t, 1.0, mode, None, "f32")
            assert np.array_equal(again[0], got[0]) and np.array_equal(again[1], got[1])


@pytest.mark.parametrize("k", [2, 200])
@pytest.mark.parametrize("rows,vocab", [(23, 50021), (23, 1003), (400, 9000)])
@pytest.mark.parametrize("temperature", [1.0, 0.01, 1e-4, 1e4])
def test_top_logits_about_the_largest_exponents(ctx, temperature, rows, vocab, k):
    """z log2(e) / T about -2^22 and 2^22, on both sides of the border in one row: every element has its share of the sum."""
    rng = np.random.default_rng(rows)
    border = 2.0**22 * np.log(2.0) * temperature
    v = np.empty((rows, vocab))
    for r in range(rows):
        sign = -1.0 if r % 4 else 1.0
        v[r] = sign * border + temperature * (0.25 * (r % 23 - 11) + (rng.uniform(-2, 2, vocab) if r % 2 else 0.0))
        v[r, rng.integers(0, vocab)] += 0.5 * temperature
    z = Rows(v, "f32")
    _check_top(_top(ctx, z, k, temperature), z, k, temperature)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("shift", [-100, -600, 90, 600, -2000])
def test_renormalised_lists_of_any_magnitude(ctx, shift, dtype):
    """log-probabilities up to a constant are the same list, however small or large their exponentials are; a mass below 1e-300 is none."""
    rng = np.random.default_rng(5)
    vocab, k = 3001, 40
    z = Rows(_logits(rng, 6, vocab), dtype)
    index, t = _lists(rng, z, k, 1.0)
    t = np.round(t * 256) / 256  # so that the constant is added exactly
    index[1, 7:] = -1
    index[2, 1::2] = index[2, 0]
    t[3, 5:] = -np.inf
    index[4] = -1
    t[5] = -np.inf
    weight = rng.uniform(0.2, 1.5, 6)
    for out, factor in (("f32", False), ("f16", True)):
        got = _distill(ctx, z, index, t + shift, 1.3, "renorm", weight, out, factor=factor)
        if shift > -700:
            _check_distill(got, z, index, t, 1.3, "renorm", weight, out, factor=factor)
        empty = slice(4 if shift > -700 else 0, 6)
        assert (got[0][empty] == 0).all() and (got[1][empty] == 0).all()


def _steps(vocab):
    """A row that rises late: zeros in the first vectors of every CTA, then values some 2^10 times as likely, then one that leaves those at 2^-117."""
    v = np.zeros(vocab, np.float32)
    v[vocab // 2:] = 6.9
    v[-3] = 88.0
    return v


@pytest.mark.parametrize("rows,vocab", [(160, 2100), (160, 12000), (2, 65536)])
def test_softmax_of_rows_that_rise_late(ctx, rows, vocab):
    """Probabilities down to 2^-126 of the largest are there, wherever the largest lies."""
    z = Rows(np.tile(_steps(vocab), (rows, 1)), "f32")
    p = Rows(np.full((rows, vocab), np.nan), "f32")
    _before()
    ctx.check(rt.lib().rt_softmax_dev(ctx._h, z.ptr, 0, rows, vocab, vocab, 1.0, p.ptr, 0, vocab))
    _sync(ctx)
    _check_prob(p.read(), z, 1.0, "f32")


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("rows,vocab", [(160, 2100), (160, 12000), (2, 65536)])
def test_gradients_far_below_the_list(ctx, rows, vocab, dtype):
    """The student's mass lies on the list; outside of it probabilities down to 2^-126 of the largest are there."""
    z = np.tile(_steps(vocab), (rows, 1))
    z[:, -3] = 0.0
    z[::2, 77] = z[1::2, vocab - 100] = 88.0
    z = Rows(z, dtype)
    index = np.array([[77, 5], [vocab - 100, 5]] * (rows // 2), np.int32)
    t = np.log(np.array([[0.75, 0.25]] * rows))
    got = _distill(ctx, z, index, t, 1.0, "renorm", None, "f32")
    _check_distill(got, z, index, t, 1.0, "renorm", None, "f32")


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_a_number_that_is_not_below_one_gives_the_last_index(ctx, dtype):
    """However the running sums were rounded: masses whose sums are not exact, and next to nothing in the last place."""
    rng = np.random.default_rng(0)
    vocab, n = 16384, 300
    p = np.zeros((n, vocab))
    for r in range(n):
        at = rng.integers(0, vocab - 1000, 60)
        p[r, at] = rng.random(60)
        p[r, at + 1] = rng.random(60) * 2.0**-33
        p[r, vocab - 1 - r] = 1e-25
        p[r, vocab - r:] = 0
    P = Rows(p, dtype)
    want = [int(np.nonzero(row)[0][-1]) for row in P.f64]
    for u in (1.0, 2.0, np.inf, np.nan):
        acc, token = _verify(ctx, P, None, [], [0] * (n + 1), [], [u] * n)
        assert (acc == 0).all() and token.tolist() == want, u


def test_results_between_the_rows(ctx):
    """Rows and results may share an allocation as long as they share no bytes: halves of the same rows, or rows in turn."""
    import torch

    rng = np.random.default_rng(2)
    rows, vocab = 4, 1000
    v = _logits(rng, rows, vocab)
    z = Rows(v, "f32")
    index, t = _lists(rng, z, 9, 1.0)
    i, tl = _dev(index, torch.int32), _dev(t, torch.float32)
    L = rt.lib()
    store = torch.empty(rows * 2016 + 2016, device="cuda")
    left, right = store[:rows * 2016].view(rows, 2016), store[1008:1008 + rows * 2016].view(rows, 2016)

    def fresh():
        store.fill_(float("nan"))
        left[:, :vocab] = torch.as_tensor(v).cuda()
        _before()

    fresh()
    ctx.check(L.rt_softmax_dev(ctx._h, left.data_ptr(), 0, rows, vocab, 2016, 1.0, right.data_ptr(), 0, 2016))
    _sync(ctx)
    _check_prob(right[:, :vocab].double().cpu().numpy(), z, 1.0, "f32")
    assert np.array_equal(left[:, :vocab].cpu().numpy(), v) and bool(torch.isnan(left[:, vocab:1008]).all())
    fresh()
    loss = _empty((rows,))
    ctx.check(L.rt_distill_dev(ctx._h, left.data_ptr(), 0, rows, vocab, 2016, 1.0, i.data_ptr(), tl.data_ptr(), 9, 1, None, loss.data_ptr(),
                               right.data_ptr(), 0, 2016, None))
    _sync(ctx)
    _check_distill((loss.cpu().numpy().astype(np.float64), right[:, :vocab].double().cpu().numpy(), None, None), z, index, t, 1.0, "tail", None, "f32")
    # one element shared, in front or behind, is one too many
    b = store.data_ptr()
    for at in (vocab - 1, 2016 - vocab + 1):
        assert L.rt_softmax_dev(ctx._h, b, 0, rows, vocab, 2016, 1.0, b + 4 * at, 0, 2016) == 7
        assert L.rt_softmax_dev(ctx._h, b + 4 * at, 0, rows, vocab, 2016, 1.0, b, 0, 2016) == 7
    # 16-bit results of the same pitch, behind the row or one element too early
    assert L.rt_softmax_dev(ctx._h, b, 0, rows, vocab, 2016, 1.0, b + 4 * vocab, 2, 4032) == 0
    assert L.rt_softmax_dev(ctx._h, b, 0, rows, vocab, 2016, 1.0, b + 4 * vocab - 2, 2, 4032) == 7
    assert L.rt_softmax_dev(ctx._h, b, 0, rows, vocab, 2016, 1.0, b + 4 * vocab, 2, 4030) == 7  # another pitch
    _sync(ctx)


@pytest.mark.parametrize("mode", ["renorm", "tail"])
@pytest.mark.parametrize("vocab", [500, 50021])
def test_rows_beside_one_with_an_index_outside(ctx, vocab, mode):
    """What such a call leaves: the other rows' losses and gradients."""
    import torch

    rng = np.random.default_rng(13)
    rows, k = 7, 5
    z = Rows(_logits(rng, rows, vocab), "f32")
    index, t = _lists(rng, z, k, 1.0)
    tl = _dev(t, torch.float32)
    for bad in (vocab, -2, 2**31 - 1, -2**31):
        wrong = index.copy()
        wrong[3, 2] = bad
        i, loss, d = _dev(wrong, torch.int32), _empty((rows,)), Rows(np.full((rows, vocab), np.nan), "f32")
        _before()
        ctx.check(rt.lib().rt_distill_dev(ctx._h, z.ptr, 0, rows, vocab, vocab, 1.0, i.data_ptr(), tl.data_ptr(), k, ops.DISTILL_MODES[mode], None,
                                          loss.data_ptr(), d.ptr, 0, vocab, None))
        with pytest.raises(rt.RtError) as e:
            _sync(ctx)
        assert e.value.status == 6
        good = [r for r in range(rows) if r != 3]
        some = Rows(z.f64[good], "f32")
        _check_distill((loss.cpu().numpy().astype(np.float64)[good], d.read()[good], None, None), some, index[good], t[good], 1.0, mode, None, "f32")
        assert d.others_untouched()


@pytest.mark.parametrize("vocab", [300, 50021])
def test_sequences_beside_one_that_does_not_fit(ctx, vocab):
    """Such a sequence stands for nothing (0, -1); the others are what they are."""
    import torch

    rng = np.random.default_rng(3)
    off, p, q, tok, ua, us = _drafts(rng, (2, 3, 2, 1), vocab)
    P, Q = Rows(p, "f32"), Rows(q, "f32")
    a, s = _dev(ua, torch.float32), _dev(us, torch.float32)
    for change, bad in ((lambda t, o: t.__setitem__(3, vocab), [1]), (lambda t, o: t.__setitem__(4, -1), [1]), (lambda t, o: t.__setitem__(0, 2**31 - 1), [0]),
                        (lambda t, o: o.__setitem__(1, 6), [0, 1]), (lambda t, o: o.__setitem__(2, 9), [1, 2]), (lambda t, o: o.__setitem__(0, 1), [0]),
                        (lambda t, o: o.__setitem__(4, 7), [3]), (lambda t, o: o.__setitem__(1, -3), [0, 1]), (lambda t, o: o.__setitem__(4, 9), [3])):
        t, o = np.asarray(tok, np.int32).copy(), np.asarray(off, np.int32).copy()
        change(t, o)
        tk, of, acc, token = _dev(t), _dev(o), _empty((4,), torch.int32), _empty((4,), torch.int32)
        _before()
        ctx.check(rt.lib().rt_verify_draft_dev(ctx._h, P.ptr, vocab, Q.ptr, vocab, 0, vocab, tk.data_ptr(), of.data_ptr(), 4, len(tok), a.data_ptr(),
                                               s.data_ptr(), acc.data_ptr(), token.data_ptr()))
        with pytest.raises(rt.RtError) as e:
            _sync(ctx)
        assert e.value.status == 6
        acc, token = acc.cpu().numpy(), token.cpu().numpy()
        # a sequence whose offsets are in order among themselves is taken as they say; only those that are as they were have a known answer
        for i in range(4):
            if i in bad and (o[i] < 0 or o[i + 1] < o[i] or o[i + 1] > len(tok) or (i == 0 and o[0]) or (i == 3 and o[4] != len(tok)) or
                             not ((t[o[i]:o[i + 1]] >= 0) & (t[o[i]:o[i + 1]] < vocab)).all()):
                assert (int(acc[i]), int(token[i])) == (0, -1), i
            elif i not in bad:
                lo, hi = off[i], off[i + 1]
                assert (int(acc[i]), int(token[i])) == R.verify(P.f64[lo + i:hi + i + 1], Q.f64[lo:hi], tok[lo:hi], ua[lo:hi], us[i]), i


@pytest.mark.parametrize("temperature", [1e-4, 1e4])
@pytest.mark.parametrize("rows,vocab,dtype", [(5, 37, "f32"), (3, 50021, "f32"), (3, 50021, "bf16"), (300, 3001, "f16"), (300, 3001, "f32")])
def test_the_ends_of_the_temperature(ctx, rows, vocab, dtype, temperature):
    rng = np.random.default_rng(vocab)
    z = Rows(_logits(rng, rows, vocab), dtype, vocab + 3, 1)
    for k in (1, 30):
        _check_top(_top(ctx, z, k, temperature), z, k, temperature)
    some = min(rows, 12)
    index, t = _lists(rng, z, 12, temperature, 0.5)
    for mode in ("renorm", "tail"):
        ls, d, f, _ = _distill(ctx, z, index, t, temperature, mode, None, "f32")
        z.rows = some
        _check_distill((ls, d, f, None), z, index, t, temperature, mode, None, "f32")
        z.rows = rows


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("vocab", [4097, 4400, 8692, 12800, 16884, 20600])
def test_top_logits_of_rows_whose_last_unit_is_short(ctx, vocab, dtype):
    """The last unit of a row holds elements for a few warps only: such rows find their bound in the CTAs that have more."""
    rng = np.random.default_rng(vocab)
    for rows in (1, 16, 120):
        z = Rows(_logits(rng, rows, vocab), dtype, vocab + 3, 1)
        for k in (8, 64, 200):
            _check_top(_top(ctx, z, k, 1.0), z, k, 1.0)
