"""Top logits, softmax, distillation and verification of drafts on the device against their 64-bit forms (vocab_reference.py).

Tolerances, with u = 2^-24 (half a step of f32, relative).  An exponential exp(x), x = (z - m) / T <= 0: the difference, the
quotient and (where the kernel forms it) the product with log2 e are rounded, at most four times by u |x|, and the exponential
itself is off by at most 4 u; a sum of such terms adds at most 64 roundings (within a thread, its warp, and of the warps), and the
average of its terms' errors, at most 4 u times the mean |x| that the sum sees, which the factor 96 covers for |x| <= 8 where the mass is.
So p is off by (4 |x| + 96) u p, a log-probability or log-sum-exp by 96 u + 4 u |x| and its own rounding u |s|.  What is written is
rounded to its type: half a step, finfo.eps / 2 relative, or half of the smallest subnormal.  An exponential below 2^-126 is taken as 0
(2^x on the special-function unit, which knows no subnormal numbers): what it would have been is less than 2^-126, and every factor it meets
on its way to a probability or gradient is at most 1 (the reciprocal of a sum that holds the maximum's 1) or the weight.
"""
import numpy as np
import pytest

import rust_trainer_b200 as rt
import vocab_reference as R
from rust_trainer_b200 import ops

pytestmark = pytest.mark.gpu
U = 2.0 ** -24
FLUSHED = 2.0 ** -126
DT = {"f32": 0, "bf16": 1, "f16": 2}


def _types():
    import torch

    return {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}


def _half_step(dtype, value):
    import torch

    f = torch.finfo(_types()[dtype])
    return np.maximum(f.eps / 2 * np.abs(value), f.smallest_normal * f.eps / 2)


class Rows:
    """[rows x vocab] values on the device as the kernels may get them: rows `ld` apart, starting `offset` elements into an allocation
    that is NaN everywhere else."""

    def __init__(self, values, dtype, ld=None, offset=0):
        import torch

        v = torch.as_tensor(np.asarray(values, np.float32)).to(_types()[dtype])
        rows, vocab = v.shape
        self.ld, self.dtype, self.vocab, self.rows = ld or vocab, dtype, vocab, rows
        self.store = torch.full((offset + rows * self.ld + 8,), float("nan"), dtype=v.dtype, device="cuda")
        self.view = self.store[offset:offset + rows * self.ld].view(rows, self.ld)
        self.view[:, :vocab] = v.cuda()
        self.f64 = v.double().numpy()

    @property
    def ptr(self):
        return self.view.data_ptr()

    def read(self):
        return self.view[:, :self.vocab].double().cpu().numpy()

    def others_untouched(self):
        import torch

        keep = self.store.clone()
        at = (self.view.data_ptr() - self.store.data_ptr()) // self.store.element_size()
        keep[at:at + self.rows * self.ld].view(self.rows, self.ld)[:, :self.vocab] = float("nan")
        return bool(torch.isnan(keep).all())


def _empty(shape, dtype=None):
    import torch

    return torch.full(shape, -77 if dtype is not None else float("nan"), dtype=dtype or torch.float32, device="cuda")


def _dev(x, dtype=None):
    import torch

    return torch.as_tensor(np.ascontiguousarray(x), dtype=dtype).cuda()


def _sync(ctx):
    ctx.synchronize()


def _before():
    import torch

    torch.cuda.synchronize()


def _logits(rng, rows, vocab, spread=2.5):
    return (rng.standard_normal((rows, vocab)) * spread).astype(np.float32)


SHAPES = [  # rows, vocab, ld, offset
    (1, 1, 1, 0), (3, 2, 2, 1), (5, 7, 9, 3), (9, 640, 640, 0), (4, 1003, 1003, 0), (3, 4099, 4104, 5), (2, 50021, 50021, 1),
    (2, 151936, 151936, 0), (3, 128257, 128300, 7), (1, 262144, 262144, 0), (1, 393216, 393217, 1)]


# ------------------------------------------------------------------ top logits


def _top(ctx, z, k, temperature, lse=True):
    import torch

    index, logp, ls = _empty((z.rows, k), torch.int32), _empty((z.rows, k)), _empty((z.rows,))
    _before()
    ctx.check(rt.lib().rt_top_logits_dev(ctx._h, z.ptr, DT[z.dtype], z.rows, z.vocab, z.ld, temperature, k, index.data_ptr(), logp.data_ptr(),
                                         ls.data_ptr() if lse else None))
    _sync(ctx)
    return index.cpu().numpy(), logp.cpu().numpy().astype(np.float64), ls.cpu().numpy().astype(np.float64)


def _check_top(got, z, k, temperature):
    index, logp, ls = got
    for r in range(z.rows):
        wi, wp, wl = R.top(z.f64[r], k, temperature)
        assert np.array_equal(index[r], wi), r
        m = np.nanmax(z.f64[r])
        for g, w in list(zip(logp[r], wp)) + [(ls[r], wl)]:
            if np.isfinite(w):
                top = abs(m / temperature) if np.isfinite(m) else 0.0
                assert abs(g - w) <= (96 + 2 * top) * U + 5 * U * abs(w), (r, g, w)
            else:
                assert np.isnan(g) if np.isnan(w) else g == w, (r, g, w)


@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("rows,vocab,ld,offset", SHAPES)
def test_top_logits(ctx, rows, vocab, ld, offset, dtype):
    rng = np.random.default_rng(rows * 31 + vocab)
    z = Rows(_logits(rng, rows, vocab), dtype, ld, offset)
    for k, temperature in {(1, 1.0), (min(vocab, 8), 0.7), (min(vocab, 64), 2.0), (min(vocab, 256), 1.0)}:
        _check_top(_top(ctx, z, k, temperature), z, k, temperature)
    assert z.others_untouched()


ORDERS = {
    "ascending": lambda v, rng: np.arange(v) * 1e-3,
    "descending": lambda v, rng: -np.arange(v) * 1e-3,
    "constant": lambda v, rng: np.full(v, 1.25),
    "two values": lambda v, rng: rng.integers(0, 2, v) * 1.0,
    "few values": lambda v, rng: np.round(rng.standard_normal(v) * 3),
    "zeros of both signs": lambda v, rng: np.where(rng.random(v) < 0.5, 0.0, -0.0),
    "all masked but ten": lambda v, rng: np.where(np.arange(v) % (v // 10 + 1) == 3, rng.standard_normal(v), -np.inf),
    "masked with the lowest value": lambda v, rng: np.where(rng.random(v) < 0.999, -3.0e38, rng.standard_normal(v)),
    "nothing but -inf": lambda v, rng: np.full(v, -np.inf),
    "large in one stretch": lambda v, rng: rng.standard_normal(v) + 50.0 * (np.abs(np.arange(v) - v // 3) < 300),
    "large every 256 vectors": lambda v, rng: rng.standard_normal(v) + 50.0 * (np.arange(v) // 4 % 256 == 7),
    "large every 64": lambda v, rng: rng.standard_normal(v) + 50.0 * (np.arange(v) % 64 == 5),
    "steep": lambda v, rng: rng.standard_normal(v) * 300.0,
}


@pytest.mark.parametrize("vocab", [37, 1003, 20000, 151936])
@pytest.mark.parametrize("order", sorted(ORDERS))
def test_top_logits_of_every_order(ctx, order, vocab):
    rng = np.random.default_rng(vocab)
    for dtype in ("f32", "bf16"):
        z = Rows(np.stack([ORDERS[order](vocab, rng) for _ in range(2)]), dtype)
        for k in (1, min(vocab, 33), min(vocab, 256)):
            _check_top(_top(ctx, z, k, 1.0), z, k, 1.0)


@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("vocab", [33, 300, 655, 1000, 2049])
def test_top_logits_of_short_rows(ctx, vocab, dtype):
    """Fewer vectors than threads, lists longer than there are vectors, more elements than are ranked by counting."""
    rng = np.random.default_rng(vocab)
    for offset in (0, 3):
        z = Rows(_logits(rng, 5, vocab), dtype, vocab + offset, offset)
        for k in {1, 29, 64, 65, 128, 129, 250, vocab}:
            if k <= min(vocab, 256):
                _check_top(_top(ctx, z, k, 1.0), z, k, 1.0)


def test_top_logits_with_values_that_are_no_numbers(ctx):
    rng = np.random.default_rng(8)
    v = _logits(rng, 5, 5003)
    v[0, [17, 4000]] = np.nan
    v[1, 9] = np.inf
    v[2, 100:4900] = np.nan
    v[3, 5:] = -np.inf
    z = Rows(v, "f32")
    for k in (1, 3, 64, 256):
        _check_top(_top(ctx, z, k, 1.0), z, k, 1.0)
    index = _top(ctx, z, 4, 1.0, lse=False)[0]
    assert index[0, :2].tolist() == [17, 4000] and index[1, 0] == 9


# ------------------------------------------------------------------ softmax


def _check_prob(got, z, temperature, out):
    for r in range(z.rows):
        s = R.log_softmax(z.f64[r], temperature)
        want = np.exp(s)
        if np.isnan(want).any():
            assert np.isnan(got[r]).all(), r
            continue
        m = z.f64[r].max()
        x = np.where(np.isfinite(z.f64[r]), (m - np.where(np.isfinite(z.f64[r]), z.f64[r], 0)) / temperature, 0.0) if np.isfinite(m) else np.zeros_like(want)
        # where |x| > 80 the value is below any f32 and only has to be small
        tol = np.minimum((4 * np.minimum(x, 200) + 96) * U, 1.0) * want + _half_step(out, want) + FLUSHED
        assert (np.abs(got[r] - want) <= tol).all(), (r, np.abs(got[r] - want).max())


@pytest.mark.parametrize("dtype,out", [("f32", "f32"), ("f32", "bf16"), ("f32", "f16"), ("bf16", "bf16"), ("bf16", "f32"), ("f16", "f16"), ("f16", "f32"),
                                       ("bf16", "f16"), ("f16", "bf16")])
@pytest.mark.parametrize("rows,vocab,ld,offset", SHAPES)
def test_softmax(ctx, rows, vocab, ld, offset, dtype, out):
    rng = np.random.default_rng(rows * 31 + vocab)
    z = Rows(_logits(rng, rows, vocab), dtype, ld, offset)
    p = Rows(np.full((rows, vocab), np.nan), out, vocab + offset, offset // 2)
    for temperature in (1.0, 0.7):
        _before()
        ctx.check(rt.lib().rt_softmax_dev(ctx._h, z.ptr, DT[dtype], rows, vocab, z.ld, temperature, p.ptr, DT[out], p.ld))
        _sync(ctx)
        _check_prob(p.read(), z, temperature, out)
        assert p.others_untouched() and z.others_untouched()


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_softmax_of_odd_rows_in_their_own_place(ctx, dtype):
    rng = np.random.default_rng(3)
    v = _logits(rng, 9, 5003)
    v[0] = -np.inf
    v[1, 4:] = -np.inf
    v[2] = -3.0e38
    v[3] = np.where(rng.random(5003) < 0.5, -3.0e38, v[3])
    v[4, 100] = np.nan
    v[5, 0] = np.inf
    v[6] = 77.0
    v[7] *= 300.0
    for temperature in (1.0, 0.5, 1e-4, 1e4):
        z = Rows(v, dtype)
        _before()
        ctx.check(rt.lib().rt_softmax_dev(ctx._h, z.ptr, DT[dtype], 9, 5003, 5003, temperature, z.ptr, DT[dtype], 5003))
        _sync(ctx)
        got = z.read()
        assert (got[0] == 0).all()
        _check_prob(got, z, temperature, dtype)


# ------------------------------------------------------------------ distillation


def _distill(ctx, z, index, t, temperature, mode, weight=None, out=None, loss=True, factor=False, inplace=False, d_ld=None, d_offset=0):
    import torch

    k = index.shape[1]
    i, tl = _dev(index, torch.int32), _dev(t, torch.float32)
    w = None if weight is None else _dev(weight, torch.float32)
    ls, f = _empty((z.rows,)), _empty((z.rows,))
    d = z if inplace else Rows(np.full((z.rows, z.vocab), np.nan), out, d_ld, d_offset) if out else None
    _before()
    ctx.check(rt.lib().rt_distill_dev(ctx._h, z.ptr, DT[z.dtype], z.rows, z.vocab, z.ld, temperature, i.data_ptr(), tl.data_ptr(), k, ops.DISTILL_MODES[mode],
                                      None if w is None else w.data_ptr(), ls.data_ptr() if loss else None, d.ptr if d else None,
                                      DT[d.dtype] if d else 0, d.ld if d else 0, f.data_ptr() if factor else None))
    _sync(ctx)
    if d is not None:
        assert d.others_untouched()
    return ls.cpu().numpy().astype(np.float64), d.read() if d is not None else None, f.cpu().numpy().astype(np.float64), d


def _check_distill(got, z, index, t, temperature, mode, weight=None, out=None, loss=True, factor=False):
    ls, d, f, _ = got
    t = np.asarray(t, np.float32).astype(np.float64)
    for r in range(z.rows):
        w = 1.0 if weight is None else float(np.float32(weight[r]))
        want, grad, parts = R.distill(z.f64[r], index[r], t[r], temperature, mode, w)
        if loss:
            if not np.isfinite(want):
                assert np.isnan(ls[r]) if np.isnan(want) else ls[r] == want, (r, ls[r], want)
            else:
                # every s is off by at most 96 u + 4 u |x|, |x| <= 40 where it counts, and the q sum to one (or to their mass)
                mass = max(1.0, float(np.exp(t[r][np.asarray(index[r]) >= 0]).sum()))
                assert abs(ls[r] - want) <= abs(w) * mass * 256 * U + 2 * U * abs(want), (r, ls[r], want)
        if factor:
            assert abs(f[r] - w / temperature) <= 2 * U * abs(w / temperature)
        if d is None:
            continue
        g = 1.0 if factor else w / temperature
        if np.isnan(grad).any():
            assert np.isnan(d[r]).all(), r
            continue
        tol = _half_step(out, g * grad) + 3 * U * np.abs(g * grad)
        if parts is not None:
            p, q = parts
            m = z.f64[r].max()
            x = np.minimum(np.where(np.isfinite(z.f64[r]), (m - np.where(np.isfinite(z.f64[r]), z.f64[r], 0)) / temperature, 0.0), 200.0)
            # outside of the list the gradient is the difference of p and r p / R, both as far off as p is (R's own sum: twice)
            tol = tol + abs(g) * ((4 * x + 192) * U * (p + np.abs(grad - p)) + 8 * U * np.abs(q))
        assert (np.abs(d[r] - g * grad) <= tol + 2 * max(1.0, abs(g)) * FLUSHED).all(), (r, np.abs(d[r] - g * grad).max(), np.argmax(np.abs(d[r] - g * grad) - tol))


def _lists(rng, z, k, temperature, noise=1.0):
    """A teacher's lists: its logits are the student's with noise."""
    index, t = [], []
    for row in z.f64:
        teacher = row + noise * rng.standard_normal(row.size)
        i, s, _ = R.top(teacher, min(k, row.size), temperature)
        index.append(np.concatenate([i, np.full(k - i.size, -1)]))
        t.append(np.concatenate([s, np.zeros(k - i.size)]))
    return np.array(index, np.int32), np.array(t, np.float32)


@pytest.mark.parametrize("mode", ["renorm", "tail"])
@pytest.mark.parametrize("dtype,out", [("f32", "f32"), ("f32", "f16"), ("bf16", "bf16"), ("f16", "f32"), ("f16", "f16"), ("bf16", "f16"), ("f32", "bf16"),
                                       ("f16", "bf16"), ("bf16", "f32")])
@pytest.mark.parametrize("rows,vocab,ld,offset", SHAPES)
def test_distill(ctx, rows, vocab, ld, offset, dtype, out, mode):
    rng = np.random.default_rng(rows * 31 + vocab)
    z = Rows(_logits(rng, rows, vocab), dtype, ld, offset)
    weight = rng.uniform(0.2, 1.5, rows)
    for k, temperature in ((1, 1.0), (17, 2.0), (256, 0.7)):
        index, t = _lists(rng, z, k, temperature)
        factor = out == "f16"
        got = _distill(ctx, z, index, t, temperature, mode, weight, out, factor=factor, d_ld=vocab + offset, d_offset=offset // 2)
        _check_distill(got, z, index, t, temperature, mode, weight, out, factor=factor)
    assert z.others_untouched()


@pytest.mark.parametrize("mode", ["renorm", "tail"])
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_distill_odd_rows(ctx, mode, dtype):
    """Lists with places left empty, an index twice, all of the mass or none of it, more than all; students that are masked, far off,
    or no numbers; rows of no weight."""
    rng = np.random.default_rng(11)
    v, k = 3001, 20
    x = _logits(rng, 16, v)
    z0 = Rows(x, dtype)
    index, t = _lists(rng, z0, k, 1.0)
    weight = np.ones(16)
    index[0] = -1                                   # nothing listed
    index[1, 3:] = -1
    index[2, 1::2] = index[2, 0]                    # eleven entries of one index
    t[3] = -np.inf                                  # a list without mass
    t[4] = np.log(0.25)                             # more than all of the mass
    x[5] = -np.inf                                  # a student that can say nothing
    x[6, index[6, 0]] = -np.inf                     # nor what the teacher says
    x[7] -= 200.0 * np.isin(np.arange(v), index[7], invert=True)  # its rest is beyond any f32 exponential
    x[8, 5] = np.nan
    x[9, 7] = np.inf
    weight[10], x[10] = 0.0, np.nan                 # a row that nobody asks for
    x[11] = -3.0e38
    x[12, np.isin(np.arange(v), index[12], invert=True)] = -np.inf  # the student has no rest
    weight[13] = -0.5
    index[14, 5:] = -1
    t[14, :5] = np.log([0.9, 0.1, 1e-9, 1e-9, 1e-9])
    x[15, index[15, 2]] = np.nan
    for out, factor in (("f32", False), ("f16", True)):
        z = Rows(x, dtype)
        got = _distill(ctx, z, index, t, 1.0, mode, weight, out, factor=factor)
        _check_distill(got, z, index, t, 1.0, mode, weight, out, factor=factor)
        assert got[0][10] == 0 and (got[1][10] == 0).all()


@pytest.mark.parametrize("mode", ["renorm", "tail"])
def test_distill_over_the_whole_vocabulary(ctx, mode):
    rng = np.random.default_rng(12)
    z = Rows(_logits(rng, 3, 200), "f32")
    index, t = _lists(rng, z, 256, 1.0)
    _check_distill(_distill(ctx, z, index, t, 1.0, mode, None, "f32"), z, index, t, 1.0, mode, None, "f32")


@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("vocab", [640, 50021, 151936])
def test_distill_alone_and_in_place(ctx, dtype, vocab):
    """The loss alone, the gradient alone, and the gradient over the logits are what one call gives for both."""
    rng = np.random.default_rng(vocab)
    x = _logits(rng, 3, vocab)
    z = Rows(x, dtype)
    index, t = _lists(rng, z, 32, 1.0)
    both = _distill(ctx, z, index, t, 1.0, "tail", None, dtype)
    assert np.array_equal(_distill(ctx, z, index, t, 1.0, "tail")[0], both[0])
    assert np.array_equal(_distill(ctx, z, index, t, 1.0, "tail", None, dtype, loss=False)[1], both[1])
    over = _distill(ctx, z, index, t, 1.0, "tail", inplace=True)
    assert np.array_equal(over[0], both[0]) and np.array_equal(over[1], both[1])


def test_a_list_with_an_index_outside_is_reported_and_spoils_no_other_row(ctx):
    rng = np.random.default_rng(13)
    z = Rows(_logits(rng, 3, 500), "f32")
    index, t = _lists(rng, z, 5, 1.0)
    for bad in (500, -2, 2**31 - 1, -2**31):
        wrong = index.copy()
        wrong[1, 2] = bad
        with pytest.raises(rt.RtError) as e:
            _distill(ctx, z, wrong, t, 1.0, "tail", None, "f32")
        assert e.value.status == 6
    _check_distill(_distill(ctx, z, index, t, 1.0, "tail", None, "f32"), z, index, t, 1.0, "tail", None, "f32")  # the context goes on


# ------------------------------------------------------------------ verification


def _verify(ctx, p, q, tok, off, ua, us):
    import torch

    n_seq = len(off) - 1
    tk, of = _dev(np.asarray(tok, np.int32), torch.int32), _dev(np.asarray(off, np.int32), torch.int32)
    a, s = _dev(np.asarray(ua, np.float32), torch.float32), _dev(np.asarray(us, np.float32), torch.float32)
    acc, token = _empty((n_seq,), torch.int32), _empty((n_seq,), torch.int32)
    _before()
    ctx.check(rt.lib().rt_verify_draft_dev(ctx._h, p.ptr, p.ld, q.ptr if q else None, q.ld if q else 0, DT[p.dtype], p.vocab, tk.data_ptr(), of.data_ptr(),
                                           n_seq, len(tok), a.data_ptr(), s.data_ptr(), acc.data_ptr(), token.data_ptr()))
    _sync(ctx)
    return acc.cpu().numpy(), token.cpu().numpy()


def _check_verify(got, p, q, tok, off, ua, us):
    ua, us = np.asarray(ua, np.float32), np.asarray(us, np.float32)
    for s in range(len(off) - 1):
        a, e = off[s], off[s + 1]
        want = R.verify(p.f64[a + s:e + s + 1], None if q is None else q.f64[a:e], tok[a:e], ua[a:e], us[s])
        assert (int(got[0][s]), int(got[1][s])) == want, s


def _soft(x):
    e = np.exp(x - x.max(1, keepdims=True))
    return e / e.sum(1, keepdims=True)


def _drafts(rng, counts, vocab, noise=0.7):
    off = np.concatenate([[0], np.cumsum(counts)]).astype(int)
    n, n_seq = int(off[-1]), len(counts)
    z = _logits(rng, n + n_seq, vocab)
    at = [off[s] + s + i for s in range(n_seq) for i in range(counts[s])]
    p = _soft(z)
    q = _soft(z[at] + noise * rng.standard_normal((n, vocab))) if n else np.zeros((0, vocab))
    tok = np.array([np.searchsorted(np.cumsum(row), u * row.sum()) for row, u in zip(q, rng.random(n))], int).clip(0, vocab - 1)
    return off, p, q, tok, rng.random(n).astype(np.float32), rng.random(n_seq).astype(np.float32)


@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("counts,vocab,ld,offset", [((0,), 1, 1, 0), ((1, 0, 2), 2, 3, 1), ((3, 3, 0, 5), 7, 7, 0), ((4,) * 9, 640, 640, 0),
                                                    ((2, 7, 1, 0, 3), 1003, 1003, 3), ((4, 600, 1), 129, 129, 0), ((5, 4), 50021, 50027, 2),
                                                    ((4, 4), 151936, 151936, 0), ((1, 0), 393216, 393216, 0)])
@pytest.mark.parametrize("certain", [False, True])
def test_verify_draft(ctx, counts, vocab, ld, offset, dtype, certain):
    rng = np.random.default_rng(vocab)
    off, p, q, tok, ua, us = _drafts(rng, counts, vocab)
    P = Rows(p, dtype, ld, offset)
    Q = None if certain or not len(tok) else Rows(q, dtype, ld + 3, offset + 1)
    for trial in range(3):
        _check_verify(_verify(ctx, P, Q, tok, off, ua, us), P, Q, tok, off, ua, us)
        ua, us = rng.random(ua.size).astype(np.float32), rng.random(us.size).astype(np.float32)


def test_verify_draft_at_its_borders(ctx):
    """Numbers of exactly 0, the largest below 1 and beyond; drafts that are exactly as likely; masses in the first and the last place only."""
    vocab, one = 4000, np.float32(1 - 2.0**-24)
    p = np.zeros((12, vocab))
    q = np.zeros((8, vocab))
    p[0, 17] = q[0, 17] = 1.0                       # as likely: stands for any number below 1
    p[1, 0], p[1, -1] = 0.5, 0.5
    p[2, 5], q[1, 5], p[2, 9], q[1, 9] = 0.25, 0.5, 0.75, 0.5
    p[3] = 1.0 / vocab
    p[4, 5], q[2, 5] = 0.25, 0.25                   # u q < p with u = 1 - 2^-24
    p[5, 3] = 1.0
    q[3, 8], p[6, 2] = 1.0, 1.0                     # impossible for the target
    p[7, 1] = 1.0
    p[8], q[4] = 0.0, 0.0                           # nobody has any mass: not even the draft
    p[9, 1] = 1.0
    p[10, 6], q[5, 6], p[10, 7] = 0.5, 1.0, -0.25   # numbers that are no probabilities count as none
    p[10, 8], p[10, 9] = np.nan, np.inf
    p[11, vocab - 1] = 1e-30
    off = [0, 1, 2, 3, 4, 5, 6]
    tok = [17, 5, 5, 8, 3, 6]
    P, Q = Rows(p, "f32"), Rows(q[:6], "f32")
    for ua in ([one] * 6, [0.0] * 6, [0.5] * 6, [1.0] * 6, [0.4999999] * 6):
        for us in ([0.0] * 6, [one] * 6, [0.5] * 6, [1.0] * 6, [0.49999997] * 6, [2.0] * 6):
            ua, us = np.asarray(ua, np.float32), np.asarray(us, np.float32)
            _check_verify(_verify(ctx, P, Q, tok, off, ua, us), P, Q, tok, off, ua, us)
            _check_verify(_verify(ctx, P, None, tok, off, ua, us), P, None, tok, off, ua, us)


def test_even_probabilities_meet_the_border_exactly(ctx):
    """2^10 probabilities of 2^-10: a number of i 2^-10 falls on a border, and belongs to what lies behind it."""
    p = Rows(np.full((64, 1024), 2.0**-10), "bf16")
    us = np.arange(64, dtype=np.float32) * np.float32(2.0**-10) * 16
    acc, token = _verify(ctx, p, None, [], list(range(0, 1)) * 65, [], us)
    assert (acc == 0).all() and np.array_equal(token, np.arange(64) * 16)


def test_drafts_that_do_not_fit_are_reported(ctx):
    rng = np.random.default_rng(3)
    off, p, q, tok, ua, us = _drafts(rng, (2, 2, 2), 300)
    P, Q = Rows(p, "f32"), Rows(q, "f32")
    for change in (lambda t, o: t.__setitem__(2, 300), lambda t, o: t.__setitem__(2, -1), lambda t, o: o.__setitem__(1, 5), lambda t, o: o.__setitem__(2, 7),
                   lambda t, o: o.__setitem__(0, 1), lambda t, o: o.__setitem__(3, 5), lambda t, o: o.__setitem__(1, -3)):
        t, o = tok.copy(), off.copy()
        change(t, o)
        with pytest.raises(rt.RtError) as e:
            _verify(ctx, P, Q, t, o, ua, us)
        assert e.value.status == 6
    _check_verify(_verify(ctx, P, Q, tok, off, ua, us), P, Q, tok, off, ua, us)


# ------------------------------------------------------------------ hosts


def test_host_forms_are_the_device_forms(ctx):
    rng = np.random.default_rng(21)
    v = _logits(rng, 4, 1003)
    z = Rows(v, "f32")
    index, logp, lse = ops.top_logits(ctx, v, 12, 1.5)
    dev = _top(ctx, z, 12, 1.5)
    assert np.array_equal(index, dev[0]) and np.array_equal(logp, dev[1].astype(np.float32)) and np.array_equal(lse, dev[2].astype(np.float32))
    w = rng.uniform(0.5, 1, 4).astype(np.float32)
    for mode in ops.DISTILL_MODES:
        got = ops.distill(ctx, v, index, logp, w, 1.5, mode, want_dlogits=True)
        want = _distill(ctx, z, index, logp, 1.5, mode, w, "f32")
        assert np.array_equal(got["loss"], want[0].astype(np.float32)) and np.array_equal(got["dlogits"], want[1].astype(np.float32))
        assert np.array_equal(ops.distill(ctx, v, index, logp, w, 1.5, mode)["loss"], got["loss"])
    _check_prob(ops.softmax(ctx, v, 0.8).astype(np.float64), z, 0.8, "f32")
    off, p, q, tok, ua, us = _drafts(rng, (3, 0, 2), 700)
    P, Q = Rows(p, "f32"), Rows(q, "f32")
    _check_verify(ops.verify_draft(ctx, p, q, tok, off, ua, us), P, Q, tok, off, ua, us)
    _check_verify(ops.verify_draft(ctx, p, None, tok, off, ua, us), P, None, tok, off, ua, us)
    assert ops.top_logits(ctx, v[:0], 3)[0].shape == (0, 3) and ops.softmax(ctx, v[:0]).shape == (0, 1003)


class Picked:
    """Some rows of a call, for the checks."""

    def __init__(self, z, at):
        self.f64, self.rows, self.vocab, self.dtype = z.f64[at], len(at), z.vocab, z.dtype


@pytest.mark.parametrize("rows,vocab,dtype", [(2600, 640, "f32"), (2600, 1003, "bf16"), (1500, 7000, "f32"), (1300, 9001, "f16"), (450, 50021, "f32"),
                                              (700, 50021, "bf16"), (130, 151936, "f32")])
def test_many_rows_follow_one_another(ctx, rows, vocab, dtype):
    """Several rows for each cluster, of which none may find what another one left: steep, even, masked and far-off ones, ones that are no numbers and ones of
    no weight, in turn."""
    rng = np.random.default_rng(rows + vocab)
    v = _logits(rng, rows, vocab)
    v[1::7] *= 30
    v[2::7] = 1.5
    v[3::7, vocab // 3:] = -np.inf
    v[4::7] += 4096
    v[5::21, vocab // 2] = np.nan
    v[6::21] = -np.inf
    z = Rows(v, dtype, vocab + 3, 1)
    k = 40
    index = rng.integers(0, vocab, (rows, k)).astype(np.int32)
    index[::5, 30:] = -1
    t = np.log(rng.dirichlet(np.ones(k), rows) * rng.uniform(0.3, 1.0, (rows, 1)))
    weight = rng.uniform(0.2, 1.5, rows)
    weight[::9] = 0
    at = np.unique(np.concatenate([np.arange(0, rows, max(1, rows * vocab // 1500000)), np.arange(rows - 30, rows)]))
    some = Picked(z, at)
    for mode in ("tail", "renorm"):
        for out in (dtype, None):
            ls, d, f, _ = _distill(ctx, z, index, t, 1.0, mode, weight, out)
            _check_distill((ls[at], None if d is None else d[at], f[at], None), some, index[at], t[at], 1.0, mode, weight[at], out)
    p = Rows(np.full((rows, vocab), np.nan), "f32")
    _before()
    ctx.check(rt.lib().rt_softmax_dev(ctx._h, z.ptr, DT[dtype], rows, vocab, z.ld, 1.0, p.ptr, 0, p.ld))
    _sync(ctx)
    _check_prob(p.read()[at], some, 1.0, "f32")
    at = at[~np.isnan(some.f64).any(1)]  # (their order takes long to find in 64 bits)
    for top in (9, 100):
        _check_top([x[at] for x in _top(ctx, z, top, 1.0)], Picked(z, at), top, 1.0)
    assert z.others_untouched()


@pytest.mark.parametrize("vocab", [640, 50021])
def test_a_teacher_that_is_no_number_reaches_its_row_only(ctx, vocab):
    """A NaN among a row's log-probabilities: with a renormalised list no entry's probability is known, with the rest as a bucket the rest's and
    the entry's own are not."""
    rng = np.random.default_rng(3)
    z = Rows(_logits(rng, 3, vocab), "f32")
    index = np.stack([rng.permutation(vocab)[:6] for _ in range(3)]).astype(np.int32)
    t = np.log(np.full((3, 6), 0.1))
    t[1, 2] = np.nan
    for mode in ("tail", "renorm"):
        loss, d = _distill(ctx, z, index, t, 1.0, mode, out="f32")[:2]
        assert np.isfinite(loss[[0, 2]]).all() and np.isnan(loss[1])
        unknown = np.isin(np.arange(vocab), index[1]) == (mode == "renorm")
        unknown[index[1, 2]] = True
        assert np.isfinite(d[[0, 2]]).all() and np.array_equal(np.isnan(d[1]), unknown)


def test_refusals(ctx):
    """Every argument that does not fit is refused before anything is launched."""
    import torch

    L, h = rt.lib(), ctx._h
    buf = torch.zeros(1 << 16, device="cuda")
    b, i = buf.data_ptr(), torch.zeros(64, dtype=torch.int32, device="cuda").data_ptr()
    before = L.rt_ctx_launch_count(h)

    def top(z=b, dt=0, rows=2, v=100, ld=100, t=1.0, k=4, idx=i, lp=b + 4096):
        return L.rt_top_logits_dev(h, z, dt, rows, v, ld, t, k, idx, lp, None)

    def dist(z=b, dt=0, rows=2, v=100, ld=100, t=1.0, idx=i, te=b + 4096, k=4, mode=0, w=None, loss=b + 8192, d=b + 16384, ddt=0, dld=100, f=None):
        return L.rt_distill_dev(h, z, dt, rows, v, ld, t, idx, te, k, mode, w, loss, d, ddt, dld, f)

    def soft(z=b, dt=0, rows=2, v=100, ld=100, t=1.0, p=b + 16384, pdt=0, pld=100):
        return L.rt_softmax_dev(h, z, dt, rows, v, ld, t, p, pdt, pld)

    def ver(p=b, pl=100, q=b + 16384, ql=100, dt=0, v=100, tok=i, off=i, n=1, nd=1, ua=b, us=b, acc=i, out=i):
        return L.rt_verify_draft_dev(h, p, pl, q, ql, dt, v, tok, off, n, nd, ua, us, acc, out)

    nan = float("nan")
    for f in (top, dist, soft):
        assert f(z=None) == 7 and f(dt=3) == 7 and f(dt=-1) == 7 and f(v=0) == 1 and f(v=393217, ld=393217) == 1 and f(ld=99) == 1
        assert f(rows=(1 << 24) + 1) == 1 and f(z=b + 2) == 7 and f(z=b + 1, dt=1) == 7
        for t in (0.0, -1.0, nan, float("inf"), 1e-5, 1e5):
            assert f(t=t) == 7
        assert f(rows=0) == 0
    assert top(k=0) == 1 and top(k=257, v=1000, ld=1000) == 1 and top(k=101) == 1 and top(idx=None) == 7 and top(lp=None) == 7 and top(lp=b + 2) == 7
    assert dist(k=0) == 1 and dist(k=257) == 1 and dist(mode=2) == 7 and dist(idx=None) == 7 and dist(te=None) == 7 and dist(loss=None, d=None) == 7
    assert dist(ddt=5) == 7 and dist(dld=99) == 1 and dist(d=b + 400) == 7 and dist(d=b, ddt=1) == 7 and dist(d=b, dld=104) == 7 and dist(w=b + 1) == 7
    assert dist(d=None, f=b) == 7 and dist(d=b - 400 + 4, z=b + 400) == 7
    assert soft(p=None) == 7 and soft(pdt=9) == 7 and soft(pld=50) == 1 and soft(p=b + 40) == 7 and soft(p=b, pdt=2) == 7
    assert ver(p=None) == 7 and ver(off=None) == 7 and ver(us=None) == 7 and ver(acc=None) == 7 and ver(out=None) == 7 and ver(tok=None) == 7 and ver(ua=None) == 7
    assert ver(pl=99) == 1 and ver(ql=99) == 1 and ver(dt=4) == 7 and ver(v=0) == 1 and ver(n=0) == 1 and ver(n=0, nd=0) == 0 and ver(us=b + 2) == 7
    assert ver(n=(1 << 24) + 1) == 1 and ver(nd=(1 << 24) + 1) == 1
    assert L.rt_ctx_launch_count(h) == before
    with pytest.raises(rt.RtError):
        ops.verify_draft(ctx, np.zeros((4, 5), np.float32), None, [1, 2, 3], [0, 4, 3][:2], [0.1] * 3, [0.5])
    st = L.rt_op_verify_draft(h, None, None, 5, None, None, 1, None, None, None, None)
    assert st == 7
    ctx.synchronize()


def test_offsets_past_32_bits(ctx):
    """The last rows of a matrix of more than 2^31 elements."""
    import torch

    vocab, ld, rows = 1001, 1 << 20, 2100
    store = torch.zeros(rows * ld, dtype=torch.bfloat16, device="cuda")
    z = store.view(rows, ld)
    rng = np.random.default_rng(1)
    v = torch.as_tensor(_logits(rng, rows, vocab)).to(torch.bfloat16)
    z[:, :vocab] = v.cuda()
    index, logp = _empty((rows, 5), torch.int32), _empty((rows, 5))
    loss = _empty((rows,))
    _before()
    L = rt.lib()
    ctx.check(L.rt_top_logits_dev(ctx._h, z.data_ptr(), 1, rows, vocab, ld, 1.0, 5, index.data_ptr(), logp.data_ptr(), None))
    ctx.check(L.rt_distill_dev(ctx._h, z.data_ptr(), 1, rows, vocab, ld, 1.0, index.data_ptr(), logp.data_ptr(), 5, 1, None, loss.data_ptr(), z.data_ptr(), 1,
                               ld, None))
    _sync(ctx)
    last = v[-1].double().numpy()
    wi, wp, _ = R.top(last, 5, 1.0)
    assert np.array_equal(index[-1].cpu().numpy(), wi) and np.abs(logp[-1].cpu().numpy() - wp).max() < 200 * U
    _, grad, _ = R.distill(last, wi, logp[-1].cpu().numpy(), 1.0, "tail")
    assert abs(float(loss[-1])) <= 256 * U
    assert np.abs(z[-1, :vocab].double().cpu().numpy() - grad).max() <= 256 * U
    assert float(z[-1, vocab:].abs().max()) == 0
    p = z.zero_()
    p[-1, :vocab] = torch.as_tensor(_soft(last[None])[0]).to(torch.bfloat16).cuda()
    off = torch.zeros(rows + 1, dtype=torch.int32, device="cuda")
    us = torch.full((rows,), 0.6, device="cuda")
    acc, token = _empty((rows,), torch.int32), _empty((rows,), torch.int32)
    _before()
    ctx.check(L.rt_verify_draft_dev(ctx._h, p.data_ptr(), ld, None, 0, 1, vocab, None, off.data_ptr(), rows, 0, None, us.data_ptr(), acc.data_ptr(), token.data_ptr()))
    _sync(ctx)
    want = R.verify(p[-1:, :vocab].double().cpu().numpy(), None, [], [], np.float32(0.6))
    assert (int(acc[-1]), int(token[-1])) == want and int(token[0]) == -1


def test_captured_and_replayed_and_beside_another_context(ctx):
    """The four calls as a graph on a stream of the host's own, replayed over new inputs, while another context runs them on its stream."""
    import torch

    rng = np.random.default_rng(4)
    rows, vocab, k = 3, 151936, 16
    values = [_logits(rng, rows, vocab) for _ in range(3)]
    z = torch.as_tensor(values[0]).cuda()
    other = rt.Context(0)

    def buffers():
        return dict(index=_empty((rows, k), torch.int32), logp=_empty((rows, k)), loss=_empty((rows,)), d=_empty((rows, vocab)), p=_empty((rows, vocab)),
                    acc=_empty((1,), torch.int32), token=_empty((1,), torch.int32))

    tok, off = _dev(np.array([5, 9]), torch.int32), _dev(np.array([0, 2]), torch.int32)
    u = _dev(np.array([0.2, 0.4, 0.6]), torch.float32)

    def calls(c, z, b):
        L, h = rt.lib(), c._h
        c.check(L.rt_top_logits_dev(h, z.data_ptr(), 0, rows, vocab, vocab, 1.0, k, b["index"].data_ptr(), b["logp"].data_ptr(), None))
        c.check(L.rt_distill_dev(h, z.data_ptr(), 0, rows, vocab, vocab, 2.0, b["index"].data_ptr(), b["logp"].data_ptr(), k, 1, None, b["loss"].data_ptr(),
                                 b["d"].data_ptr(), 0, vocab, None))
        c.check(L.rt_softmax_dev(h, z.data_ptr(), 0, rows, vocab, vocab, 1.0, b["p"].data_ptr(), 0, vocab))
        c.check(L.rt_verify_draft_dev(h, b["p"].data_ptr(), vocab, None, 0, 0, vocab, tok.data_ptr(), off.data_ptr(), 1, 2, u.data_ptr(), u[2:].data_ptr(),
                                      b["acc"].data_ptr(), b["token"].data_ptr()))

    want = []
    for v in values:
        b = buffers()
        zz = torch.as_tensor(v).cuda()
        _before()
        calls(ctx, zz, b)
        _sync(ctx)
        want.append({n: x.cpu().numpy().copy() for n, x in b.items()})
    stream = torch.cuda.Stream()
    mine, b, b2 = rt.Context(0), buffers(), buffers()
    mine.check(rt.lib().rt_ctx_set_stream(mine._h, stream.cuda_stream))
    graph = torch.cuda.CUDAGraph()
    _before()
    with torch.cuda.graph(graph, stream=stream):
        calls(mine, z, b)
    z2 = torch.as_tensor(values[2]).cuda()
    for v, w in zip(values, want):
        z.copy_(torch.as_tensor(v))
        _before()
        graph.replay()
        for _ in range(3):
            calls(other, z2, b2)
        _before()
        for n in w:
            assert np.array_equal(b[n].cpu().numpy(), w[n]), n
            assert np.array_equal(b2[n].cpu().numpy(), want[2][n]), n
    mine.synchronize()
    other.synchronize()
    mine.close()
    other.close()
