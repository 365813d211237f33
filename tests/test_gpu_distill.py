"""A teacher's top logits, distillation and the check of drafts through whole models.

Gradients: a logit gradient g of sum 0 is a sum of scored targets, sum_v c_v (p - onehot_v) with c = -g, so that `forward_backward` with
every token of the vocabulary as a target of the same position gives the gradient that any distillation loss has to have; both sides
round their logit gradients to f16 rows, so the bar is that of the other objectives (relative L2 1e-2, cosine 0.999).  Losses: the
logits are the same f32 numbers on both sides, so they agree as the row operation does, to 256 * 2^-24 of the weight.
"""
import numpy as np
import pytest

import rust_trainer_b200 as rt
import vocab_reference as R
from conftest import cosine, rel_l2
from rust_trainer_b200 import evalgate, packing, synth
from rust_trainer_b200 import objectives as obj
from test_gpu_model import _gpu_flat, _setup

pytestmark = pytest.mark.gpu
U = 2.0 ** -24


def _model(ctx, preset="tiny-qwen3", quant="Q8_0", seed=0, **kw):
    spec = synth.preset(preset, quant=quant, seed=seed, w_std=0.08)
    m = rt.Model(ctx, spec.config(), synth.build_tensors(spec), **kw)
    m.attach_lora(8, 16.0, None, 5)
    m.load_adapters(synth.lora_adapters(spec, 8, 16.0, seed=seed + 2, b_std=0.02))
    return spec, m


def _seqs(spec, lens, seed=3):
    toks = synth.token_batch(spec, len(lens), max(lens), seed)
    return [toks[i][:n] for i, n in enumerate(lens)]


def _logits(m, seqs, pos):
    return m.score(seqs, pos, np.zeros(len(pos), np.int32), want_logits=True)[2].copy()


@pytest.mark.parametrize("preset", ["tiny-qwen3", "tiny-qwen2", "tiny-llama"])
def test_top_logits_are_those_of_the_rows(ctx, preset):
    spec, m = _model(ctx, preset)
    seqs = _seqs(spec, [40, 17, 1])
    pos = np.array([0, 5, 39, 41, 56, 57, 5], np.int32)
    z = _logits(m, seqs, pos)
    for k, t in ((1, 1.0), (64, 2.0), (256, 0.7)):
        index, logp, lse = m.top_logits(seqs, pos, k, t)
        for r in range(len(pos)):
            wi, wp, wl = R.top(z[r], k, t)
            assert np.array_equal(index[r], wi)
            assert np.abs(logp[r] - wp).max() <= 256 * U and abs(lse[r] - wl) <= 256 * U
    m.close()


def test_top_logits_of_packed_groups_and_in_chunks(ctx):
    spec, m = _model(ctx)
    rng = np.random.default_rng(0)
    prompt = rng.integers(0, spec.vocab, 30)
    seqs = [np.concatenate([prompt, [i], rng.integers(0, spec.vocab, 9 + i)]).astype(np.int32) for i in range(3)]
    g = packing.pack(seqs)
    at = np.array([g.index(k, p) for k in range(3) for p in (10, 32, 38)], np.int32)
    index, logp, _ = m.top_logits(None, at, 12, groups=[g])
    plain = m.top_logits(seqs, [sum(s.size for s in seqs[:k]) + p for k in range(3) for p in (10, 32, 38)], 12)
    assert (index == plain[0]).mean() > 0.9 and np.abs(logp - plain[1]).max() < 2e-2  # the same rows through other tiles, in f16
    _, small = _model(ctx, head_rows=4)
    assert np.array_equal(small.top_logits(None, at, 12, groups=[g])[0], index)
    m.close()
    small.close()


def _through_targets(m, seqs, pos, grads):
    """The adapter gradients that logit gradients of sum 0 have."""
    v = grads.shape[1]
    m.zero_grad()
    m.forward_backward(seqs, np.repeat(pos, v), np.tile(np.arange(v), len(pos)), -grads.ravel())
    return _gpu_flat(m, "ga", "gb")


@pytest.mark.parametrize("mode", ["renorm", "tail"])
@pytest.mark.parametrize("preset,t", [("tiny-qwen3", 1.0), ("tiny-qwen2", 2.0), ("tiny-llama", 0.7)])
def test_distillation_gradient(ctx, preset, t, mode):
    spec, student = _model(ctx, preset)
    _, teacher = _model(ctx, preset, seed=9)
    seqs, pos = _seqs(spec, [30, 21]), np.array([3, 20, 29, 35, 50], np.int32)
    w = np.array([0.2, 0.1, 0.3, 0.0, 0.4], np.float32)
    index, tl, _ = teacher.top_logits(seqs, pos, 20, t)
    index[1, 7:] = -1      # lists are shorter than k
    index[2, 3] = index[2, 0]  # or say something twice
    z = _logits(student, seqs, pos)
    student.zero_grad()
    loss = student.distill_backward(seqs, pos, index, tl, w, t, mode)
    got = _gpu_flat(student, "ga", "gb")
    want = [R.distill(z[r], index[r], tl[r], t, mode, float(w[r])) for r in range(len(pos))]
    assert np.abs(loss - [x[0] for x in want]).max() <= 256 * U
    rows = np.array([float(w[r]) / t * want[r][1] for r in range(len(pos))])
    assert np.abs(rows.sum(1)).max() < 1e-6
    expect = _through_targets(student, seqs, pos, rows)
    assert rel_l2(got, expect) < 1e-2 and cosine(got, expect) > 0.999
    student.close()
    teacher.close()


def test_a_list_of_one_certain_token_is_the_token_as_a_target(ctx):
    spec, m = _model(ctx)
    seqs, pos, tok = _seqs(spec, [25]), np.array([4, 9, 23], np.int32), np.array([7, 100, 3], np.int32)
    w = np.full(3, 1 / 3, np.float32)
    m.zero_grad()
    logp, _ = m.forward_backward(seqs, pos, tok, w)
    want = _gpu_flat(m, "ga", "gb")
    m.zero_grad()
    loss = m.distill_backward(seqs, pos, tok[:, None], np.zeros((3, 1)), w)
    assert np.abs(loss + w * logp).max() <= 256 * U
    assert rel_l2(_gpu_flat(m, "ga", "gb"), want) < 1e-3  # both round p - onehot to f16
    m.close()


def test_recurring_batches_replay_and_other_passes_stay_what_they_were(ctx):
    """The same shapes in turn, captured once they recur, between scoring and training passes on the same model."""
    spec, m = _model(ctx)
    seqs, pos = _seqs(spec, [33, 20]), np.array([5, 30, 40], np.int32)
    tok, w = np.array([1, 2, 3], np.int32), np.full(3, 1 / 3, np.float32)
    rng = np.random.default_rng(1)
    lists = [(rng.integers(0, spec.vocab, (3, 6)), np.log(rng.dirichlet(np.ones(7), 3)[:, :6])) for _ in range(2)]

    def distilled(l, mode, t):
        m.zero_grad()
        return m.distill_backward(seqs, pos, *l, w, t, mode), _gpu_flat(m, "ga", "gb")

    def trained():
        m.zero_grad()
        return m.forward_backward(seqs, pos, tok, w)[0], _gpu_flat(m, "ga", "gb")

    first = {(i, mode, t): distilled(lists[i], mode, t) for i in (0, 1) for mode in ("renorm", "tail") for t in (1.0, 2.0)}
    score = trained()
    for _ in range(3):
        for (i, mode, t), (loss, grad) in first.items():
            again = distilled(lists[i], mode, t)
            assert np.array_equal(again[0], loss) and np.array_equal(again[1], grad)
        again = trained()
        assert np.array_equal(again[0], score[0]) and np.array_equal(again[1], score[1])
        m.top_logits(seqs, pos, 5)
    m.close()


def _softmax(z, t):
    return np.exp(np.array([R.log_softmax(r, t) for r in z]))


@pytest.mark.parametrize("head_rows", [0, 7])
@pytest.mark.parametrize("drafted", [True, False])
def test_verified_drafts(ctx, drafted, head_rows):
    """Against the 64-bit form on the models' own logits; a chunk of seven head rows cuts the batch between sequences."""
    spec, m = _model(ctx, head_rows=head_rows)
    _, d = _model(ctx, seed=4, head_rows=head_rows)
    lens, start = [20, 9, 5, 33, 12], [15, 8, 5, 27, 10]  # 5, 1, 0, 6 and 2 drafted tokens
    seqs = _seqs(spec, lens)
    rng = np.random.default_rng(2)
    t = 1.3
    offs = np.cumsum([0] + lens)
    for trial in range(4):
        n = sum(lens) - sum(start)
        ua, us = rng.random(n, dtype=np.float32) * np.float32(0.02 if not drafted else 1.0), rng.random(5, dtype=np.float32)
        if trial == 0:
            ua[:] = 0  # everything that is possible stands
        acc, tok = m.verify_draft(seqs, start, ua, us, t, d if drafted else None)
        at = 0
        for s in range(5):
            k = lens[s] - start[s]
            rows = np.arange(offs[s] + start[s] - 1, offs[s] + lens[s])
            p = _softmax(_logits(m, seqs, rows), t)
            q = _softmax(_logits(d, seqs, rows[:-1]), t) if drafted and k else None
            assert (int(acc[s]), int(tok[s])) == R.verify(p, q, seqs[s][start[s]:], ua[at:at + k], us[s]), (trial, s)
            at += k
        if trial == 0:
            assert acc.tolist() == [5, 1, 0, 6, 2]
    m.close()
    d.close()


def test_objective_and_gate_wrappers(ctx):
    spec, student = _model(ctx)
    _, teacher = _model(ctx, seed=6)
    exs = [(t, int(t.size * 0.6)) for t in _seqs(spec, [30, 22, 18])]
    lists = obj.teacher_top_logits(teacher, exs, 16, 2.0)
    student.zero_grad()
    loss = obj.distill_batch_grad(student, exs, lists, 2.0)
    g = _gpu_flat(student, "ga", "gb")
    assert np.isfinite(loss) and loss > 0 and np.isfinite(g).all() and np.abs(g).max() > 0
    student.zero_grad()
    # the model as its own teacher has nothing to learn: its loss is what rounding leaves
    own = obj.teacher_top_logits(student, exs, 16, 2.0)
    assert abs(obj.distill_batch_grad(student, exs, own, 2.0)) <= 4 * 256 * U
    got = evalgate.accepted_prefix(teacher, exs, np.random.default_rng(0), 1.0, student)
    assert [n for _, n, _ in got] == [t.size - a for t, a in exs] and all(0 <= n <= k and 0 <= x < spec.vocab for n, k, x in got)
    assert evalgate.accepted_prefix(teacher, [], np.random.default_rng(0)) == []
    # a model that drafts for itself with the numbers 0 is believed everything
    zero = type("Zero", (), {"random": staticmethod(lambda n, dtype: np.zeros(n, dtype))})
    assert [n for n, k, _ in evalgate.accepted_prefix(teacher, exs, zero, 1.0, student)] == [k for _, k, _ in got]
    student.close()
    teacher.close()


def test_model_level_refusals(ctx):
    spec, m = _model(ctx, head_rows=8)
    _, d = _model(ctx, seed=1)
    seqs, pos, w = _seqs(spec, [20, 10]), np.array([3, 25], np.int32), np.ones(2, np.float32)
    i, t = np.zeros((2, 3), np.int32), np.full((2, 3), -2.0, np.float32)

    def refused(status, f):
        with pytest.raises(rt.RtError) as e:
            f()
        assert e.value.status == status, (status, e.value)

    refused(1, lambda: m.top_logits(seqs, pos, 0))
    refused(1, lambda: m.top_logits(seqs, pos, 257))
    refused(7, lambda: m.top_logits(seqs, pos, 3, 0.0))
    refused(6, lambda: m.top_logits(seqs, [30], 3))
    refused(7, lambda: m.top_logits(None, pos, 3))
    refused(1, lambda: m.distill_backward(seqs, pos, i[:1], t[:1], w))
    refused(7, lambda: m.distill_backward(seqs, pos, i, t, w, mode="reverse"))
    refused(7, lambda: m.distill_backward(seqs, pos, i, t, w, temperature=float("nan")))
    refused(7, lambda: m.distill_backward(seqs, pos[:0], i[:0], t[:0], w[:0]))
    refused(1, lambda: m.distill_backward(seqs, pos, np.zeros((2, 257), np.int32), np.zeros((2, 257), np.float32), w))
    for bad in (-2, spec.vocab):
        wrong = i.copy()
        wrong[1, 1] = bad
        refused(6, lambda: m.distill_backward(seqs, pos, wrong, t, w))
    refused(1, lambda: m.verify_draft(seqs, [19], [0.5], [0.5]))
    refused(1, lambda: m.verify_draft(seqs, [19, 9], [0.5], [0.5, 0.5]))
    refused(6, lambda: m.verify_draft(seqs, [0, 10], [0.5] * 20, [0.5, 0.5]))
    refused(7, lambda: m.verify_draft(seqs, [19, 10], [0.5], [0.5, 0.5], draft=m))
    refused(7, lambda: m.verify_draft(seqs, [19, 10], [0.5], [0.5, 0.5], temperature=-1.0, draft=d))
    refused(8, lambda: m.verify_draft(seqs, [12, 10], [0.5] * 8, [0.5, 0.5], draft=d))
    assert m.verify_draft(seqs, [13, 10], [0.5] * 7, [0.5, 0.5], draft=d)[0].shape == (2,)
    # no batch is staged behind these passes, and the model goes on
    assert rt.lib().rt_model_run_staged(m._h, 1) == 7
    assert np.isfinite(m.score(seqs, pos, [1, 2])[0]).all()
    m.close()
    d.close()
