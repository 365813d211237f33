"""The gradients of distillation through a model with a large vocabulary, where most of a row's gradient elements are tiny and of one sign.

The rows of the head's weights share a large common part, c.  A row of logit gradients sums to zero, so that c has no part in what reaches
the model; whatever the small elements lose by rounding to 16 bits comes through multiplied by c.  The expected gradient is the one that
forward_backward gives with every token of the vocabulary as a target of the same position (test_gpu_distill.py), whose rows' rounding is
the same for every target and cancels with the weights' sum.

Tolerance: that of the other objectives, 1e-2, and what the rounding of rows to f16 may add through c.  Either side rounds every element g_v (a
single row's, or a target's weight times p_v - 1) by at most 2^-11 of it, which moves what reaches the model, sum g_v W_v, by at most 2^-11 sum |g_v| |W_v|."""
import numpy as np
import pytest

import rust_trainer_b200 as rt
import vocab_reference as R
from conftest import cosine, rel_l2
from rust_trainer_b200 import quants, synth
from test_gpu_distill import U, _logits, _model, _seqs, _through_targets
from test_gpu_model import _gpu_flat

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def large(ctx):
    spec = synth.preset("tiny-qwen3", vocab=131072, quant="Q8_0", w_std=0.08, tie_embeddings=False)
    tensors = synth.build_tensors(spec)
    rng = np.random.default_rng(0)
    w = rng.standard_normal((spec.vocab, spec.hidden), dtype=np.float32) * np.float32(0.2)  # logits of a spread of 2.3 or so
    w += np.float32(4.0) * rng.standard_normal(spec.hidden, dtype=np.float32)
    q8 = quants.BY_NAME["Q8_0"]
    tensors["output.weight"] = (q8, spec.vocab, spec.hidden, quants.quantize(w, q8))
    w = w.astype(np.float64)
    m = rt.Model(ctx, spec.config(), tensors)
    m.attach_lora(8, 16.0, None, 5)
    m.load_adapters(synth.lora_adapters(spec, 8, 16.0, seed=2, b_std=0.02))
    yield spec, m, w
    m.close()


@pytest.mark.parametrize("mode", ["renorm", "tail"])
@pytest.mark.parametrize("noise", [0.3, 0.1])
def test_small_gradients_are_not_lost_together(large, mode, noise):
    spec, m, weight = large
    seqs, pos, k = _seqs(spec, [24]), np.array([19], np.int32), 32
    z = _logits(m, seqs, pos)[0].astype(np.float64)
    index, tl, _ = R.top(z + noise * np.random.default_rng(1).standard_normal(z.size), k, 1.0)
    m.zero_grad()
    w = np.ones(1, np.float32)
    loss = m.distill_backward(seqs, pos, index[None], tl[None], w, 1.0, mode)
    got = _gpu_flat(m, "ga", "gb")
    want, grad, _ = R.distill(z, index, tl.astype(np.float32), 1.0, mode)
    assert abs(loss[0] - want) <= 256 * U
    expect = _through_targets(m, seqs, pos, grad[None])
    rounding = 2 * 2.0**-11 * (np.abs(grad) * np.linalg.norm(weight, axis=1)).sum() / np.linalg.norm(grad @ weight)
    assert rounding < 0.2 and rel_l2(got, expect) < 1e-2 + rounding, (rounding, rel_l2(got, expect))


@pytest.mark.parametrize("preset", ["tiny-qwen3", "tiny-llama"])
def test_lists_of_more_than_all_mass(ctx, preset):
    """Entries that add up to m >= 1, or that f16 could not hold: p - m q for a list q that is normalised, so that (G(m) - G(1)) / (m - 1) is
    the same for every m, G(1) being the normalised list's."""
    spec, m = _model(ctx, preset)
    seqs, pos = _seqs(spec, [30]), np.array([3, 11, 20, 29], np.int32)
    rng = np.random.default_rng(3)
    index = np.stack([rng.permutation(spec.vocab)[:6] for _ in range(4)]).astype(np.int32)
    t = np.log(rng.dirichlet(np.ones(6), 4))
    w = np.full(4, 0.25, np.float32)

    def gradient(shift, mode):
        m.zero_grad()
        m.distill_backward(seqs, pos, index, t + shift, w, 1.0, mode)
        g = _gpu_flat(m, "ga", "gb").astype(np.float64)
        assert np.isfinite(g).all()
        return g

    one = gradient(0.0, "renorm")
    want = gradient(np.log(3.0), "tail") - one
    for mass in (2.0, 100.0, 3e4, 1e9):
        got = (gradient(np.log(mass), "tail") - one) * 2 / (mass - 1)
        assert rel_l2(got, want) < 1e-2 and cosine(got, want) > 0.999, mass
    m.close()


def test_a_verification_that_fails_leaves_no_batch_behind(ctx):
    """The drafting model refuses its pass (it has no weights yet) when the target's has run."""
    spec, m = _model(ctx, head_rows=16)
    d = rt.Model.__new__(rt.Model)
    with pytest.raises(rt.RtError):
        d.__init__(ctx, spec.config(), {}, head_rows=16)
    seqs = _seqs(spec, [20])
    with pytest.raises(rt.RtError) as e:
        m.verify_draft(seqs, [15], [0.5] * 5, [0.5], draft=d)
    assert "finalize" in str(e.value)
    assert rt.lib().rt_model_run_staged(m._h, 0) == 7
    assert np.isfinite(m.score(seqs, np.array([3], np.int32), [1])[0]).all()
    m.close()
    d.close()


def test_no_scoring_batch_is_staged_behind_a_teachers_pass(ctx):
    spec, m = _model(ctx)
    seqs, pos = _seqs(spec, [20, 9]), np.array([3, 8, 25], np.int32)
    m.top_logits(seqs, pos, 4)
    assert rt.lib().rt_model_run_staged(m._h, 0) == 7
    assert np.isfinite(m.score(seqs, pos, [1, 2, 3])[0]).all()
    m.close()


@pytest.mark.parametrize("mode", ["renorm", "tail"])
def test_distillation_in_chunks_of_the_head(ctx, mode):
    """Five targets through a head of two rows at a time: the losses of one chunk, and its gradients."""
    spec, m = _model(ctx)
    _, small = _model(ctx, head_rows=2)
    seqs, pos = _seqs(spec, [30, 12]), np.array([3, 20, 29, 31, 40], np.int32)
    w = np.array([0.2, 0.1, 0.3, 0.0, 0.4], np.float32)
    rng = np.random.default_rng(7)
    index = rng.integers(0, spec.vocab, (5, 9)).astype(np.int32)
    t = np.log(rng.dirichlet(np.ones(10), 5)[:, :9])
    out = []
    for x in (m, small):
        x.zero_grad()
        out.append((x.distill_backward(seqs, pos, index, t, w, 1.5, mode), _gpu_flat(x, "ga", "gb")))
    assert np.abs(out[0][0] - out[1][0]).max() <= 256 * U
    assert rel_l2(out[1][1], out[0][1]) < 1e-2 and cosine(out[1][1], out[0][1]) > 0.999
    m.close()
    small.close()
