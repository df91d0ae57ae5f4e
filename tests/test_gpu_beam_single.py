"""Beam search of one beam: greedy decoding. Its lists have a single entry where
there is no EOS id. The scratch is filled with NaN bits in front of every call,
so that nothing may come from what it held."""
import numpy as np
import pytest
import torch

from tests.test_gpu_beam import TYPES, _ctx, beams, check, empty_pool, lse_tol, rows_at

pytestmark = pytest.mark.gpu


@pytest.fixture(autouse=True)
def scratch_of_nan(monkeypatch):
    from zllm_amd import beam, distill
    make = beam._work

    def work(nbytes, dev):
        t, at = make(nbytes, dev)
        if t is not None:
            t.fill_(0xff)
        return t, at
    monkeypatch.setattr(beam, "_work", work)
    monkeypatch.setattr(distill, "_work", work)


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("G,V", [(1, 1), (3, 7), (5, 4099), (2, 50257)])
def test_one_beam_without_an_end(G, V, dtype):
    rng = np.random.default_rng(G + V)
    for shift in (0, 1, 5):
        x = rng.normal(0, 2, (G, V)).astype(np.float32)
        check(rows_at(x, dtype, shift, 3), beams(rng, G, 1), empty_pool(G, 1), 1, what=f"one beam shift={shift}")


def test_one_beam_of_ties_and_orders():
    """Equal values, sorted rows, rows of nothing, one id, huge values."""
    rng = np.random.default_rng(8)
    V = 70001
    x = rng.normal(0, 2, (7, V)).astype(np.float32)
    x[0] = 1.5
    x[1].sort()
    x[2] = -np.inf
    x[3] = np.nan
    x[3, V - 1] = -4.0
    x[4] = -1e30
    x[5, 100:3000] = 30.0
    for dtype in ("f32", "bf16"):
        check(rows_at(x, dtype, 1, 2), beams(rng, 7, 1), empty_pool(7, 1), 1, what="one beam, orders")


def test_one_beam_over_several_steps():
    """BeamSearch as it is by default (no EOS id): the likeliest id at every
    step, its score the sum of the log-probabilities over the length."""
    from zllm_amd.beam import BeamSearch
    rng = np.random.default_rng(5)
    G, V, steps = 4, 600, 6
    x = rng.normal(0, 2, (steps, G, V)).astype(np.float32)
    print(f"[case] BeamSearch one beam G={G} V={V} steps={steps}", flush=True)
    search = BeamSearch(_ctx(), G, 1, steps)
    for t in range(steps):
        assert not search.finished()
        search.step(torch.from_numpy(x[t]).cuda())
        assert (search.parents == 0).all()
    d = x.astype(np.float64)
    lp = d - np.log(np.exp(d).sum(2, keepdims=True))
    for g, hyps in enumerate(search.sequences()):
        assert len(hyps) == 1 and hyps[0].tokens == x[:, g].argmax(1).tolist() and not hyps[0].finished
        # a step's rounding: its logarithm's and the running sum's to 32 bits
        want = lp[:, g].max(1).sum()
        assert abs(hyps[0].score * steps - want) <= steps * (lse_tol(V) + 2.0 ** -23 * abs(want))


@pytest.mark.parametrize("W,eos,K", [(2, (), 1), (2, (3,), 2), (5, (1, 2), 17)])
def test_wider_beams_and_lists(W, eos, K):
    from tests.test_gpu_distill import check_teacher
    rng = np.random.default_rng(W)
    x = rng.normal(0, 2, (3 * W, 999)).astype(np.float32)
    for dtype in TYPES:
        xt = rows_at(x, dtype, 1, 2)
        check(xt, beams(rng, 3, W), empty_pool(3, W), W, eos, what="scratch of NaN")
        check_teacher(xt, K, 1.5, "scratch of NaN")
