"""The scheduler's sampling, row by row, on logits that are given: every request's tokens and
its generator's state are those of sample_logits on its own rows."""
from __future__ import annotations

import numpy as np
import pytest
import torch

from sunnynet_amd.runtime import serve as serve_module
from sunnynet_amd.runtime.serve import BatchScheduler, sample_logits

pytestmark = pytest.mark.gpu
INF, NAN = np.inf, np.nan


class Given:
    """A handle whose steps return given logits: steps (n, rows, V)."""

    def __init__(self, steps, dev):
        self.steps = [torch.tensor(s, dtype=torch.float32, device=dev) for s in steps]
        self.device, self.max_batch, self.at = dev, self.steps[0].shape[0], 0

    def get_state(self, n):
        return torch.zeros(n, 1, device=self.device), torch.zeros(n, 1, device=self.device)

    def set_state(self, s, h):
        pass

    def step_batch(self, tokens):
        self.at += 1
        return self.steps[self.at - 1][:tokens.shape[0]]


def serve(steps, settings, dev, prompts=None):
    """Every request steps through all the logits; checks its tokens and its generator."""
    sch = BatchScheduler(Given(steps, dev))
    prompts = prompts or [1] * len(settings)
    reqs = [sch.submit([1] * n, len(steps) - n + 1, seed=i, **s) for i, (n, s) in enumerate(zip(prompts, settings))]
    gens = [np.random.default_rng(i) for i in range(len(settings))]
    for r, g in zip(reqs, gens):           # a half word held back stays held back
        assert r.rng.integers(9, dtype=np.int32) == g.integers(9, dtype=np.int32)
    sch.run()
    rows = np.asarray(steps, dtype=np.float32)
    for i, (r, g, n) in enumerate(zip(reqs, gens, prompts)):
        want = [sample_logits(rows[t, i], r.temperature, r.top_p, r.top_k, g, r.min_p) for t in range(n - 1, len(steps))]
        assert r.output == want, i
        assert r.rng.bit_generator.state == g.bit_generator.state, i
    return sch


@pytest.mark.filterwarnings("ignore::RuntimeWarning")
def test_rows_without_a_distribution_draw_nothing(gpu):
    """Non-finite maxima, a temperature that makes them so, and a min_p above every weight: the
    token is the argmax, and the next draw is the one it would have been."""
    rng = np.random.default_rng(1)
    steps = 2 * rng.standard_normal((9, 6, 50))
    steps[2, 0, 7], steps[3, 1, 5], steps[4, 1], steps[5, 2, 30:] = INF, NAN, -INF, -INF
    steps[6, 3] = -INF
    serve(steps, [dict(temperature=0.8, top_k=9, top_p=0.9), dict(temperature=1.0), dict(temperature=1.0, top_p=0.7),
                  dict(temperature=2.0, top_k=5), dict(temperature=1.0, min_p=2.0), dict(temperature=1e-320)], gpu)


def test_other_generators_sample_on_the_host(gpu):
    """A generator that cannot take a number back, with rows that need it to."""
    rng = np.random.default_rng(2)
    steps = rng.standard_normal((6, 2, 40))
    steps[1, 0, 3], steps[2, 1] = INF, -INF
    sch = BatchScheduler(Given(steps, gpu))
    reqs = [sch.submit([1], 6, temperature=1.0) for _ in range(2)]
    kinds = [np.random.MT19937, np.random.SFC64]
    gens = [np.random.Generator(k(5)) for k in kinds]
    for r, k in zip(reqs, kinds):
        r.rng = np.random.Generator(k(5))
    sch.run()
    for i, (r, g) in enumerate(zip(reqs, gens)):
        assert r.output == [sample_logits(steps[t, i].astype(np.float32), 1.0, rng=g) for t in range(6)]


def test_neighbours_do_not_move_a_row_to_the_host(gpu, monkeypatch):
    """Equal logits at the nucleus' border go by index on the device and in no fixed order on the
    host: a request's tokens are its own whether or not a neighbour's settings need the host."""
    rng = np.random.default_rng(3)
    tied = np.round(rng.standard_normal((40, 3, 300)))
    own = [dict(temperature=1.0, top_p=0.5), dict(temperature=1.3, top_p=0.6)]
    out = []
    for other in (dict(temperature=1.0), dict(temperature=1.0, top_k=-3)):
        sch = BatchScheduler(Given(tied, gpu))
        reqs = [sch.submit([1], 40, seed=i, **s) for i, s in enumerate([*own, other])]
        sch.run()
        out.append([r.output for r in reqs])
    assert out[0][:2] == out[1][:2]
    gen = np.random.default_rng(2)         # the neighbour itself is sampled on the host
    assert out[1][2] == [sample_logits(tied[t, 2].astype(np.float32), 1.0, 1.0, -3, gen) for t in range(40)]


def test_a_batch_of_rows_for_both(gpu):
    rng = np.random.default_rng(4)
    serve(2 * rng.standard_normal((12, 5, 90)), [dict(temperature=1.0, top_k=-5), dict(), dict(temperature=0.7, top_k=9),
                                                 dict(temperature=1.1, top_p=0.8), dict(temperature=0.5, top_k=-1)], gpu,
          prompts=[1, 3, 1, 7, 4])


def test_steps_inside_prompts_choose_nothing(gpu, monkeypatch):
    """Steps that leave every request inside its prompt do not sample or copy logits."""
    calls = []
    plain = serve_module.sample_tokens
    monkeypatch.setattr(serve_module, "sample_tokens", lambda *a: calls.append(a[0].shape[0]) or plain(*a))
    rng = np.random.default_rng(6)
    serve(rng.standard_normal((8, 2, 30)), [dict(temperature=1.0), dict(temperature=0.5, top_k=4)], gpu, prompts=[5, 7])
    assert len(calls) == 4                 # from the fifth step on


@pytest.mark.filterwarnings("ignore::RuntimeWarning")
def test_settings_that_only_the_host_knows(gpu):
    """top_k that is no whole number, and temperatures that are not finite."""
    rng = np.random.default_rng(7)
    steps = rng.standard_normal((7, 6, 60))
    steps[2, 3, 10:] = -INF                # at an infinite temperature no distribution, by the host's rule
    settings = [dict(temperature=1.0, top_k=INF), dict(temperature=1.0, top_k=np.int64(5)), dict(temperature=INF),
                dict(temperature=INF, top_p=0.5), dict(temperature=NAN), dict(temperature=0.9, top_k=None)]
    serve(steps, settings, gpu)
