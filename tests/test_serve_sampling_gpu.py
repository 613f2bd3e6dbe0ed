"""The scheduler's sampling on the device: every token of every request is the one that
the host sampler draws from the same logits with the request's own generator, whatever
mix of greedy, filtered and prefilling requests a step holds."""
from __future__ import annotations

import numpy as np
import pytest
import torch

from sunnynet_amd.blob import pack_sunny_blob
from sunnynet_amd.config import TINY
from sunnynet_amd.runtime import serve
from sunnynet_amd.runtime.model import HipModel
from sunnynet_amd.runtime.serve import BatchScheduler, sample_logits
from sunnynet_amd.weights import init_sunnynet

pytestmark = pytest.mark.gpu

SETTINGS = [dict(), dict(temperature=0.8, top_k=40, top_p=0.95), dict(temperature=1.0), dict(temperature=1.5, top_p=0.7),
            dict(temperature=0.6, top_k=5), dict(temperature=2.0, min_p=0.2), dict(temperature=None),
            dict(temperature=0.9, top_k=3, top_p=0.5, min_p=0.01), dict(temperature=1.0, top_k=10 ** 7)]


class Recorder:
    """A handle whose steps' logits are kept, with the active requests of each step."""

    def __init__(self, model):
        self._m, self.seen = model, []

    def __getattr__(self, n):
        return getattr(self._m, n)

    def step_batch(self, tokens):
        out = self._m.step_batch(tokens)
        self.seen.append(out.float().cpu().numpy())
        return out


def serve_all(tmp_path, settings, monkeypatch=None, host=False):
    path = tmp_path / "m.bin"
    path.write_bytes(pack_sunny_blob(init_sunnynet(TINY, 0)))
    c = TINY
    m = Recorder(HipModel(path, c.vocab_size, c.dim, c.inner, c.rank, c.taps, c.layers, max_batch=6))
    sch = BatchScheduler(m)
    rng = np.random.default_rng(3)
    reqs = [sch.submit(rng.integers(0, c.vocab_size, int(rng.integers(1, 9))).tolist(), int(rng.integers(1, 12)),
                       seed=100 + i, **s) for i, s in enumerate(settings * 2)]
    gens = {id(r): np.random.default_rng(100 + i) for i, r in enumerate(reqs)}
    while sch.active or sch.waiting:
        had = {id(r): len(r.output) for r in reqs}
        sch._admit()
        order = list(sch.active)
        sch.step()
        for row, r in zip(m.seen[-1], order):
            if len(r.output) > had[id(r)]:
                want = sample_logits(row, r.temperature, r.top_p, r.top_k, gens[id(r)], r.min_p)
                assert r.output[-1] == want
    m.close()
    assert all(r.done and r.output for r in reqs)
    return [r.output for r in reqs]


def test_tokens_are_the_host_samplers(gpu, tmp_path, monkeypatch):
    calls = []
    plain = serve.sample_tokens
    monkeypatch.setattr(serve, "sample_tokens", lambda *a: calls.append(a[0].shape[0]) or plain(*a))
    first = serve_all(tmp_path, SETTINGS)
    assert calls and max(calls) == 6
    assert serve_all(tmp_path, SETTINGS) == first                 # seeded: reproducible


def test_settings_the_device_does_not_know_stay_on_the_host(gpu, tmp_path, monkeypatch):
    def never(*a):
        raise AssertionError("sample_tokens called")
    monkeypatch.setattr(serve, "sample_tokens", never)
    serve_all(tmp_path, [dict(temperature=1.0, top_k=-5)])
    serve_all(tmp_path, [dict()])                                  # greedy requests alone


def test_settings_changed_between_steps(gpu, tmp_path):
    """A request's settings hold from the next step on, and a greedy one's filters are not read."""
    path = tmp_path / "m.bin"
    path.write_bytes(pack_sunny_blob(init_sunnynet(TINY, 0)))
    c = TINY
    m = Recorder(HipModel(path, c.vocab_size, c.dim, c.inner, c.rank, c.taps, c.layers, max_batch=3))
    sch = BatchScheduler(m)
    reqs = [sch.submit([5], 24, seed=1, temperature=3.0), sch.submit([6], 24, seed=2, temperature=0.0, top_p=None),
            sch.submit([7], 24, seed=3, temperature=1.0, top_k=9)]
    gens = [np.random.default_rng(s) for s in (1, 2, 3)]
    for step in range(24):
        if step == 8:
            reqs[0].top_k, reqs[2].temperature = 2, 0.01
        if step == 16:
            reqs[0].temperature, reqs[2].top_p, reqs[2].temperature = 0.0, 0.3, 5.0
        sch.step()
        for row, r, gen in zip(m.seen[-1], reqs, gens):
            assert r.output[step] == sample_logits(row, r.temperature, r.top_p, r.top_k, gen, r.min_p)
    m.close()


def test_fields_keep_their_places():
    r = serve.Request([1], 2, 0.5, 0.9, 3, 7, 11)
    assert (r.temperature, r.top_p, r.top_k, r.eos, r.seed, r.min_p) == (0.5, 0.9, 3, 7, 11, 0.0)


def test_min_p_of_the_host_sampler():
    z = np.log(np.array([0.5, 0.3, 0.15, 0.05]))
    draws = {sample_logits(z, 1.0, 1.0, 0, np.random.default_rng(i), 0.4) for i in range(50)}
    assert draws == {0, 1}


def test_device_loop_without_host_round_trips(gpu, tmp_path):
    """A sampled token loop that stays on the device: step, sample, step."""
    path = tmp_path / "m.bin"
    path.write_bytes(pack_sunny_blob(init_sunnynet(TINY, 1)))
    c = TINY
    m = HipModel(path, c.vocab_size, c.dim, c.inner, c.rank, c.taps, c.layers, max_batch=3)
    u = torch.rand(8, 3, dtype=torch.float64, device="cuda")
    tok = torch.tensor([1, 2, 3], dtype=torch.int32, device="cuda")
    from sunnynet_amd.runtime import sample_tokens
    toks, logits = [], []
    for t in range(8):
        logits.append(m.step_batch(tok).clone())
        tok = sample_tokens(logits[-1], u[t], 0.9, 50, 0.9)
        toks.append(tok)
    for t in range(8):
        again = sample_tokens(logits[t], u[t], 0.9, 50, 0.9)
        assert torch.equal(again, toks[t])
    m.close()
