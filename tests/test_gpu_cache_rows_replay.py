"""Beam selection, reordering and eviction captured and replayed with other inputs, and side by side on two streams."""
import ctypes as C

import numpy as np
import pytest
import torch

import plain_cache4 as P

pytestmark = pytest.mark.gpu


def arr(ts):
    return (C.c_void_p * len(ts))(*[t.data_ptr() for t in ts])


class Search:
    """Buffers of groups of beams with half caches and row weights; a step selects, reorders in place and evicts into other planes."""

    def __init__(self, lcu, groups, beams, kv, ctx, vocab, keep, recent, seed):
        self.lcu, self.groups, self.beams, self.kv, self.ctx, self.vocab, self.keep, self.recent = lcu, groups, beams, kv, ctx, vocab, keep, recent
        self.rng, n = np.random.default_rng(seed), groups * beams
        self.logits = torch.zeros(n, vocab, device="cuda")
        self.scores = torch.zeros(groups, beams, device="cuda")
        self.parents, self.tokens = (torch.zeros(groups, beams, dtype=torch.int32, device="cuda") for _ in range(2))
        self.out = torch.zeros(groups, beams, device="cuda")
        self.keys, self.weights = torch.zeros(n, kv, ctx, 64, dtype=torch.float16, device="cuda"), torch.zeros(n, kv, ctx, 1, device="cuda")
        self.lengths, self.left = (torch.zeros(n, dtype=torch.int32, device="cuda") for _ in range(2))
        self.kept = torch.zeros(n, kv, keep, dtype=torch.int32, device="cuda")
        self.to = [torch.zeros(n, kv, keep, 64, dtype=torch.float16, device="cuda"), torch.zeros(n, kv, keep, 1, device="cuda")]
        self.ws = torch.empty(lcu.lib.lcu_beam_select_workspace(groups, beams, vocab, beams), dtype=torch.uint8, device="cuda")

    def fill(self):
        r = self.rng
        self.logits.copy_(torch.from_numpy(r.standard_normal(tuple(self.logits.shape)).astype(np.float32) * 2))
        self.scores.copy_(torch.from_numpy(r.standard_normal(tuple(self.scores.shape)).astype(np.float32)))
        self.keys.copy_(torch.from_numpy(r.standard_normal(tuple(self.keys.shape)).astype(np.float16)))
        self.weights.copy_(torch.from_numpy(r.random(tuple(self.weights.shape)).astype(np.float32)))
        self.lengths.copy_(torch.from_numpy(np.repeat(r.integers(1, self.ctx + 1, self.groups), self.beams).astype(np.int32)))
        for t in self.to:
            t.fill_(7)
        torch.cuda.synchronize()
        self.was = [t.clone() for t in (self.keys, self.weights)]

    def step(self, stream):
        lib, check, n = self.lcu.lib, self.lcu.check, self.groups * self.beams
        check(lib.lcu_beam_select(self.parents.data_ptr(), self.tokens.data_ptr(), self.out.data_ptr(), self.logits.data_ptr(), self.vocab, 2, self.scores.data_ptr(),
                                  self.groups, self.beams, self.vocab, self.beams, self.ws.data_ptr(), self.ws.numel(), stream))
        both, rb = arr([self.keys, self.weights]), (C.c_int * 2)(128, 4)
        check(lib.lcu_cache_reorder(both, both, rb, 2, self.parents.data_ptr(), self.lengths.data_ptr(), self.groups, self.beams, self.kv, self.ctx, stream))
        check(lib.lcu_cache_evict(arr(self.to), both, rb, 2, self.weights.data_ptr(), self.kept.data_ptr(), self.left.data_ptr(), self.lengths.data_ptr(), n, self.kv,
                                  self.ctx, self.keep, self.keep, self.recent, stream))

    def holds(self):
        torch.cuda.synchronize()
        x, scores = self.logits.double().cpu().numpy().reshape(self.groups, self.beams, self.vocab), self.scores.double().cpu().numpy()
        for g in range(self.groups):
            p, t, s = P.beam_select(x[g], scores[g], self.beams)
            assert self.parents[g].tolist() == p.tolist() and self.tokens[g].tolist() == t.tolist()
            assert np.abs(self.out[g].cpu().numpy() - s).max() <= 2.0 ** -18 + 2.0 ** -24 * np.abs(s).max()
            for b in range(self.beams):
                at, frm, n = g * self.beams + b, g * self.beams + p[b], int(self.lengths[g * self.beams])
                for now, was in zip((self.keys, self.weights), self.was):
                    assert torch.equal(now[at, :, :n], was[frm, :, :n]) and torch.equal(now[at, :, n:], was[at, :, n:])
                assert int(self.left[at]) == min(n, self.keep)
                for h in range(self.kv):
                    rows = P.evict(self.weights[at, h, :, 0].cpu().numpy(), n, self.keep, self.recent)
                    assert self.kept[at, h].tolist() == rows + [-1] * (self.keep - len(rows))
                    for to, now in zip(self.to, (self.keys, self.weights)):
                        assert torch.equal(to[at, h, :len(rows)], now[at, h, rows]) and (to[at, h, len(rows):] == 7).all()


SHAPES = [(2, 3, 2, 300, 9000, 120, 17), (1, 4, 3, 17000, 700, 4000, 100)]


@pytest.mark.parametrize("shape", SHAPES)
def test_replayed_searches_follow_their_inputs(lcu, shape):
    s = Search(lcu, *shape, seed=1)
    side = torch.cuda.Stream()
    s.fill()
    s.step(side.cuda_stream)
    s.holds()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        s.step(torch.cuda.current_stream().cuda_stream)
    for _ in range(3):
        s.fill()
        graph.replay()
        s.holds()


def test_searches_on_two_streams(lcu):
    both, streams = [Search(lcu, *SHAPES[0], seed=k) for k in (2, 3)], [torch.cuda.Stream() for _ in range(2)]
    for _ in range(4):
        for s in both:
            s.fill()
        for s, stream in zip(both, streams):
            s.step(stream.cuda_stream)
        for s in both:
            s.holds()
