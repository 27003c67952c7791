"""Whole passes through the public functions, gradients included, recorded as CUDA graphs: replayed on other inputs, two graphs in
turn, on a stream of the caller's, and eager passes on two streams at once."""

import pytest
import torch

from dual_mod_public_b200.ops import cached_attention, packed_attention, token_logprobs

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


def rnd(*shape, seed):
    return torch.randn(*shape, generator=torch.Generator(device=DEV).manual_seed(seed), device=DEV).bfloat16()


class Pass:
    """Attention over two documents, scores of the next tokens, gradients, and one token over the keys as a cache."""

    def __init__(self, seed, T=300, dim=64):
        g = torch.Generator().manual_seed(seed)
        self.q, self.k, self.v = (rnd(T, h, dim, seed=seed + i).requires_grad_() for i, h in enumerate((4, 2, 2)))
        self.w = rnd(4 * dim, 500, seed=seed + 3) * 0.1
        self.y = torch.randint(0, 500, (T,), generator=g).to(DEV)
        self.cu = torch.tensor([0, 100 + seed, T], dtype=torch.int32, device=DEV)
        self.n = torch.tensor([T - 7], dtype=torch.int32, device=DEV)

    def __call__(self):
        o = packed_attention(self.q, self.k, self.v, self.cu)
        r = token_logprobs(o.reshape(len(o), -1) @ self.w, self.y, top=3)
        grads = torch.autograd.grad((r.logp, r.entropy), (self.q, self.k, self.v), (torch.ones_like(r.logp), torch.ones_like(r.entropy)))
        with torch.no_grad():
            one = cached_attention(self.q[-1:], self.k[None], self.v[None], self.n)
        return [o.detach(), r.logp.detach(), r.entropy.detach(), r.top_logp, r.top_ids, one, *grads]

    def take(self, other):
        with torch.no_grad():
            for name in ("q", "k", "v", "y", "cu", "n", "w"):
                getattr(self, name).copy_(getattr(other, name))

    def record(self):
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            self()
        torch.cuda.current_stream().wait_stream(side)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            held = self()
        return graph, held


def same(a, b):
    return all(torch.equal(x, y) for x, y in zip(a, b))


@pytest.mark.parametrize("dim", [64, 128])
def test_recorded_passes(dim):
    inputs = [Pass(s, dim=dim) for s in (1, 2, 3)]
    want = [[t.clone() for t in p()] for p in inputs]
    assert not same(want[0], want[1])
    a, b = Pass(1, dim=dim), Pass(2, dim=dim)
    (ga, out_a), (gb, out_b) = a.record(), b.record()
    for turn in (0, 2, 1, 0):
        a.take(inputs[turn])
        b.take(inputs[(turn + 1) % 3])
        ga.replay()
        gb.replay()
        assert same(out_a, want[turn]) and same(out_b, want[(turn + 1) % 3])
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        a.take(inputs[1])
        ga.replay()
        got = [t.clone() for t in out_a]
    s.synchronize()
    assert same(got, want[1])


def test_two_streams_at_once():
    passes = [Pass(s, T=1500) for s in (1, 2)]
    want = [[t.clone() for t in p()] for p in passes]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in passes]
    got = [[] for _ in passes]
    for _ in range(5):
        for p, s, out in zip(passes, streams, got):
            with torch.cuda.stream(s):
                out.append(p())
    torch.cuda.synchronize()
    for out, w in zip(got, want):
        assert all(same(o, w) for o in out)
