"""GPU tests of the tree attention and of the sampler's several launches where they meet: on two streams at once, and in turn
over one workspace, eager and captured. Attention is compared with calls of its own, bit for bit, tokens with the 64-bit
form."""
import pytest
import torch

import _draft_tree_ref as R
import efm_capi as C
from _util import ptr, stream

pytestmark = pytest.mark.gpu


class _Attention:
    """Attention that is split over workgroups, and so uses its workspace."""

    def __init__(self, hq, hkv, hd, n, prefix, seed=1):
        g = torch.Generator(device="cuda").manual_seed(seed)
        self.n, self.rows = n, prefix + n
        self.ctx = C.make_attention_ctx(hq, hkv, hd, rope=False)
        self.q = torch.randn(n, hq, hd, generator=g, device="cuda").bfloat16()
        self.kv = torch.randn(2, self.rows, hkv, hd, generator=g, device="cuda").bfloat16()
        self.mask = R.words(R.bits(R.random_tree(n, torch.Generator().manual_seed(n)))).cuda()
        self.length = torch.tensor([self.rows], dtype=torch.int32, device="cuda")
        self.o = torch.zeros(n, hq * hd, dtype=torch.bfloat16, device="cuda")
        self.bytes = C.load().efm_attention_tree_workspace_bytes(self.ctx, n, self.rows)
        assert self.bytes > 0

    def launch(self, ws):
        C.call("efm_attention_tree", self.ctx, ptr(self.q), ptr(self.kv[0]), ptr(self.kv[1]), ptr(self.mask), ptr(self.o), self.n, 0,
               ptr(self.length), self.rows, ptr(ws), ws.numel(), stream())

    def new(self, seed):
        self.q.copy_(torch.randn(self.q.shape, generator=torch.Generator().manual_seed(seed)).bfloat16())

    def alone(self):
        """Outputs of a call with a workspace that nothing else uses."""
        kept = self.o.clone()
        self.launch(torch.full((self.bytes,), 0xff, dtype=torch.uint8, device="cuda"))
        torch.cuda.synchronize()
        want = self.o.clone()
        self.o.copy_(kept)
        return want


class _Sampler:
    def __init__(self, rows, vocab, dtype=torch.float32, k=0, p=1.0, min_p=0.0):
        self.rows, self.vocab, self.f = rows, vocab, dict(k=k, p=p, min_p=min_p)
        self.x, self.u = torch.zeros(rows, vocab, dtype=dtype, device="cuda"), torch.zeros(rows, device="cuda")
        self.out = torch.zeros(rows, dtype=torch.int32, device="cuda")
        self.bytes = C.load().efm_sampler_filtered_workspace_bytes(rows, vocab)
        assert self.bytes > 0

    def new(self, seed):
        g = torch.Generator(device="cuda").manual_seed(seed)
        x = (0.5 if seed % 3 == 2 else 2.5) * torch.randn(self.rows, self.vocab, generator=g, device="cuda")   # flat rows now and then
        self.x.copy_(x), self.u.copy_(torch.rand(self.rows, generator=g, device="cuda"))

    def launch(self, ws):
        dt = C.EFM_DTYPE_BF16 if self.x.dtype == torch.bfloat16 else C.EFM_DTYPE_F32
        C.call("efm_sampler_filtered", self.rows, self.vocab, ptr(self.x), dt, 0, 1.0, self.f["k"], self.f["p"], self.f["min_p"], ptr(self.u),
               ptr(self.out), ptr(ws), ws.numel(), stream())

    def alone(self):
        return R.sample(self.x, self.u, **self.f)


def _sets():
    return ([_Attention(28, 4, 128, 33, 9000), _Sampler(33, 151936, p=0.9), _Sampler(5, 60000, torch.bfloat16, k=100, p=0.95)],
            [_Attention(14, 2, 64, 100, 3000, seed=2), _Sampler(64, 50000, k=50, min_p=0.01), _Sampler(20, 151936, torch.bfloat16, p=0.95),
             _Sampler(3, 151936, min_p=0.02)])


def _workspace(ops):
    return torch.full((max(op.bytes for op in ops),), 0xff, dtype=torch.uint8, device="cuda")


def _check(ops, wants, what):
    for i, (op, want) in enumerate(zip(ops, wants)):
        assert torch.equal(op.o if isinstance(op, _Attention) else op.out, want), (what, i)


def test_two_streams_at_once(gpu):
    """Attention and samplers in turn on each of two streams, which share nothing; a workspace a stream."""
    sets = _sets()
    spaces, streams = [_workspace(ops) for ops in sets], [torch.cuda.Stream(), torch.cuda.Stream()]
    for step in range(6):
        for ops in sets:
            for op in ops:
                op.new(step)
        torch.cuda.synchronize()
        wants = [[op.alone() for op in ops] for ops in sets]
        torch.cuda.synchronize()
        for _ in range(3):
            for i in range(max(map(len, sets))):
                for ops, ws, s in zip(sets, spaces, streams):
                    with torch.cuda.stream(s):
                        ops[i % len(ops)].launch(ws)
        torch.cuda.synchronize()
        for ops, want in zip(sets, wants):
            _check(ops, want, step)


@pytest.mark.parametrize("which", [0, 1])
def test_one_workspace_in_turn(gpu, which):
    """Attention and samplers one after another over one workspace, eager, and captured with eager calls between replays."""
    ops = _sets()[which]
    ws = _workspace(ops)
    for op in ops:
        op.new(99)
        op.launch(ws)
    side, graph = torch.cuda.Stream(), torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph, stream=side, capture_error_mode="thread_local"):
        for op in ops + ops[::-1]:
            op.launch(ws)
    for step in range(6):
        for op in ops:
            op.new(step)
        wants = [op.alone() for op in ops]
        for op in ops[::-1] + ops:
            op.launch(ws)
        torch.cuda.synchronize()
        _check(ops, wants, f"eager {step}")
        for op in ops:
            op.new(step + 50)
        wants = [op.alone() for op in ops]
        graph.replay()
        torch.cuda.synchronize()
        _check(ops, wants, f"replay {step}")
