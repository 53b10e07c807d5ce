"""GPU tests of the tree attention over a cache whose rows past the length hold what earlier texts left there."""
import math

import pytest
import torch

import _draft_tree_ref as R
import efm_capi as C
from _util import ptr, stream

pytestmark = pytest.mark.gpu

# both kernels: little work, much work
CASES = [pytest.param(14, 2, 64, 250, 910, id="few-64"), pytest.param(12, 2, 128, 200, 2001, id="few-128"),
         pytest.param(12, 2, 128, 1000, 1990, id="rows-128"), pytest.param(28, 4, 64, 1001, 2900, id="rows-64")]


class _Call:
    def __init__(self, hq, hkv, hd, n, prefix):
        g = torch.Generator(device="cuda").manual_seed(n)
        self.n, self.rows, self.bound = n, prefix + n, prefix + n + 128
        self.ctx = C.make_attention_ctx(hq, hkv, hd, rope=False)
        self.q = torch.randn(n, hq, hd, generator=g, device="cuda").bfloat16()
        self.kv = torch.randn(2, self.bound, hkv, hd, generator=g, device="cuda").bfloat16()
        self.mask = R.words(R.bits(R.random_tree(n, torch.Generator().manual_seed(n)))).cuda()
        self.length = torch.tensor([self.rows], dtype=torch.int32, device="cuda")
        self.o = torch.empty(n, hq * hd, dtype=torch.bfloat16, device="cuda")
        size = C.load().efm_attention_tree_workspace_bytes(self.ctx, n, self.bound)
        self.ws = torch.empty(max(size, 256), dtype=torch.uint8, device="cuda")

    def launch(self):
        C.call("efm_attention_tree", self.ctx, ptr(self.q), ptr(self.kv[0]), ptr(self.kv[1]), ptr(self.mask), ptr(self.o), self.n, 0,
               ptr(self.length), self.bound, ptr(self.ws), self.ws.numel(), stream())

    def run(self, left):
        """(outputs, least time of 9 times of 10 calls in us) with `left` in the rows past the length."""
        self.kv[:, self.rows:] = left
        times = []
        for _ in range(9):
            a, b = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
            a.record()
            for _ in range(10):
                self.launch()
            b.record()
            torch.cuda.synchronize()
            times.append(a.elapsed_time(b) * 100)
        return self.o.clone(), min(times)


@pytest.mark.parametrize("hq,hkv,hd,n,prefix", CASES)
def test_rows_past_the_length_cost_nothing(gpu, hq, hkv, hd, n, prefix):
    """The same outputs, bit for bit, and about the same time whatever those rows hold. (Searched for what each row sees
    of them, a call takes 2 to 20 times as long; the margin is that of a noisy clock.)"""
    call = _Call(hq, hkv, hd, n, prefix)
    want, clean = call.run(0.0)
    for left in (math.nan, math.inf, -math.inf):
        got, other = call.run(left)
        print(f"zeros {clean:.1f} {left} {other:.1f} us")
        assert torch.equal(got, want)
        assert other < 1.5 * clean
