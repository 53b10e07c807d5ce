"""GPU tests of the filtered sampler over rows in which part of the vocabulary is masked (a grammar, banned ids, a
vocabulary's padding), against the plain 64-bit form (_draft_tree_ref). Tokens have to be equal."""
import math

import pytest
import torch

import _draft_tree_ref as R
import efm_capi as C
from _util import ptr, stream

pytestmark = pytest.mark.gpu

F32_MIN, BF16_MIN = torch.finfo(torch.float32).min, torch.finfo(torch.bfloat16).min
# largest logits on both sides of the powers of two: the keys' ranges then begin at other bits
TOPS = [1.5, 3.0, 6.0, 10.0, 20.0, 40.0, 100.0, 0.3, -0.7, -1.5, -3.0, -20.0]


def _sample(x, u, t=1.0, k=0, p=1.0, min_p=0.0):
    rows, vocab = x.shape
    out = torch.full((rows + 1,), -77, dtype=torch.int32, device="cuda")
    ws = torch.full((max(C.load().efm_sampler_filtered_workspace_bytes(rows, vocab), 256),), 0xff, dtype=torch.uint8, device="cuda")
    dt = C.EFM_DTYPE_BF16 if x.dtype == torch.bfloat16 else C.EFM_DTYPE_F32
    C.call("efm_sampler_filtered", rows, vocab, ptr(x), dt, 0, t, k, p, min_p, ptr(u), ptr(out), ptr(ws), ws.numel(), stream())
    torch.cuda.synchronize()
    assert int(out[rows]) == -77
    return out[:rows]


def _masked(seed, vocab, allowed, mask, dtype):
    """A row for each of TOPS: `allowed` ids with logits up to the top, `mask` everywhere else."""
    g = torch.Generator(device="cuda").manual_seed(seed)
    x = torch.full((len(TOPS), vocab), mask, device="cuda")
    for r, top in enumerate(TOPS):
        ids = torch.randperm(vocab, generator=g, device="cuda")[:allowed]
        x[r, ids] = top - 6 * torch.rand(allowed, generator=g, device="cuda")
        x[r, ids[allowed // 2]] = top
    return x.to(dtype), torch.rand(len(TOPS), generator=g, device="cuda")


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("mask", [-1e4, -1e9, -1e30, "lowest", -math.inf, math.nan])
@pytest.mark.parametrize("vocab", [300, 1000, 2048, 10000, 151936])
def test_fewer_and_more_allowed_ids_than_top_k(gpu, vocab, mask, dtype):
    value = (BF16_MIN if dtype == torch.bfloat16 else F32_MIN) if mask == "lowest" else mask
    for allowed in (1, 26, 290, 700, 3000):
        if allowed > vocab:
            continue
        x, u = _masked(vocab + allowed, vocab, allowed, value, dtype)
        for f in (dict(k=50), dict(k=50, p=0.9), dict(k=299), dict(k=700, min_p=0.01), dict(k=5000), dict(k=5000, p=0.7, t=3.0)):
            assert torch.equal(_sample(x, u, **f), R.sample(x, u, **f)), (allowed, f)


@pytest.mark.parametrize("f", [dict(k=5000), dict(k=5000, p=0.95), dict(p=0.95), dict(min_p=0.02)], ids=str)
@pytest.mark.parametrize("t", [0.7, 1e9])
def test_finite_masks_at_any_temperature(gpu, f, t):
    """A temperature at which masks of -1e9 have mass, and one at which they have none."""
    x, u = _masked(1, 30000, 3000, -1e9, torch.float32)
    assert torch.equal(_sample(x, u, t=t, **f), R.sample(x, u, t=t, **f))


@pytest.mark.parametrize("f", [dict(k=50), dict(k=50, p=0.99), dict(k=40, min_p=0.01)], ids=str)
@pytest.mark.parametrize("vocab", [10000, 151936])
@pytest.mark.parametrize("gap", [4e-36, 1e-30, 1e-7, 3e-38])
def test_groups_whose_maxima_are_close(gpu, gap, vocab, f):
    """Two groups of neighbouring ids are allowed, with largest logits that differ by next to nothing and others units
    below."""
    g = torch.Generator(device="cuda").manual_seed(4)
    x = torch.full((8, vocab), -math.inf, device="cuda")
    x[:, 256:272] = -1 - 4 * torch.rand(8, 16, generator=g, device="cuda")
    x[:, 1024:1040] = -1 - 4 * torch.rand(8, 16, generator=g, device="cuda")
    x[:, 260], x[:, 1030] = 0.0, -gap
    u = (torch.arange(8, device="cuda") + 0.5) / 8
    u[0], u[7] = 0.0, 1.0
    assert torch.equal(_sample(x, u, **f), R.sample(x, u, **f))


def _time(x, u, **f):
    """The least of 7 times of 10 calls, in us a call."""
    rows, vocab = x.shape
    out = torch.empty(rows, dtype=torch.int32, device="cuda")
    ws = torch.empty(max(C.load().efm_sampler_filtered_workspace_bytes(rows, vocab), 256), dtype=torch.uint8, device="cuda")
    times = []
    for _ in range(7):
        a, b = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
        a.record()
        for _ in range(10):
            C.call("efm_sampler_filtered", rows, vocab, ptr(x), C.EFM_DTYPE_F32, 0, 1.0, f["k"], f.get("p", 1.0), 0.0, ptr(u), ptr(out), ptr(ws),
                   ws.numel(), stream())
        b.record()
        torch.cuda.synchronize()
        times.append(a.elapsed_time(b) * 100)
    return min(times)


@pytest.mark.parametrize("mask", [-1e4, -1e9, "lowest"])
@pytest.mark.parametrize("rows,vocab,first", [(1, 151936, 151643), (33, 151936, 151643), (33, 151936, 2000), (4, 16000, 15000)])
def test_masked_ids_do_not_cost_the_short_list(gpu, rows, vocab, first, mask):
    """A few logits of a finite mask value, or nearly all of a row: the same tokens as with -inf, in about the same time. (With
    a list of all that is not -inf a call takes 20 to 40 times as long; the margin is that of a noisy clock.)"""
    g = torch.Generator(device="cuda").manual_seed(6)
    x = 2.5 * torch.randn(rows, vocab, generator=g, device="cuda")
    x[:, 7:1900:100] += 10
    masked, infinite = x.clone(), x.clone()
    masked[:, first:], infinite[:, first:] = F32_MIN if mask == "lowest" else mask, -math.inf
    u = torch.rand(rows, generator=g, device="cuda")
    for f in (dict(k=50), dict(k=200, p=0.9)):
        assert torch.equal(_sample(masked, u, **f), R.sample(infinite, u, **f))
        clean, other = _time(x, u, **f), _time(masked, u, **f)
        print(f"{f} clean {clean:.1f} masked {other:.1f} us")
        assert other < 3 * clean


@pytest.mark.parametrize("f", [dict(), dict(k=50), dict(k=3000, p=0.9), dict(p=0.9), dict(min_p=0.1)], ids=str)
@pytest.mark.parametrize("vocab", [5000, 60000])
def test_logits_near_the_ends_of_fp32(gpu, vocab, f):
    """The largest temperature, logits whose distances have mass and ones whose distance is no finite fp32 number."""
    g = torch.Generator(device="cuda").manual_seed(8)
    x = 3.3e38 - 4e37 * torch.rand(6, vocab, generator=g, device="cuda")
    x[:, ::3] = -3.3e38
    u = torch.rand(6, generator=g, device="cuda")
    assert torch.equal(_sample(x, u, t=1e36, **f), R.sample(x, u, t=1e36, **f))
