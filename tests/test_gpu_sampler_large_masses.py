"""GPU tests of the filtered sampler where a row's mass passes 2^63: more than 2^19 ids of nearly equal mass. The
expected tokens come from unsigned 64-bit sums and Python's integers."""
import math

import numpy as np
import pytest
import torch

import efm_capi as C
from _util import ptr, stream

pytestmark = pytest.mark.gpu

VOCAB = (1 << 20) - 1
DRAWS = [0.0, 0.1, 0.49, 0.5, 0.51, 0.6, 0.9, 0.999, 1 - 2.0 ** -24, 1.0, 3.0, math.inf, -1.0, math.nan]


def _sample(x, u, t, p, min_p, k):
    rows, vocab = x.shape
    out = torch.empty(rows, dtype=torch.int32, device="cuda")
    ws = torch.full((C.load().efm_sampler_filtered_workspace_bytes(rows, vocab),), 0xff, dtype=torch.uint8, device="cuda")
    dt = C.EFM_DTYPE_BF16 if x.dtype == torch.bfloat16 else C.EFM_DTYPE_F32
    C.call("efm_sampler_filtered", rows, vocab, ptr(x), dt, 0, t, k, p, min_p, ptr(u), ptr(out), ptr(ws), ws.numel(), stream())
    torch.cuda.synchronize()
    return out.tolist()


def _expected(row, draws, t, p, min_p, k):
    """Tokens of one row of finite logits."""
    f32 = np.float32
    x = row.astype(np.float64)
    w = np.rint(np.exp((x - x.max()) / float(f32(t))) * 2.0 ** 44).astype(np.uint64)
    order = np.argsort(-x, kind="stable")
    order = order[:k] if k > 0 else order
    order = order[w[order] >= max(1, math.ceil(float(f32(min_p)) * 2.0 ** 44))]
    mass = np.cumsum(w[order], dtype=np.uint64)
    if p < 1:
        need = max(1, math.ceil(float(f32(p)) * float(int(mass[-1]))))
        order = order[:int(np.searchsorted(mass, np.uint64(need), side="left")) + 1]
    ids = np.sort(order)
    mass = np.cumsum(w[ids], dtype=np.uint64)
    total, tokens = int(mass[-1]), []
    for u in draws:
        u = 0.0 if math.isnan(u) else min(max(float(f32(u)), 0.0), 1.0)
        r = min(int(u * float(total)), total - 1)
        tokens.append(int(ids[int(np.searchsorted(mass, np.uint64(r), side="right"))]))
    return tokens


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("f", [dict(), dict(p=0.7), dict(p=0.4), dict(min_p=0.5), dict(k=VOCAB - 1), dict(k=900000, p=0.9)], ids=str)
@pytest.mark.parametrize("kind", ["equal", "flat", "uneven"])
def test_draws_over_all_of_the_mass(gpu, dtype, f, kind):
    """Equal logits, nearly equal ones (a high temperature), and a bulk beside lighter ids."""
    g = torch.Generator().manual_seed(1)
    x, t = torch.randn(VOCAB, generator=g), 1.0
    if kind == "equal":
        x = torch.full((VOCAB,), 2.0)
    elif kind == "flat":
        t = 1e6
    else:
        x = torch.where(x < -1.5, -0.5 - 0.1 * x.abs(), torch.zeros(()))
    x = x.to(dtype)
    args = (t, f.get("p", 1.0), f.get("min_p", 0.0), f.get("k", 0))
    u = torch.tensor(DRAWS, device="cuda")
    got = _sample(x.cuda().expand(len(DRAWS), -1).contiguous(), u, *args)
    assert got == _expected(x.float().numpy(), DRAWS, *args)
