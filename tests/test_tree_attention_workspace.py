"""CPU test that the tree attention's workspace query covers what calls ask for. A call without a workspace names its need and
is refused before any launch; where it needs none it would launch, and fails for want of a device."""
import random
import re

import pytest
import torch

import efm_capi as C

P = 4096   # an address that is never read

pytestmark = pytest.mark.skipif(torch.cuda.device_count() > 0, reason="calls that need no workspace would launch")


def _need(ctx, n, rows, device_len):
    lib = C.load()
    rc = lib.efm_attention_tree(ctx, P, P, P, P, P, n, 0 if device_len else rows, P if device_len else None, rows, None, 0, None)
    if rc != C.EFM_ERR_WORKSPACE:
        assert rc == C.EFM_ERR_DEVICE
        return 0
    return int(re.search(r"workspace of (\d+) bytes", lib.efm_last_error().decode()).group(1))


@pytest.mark.parametrize("hq,hkv,hd", [(14, 2, 64), (12, 2, 128), (16, 2, 128), (28, 4, 128), (8, 8, 64), (1, 1, 128), (64, 8, 128)])
def test_query_covers_every_smaller_call(hq, hkv, hd):
    """Sizes on both sides of the border between the two kernels, of one tile to hundreds of splits."""
    rng, ctx = random.Random(hq * hd), C.make_attention_ctx(hq, hkv, hd, rope=False)
    size, split, whole, tight = C.load().efm_attention_tree_workspace_bytes, 0, 0, 0.0
    for _ in range(1500):
        n = round(1024 ** rng.random())
        rows = n + round(2 ** (17 * rng.random()))
        need = _need(ctx, n, rows, rng.random() < 0.5)
        split, whole = split + (need > 0), whole + (need == 0)
        for n2, rows2 in ((n, rows), (rng.randint(n, 1024), rows), (n, rng.randint(rows, 1 << 18)), (rng.randint(n, 1024), rng.randint(rows, 1 << 18))):
            if rows2 >= n2:
                assert need <= size(ctx, n2, rows2), (n, rows, n2, rows2)
        tight = max(tight, need / max(size(ctx, n, rows), 1))
    assert split > 100 and whole > 100 and tight > 0.2   # both kinds were met, and the query is no arbitrary large number
