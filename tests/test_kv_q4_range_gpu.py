"""GPU tests of the 4-bit cache over its range: long sums, steps far apart, values beyond fp16, long rolls.  Tolerances not derived
here: test_kv_q4_gpu.py."""
import math

import numpy as np
import pytest
import torch

from test_kv_q4_gpu import long_cache, prefill_bound

pytestmark = pytest.mark.gpu


# ------------------------------------------------------------------------------------------------- sums over long contexts
def powers_of_two(ops, n_kv, hd, n, seed):
    """A cache of n rows whose scores against q = (1, 0, ...) are whole numbers from -7 to 0 and whose values are one fp16 number of
    [1, 2) per row and group.  With weights that are powers of two and values that fp16 holds, attention rounds nothing but its sums."""
    gen = torch.Generator(device="cuda").manual_seed(seed)
    cache = ops.KVCacheQ4(1, n_kv, n, hd).layer(0)
    k = torch.zeros(n, n_kv, hd, device="cuda")
    k[..., 0] = -torch.randint(0, 8, (n, n_kv), device="cuda", generator=gen).float()
    k[::128, :, 0] = 0
    v = (1 + torch.rand(n, n_kv, hd // 64, device="cuda", generator=gen)).half().float()
    ops.kv_store_q4_batch(cache, k, v.repeat_interleave(64, -1), n_kv, hd, n, 0, n)
    w = torch.exp2(k[..., 0].double())
    return cache, w, v.double()


# 32/8 heads: whole tiles; one kv head: its rows in slices
@pytest.mark.parametrize("n_head,n_kv,hd,past,batch,slices", [(32, 8, 128, 131072, 512, 1), (32, 8, 64, 131072, 512, 1), (16, 1, 128, 131072, 140, 8),
                                                              (16, 1, 64, 200000, 140, 8), (32, 8, 128, 7800, 512, 1), (12, 4, 128, 8000, 1111, 1)])
@pytest.mark.parametrize("half", [False, True])
def test_a_long_chunk_keeps_its_sums(ops, n_head, n_kv, hd, past, batch, slices, half):
    """The tensor core's additions cut off, and what they cut off adds up with the rows of one sum: at most 63 blocks of 128 are in
    one, eight products each, a product up to two last places short (2 * 2^-23) of the sum so far, on average half of the whole.  The
    sum of the weights is rounded to nearest once per block and softmax team, and 2^-20 is left for the rest."""
    n = past + batch
    cache, w, v = powers_of_two(ops, n_kv, hd, n, 400)
    q = torch.zeros(batch, n_head, hd, device="cuda")
    q[..., 0] = 1
    out = torch.empty(batch, n_head, hd, dtype=torch.float16 if half else torch.float32, device="cuda")
    ops.attn_prefill_q4(q, None, None, cache, out, n_head, n_kv, hd, n, past, batch, float(np.log(2.0)), ops.FUSE_NONE)
    want = (torch.cumsum(w[..., None] * v, 0) / torch.cumsum(w, 0)[..., None])[past:]              # [batch][n_kv][groups]
    want = want.repeat_interleave(n_head // n_kv, 1).repeat_interleave(64, -1)
    err = float(((out.double() - want) / want).abs().max())
    bound = 63 * 8 * 2.0 ** -23 + (n / slices / 256 + 2) * 2.0 ** -24 + 2.0 ** -20 + (2.0 ** -11 if half else 0)
    assert err <= bound, (err, bound)
    assert ops.prefill_status(n_head, n_kv, hd, batch, ops.prefill_q4_workspace(n_head, n_kv, hd, batch, n)) == 0


@pytest.mark.parametrize("n_head,n_kv,hd,past,batch", [(32, 8, 128, 8192, 512), (32, 8, 64, 20000, 512), (16, 2, 128, 70000, 512), (12, 4, 128, 8003, 1111)])
def test_a_long_chunk_repeats_itself(ops, n_head, n_kv, hd, past, batch):
    """Rows whose maxima move along the context, several times over: the same bits, and within the bound of the fp16 operands."""
    n, scale = past + batch, 1.0 / math.sqrt(hd)
    raw, K, V = long_cache(ops, n_kv, hd, n)
    gen = torch.Generator(device="cuda").manual_seed(401)
    q = 2 * torch.randn(batch, n_head, hd, device="cuda", generator=gen)
    outs = [torch.empty(batch, n_head, hd, device="cuda") for _ in range(6)]
    for out in outs:
        ops.attn_prefill_q4(q, None, None, raw, out, n_head, n_kv, hd, n, past, batch, scale, ops.FUSE_NONE)
    assert all(torch.equal(out, outs[0]) for out in outs)
    unseen = torch.arange(n, device="cuda")[None] > torch.arange(past, n, device="cuda")[:, None]
    for h in (0, n_head - 1):
        k, v, x = K[h * n_kv // n_head], V[h * n_kv // n_head], q[:, h].double()
        want = torch.softmax((x @ k.T * scale).masked_fill(unseen, -math.inf), -1) @ v
        bound = prefill_bound(float((x.abs() @ k.abs().T).max()), scale, v.cpu().numpy(), False)
        assert float((outs[0][:, h] - want).abs().max()) <= bound
        # ... which is for the worst case: roundings of random sign leave a tenth of it in the mean
        assert float((outs[0][:, h] - want).norm() / want.norm()) <= 1e-3
