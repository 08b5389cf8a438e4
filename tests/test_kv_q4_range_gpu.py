"""GPU tests of the 4-bit cache over its range: long sums, steps that are small or far apart, values beyond fp16, long rolls.
Tolerances that are not derived here: test_kv_q4_gpu.py."""
import math

import numpy as np
import pytest
import torch

import q4_reference as ref
from test_kv_q4_gpu import decode_bound, dev, filled, long_cache, prefill_bound, rows

pytestmark = pytest.mark.gpu


def dpos(p):
    return torch.tensor([p], dtype=torch.int32, device="cuda")


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


@pytest.mark.parametrize("n_head,n_kv,hd,past,batch,half", [(32, 8, 128, 9000, 512, False), (16, 1, 64, 70000, 140, True)])
def test_a_long_chunk_captured(ops, n_head, n_kv, hd, past, batch, half):
    """A call whose sums pass through the workspace, replayed over a workspace that held something else in between: the same bits."""
    n, scale = past + batch, 1.0 / math.sqrt(hd)
    raw, _, _ = long_cache(ops, n_kv, hd, n)
    gen = torch.Generator(device="cuda").manual_seed(402)
    q = 2 * torch.randn(batch, n_head, hd, device="cuda", generator=gen)
    kn, vn = (torch.randn(batch, n_kv, hd, device="cuda", generator=gen) for _ in range(2))
    ws = torch.empty(ops.prefill_q4_workspace(n_head, n_kv, hd, batch, n).numel(), dtype=torch.uint8, device="cuda")
    want, got = (torch.zeros(batch, n_head, hd, dtype=torch.float16 if half else torch.float32, device="cuda") for _ in range(2))

    def call(out):
        ops.attn_prefill_q4(q, kn, vn, raw, out, n_head, n_kv, hd, n, past, batch, scale, ops.FUSE_ALL, (1, hd, 1e6, None), ws)

    call(want)
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        call(got)
    for fill in (0, 255):                                  # (255: NaN wherever it is read as a number)
        got.zero_()
        ws.fill_(fill)
        g.replay()
        torch.cuda.synchronize()
        assert torch.equal(got, want) and bool(torch.isfinite(got).all())


# ------------------------------------------------------------------------------------------------- steps
def repeated_row(rng, n_kv, hd, n, step, at, amp=1.0):
    """A cache of n rows that are all alike -- K zero, V of about 15 steps -- but for row `at`, whose K is amp times a random row and
    whose V is zero.  The cache (on the GPU; every kv head the same), K and V of row `at`, V of the others."""
    block = np.zeros((1, 1, 18 * hd), np.uint8)
    zero = np.zeros((16, 1, hd), np.float32)
    v = (step * rng.integers(0, 16, (1, 1, hd))).astype(np.float32)
    v[..., ::64], v[..., 1::64] = 0, 15 * step
    ref.write_rows(block, hd, range(16), zero, np.repeat(v, 16, 0))
    cache = dev(block).expand(n_kv, (n + 15) // 16, 18 * hd).contiguous()
    k = (amp * rng.standard_normal((1, 1, hd))).astype(np.float32)
    ref.write_rows(block, hd, [at % 16], k, zero[:1])
    cache[:, at // 16] = dev(block[:, 0])
    K, V = ref.read_rows(block, hd, 16)
    return cache, K[0, at % 16], V[0, (at + 1) % 16]


def repeated_row_attention(q, k, v, n, scale):
    """q [n_head][hd] over that cache: n - 1 rows of score 0 and value v, one of score q . k and value 0.  And the bound's `most`."""
    s = (q.astype(np.float64) @ k) * np.float32(scale)
    rest = (n - 1) * np.exp(-s)
    return (rest / (1 + rest))[:, None] * v, float((np.abs(q.astype(np.float64)) @ np.abs(k)).max())


# Many kv heads leave one CTA to each, whose eight warps walk 885 rows apiece.
@pytest.mark.parametrize("step", [1e-2, 1e-4, 1e-5, 2.0 ** -24])
@pytest.mark.parametrize("group,hd", [(1, 64), (3, 128), (4, 64), (8, 64), (8, 128)])
def test_decode_counts_small_values_behind_a_dominant_row(ops, group, hd, step):
    """One row has nearly all of the weight, the others a sum of weights of the size of the bound ten times over: what they add to the
    output is not lost, however small the steps of their values."""
    rng = np.random.default_rng(300)
    n_kv, n, at = 160, 8 * 885, 1234
    n_head, scale = n_kv * group, 1.0 / math.sqrt(hd)
    cache, k, v = repeated_row(rng, n_kv, hd, n, step, at)
    # the dominant row's score is 13 to 17
    q = np.stack([k * (13 + 4 * i / group) / (scale * (k @ k)) for i in range(group)]).astype(np.float32)
    out = torch.empty(n_head, hd, device="cuda")
    ops.attn_decode_q4(dev(np.tile(q, (n_kv, 1))), None, None, cache, out, n_head, n_kv, hd, n, dpos(n - 1), scale, ops.FUSE_NONE)
    want, most = repeated_row_attention(q, k, v, n, scale)
    err = np.abs(out.view(n_kv, group, hd).cpu().numpy() - want).max()
    assert err <= decode_bound(most, scale, v), (err, decode_bound(most, scale, v))


@pytest.mark.parametrize("step", [1e-2, 1e-5])
@pytest.mark.parametrize("hd", [64, 128])
def test_short_chunk_counts_small_values_behind_a_dominant_row(ops, hd, step):
    rng = np.random.default_rng(301)
    n_kv, group, batch = 24, 4, 2
    n, at, scale = 12 * 8 * 885, 1234, 1.0 / math.sqrt(hd)
    n_head = n_kv * group
    cache, k, v = repeated_row(rng, n_kv, hd, n, step, at)
    q = np.stack([k * (13 + 4 * i / group) / (scale * (k @ k)) for i in range(group)]).astype(np.float32)
    out = torch.empty(batch, n_head, hd, device="cuda")
    ops.attn_prefill_q4(dev(np.tile(q, (batch, n_kv, 1))), None, None, cache, out, n_head, n_kv, hd, n, n - batch, batch, scale, ops.FUSE_NONE)
    for b in range(batch):
        want, most = repeated_row_attention(q, k, v, n - batch + b + 1, scale)
        err = np.abs(out[b].view(n_kv, group, hd).cpu().numpy() - want).max()
        assert err <= decode_bound(most, scale, v), (err, decode_bound(most, scale, v))


AMPLITUDES = {"growing": lambda n: np.logspace(-6, 4, n), "falling": lambda n: np.logspace(4, -6, n),
              "one large": lambda n: np.where(np.arange(n) == n // 3, 1e4, 1e-3), "none, then small": lambda n: np.where(np.arange(n) < n // 2, 0, 1e-5)}


@pytest.mark.parametrize("order", sorted(AMPLITUDES))
@pytest.mark.parametrize("n_head,n_kv,hd", [(2, 2, 128), (3, 1, 64), (8, 2, 128), (4, 1, 64), (8, 1, 64), (14, 2, 128), (16, 1, 128)])
def test_decode_with_steps_far_apart(ops, n_head, n_kv, hd, order):
    """Steps that grow, fall or jump along the context: those of ten orders of magnitude are summed in one scale after another."""
    rng = np.random.default_rng(302)
    n, scale = 1500, 0.3 / math.sqrt(hd)
    k, v = rows(rng, n, n_kv, hd), rng.standard_normal((n, n_kv, hd)).clip(-6, 6)
    v = (v * AMPLITUDES[order](n)[:, None, None]).astype(np.float32)
    cache = np.zeros((n_kv, (n + 15) // 16, 18 * hd), np.uint8)
    ref.write_rows(cache, hd, range(n), k, v)
    K, V = ref.read_rows(cache, hd, n)
    q = rng.standard_normal((1, n_head, hd)).astype(np.float32)
    out = torch.empty(n_head, hd, device="cuda")
    for length in (n, 500, 40):
        ops.attn_decode_q4(dev(q[0]), None, None, dev(cache), out, n_head, n_kv, hd, n, dpos(length - 1), scale, ops.FUSE_NONE)
        want, most = ref.attend(q, K[:, :length], V[:, :length], length - 1, scale)
        err = np.abs(out.cpu().numpy() - want[0]).max()
        assert err <= decode_bound(most, scale, V[:, :length]), (length, err, decode_bound(most, scale, V[:, :length]))


@pytest.mark.parametrize("n_head,n_kv,hd", [(2, 2, 64), (8, 2, 128), (4, 1, 64), (7, 1, 64), (14, 2, 128), (16, 1, 128)])
@pytest.mark.parametrize("amp_old,amp_new", [(1e-3, 9000.0), (0.01, 400.0), (9000.0, 1e-3), (1.0, 1.0)])
def test_decode_with_a_step_of_its_own_for_the_appended_row(ops, n_head, n_kv, hd, amp_old, amp_new):
    rng = np.random.default_rng(303)
    scale = 1.0 / math.sqrt(hd)
    for length in (1, 17, 300, 1030):
        cache = np.zeros((n_kv, (length + 20) // 16 + 1, 18 * hd), np.uint8)
        n_ctx = 16 * cache.shape[1]
        k, v = rows(rng, length, n_kv, hd), rng.standard_normal((length, n_kv, hd)).clip(-6, 6)
        v[:-1] *= amp_old
        v[-1] *= amp_new
        v = v.astype(np.float32)
        if length > 1:
            ref.write_rows(cache, hd, range(length - 1), k[:-1], v[:-1])
        q = rng.standard_normal((1, n_head, hd)).astype(np.float32)
        d_cache, out = dev(cache), torch.empty(n_head, hd, device="cuda")
        ops.attn_decode_q4(dev(q[0]), dev(k[-1]), dev(v[-1]), d_cache, out, n_head, n_kv, hd, n_ctx, dpos(length - 1), scale, ops.FUSE_KV_APPEND)
        ref.write_rows(cache, hd, [length - 1], k[-1:], v[-1:])
        assert np.array_equal(d_cache.cpu().numpy(), cache)
        K, V = ref.read_rows(cache, hd, length)
        want, most = ref.attend(q, K, V, length - 1, scale)
        err = np.abs(out.cpu().numpy() - want[0]).max()
        assert err <= decode_bound(most, scale, V), (length, err, decode_bound(most, scale, V))


@pytest.mark.parametrize("bad", [1e6, np.nan])
@pytest.mark.parametrize("n_head,n_kv,chunk", [(4, 1, 0), (8, 1, 0), (8, 1, 3)])
def test_a_step_that_is_not_finite_stays_in_its_group(ops, n_head, n_kv, chunk, bad):
    """A range beyond 15 fp16 steps, or a NaN, in the first 64 values of a row: the other 64 of the output are what they would be."""
    rng = np.random.default_rng(304)
    hd, n, scale = 128, 333, 0.0884
    cache = filled(rng, n_kv, hd, n, n)
    v = rows(rng, 1, n_kv, hd)
    v[0, :, 3] = bad
    ref.write_rows(cache, hd, [200], rows(rng, 1, n_kv, hd), v)
    m = max(chunk, 1)
    q = rng.standard_normal((m, n_head, hd)).astype(np.float32)
    out = torch.empty(m, n_head, hd, device="cuda")
    if chunk:
        ops.attn_prefill_q4(dev(q), None, None, dev(cache), out, n_head, n_kv, hd, n, n - m, m, scale, ops.FUSE_NONE)
    else:
        ops.attn_decode_q4(dev(q[0]), None, None, dev(cache), out[0], n_head, n_kv, hd, n, dpos(n - 1), scale, ops.FUSE_NONE)
    K, V = ref.read_rows(cache, hd, n)
    assert not np.isfinite(V[:, 200, :64]).any() and np.isfinite(np.delete(V, 200, 1)).all()
    want, most = ref.attend(q, K, np.nan_to_num(V), n - m, scale)
    got = out.cpu().numpy()
    assert not np.isfinite(got[..., :64]).any()
    assert np.abs(got[..., 64:] - want[..., 64:]).max() <= decode_bound(most, scale, V[..., 64:])


# ------------------------------------------------------------------------------------------------- values beyond fp16
@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("batch", [1, 5, 600])
@pytest.mark.parametrize("which,where", [("k", 7), ("v", 7), ("k", 40), ("v", 40)])
def test_a_value_beyond_fp16(ops, which, where, batch, hd):
    """The format holds 1e5 behind a minimum and a step that fit fp16.  Decode and a short chunk work on the codes; a long chunk works on
    fp16 copies, where such a row is NaN and shows, and is never another finite number.  Row 7 lies in front of the chunk, row 40 is
    its first."""
    rng = np.random.default_rng(305)
    n_head, n_kv, past, scale = 4, 2, 40, 1.0 / math.sqrt(hd)
    n = past + batch
    q, k, v = rng.standard_normal((batch, n_head, hd)).astype(np.float32), rows(rng, n, n_kv, hd), rows(rng, n, n_kv, hd)
    q[..., :64] *= 1e-5 if which == "k" else 1
    (k if which == "k" else v)[where, 1, 3] = 1e5
    q[..., 3] = -np.abs(q[..., 3])
    cache = np.zeros((n_kv, (n + 15) // 16, 18 * hd), np.uint8)
    ref.write_rows(cache, hd, range(past), k[:past], v[:past])
    d_cache, out = dev(cache), torch.empty(batch, n_head, hd, device="cuda")
    if batch == 1:
        ops.attn_decode_q4(dev(q[0]), dev(k[past]), dev(v[past]), d_cache, out[0], n_head, n_kv, hd, n, dpos(past), scale, ops.FUSE_KV_APPEND)
    else:
        ops.attn_prefill_q4(dev(q), dev(k[past:]), dev(v[past:]), d_cache, out, n_head, n_kv, hd, n, past, batch, scale, ops.FUSE_KV_APPEND)
    ref.write_rows(cache, hd, range(past, n), k[past:], v[past:])
    assert np.array_equal(d_cache.cpu().numpy(), cache)
    K, V = ref.read_rows(cache, hd, n)
    assert (K if which == "k" else V)[1, where].max() > 65520
    want, most = ref.attend(q, K, V, past, scale)
    got = out.cpu().numpy()
    if batch < 100:
        assert np.abs(got - want).max() <= decode_bound(most, scale, V)
        return
    # the first kv head's heads have nothing to do with it, nor has the second half of V
    assert np.abs(got[:, :2] - want[:, :2]).max() <= prefill_bound(most, scale, V[0], False)
    if which == "k":
        assert np.isnan(got[:, 2:]).all()
    else:
        assert np.isnan(got[:, 2:, :64]).all()
        if hd == 128:
            assert np.abs(got[:, 2:, 64:] - want[:, 2:, 64:]).max() <= prefill_bound(most, scale, V[1, :, 64:], False)
    # read back, the value is the nearest fp16 number
    kh, vh = (torch.empty(n_kv, n, hd, dtype=torch.float16, device="cuda") for _ in range(2))
    ops.kv_load_q4(d_cache, kh, vh, n_kv, hd, n, 0, n)
    assert float((kh if which == "k" else vh)[1, where, 3]) == math.inf


# ------------------------------------------------------------------------------------------------- rolls of many steps
def row_bytes(cache, hd, which):
    """Codes (a byte per pair of dims) and scales of every row of a cache on the GPU, uint8 [heads][rows][bytes]."""
    even = np.arange(0, hd, 2)
    at = np.stack([(ref.v_byte if which else ref.k_byte)(hd, s, even) for s in range(16)])
    scale = 16 * hd + which * hd + np.arange(hd).reshape(16, -1)
    at = torch.from_numpy(np.concatenate((at, scale), 1)).cuda()
    return cache[..., at.reshape(-1)].view(cache.shape[0], -1, at.shape[1])


@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("n_layer,n_kv,n_ctx,n_keep,shift", [(1, 2, 2049, 0, 1), (2, 2, 4000, 7, 13), (1, 3, 5000, 20, 16), (1, 2, 12345, 1000, 5555),
                                                             (2, 1, 30011, 3, 511), (1, 1, 8192, 5, 4094), (1, 2, 6000, 100, 5900), (1, 1, 2600, 515, 512)])
def test_a_roll_of_many_steps(ops, hd, n_layer, n_kv, n_ctx, n_keep, shift):
    """Contexts of more steps than are in flight at once, so that a window is filled while another leaves and used again: every byte."""
    gen = torch.Generator(device="cuda").manual_seed(306)
    cache = ops.KVCacheQ4(n_layer, n_kv, n_ctx, hd)
    cache.buf.copy_(torch.randint(0, 256, cache.buf.shape, dtype=torch.uint8, device="cuda", generator=gen))
    before = cache.buf.view(n_layer * n_kv, -1, 18 * hd).clone()
    for _ in range(2):                                     # the second one rolls what the first one left
        cache.shift(n_keep, shift)
        after = cache.buf.view_as(before)
        for which in (0, 1):
            want, got = row_bytes(before, hd, which), row_bytes(after, hd, which)
            moved = torch.cat((want[:, :n_keep], want[:, n_keep + shift: n_ctx], torch.zeros_like(want[:, :shift]), want[:, n_ctx:]), 1)
            assert torch.equal(got, moved)
        before = after.clone()


# ------------------------------------------------------------------------------------------------- what stands around the attention
def test_block_output_of_a_long_context(ops):
    """The blocks next to the fp32 output and instead of it, behind more rows than go into one sum."""
    n_head, n_kv, hd, past, batch = 8, 2, 128, 9000, 149
    n = past + batch
    raw, _, V = long_cache(ops, n_kv, hd, n)
    q = torch.randn(batch, n_head, hd, device="cuda", generator=torch.Generator(device="cuda").manual_seed(307))
    f32, blk = torch.empty(batch, n_head, hd, device="cuda"), [torch.zeros(n_head * batch * 144, dtype=torch.uint8, device="cuda") for _ in range(2)]
    for out, b in ((f32, blk[0]), (None, blk[1])):
        ops.attn_prefill_q4(q, None, None, raw, out, n_head, n_kv, hd, n, past, batch, 0.0884, ops.FUSE_NONE, ext=dict(out_mmq=b))
    assert torch.equal(blk[0], blk[1])
    b = blk[0].view(n_head, batch, 144)
    d = b[..., :16].contiguous().view(torch.float32)
    val = (b[..., 16:].contiguous().view(torch.int8).view(n_head, batch, 4, 32).float() * d[..., None]).reshape(n_head, batch, hd).transpose(0, 1)
    assert ((val - f32).abs() <= 0.5001 * d.transpose(0, 1).repeat_interleave(32, -1) + 1e-7).all()
    # Without the blocks the rows are cut into slices, whose weights are relative to maxima of their own: both calls round each weight to
    # fp16, by 2^-11 of it at most, so the two means of the values lie within twice that of the largest value, and the sums' share.
    other = torch.empty_like(f32)
    ops.attn_prefill_q4(q, None, None, raw, other, n_head, n_kv, hd, n, past, batch, 0.0884, ops.FUSE_NONE)
    assert float((other - f32).abs().max()) <= (2 * 2.0 ** -11 + 2 * 63 * 8 * 2.0 ** -23) * float(V.abs().max())


@pytest.mark.parametrize("batch", [1, 4, 200])
def test_a_bias_at_any_address(ops, batch):
    """Biases are read one number at a time: those of a packed parameter block may begin anywhere."""
    rng = np.random.default_rng(308)
    n_head, n_kv, hd, past = 12, 4, 64, 30
    n, scale, rope = past + batch, 0.125, (1, hd, 1e4, None)
    base, q = dev(filled(rng, n_kv, hd, n, past)), dev(rng.standard_normal((batch, n_head, hd)).astype(np.float32))
    k, v = (dev(rows(rng, batch, n_kv, hd)) for _ in range(2))
    sizes = [n_head * hd, n_kv * hd, n_kv * hd]
    packed = dev(rng.standard_normal(sum(sizes) + 3).astype(np.float32))
    res = []
    for shift in (0, 1, 3):
        where = packed.new_empty(packed.numel() + 3)
        where[shift: shift + packed.numel()] = packed
        bias = dict(zip(("bias_q", "bias_k", "bias_v"), where[shift:].split(sizes + [where.numel() - shift - sum(sizes)])))
        cache, out = base.clone(), torch.empty(batch, n_head, hd, device="cuda")
        if batch == 1:
            ops.attn_decode_q4(q[0], k[0], v[0], cache, out[0], n_head, n_kv, hd, n, dpos(past), scale, ops.FUSE_ALL, rope, ext=bias)
        else:
            ops.attn_prefill_q4(q, k, v, cache, out, n_head, n_kv, hd, n, past, batch, scale, ops.FUSE_ALL, rope, ext=bias)
        res.append((cache, out))
    assert all(torch.equal(x, y) for r in res for x, y in zip(r, res[0]))


def test_extras_on_another_device_are_refused(ops):
    c, x = ops.KVCacheQ4(1, 2, 64, 128).layer(0), torch.zeros(1, 2, 128, device="cuda")
    good = dict(bias_q=torch.zeros(256, device="cuda"))
    ops.attn_decode_q4(x, x, x, c, x.clone(), 2, 2, 128, 64, dpos(0), 0.1, ops.FUSE_KV_APPEND, ext=good)
    for bad in (dict(bias_q=torch.zeros(256)), dict(norm_k=torch.zeros(128)), dict(bias_q=torch.zeros(128, device="cuda"))):
        with pytest.raises(ValueError, match=list(bad)[0] + ": "):
            ops.attn_decode_q4(x, x, x, c, x.clone(), 2, 2, 128, 64, dpos(0), 0.1, ops.FUSE_KV_APPEND, ext=bad)
        with pytest.raises(ValueError, match=list(bad)[0] + ": "):
            ops.attn_prefill_q4(x, x, x, c, x.clone(), 2, 2, 128, 64, 0, 1, 0.1, ops.FUSE_KV_APPEND, ext=bad)
