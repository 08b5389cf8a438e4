"""GPU tests of the 4-bit KV cache: store, read back, roll, decode and prefill attention against a plain 64-bit reference.

Tolerances.  Bytes of the cache are compared exactly: the format defines them.  A value read back is the exact m + d * code
rounded to fp16, half a step: 2^-11 of the value (2^-25 among the subnormals).  Decode is fp32 work: a weight e^(s - max) is off
by its exponent's absolute error -- scores are sums of products accumulated in fp32 on operands of 22 bits, at most
2^-20 of scale * sum |q_i k_i| -- and the exp2 unit's 2^-21; the output is a mean of values under such weights, so
it is off by at most (2 (2^-20 scale sum |q k| + 2^-21) + 2^-20) max |v|.  Prefill runs on fp16 operands: q and k are off by
2^-11 each, so a score by 2 * 2^-11 scale * sum |q_i k_i|, a weight by that and by its own rounding 2^-11, a value by 2^-11; the bound
is the sum of these times max |v| (and 2^-11 more for an fp16 output)."""
import math

import numpy as np
import pytest
import torch

import q4_reference as ref

pytestmark = pytest.mark.gpu


def dev(a):
    return torch.from_numpy(np.ascontiguousarray(a)).cuda()


def rows(rng, n, heads, hd):
    """Rows like those of a model: channels of different spread, a few with an offset."""
    spread = np.exp(0.4 * rng.standard_normal((heads, hd)))
    offset = 4.0 * rng.standard_normal((heads, hd)) * (rng.random((heads, hd)) < 0.05)
    return (rng.standard_normal((n, heads, hd)) * spread + offset).astype(np.float32)


def filled(rng, heads, hd, n_ctx, n):
    """A cache whose first n rows are written; the rest is garbage, NaN steps and offsets among it."""
    cache = rng.integers(0, 256, (heads, (n_ctx + 15) // 16, 18 * hd), dtype=np.uint8)
    cache[:, :, 16 * hd:] = 255
    if n:
        ref.write_rows(cache, hd, range(n), rows(rng, n, heads, hd), rows(rng, n, heads, hd))
    return cache


def decode_bound(most, scale, V):
    return (2 * (2.0 ** -20 * scale * most + 2.0 ** -21) + 2.0 ** -20) * np.abs(V).max()


def prefill_bound(most, scale, V, half):
    return (2 * 2.0 ** -11 * scale * most + 2 * 2.0 ** -11 + (2.0 ** -11 if half else 0)) * np.abs(V).max()


# ------------------------------------------------------------------------------------------------- store and load
@pytest.mark.parametrize("heads,hd,n_ctx,base,batch", [(2, 128, 64, 0, 64), (3, 64, 50, 7, 1), (1, 128, 33, 15, 18), (8, 64, 40, 16, 16),
                                                       (5, 128, 200, 3, 190), (1, 64, 1, 0, 1)])
def test_store_writes_the_formats_bytes_and_nothing_else(ops, heads, hd, n_ctx, base, batch):
    rng = np.random.default_rng(100)
    k, v = rows(rng, batch, heads, hd), rows(rng, batch, heads, hd)
    want = rng.integers(0, 256, (heads, (n_ctx + 15) // 16, 18 * hd), dtype=np.uint8)
    cache = dev(want)
    ops.kv_store_q4_batch(cache, dev(k), dev(v), heads, hd, n_ctx, base, batch)
    ref.write_rows(want, hd, range(base, base + batch), k, v)
    torch.cuda.synchronize()
    assert np.array_equal(cache.cpu().numpy(), want)
    # one row at a device position, over what is there; a position outside the cache writes nothing
    for pos, row in ((base, batch - 1), (n_ctx, 0), (-1, 0)):
        ops.kv_store_q4_ind(cache, dev(k[row]), dev(v[row]), heads, hd, n_ctx, torch.tensor([pos], dtype=torch.int32, device="cuda"))
        if 0 <= pos < n_ctx:
            ref.write_rows(want, hd, [pos], k[row: row + 1], v[row: row + 1])
    torch.cuda.synchronize()
    assert np.array_equal(cache.cpu().numpy(), want)


@pytest.mark.parametrize("hd", [64, 128])
def test_store_at_the_borders_of_the_quantiser(ops, hd):
    """Constant groups, zeros, ties between codes, subnormal steps, huge and non-finite values."""
    rng = np.random.default_rng(101)
    x = rng.standard_normal((40, 1, hd)).astype(np.float32)
    x[0], x[1], x[2] = 0, 1.0, 70.0 / 3
    x[3] = rng.integers(-30, 31, hd)                     # ties: halves of integer steps
    x[4] = np.tile(np.arange(16) * 2.0, hd // 16)        # step exactly 2
    x[5] = np.tile(np.arange(31) * 0.5, 5)[:hd]          # every second value lies between two codes
    x[6] *= 1e-7
    x[7] *= 1e-12
    x[8] *= 60000.0 / np.abs(x[8]).max()
    x[9, 0, 5] = np.inf
    x[10, 0, hd - 1] = np.nan
    x[11, 0, 3] = -1e6                                   # minimum beyond fp16
    x[12, 0, 3] = 1e5                                    # maximum beyond fp16 only: representable
    x[13] = -0.0
    x[14] = np.float32(1e-40)
    for i in range(15, 40):                              # ties by construction: m and d powers of two
        x[i] = rng.integers(0, 31, hd) * 0.5 - 4.0
        x[i, 0, 0], x[i, 0, hd - 1], x[i, 0, 63] = -4.0, -4.0 + 15.0, 11.0
        x[i, 0, hd - 64] = -4.0
    y = np.ascontiguousarray(x[::-1])
    want = np.zeros((1, 3, 18 * hd), np.uint8)
    cache = dev(want)
    ops.kv_store_q4_batch(cache, dev(x), dev(y), 1, hd, 40, 0, 40)
    torch.cuda.synchronize()
    got = cache.cpu().numpy()
    ref.write_rows(want, hd, range(40), x, y)
    gk, gv = ref.read_rows(got, hd, 40)
    wk, wv = ref.read_rows(want, hd, 40)
    for g, w in ((gk, wk), (gv, wv)):
        assert np.array_equal(np.isnan(g), np.isnan(w))
        assert np.array_equal(np.nan_to_num(g), np.nan_to_num(w))
    assert np.isnan(gk[0, 9]).any() and np.isnan(gk[0, 10]).any() and np.isnan(gk[0, 11]).any() and not np.isnan(gk[0, 12]).any()


@pytest.mark.parametrize("heads,hd,n_ctx,base,n", [(2, 128, 100, 0, 100), (3, 64, 77, 5, 1), (1, 128, 64, 15, 34), (4, 64, 300, 33, 250)])
def test_load_gives_the_rows_as_fp16(ops, heads, hd, n_ctx, base, n):
    rng = np.random.default_rng(102)
    cache = filled(rng, heads, hd, n_ctx, base + n)
    dst_ctx, dst_base = n + 9, 4
    kc = torch.full((heads, dst_ctx, hd), 7.0, dtype=torch.float16, device="cuda")
    vc = kc.clone()
    ops.kv_load_q4(dev(cache), kc, vc, heads, hd, n_ctx, base, n, dst_ctx, dst_base)
    torch.cuda.synchronize()
    for got, want in zip((kc, vc), ref.read_rows(cache, hd, base + n)):
        g = got.cpu().numpy().astype(np.float64)
        w = want[:, base:]
        assert (np.abs(g[:, dst_base: dst_base + n] - w) <= 2.0 ** -11 * (1 + 2.0 ** -11) * np.abs(w) + 2.0 ** -25).all()
        assert (g[:, :dst_base] == 7).all() and (g[:, dst_base + n:] == 7).all()


# ------------------------------------------------------------------------------------------------- roll
@pytest.mark.parametrize("layers,n_kv,hd,n_ctx,n_keep,shift", [(2, 3, 128, 1000, 4, 498), (3, 2, 64, 513, 0, 1), (1, 1, 128, 300, 10, 290),
                                                               (2, 2, 128, 512, 16, 128), (1, 2, 64, 17, 3, 7), (1, 1, 128, 1, 0, 1),
                                                               (1, 1, 64, 640, 33, 16)])
def test_shift_moves_rows_bytewise(ops, layers, n_kv, hd, n_ctx, n_keep, shift):
    rng = np.random.default_rng(103)
    heads = layers * n_kv
    cache = ops.KVCacheQ4(layers, n_kv, n_ctx, hd)
    before = filled(rng, heads, hd, n_ctx, n_ctx)
    cache.buf.copy_(dev(before).view_as(cache.buf))
    cache.shift(n_keep, shift)
    torch.cuda.synchronize()
    got = cache.buf.cpu().numpy().reshape(before.shape)
    for g, b in zip(ref.read_rows(got, hd, n_ctx), ref.read_rows(before, hd, n_ctx)):
        want = np.zeros_like(b)
        want[:, :n_keep] = b[:, :n_keep]
        want[:, n_keep: n_ctx - shift] = b[:, n_keep + shift:]
        assert np.array_equal(g, want)


# ------------------------------------------------------------------------------------------------- decode
SHAPES = [(12, 2, 128), (28, 4, 128), (8, 8, 128), (16, 1, 128), (9, 1, 64), (32, 8, 64), (13, 1, 128)]


@pytest.mark.parametrize("n_head,n_kv,hd", SHAPES)
@pytest.mark.parametrize("length", [1, 2, 16, 17, 129, 700])
def test_decode_appends_and_attends(ops, n_head, n_kv, hd, length):
    rng = np.random.default_rng(104 + length)
    n_ctx, rope_type, theta = length + 20, length % 2, 1e6
    cache = filled(rng, n_kv, hd, n_ctx, length - 1)
    q, k, v = rng.standard_normal((1, n_head, hd)).astype(np.float32), rows(rng, 1, n_kv, hd), rows(rng, 1, n_kv, hd)
    scale = 1.0 / math.sqrt(hd)
    d_cache, out = dev(cache), torch.full((n_head, hd), 9.0, device="cuda")
    pos = torch.tensor([length - 1], dtype=torch.int32, device="cuda")
    ops.attn_decode_q4(dev(q[0]), dev(k[0]), dev(v[0]), d_cache, out, n_head, n_kv, hd, n_ctx, pos, scale, ops.FUSE_ALL,
                       (rope_type, hd, theta, None))
    torch.cuda.synchronize()
    ref.write_rows(cache, hd, [length - 1], ref.rope(k, [length - 1], rope_type, hd, theta).astype(np.float32), v)
    assert np.array_equal(d_cache.cpu().numpy(), cache)
    K, V = ref.read_rows(cache, hd, length)
    want, most = ref.attend(ref.rope(q, [length - 1], rope_type, hd, theta), K, V, length - 1, scale)
    err = np.abs(out.cpu().numpy() - want[0]).max()
    assert err <= decode_bound(most, scale, V), (err, decode_bound(most, scale, V))


def long_cache(ops, heads, hd, n):
    """A long cache made on the GPU by the store call (checked above), and its rows in float64 on the GPU."""
    gen = torch.Generator(device="cuda").manual_seed(5)
    cache = ops.KVCacheQ4(1, heads, n, hd)
    k, v = (torch.randn(n, heads, hd, device="cuda", generator=gen) for _ in range(2))
    ops.kv_store_q4_batch(cache.layer(0), k, v, heads, hd, n, 0, n)
    even = np.arange(hd)
    out = []
    raw = cache.layer(0)
    for which in (0, 1):
        byte = np.stack([(ref.v_byte if which else ref.k_byte)(hd, s, even - even % 2) for s in range(16)]).reshape(-1)
        b = raw[:, :, torch.from_numpy(byte).cuda()].view(heads, -1, 16, hd)
        code = torch.where(torch.from_numpy(even % 2 == 1).cuda(), b >> 4, b & 15).double().view(heads, -1, hd // 64, 64)
        at = 16 * hd + which * hd
        sc = raw[:, :, at: at + hd].contiguous().view(torch.float16).view(heads, -1, hd // 64, 2).double()
        out.append((sc[..., 1:] + sc[..., :1] * code).view(heads, -1, hd)[:, :n])
    return raw, out[0], out[1]


@pytest.mark.parametrize("n_head,n_kv,hd,length", [(16, 2, 128, 40000), (32, 8, 64, 32001), (16, 1, 128, 9999), (4, 1, 128, 4097), (28, 4, 128, 2048)])
def test_decode_over_long_caches(ops, n_head, n_kv, hd, length):
    raw, K, V = long_cache(ops, n_kv, hd, length)
    q = torch.randn(n_head, hd, device="cuda", generator=torch.Generator(device="cuda").manual_seed(6))
    scale = 1.0 / math.sqrt(hd)
    out = torch.empty(n_head, hd, device="cuda")
    for n in (length, length - 1, length // 2 + 1):
        ops.attn_decode_q4(q, None, None, raw, out, n_head, n_kv, hd, length, torch.tensor([n - 1], dtype=torch.int32, device="cuda"),
                           scale, ops.FUSE_NONE)
        qd = q.double().view(n_kv, -1, hd)
        want = torch.softmax(qd @ K[:, :n].transpose(1, 2) * scale, -1) @ V[:, :n]
        most = float((qd.abs() @ K[:, :n].abs().transpose(1, 2)).max())
        err = float((out.view_as(want) - want).abs().max())
        assert err <= decode_bound(most, scale, V.cpu().numpy()), err


@pytest.mark.parametrize("amp_q,amp_k,amp_v", [(1e-4, 300.0, 1e-3), (300.0, 1e-3, 20000.0), (1.0, 1.0, 50.0), (1e-20, 1.0, 1e-5)])
def test_decode_keeps_its_accuracy_at_any_scale(ops, amp_q, amp_k, amp_v):
    """Steps far below and above one, among them those that make the kernel lower the scale of its weights half way."""
    rng = np.random.default_rng(110)
    n_head, n_kv, hd, n = 8, 1, 128, 333
    cache = np.zeros((n_kv, (n + 15) // 16, 18 * hd), np.uint8)
    k, v = amp_k * rows(rng, n, n_kv, hd), amp_v * rng.standard_normal((n, n_kv, hd))
    v[: n // 2] *= 0.01
    v = np.clip(v, -60000, 60000)
    ref.write_rows(cache, hd, range(n), k.astype(np.float32), v.astype(np.float32))
    q = (amp_q * rng.standard_normal((1, n_head, hd))).astype(np.float32)
    out = torch.empty(n_head, hd, device="cuda")
    scale = 0.3 / (amp_q * amp_k * hd)
    ops.attn_decode_q4(dev(q[0]), None, None, dev(cache), out, n_head, n_kv, hd, n, torch.tensor([n - 1], dtype=torch.int32, device="cuda"),
                       scale, ops.FUSE_NONE)
    K, V = ref.read_rows(cache, hd, n)
    want, most = ref.attend(q, K, V, n - 1, np.float32(scale))
    err = np.abs(out.cpu().numpy() - want[0]).max()
    assert err <= decode_bound(most, scale, V), (err, decode_bound(most, scale, V))


def test_decode_shows_a_nan_and_an_empty_cache_gives_zero(ops):
    rng = np.random.default_rng(111)
    n_head, n_kv, hd, n = 4, 2, 128, 40
    cache = filled(rng, n_kv, hd, n, n)
    bad = rows(rng, 1, n_kv, hd)
    bad[0, 1, 3] = np.nan
    ref.write_rows(cache, hd, [20], bad, rows(rng, 1, n_kv, hd))
    q = rng.standard_normal((n_head, hd)).astype(np.float32)
    out = torch.empty(n_head, hd, device="cuda")
    ops.attn_decode_q4(dev(q), None, None, dev(cache), out, n_head, n_kv, hd, n, torch.tensor([n - 1], dtype=torch.int32, device="cuda"), 0.1,
                       ops.FUSE_NONE)
    got = out.cpu().numpy()
    assert np.isfinite(got[:2]).all() and np.isnan(got[2:]).all()
    ops.attn_decode_q4(dev(q), None, None, dev(cache), out, n_head, n_kv, hd, n, torch.tensor([-1], dtype=torch.int32, device="cuda"), 0.1,
                       ops.FUSE_NONE)
    assert (out == 0).all()


# ------------------------------------------------------------------------------------------------- prefill
@pytest.mark.parametrize("half", [False, True])
@pytest.mark.parametrize("n_head,n_kv,hd,past,batch", [(12, 2, 128, 0, 1), (12, 2, 128, 0, 45), (8, 8, 128, 17, 33), (9, 3, 128, 130, 50), (4, 1, 64, 30, 19),
                                                       (32, 8, 64, 0, 3), (16, 1, 128, 5, 16), (5, 5, 64, 28, 8), (8, 8, 128, 60, 41),
                                                       # more (token, head) pairs than are taken from the 4-bit rows: the fp16 copies
                                                       (12, 2, 128, 20, 190), (8, 8, 128, 131, 140), (9, 3, 128, 130, 131), (4, 1, 64, 35, 530),
                                                       (32, 8, 64, 0, 70), (16, 16, 64, 0, 200), (12, 12, 128, 0, 100),
                                                       # ... cut into slices of at least 512 rows: 3, 5, 4, 5; 3, 3, 4
                                                       (8, 2, 128, 1500, 140), (5, 1, 128, 2500, 210), (9, 3, 128, 2000, 160), (32, 2, 128, 2560, 70),
                                                       (8, 8, 64, 1600, 260), (16, 1, 64, 1500, 129), (12, 4, 64, 2047, 190)])
def test_prefill_appends_and_attends(ops, n_head, n_kv, hd, past, batch, half):
    rng = np.random.default_rng(120)
    n_ctx, rope_type, theta = past + batch + 5, past % 2, 5e5
    cache = filled(rng, n_kv, hd, n_ctx, past)
    q, k, v = rng.standard_normal((batch, n_head, hd)).astype(np.float32), rows(rng, batch, n_kv, hd), rows(rng, batch, n_kv, hd)
    scale = 1.0 / math.sqrt(hd)
    d_cache = dev(cache)
    out = torch.full((batch + 1, n_head, hd), 9.0, dtype=torch.float16 if half else torch.float32, device="cuda")
    ops.attn_prefill_q4(dev(q), dev(k), dev(v), d_cache, out, n_head, n_kv, hd, n_ctx, past, batch, scale, ops.FUSE_ALL, (rope_type, hd, theta, None))
    torch.cuda.synchronize()
    pos = np.arange(past, past + batch)
    ref.write_rows(cache, hd, pos, ref.rope(k, pos, rope_type, hd, theta).astype(np.float32), v)
    assert np.array_equal(d_cache.cpu().numpy(), cache)
    K, V = ref.read_rows(cache, hd, past + batch)
    want, most = ref.attend(ref.rope(q, pos, rope_type, hd, theta), K, V, past, scale)
    got = out.float().cpu().numpy()
    err = np.abs(got[:batch] - want).max()
    assert err <= prefill_bound(most, scale, V, half), (err, prefill_bound(most, scale, V, half))
    assert (got[batch] == 9).all()
