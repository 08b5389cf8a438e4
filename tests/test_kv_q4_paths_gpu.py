"""GPU tests of the 4-bit cache's calls as a program makes them: bias, norm and quantised outputs around them, partial rotation,
launch overlap, graphs, streams, a whole conversation, large caches, and refusals.  Tolerances: test_kv_q4_gpu.py."""
import math

import numpy as np
import pytest
import torch

import q4_reference as ref
from test_kv_q4_gpu import decode_bound, dev, filled, prefill_bound, rows

pytestmark = pytest.mark.gpu


def dpos(p):
    return torch.tensor([p], dtype=torch.int32, device="cuda")


def normed(x, bias, w, eps):
    x = x.astype(np.float32) + bias.astype(np.float32)
    if w is None:
        return x
    x = x.astype(np.float64)
    return (x / np.sqrt((x ** 2).mean(-1, keepdims=True) + eps) * w).astype(np.float32)


@pytest.mark.parametrize("batch", [21, 140])
@pytest.mark.parametrize("n_head,n_kv,hd,n_rot,rope_type,norm", [(12, 2, 128, 128, 1, True), (14, 2, 64, 32, 1, False), (8, 8, 128, 96, 0, False),
                                                                (20, 2, 64, 64, 0, True)])
def test_bias_norm_and_partial_rotation_in_front(ops, n_head, n_kv, hd, n_rot, rope_type, norm, batch):
    """A chunk through the prefill call and one more token through the decode call."""
    rng = np.random.default_rng(200)
    past, n_ctx, theta, eps = 19, 200, 1e4, 1e-6
    cache = filled(rng, n_kv, hd, n_ctx, past)
    n = batch + 1
    q, k, v = rng.standard_normal((n, n_head, hd)).astype(np.float32), rows(rng, n, n_kv, hd), rows(rng, n, n_kv, hd)
    ff = (1 + rng.random(n_rot // 2)).astype(np.float32)
    b = {m: rng.standard_normal((h, hd)).astype(np.float32) for m, h in (("bias_q", n_head), ("bias_k", n_kv), ("bias_v", n_kv))}
    w = {m: (1 + 0.2 * rng.standard_normal(hd)).astype(np.float32) for m in ("norm_q", "norm_k")} if norm else {}
    ext = {m: dev(x) for m, x in {**b, **w}.items()}
    if norm:
        ext["norm_eps"] = eps
    d_cache, d_ff = dev(cache), dev(ff)
    rope, scale = (rope_type, n_rot, theta, d_ff), 1.0 / math.sqrt(hd)
    out = torch.empty(n, n_head, hd, device="cuda")
    ops.attn_prefill_q4(dev(q[:batch]), dev(k[:batch]), dev(v[:batch]), d_cache, out[:batch], n_head, n_kv, hd, n_ctx, past, batch, scale,
                        ops.FUSE_ALL, rope, ext=ext)
    ops.attn_decode_q4(dev(q[batch]), dev(k[batch]), dev(v[batch]), d_cache, out[batch], n_head, n_kv, hd, n_ctx, dpos(past + batch), scale,
                       ops.FUSE_ALL, rope, ext=ext)
    torch.cuda.synchronize()
    pos = np.arange(past, past + n)
    qr = ref.rope(normed(q, b["bias_q"], w.get("norm_q"), eps), pos, rope_type, n_rot, theta, ff)
    kr = ref.rope(normed(k, b["bias_k"], w.get("norm_k"), eps), pos, rope_type, n_rot, theta, ff).astype(np.float32)
    want = cache.copy()
    ref.write_rows(want, hd, pos, kr, v + b["bias_v"])
    got = d_cache.cpu().numpy()
    if not norm:                       # (a norm is a sum in fp32: its last bit may move a code)
        assert np.array_equal(got, want)
    K, V = ref.read_rows(got, hd, past + n)
    Kw, _ = ref.read_rows(want, hd, past + n)
    assert np.abs(K - Kw).max() <= 0.6 * np.abs(Kw).max() / 7 and (np.abs(K - Kw) > 1e-2).mean() < 1e-3
    res, most = ref.attend(qr, K, V, past, scale)
    err = np.abs(out.cpu().numpy() - res)
    assert err[:batch].max() <= prefill_bound(most, scale, V, False)
    # q's norm is another fp32 sum: 2^-20 of the scores covers it
    assert err[batch].max() <= 2 * decode_bound(most, scale, V)


def test_decode_writes_the_quantised_activation(ops, oracle):
    rng = np.random.default_rng(201)
    n_head, n_kv, hd, n = 12, 2, 128, 300
    cache = dev(filled(rng, n_kv, hd, n, n))
    q = dev(rng.standard_normal((n_head, hd)).astype(np.float32))
    out = torch.empty(n_head, hd, device="cuda")
    qs, sc = torch.empty(n_head * hd, dtype=torch.int8, device="cuda"), torch.empty(n_head * hd // 32, device="cuda")
    for o in (out, None):
        ops.attn_decode_q4(q, None, None, cache, o, n_head, n_kv, hd, n, dpos(n - 1), 0.09, ops.FUSE_NONE, ext=dict(out_qs=qs, out_scales=sc))
        torch.cuda.synchronize()
        want_q, want_d = oracle.quantize_q8_1(out.cpu().numpy().reshape(-1))
        assert np.array_equal(qs.cpu().numpy(), want_q) and np.array_equal(sc.cpu().numpy(), want_d)


def test_prefill_block_output_and_other_kernel(ops):
    """out_mmq next to and instead of the fp32 output; the warp-level kernel with both output types."""
    rng = np.random.default_rng(202)
    n_head, n_kv, hd, past, batch = 8, 2, 128, 40, 149      # (too many pairs to be taken from the 4-bit rows)
    n_ctx = past + batch
    base = filled(rng, n_kv, hd, n_ctx, past)
    q, k, v = (dev(x) for x in (rng.standard_normal((batch, n_head, hd)).astype(np.float32), rows(rng, batch, n_kv, hd), rows(rng, batch, n_kv, hd)))
    rope = (1, hd, 1e6, None)

    def run(out, **kw):
        cache = dev(base)
        ops.attn_prefill_q4(q, k, v, cache, out, n_head, n_kv, hd, n_ctx, past, batch, 0.0884, ops.FUSE_ALL, rope, **kw)
        torch.cuda.synchronize()
        assert ops.prefill_status(n_head, n_kv, hd, batch, ops.prefill_q4_workspace(n_head, n_kv, hd, batch, n_ctx)) == 0
        return cache

    f32, f16 = torch.empty(batch, n_head, hd, device="cuda"), torch.empty(batch, n_head, hd, dtype=torch.float16, device="cuda")
    blk = [torch.zeros(n_head * batch * 144, dtype=torch.uint8, device="cuda") for _ in range(3)]
    a = run(f32)
    assert torch.equal(a, run(f16)) and torch.equal(f16, f32.half())
    again = torch.empty_like(f32)
    run(again, ext=dict(out_mmq=blk[0]))
    run(None, ext=dict(out_mmq=blk[1]))
    run(f16, ext=dict(out_mmq=blk[2]))
    assert torch.equal(again, f32) and torch.equal(blk[0], blk[1]) and torch.equal(blk[0], blk[2])
    b = blk[0].view(n_head, batch, 144)
    d = b[..., :16].contiguous().view(torch.float32)
    val = (b[..., 16:].contiguous().view(torch.int8).view(n_head, batch, 4, 32).float() * d[..., None]).reshape(n_head, batch, hd).transpose(0, 1)
    step = d.transpose(0, 1).repeat_interleave(32, -1)
    assert ((val - f32).abs() <= 0.5001 * step + 1e-7).all()
    try:
        ops.set_prefill_impl(1)
        m32, m16 = torch.empty_like(f32), torch.empty_like(f16)
        run(m32)
        run(m16)
    finally:
        ops.set_prefill_impl(0)
    K, V = ref.read_rows(a.cpu().numpy(), hd, n_ctx)
    want, most = ref.attend(ref.rope(q.cpu().numpy(), np.arange(past, n_ctx), 1, hd, 1e6), K, V, past, 0.0884)
    assert np.abs(m32.cpu().numpy() - want).max() <= prefill_bound(most, 0.0884, V, False)
    assert torch.equal(m16, m32.half())


@pytest.mark.parametrize("half", [False, True])
@pytest.mark.parametrize("n_head,n_kv,hd,past,batch", [(12, 2, 128, 600, 5), (8, 8, 128, 512, 1), (32, 8, 64, 1003, 3), (16, 1, 128, 2000, 9),
                                                       (28, 4, 128, 900, 18), (9, 1, 64, 700, 40), (5, 5, 64, 527, 17)])
def test_short_chunk_behind_a_long_context(ops, n_head, n_kv, hd, past, batch, half):
    """Walked from the 4-bit rows themselves: fp32 accuracy, each token with the positions up to its own."""
    rng = np.random.default_rng(204)
    n_ctx, rope_type, theta = past + batch + 9, past % 2, 5e5
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
    bound = decode_bound(most, scale, V) + (2.0 ** -11 * np.abs(want).max() if half else 0)
    assert np.abs(got[:batch] - want).max() <= bound
    assert (got[batch] == 9).all()
    assert ops.prefill_status(n_head, n_kv, hd, batch, ops.prefill_q4_workspace(n_head, n_kv, hd, batch, n_ctx)) == 0


@pytest.mark.parametrize("n_head,n_kv,hd,past", [(4, 4, 128, 700), (12, 2, 128, 45), (6, 3, 64, 640), (8, 8, 64, 0)])
def test_short_chunk_hides_a_later_tokens_nan(ops, n_head, n_kv, hd, past):
    """The last token's key and value are not finite: the tokens before it give the bits they give without it."""
    rng = np.random.default_rng(206)
    batch = 7
    n_ctx = past + batch
    cache = filled(rng, n_kv, hd, n_ctx, past)
    q, k, v = rng.standard_normal((batch, n_head, hd)).astype(np.float32), rows(rng, batch, n_kv, hd), rows(rng, batch, n_kv, hd)
    outs = []
    for bad in (False, True):
        if bad:
            k[-1, :, 5] = v[-1, :, 9] = np.nan
        out = torch.empty(batch, n_head, hd, device="cuda")
        ops.attn_prefill_q4(dev(q), dev(k), dev(v), dev(cache), out, n_head, n_kv, hd, n_ctx, past, batch, 0.1, ops.FUSE_KV_APPEND)
        outs.append(out.cpu().numpy())
    assert np.isfinite(outs[0]).all() and np.array_equal(outs[0][:-1], outs[1][:-1])
    assert np.isnan(outs[1][-1]).all()


@pytest.mark.parametrize("amp_q,amp_k,amp_v", [(1e-4, 300.0, 1e-3), (300.0, 1e-3, 20000.0), (1.0, 1.0, 50.0), (1e-20, 1.0, 1e-5)])
@pytest.mark.parametrize("hd,past,batch", [(128, 327, 6), (64, 327, 6), (128, 1700, 300), (64, 1700, 600)])
def test_chunk_at_any_scale(ops, hd, past, batch, amp_q, amp_k, amp_v):
    """The values of the decode test of this name, for a chunk that takes the 4-bit rows and one whose fp16 copies are read in slices."""
    short = batch < 100
    rng = np.random.default_rng(207)
    n_head, n_kv = 4, 1
    n_ctx = past + batch
    cache = np.zeros((n_kv, (n_ctx + 15) // 16, 18 * hd), np.uint8)
    k, v = amp_k * rows(rng, n_ctx, n_kv, hd), amp_v * rng.standard_normal((n_ctx, n_kv, hd))
    v[: n_ctx // 2] *= 0.01
    v = np.clip(v, -60000, 60000)
    ref.write_rows(cache, hd, range(n_ctx), k.astype(np.float32), v.astype(np.float32))
    q = (amp_q * rng.standard_normal((batch, n_head, hd))).astype(np.float32)
    scale = 0.3 / (amp_q * amp_k * hd)
    out = torch.empty(batch, n_head, hd, device="cuda")
    ops.attn_prefill_q4(dev(q), None, None, dev(cache), out, n_head, n_kv, hd, n_ctx, past, batch, scale, ops.FUSE_NONE)
    K, V = ref.read_rows(cache, hd, n_ctx)
    want, most = ref.attend(q, K, V, past, np.float32(scale))
    err = np.abs(out.cpu().numpy() - want).max()
    # the scaled queries of the second way are fp16 and may be subnormal there: off by up to 2^-25 each, in a power of two
    small = 2 * math.log(2) * 2.0 ** -25 * np.abs(K).sum(-1).max() * np.abs(V).max()
    bound = decode_bound(most, scale, V) if short else prefill_bound(most, scale, V, False) + small
    assert err <= bound, (err, bound)


def test_short_chunk_over_many_slices_and_in_a_graph(ops):
    """20000 rows, so that a chunk's slices merge in two levels; the same bits from a graph, and from both kernels to their bounds."""
    n_head, n_kv, hd, past, batch = 8, 2, 128, 20000, 6
    n_ctx = past + batch
    gen = torch.Generator(device="cuda").manual_seed(11)
    base = ops.KVCacheQ4(1, n_kv, n_ctx, hd).layer(0)
    k, v = (torch.randn(past, n_kv, hd, device="cuda", generator=gen) for _ in range(2))
    ops.kv_store_q4_batch(base, k, v, n_kv, hd, n_ctx, 0, past)
    q = torch.randn(batch, n_head, hd, device="cuda", generator=gen)
    kn, vn = (torch.randn(batch, n_kv, hd, device="cuda", generator=gen) for _ in range(2))
    ws = torch.empty(ops.prefill_q4_workspace(n_head, n_kv, hd, batch, n_ctx).numel(), dtype=torch.uint8, device="cuda")

    def call(cache, out):
        ops.attn_prefill_q4(q, kn, vn, cache, out, n_head, n_kv, hd, n_ctx, past, batch, 0.0884, ops.FUSE_KV_APPEND, None, ws)

    a, b = base.clone(), base.clone()
    want, got, other = (torch.zeros(batch, n_head, hd, device="cuda") for _ in range(3))
    call(a, want)
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        call(b, got)
    for _ in range(3):
        b.copy_(base)
        got.zero_()
        g.replay()
        torch.cuda.synchronize()
        assert torch.equal(got, want) and torch.equal(a, b)
    kh, vh = (torch.zeros(n_kv, n_ctx, hd, dtype=torch.float16, device="cuda") for _ in range(2))
    ops.kv_load_q4(a, kh, vh, n_kv, hd, n_ctx, 0, n_ctx)
    K, V = kh.double().repeat_interleave(n_head // n_kv, 0), vh.double().repeat_interleave(n_head // n_kv, 0)
    s = torch.einsum("bhd,hnd->bhn", q.double(), K) * 0.0884
    s.masked_fill_(torch.arange(n_ctx, device="cuda")[None, None] > torch.arange(past, n_ctx, device="cuda")[:, None, None], -math.inf)
    exact = torch.einsum("bhn,hnd->bhd", torch.softmax(s, -1), V)
    most = float(torch.einsum("bhd,hnd->bhn", q.double().abs(), K.abs()).max())
    bound = prefill_bound(most, 0.0884, vh.float().cpu().numpy(), False)          # (kh and vh are the rows rounded to fp16)
    assert float((want - exact).abs().max()) <= bound
    try:
        ops.set_prefill_impl(1)                            # the fp16 copies and the warp-level kernel
        call(b, other)
    finally:
        ops.set_prefill_impl(0)
    assert float((other - exact).abs().max()) <= bound


@pytest.mark.parametrize("batch", [3, 25])
def test_many_heads_in_the_prologue(ops, batch):
    """More head rows than a prologue CTA has in flight at once."""
    rng = np.random.default_rng(203)
    n_head, n_kv, hd = 96, 16, 64
    q, k, v = rng.standard_normal((batch, n_head, hd)).astype(np.float32), rows(rng, batch, n_kv, hd), rows(rng, batch, n_kv, hd)
    cache = np.zeros((n_kv, 2, 18 * hd), np.uint8)
    d_cache, out = dev(cache), torch.empty(batch, n_head, hd, device="cuda")
    ops.attn_prefill_q4(dev(q), dev(k), dev(v), d_cache, out, n_head, n_kv, hd, 27, 0, batch, 0.125, ops.FUSE_ALL, (1, hd, 1e6, None))
    pos = np.arange(batch)
    ref.write_rows(cache, hd, pos, ref.rope(k, pos, 1, hd, 1e6).astype(np.float32), v)
    assert np.array_equal(d_cache.cpu().numpy(), cache)
    K, V = ref.read_rows(cache, hd, batch)
    want, most = ref.attend(ref.rope(q, pos, 1, hd, 1e6), K, V, 0, 0.125)
    assert np.abs(out.cpu().numpy() - want).max() <= prefill_bound(most, 0.125, V, False)


# ------------------------------------------------------------------------------------------------- a run of them together
@pytest.mark.parametrize("n_head,n_kv,hd", [(12, 2, 128), (18, 2, 64)])
def test_a_conversation(ops, n_head, n_kv, hd):
    """Prompt in two chunks, decode steps, the context rolled, more steps, on two layers; the cache's bytes and every output against
    the 64-bit reference.  The rows one call appends are the bytes another would."""
    rng = np.random.default_rng(210)
    n_layer, n_ctx, theta, scale = 2, 75, 1e6, 1.0 / math.sqrt(hd)
    cache = ops.KVCacheQ4(n_layer, n_kv, n_ctx, hd)
    want = cache.buf.cpu().numpy()
    rope = (1, hd, theta, None)

    def step(n_past, n, call):
        for l in range(n_layer):
            q, k, v = rng.standard_normal((n, n_head, hd)).astype(np.float32), rows(rng, n, n_kv, hd), rows(rng, n, n_kv, hd)
            pos = np.arange(n_past, n_past + n)
            kr = ref.rope(k, pos, 1, hd, theta).astype(np.float32)
            ref.write_rows(want[l], hd, pos, kr, v)
            out = torch.empty(n, n_head, hd, device="cuda")
            if call == "prefill":
                ops.attn_prefill_q4(dev(q), dev(k), dev(v), cache.layer(l), out, n_head, n_kv, hd, n_ctx, n_past, n, scale, ops.FUSE_ALL, rope)
            elif call == "decode":
                ops.attn_decode_q4(dev(q[0]), dev(k[0]), dev(v[0]), cache.layer(l), out[0], n_head, n_kv, hd, n_ctx, dpos(n_past), scale, ops.FUSE_ALL, rope)
            else:                                          # the unfused sequence
                ops.kv_store_q4_ind(cache.layer(l), dev(kr[0]), dev(v[0]), n_kv, hd, n_ctx, dpos(n_past))
                ops.attn_decode_q4(dev(q[0]), None, None, cache.layer(l), out[0], n_head, n_kv, hd, n_ctx, dpos(n_past), scale, ops.FUSE_ROPE_Q, rope)
            K, V = ref.read_rows(want[l], hd, n_past + n)
            res, most = ref.attend(ref.rope(q, pos, 1, hd, theta), K, V, n_past, scale)
            bound = prefill_bound(most, scale, V, False) if call == "prefill" else decode_bound(most, scale, V)
            assert np.abs(out.cpu().numpy() - res).max() <= bound, (call, n_past)
        assert np.array_equal(cache.buf.cpu().numpy(), want), (call, n_past)

    step(0, 37, "prefill")
    step(37, 20, "prefill")
    for p in range(57, 75):
        step(p, 1, "decode" if p % 2 else "store")
    n_keep, shift = 5, 34
    cache.shift(n_keep, shift)
    torch.cuda.synchronize()
    for l in range(n_layer):
        K, V = ref.read_rows(want[l], hd, n_ctx)
        gK, gV = ref.read_rows(cache.layer(l).cpu().numpy(), hd, n_ctx)
        for g, x in ((gK, K), (gV, V)):
            moved = np.concatenate((x[:, :n_keep], x[:, n_keep + shift:], np.zeros_like(x[:, :shift])), 1)
            assert np.array_equal(g, moved)
    want[:] = cache.buf.cpu().numpy()
    for p in range(n_ctx - shift, n_ctx - shift + 9):
        step(p, 1, "decode")
    # taken over into an fp16 cache, the rows are those the reference reads
    half = ops.KVCache(n_layer, n_kv, 96, hd)
    for l in range(n_layer):
        ops.kv_load_q4(cache.layer(l), *half.layer(l), n_kv, hd, n_ctx, 0, n_ctx, 96, 0)
        for g, x in zip(half.layer(l), ref.read_rows(want[l], hd, n_ctx)):
            assert np.abs(g[:, :n_ctx].float().cpu().numpy() - x).max() <= 2.0 ** -11 * np.abs(x).max()


# ------------------------------------------------------------------------------------------------- order and overlap
@pytest.mark.parametrize("mode", [0, 1, 2])
def test_launch_overlap(ops, mode):
    """The unfused pair and the fused call under every launch mode, back to back over layers of their own, with a decoy in
    the row the store call overwrites."""
    rng = np.random.default_rng(220)
    n_head, n_kv, hd, n, layers = 16, 2, 128, 700, 6
    scale = 1.0 / math.sqrt(hd)
    q = [dev(rng.standard_normal((n_head, hd)).astype(np.float32)) for _ in range(layers)]
    kv = [(rows(rng, 1, n_kv, hd), rows(rng, 1, n_kv, hd)) for _ in range(layers)]
    base = []
    for l in range(layers):
        c = filled(rng, n_kv, hd, n + 3, n - 1)
        ref.write_rows(c, hd, [n - 1], 100 * np.ones((1, n_kv, hd), np.float32), 100 * np.ones((1, n_kv, hd), np.float32))
        base.append(c)
    outs = {}
    for m in (0, mode):
        for fused in (False, True):
            caches = [dev(c) for c in base]
            new = [(dev(k[0]), dev(v[0])) for k, v in kv]
            out = torch.empty(layers, n_head, hd, device="cuda")
            pos = dpos(n - 1)
            torch.cuda.synchronize()
            ops.set_decode_overlap(m)
            try:
                for l in range(layers):
                    if fused:
                        ops.attn_decode_q4(q[l], new[l][0], new[l][1], caches[l], out[l], n_head, n_kv, hd, n + 3, pos, scale, ops.FUSE_KV_APPEND)
                    else:
                        ops.kv_store_q4_ind(caches[l], new[l][0], new[l][1], n_kv, hd, n + 3, pos)
                        ops.attn_decode_q4(q[l], None, None, caches[l], out[l], n_head, n_kv, hd, n + 3, pos, scale, ops.FUSE_NONE)
                torch.cuda.synchronize()
            finally:
                ops.set_decode_overlap(0)
            outs[m, fused] = (out, torch.stack(caches))
    first = outs[0, False]
    for got in outs.values():
        assert torch.equal(got[0], first[0]) and torch.equal(got[1], first[1])
    want = base[0].copy()
    ref.write_rows(want, hd, [n - 1], *kv[0])
    assert np.array_equal(first[1][0].cpu().numpy(), want)


def test_graph_replays_across_block_and_slice_borders(ops):
    """One captured step with the position in device memory, replayed over 60 tokens: the same outputs and bytes as eager calls."""
    rng = np.random.default_rng(221)
    n_head, n_kv, hd, n_ctx, start, steps = 14, 2, 128, 400, 250, 60
    base = dev(filled(rng, n_kv, hd, n_ctx, start))
    q, k, v = (dev(rng.standard_normal((steps, h, hd)).astype(np.float32)) for h in (n_head, n_kv, n_kv))
    rope, scale = (1, hd, 1e6, None), 0.0884

    def program(cache, sq, sk, sv, out, pos, ws):
        ops.attn_decode_q4(sq, sk, sv, cache, out, n_head, n_kv, hd, n_ctx, pos, scale, ops.FUSE_ALL, rope, ws)

    eager_cache, graph_cache = base.clone(), base.clone()
    eager, graph = (torch.empty(steps, n_head, hd, device="cuda") for _ in range(2))
    ws = torch.empty_like(ops.decode_q4_workspace(n_head, n_kv, hd))
    sq, sk, sv, so, sp = q[0].clone(), k[0].clone(), v[0].clone(), torch.empty(n_head, hd, device="cuda"), dpos(start)
    program(base.clone(), sq, sk, sv, so, sp, ws)
    g = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(g):
        program(graph_cache, sq, sk, sv, so, sp, ws)
    for i in range(steps):
        program(eager_cache, q[i], k[i], v[i], eager[i], dpos(start + i), None)
        for dst, src in ((sq, q[i]), (sk, k[i]), (sv, v[i])):
            dst.copy_(src)
        sp.fill_(start + i)
        g.replay()
        graph[i].copy_(so)
    torch.cuda.synchronize()
    assert torch.equal(eager, graph) and torch.equal(eager_cache, graph_cache)


def test_two_streams_with_workspaces_of_their_own(ops):
    rng = np.random.default_rng(222)
    n_head, n_kv, hd, n = 16, 2, 128, 20000
    gen = torch.Generator(device="cuda").manual_seed(3)
    caches, qs, want = [], [], []
    for i in range(2):
        c = ops.KVCacheQ4(1, n_kv, n, hd).layer(0)
        k, v = (torch.randn(n, n_kv, hd, device="cuda", generator=gen) for _ in range(2))
        ops.kv_store_q4_batch(c, k, v, n_kv, hd, n, 0, n)
        caches.append(c)
        qs.append(torch.randn(n_head, hd, device="cuda", generator=gen))
        o = torch.empty(n_head, hd, device="cuda")
        ops.attn_decode_q4(qs[i], None, None, c, o, n_head, n_kv, hd, n, dpos(n - 1), 0.0884, ops.FUSE_NONE)
        want.append(o)
    pos = dpos(n - 1)
    streams = [torch.cuda.Stream() for _ in range(2)]
    ws = [torch.empty_like(ops.decode_q4_workspace(n_head, n_kv, hd)) for _ in range(2)]
    out = torch.zeros(2, 20, n_head, hd, device="cuda")
    torch.cuda.synchronize()
    for r in range(20):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                ops.attn_decode_q4(qs[i], None, None, caches[i], out[i, r], n_head, n_kv, hd, n, pos, 0.0884, ops.FUSE_NONE, None, ws[i])
    torch.cuda.synchronize()
    for i in range(2):
        assert all(torch.equal(out[i, r], want[i]) for r in range(20))
    # and through set_stream, which the other calls of this module take as well
    try:
        ops.set_stream(streams[0])
        o = torch.empty(n_head, hd, device="cuda")
        torch.cuda.synchronize()
        ops.attn_decode_q4(qs[1], None, None, caches[1], o, n_head, n_kv, hd, n, pos, 0.0884, ops.FUSE_NONE)
        streams[0].synchronize()
        assert torch.equal(o, want[1])
    finally:
        ops.set_stream(None)


@pytest.mark.parametrize("hd,past,batch", [(128, 50, 40), (128, 50, 160), (128, 1500, 160), (64, 1600, 270)])
def test_prefill_captured(ops, hd, past, batch):
    rng = np.random.default_rng(223)
    n_head, n_kv = 8, 2
    n_ctx = past + batch
    base = dev(filled(rng, n_kv, hd, n_ctx, past))
    q, k, v = (dev(rng.standard_normal((batch, h, hd)).astype(np.float32)) for h in (n_head, n_kv, n_kv))
    ws = torch.empty(2 * ops.prefill_q4_workspace(n_head, n_kv, hd, batch, n_ctx).numel(), dtype=torch.uint8, device="cuda")
    want, got = (torch.zeros(batch, n_head, hd, dtype=torch.float16, device="cuda") for _ in range(2))

    def call(cache, out):
        ops.attn_prefill_q4(q, k, v, cache, out, n_head, n_kv, hd, n_ctx, past, batch, 0.0884, ops.FUSE_ALL, (0, hd, 5e5, None), ws)

    a, b = base.clone(), base.clone()
    call(a, want)
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        call(b, got)
    for _ in range(3):
        b.copy_(base)
        got.zero_()
        g.replay()
        torch.cuda.synchronize()
        assert torch.equal(got, want) and torch.equal(a, b)


@pytest.mark.parametrize("n_head,n_kv,hd,batch", [(8, 2, 128, 30), (12, 4, 64, 30), (8, 2, 128, 150)])
def test_unfused_prefill_reads_what_the_store_call_wrote(ops, n_head, n_kv, hd, batch):
    """Rows stored by the unfused call, then the chunk with and without the rotation of q: the fused call's bytes and outputs."""
    rng = np.random.default_rng(224)
    past = 21
    n_ctx, scale, rope = past + batch, 1.0 / math.sqrt(hd), (1, hd, 1e6, None)
    base = filled(rng, n_kv, hd, n_ctx, past)
    q, k, v = rng.standard_normal((batch, n_head, hd)).astype(np.float32), rows(rng, batch, n_kv, hd), rows(rng, batch, n_kv, hd)
    pos = np.arange(past, n_ctx)
    kr = ref.rope(k, pos, 1, hd, 1e6).astype(np.float32)
    a, b = dev(base), dev(base)
    fused, unfused, raw = (torch.empty(batch, n_head, hd, device="cuda") for _ in range(3))
    ops.attn_prefill_q4(dev(q), dev(k), dev(v), a, fused, n_head, n_kv, hd, n_ctx, past, batch, scale, ops.FUSE_ALL, rope)
    ops.kv_store_q4_batch(b, dev(kr), dev(v), n_kv, hd, n_ctx, past, batch)
    ops.attn_prefill_q4(dev(q), None, None, b, unfused, n_head, n_kv, hd, n_ctx, past, batch, scale, ops.FUSE_ROPE_Q, rope)
    ops.attn_prefill_q4(dev(ref.rope(q, pos, 1, hd, 1e6).astype(np.float32)), None, None, b, raw, n_head, n_kv, hd, n_ctx, past, batch, scale,
                        ops.FUSE_NONE)
    torch.cuda.synchronize()
    assert torch.equal(a, b) and torch.equal(fused, unfused)
    K, V = ref.read_rows(b.cpu().numpy(), hd, n_ctx)
    want, most = ref.attend(ref.rope(q, pos, 1, hd, 1e6), K, V, past, scale)
    for got in (fused, raw):
        assert np.abs(got.cpu().numpy() - want).max() <= prefill_bound(most, scale, V, False)
    # the append without any rotation
    c, out = dev(base), torch.empty(n_head, hd, device="cuda")
    ops.attn_decode_q4(dev(q[0]), dev(k[0]), dev(v[0]), c, out, n_head, n_kv, hd, n_ctx, dpos(past), scale, ops.FUSE_KV_APPEND)
    w = base.copy()
    ref.write_rows(w, hd, [past], k[:1], v[:1])
    assert np.array_equal(c.cpu().numpy(), w)
    K, V = ref.read_rows(w, hd, past + 1)
    want, most = ref.attend(q[:1], K, V, past, scale)
    assert np.abs(out.cpu().numpy() - want[0]).max() <= decode_bound(most, scale, V)


@pytest.mark.parametrize("n_head,n_kv", [(4, 1), (7, 1)])
def test_a_bad_query_head_stays_alone(ops, n_head, n_kv):
    rng = np.random.default_rng(225)
    hd, n = 128, 100
    cache = dev(filled(rng, n_kv, hd, n, n))
    q = rng.standard_normal((n_head, hd)).astype(np.float32)
    good, out = torch.empty(n_head, hd, device="cuda"), torch.empty(n_head, hd, device="cuda")
    ops.attn_decode_q4(dev(q), None, None, cache, good, n_head, n_kv, hd, n, dpos(n - 1), 0.0884, ops.FUSE_NONE)
    for bad in (np.nan, np.inf, -np.inf):
        x = q.copy()
        x[1, 77] = bad
        ops.attn_decode_q4(dev(x), None, None, cache, out, n_head, n_kv, hd, n, dpos(n - 1), 0.0884, ops.FUSE_NONE)
        assert torch.isnan(out[1]).all() and torch.equal(out[2:], good[2:]) and torch.equal(out[0], good[0])
    # the same over rows whose steps are all zero
    flat = np.zeros((n_kv, (n + 15) // 16, 18 * hd), np.uint8)
    same = np.ones((n, n_kv, hd), np.float32)
    ref.write_rows(flat, hd, range(n), same, 3 * same)
    x = q.copy()
    x[1, 77] = np.nan
    ops.attn_decode_q4(dev(x), None, None, dev(flat), out, n_head, n_kv, hd, n, dpos(n - 1), 0.0884, ops.FUSE_NONE)
    rest = [h for h in range(n_head) if h != 1]
    assert torch.isnan(out[1]).all() and float((out[rest] - 3).abs().max()) <= decode_bound(hd * 4, 0.0884, np.float64(3))
    x = q.copy()
    x[2] = 0                                              # all scores alike: the mean of the values
    ops.attn_decode_q4(dev(x), None, None, cache, out, n_head, n_kv, hd, n, dpos(n - 1), 0.0884, ops.FUSE_NONE)
    V = ref.read_rows(cache.cpu().numpy(), hd, n)[1]
    assert np.abs(out[2].cpu().numpy() - V[0].mean(0)).max() <= decode_bound(0, 1, V)


# ------------------------------------------------------------------------------------------------- large caches, odd positions
def test_store_of_more_blocks_than_one_grid_plane(ops):
    n_kv, hd, n, base = 1, 64, 65535 * 16 + 300, 5
    gen = torch.Generator(device="cuda").manual_seed(9)
    k, v = (torch.randn(n, n_kv, hd, device="cuda", generator=gen) for _ in range(2))
    cache = ops.KVCacheQ4(1, n_kv, n + 10, hd).layer(0)
    ops.kv_store_q4_batch(cache, k, v, n_kv, hd, n + 10, base, n)
    for at, m in ((0, 40), (65535 * 16 - 60, 120), (n - 50, 50)):
        kh, vh = (torch.zeros(n_kv, m, hd, dtype=torch.float16, device="cuda") for _ in range(2))
        ops.kv_load_q4(cache, kh, vh, n_kv, hd, n + 10, base + at, m)
        for g, x in ((kh, k), (vh, v)):
            w = ref.values(*ref.quantise(np.ascontiguousarray(x[at: at + m].cpu().numpy().transpose(1, 0, 2))))
            assert (np.abs(g.float().cpu().numpy() - w) <= 2.0 ** -11 * (1 + 2.0 ** -11) * np.abs(w) + 2.0 ** -25).all()


def test_offsets_beyond_two_gigabytes(ops):
    n_kv, hd, n_ctx, n_head = 8, 128, 2_000_016, 8
    assert ops.kv_q4_bytes(n_kv, hd, n_ctx) > 2 ** 31
    cache = ops.KVCacheQ4(1, n_kv, n_ctx, hd).layer(0)
    rng = np.random.default_rng(230)
    n = 40
    k, v = rows(rng, n, n_kv, hd), rows(rng, n, n_kv, hd)
    ops.kv_store_q4_batch(cache, dev(k), dev(v), n_kv, hd, n_ctx, n_ctx - n, n)
    kh, vh = (torch.zeros(n_kv, n, hd, dtype=torch.float16, device="cuda") for _ in range(2))
    ops.kv_load_q4(cache, kh, vh, n_kv, hd, n_ctx, n_ctx - n, n)
    vals = [ref.values(*ref.quantise(np.transpose(x, (1, 0, 2)))) for x in (k, v)]
    for g, w in zip((kh, vh), vals):
        assert (np.abs(g.float().cpu().numpy() - w) <= 2.0 ** -11 * (1 + 2.0 ** -11) * np.abs(w) + 2.0 ** -25).all()
    assert not cache[:, : (n_ctx - n) // 16].any()
    # all other rows are zero: their scores are 0 and their values add nothing
    q = rng.standard_normal((n_head, hd)).astype(np.float32)
    out = torch.empty(n_head, hd, device="cuda")
    scale = 0.3
    ops.attn_decode_q4(dev(q), None, None, cache, out, n_head, n_kv, hd, n_ctx, dpos(n_ctx - 1), scale, ops.FUSE_NONE)
    s = np.einsum("hd,hnd->hn", q.astype(np.float64), vals[0]) * np.float32(scale)
    want = np.einsum("hn,hnd->hd", np.exp(s), vals[1]) / (np.exp(s).sum(-1) + n_ctx - n)[:, None]
    most = np.einsum("hd,hnd->hn", np.abs(q), np.abs(vals[0])).max()
    err = np.abs(out.cpu().numpy() - want)
    # the weights of the 40 rows among two million: the bound scales with the largest output instead of the largest value
    assert err.max() <= (2 * (2.0 ** -20 * scale * most + 2.0 ** -21) + 2.0 ** -20) * np.abs(want).max() * 4, (err.max(), np.abs(want).max())


def test_positions_outside_the_cache(ops):
    rng = np.random.default_rng(231)
    n_head, n_kv, hd, n_ctx = 4, 2, 64, 50
    host = filled(rng, n_kv, hd, n_ctx, n_ctx)
    q = dev(rng.standard_normal((n_head, hd)).astype(np.float32))
    outs = []
    for p in (n_ctx - 1, n_ctx, n_ctx + 1000, 2 ** 31 - 1):
        cache, out = dev(host), torch.empty(n_head, hd, device="cuda")
        ops.attn_decode_q4(q, None, None, cache, out, n_head, n_kv, hd, n_ctx, dpos(p), 0.125, ops.FUSE_NONE)
        outs.append(out)
        assert np.array_equal(cache.cpu().numpy(), host)
    assert all(torch.equal(o, outs[0]) for o in outs)


@pytest.mark.parametrize("n_head,n_kv,hd", [(40, 40, 64), (128, 64, 128), (100, 100, 64), (160, 160, 64)])
@pytest.mark.parametrize("length", [300, 600, 1500, 3000, 5000])
def test_more_kv_heads_than_slices(ops, n_head, n_kv, hd, length):
    """Many kv heads leave few slices to each: every row has to be in one of them."""
    gen = torch.Generator(device="cuda").manual_seed(7)
    cache = ops.KVCacheQ4(1, n_kv, length, hd).layer(0)
    k, v = (torch.randn(length, n_kv, hd, device="cuda", generator=gen) for _ in range(2))
    ops.kv_store_q4_batch(cache, k, v, n_kv, hd, length, 0, length)
    kh, vh = (torch.zeros(n_kv, length, hd, dtype=torch.float16, device="cuda") for _ in range(2))
    ops.kv_load_q4(cache, kh, vh, n_kv, hd, length, 0, length)
    q = torch.randn(n_head, hd, device="cuda", generator=gen)
    out = torch.empty(n_head, hd, device="cuda")
    ops.attn_decode_q4(q, None, None, cache, out, n_head, n_kv, hd, length, dpos(length - 1), 0.1, ops.FUSE_NONE)
    qd, K, V = q.double().view(n_kv, -1, hd), kh.double(), vh.double()
    want = torch.softmax(qd @ K.transpose(1, 2) * 0.1, -1) @ V
    # kh and vh are the rows rounded to fp16: 2^-11 of a value, and of a score's sum of products
    most = float((qd.abs() @ K.abs().transpose(1, 2)).max())
    err = float((out.view_as(want) - want).abs().max())
    assert err <= (2 * 2.0 ** -11 * 0.1 * most + 2.0 ** -11) * float(V.abs().max())


@pytest.mark.parametrize("n_head,hd,length", [(4, 128, 40000), (16, 128, 70001), (3, 64, 40000)])
def test_one_kv_head_merges_more_than_sixteen_groups(ops, n_head, hd, length):
    """One kv head at a long context has 19 groups of slices, which merge in two passes: both caches."""
    gen = torch.Generator(device="cuda").manual_seed(8)
    cache = ops.KVCacheQ4(1, 1, length, hd).layer(0)
    k, v = (torch.randn(length, 1, hd, device="cuda", generator=gen) for _ in range(2))
    v[..., hd // 2:] += 1.0
    ops.kv_store_q4_batch(cache, k, v, 1, hd, length, 0, length)
    kh, vh = (torch.zeros(1, length, hd, dtype=torch.float16, device="cuda") for _ in range(2))
    ops.kv_load_q4(cache, kh, vh, 1, hd, length, 0, length)
    q = torch.randn(n_head, hd, device="cuda", generator=gen).half().float()
    qd, K, V = q.double(), kh[0].double(), vh[0].double()
    want = torch.softmax(qd @ K.T * 0.1, -1) @ V
    most = float((qd.abs() @ K.abs().T).max())
    # the rows of the 4-bit cache are within 2^-11 of kh and vh; the fp16 kernel rounds its weights to fp16, 2^-11 as well
    bound = (2 * 2.0 ** -11 * 0.1 * most + 2 * 2.0 ** -11) * float(V.abs().max())
    out = torch.empty(n_head, hd, device="cuda")
    ops.attn_decode_q4(q, None, None, cache, out, n_head, 1, hd, length, dpos(length - 1), 0.1, ops.FUSE_NONE)
    assert float((out - want).abs().max()) <= bound and float((out - want).norm() / want.norm()) < 1e-3
    ops.flash_attention_decode_ind(q, kh, vh, out, n_head, 1, hd, length, dpos(length - 1), 0.1)
    assert float((out - want).abs().max()) <= bound and float((out - want).norm() / want.norm()) < 1e-3


def test_more_workspaces_than_counter_slots(ops):
    rng = np.random.default_rng(232)
    n_head, n_kv, hd, n = 8, 1, 128, 5000
    gen = torch.Generator(device="cuda").manual_seed(4)
    cache = ops.KVCacheQ4(1, n_kv, n, hd).layer(0)
    ops.kv_store_q4_batch(cache, *(torch.randn(n, n_kv, hd, device="cuda", generator=gen) for _ in range(2)), n_kv, hd, n, 0, n)
    q = torch.randn(n_head, hd, device="cuda", generator=gen)
    pos, size = dpos(n - 1), ops.decode_q4_workspace(n_head, n_kv, hd).numel()
    ws = [torch.empty(size, dtype=torch.uint8, device="cuda").fill_(255) for _ in range(70)]
    out = torch.empty(70, n_head, hd, device="cuda")
    for i in range(70):
        ops.attn_decode_q4(q, None, None, cache, out[i], n_head, n_kv, hd, n, pos, 0.0884, ops.FUSE_NONE, None, ws[i])
    torch.cuda.synchronize()
    assert all(torch.equal(out[i], out[0]) for i in range(70))


def test_refusals(ops):
    from orin_llm_b200 import capi
    L = capi.lib()
    t = torch.zeros(1 << 20, dtype=torch.uint8, device="cuda")
    p = t.data_ptr()
    s = torch.cuda.current_stream().cuda_stream
    A, U, W = capi.ERR_ARG, capi.ERR_UNSUPPORTED, capi.ERR_WORKSPACE

    def store(c=p, k=p, v=p, heads=2, hd=128, n_ctx=64, base=0, batch=1, d=None):
        return L.oattn_kv_store_q4(c, k, v, heads, hd, n_ctx, base, batch, d, s)
    assert [store(c=None), store(k=None), store(heads=0), store(n_ctx=0), store(batch=0), store(base=-1), store(base=64), store(base=1, batch=64),
            store(c=p + 8), store(k=p + 4), store(d=p, batch=2), store(base=2 ** 31 - 1, batch=2)] == [A] * 12
    assert [store(hd=96), store(hd=0), store(n_ctx=(1 << 30) + 1)] == [U] * 3

    def load(c=p, k=p, v=p, heads=2, hd=128, n_ctx=64, base=0, n=1, dc=1, db=0):
        return L.oattn_kv_load_q4(c, k, v, heads, hd, n_ctx, base, n, dc, db, s)
    assert [load(c=None), load(k=None), load(n=0), load(base=64), load(base=-1), load(base=60, n=5, dc=5), load(n=2), load(db=1), load(db=-1), load(dc=0),
            load(c=p + 4), load(v=p + 2)] == [A] * 12
    assert load(hd=32) == U

    def shift(c=p, layers=1, n_kv=2, hd=128, n_ctx=64, keep=0, sh=1):
        return L.oattn_kv_shift_q4(c, layers, n_kv, hd, n_ctx, keep, sh, s)
    assert [shift(c=None), shift(layers=0), shift(n_kv=0), shift(keep=-1), shift(sh=0), shift(keep=64), shift(keep=60, sh=5), shift(c=p + 1)] == [A] * 8
    assert [shift(hd=256), shift(layers=40000)] == [U] * 2

    rp = capi.RopeParams(1, 128, 1e6, 0)

    def decode(q=p, k=p, v=p, c=p, o=p, nh=8, nkv=2, hd=128, n_ctx=64, d=p, sc=0.1, fuse=7, rope=rp, ext=None, w=p, wb=1 << 20):
        return L.oattn_decode_q4(q, k, v, c, o, nh, nkv, hd, n_ctx, d, sc, fuse, rope, ext, w, wb, s)
    assert [decode(q=None), decode(k=None), decode(c=None), decode(o=None), decode(d=None), decode(sc=0.0), decode(sc=float("nan")), decode(fuse=8),
            decode(fuse=2), decode(rope=None), decode(q=p + 4), decode(o=p + 8), decode(n_ctx=0), decode(nkv=0)] == [A] * 14
    assert [decode(hd=80), decode(nh=7), decode(nh=34, nkv=2), decode(rope=capi.RopeParams(1, 130, 1e6, 0))] == [U] * 4
    assert [decode(w=None), decode(w=p + 128), decode(wb=1000)] == [W] * 3
    ext = capi.Ext()
    ext.bias_k = p
    assert decode(fuse=0, ext=ext) == A                                # a bias of a row that is not appended
    ext = capi.Ext()
    ext.out_mmq = p
    assert decode(ext=ext) == U                                        # the prefill form

    need = L.oattn_prefill_q4_workspace_bytes(8, 2, 128, 4, 20)

    def prefill(q=p, k=p, v=p, c=p, o=p, h=None, nh=8, nkv=2, hd=128, n_ctx=64, past=16, batch=4, sc=0.1, fuse=7, rope=rp, ext=None, w=p, wb=1 << 20):
        return L.oattn_prefill_q4(q, k, v, c, o, h, nh, nkv, hd, n_ctx, past, batch, sc, fuse, rope, ext, w, wb, s)
    assert [prefill(q=None), prefill(v=None), prefill(c=None), prefill(o=None), prefill(h=p), prefill(past=61), prefill(past=-1), prefill(batch=0),
            prefill(sc=-1.0), prefill(fuse=16), prefill(fuse=3), prefill(q=p + 4), prefill(o=None, h=p + 2), prefill(past=2 ** 31 - 2)] == [A] * 14
    assert [prefill(hd=96), prefill(nh=9)] == [U] * 2
    assert [prefill(w=None), prefill(w=p + 64), prefill(wb=need - 1)] == [W] * 3
    torch.cuda.synchronize()
    assert not t.any()                                                 # nothing was written

    # what only the Python layer can see
    c = ops.KVCacheQ4(1, 2, 64, 128).layer(0)
    x = torch.zeros(1, 2, 128, device="cuda")
    with pytest.raises(ValueError, match="k:"):
        ops.kv_store_q4_batch(c, x.cpu(), x, 2, 128, 64, 0, 1)
    with pytest.raises(ValueError, match="float32"):
        ops.kv_store_q4_batch(c, x.half(), x, 2, 128, 64, 0, 1)
    with pytest.raises(ValueError, match="at least"):
        ops.kv_store_q4_batch(c, x, x, 2, 128, 64, 0, 2)
    with pytest.raises(ValueError, match="not contiguous"):
        ops.kv_store_q4_ind(c, torch.zeros(128, 2, device="cuda").t(), x, 2, 128, 64, dpos(0))
    with pytest.raises(ValueError, match="int32"):
        ops.kv_store_q4_ind(c, x, x, 2, 128, 64, torch.zeros(1, dtype=torch.int64, device="cuda"))
    with pytest.raises(capi.AttnError):
        ops.kv_store_q4_batch(c, x, x, 2, 128, 64, 64, 1)
    with pytest.raises(TypeError, match="out"):
        ops.attn_decode_q4(x, x, x, c, None, 2, 2, 128, 64, dpos(0), 0.1, ops.FUSE_KV_APPEND)
    with pytest.raises(ValueError, match="kc"):
        ops.kv_load_q4(c, x.half(), torch.zeros(2, 9, 128, dtype=torch.float16, device="cuda"), 2, 128, 64, 0, 9)
    with pytest.raises(ValueError, match="unknown extension"):
        ops.attn_decode_q4(x, x, x, c, x.clone(), 2, 2, 128, 64, dpos(0), 0.1, ops.FUSE_KV_APPEND, ext=dict(nonsense=1))
