"""CPU tests of the 4-bit KV cache: sizes, the format's addresses, and what the calls refuse before they reach a GPU."""
import numpy as np
import pytest
import torch

import q4_reference as ref
from orin_llm_b200 import build, capi


@pytest.fixture(scope="module")
def ops():
    build.build()
    from orin_llm_b200 import ops as _ops
    return _ops


def test_sizes(ops):
    L = capi.lib()
    for n_kv, hd, n_ctx in ((1, 64, 1), (8, 128, 16), (8, 128, 17), (3, 64, 4095), (2, 128, 1 << 20)):
        want = n_kv * ((n_ctx + 15) // 16) * 18 * hd
        assert L.oattn_kv_q4_bytes(n_kv, hd, n_ctx) == ops.kv_q4_bytes(n_kv, hd, n_ctx) == want
    for n_kv, hd, n_ctx in ((0, 64, 1), (1, 96, 16), (1, 128, 0), (-1, 128, 5), (1, 128, (1 << 30) + 1)):
        assert L.oattn_kv_q4_bytes(n_kv, hd, n_ctx) == ops.kv_q4_bytes(n_kv, hd, n_ctx) == 0
    head = L.oattn_prefill_workspace_bytes(32, 8, 128, 512)
    # the rows in fp16 and the slices' outputs, maxima and sums
    assert L.oattn_prefill_q4_workspace_bytes(32, 8, 128, 512, 8704) == head + 2 * 8 * 8704 * 128 * 2 + 148 * 128 * (128 * 4 + 8)
    # ... or, where that is more, a short chunk's fp32 queries and partial results
    assert (L.oattn_prefill_q4_workspace_bytes(8, 2, 64, 1200, 1200) ==
            L.oattn_prefill_workspace_bytes(8, 2, 64, 1200) + max(1200 * 8 * 64 * 4 + (4 << 20), 2 * 2 * 1200 * 64 * 2 + 148 * 128 * (64 * 4 + 8)))
    assert L.oattn_prefill_q4_workspace_bytes(32, 8, 128, 512, 511) == 0          # fewer rows than the chunk alone has
    assert L.oattn_prefill_q4_workspace_bytes(32, 8, 96, 512, 8704) == 0


@pytest.mark.parametrize("hd", [64, 128])
def test_every_byte_of_a_block_has_one_place(hd):
    seen = np.zeros(18 * hd, int)
    for s in range(16):
        for D in range(0, hd, 2):
            seen[ref.k_byte(hd, s, D)] += 1
            seen[ref.v_byte(hd, s, D)] += 1
    assert (seen[: 16 * hd] == 1).all() and (seen[16 * hd:] == 0).all()


def test_reference_writes_what_it_reads():
    rng = np.random.default_rng(1)
    for hd in (64, 128):
        k, v = rng.standard_normal((20, 3, hd)).astype(np.float32), rng.standard_normal((20, 3, hd)).astype(np.float32)
        cache = np.zeros((3, 2, 18 * hd), np.uint8)
        ref.write_rows(cache, hd, range(20), k, v)
        for got, x in zip(ref.read_rows(cache, hd, 20), (k, v)):
            x = np.transpose(x, (1, 0, 2))
            q, d, m = ref.quantise(x)
            assert np.array_equal(got, ref.values(q, d, m))
            # half a step, and what the fp16 offset adds
            assert (np.abs(got - x).reshape(3, 20, -1, 64) <= (0.502 * d.astype(float) + 2.0 ** -11 * np.abs(m.astype(float)))[..., None]).all()


def test_no_compute_without_device():
    if torch.cuda.is_available():
        pytest.skip("GPU present; covered by the gpu tests")
    build.build()
    L = capi.lib()
    assert L.oattn_kv_store_q4(256, 256, 256, 1, 128, 16, 0, 1, None, None) == capi.ERR_DEVICE
    assert L.oattn_kv_load_q4(256, 256, 256, 1, 128, 16, 0, 1, 1, 0, None) == capi.ERR_DEVICE
    assert L.oattn_kv_shift_q4(256, 1, 1, 128, 16, 0, 1, None) == capi.ERR_DEVICE
    assert L.oattn_decode_q4_workspace_bytes(8, 2, 128) == 0
    assert L.oattn_decode_q4(256, None, None, 256, 256, 8, 2, 128, 16, 256, 0.1, 0, None, None, 256, 1 << 24, None) == capi.ERR_DEVICE
    assert L.oattn_prefill_q4(256, None, None, 256, 256, None, 8, 2, 128, 16, 0, 4, 0.1, 0, None, None, 256, 1 << 24, None) == capi.ERR_DEVICE


def test_tensors_the_calls_refuse(ops):
    """Wrong type, size, stride, device: refused by the Python layer, which knows them (the C entry sees addresses)."""
    c = torch.zeros(2, 1, 18 * 128, dtype=torch.uint8)
    x = torch.zeros(4, 2, 128)
    with pytest.raises(ValueError, match="current CUDA device"):
        ops.kv_store_q4_batch(c, x, x, 2, 128, 16, 0, 4)                       # a CPU cache
    with pytest.raises(ValueError, match="uint8"):
        ops.kv_store_q4_batch(c.float(), x, x, 2, 128, 16, 0, 4)
    with pytest.raises(ValueError, match="at least"):
        ops.kv_shift_q4(c, 2, 2, 128, 16, 0, 1)                                # two layers' worth is needed
    with pytest.raises(ValueError, match="not contiguous"):
        ops.kv_load_q4(torch.zeros(2, 2, 18 * 128, dtype=torch.uint8)[:, :1].expand(2, 1, 18 * 128), x, x, 2, 128, 16, 0, 1)
    with pytest.raises(TypeError, match="cache"):
        ops.kv_load_q4(None, x, x, 2, 128, 16, 0, 1)
    for bad in (dict(head_dim=96), dict(n_kv=0), dict(n_ctx=0)):
        a = dict(n_layer=1, n_kv=2, head_dim=128, n_ctx=16, n_keep=0, shift=1)
        a.update(bad)
        with pytest.raises(capi.AttnError):
            ops.kv_shift_q4(c, **a)
    with pytest.raises(capi.AttnError):
        ops.KVCacheQ4(1, 2, 16, 80, device="cpu")
    cache = ops.KVCacheQ4(2, 3, 33, 64, device="cpu")
    assert cache.buf.shape == (2, 3, 3, 18 * 64) and cache.layer(1).numel() == ops.kv_q4_bytes(3, 64, 33)
