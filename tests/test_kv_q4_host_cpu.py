"""CPU tests of the host side of the 4-bit cache: what the default workspace of the prefill call grows to."""
import pytest
import torch

from orin_llm_b200 import build, capi


@pytest.fixture
def ops(monkeypatch):
    """The module with no workspace yet, and with storage-less blocks in place of the GPU's."""
    build.build()
    from orin_llm_b200 import ops as _ops
    real = torch.empty
    monkeypatch.setitem(_ops._state, "prefill_q4_ws", {})
    monkeypatch.setattr(torch, "empty", lambda *a, **k: real(*a, **{**k, "device": "meta"}))
    monkeypatch.setattr(torch._C, "_cuda_getDevice", lambda: 0)
    return _ops


def kept(ops):
    return [b for have in ops._state["prefill_q4_ws"].values() for _, _, b in have]


@pytest.mark.parametrize("n_ctx,lengths,most", [(32768, range(45, 513), 1), (32768, range(1, 4097), 4), (300, range(1, 301), 1), (40, [1, 40], 1)])
def test_longer_and_longer_prompts_keep_few_workspaces(ops, n_ctx, lengths, most):
    L = capi.lib()
    for n in lengths:
        ws = ops.prefill_q4_workspace(32, 8, 128, n, n_ctx)
        assert ws.numel() >= L.oattn_prefill_q4_workspace_bytes(32, 8, 128, n, n_ctx)
    assert len(kept(ops)) <= most


def test_longer_and_longer_contexts_keep_few_workspaces(ops):
    L = capi.lib()
    for rows in range(100, 20000, 37):
        ws = ops.prefill_q4_workspace(12, 2, 64, min(rows, 700), rows)
        assert ws.numel() >= L.oattn_prefill_q4_workspace_bytes(12, 2, 64, min(rows, 700), rows)
    # 100 rows doubled until they are 20000
    assert len(kept(ops)) <= 9
    # all of them together are less than what the last two would be, and a small context's block holds no more than its own rows
    sizes = [b.numel() for b in kept(ops)]
    assert sum(sizes) <= 2.5 * sizes[-1] + 9 * L.oattn_prefill_q4_workspace_bytes(12, 2, 64, 700, 700)
    assert sizes[0] == L.oattn_prefill_q4_workspace_bytes(12, 2, 64, 100, 100)


def test_a_chunk_longer_than_its_rows_has_no_workspace(ops):
    with pytest.raises(capi.AttnError):
        ops.prefill_q4_workspace(8, 2, 128, 600, 100)
    ops.prefill_q4_workspace(8, 2, 128, 100, 300)
    with pytest.raises(capi.AttnError):
        ops.prefill_q4_workspace(8, 2, 128, 1000, 300)


# ------------------------------------------------------------------------------------------------- the compiled binding
class Compiled(Exception):
    pass


@pytest.fixture
def binding(monkeypatch, tmp_path):
    """The built binding's files at a place of their own, a compiler that only says that it was called, and nothing loaded yet."""
    import os
    import shutil
    from orin_llm_b200 import ops as _ops
    build.build()
    path = str(tmp_path / "_q4_binding.so")
    for end in ("", ".for"):
        shutil.copy2(build.build_binding() + end, path + end)

    def run(cmd, *a, **k):
        raise Compiled(os.path.basename(cmd[0]))
    monkeypatch.setattr(build, "BINDING_LIB", path)
    monkeypatch.setattr(build.subprocess, "run", run)
    monkeypatch.setattr(_ops, "_binding", None)
    return _ops, path


def test_a_current_binding_is_not_built_again(binding):
    _, path = binding
    assert build.build_binding() == path


@pytest.mark.parametrize("stale", ["torch", "older", "no stamp"])
def test_a_stale_binding_is_not_loaded(binding, stale):
    """Made for another torch or Python, or before its source or header changed: built again, not mapped."""
    import os
    ops, path = binding
    if stale == "torch":
        open(path + ".for", "w").write("1.0.0 3.0.0")
    elif stale == "older":
        t = os.path.getmtime(build.BINDING_SRC) - 60
        os.utime(path, (t, t))
    else:
        os.remove(path + ".for")
    with pytest.raises(Compiled, match="g\\+\\+"):
        ops._q4()


def test_a_binding_that_cannot_be_built_says_so(binding, monkeypatch):
    ops, path = binding
    open(path + ".for", "w").write("1.0.0 3.0.0")

    def run(cmd, *a, **k):
        raise FileNotFoundError(cmd[0])
    monkeypatch.setattr(build.subprocess, "run", run)
    with pytest.raises(RuntimeError, match="_q4_binding.so is missing or was built for"):
        ops._q4()


def test_the_library_is_not_built_again_under_its_binding(binding, monkeypatch):
    """It may be loaded already: the binding would be linked to a second one, which was never initialised."""
    ops, path = binding
    open(path + ".for", "w").write("1.0.0 3.0.0")
    monkeypatch.setattr(build, "needs_build", lambda: True)
    with pytest.raises(Compiled, match="g\\+\\+"):
        ops._q4()


def test_a_binding_without_its_source_is_current(binding, monkeypatch):
    """An installed package has no header and may have no source."""
    _, path = binding
    monkeypatch.setattr(build, "BINDING_SRC", path + ".cpp")
    monkeypatch.setattr(build, "HERE", path + ".package")
    assert build.build_binding() == path


# ------------------------------------------------------------------------------------------------- tensors around the attention
N_HEAD, N_KV, HD, BATCH = 6, 2, 128, 3
EXTRAS = {"bias_q": (torch.float32, N_HEAD * HD), "bias_k": (torch.float32, N_KV * HD), "bias_v": (torch.float32, N_KV * HD),
          "norm_q": (torch.float32, HD), "norm_k": (torch.float32, HD), "out_qs": (torch.int8, N_HEAD * HD),
          "out_scales": (torch.float32, N_HEAD * HD // 32), "out_mmq": (torch.uint8, BATCH * N_HEAD * 144)}


def call_with(extra, prefill):
    from orin_llm_b200 import ops as _ops
    build.build()
    cache, x = torch.zeros(N_KV, 1, 18 * HD, dtype=torch.uint8), torch.zeros(BATCH, N_HEAD, HD)
    ws = torch.zeros(1, dtype=torch.uint8)
    if prefill:
        _ops.attn_prefill_q4(x, x, x, cache, x, N_HEAD, N_KV, HD, 16, 0, BATCH, 0.1, _ops.FUSE_KV_APPEND, None, ws, extra)
    else:
        _ops.attn_decode_q4(x, x, x, cache, x, N_HEAD, N_KV, HD, 16, torch.zeros(1, dtype=torch.int32), 0.1, _ops.FUSE_KV_APPEND, None, ws, extra)


@pytest.mark.parametrize("prefill", [False, True])
@pytest.mark.parametrize("name", sorted(EXTRAS))
def test_extras_of_the_wrong_kind_are_refused(name, prefill):
    """Before anything is launched, and by name.  (What is in order gets as far as the cache, which is not on a GPU here.)"""
    dtype, numel = EXTRAS[name]
    with pytest.raises(ValueError, match="current CUDA device"):
        call_with({name: torch.zeros(numel, dtype=dtype)}, prefill)
    if name != "out_mmq" or prefill:                       # (a decode call takes the blocks of one token, which the C entry refuses)
        with pytest.raises(ValueError, match="%s: .*at least" % name):
            call_with({name: torch.zeros(numel - 1, dtype=dtype)}, prefill)
    with pytest.raises(ValueError, match=name + ": "):
        call_with({name: torch.zeros(numel, dtype=torch.float16)}, prefill)
    with pytest.raises(ValueError, match="%s: .*not contiguous" % name):
        call_with({name: torch.zeros(2, numel, dtype=dtype).t()}, prefill)
    with pytest.raises(TypeError, match=name + ": a tensor"):
        call_with({name: 12345}, prefill)


@pytest.mark.parametrize("prefill", [False, True])
def test_extras_that_are_no_extras(prefill):
    for extra in ({}, {"norm_eps": 1e-6}, {"bias_q": None, "out_mmq_ds4": True}):
        with pytest.raises(ValueError, match="current CUDA device"):
            call_with(extra, prefill)
    with pytest.raises(ValueError, match="unknown extension"):
        call_with({"nonsense": 1}, prefill)
    with pytest.raises(TypeError, match="dict"):
        call_with([1], prefill)
    with pytest.raises(TypeError):
        call_with({"norm_eps": "small"}, prefill)
