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
