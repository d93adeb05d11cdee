"""CPU tests of what the low-bit operators tell a tracer and a caller."""
import pytest
import torch

import b200q  # noqa: F401  (registers the operators)


@pytest.mark.parametrize("shape,order", [((5, 3, 256), (1, 0, 2)), ((4, 6), (1, 0)), ((2, 3, 4, 32), (0, 2, 1, 3))])
def test_fake_norms_are_contiguous(shape, order):
    """The kernels write contiguous outputs whatever x's strides are."""
    with torch._subclasses.FakeTensorMode():
        x = torch.empty(shape, dtype=torch.bfloat16, device="cuda").permute(order)
        ops = torch.ops.b200q
        outs = [ops.norm_modulate(x), ops.gated_residual(x, x), *ops.gated_residual_norm(x, x),
                ops.gated_residual_norm_quant_i8(x, x)[0]]
        for o in outs:
            assert o.shape == x.shape and o.dtype == x.dtype and o.is_contiguous()


def test_w4a16_workspaces():
    """The workspace of a call without shape-only guesses: the size function covers every group
    size and type, and calls whose scales are not of x's type get one for their K slices."""
    from b200q._patches import _native
    L = _native.lib()
    for M, N, K in ((1, 5120, 5120), (2, 1024, 2048), (16, 5120, 13824), (40, 515, 1024), (300, 129, 256)):
        every = [L.b200q_w4a16_workspace_bytes(M, N, K, g, x, s)
                 for g in (32, 64, 128) for x in (0, 1) for s in (1, 2, 3)]
        assert max(every) == L.b200q_w4a16_workspace_size(M, N, K)
    assert L.b200q_w4a16_workspace_bytes(1, 5120, 5120, 128, 0, 1) == 0  # the integer kernel
    assert L.b200q_w4a16_workspace_bytes(1, 5120, 5120, 128, 0, 3) > 0
    for bad in ((0, 8, 64, 64), (2, 8, 64, 48), (2, 8, 96, 64)):
        assert L.b200q_w4a16_workspace_bytes(*bad, 0, 1) == 0


def test_build_without_a_host_compiler(tmp_path, monkeypatch, capsys):
    """The library is whole without the bindings: a machine that cannot compile them gets it,
    and a message, in place of an error."""
    import importlib.util
    import os
    from conftest import PACK_DIR
    spec = importlib.util.spec_from_file_location("b200q_build_test", PACK_DIR / "csrc" / "build.py")
    build = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(build)
    monkeypatch.setattr(build, "OUT", str(tmp_path / "libb200q.so"))
    monkeypatch.setattr(build, "BINDINGS", str(tmp_path / "b200q_bindings.so"))
    monkeypatch.setattr(build, "newer", lambda target, sources: target.endswith(".o"))  # objects are there
    linked = ["true"]
    monkeypatch.setattr(build, "link_cmd", lambda objects: linked)
    monkeypatch.setenv("CXX", "no-such-compiler")
    assert build.build() == build.OUT
    assert "no-such-compiler" in capsys.readouterr().out and not os.path.exists(build.BINDINGS)
    monkeypatch.delenv("CXX")
    assert build.bindings_lack() is None
    linked[0] = "false"  # what does not link is still an error
    with pytest.raises(RuntimeError):
        build.build()
