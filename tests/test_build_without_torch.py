"""The library, its host program and the oracle build where torch is not
installed: the binding of the long-context operators alone needs it."""
import importlib
import sys

STEPS = ("build_synth", "build_i4d", "build_torch", "build_host", "build_oracle")


def test_without_torch_all_but_the_binding_is_built(pkg, monkeypatch, capsys):
    build = importlib.import_module("4pe_u250_b200.build")
    done = []
    for step in STEPS:
        if step != "build_torch":
            monkeypatch.setattr(build, step, lambda step=step: done.append(step))
    monkeypatch.setitem(sys.modules, "torch", None)  # an import of it fails
    build.main()
    assert sorted(done) == sorted(s for s in STEPS if s != "build_torch")
    assert "torch" in capsys.readouterr().out


def test_a_binding_that_does_not_build_is_an_error(pkg, monkeypatch):
    build = importlib.import_module("4pe_u250_b200.build")
    done = []
    for step in STEPS:
        monkeypatch.setattr(build, step, lambda step=step: done.append(step))

    def broken():
        raise ImportError("a header")
    monkeypatch.setattr(build, "build_torch", broken)
    try:
        build.main()
    except ImportError:
        assert "build_oracle" in done
    else:
        raise AssertionError("accepted")
