"""How the calls of the operators around the expert layer are reached: the
binding's absence and its build, without a GPU."""

import os
import subprocess
import sys
import sysconfig

import pytest
import torch

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


@pytest.fixture
def bare(tmp_path):
    """A folder with the package as it is, but for the binding."""
    package = tmp_path / "dw_tpu_b200"
    package.mkdir()
    for name in os.listdir(os.path.join(ROOT, "dw_tpu_b200")):
        if not name.startswith(("_bind", "__pycache__")):
            (package / name).symlink_to(os.path.join(ROOT, "dw_tpu_b200", name))
    return tmp_path


def _run(code, cwd):
    r = subprocess.run([sys.executable, "-c", code], cwd=cwd, capture_output=True, text=True)
    assert r.returncode == 0, r.stderr[-2000:]


def test_the_expert_layer_needs_no_binding(bare):
    """The package imports, and the ops that the binding has no part in reach the
    library; its own calls say what is missing."""
    _run("import os, torch, dw_tpu_b200 as dw\n"
         "assert os.path.dirname(dw.__file__) == os.path.join(os.getcwd(), 'dw_tpu_b200')\n"
         "x = torch.zeros((4, 64), dtype=torch.bfloat16)\n"
         "for call in (lambda: dw.route_topk(x, 2), lambda: dw.dispatch_gather(x, x[0].int())):\n"
         "    try: call()\n"
         "    except ValueError as e: assert 'CUDA' in str(e), e\n"
         "    else: raise SystemExit('no refusal')\n"
         "for call in (lambda: dw.dense_matmul(x, x), lambda: dw.pre_norm(x, x[0]),\n"
         "             lambda: dw.route_grouped_topk(x, 4, 8, 4)):\n"
         "    try: call()\n"
         "    except ImportError as e: assert 'build it' in str(e), e\n"
         "    else: raise SystemExit('no refusal')\n", bare)


def test_a_binding_of_another_torch_is_refused(monkeypatch):
    from dw_tpu_b200 import _lib
    monkeypatch.setattr(_lib, "_bind", None)
    monkeypatch.setattr(torch, "__version__", "2.0.1+other")
    with pytest.raises(ImportError, match="built for torch .* this is 2.0.1.other: build it"):
        _lib.bind()
    monkeypatch.undo()
    mod = _lib.bind()
    assert mod.torch_version == str(torch.__version__)
    assert mod.__file__.endswith(sysconfig.get_config_var("EXT_SUFFIX"))


def test_a_binding_of_an_older_build_is_refused(bare):
    """One without its torch's version, under the plain name."""
    (bare / "dw_tpu_b200" / "_bind.py").write_text("")
    _run("import torch, dw_tpu_b200 as dw\n"
         "x = torch.zeros((4, 64), dtype=torch.bfloat16)\n"
         "try: dw.dense_matmul(x, x)\n"
         "except ImportError as e: assert 'built for torch another version' in str(e), e\n"
         "else: raise SystemExit('no refusal')\n", bare)


def test_forward_mode_derivatives_are_refused():
    """A tangent would be lost without a word."""
    import torch.autograd.forward_ad as fw

    import dw_tpu_b200 as dw
    x, w = torch.zeros((4, 64), dtype=torch.bfloat16), torch.zeros((64, 64), dtype=torch.bfloat16)
    v, f = torch.ones(64, dtype=torch.bfloat16), torch.zeros((4, 64))
    with fw.dual_level():
        def dual(t):
            return fw.make_dual(t.clone(), torch.ones_like(t))
        calls = [lambda: dw.dense_matmul(dual(x), w), lambda: dw.dense_matmul(x, dual(w)),
                 lambda: dw.dense_matmul(x, w, bias=dual(v)),
                 lambda: dw.dense_matmul(x, w, residual=dual(x)),
                 lambda: dw.dense_matmul(x, w, out=dual(x)),
                 lambda: dw.route_grouped_topk(dual(f), 4, 8, 4),
                 lambda: dw.route_grouped_topk(dual(f.half()), 4, 8, 4),
                 lambda: dw.route_grouped_topk(f, 4, 8, 4, bias=dual(f[0])),
                 lambda: dw.pre_norm(dual(x), v), lambda: dw.pre_norm(x, dual(v)),
                 lambda: dw.pre_norm(x, v, dual(v)), lambda: dw.post_norm(dual(x), x),
                 lambda: dw.post_norm(x, x, residual_out=dual(x)),
                 lambda: dw.pre_norm(x, v, out=dual(x)),
                 lambda: dw.post_norm(x, dual(x)), lambda: dw.post_norm(x, x, gate=dual(v)),
                 lambda: dw.post_norm(x, x, norm_weight=dual(v)),
                 lambda: dw.post_norm(x, x, next_weight=v, next_bias=dual(v))]
        for grad in (True, False):
            with torch.set_grad_enabled(grad):
                for call in calls:
                    with pytest.raises(ValueError, match="inference only"):
                        call()
        # No tangent, or none that is recorded: as far as the CUDA check.
        with pytest.raises(ValueError, match="CUDA"):
            dw.dense_matmul(x, w)
        with fw._set_fwd_grad_enabled(False), pytest.raises(ValueError, match="CUDA"):
            dw.dense_matmul(dual(x), w)


@pytest.mark.parametrize("kw,message", [
    (dict(logits=(1 << 20) + 4), "misaligned"), (dict(dt=4), "dtype"), (dict(ld=63), "shorter"),
    (dict(ids=(1 << 20) + 4 * 64 * 8 - 4), "overlaps"), (dict(t=-1), "bad shape"),
])
def test_refusals_of_64_bit_logits(kw, message):
    from dw_tpu_b200 import _lib
    a = dict(logits=1 << 20, dt=_lib.F64, ld=64, t=4, e=64, k=4, groups=8, keep=4, scoring=1, gs=1,
             renorm=1, scale=1.0, bias=None, nv=-1, ids=2 << 20, w32=None, w16=None, stream=None)
    a.update(kw)
    assert _lib.load().dwm_route_grouped_topk(*a.values()) == -1
    assert message in _lib.last_error()
