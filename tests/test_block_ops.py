"""Refusals of the operators around the expert layer (dense_matmul,
route_grouped_topk, pre_norm / post_norm): host checks only, no GPU."""

import pytest
import torch

FAKE = 1 << 20  # never dereferenced: every call below fails its checks
MB = 1 << 20


@pytest.fixture(scope="module")
def lib():
    from dw_tpu_b200 import _lib
    return _lib.load()


def _dense(lib, **kw):
    a = dict(x=FAKE, ldx=64, w=2 * FAKE, ldw=64, m=16, n=32, k=64, bias=None, bdt=1, act=0,
             limit=0.0, res=None, rdt=0, ldr=0, rs=1.0, out=8 * FAKE, odt=0, ldo=32, stream=None)
    assert set(kw) <= set(a)
    a.update(kw)
    return lib.dwm_dense_matmul(*a.values())


@pytest.mark.parametrize("kw,message", [
    (dict(k=63), "multiple of 8"), (dict(k=0), "bad shape"), (dict(n=0), "bad shape"),
    (dict(m=-1), "bad shape"), (dict(act=9), "activation"), (dict(act=-1), "activation"),
    (dict(act=1, n=33), "odd"), (dict(act=2, limit=0.0), "act_limit"),
    (dict(odt=2), "bf16 or f32"), (dict(bias=FAKE, bdt=2), "bf16 or f32"),
    (dict(ldx=60), "shorter"), (dict(ldw=56), "shorter"), (dict(ldo=31), "shorter"),
    (dict(res=FAKE, ldr=16), "shorter"), (dict(ldx=68), "16 bytes"), (dict(ldw=68), "16 bytes"),
    (dict(ldw=1 << 40), "too long"), (dict(x=None), "NULL"), (dict(out=None), "NULL"),
    (dict(x=FAKE + 8), "aligned"), (dict(w=FAKE + 2), "aligned"), (dict(out=8 * FAKE + 1), "misaligned"),
    (dict(odt=1, out=8 * FAKE + 2), "misaligned"), (dict(out=FAKE), "overlaps an input"),
    (dict(out=2 * FAKE + 32), "overlaps an input"),
    (dict(bias=8 * FAKE + 64, bdt=1), "overlaps an input"),
    (dict(res=8 * FAKE + 64, ldr=32), "overlaps the residual"),
    (dict(res=8 * FAKE, ldr=64), "overlaps the residual"),
    (dict(res=8 * FAKE, ldr=32, rdt=1), "overlaps the residual"),
])
def test_dense_refusals(lib, kw, message):
    from dw_tpu_b200 import _lib
    assert _dense(lib, **kw) == -1
    assert message in _lib.last_error()


@pytest.mark.parametrize("kw,ok", [
    (dict(ldx=512, ldo=512, out=FAKE + 128), True),       # the columns behind x's
    (dict(ldx=512, ldo=512, out=FAKE + 126), False),
    (dict(ldx=512, ldo=512, out=FAKE + 1024 - 64), True),  # and before the next row's
    (dict(ldx=512, ldo=512, out=FAKE + 1024 - 62), False),
    (dict(ldx=512, ldo=520, out=FAKE + 128), False),      # rows of other distances
    (dict(ldx=512, ldo=512, out=FAKE - 64), True),
    (dict(ldx=512, ldo=512, out=FAKE - 62), False),
])
def test_dense_columns_of_one_tensor(lib, kw, ok):
    """x and out may be columns of the same rows; they may not share a byte.
    (k = 64: 128 bytes of x and 64 of out a row; the residual's overlap stops
    the calls that get past the check of x.)"""
    from dw_tpu_b200 import _lib
    assert _dense(lib, **kw, res=kw["out"] + 2, ldr=kw["ldo"]) == -1
    assert _lib.last_error().endswith("without being it" if ok else "an input")


def test_empty_batches_are_no_work(lib):
    assert _dense(lib, m=0, x=None, out=None) == 0
    assert _route(lib, t=0, logits=None, ids=None) == 0
    assert _norm(lib, t=0, y=None, res=None, r=None, ho=None) == 0


def _route(lib, **kw):
    a = dict(logits=FAKE, dt=1, ld=64, t=4, e=64, k=4, groups=8, keep=4, scoring=1, gs=1, renorm=1,
             scale=1.0, bias=None, nv=-1, ids=2 * FAKE, w32=None, w16=None, stream=None)
    assert set(kw) <= set(a)
    a.update(kw)
    return lib.dwm_route_grouped_topk(*a.values())


@pytest.mark.parametrize("kw,message", [
    (dict(dt=2), "dtype"), (dict(t=-1), "bad shape"), (dict(e=0), "bad shape"),
    (dict(e=2048, groups=8), "bad shape"), (dict(groups=0), "num_groups"),
    (dict(groups=7), "num_groups"), (dict(groups=64), "num_groups"), (dict(keep=0), "topk_groups"),
    (dict(keep=9), "topk_groups"), (dict(k=0), "top_k"), (dict(k=33), "top_k"),
    (dict(k=9, keep=1), "top_k"), (dict(scoring=3), "scoring"), (dict(gs=2), "group score"),
    (dict(ld=63), "shorter"), (dict(logits=None), "NULL"), (dict(ids=None), "NULL"),
])
def test_route_refusals(lib, kw, message):
    from dw_tpu_b200 import _lib
    assert _route(lib, **kw) == -1
    assert message in _lib.last_error()


def _norm(lib, **kw):
    a = dict(y=MB, ydt=0, ldy=64, res=2 * MB, rdt=0, ldres=64, t=4, h=64, kind=0, eps=1e-6,
             inner=1, w2=3 * MB, b2=None, gate=None, gmode=0, ldg=0, scale=1.0, rs=1.0,
             w1=4 * MB, b1=None, wdt=0, r=5 * MB, ldr=64, ho=6 * MB, hdt=0, ldh=64, stream=None)
    assert set(kw) <= set(a)
    a.update(kw)
    return lib.dwm_block_norm(*a.values())


@pytest.mark.parametrize("kw,message", [
    (dict(t=-1), "bad shape"), (dict(h=0), "bad shape"), (dict(h=16385), "exceeds"),
    (dict(kind=2), "norm kind"), (dict(eps=0.0), "eps"), (dict(eps=float("nan")), "eps"),
    (dict(rdt=2), "bf16 or f32"), (dict(ydt=2), "bf16 or f32"), (dict(wdt=2), "bf16 or f32"),
    (dict(gmode=2), "gate mode"), (dict(gate=MB, gmode=0), "gate mode"),
    (dict(gate=MB, gmode=4), "gate mode"), (dict(res=None), "NULL residual"),
    (dict(r=None), "NULL r_out"), (dict(w2=None), "needs its weight"),
    (dict(w1=None), "needs its weight"), (dict(y=None), "without y"),
    (dict(y=None, r=None, inner=0, ho=None), "without y"), (dict(ldy=63), "stride"),
    (dict(ldres=0), "stride"), (dict(ldr=1), "stride"), (dict(ldh=63), "stride"),
    (dict(gate=7 * MB, gmode=3, ldg=63), "stride"), (dict(gate=7 * MB, gmode=1, ldg=0), "stride"),
    (dict(r=6 * MB), "two outputs"), (dict(r=2 * MB + 128), "r_out overlaps"),
    (dict(r=2 * MB, ldr=128), "r_out overlaps"), (dict(ho=MB, hdt=1), "h_out overlaps"),
    (dict(ho=3 * MB - 64), "weight or the gate"), (dict(r=4 * MB), "weight or the gate"),
    (dict(gate=5 * MB, gmode=2), "weight or the gate"),
])
def test_norm_refusals(lib, kw, message):
    from dw_tpu_b200 import _lib
    assert _norm(lib, **kw) == -1
    assert message in _lib.last_error()


def test_python_refusals_without_gpu():
    import dw_tpu_b200 as dw
    bf, f32 = torch.bfloat16, torch.float32
    x, w = torch.zeros((4, 64), dtype=bf), torch.zeros((32, 64), dtype=bf)
    for call in (lambda: dw.dense_matmul(x, w), lambda: dw.pre_norm(x, torch.ones(64)),
                 lambda: dw.route_grouped_topk(x, 4, 8, 4)):
        with pytest.raises(ValueError, match="CUDA"):
            call()
    with pytest.raises(ValueError, match="act"):
        dw.dense_matmul(x, w, act="tanh")
    with pytest.raises(ValueError, match="act_limit"):
        dw.dense_matmul(x, w, act="swiglu_clamp")
    with pytest.raises(ValueError, match="out_dtype"):
        dw.dense_matmul(x, w, out=torch.zeros((4, 32), dtype=bf), out_dtype=f32)
    with pytest.raises(ValueError, match="gradient"):
        dw.dense_matmul(x, w.clone().requires_grad_())
    with pytest.raises(ValueError, match="gradient"):
        dw.pre_norm(x, torch.ones(64, requires_grad=True))
    with pytest.raises(ValueError, match="next_weight"):
        dw.post_norm(x, x, out=x)
    with pytest.raises(ValueError, match="gradient"):
        dw.route_grouped_topk(x.float().requires_grad_(), 4, 8, 4)


@pytest.mark.parametrize("kw,message", [
    (dict(m=2 ** 31 - 100), "too large"), (dict(n=2 ** 31 - 100), "too large"),
    (dict(k=2 ** 31 - 104), "too large"),
])
def test_dense_sizes_past_the_tiles(lib, kw, message):
    from dw_tpu_b200 import _lib
    assert _dense(lib, **kw) == -1
    assert message in _lib.last_error()


@pytest.mark.parametrize("kw,message", [
    (dict(logits=FAKE + 2), "misaligned"), (dict(ids=2 * FAKE + 2), "misaligned"),
    (dict(bias=FAKE + 1), "misaligned"), (dict(w32=FAKE + 2), "misaligned"),
    (dict(w16=FAKE + 1), "misaligned"), (dict(ids=FAKE + 16), "overlaps"),
    (dict(w16=2 * FAKE + 56), "overlaps"), (dict(w32=2 * FAKE), "overlaps"),
    (dict(bias=2 * FAKE + 60), "overlaps"),
])
def test_route_memory_refusals(lib, kw, message):
    from dw_tpu_b200 import _lib
    assert _route(lib, **kw) == -1
    assert message in _lib.last_error()


@pytest.mark.parametrize("kw", [
    dict(y=MB + 1), dict(res=2 * MB + 1), dict(rdt=1, res=2 * MB + 2), dict(w1=4 * MB + 1),
    dict(w2=3 * MB + 1), dict(b1=7 * MB + 1), dict(b2=7 * MB + 1), dict(r=5 * MB + 1),
    dict(ho=6 * MB + 1), dict(hdt=1, ho=6 * MB + 2), dict(gate=7 * MB + 1, gmode=2),
])
def test_norm_misaligned(lib, kw):
    from dw_tpu_b200 import _lib
    assert _norm(lib, **kw) == -1
    assert "misaligned" in _lib.last_error()
