"""dense_matmul, route_grouped_topk and pre_norm / post_norm on the GPU against
64-bit restatements of their formulas.

Tolerances. A value is rounded once on its way out (half a step:
eps / 2 of the value), on top of f32 arithmetic, whose error is counted
against the absolute values that were summed."""

import math

import pytest
import torch

pytestmark = pytest.mark.gpu

BF, F32, F64 = torch.bfloat16, torch.float32, torch.float64
HALF = {BF: 2.0 ** -8, F32: 2.0 ** -24}


@pytest.fixture(scope="module")
def dw():
    import dw_tpu_b200
    return dw_tpu_b200


@pytest.fixture(autouse=True)
def _no_device_error():
    yield
    from dw_tpu_b200 import _lib
    _lib.raise_on_device_error()


def _randn(seed, *shape, scale=1.0, mean=0.0, dtype=BF):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return (torch.randn(shape, generator=g, device="cuda") * scale + mean).to(dtype)


def _close(got, ref, tol, what=""):
    assert got.shape == ref.shape
    err = (got.double() - ref).abs()
    bad = ~(err <= tol)
    assert not bad.any(), (f"{what}: {int(bad.sum())} of {bad.numel()} off, worst "
                           f"{float((err / tol).nan_to_num(1e9).max()):.3g} tolerances at "
                           f"{bad.nonzero()[0].tolist()}")


# ---------------------------------------------------------------------------
# dense_matmul
# ---------------------------------------------------------------------------

LIMIT = 0.8


def _dense_ref(x, w, bias, act, residual, rs, out_dtype):
    """(reference, tolerance) in 64 bits. k products are added in f32 in some
    order, each addition off by a step (2^-23, the tensor core may truncate) of
    a sum that the absolute values bound; the activations pass that on with a
    slope of at most 1.13 and add 2^-20 of their own (the MUFU forms and erff)."""
    xd, wd = x.double(), w.double()
    z = xd @ wd.T
    e = (x.shape[1] + 4) * 2.0 ** -23 * (xd.abs() @ wd.abs().T)
    if bias is not None:
        z = z + bias.double()
        e = e + 2.0 ** -23 * (z.abs() + bias.double().abs())
    if act in ("swiglu", "swiglu_clamp"):
        h = z.shape[1] // 2
        g, u, eg, eu = z[:, :h], z[:, h:], e[:, :h], e[:, h:]
        if act == "swiglu_clamp":
            g, u = g.clamp(max=LIMIT), u.clamp(-LIMIT, LIMIT)
        s = g * torch.sigmoid(g)
        a = s * u
        e = 1.13 * eg * (u.abs() + eu) + s.abs() * eu + 2.0 ** -20 * a.abs()
    elif act == "silu":
        a = z * torch.sigmoid(z)
        e = 1.13 * e + 2.0 ** -20 * a.abs()
    elif act == "gelu":
        a = 0.5 * z * torch.erfc(-z / math.sqrt(2.0))
        # 1 + erf(v) is off by a few steps of 1, however small it is.
        e = 1.13 * e + 2.0 ** -21 * z.abs()
    elif act == "gelu_tanh":
        a = z * torch.sigmoid(math.sqrt(8 / math.pi) * (z + 0.044715 * z ** 3))
        # The exponent's own rounding: |2u| 2^-22 of the result.
        e = 1.13 * e + 2.0 ** -20 * a.abs() * (1 + z.abs() + z.abs() ** 3)
    else:
        a = z
    if residual is not None:
        r = rs * residual.double()
        e = e + 2.0 ** -23 * (a.abs() + r.abs())
        a = a + r
    return a, e + HALF[out_dtype] * (a.abs() + e) + 1e-38


def _dense_case(dw, m, k, n, act=None, bias=None, res=None, out_dtype=BF, seed=0):
    x, w = _randn(seed, m, k), _randn(seed + 1, n, k, scale=k ** -0.5)
    n_out = n // 2 if act in ("swiglu", "swiglu_clamp") else n
    b = _randn(seed + 2, n, scale=0.3, dtype=bias) if bias else None
    r = _randn(seed + 3, m, n_out, dtype=res) if res else None
    got = dw.dense_matmul(x, w, bias=b, act=act, act_limit=LIMIT, residual=r, residual_scale=0.75,
                          out_dtype=out_dtype)
    assert got.dtype == out_dtype
    ref, tol = _dense_ref(x, w, b, act, r, 0.75, out_dtype)
    _close(got, ref, tol, f"m={m} k={k} n={n} {act}")
    return got


@pytest.mark.parametrize("m", [1, 2, 15, 16, 17, 33, 64, 65, 128, 129, 257, 300])
@pytest.mark.parametrize("k,n", [(8, 1), (64, 16), (72, 130), (1000, 777), (2048, 256)])
def test_dense_sizes(dw, m, k, n):
    _dense_case(dw, m, k, n, seed=m + k + n)


@pytest.mark.parametrize("m,k,n", [(1, 4096, 256), (3, 512, 4096), (64, 4096, 4096),
                                   (1024, 2048, 4096), (2049, 520, 1030), (700, 4096, 257),
                                   (5000, 64, 8)])
@pytest.mark.parametrize("out_dtype", [BF, F32])
def test_dense_larger(dw, m, k, n, out_dtype):
    _dense_case(dw, m, k, n, bias=F32, out_dtype=out_dtype, seed=m + n)


@pytest.mark.parametrize("act", [None, "silu", "gelu", "gelu_tanh", "swiglu", "swiglu_clamp"])
@pytest.mark.parametrize("m", [5, 100, 600])
@pytest.mark.parametrize("n", [2, 62, 514, 1026])
def test_dense_epilogue(dw, act, m, n):
    """Every activation with bias, residual and both output types; widths whose
    halves end inside a tile."""
    for i, (b, r, o) in enumerate([(F32, None, BF), (BF, BF, F32), (None, F32, BF), (BF, F32, F32)]):
        _dense_case(dw, m, 136, n, act=act, bias=b, res=r, out_dtype=o, seed=10 * i + n)


@pytest.mark.parametrize("m,n", [(7, 40), (300, 520), (1000, 1000)])
@pytest.mark.parametrize("out_dtype", [BF, F32])
def test_dense_strides_and_untouched_surroundings(dw, m, n, out_dtype):
    """Rows of x, w, residual and out inside wider tensors: what is between and
    behind the rows is neither read (NaN) nor written."""
    k = 200
    x = torch.full((m + 1, k + 24), math.nan, dtype=BF, device="cuda")
    w = torch.full((n + 1, k + 8), math.nan, dtype=BF, device="cuda")
    x[:m, 16:16 + k] = _randn(1, m, k)
    w[:n, :k] = _randn(2, n, k, scale=0.1)
    for pad, off in ((5, 3), (16, 8)):
        r = torch.full((m + 1, n + pad), math.nan, dtype=BF, device="cuda")
        r[:m, off:off + n] = _randn(3, m, n)
        out = torch.full((m + 2, n + pad + off), -7.0, dtype=out_dtype, device="cuda")
        xv, wv, rv, ov = x[:m, 16:16 + k], w[:n, :k], r[:m, off:off + n], out[:m, off:off + n]
        dw.dense_matmul(xv, wv, residual=rv, residual_scale=0.75, out=ov)
        ref, tol = _dense_ref(xv, wv, None, None, rv, 0.75, out_dtype)
        _close(ov, ref, tol)
        ov.fill_(-7.0)
        assert bool((out == -7.0).all())


@pytest.mark.parametrize("m,dtype", [(9, BF), (500, F32)])
def test_dense_adds_to_the_residual_in_place(dw, m, dtype):
    x, w = _randn(1, m, 256), _randn(2, 384, 256, scale=0.06)
    r = _randn(3, m, 384, dtype=dtype)
    ref, tol = _dense_ref(x, w, None, "silu", r, 0.5, dtype)
    got = dw.dense_matmul(x, w, act="silu", residual=r, residual_scale=0.5, out=r)
    assert got is r
    _close(r, ref, tol)


@pytest.mark.parametrize("m", [1, 40, 600])
def test_dense_rows_are_their_own(dw, m):
    """NaN and infinities of one row of x stay in that row; a row's bits do not
    depend on the other rows' values."""
    x, w = _randn(1, m + 3, 512), _randn(2, 300, 512, scale=0.05)
    base = dw.dense_matmul(x, w)
    y = x.clone()
    y[0, 5], y[m, 7], y[m + 1, 100] = math.inf, math.nan, -math.inf
    got = dw.dense_matmul(y, w)
    keep = [i for i in range(m + 3) if i not in (0, m, m + 1)]
    assert torch.equal(got[keep], base[keep])
    assert bool(got[m].isnan().all())
    assert bool(got[0].isinf().all()) and bool(got[m + 1].isinf().all())


@pytest.mark.parametrize("m", [1, 8, 9, 33, 70])
@pytest.mark.parametrize("k", [2056, 4096, 8192])
@pytest.mark.parametrize("n", [2, 66, 256])
def test_dense_long_k(dw, m, k, n):
    """Few columns of w: their k is shared by several CTAs, and ends inside a step."""
    _dense_case(dw, m, k, n, bias=F32, res=BF, out_dtype=F32, seed=m + k + n)
    _dense_case(dw, m, k, n, act="swiglu", bias=BF, res=F32, out_dtype=BF, seed=m * k + n)


@pytest.mark.parametrize("m", [2, 13, 100, 333])
@pytest.mark.parametrize("k,n", [(8, 4000), (520, 1032), (1000, 776)])
@pytest.mark.parametrize("act", ["gelu", "swiglu"])
def test_dense_few_hundred_rows(dw, m, k, n, act):
    """In place, in rows that start anywhere, with a row of NaN."""
    x, w = _randn(1, m, k), _randn(2, n, k, scale=k ** -0.5)
    cols = n // 2 if act == "swiglu" else n
    ref, tol = None, None
    for pad, off in ((0, 0), (7, 3)):
        buf = torch.full((m, cols + pad), -7.0, dtype=BF, device="cuda")
        r = buf[:, off:off + cols]
        r.copy_(_randn(3, m, cols))
        if ref is None:
            ref, tol = _dense_ref(x, w, None, act, r, 0.5, BF)
            base = dw.dense_matmul(x, w, act=act, residual=r, residual_scale=0.5)
            _close(base, ref, tol)
        dw.dense_matmul(x, w, act=act, residual=r, residual_scale=0.5, out=r)
        assert torch.equal(r, base)
        r.fill_(-7.0)
        assert bool((buf == -7.0).all())
    x[m // 2, 3] = math.nan
    got = dw.dense_matmul(x, w, act=act, residual=_randn(3, m, cols), residual_scale=0.5)
    keep = [i for i in range(m) if i != m // 2]
    assert torch.equal(got[keep], base[keep]) and bool(got[m // 2].isnan().all())


@pytest.mark.parametrize("n,pad,off", [(1544, 0, 0), (1544, 24, 8), (1546, 0, 0), (1544, 3, 1)])
@pytest.mark.parametrize("res,out_dtype", [(None, BF), (BF, BF), (F32, BF), (BF, F32), (F32, F32)])
def test_dense_many_rows(dw, n, pad, off, res, out_dtype):
    """Rows for several 256-row tiles (the last of one row), every epilogue with a
    residual of either type, in rows that start on 16 bytes and that do not;
    what lies between the rows stays as it was."""
    m, k = 2049, 1032
    x, w, b = _randn(1, m, k), _randn(2, n, k, scale=k ** -0.5), _randn(3, n, scale=0.3)
    for act in (None, "gelu_tanh", "swiglu_clamp"):
        cols = n // 2 if act == "swiglu_clamp" else n
        r = None
        if res is not None:
            r = torch.full((m, cols + pad + off), math.nan, dtype=res, device="cuda")
            r[:, off:off + cols] = _randn(4, m, cols, dtype=res)
            r = r[:, off:off + cols]
        buf = torch.full((m + 1, cols + pad + off), -7.0, dtype=out_dtype, device="cuda")
        out = buf[:m, off:off + cols]
        args = dict(bias=b, act=act, act_limit=LIMIT, residual_scale=0.75)
        ref, tol = _dense_ref(x, w, b, act, r, 0.75, out_dtype)
        got = dw.dense_matmul(x, w, residual=r, out=out, **args)
        assert got is out
        _close(out, ref, tol, f"{act}")
        if res == out_dtype:  # in place
            again = r.clone() if pad == 0 else r
            dw.dense_matmul(x, w, residual=again, out=again, **args)
            assert torch.equal(again, out)
        out.fill_(-7.0)
        assert bool((buf == -7.0).all())


@pytest.mark.parametrize("m", [3, 700])
def test_dense_clamp_keeps_nan(dw, m):
    x, w = _randn(1, m, 128), _randn(2, 512, 128)
    x[1, 7] = math.nan
    got = dw.dense_matmul(x, w, act="swiglu_clamp", act_limit=1.0)
    assert bool(got[1].isnan().all()) and not bool(got[0].isnan().any())


def test_dense_empty(dw):
    assert dw.dense_matmul(_randn(1, 0, 64), _randn(2, 32, 64)).shape == (0, 32)


@pytest.mark.parametrize("m,n", [(3, 264), (700, 512)])
def test_dense_offsets_past_32_bits(dw, m, n):
    """Rows of x, residual and out whose offsets pass 2^31 elements."""
    k, ld = 128, (1 << 31) // (m - 1) // 8 * 8 + 520
    buf = torch.empty((m - 1) * ld + n, dtype=BF, device="cuda")
    assert (m - 1) * ld > 1 << 31
    view = buf.as_strided((m, n), (ld, 1))
    view.copy_(_randn(1, m, n))
    xv = view[:, :k]
    w = _randn(2, n - 256, k, scale=0.1)
    r = view[:, 256:]
    ref, tol = _dense_ref(xv, w, None, None, r, 1.0, BF)
    got = dw.dense_matmul(xv, w, residual=r)
    _close(got, ref, tol)
    dw.dense_matmul(xv, w, residual=r, out=r)  # other columns of x's rows
    assert torch.equal(r, got)


@pytest.mark.parametrize("m,n", [(2, 256), (96, 1000), (1500, 2048)])
def test_dense_same_bits_again_other_stream_and_graph(dw, m, n):
    x, w = _randn(1, m, 1024), _randn(2, n, 1024, scale=0.03)
    r = _randn(3, m, n // 2, dtype=F32)
    args = dict(act="swiglu", residual=r)
    base = dw.dense_matmul(x, w, **args)
    assert torch.equal(dw.dense_matmul(x, w, **args), base)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        other = dw.dense_matmul(x, w, **args)
    # Two captured graphs of the same call, replayed together on two streams.
    outs, graphs = [torch.empty_like(base) for _ in range(2)], []
    torch.cuda.current_stream().wait_stream(s)
    assert torch.equal(other, base)
    for o in outs:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            dw.dense_matmul(x, w, out=o, **args)
        graphs.append(g)
    x.copy_(_randn(4, m, 1024))
    base = dw.dense_matmul(x, w, **args)
    torch.cuda.synchronize()
    for _ in range(3):
        with torch.cuda.stream(s):
            graphs[0].replay()
        graphs[1].replay()
    torch.cuda.synchronize()
    assert torch.equal(outs[0], base) and torch.equal(outs[1], base)


# ---------------------------------------------------------------------------
# route_grouped_topk
# ---------------------------------------------------------------------------

def _route_ref(x, k, groups, keep, renorm, scoring, group_score, scale, bias):
    x = x.double().cpu()
    t, e = x.shape
    per = e // groups
    if scoring == "softmax":
        d = x - x.amax(1, keepdim=True)
        d[x == x.amax(1, keepdim=True)] = 0.0
        s = torch.exp(d) / torch.exp(d).sum(1, keepdim=True)
        s[(x == -math.inf).all(1)] = 0.0
    elif scoring == "sigmoid":
        s = 1 / (1 + torch.exp(-x))
    else:
        s = (x.clamp(min=0) + torch.log1p(torch.exp(-x.abs()))).sqrt()
    c = x if bias is None else s + bias.double().cpu()
    cg = c.reshape(t, groups, per)
    if group_score == "max":
        v = cg.amax(2)
    else:
        top, at = cg.sort(dim=2, descending=True, stable=True)
        if bias is None:
            top = s.reshape(t, groups, per).gather(2, at)
        v = top[:, :, :2].sum(2)
    best = v.sort(dim=1, descending=True, stable=True)[1][:, :keep]
    open_ = torch.zeros((t, groups), dtype=torch.bool).scatter_(1, best, True)
    # Closed experts behind every open one, -inf or not.
    order = c.sort(dim=1, descending=True, stable=True)[1]
    is_open = open_.repeat_interleave(per, 1).gather(1, order)
    ids = order.gather(1, (~is_open).to(torch.int8).sort(dim=1, stable=True)[1])[:, :k]
    w = s.gather(1, ids)
    if renorm:
        total = w.sum(1, keepdim=True)
        w = torch.where(total == 0, torch.zeros_like(w), w / total)
    return w * scale, ids.int()


def _route_case(dw, x, k, groups, keep, renorm=True, scoring="sigmoid", group_score="top2",
                scale=2.5, bias=None, **kw):
    w, ids = dw.route_grouped_topk(x, k, groups, keep, renorm, scoring, group_score, scale, F32,
                                   bias, **kw)
    rw, ri = _route_ref(x, k, groups, keep, renorm, scoring, group_score, scale, bias)
    assert ids.dtype == torch.int32 and torch.equal(ids.cpu(), ri)
    # f32 exp, division and a sum of at most 32 weights.
    _close(w.cpu(), rw, 2.0 ** -19 * rw.abs() + 1e-37)
    w16, ids16 = dw.route_grouped_topk(x, k, groups, keep, renorm, scoring, group_score, scale, BF,
                                       bias, **kw)
    assert torch.equal(ids16, ids) and torch.equal(w16, w.to(BF))
    return w, ids


@pytest.mark.parametrize("scoring", ["softmax", "sigmoid", "sqrtsoftplus"])
@pytest.mark.parametrize("group_score", ["max", "top2"])
@pytest.mark.parametrize("dtype", [F32, BF])
@pytest.mark.parametrize("with_bias", [False, True])
def test_route_scorings(dw, scoring, group_score, dtype, with_bias):
    for t, e, groups, keep, k in [(333, 256, 8, 4, 8), (50, 160, 8, 3, 6), (65, 48, 3, 2, 9)]:
        x = _randn(t + e, t, e, scale=1.5, dtype=dtype)
        b = _randn(7, e, scale=0.1, dtype=F32) if with_bias else None
        for renorm in (False, True):
            _route_case(dw, x, k, groups, keep, renorm, scoring, group_score, bias=b)


@pytest.mark.parametrize("t", [0, 1, 2, 5, 1023])
@pytest.mark.parametrize("e,groups,keep,k", [
    (1, 1, 1, 1), (2, 2, 1, 1), (8, 8, 8, 8), (31, 31, 7, 7), (32, 32, 32, 32), (33, 1, 1, 32),
    (34, 17, 16, 32), (64, 2, 1, 32), (100, 5, 5, 3), (513, 27, 26, 17), (1024, 32, 1, 32),
    (1024, 4, 3, 32), (992, 31, 30, 32)])
def test_route_sizes(dw, t, e, groups, keep, k):
    x = _randn(t + e, t, e, scale=2.0, dtype=F32)
    b = _randn(9, e, scale=0.2, dtype=F32)
    _route_case(dw, x, k, groups, keep, bias=b)
    _route_case(dw, x, k, groups, keep, scoring="softmax", group_score="max")


@pytest.mark.parametrize("with_bias", [False, True])
@pytest.mark.parametrize("scoring", ["softmax", "sigmoid", "sqrtsoftplus"])
def test_route_ties_go_to_the_lower_index(dw, scoring, with_bias):
    """Logits of three values only: almost every comparison is a tie, and the
    group sums tie too."""
    g = torch.Generator().manual_seed(1)
    x = torch.randint(-1, 2, (500, 128), generator=g).float().cuda()
    b = torch.randint(0, 2, (128,), generator=g).float().cuda() * 0.5 if with_bias else None
    for gs in ("max", "top2"):
        _route_case(dw, x, 8, 8, 3, scoring=scoring, group_score=gs, bias=b)
    _route_case(dw, torch.zeros((3, 128), device="cuda"), 8, 8, 3, scoring=scoring, bias=b)


def test_route_near_ties_are_ordered_in_64_bits(dw):
    """Logits one f32 step apart, and sigmoids that round to 1 in f32: the f32
    scores tie (or swap), the order of the 64-bit ones holds."""
    e = 64
    base = torch.linspace(17.0, 24.0, e)  # 1 - sigmoid: 4e-8 .. 4e-11
    g = torch.Generator().manual_seed(2)
    x = torch.stack([base[torch.randperm(e, generator=g)] for _ in range(200)]).cuda()
    b = torch.full((e,), 0.25, device="cuda")
    _route_case(dw, x, 8, 4, 2, bias=b)
    _route_case(dw, x, 8, 4, 2)
    ulp = torch.arange(e, dtype=torch.int32)
    near = (torch.tensor(0.7).view(torch.int32) + ulp).view(F32)
    y = torch.stack([near[torch.randperm(e, generator=g)] for _ in range(200)]).cuda()
    for scoring in ("softmax", "sigmoid", "sqrtsoftplus"):
        _route_case(dw, y, 8, 4, 2, scoring=scoring, bias=b)
        _route_case(dw, y, 8, 4, 2, scoring=scoring)
    # A bias far above the scores hides them from f32 altogether.
    big = torch.full((e,), 1.0e6, device="cuda")
    _route_case(dw, _randn(3, 100, e, dtype=F32), 8, 4, 2, bias=big)


def test_route_masked_and_non_finite(dw):
    x = _randn(1, 64, 96, dtype=F32)
    x[:, 40:] = -math.inf              # masked experts, whole groups among them
    x[1] = -math.inf                   # nothing left
    x[2, 3], x[2, 90] = math.inf, math.inf
    x[3, :] = -math.inf
    x[3, 95] = 0.0
    x[4] = -3.0e38
    for scoring in ("softmax", "sigmoid", "sqrtsoftplus"):
        for gs in ("max", "top2"):
            ok = x if scoring != "sqrtsoftplus" else torch.cat([x[:2], x[3:]])  # inf / inf
            _route_case(dw, ok, 8, 6, 3, scoring=scoring, group_score=gs)
    b = torch.zeros(96, device="cuda")
    b[:50] = -math.inf
    _route_case(dw, x[5:], 8, 6, 3, bias=b)
    # NaN: below every number, in its own row only, ids still distinct.
    y = x.clone()
    y[10, :39], y[11, 0] = math.nan, math.nan
    w, ids = dw.route_grouped_topk(y, 8, 6, 3, dtype=F32)
    rw, ri = dw.route_grouped_topk(x, 8, 6, 3, dtype=F32)
    rest = [i for i in range(64) if i not in (10, 11)]
    assert torch.equal(ids[rest], ri[rest]) and torch.equal(w[rest], rw[rest])
    assert all(len(set(r)) == 8 for r in ids.tolist())
    assert 0 not in ids[11].tolist()
    assert ids[10].tolist()[0] == 39


# From some tokens an SM on, several tokens share a warp.
MANY = 2001


@pytest.mark.parametrize("e,groups,keep,k", [
    (1, 1, 1, 1), (8, 8, 8, 8), (31, 31, 7, 7), (32, 32, 32, 32), (33, 1, 1, 32), (34, 17, 16, 32),
    (64, 2, 1, 32), (100, 5, 5, 3), (160, 8, 3, 6), (256, 8, 4, 8), (250, 5, 2, 8), (513, 27, 26, 17),
    (1024, 32, 1, 32), (1024, 4, 3, 32), (992, 31, 30, 32)])
def test_route_many_tokens(dw, e, groups, keep, k):
    for dtype in (F32, BF):
        x = _randn(e + k, MANY, e, scale=2.0, dtype=dtype)
        b = _randn(9, e, scale=0.2, dtype=F32)
        _route_case(dw, x, k, groups, keep, bias=b)
        _route_case(dw, x, k, groups, keep, False, "softmax", "max")
        _route_case(dw, x, k, groups, keep, scoring="sqrtsoftplus")
        _route_case(dw, x, k, groups, keep, scoring="softmax", bias=b)


def _undecided(x, groups, keep, scoring, bias):
    """Rows whose order of groups 64-bit arithmetic leaves open. The sum of the
    scores of logits p and q steps of d = 2^-24 above another is 2 s + (p + q) s' d
    + (p^2 + q^2) s'' d^2 / 2, so two groups of the same p + q may differ by as little
    as s'' d^2 = 2^-50. A score (at most 2) has errors of half a step of 2^-52 or a
    step of a value below 1 from exp, log1p, their sum and the root, 2^-51 together;
    with the bias and the sum of two (at most 4) that makes 2^-49 at most. Where two
    sums computed here are 2^-47 or less apart, they may truly be 2^-48 apart in
    either order, or 2^-48 the other way in the kernel's own arithmetic."""
    x = x.double().cpu()
    s = {"softmax": lambda v: v.softmax(1), "sigmoid": torch.sigmoid,
         "sqrtsoftplus": lambda v: (v.clamp(min=0) + torch.log1p(torch.exp(-v.abs()))).sqrt()}
    s = s[scoring](x)
    c = s if bias is None else s + bias.double().cpu()
    v = c.reshape(len(x), groups, -1).topk(2, dim=2)[0].sum(2).sort(dim=1, descending=True)[0]
    return v[:, keep - 1] - v[:, keep] <= 2.0 ** -47


def test_route_many_tokens_ties_and_masks(dw):
    """Ties, values one f32 step apart, masked experts and NaN, between ordinary
    tokens of the same warp."""
    g = torch.Generator().manual_seed(4)
    e = 128
    near = (torch.tensor(0.7).view(torch.int32) + torch.arange(e, dtype=torch.int32)).view(F32)
    x = torch.randn((MANY, e), generator=g) * 1.5
    x[::5] = torch.randint(-1, 2, x[::5].shape, generator=g).float()
    x[1::7] = torch.stack([near[torch.randperm(e, generator=g)] for _ in range(len(x[1::7]))])
    x[2::11, 16:112] = -math.inf
    x[3::97] = -math.inf
    x = x.cuda()
    b = (torch.randint(0, 2, (e,), generator=g).float() * 0.5).cuda()
    steps = torch.zeros(MANY, dtype=torch.bool)
    steps[1::7] = True
    steps[2::11] = steps[3::97] = False
    for scoring in ("softmax", "sigmoid", "sqrtsoftplus"):
        for bias in (None, b):
            _route_case(dw, x, 8, 8, 3, scoring=scoring, group_score="max", bias=bias)
            w, ids = dw.route_grouped_topk(x, 8, 8, 3, True, scoring, "top2", 2.5, F32, bias)
            rw, ri = _route_ref(x, 8, 8, 3, True, scoring, "top2", 2.5, bias)
            sure = ~(steps & _undecided(x, 8, 3, scoring, bias))
            assert int((~sure).sum()) < MANY // 20
            assert torch.equal(ids.cpu()[sure], ri[sure])
            # (The others' weights are as close as their logits: 128 steps of 2^-24.)
            _close(w.cpu(), rw, 2.0 ** -19 * rw.abs() + 1e-37 + 2.0 ** -16 * ~sure[:, None])
    y = x.clone()
    y[10, 1:] = math.nan
    w, ids = dw.route_grouped_topk(y, 8, 8, 3, dtype=F32, num_valid_tokens=MANY - 3)
    rw, ri = dw.route_grouped_topk(x, 8, 8, 3, dtype=F32)
    rest = [i for i in range(MANY - 3) if i != 10]
    assert torch.equal(ids[rest], ri[rest]) and torch.equal(w[rest], rw[rest])
    assert ids[10, 0] == 0 and len(set(ids[10].tolist())) == 8
    assert not bool(ids[MANY - 3:].any()) and not bool(w[MANY - 3:].any())


@pytest.mark.parametrize("valid", [0, 1, 7, 100])
def test_route_padding_strides_stream(dw, valid):
    buf = torch.full((12, 70), math.nan, device="cuda")
    buf[:9, 3:67] = _randn(1, 9, 64, dtype=F32)
    x = buf[:9, 3:67]
    w, ids = dw.route_grouped_topk(x, 4, 8, 2, dtype=F32, num_valid_tokens=valid)
    rw, ri = _route_ref(x, 4, 8, 2, True, "sigmoid", "top2", 1.0, None)
    rw[valid:], ri[valid:] = 0, 0
    assert torch.equal(ids.cpu(), ri)
    _close(w.cpu(), rw, 2.0 ** -19 * rw + 1e-37)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        w2, ids2 = dw.route_grouped_topk(x, 4, 8, 2, dtype=F32, num_valid_tokens=valid)
    s.synchronize()
    assert torch.equal(ids, ids2) and torch.equal(w, w2)


def test_route_without_groups_is_route_topk(dw):
    """One group: route_topk's choice (f32 logits apart enough to order in f32)."""
    x = torch.stack([torch.randperm(256, generator=torch.Generator().manual_seed(i))
                     for i in range(40)]).float().cuda() / 64 - 2
    w, ids = dw.route_grouped_topk(x, 8, 1, 1, dtype=F32)
    rw, ri = dw.route_topk(x, 8, dtype=F32)
    assert torch.equal(ids, ri)
    _close(w, rw.double(), 2.0 ** -19 * rw.double())


# ---------------------------------------------------------------------------
# pre_norm / post_norm
# ---------------------------------------------------------------------------

EPS = 1e-5


def _norm64(v, w, b, kind):
    mean = v.mean(1, keepdim=True) if kind == "layer" else torch.zeros_like(v[:, :1])
    rstd = ((v - mean).square().mean(1, keepdim=True) + EPS).rsqrt()
    out = (v - mean) * rstd * w
    return (out if b is None else out + b), rstd


def _post_ref(y, res, w2, b2, gate, scale, rs, w1, b1, kind, r_dtype, h_dtype):
    """References and tolerances. F = 2^-18 covers the f32 arithmetic of a
    value against the absolute values it is made of: at most 32 + 5 + 16
    additions in sequence for a sum over the row, an rsqrtf of 2 steps and
    some ten single operations, together below 2^6 steps of 2^-24."""
    F = 2.0 ** -18
    d = lambda t: None if t is None else t.double()  # noqa: E731
    y, res, w2, b2, gate, w1, b1 = map(d, (y, res, w2, b2, gate, w1, b1))
    n, size = y, y.abs()
    if w2 is not None:
        n, rstd = _norm64(y, w2, b2, kind)
        # v and its mean apart, and the bias
        size = rstd * (y.abs() + y.abs().mean(1, keepdim=True)) * w2.abs()
        if b2 is not None:
            size = size + b2.abs()
    if gate is not None:
        n, size = n * gate, size * gate.abs()
    r = rs * res + scale * n
    size = (rs * res).abs() + abs(scale) * size
    out = [(r, HALF[r_dtype] * r.abs() + F * size + 1e-38)]
    if w1 is not None:
        h, rstd = _norm64(r, w1, b1, kind)
        hs = rstd * (size + size.mean(1, keepdim=True)) * w1.abs()
        # The row's own errors change the statistics by as much again.
        hs = 2 * hs + h.abs() * rstd * size.square().mean(1, keepdim=True).sqrt()
        if b1 is not None:
            hs = hs + b1.abs()
        out.append((h, HALF[h_dtype] * h.abs() + F * hs + 1e-38))
    return out


def _gate(mode, t, h, dtype):
    shape = {"none": None, "token": (t, 1), "channel": (h,), "full": (t, h)}[mode]
    return None if shape is None else _randn(31, *shape, scale=0.5, mean=0.4, dtype=dtype)


@pytest.mark.parametrize("kind", ["rms", "layer"])
@pytest.mark.parametrize("t,h", [(1, 1), (1, 4096), (2, 7), (3, 8), (5, 100), (9, 1000), (7, 1024),
                                 (130, 1032), (64, 4096), (33, 5003), (4, 8192), (3, 8200),
                                 (2, 16384), (3, 16383), (1000, 512)])
def test_norm_sizes(dw, kind, t, h):
    w, b = _randn(1, h, scale=0.3, mean=1.0), _randn(2, h, scale=0.2) if kind == "layer" else None
    for dt in (BF, F32):
        x = _randn(t + h, t, h, scale=1.5, mean=0.3, dtype=dt)
        got = dw.pre_norm(x, w, b, eps=EPS, kind=kind)
        ref = _post_ref(torch.zeros_like(x), x, None, None, None, 0.0, 1.0, w, b, kind, F32, BF)[1]
        _close(got, *ref, f"pre {t}x{h}")
        y = _randn(t * h + 1, t, h, mean=0.1)
        gate = _gate("full", t, h, BF)
        r, hn = dw.post_norm(y, x, norm_weight=w, norm_bias=b, gate=gate, scale=1.25,
                             residual_scale=0.5, next_weight=w, next_bias=b, eps=EPS, kind=kind)
        (rr, rt), (hr, ht) = _post_ref(y, x, w, b, gate, 1.25, 0.5, w, b, kind, dt, BF)
        assert r.dtype == dt and hn.dtype == BF
        _close(r, rr, rt, f"r {t}x{h}")
        _close(hn, hr, ht, f"h {t}x{h}")


@pytest.mark.parametrize("gate", ["none", "token", "channel", "full"])
@pytest.mark.parametrize("inner", [False, True])
@pytest.mark.parametrize("nxt", [False, True])
@pytest.mark.parametrize("h", [264, 4001])
def test_post_norm_forms_and_types(dw, gate, inner, nxt, h):
    t = 37
    for i, (ydt, rdt, wdt, gdt, hdt) in enumerate([(BF, BF, BF, BF, BF), (F32, F32, F32, F32, F32),
                                                   (BF, F32, F32, BF, BF), (F32, BF, BF, F32, F32)]):
        kind = "rms" if i % 2 else "layer"
        y, x = _randn(i, t, h, dtype=ydt), _randn(i + 9, t, h, scale=2.0, dtype=rdt)
        w2 = _randn(3, h, mean=1.0, dtype=wdt) if inner else None
        b2 = _randn(4, h, dtype=wdt) if inner and i > 1 else None
        w1 = _randn(5, h, mean=1.0, dtype=wdt) if nxt else None
        b1 = _randn(6, h, dtype=wdt) if nxt and i > 1 else None
        g = _gate(gate, t, h, gdt)
        r, hn = dw.post_norm(y, x, norm_weight=w2, norm_bias=b2, gate=g, scale=-0.5,
                             residual_scale=1.5, next_weight=w1, next_bias=b1, eps=EPS, kind=kind,
                             out_dtype=hdt)
        refs = _post_ref(y, x, w2, b2, g, -0.5, 1.5, w1, b1, kind, rdt, hdt)
        _close(r, *refs[0])
        if nxt:
            assert hn.dtype == hdt
            _close(hn, *refs[1])
        else:
            assert hn is None


@pytest.mark.parametrize("t,h", [(5000, 100), (4999, 512), (2500, 333), (1301, 4096), (1300, 2000),
                                 (700, 5003), (601, 8192), (401, 9001), (307, 16384)])
@pytest.mark.parametrize("gate", ["none", "token", "channel", "full"])
def test_norm_many_rows(dw, t, h, gate):
    """More rows than the CTAs take at once, in every form; again in place, and
    several times over: the same bits."""
    for i, (ydt, rdt, wdt, hdt) in enumerate([(BF, BF, BF, BF), (BF, F32, F32, BF),
                                              (F32, BF, BF, F32)]):
        kind = ("rms", "layer")[(i + h) % 2]
        y, x = _randn(i, t, h, mean=0.2, dtype=ydt), _randn(i + 9, t, h, scale=2.0, dtype=rdt)
        w, b = _randn(3, h, mean=1.0, dtype=wdt), _randn(4, h, dtype=wdt)
        g = _gate(gate, t, h, ydt)
        for inner, nxt in ((True, True), (False, True), (True, False)):
            args = dict(norm_weight=w if inner else None, gate=g, scale=0.75, residual_scale=1.5,
                        next_weight=w if nxt else None, next_bias=b if nxt else None, eps=EPS,
                        kind=kind, out_dtype=hdt)
            r, hn = dw.post_norm(y, x, **args)
            refs = _post_ref(y, x, w if inner else None, None, g, 0.75, 1.5, w if nxt else None,
                             b, kind, rdt, hdt)
            _close(r, *refs[0], f"r {kind} {inner} {nxt}")
            if nxt:
                _close(hn, *refs[1], f"h {kind} {inner}")
            x2, y2 = x.clone(), y.clone()
            r2, h2 = dw.post_norm(y2, x2, residual_out=x2, out=y2 if nxt and ydt == hdt else None,
                                  **args)
            assert torch.equal(r2, r) and (hn is None or torch.equal(h2, hn))


@pytest.mark.parametrize("t,h", [(8192, 2048), (5000, 104), (1500, 5003)])
def test_pre_norm_many_rows_same_bits(dw, t, h):
    """An RMS norm alone has one sum a row, whose slots the next row reuses."""
    x, w = _randn(1, t, h), _randn(2, h, mean=1.0)
    ref, tol = _post_ref(torch.zeros_like(x), x, None, None, None, 0.0, 1.0, w, None, "rms", F32,
                         BF)[1]
    base = dw.pre_norm(x, w, eps=EPS)
    _close(base, ref, tol)
    for _ in range(20):
        assert torch.equal(dw.pre_norm(x, w, eps=EPS), base)


@pytest.mark.parametrize("h,pad,off", [(512, 8, 8), (512, 3, 1), (333, 5, 2), (4096, 16, 8)])
def test_norm_strides_and_untouched_surroundings(dw, h, pad, off):
    t = 11

    def inside(seed, dtype=BF, **kw):
        buf = torch.full((t + 1, h + pad + off), math.nan, dtype=dtype, device="cuda")
        v = buf[:t, off:off + h]
        v.copy_(_randn(seed, t, h, dtype=dtype, **kw))
        return v

    y, x, g = inside(1), inside(2, F32), inside(3)
    w = _randn(4, h, mean=1.0)
    bufs = [torch.full((t + 2, h + pad + off), -7.0, dtype=dt, device="cuda") for dt in (F32, BF)]
    ro, ho = (b[:t, off:off + h] for b in bufs)
    dw.post_norm(y, x, norm_weight=w, gate=g, next_weight=w, eps=EPS, residual_out=ro, out=ho)
    refs = _post_ref(y, x, w, None, g, 1.0, 1.0, w, None, "rms", F32, BF)
    _close(ro, *refs[0])
    _close(ho, *refs[1])
    for v, b in ((ro, bufs[0]), (ho, bufs[1])):
        v.fill_(-7.0)
        assert bool((b == -7.0).all())


@pytest.mark.parametrize("h", [1024, 4096, 1001])
def test_norm_in_place(dw, h):
    t = 70
    w = _randn(4, h, mean=1.0)
    y, x = _randn(1, t, h), _randn(2, t, h)
    r, hn = dw.post_norm(y, x, norm_weight=w, next_weight=w, eps=EPS)
    y1, x1 = y.clone(), x.clone()
    a, b = dw.post_norm(y1, x1, norm_weight=w, next_weight=w, eps=EPS, residual_out=x1, out=y1)
    assert a is x1 and b is y1
    assert torch.equal(x1, r) and torch.equal(y1, hn)
    p = dw.pre_norm(x, w, eps=EPS)
    x2 = x.clone()
    dw.pre_norm(x2, w, eps=EPS, out=x2)
    assert torch.equal(x2, p)
    # The block's output and the stream are one tensor: read twice, written once.
    r2, _ = dw.post_norm(x, x, scale=0.5, next_weight=w, eps=EPS)
    x3 = x.clone()
    dw.post_norm(x3, x3, scale=0.5, next_weight=w, eps=EPS, residual_out=x3)
    assert torch.equal(x3, r2)


def test_norm_special_rows(dw):
    """A zero row and a constant row (layer norm: no spread) are finite; NaN and
    infinities stay in their row; no rows are no work."""
    h = 600
    w, b = _randn(1, h, mean=1.0), _randn(2, h)
    x = _randn(3, 6, h, dtype=F32)
    x[0], x[1], x[2, 5], x[3, 9] = 0.0, 3.0, math.nan, math.inf
    base = dw.pre_norm(_randn(3, 6, h, dtype=F32), w, b, eps=EPS, kind="layer")
    got = dw.pre_norm(x, w, b, eps=EPS, kind="layer")
    assert torch.equal(got[4:], base[4:])
    assert torch.equal(got[0], b)
    # mean(3) is 3 to 2^-18, so what is left of the row is at most 3 2^-18 / sqrt(eps).
    _close(got[1], b.double(), 2.0 ** -8 * b.double().abs() + 3 * 2.0 ** -18 / EPS ** 0.5 * w.abs())
    assert bool(got[2].isnan().all()) and bool(got[3].isnan().any())
    assert bool((dw.pre_norm(x[:1], w, eps=EPS) == 0).all())
    e = torch.empty((0, h), device="cuda")
    r, hn = dw.post_norm(e, e, next_weight=w)
    assert r.shape == hn.shape == (0, h)


def test_norm_offsets_past_32_bits(dw):
    t, h, ld = 3, 1024, (1 << 30) + 1024
    x = torch.empty((t - 1) * ld + h, dtype=BF, device="cuda").as_strided((t, h), (ld, 1))
    x.copy_(_randn(1, t, h))
    w, y = _randn(2, h, mean=1.0), _randn(3, t, h)
    base = dw.post_norm(y, x.contiguous(), next_weight=w)
    r, hn = dw.post_norm(y, x, next_weight=w, residual_out=x)
    assert r is x and torch.equal(x, base[0]) and torch.equal(hn, base[1])


def test_norm_stream_and_graph(dw):
    t, h = 300, 4096
    w, g = _randn(2, h, mean=1.0), _randn(5, t, 1)
    y, x = _randn(3, t, h), _randn(1, t, h)
    base = dw.post_norm(y, x, norm_weight=w, gate=g, next_weight=w)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        other = dw.post_norm(y, x, norm_weight=w, gate=g, next_weight=w)
    s.synchronize()
    assert torch.equal(base[0], other[0]) and torch.equal(base[1], other[1])
    ro, ho = torch.empty_like(x), torch.empty_like(x)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        dw.post_norm(y, x, norm_weight=w, gate=g, next_weight=w, residual_out=ro, out=ho)
    x.copy_(_randn(8, t, h))
    base = dw.post_norm(y, x, norm_weight=w, gate=g, next_weight=w)
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(ro, base[0]) and torch.equal(ho, base[1])


def test_refusals_on_the_gpu(dw):
    x, w = _randn(1, 4, 64), _randn(2, 32, 64)
    for bad in (lambda: dw.dense_matmul(x.float(), w), lambda: dw.dense_matmul(x, w.T),
                lambda: dw.dense_matmul(x, w[:, :32]), lambda: dw.dense_matmul(x, w.cpu()),
                lambda: dw.dense_matmul(x, w, bias=torch.zeros(31, device="cuda")),
                lambda: dw.dense_matmul(x, w, residual=torch.zeros((4, 64), device="cuda")),
                lambda: dw.dense_matmul(x, w, out=x[:, :32]),
                lambda: dw.dense_matmul(x[:, 4:60], w[:, 4:60]),
                lambda: dw.pre_norm(x, w[0, :32]), lambda: dw.pre_norm(x.half(), w[0]),
                lambda: dw.pre_norm(x, w[0], w[1].float()),
                lambda: dw.pre_norm(x.T, torch.ones(4, device="cuda")),
                lambda: dw.post_norm(x, x[:, :32]), lambda: dw.post_norm(x, x, gate=w[:3]),
                lambda: dw.post_norm(x, x, norm_bias=w[0]),
                lambda: dw.post_norm(x, x, residual_out=x.float()),
                lambda: dw.route_grouped_topk(x, 4, 7, 2), lambda: dw.route_grouped_topk(x, 9, 8, 1),
                lambda: dw.route_grouped_topk(x, 4, 8, 2, scoring_fn="relu"),
                lambda: dw.route_grouped_topk(x, 4, 8, 2, group_score="sum"),
                lambda: dw.route_grouped_topk(x, 4, 8, 2, bias=torch.zeros(63, device="cuda"))):
        with pytest.raises(ValueError):
            bad()


def test_a_stream_of_its_own_needs_outputs(dw):
    """The tensors that a call allocates belong to the current stream."""
    from dw_tpu_b200 import ops
    x, w = _randn(1, 64, 256), _randn(2, 128, 256)
    base, s = dw.dense_matmul(x, w), torch.cuda.Stream()
    with pytest.raises(ValueError, match="outputs given"):
        ops.dense_matmul_out(x, w, None, stream=s.cuda_stream)
    with pytest.raises(ValueError, match="outputs given"):
        ops.block_norm_out(x, weight=w[0], stream=s.cuda_stream)
    with pytest.raises(ValueError, match="outputs given"):
        ops.block_norm_out(x, y=x, norm_weight=w[0], stream=s.cuda_stream)
    out = torch.empty_like(base)
    s.wait_stream(torch.cuda.current_stream())
    ops.dense_matmul_out(x, w, out, stream=s.cuda_stream)
    s.synchronize()
    assert torch.equal(out, base)


def test_calls_on_two_streams_at_once(dw):
    """Each stream's chain of calls overlaps its own launches; the other's run
    between them."""
    x, w, r = _randn(1, 1500, 1024), _randn(2, 2048, 1024, scale=0.03), _randn(3, 1500, 1024)
    nw = _randn(4, 1024, mean=1.0)

    def chain(v):
        for _ in range(4):
            a = dw.dense_matmul(v, w, act="swiglu")
            v, hn = dw.post_norm(a, v, norm_weight=nw, next_weight=nw)
            ids = dw.route_grouped_topk(hn[:, :256], 8, 8, 4)[1]
        return v, hn, ids

    base = [[t.clone() for t in chain(v)] for v in (x, r)]
    torch.cuda.synchronize()
    streams, got = [torch.cuda.Stream() for _ in range(2)], [None, None]
    for _ in range(3):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                got[i] = chain((x, r)[i])
    torch.cuda.synchronize()
    for b, g in zip(base, got):
        assert all(torch.equal(p, q) for p, q in zip(b, g))
