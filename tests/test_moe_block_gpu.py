"""MoEBlock: the norms, router, group-limited routing, FP4 experts and shared
expert of a block run together, against a plain fp32 restatement and against
its operators called one by one."""

import pytest
import torch

from tests.gpu_util import gemm_rel_tol, torch_layer_reference, torch_round_bf16

pytestmark = pytest.mark.gpu

BF, F32 = torch.bfloat16, torch.float32
E, H, I, K = 16, 512, 256, 4


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


def _block(dw, max_tokens, shared=True, post=True, nxt=True, act_limit=None, **kw):
    from dw_tpu_b200 import synthetic
    raw = synthetic.moe_weights(E, H, I, seed=5, device="cuda")
    for name in ("s13", "s2"):  # keep activations O(1): scales 2^-9..2^-6
        setattr(raw, name, synthetic.random_e8m0(getattr(raw, name).shape, 6, "cuda", lo=118,
                                                 hi=121))
    layer = dw.MoELayer(raw.to_b200(), K, max_tokens, act_limit=act_limit)
    args = dict(num_groups=4, topk_groups=2, routed_scale=2.0,
                router_bias=_randn(3, E, scale=0.05, dtype=F32))
    if shared:
        args.update(shared_w13=_randn(7, 2 * I, H, scale=H ** -0.5),
                    shared_w2=_randn(8, H, I, scale=I ** -0.5))
    if post:
        args.update(post_weight=_randn(9, H, scale=0.2, mean=1.0))
    if nxt:
        args.update(next_weight=_randn(10, H, scale=0.2, mean=1.0))
    args.update(kw)
    block = dw.MoEBlock(layer, _randn(1, E, H, scale=0.05), _randn(2, H, scale=0.2, mean=1.0),
                        **args)
    return block, raw


def _norm(v, w, eps=1e-6):
    return v * torch.rsqrt(v.square().mean(1, keepdim=True) + eps) * w.float()


def _reference(block, raw, x, h, gate, limit):
    """x' and h' in fp32 from the block's own routing and normed input (both
    checked by their own tests), rounding where the block does."""
    t = x.shape[0]
    ids, w = block.layer.ids[:t], block.layer.w16[:t]
    y = torch_layer_reference(h, ids, w, raw.w13, raw.s13, raw.w2, raw.s2, limit).float()
    if block.shared_w13 is not None:
        a = h.float() @ block.shared_w13.float().T
        g, u = a[:, :I], a[:, I:]
        if limit is not None:
            g, u = g.clamp(max=limit), u.clamp(-limit, limit)
        y = torch_round_bf16(y + torch_round_bf16(g * torch.sigmoid(g) * u) @
                             block.shared_w2.float().T)
    if block.post_weight is not None:
        y = _norm(y, block.post_weight)
    if gate is not None:
        y = y * gate.float()
    r = block.residual_scale * x.float() + block.scale * y
    return r, None if block.next_weight is None else _norm(r, block.next_weight)


def _rel(a, b):
    return float((a.float() - b).norm() / b.norm())


@pytest.mark.parametrize("t", [1, 5, 64, 700])
@pytest.mark.parametrize("shared,post,nxt,limit,dtype,gated", [
    (True, True, True, None, BF, False), (True, False, True, 7.0, F32, True),
    (False, True, False, None, F32, True), (False, False, True, None, BF, False)])
def test_block_matches_reference(dw, t, shared, post, nxt, limit, dtype, gated):
    block, raw = _block(dw, 700, shared, post, nxt, limit, scale=0.75, residual_scale=1.25)
    x = _randn(20 + t, t, H, dtype=dtype)
    gate = _randn(21, t, 1, mean=0.5) if gated else None
    r, hn = block(x, gate=gate)
    assert r.dtype == dtype
    # The routing is that of the block's own logits.
    w, ids = dw.route_grouped_topk(block.logits[:t], K, 4, 2, routed_scale=2.0,
                                   bias=block.router_bias)
    assert torch.equal(ids, block.layer.ids[:t]) and torch.equal(w, block.layer.w16[:t])
    h = block.h[:t]
    ref_h = _norm(x.float(), block.norm_weight)
    assert _rel(h, ref_h) < 2 ** -8
    rr, hr = _reference(block, raw, x, h, gate, limit)
    # Two products deep, and one rounding to bf16 of the result.
    tol = 2 * gemm_rel_tol(H) + 2 ** -8
    assert _rel(r, rr) < tol
    if nxt:
        assert hn.dtype == BF and _rel(hn, hr) < tol
    else:
        assert hn is None


def test_block_is_its_operators(dw):
    t = 33
    block, _ = _block(dw, 64)
    x = _randn(30, t, H)
    r, hn = block(x)
    h = dw.pre_norm(x, block.norm_weight)
    logits = dw.dense_matmul(h, block.router, out_dtype=F32)
    w, ids = dw.route_grouped_topk(logits, K, 4, 2, routed_scale=2.0, bias=block.router_bias)
    y = block.layer.experts(h, ids, w, torch.empty((t, H), device="cuda"))
    s1 = dw.dense_matmul(h, block.shared_w13, act="swiglu")
    y = dw.dense_matmul(s1, block.shared_w2, residual=y)
    r2, hn2 = dw.post_norm(y, x, norm_weight=block.post_weight, next_weight=block.next_weight)
    assert torch.equal(r, r2) and torch.equal(hn, hn2)
    # Two blocks in a row: the second takes the first one's h'; the stream in place.
    r3, _ = block(r, h=hn)
    again, _ = block(r.clone(), h=hn.clone())
    assert torch.equal(r3, again)
    stream = r.clone()
    got, _ = block(stream, h=hn, out=stream)
    assert got is stream and torch.equal(stream, r3)


@pytest.mark.parametrize("t,valid", [(48, 20), (48, 0)])
def test_block_padding(dw, t, valid):
    """Padding tokens get the shared expert alone, and do not change the others."""
    block, _ = _block(dw, 64)
    x = _randn(31, t, H)
    r, hn = block(x, num_valid_tokens=valid)
    assert bool((block.layer.w16[valid:t] == 0).all())
    assert bool((block.routed[valid:t] == 0).all())
    r, hn = r.clone(), hn.clone()
    if valid:
        full = block(x)
        # The same experts' rows, in groups of other sizes: f32 sums in another order.
        assert _rel(r[:valid], full[0][:valid].float()) < gemm_rel_tol(H)


def test_block_graph_and_stream(dw):
    t = 64
    block, _ = _block(dw, t)
    x = _randn(32, t, H)
    base = [v.clone() for v in block(x)]
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        other = [v.clone() for v in block(x)]
    s.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(base, other))
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        got = block(x)
    x.copy_(_randn(33, t, H))
    for _ in range(2):
        g.replay()
    torch.cuda.synchronize()
    got = [v.clone() for v in got]
    assert all(torch.equal(a, b) for a, b in zip(got, block(x)))


def test_block_refusals(dw):
    block, raw = _block(dw, 8)
    layer, router, nw = block.layer, block.router, block.norm_weight
    with pytest.raises(ValueError, match="max_tokens"):
        block(_randn(1, 9, H))
    with pytest.raises(ValueError, match="h must"):
        block(_randn(1, 4, H), h=_randn(1, 4, H, dtype=F32))
    with pytest.raises(ValueError, match="router"):
        dw.MoEBlock(layer, router.T, nw)
    with pytest.raises(ValueError, match="together"):
        dw.MoEBlock(layer, router, nw, shared_w2=block.shared_w2)
    with pytest.raises(ValueError, match="shared_w13"):
        dw.MoEBlock(layer, router, nw, shared_w13=block.shared_w2, shared_w2=block.shared_w13)


def test_block_without_tokens(dw):
    block, _ = _block(dw, 8)
    r, hn = block(_randn(1, 0, H))
    assert r.shape == hn.shape == (0, H)
