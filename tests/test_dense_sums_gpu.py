"""f32 results of dense_matmul over a long k: what the sums of the tensor cores lose.

A tensor core adds 16 products at a time to an f32 sum and cuts the result off: on
average half a step (2^-24 to 2^-25) of the sum so far, always towards zero, so a sum
of J additions loses J 2^-24 of it at most on average (2/3 of that where its size grows
as a random walk's). A sum is cut into parts of at most 2048 k, 128 additions, which
are added in f32 with rounding: 2^-17 of the result, 7.6e-6 (and the activation's own
2^-20). SwiGLU is a product of two such sums, one of them with a slope of at most 1.13
relative to itself where it is positive, and up to |z| more where it is negative."""

import pytest
import torch

pytestmark = pytest.mark.gpu

BF, F32 = torch.bfloat16, torch.float32
LOSS = 2.0 ** -17 * 2 / 3  # random operands: 5.1e-6


@pytest.fixture(autouse=True)
def _no_device_error():
    yield
    from dw_tpu_b200 import _lib
    _lib.raise_on_device_error()


def _operands(m, k, n, seed=0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    x = torch.randn((m, k), generator=g, device="cuda").to(BF)
    w = (torch.randn((n, k), generator=g, device="cuda") * k ** -0.5).to(BF)
    return x, w


def _off(got, ref):
    return float((got.double() - ref).norm() / ref.norm())


# Pair kernel (prompts of many tiles), split kernel with k over one CTA (decode batches
# with many rows of w) and over more, few rows.
SHAPES = [(2048, 8192, 4096), (1024, 8200, 8200), (300, 16384, 9000), (64, 8192, 32768),
          (16, 12288, 40960), (129, 8192, 20000), (1024, 8192, 256), (4, 8192, 512),
          (64, 65536, 512), (20, 16384, 20000)]


@pytest.mark.parametrize("m,k,n", SHAPES)
def test_f32_results_of_a_long_k(m, k, n):
    import dw_tpu_b200 as dw
    x, w = _operands(m, k, n)
    z = x.double() @ w.double().T
    assert _off(dw.dense_matmul(x, w, out_dtype=F32), z) < LOSS + 2.0 ** -20
    g, u = z[:, :n // 2], z[:, n // 2:]
    swiglu = g * torch.sigmoid(g) * u
    assert _off(dw.dense_matmul(x, w, act="swiglu", out_dtype=F32), swiglu) < 2.13 * LOSS + 2.0 ** -19


@pytest.mark.parametrize("m,k,n", SHAPES)
def test_every_value_of_a_long_k(m, k, n):
    """Each part of the sum once, in its place: whole numbers whose sums f32 holds, with
    bias, residual and rows off 16 bytes; and the same bits again."""
    import dw_tpu_b200 as dw
    g = torch.Generator(device="cuda").manual_seed(k)
    x = torch.randint(-3, 4, (m, k), generator=g, device="cuda").to(BF)
    w = torch.randint(-3, 4, (n, k), generator=g, device="cuda").to(BF)
    z = x.double() @ w.double().T
    b = torch.randint(-9, 10, (n,), generator=g, device="cuda").to(F32)
    r = torch.randint(-99, 100, (m, n), generator=g, device="cuda").to(F32)
    assert torch.equal(dw.dense_matmul(x, w, out_dtype=F32).double(), z)
    got = dw.dense_matmul(x, w, bias=b, residual=r, residual_scale=0.5, out_dtype=F32)
    assert torch.equal(got.double(), z + b + 0.5 * r)
    wide = torch.empty((m, n + 3), device="cuda")
    off = dw.dense_matmul(x, w, bias=b, residual=r, residual_scale=0.5, out=wide[:, 1:n + 1])
    assert torch.equal(off, got)
    assert torch.equal(dw.dense_matmul(x, w, bias=b, residual=got, out=got).double(),
                       2 * z + 2 * b + 0.5 * r)


def test_two_streams_and_a_graph():
    """Calls of every kernel with sums in parts, on two streams at once and replayed."""
    import dw_tpu_b200 as dw
    data = [_operands(m, k, n, seed=i) for i, (m, k, n) in
            enumerate([(1024, 4096, 4096), (64, 8192, 16384), (129, 8192, 4096), (16, 12288, 4096)])]
    alone = [dw.dense_matmul(x, w, out_dtype=F32) for x, w in data]
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    for s in streams:
        s.wait_stream(torch.cuda.current_stream())
    got = []
    for turn in range(10):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                x, w = data[(turn + 2 * i) % 4]
                got.append(((turn + 2 * i) % 4, dw.dense_matmul(x, w, out_dtype=F32)))
    torch.cuda.synchronize()
    assert all(torch.equal(y, alone[i]) for i, y in got)
    outs = [torch.empty_like(y) for y in alone]
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        for (x, w), out in zip(data, outs):
            dw.dense_matmul(x, w, out=out)
    for _ in range(3):
        for out in outs:
            out.fill_(float("nan"))
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(y, z) for y, z in zip(outs, alone))
