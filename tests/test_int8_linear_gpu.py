"""8-bit integer quantisation and linear against their definitions in 64 bits.

The quantised integers and the integer sums are exact, so they are compared bit for bit.  The
scaled result rounds three times in f32 (the row's scale, the product of the scales, the product
with the sum and, past 2^24, the sum's conversion: 4 x 2^-24 relative) and once to bf16 (2^-8).
"""
import pytest
import torch

import ds_kernels

pytestmark = pytest.mark.gpu
bf16 = torch.bfloat16


def rows(m, k, seed, spread=True):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(m, k, generator=g)
    if spread:
        x = x * torch.exp(2 * torch.randn(m, 1, generator=g))
    return x.to(bf16)


def quant64(x):
    """(q, scale in 64 bits) of CPU bf16 rows."""
    x = x.double()
    a = x.abs().amax(-1, keepdim=True)
    bad = ~torch.isfinite(a)
    q = torch.where((a > 0) & ~bad, torch.round(127 * x / a), torch.zeros_like(x))
    s = torch.where(bad, torch.full_like(a, float("nan")), a / 127)
    return q.to(torch.int8), s[..., 0]


def weights(n, k, seed):
    g = torch.Generator().manual_seed(seed)
    w = torch.randint(-127, 128, (n, k), generator=g, dtype=torch.int8)
    return w, (torch.rand(n, generator=g) + 0.5) * 1e-3


def linear64(x, w, ws):
    q, s = quant64(x)
    return (q.double() @ w.double().t()) * s[:, None] * ws.double()


def check(out, ref):
    o, err = out.cpu().double(), None
    err = (o - ref).abs()
    tol = ref.abs() * (2.0 ** -8 + 4 * 2.0 ** -24) + 2.0 ** -133
    assert (err <= tol).all(), (err - tol).max()


@pytest.mark.parametrize("m,k", [(1, 16), (3, 48), (7, 1424), (130, 2048), (2, 8208), (1, 65536)])
def test_quantize_is_exact(m, k):
    x = rows(m, k, m + k)
    x[0, :k // 2] = x[0].abs().max() / 2          # 127 x / a = 63.5: a tie in every place
    q, s = ds_kernels.int8_quantize(x.cuda())
    rq, rs = quant64(x)
    assert torch.equal(q.cpu(), rq)
    assert ((s.cpu().double() - rs).abs() <= rs * 2.0 ** -24).all()


@pytest.mark.parametrize("top", [2.0 ** -133, 3 * 2.0 ** -133, 2.0 ** -126, 1e-30, 1e30, 3.3895e38])
def test_quantize_at_the_ends_of_the_range(top):
    g = torch.Generator().manual_seed(1)
    x = (torch.rand(4, 64, generator=g, dtype=torch.float64) * 2 - 1) * top
    x[:, 0] = top
    x = x.to(bf16)
    q, s = ds_kernels.int8_quantize(x.cuda())
    rq, rs = quant64(x)
    assert torch.equal(q.cpu(), rq)
    assert ((s.cpu().double() - rs).abs() <= rs * 2.0 ** -24 + 2.0 ** -150).all()


def test_every_pair_of_mantissas_goes_to_its_side():
    # all 128 mantissas of the value against all of the row's maximum, over nine binades
    m = (1 + torch.arange(128) / 128.0)
    x = torch.cat([m * 2.0 ** -e for e in range(9)])[None].expand(128, -1) * 1.0
    x = torch.where(x <= m[:, None], x, torch.zeros_like(x))
    x = torch.cat([x, m[:, None].expand(-1, 16)], dim=1).to(bf16)
    q, _ = ds_kernels.int8_quantize(x.cuda())
    assert torch.equal(q.cpu(), quant64(x)[0])


@pytest.mark.parametrize("value", [float("inf"), -float("inf"), float("nan")])
def test_a_row_that_is_not_finite_spoils_itself_alone(value):
    x = rows(5, 64, 3)
    x[2, 17] = value
    x[4] = 0
    w, ws = weights(24, 64, 4)
    q, s = ds_kernels.int8_quantize(x.cuda())
    assert torch.isnan(s[2]) and (q[2] == 0).all() and s[4] == 0 and (q[4] == 0).all()
    out = ds_kernels.int8_linear(x.cuda(), w.cuda(), ws.cuda())
    assert torch.isnan(out[2]).all() and (out[4] == 0).all()
    keep = [0, 1, 3, 4]
    check(out[keep], linear64(x[keep], w, ws))


@pytest.mark.parametrize("m", [1, 2, 7, 8, 9, 16, 17, 31, 33, 64, 65, 127, 128, 129, 257, 640])
@pytest.mark.parametrize("k,n", [(16, 8), (144, 136), (2048, 264), (1424, 2840)])
def test_linear(m, k, n):
    x, (w, ws) = rows(m, k, m), weights(n, k, n)
    check(ds_kernels.int8_linear(x.cuda(), w.cuda(), ws.cuda()), linear64(x, w, ws))


@pytest.mark.parametrize("m,k,n", [(1, 8192, 2048), (64, 2048, 9792), (64, 8192, 2048), (5, 32768, 128),
                                   (3, 131072, 8), (300, 16, 4096), (2049, 512, 776), (1, 64, 40000)])
def test_linear_shapes_of_the_decode_and_prefill_paths(m, k, n):
    x, (w, ws) = rows(m, k, m), weights(n, k, n)
    check(ds_kernels.int8_linear(x.cuda(), w.cuda(), ws.cuda()), linear64(x, w, ws))


def test_the_largest_sums_do_not_wrap():
    k = 131072
    x = torch.ones(2, k, dtype=bf16)
    x[1] = -1
    w = torch.full((16, k), -128, dtype=torch.int8)
    w[8:] = 127
    out = ds_kernels.int8_linear(x.cuda(), w.cuda(), torch.ones(16, device="cuda"))
    check(out, linear64(x, w, torch.ones(16)))


def test_strided_rows_leading_dims_and_misaligned_views():
    w, ws = weights(40, 64, 5)
    big = rows(6, 200, 6).cuda()
    for x in (big[:, 8:72], big[:, 3:67], big[::2, 16:80], big[:, :64].reshape(2, 3, 64),
              big[:, :128].t()[:64].t(), big.t()[:64, :].t()):
        out = ds_kernels.int8_linear(x, w.cuda(), ws.cuda())
        assert out.shape == (*x.shape[:-1], 40)
        check(out.reshape(-1, 40), linear64(x.reshape(-1, 64).cpu(), w, ws))
        q, _ = ds_kernels.int8_quantize(x)
        assert torch.equal(q.reshape(-1, 64).cpu(), quant64(x.reshape(-1, 64).cpu())[0])


def test_one_row_expanded_and_empty_batches():
    w, ws = weights(16, 32, 7)
    x = rows(1, 32, 8)
    out = ds_kernels.int8_linear(x.cuda().expand(5, 32), w.cuda(), ws.cuda())
    check(out, linear64(x.expand(5, 32), w, ws))
    assert ds_kernels.int8_linear(x.cuda()[:0], w.cuda(), ws.cuda()).shape == (0, 16)
    assert ds_kernels.int8_linear(x.cuda(), w.cuda()[:0], ws.cuda()[:0]).shape == (1, 0)
    assert ds_kernels.int8_linear(x.cuda()[0], w.cuda(), ws.cuda()).shape == (16,)


def test_bits_do_not_depend_on_the_batch():
    # a row's result is the same alone and among others (exact sums; one scaling)
    x, (w, ws) = rows(300, 2048, 9), weights(520, 2048, 10)
    x, w, ws = x.cuda(), w.cuda(), ws.cuda()
    whole = ds_kernels.int8_linear(x, w, ws)
    for m in (1, 5, 16, 33, 64, 100, 129):
        assert torch.equal(ds_kernels.int8_linear(x[:m], w, ws), whole[:m])


def test_other_stream_own_workspace_and_graph_replay():
    x, (w, ws) = rows(33, 1024, 11).cuda(), weights(264, 1024, 12)
    w, ws = w.cuda(), ws.cuda()
    want = ds_kernels.int8_linear(x, w, ws)
    space = torch.empty(ds_kernels.int8_linear_workspace_size(33, 264, 1024), dtype=torch.uint8, device="cuda")
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        assert torch.equal(ds_kernels.int8_linear(x, w, ws, workspace=space), want)
    torch.cuda.current_stream().wait_stream(side)
    static, graph = x.clone(), torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = ds_kernels.int8_linear(static, w, ws)
    for seed in (13, 14):
        y = rows(33, 1024, seed).cuda()
        static.copy_(y)
        graph.replay()
        assert torch.equal(out, ds_kernels.int8_linear(y, w, ws))


def test_custom_operators():
    x, (w, ws) = rows(7, 64, 15).cuda(), weights(24, 64, 16)
    w, ws = w.cuda(), ws.cuda()
    torch.library.opcheck(torch.ops.ds_kernels.int8_quantize.default, (x,))
    torch.library.opcheck(torch.ops.ds_kernels.int8_linear.default, (x, w, ws))

    def f(x):
        q, s = ds_kernels.int8_quantize(x)
        return ds_kernels.int8_linear(x, w, ws) * 2, q, s

    for got, want in zip(torch.compile(f, fullgraph=True)(x), f(x)):
        assert torch.equal(got, want)


@pytest.mark.parametrize("m,k,n", [(8200, 272, 2072), (4500, 912, 4616)])
def test_linear_with_several_tiles_for_each_pair_of_ctas(m, k, n):
    """297 and 342 tiles of 256 x 256 for at most 74 pairs, ragged at every edge: accumulators, ring and
    channel scales go on from tile to tile.  More tiles than the ring has stages, and fewer."""
    x, (w, ws) = rows(m, k, m), weights(n, k, n)
    check(ds_kernels.int8_linear(x.cuda(), w.cuda(), ws.cuda()), linear64(x, w, ws))


@pytest.mark.parametrize("k", [1136, 1152, 2160, 2304, 2560, 3136, 5248])
@pytest.mark.parametrize("m", [1, 2, 3, 4, 5, 16, 17, 33, 64, 100, 128])
def test_linear_with_parts_of_k_for_clusters_of_3_6_and_7(m, k):
    for n in (8, 264):
        x, (w, ws) = rows(m, k, m), weights(n, k, n)
        check(ds_kernels.int8_linear(x.cuda(), w.cuda(), ws.cuda()), linear64(x, w, ws))
