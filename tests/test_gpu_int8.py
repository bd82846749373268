"""The 8-bit projections against their definition in 64 bits.

Codes have to be equal: they are defined by real arithmetic.  An output is the exact sum,
rounded to fp32 (2^-24), times two scales (2^-24 each), and half a step of its type.  A
gated one is silu(g) u: g is off by 3 * 2^-24 of itself, which silu amplifies by at most
1 + |g|; the exponential's argument g log2(e) rounds once and its constant once, 2 |g| *
2^-24 of the exponential; the exponential itself, the sum, the quotient and the product
with u (off by 3 * 2^-24) come to less than 9 * 2^-24 (exponential and reciprocal within
2 ulp)."""
from __future__ import annotations

import pytest
import torch

from dflash_mlx import Int8Weight, linear_i8, matmul_i8, pack_weight_i8, quantize_rows_i8, quantize_weight_i8

pytestmark = pytest.mark.gpu

TYPES = (torch.bfloat16, torch.float16)


def quantised(x):
    """(codes, scales) of rows in 64 bits, on the CPU."""
    x = x.double()
    a = x.abs().amax(-1).clamp_min(2.0 ** -100)
    return (127 * x / a[..., None]).round().long(), a / 127


def product(codes, scale, w_codes, w_scale, gated=False):
    """(outputs, the gates) in 64 bits; the sums of codes are exact."""
    y = (codes.double() @ w_codes.double().T) * scale.double()[:, None] * w_scale.double()
    if not gated:
        return y, torch.zeros_like(y)
    g, u = y.chunk(2, -1)
    return g * torch.sigmoid(g) * u, g


def check(got, want, gate=None):
    gate = torch.zeros_like(want) if gate is None else gate
    tol = (12 + 5 * gate.abs()) * 2.0 ** -24 * want.abs() + torch.finfo(got.dtype).eps / 2 * want.abs()
    tol += torch.finfo(got.dtype).smallest_normal * torch.finfo(got.dtype).eps  # a step of the least values
    bad = (got.cpu().double() - want).abs() > tol
    assert not bad.any(), f"{int(bad.sum())} of {bad.numel()} beyond the tolerance"


def rows(M, K, dtype, seed):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(M, K, generator=g) * (0.1 + torch.rand(M, 1, generator=g))
    return (x * (1 + 20 * (torch.rand(K, generator=g) < 0.02))).to(dtype)


def weight(N, K, seed, scale=1.0):
    g = torch.Generator().manual_seed(seed)
    codes = torch.randint(-127, 128, (N, K), generator=g, dtype=torch.int8)
    return codes, scale * (0.5 + torch.rand(N, generator=g)) / 127 * K ** -0.5


SHAPES = [(1, 1, 1), (1, 16, 64), (2, 70001, 64), (3, 5, 7), (4, 48, 1024), (8, 2560, 640), (15, 1000, 2560), (16, 33, 129),
          (16, 2560, 9216), (17, 64, 128), (31, 257, 640), (33, 4099, 256), (48, 100, 4000), (64, 50, 200), (64, 5120, 2560),
          (65, 130, 1000), (96, 999, 512), (120, 1024, 2560), (128, 256, 256), (129, 257, 384), (200, 300, 513),
          (257, 512, 384), (300, 40, 2049), (513, 1537, 192), (700, 5003, 1001), (1000, 16, 64), (1024, 2304, 640)]


@pytest.mark.parametrize("shape", SHAPES, ids=str)
@pytest.mark.parametrize("dtype", TYPES)
def test_linear(device, shape, dtype):
    M, N, K = shape
    x = rows(M, K, dtype, seed=M + N + K)
    w_codes, w_scale = weight(N, K, seed=N * K)
    w = pack_weight_i8(w_codes.to(device), w_scale.to(device))
    codes, scale = quantised(x)
    want, _ = product(codes, scale, w_codes, w_scale)
    got_codes, got_scale = quantize_rows_i8(x.to(device))
    assert torch.equal(got_codes.cpu().long(), codes)
    assert ((got_scale.cpu().double() - scale).abs() <= 2.0 ** -24 * scale).all()
    out = linear_i8(x.to(device), w)
    assert out.dtype is dtype and out.shape == (M, N)
    check(out, want)
    # the halves give the same bits
    assert torch.equal(matmul_i8(got_codes, got_scale, w, out_dtype=dtype), out)


@pytest.mark.parametrize("M,N,K", [(1, 2, 1), (1, 18432, 256), (3, 34, 70), (16, 512, 2560), (16, 98, 513), (40, 1026, 640),
                                   (64, 2048, 512), (100, 1000, 640), (120, 18432, 320), (257, 514, 1000),
                                   (600, 3074, 256)])
@pytest.mark.parametrize("out_dtype", [torch.bfloat16, torch.float16, torch.float32])
def test_gated(device, M, N, K, out_dtype):
    x = rows(M, K, torch.bfloat16, seed=M * N + K)
    w_codes, w_scale = weight(N, K, seed=N + K)
    w = pack_weight_i8(w_codes.to(device), w_scale.to(device), gated=True)
    codes, scale = quantised(x)
    want, gate = product(codes, scale.float(), w_codes, w_scale, gated=True)
    out = linear_i8(x.to(device), w, out_dtype=out_dtype)
    assert out.dtype is out_dtype and out.shape == (M, N // 2)
    check(out, want, gate)


@pytest.mark.parametrize("M", [1, 2, 5, 16, 17, 64, 65, 130, 300])
@pytest.mark.parametrize("out_dtype", [torch.bfloat16, torch.float16, torch.float32])
def test_output_types_and_largest_sums(device, M, out_dtype):
    """All codes 127: the sum of the largest K stays in 32 bits, fp32's 24 bits do not hold it."""
    N, K = 20, 131072
    c = torch.full((M, K), 127, dtype=torch.int8)
    c[:, ::7] = -127
    w = torch.full((N, K), 127, dtype=torch.int8)
    w[1] = -127
    w[2] = c[0]
    w_scale = torch.linspace(1, 2, N) / K / 127
    scale = torch.linspace(1, 2, M) / 127
    got = matmul_i8(c.to(device), scale.to(device), pack_weight_i8(w.to(device), w_scale.to(device)), out_dtype=out_dtype)
    want, _ = product(c, scale, w, w_scale)
    check(got, want)
    assert abs(float(want[0, 2]) / (127 * 127 * K * float(scale[0]) * float(w_scale[2])) - 1) < 1e-12


def test_codes_at_ties(device):
    """Every pair of mantissas, ties among them: codes as real arithmetic gives them."""
    for dtype, bits in ((torch.bfloat16, 7), (torch.float16, 10)):
        m = torch.arange(2 ** bits, 2 ** (bits + 1)).double()
        a = m[:: max(1, 2 ** bits // 128)]  # the row's largest
        for s in range(0, 9):
            x = torch.cat((a[:, None], -(m * 2.0 ** -s).minimum(a[:, None])), 1).to(dtype)
            assert torch.equal(quantize_rows_i8(x.to(device))[0].cpu().long(), quantised(x)[0])


@pytest.mark.parametrize("dtype", TYPES)
def test_rows_of_extremes(device, dtype):
    """Zeros, the least and the largest values, NaN and infinities."""
    K = 100
    big, small = torch.finfo(dtype).max, torch.finfo(dtype).smallest_normal * torch.finfo(dtype).eps
    x = torch.zeros(7, K, dtype=dtype)
    x[1, 3], x[1, 4] = big, -big
    x[2, 5], x[2, 6] = small, -small
    x[3, 7] = torch.nan
    x[4, 99] = torch.inf
    x[5, 0] = -torch.inf
    x[6] = 1
    codes, scale = quantize_rows_i8(x.to(device))
    codes, scale = codes.cpu().long(), scale.cpu()
    live = [0, 1, 2, 6]
    want, want_s = quantised(x[live])
    assert torch.equal(codes[live], want)
    assert ((scale[live].double() - want_s).abs() <= 2.0 ** -24 * want_s).all()
    assert (codes[3:6] == 0).all() and torch.isnan(scale[3:6]).all()
    w = pack_weight_i8(*(t.to(device) for t in weight(33, K, 1)))
    out = linear_i8(x.to(device), w).cpu()
    assert torch.isnan(out[3:6]).all() and (out[0] == 0).all()
    if dtype is torch.bfloat16:  # (fp16 outputs of the largest inputs overflow)
        assert torch.isfinite(out[live]).all()
    # a row's NaN stays the row's, also where a launch takes many rows
    many = torch.ones(200, K, dtype=dtype, device=device)
    many[77, 5] = torch.nan
    out = linear_i8(many, w)
    assert torch.isnan(out[77]).all() and torch.equal(out[:77], out[:1].expand(77, -1))
    assert torch.equal(out[78:], out[:1].expand(122, -1))


@pytest.mark.parametrize("M", [1, 3, 16, 70, 300])
@pytest.mark.parametrize("N,gated", [(90, False), (83, False), (90, True)])
def test_strides(device, M, N, gated):
    """Inputs and outputs inside wider tensors, rows that begin at any element."""
    K = 328
    x = rows(M, K, torch.bfloat16, seed=5).to(device)
    w = pack_weight_i8(*(t.to(device) for t in weight(N, K, 2)), gated=gated)
    want = linear_i8(x, w)
    cols = w.cols
    for first in (0, 1, 5):
        wide = torch.full((M, K + 11), 3.0, dtype=torch.bfloat16, device=device)
        wide[:, first:first + K] = x
        for dt in (torch.bfloat16, torch.float32):
            out = torch.full((M, cols + 9), 7.0, dtype=dt, device=device)
            view = out[:, first:first + cols]
            assert linear_i8(wide[:, first:first + K], w, out=view) is view
            assert torch.equal(view.bfloat16(), want)
            assert (out[:, :first] == 7).all() and (out[:, first + cols:] == 7).all()
    codes, scale = quantize_rows_i8(x)
    assert torch.equal(matmul_i8(codes.t().contiguous().t(), scale, w), want)
    wide = torch.zeros((M, K + 24), dtype=torch.int8, device=device)
    for first in (0, 1, 16):
        wide.fill_(99)
        wide[:, first:first + K] = codes
        assert torch.equal(matmul_i8(wide[:, first:first + K], scale, w), want)
    alone = torch.empty(M * K, dtype=torch.int8, device=device).view(M, K)  # rows of 328 bytes, the last at the end
    alone.copy_(codes)
    assert torch.equal(matmul_i8(alone, scale, w), want)
    assert torch.equal(linear_i8(x.t().contiguous().t(), w), want)
    assert torch.equal(linear_i8(x[:1].expand(M, -1), w), want[:1].expand(M, -1))


def test_shapes_of_more_axes(device):
    x = rows(24, 64, torch.bfloat16, seed=9).to(device).view(2, 3, 4, 64)
    w = quantize_weight_i8(rows(40, 64, torch.bfloat16, seed=8).to(device))
    want = linear_i8(x.view(24, 64), w)
    assert torch.equal(linear_i8(x, w), want.view(2, 3, 4, 40))
    assert torch.equal(linear_i8(x[0, 0, 0], w), want[0])
    assert torch.equal(linear_i8(x.transpose(0, 2), w), want.view(2, 3, 4, 40).transpose(0, 2))
    assert linear_i8(x[:, :0], w).shape == (2, 0, 4, 40)
    c, s = quantize_rows_i8(x)
    assert c.shape == x.shape and s.shape == (2, 3, 4)
    assert torch.equal(matmul_i8(c, s, w), want.view(2, 3, 4, 40))


@pytest.mark.parametrize("dtype", TYPES)
def test_quantised_weights(device, dtype):
    """A weight's channels are rows: the product is near the unquantised one by 8 bits.

    Codes of x and w are each off by at most half a step of their row's largest over 127:
    random signs, K = 512 products: the error's norm is about 2^0.5 (a / 127 / 12^0.5) /
    rms of normal rows with a of 3.5 to 4 deviations, 1.2e-2; three times that bounds it."""
    x, w = rows(50, 512, dtype, 3)[:, :512], torch.randn(300, 512, generator=torch.Generator().manual_seed(4)).to(dtype)
    x = torch.randn(50, 512, generator=torch.Generator().manual_seed(6)).to(dtype)
    packed = quantize_weight_i8(w.to(device))
    assert isinstance(packed, Int8Weight) and (packed.N, packed.K, packed.cols) == (300, 512, 300)
    out = linear_i8(x.to(device), packed, out_dtype=torch.float32).cpu().double()
    want = x.double() @ w.double().T
    assert (out - want).norm() / want.norm() < 3 * 1.2e-2
    wc, ws = quantised(w)
    exact, _ = product(*quantised(x), wc, ws.float())
    assert ((out - exact).abs() <= 5 * 2.0 ** -24 * exact.abs() + 1e-30).all()


@pytest.mark.parametrize("M", [1, 7, 16, 48, 128, 400])
def test_captured_and_repeated(device, M):
    """Replays on other inputs give the eager bits; so does every call again."""
    K, N = 1280, 2000
    x = rows(M, K, torch.bfloat16, 1).to(device)
    w = pack_weight_i8(*(t.to(device) for t in weight(N, K, 2)), gated=True)
    linear_i8(x, w)
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=stream):
        out = linear_i8(x, w)
    for k in range(4):
        x.copy_(rows(M, K, torch.bfloat16, 10 + k))
        graph.replay()
        assert torch.equal(out, linear_i8(x, w)) and torch.equal(out, linear_i8(x, w))
        torch.cuda.synchronize()


@pytest.mark.parametrize("M,H", [(1, 16), (3, 256), (16, 2560), (5, 8192), (2, 20480), (600, 512), (513, 2576)])
@pytest.mark.parametrize("add,capture", [(True, True), (False, False)])
def test_add_rmsnorm(device, M, H, add, capture):
    """h_out exactly; the codes and scales are those of a bf16 rounding of the norm, whose fp32
    is off by at most 2^-19 of itself (sums of 20 + 10 + 16 terms at 2^-24 each, halved by the
    root, and four steps more).  So a value within 2^-19 of a border, about one of 2^10, may
    round the other way, by a whole step of 2^-7 of itself: its code moves by 127 * 2^-7 < 1,
    and where the row's largest does, which the scale shows, by as much again."""
    from dflash_mlx import _lib

    g = torch.Generator().manual_seed(M + H)
    h, r = (torch.randn(M, H, generator=g).bfloat16() for _ in range(2))
    w = (1 + 0.1 * torch.randn(H, generator=g)).bfloat16()
    hd, rd, wd = (t.to(device) for t in (h, r, w))
    out, cap = torch.empty_like(hd), torch.full((M, 2 * H), 7.0, dtype=torch.bfloat16, device=device)
    codes = torch.full((M, H + 16), 99, dtype=torch.int8, device=device)
    scale = torch.empty(M, device=device)
    _lib.call("dflash_add_rmsnorm_i8", hd.data_ptr(), rd.data_ptr() if add else None, wd.data_ptr(), out.data_ptr(),
              cap.data_ptr() if capture else None, 2 * H, codes.data_ptr(), H + 16, scale.data_ptr(), M, H, 1e-6,
              _lib.stream_handle(device))
    want_h = (h.float() + r.float()).bfloat16() if add else h
    assert torch.equal(out.cpu(), want_h)
    assert (codes[:, H:] == 99).all()
    if capture:
        assert torch.equal(cap[:, :H].cpu(), want_h) and (cap[:, H:] == 7).all()
    d = want_h.double()
    x = (d / (d.square().mean(1, keepdim=True) + 1e-6).sqrt() * w.double()).bfloat16()
    want, want_s = quantised(x)
    moved = (codes[:, :H].cpu().long() - want).abs()
    scale = scale.cpu().double()
    assert moved.max() <= 2
    assert ((scale - want_s).abs() <= 2.0 ** -7 * (1 + 2.0 ** -10) * want_s).all()
    same = (scale - want_s).abs() <= 2.0 ** -22 * want_s
    assert not same.any() or moved[same].max() <= 1
    assert same.sum() >= M // 2 and (moved[same] > 0).sum() <= 1 + 0.004 * moved[same].numel()


@pytest.mark.parametrize("M", [1, 2, 3])
@pytest.mark.parametrize("N,K,gated", [(40, 1, False), (2, 17, True), (5120, 2560, False), (5120, 2559, True), (4096, 9984, False),
                                       (4100, 12300, False), (33024, 200, True), (48, 40960, False), (32784, 264, False),
                                       (48, 40961, True)])
@pytest.mark.parametrize("dtype", TYPES)
def test_few_rows_quantised_on_the_way(device, M, N, K, gated, dtype):
    """As by its two halves, to the bit: one row in LDS where it holds the codes, else by a launch before."""
    g = torch.Generator().manual_seed(M * K + N)
    x = torch.zeros(M, K + 3, dtype=dtype)
    x[:, :K] = torch.randn(M, K, generator=g) * torch.logspace(-3, 3, M)[:, None]
    x[:, K:] = torch.nan
    if M > 2:
        x[1, :K] = 0
        x[2, K // 2] = torch.inf
    x = x.to(device)[:, :K]
    w = pack_weight_i8(torch.randint(-127, 128, (N, K), generator=g, dtype=torch.int8).to(device),
                       torch.rand(N, generator=g).to(device) / K, gated=gated)
    for out_dtype in (torch.float32, dtype):
        got = linear_i8(x, w, out_dtype=out_dtype)
        want = matmul_i8(*quantize_rows_i8(x), w, out_dtype=out_dtype)
        assert torch.equal(got.isnan(), want.isnan()) and torch.equal(got.nan_to_num(), want.nan_to_num())
        if M > 2:
            assert got[2].isnan().all()


def test_outputs_over_their_inputs_are_refused(device):
    w = pack_weight_i8(torch.ones(32, 32, dtype=torch.int8, device=device), torch.ones(32, device=device))
    buf = torch.zeros(3, 32, dtype=torch.bfloat16, device=device)
    with pytest.raises(ValueError, match="apart"):
        linear_i8(buf, w, out=buf)
    with pytest.raises(ValueError, match="apart"):
        linear_i8(buf[:2], w, out=buf[1:])
    linear_i8(buf[:1], w, out=buf[1:2])
    codes, scale = quantize_rows_i8(buf)
    with pytest.raises(ValueError, match="apart"):
        matmul_i8(codes[:1], scale[:1], w, out=codes.view(torch.bfloat16).view(-1)[:32].view(1, 32))


def test_rows_do_not_depend_on_their_number(device):
    """A row's output is the same bits whatever rows are beside it."""
    K, N = 640, 1100
    x = rows(600, K, torch.bfloat16, 1).to(device)
    w = pack_weight_i8(*(t.to(device) for t in weight(N, K, 2)))
    want = linear_i8(x, w)
    for M in (1, 2, 4, 5, 8, 16, 17, 32, 33, 64, 65, 128, 129, 256, 300, 512):
        assert torch.equal(linear_i8(x[:M], w), want[:M])


def test_far_offsets(device):
    """Outputs and codes behind 2^31 elements."""
    M, N, K = 70000, 33000, 64
    x = rows(M, K, torch.bfloat16, 1).to(device)
    w = pack_weight_i8(*(t.to(device) for t in weight(N, K, 2)))
    out = linear_i8(x, w)
    assert out.numel() > 2 ** 31
    assert torch.equal(out[-300:], linear_i8(x[-300:], w)) and torch.equal(out[65000:65064], linear_i8(x[65000:65064], w))


def test_refusals(device):
    x = torch.zeros(4, 64, dtype=torch.bfloat16, device=device)
    w = quantize_weight_i8(x)
    c, s = quantize_rows_i8(x)
    for bad in (lambda: linear_i8(x[:, :63], w), lambda: matmul_i8(c[:, :63], s, w), lambda: matmul_i8(c, s[:3], w),
                lambda: pack_weight_i8(c, s[:3]), lambda: pack_weight_i8(c[:3], s[:3], gated=True),
                lambda: pack_weight_i8(c[0], s), lambda: linear_i8(x, w, out=torch.zeros(4, 5, device=device)),
                lambda: linear_i8(x, w, out=torch.zeros(1, 4, device=device).expand(4, 4)),
                lambda: linear_i8(x, w, out=torch.zeros(4, 4, device=device).t()),
                lambda: quantize_rows_i8(torch.zeros(1, 131073, dtype=torch.bfloat16, device=device)),
                lambda: quantize_rows_i8(x[:, :0]), lambda: Int8Weight(w.codes[:-1], w.scales, 4, 64, False),
                lambda: Int8Weight(w.codes, w.scales[:-1], 4, 64, False), lambda: Int8Weight(w.codes, w.scales, 3, 64, True),
                lambda: linear_i8(x[0, 0], w)):
        with pytest.raises(ValueError):
            bad()
    for bad in (lambda: linear_i8(x.float(), w), lambda: linear_i8(x, x), lambda: matmul_i8(x, s, w),
                lambda: linear_i8(x, w, out_dtype=torch.float64), lambda: quantize_rows_i8(c),
                lambda: linear_i8(x, w, out=torch.zeros(4, 4, dtype=torch.int32, device=device))):
        with pytest.raises(TypeError):
            bad()
