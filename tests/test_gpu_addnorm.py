"""add_rmsnorm through the C-ABI against the reference's rmsnorm (src/kernels/rmsnorm.rs:10-21).

Two references in numpy: the definition's own f32 steps, which 8-bit codes and f32 outputs follow bit for
bit, and the formula in 64 bits. Tolerance of the second, in units u = 2^-24 (half a step of f32): the
squares and their mean carry 2 u, the addition of eps 1 u, halved by the root: 1.5 u; the root, the division
and two products 1 u each: 5.5 u, taken as 6 u; a bf16 output adds half a step of bf16, 2^-8.
"""
import numpy as np
import pytest
import torch

import bebelm_b200 as bb
import oracle

pytestmark = pytest.mark.gpu
U = 2.0 ** -24
EPS = np.float32(1e-5)


def steps(h, gain, eps=EPS):
    """t of float32 rows h, each step rounded to f32 as the definition says."""
    h = np.asarray(h, np.float32)
    ss = (h * h).astype(np.float64).sum(-1, keepdims=True)
    mean = (ss / h.shape[-1]).astype(np.float32)
    r = np.float32(1.0) / np.sqrt(mean + np.float32(eps))
    return (h * r) * gain


def codes_of(t, group):
    rows, n = t.shape
    g = t.reshape(rows, -1, group or n)
    a = np.abs(g).max(-1, keepdims=True)
    inv = np.divide(np.float32(127), a, out=np.zeros_like(a), where=a > 0)
    z = g * inv
    w = np.trunc(z)
    q = np.clip(w + np.sign(z) * (np.abs(z - w) >= 0.5), -127, 127)
    return q.reshape(rows, n).astype(np.int8), (a / np.float32(127)).reshape(rows, -1)


def inputs(rows, n, dtype, seed, residual=True):
    g = torch.Generator(device="cuda").manual_seed(seed)
    x = torch.randn(rows, n, device="cuda", generator=g).to(dtype)
    r = (3 * torch.randn(rows, n, device="cuda", generator=g)).to(dtype) if residual else None
    return x, r, 1 + 0.1 * torch.randn(n, device="cuda", generator=g)


def check(x, r, gain, y, h):
    want_h = x if r is None else (x.float() + r.float()).to(x.dtype)
    assert torch.equal(h, want_h)
    hf = want_h.float().cpu().numpy()
    t = steps(hf, gain.cpu().numpy())
    h64 = hf.astype(np.float64)
    exact = h64 / np.sqrt((h64 ** 2).mean(-1, keepdims=True) + float(EPS)) * gain.double().cpu().numpy()
    got = y.float().cpu().numpy()
    if y.dtype == torch.float32:
        np.testing.assert_array_equal(got, t)
        assert (np.abs(got - exact) <= 6 * U * np.abs(exact)).all()
    else:
        np.testing.assert_array_equal(got, torch.from_numpy(t).to(torch.bfloat16).float().numpy())
        assert (np.abs(got - exact) <= (6 * U + 2.0 ** -8) * np.abs(exact)).all()


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("rows,n", [(1, 1), (1, 2048), (3, 7), (5, 64), (2, 255), (7, 256), (4, 257), (3, 1000), (6, 1024),
                                    (2, 1032), (33, 2048), (3, 2049), (2, 8192), (1, 8200), (2, 16392), (1, 32768), (3, 32761)])
def test_float_outputs(rows, n, dtype):
    for residual in (True, False):
        x, r, gain = inputs(rows, n, dtype, rows * 40000 + n, residual)
        for od in (bb.F32, bb.BF16):
            y, h = bb.add_rmsnorm(x, gain, r, out_dtype=od)
            assert y.dtype == (torch.float32 if od == bb.F32 else torch.bfloat16)
            check(x, r, gain, y, h)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("rows,n", [(700, 2048), (610, 2049), (1200, 1032), (80, 16392), (170, 8192), (1300, 1024)])
def test_rows_that_fill_the_device(rows, n, dtype):
    x, r, gain = inputs(rows, n, dtype, rows + n)
    for od in (bb.F32, bb.BF16):
        check(x, r, gain, *bb.add_rmsnorm(x, gain, r, out_dtype=od))
    for group in (0, 64):
        if group and n % group:
            continue
        q, sc, h = bb.add_rmsnorm(x, gain, r, out_dtype=bb.INT8, group=group)
        want, want_sc = codes_of(steps(h.float().cpu().numpy(), gain.cpu().numpy()), group)
        np.testing.assert_array_equal(q.cpu().numpy(), want)
        np.testing.assert_array_equal(sc.cpu().numpy().reshape(want_sc.shape), want_sc)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("group", [0, 32, 64, 128, 256])
@pytest.mark.parametrize("rows,n", [(1, 256), (1, 2048), (9, 512), (5, 1280), (3, 8192), (2, 8448), (1, 32768), (130, 768)])
def test_codes_are_the_definitions(rows, n, group, dtype):
    x, r, gain = inputs(rows, n, dtype, rows * 999 + n + group)
    q, sc, h = bb.add_rmsnorm(x, gain, r, out_dtype=bb.INT8, group=group)
    hf = (x.float() + r.float()).to(dtype)
    assert torch.equal(h, hf)
    wq, ws = codes_of(steps(hf.float().cpu().numpy(), gain.cpu().numpy()), group)
    np.testing.assert_array_equal(q.cpu().numpy(), wq)
    np.testing.assert_array_equal(sc.cpu().numpy(), ws)


@pytest.mark.parametrize("rows,n,group", [(3, 96, 32), (2, 2080, 32), (3, 224, 0), (4, 41, 0), (2, 1033, 0), (2, 4160, 64)])
def test_codes_of_odd_sizes(rows, n, group):
    x, r, gain = inputs(rows, n, torch.float32, n)
    q, sc, _ = bb.add_rmsnorm(x, gain, r, out_dtype=bb.INT8, group=group)
    wq, ws = codes_of(steps((x + r).cpu().numpy(), gain.cpu().numpy()), group)
    np.testing.assert_array_equal(q.cpu().numpy(), wq)
    np.testing.assert_array_equal(sc.cpu().numpy(), ws)


def test_equals_the_oracles_rmsnorm():
    """Without a residual the f32 output is the reference's rmsnorm, whose sequential f64 sum has the
    same value (its partial sums are exact in f64 for these inputs)."""
    x, gain = oracle.normal(5, (4, 2048)), (1 + 0.1 * oracle.normal(6, 2048)).astype(np.float32)
    y, h = bb.add_rmsnorm(torch.from_numpy(x).cuda(), torch.from_numpy(gain).cuda())
    for i in range(4):
        np.testing.assert_array_equal(y[i].cpu().numpy(), oracle.rmsnorm(x[i], gain, 1e-5))
    yh, hh = bb.add_rmsnorm(x, gain)
    np.testing.assert_array_equal(yh, y.cpu().numpy())
    assert hh is x or np.array_equal(hh, x)


def test_host_buffers():
    x, r, gain = inputs(19, 2048, torch.float32, 3)
    dev = bb.add_rmsnorm(x, gain, r, out_dtype=bb.INT8, group=256)
    host = bb.add_rmsnorm(x.cpu().numpy(), gain.cpu().numpy(), r.cpu().numpy(), out_dtype=bb.INT8, group=256)
    for a, b in zip(dev, host):
        np.testing.assert_array_equal(a.cpu().numpy(), b)
    y, h = bb.add_rmsnorm(x.cpu().numpy(), gain.cpu().numpy(), r.cpu().numpy())
    check(x, r, gain, torch.from_numpy(y), torch.from_numpy(h).cuda())


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_strided_and_unaligned_rows(dtype):
    """Rows inside wider buffers, at odd offsets, with nothing beside them touched."""
    g = torch.Generator(device="cuda").manual_seed(4)
    for off, n, width in ((0, 2048, 2304), (3, 2048, 2061), (1, 513, 517), (8, 256, 264)):
        buf = torch.randn(6, width, device="cuda", generator=g).to(dtype)
        rbuf = torch.randn(6, width + 5, device="cuda", generator=g).to(dtype)
        hbuf = torch.full((6, width + 2), 7.0, device="cuda", dtype=dtype)
        gain = (1 + 0.1 * torch.randn(n + 1, device="cuda", generator=g))[1:]  # 4-byte aligned only
        x, r, h = buf[:, off:off + n], rbuf[:, 2:2 + n], hbuf[:, 1:1 + n]
        y, hh = bb.add_rmsnorm(x, gain.contiguous(), r, sum_out=h)
        assert hh.data_ptr() == h.data_ptr()
        check(x.contiguous(), r.contiguous(), gain, y, h.contiguous())
        assert (hbuf[:, 0] == 7).all() and (hbuf[:, 1 + n:] == 7).all()
        y2, _ = bb.add_rmsnorm(x, gain, r)  # an unaligned gain
        assert torch.equal(y, y2)


def test_in_place_sum():
    for dtype in (torch.float32, torch.bfloat16):
        x, r, gain = inputs(300, 2048, dtype, 8)
        want, wh = bb.add_rmsnorm(x, gain, r)
        a = x.clone()
        y, h = bb.add_rmsnorm(a, gain, r, sum_out=a)
        assert h is a and torch.equal(a, wh) and torch.equal(y, want)
        b = r.clone()
        y, h = bb.add_rmsnorm(x, gain, b, sum_out=b, out=x)  # y over x, the sum over the residual
        assert torch.equal(b, wh) and torch.equal(x, want)


def test_zero_rows_and_extremes():
    gain = torch.ones(64, device="cuda")
    x = torch.zeros(3, 64, device="cuda")
    x[1] = 1e-30
    x[2, 5] = float("nan")
    q, sc, _ = bb.add_rmsnorm(x, gain, out_dtype=bb.INT8)
    assert (q[0] == 0).all() and sc[0] == 0
    assert (q[1] == 127).all()  # equal values: each is the maximum
    y, _ = bb.add_rmsnorm(x, gain)
    assert (y[0] == 0).all() and torch.isfinite(y[1]).all() and torch.isnan(y[2]).all()
    y, h = bb.add_rmsnorm(torch.empty(0, 64, device="cuda"), gain)
    assert y.shape == (0, 64)


def test_on_another_stream_and_in_a_graph():
    x, r, gain = inputs(5, 2048, torch.float32, 10)
    want, wh = bb.add_rmsnorm(x, gain, r)
    s = torch.cuda.Stream()
    y, h = torch.empty_like(x), torch.empty_like(x)
    s.wait_stream(torch.cuda.current_stream())
    bb.add_rmsnorm(x, gain, r, out=y, sum_out=h, stream=s)
    s.synchronize()
    assert torch.equal(y, want) and torch.equal(h, wh)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        bb.add_rmsnorm(x, gain, r, out=y, sum_out=h)
    x.mul_(2)
    graph.replay()
    want, wh = bb.add_rmsnorm(x, gain, r)
    assert torch.equal(y, want) and torch.equal(h, wh)


def float_row_and_codes(x, gain, group, r=None):
    """The float output and what the 8-bit one stands for."""
    y, _ = bb.add_rmsnorm(x, gain, r, out_dtype=bb.F32)
    q, sc, _ = bb.add_rmsnorm(x, gain, r, out_dtype=bb.INT8, group=group)
    rows, n = x.shape
    sc = sc.view(rows, -1)
    return y, q, sc, (q.view(rows, sc.shape[1], -1).float() * sc[..., None]).view(rows, n)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("n,group", [(64, 0), (256, 32), (2048, 256), (2048, 0), (41, 0), (16384, 128)])
def test_8_bit_rows_that_are_not_finite(n, group, dtype):
    """A group of 8-bit outputs with a NaN or an infinity among its values reads back as NaN: its scale is NaN, its codes 0.
    Groups and rows beside it are as they are without it."""
    x, r, gain = inputs(6, n, dtype, n)
    clean = bb.add_rmsnorm(x, gain, r, out_dtype=bb.INT8, group=group)
    x[1, n // 2] = float("nan")
    x[2, n - 1] = float("inf")
    x[4, 0], x[4, n // 3] = float("-inf"), float("inf")
    y, q, sc, back = float_row_and_codes(x, gain, group, r)
    assert torch.isnan(y[1]).all() and torch.isnan(sc[1]).all()  # one NaN makes the row's sum one
    for row in (1, 2, 4):
        broken = (~torch.isfinite(y[row])).view(-1, group or n).any(-1)
        assert broken.any() and torch.equal(torch.isnan(sc[row]), broken)
        assert torch.equal(torch.isnan(back[row]), broken.repeat_interleave(group or n))
        assert (q[row].view(-1, group or n)[broken] == 0).all()
    for row in (0, 3, 5):
        assert torch.equal(q[row], clean[0][row]) and torch.equal(sc[row], clean[1][row].view(-1))


@pytest.mark.parametrize("bad", [float("nan"), float("inf"), float("-inf")])
@pytest.mark.parametrize("group", [0, 64])
def test_8_bit_rows_under_a_gain_that_is_not_finite(group, bad):
    x, r, gain = inputs(3, 512, torch.float32, 3)
    want = bb.add_rmsnorm(x, gain, r, out_dtype=bb.INT8, group=group)
    gain[100] = bad
    _, q, sc, back = float_row_and_codes(x, gain, group, r)
    g = group or 512
    hit = torch.arange(512 // g, device="cuda") == 100 // g
    assert torch.equal(torch.isnan(sc), hit.expand(3, -1)) and torch.isnan(back[:, 100]).all()
    keep = ~hit.repeat_interleave(g)
    assert torch.equal(q[:, keep], want[0][:, keep]) and (q[:, ~keep] == 0).all()


@pytest.mark.parametrize("group", [0, 32])
@pytest.mark.parametrize("unit", [-149, -140, -126, -122, -120, -100])
def test_8_bit_rows_of_tiny_values(unit, group):
    """Below 3.8e-37 the factor 127 / a is above f32's range. The codes are those of the same values 2^64 times as large, where
    it is in range, and zeros stay zeros. h = 1 and 0 with eps = 0 makes t whole multiples of the gain's 2^unit."""
    rows, n = 3, 256
    x = torch.ones(rows, n, device="cuda")
    x[1] = -1
    g = torch.Generator(device="cuda").manual_seed(unit & 0xff)
    gain = torch.randint(-9, 10, (n,), device="cuda", generator=g).double()
    gain[3::5] = 0
    small = (gain * 2.0 ** unit).float()
    q, sc, _ = bb.add_rmsnorm(x, small, eps=0.0, out_dtype=bb.INT8, group=group)
    want, want_sc, _ = bb.add_rmsnorm(x, gain.float(), eps=0.0, out_dtype=bb.INT8, group=group)
    assert torch.equal(q, want) and (q[:, 3::5] == 0).all() and want.abs().max() == 127
    exact = gain.view(-1, group or n).abs().amax(-1) * 2.0 ** unit / 127
    # a / 127 rounded to f32: half a step, 2^-24 of it or half of the smallest denormal
    assert ((sc.double() - exact).abs() <= (exact * 2.0 ** -24).clamp(min=2.0 ** -150)).all()
