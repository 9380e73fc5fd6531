"""Products with 4-bit weights and group scales against the formula in 64 bits.

Two kinds of inputs. Whole-numbered activations with scales that are powers of two: every product,
group sum and total is a whole multiple of one power of two below 2^24 of them, so any order of f32 additions
gives the exact result and the outputs must be equal. Normal activations: the products c - z times a
bf16 term are exact; the tensor cores add 16 of them and the running sum per step, each addition within
one f32 step (2^-23) of the sum of absolute terms A_g of the group; with s steps a group (group / 16 per
bf16 term of an activation, 3 terms for f32) and 17 additions a step that is 17 s 2^-23 A_g. The groups
are then scaled and added in f32: one rounding each for the scale product, the activations' scale and the
addition, (groups + 2) 2^-24 A. A bf16 output adds half a step, 2^-8 of the value.

Up to 8 tokens (16 through small layers) the activations are whole numbers instead, kept to 2^-23 of the largest M of 128: 2^-23 M Σ|w|, and
their sums are exact. For these normal activations M < 5.5 against a mean of 0.8, so that is about 7 2^-23 A,
within the 17 s above. More f32 tokens are two f16 terms, within 2^-24 of each activation: 2^-24 A more
than the bf16 terms' 0, again within it.
"""
import numpy as np
import pytest
import torch

import bebelm_b200 as bb

pytestmark = pytest.mark.gpu

KINDS = {"f32": torch.float32, "bf16": torch.bfloat16, "int8": torch.int8}


def weights(n_out, n_in, group, seed, zeros=True, scales=torch.float16, exact=False):
    g = torch.Generator(device="cuda").manual_seed(seed)
    codes = torch.randint(0, 256, (n_out, n_in // 2), device="cuda", generator=g, dtype=torch.uint8)
    ng = n_in // group
    if exact:
        sc = torch.exp2(-torch.randint(0, 3, (n_out, ng), device="cuda", generator=g).float()).to(scales)
    else:
        sc = (0.02 * torch.randn(n_out, ng, device="cuda", generator=g)).to(scales)
    z = torch.randint(0, 16, (n_out, ng), device="cuda", generator=g, dtype=torch.uint8) if zeros else None
    return codes, sc, z


def activations(t, n_in, kind, x_group, seed, exact=False):
    g = torch.Generator(device="cuda").manual_seed(seed + 77)
    if kind == "int8":
        hi = 4 if exact else 128
        x = torch.randint(-hi + 1, hi, (t, n_in), device="cuda", generator=g).to(torch.int8)
        ng = n_in // x_group if x_group else 1
        if exact:
            xs = torch.exp2(-torch.randint(0, 3, (t, ng), device="cuda", generator=g).float())
        else:
            xs = 0.01 + torch.rand(t, ng, device="cuda", generator=g)
        return x, xs
    if exact:
        return torch.randint(-3, 4, (t, n_in), device="cuda", generator=g).to(KINDS[kind]), None
    return torch.randn(t, n_in, device="cuda", generator=g).to(KINDS[kind]), None


def dense(codes, sc, z, group):
    n_out, half = codes.shape
    w = torch.empty(n_out, 2 * half, dtype=torch.float64, device=codes.device)
    w[:, 0::2], w[:, 1::2] = (codes & 15).double(), (codes >> 4).double()
    w -= 8 if z is None else z.double().repeat_interleave(group, 1)
    return w * sc.double().repeat_interleave(group, 1)


def floats(x, xs):
    x = x.double()
    return x if xs is None else x * xs.double().repeat_interleave(x.shape[1] // xs.shape[1], 1)


def check(case, exact):
    t, n_in, n_out, group, kind, x_group, zeros, sdt, ydt = case
    codes, sc, z = weights(n_out, n_in, group, hash(case[:4]) & 0xffff, zeros, sdt, exact)
    x, xs = activations(t, n_in, kind, x_group, n_in + t, exact)
    w = bb.W4Weights(codes, sc, z, group=group)
    y = w.matmul(x, xs, out_dtype=ydt)
    assert y.shape == (t, n_out)
    assert torch.equal(y, w.matmul(x, xs, out_dtype=ydt))  # the same bits again
    wd, xd = dense(codes, sc, z, group), floats(x, xs)
    want = xd @ wd.t()
    if exact and ydt == bb.F32:
        assert torch.equal(y.double(), want)
    else:
        a = xd.abs() @ wd.abs().t()
        steps = max(1, group // 16) * (3 if kind == "f32" else 1)
        tol = (17 * steps * 2.0 ** -23 + (n_in / min(group, x_group or group) + 2) * 2.0 ** -24) * a
        if ydt == bb.BF16:
            tol = tol * (1 + 2.0 ** -8) + 2.0 ** -8 * want.abs()
        bad = (y.double() - want).abs() > tol
        assert not bad.any(), (int(bad.sum()), float(((y.double() - want).abs() / a.clamp(min=1e-30)).max()))
    w.close()


CASES = [
    # tokens, n_in, n_out, group, kind, x_group, zeros, scales, out
    (1, 32, 1, 32, "f32", 0, False, torch.float16, bb.F32),
    (1, 2048, 2048, 128, "f32", 0, True, torch.float16, bb.F32),
    (1, 2048, 512, 32, "bf16", 0, True, torch.bfloat16, bb.F32),
    (3, 96, 17, 32, "bf16", 0, True, torch.float16, bb.BF16),
    (2, 192, 130, 64, "int8", 0, True, torch.float16, bb.F32),
    (5, 2080, 515, 32, "f32", 0, True, torch.bfloat16, bb.F32),
    (7, 1024, 100, 64, "int8", 32, False, torch.float16, bb.F32),
    (8, 512, 333, 128, "int8", 256, True, torch.bfloat16, bb.F32),
    (9, 768, 48, 256, "int8", 64, True, torch.float16, bb.BF16),
    (16, 640, 1000, 640, "f32", 0, True, torch.float16, bb.F32),
    (17, 2048, 129, 128, "bf16", 0, False, torch.float16, bb.BF16),
    (31, 320, 64, 64, "f32", 0, True, torch.float16, bb.F32),
    (32, 8192, 40, 128, "bf16", 0, True, torch.float16, bb.F32),
    (33, 256, 200, 32, "f32", 0, True, torch.float16, bb.F32),
    (64, 2048, 300, 128, "int8", 128, True, torch.float16, bb.F32),
    (65, 416, 257, 32, "int8", 0, False, torch.bfloat16, bb.F32),
    (100, 1024, 128, 256, "bf16", 0, True, torch.float16, bb.BF16),
    (129, 160, 385, 32, "bf16", 0, True, torch.float16, bb.F32),
    (200, 2048, 2048, 64, "f32", 0, True, torch.bfloat16, bb.F32),
    (257, 512, 640, 128, "int8", 32, True, torch.float16, bb.BF16),
    (513, 1280, 1000, 128, "bf16", 0, True, torch.float16, bb.F32),
    # 9 to 16 tokens through layers above and below the size where the kernels change
    (9, 2048, 8192, 128, "f32", 0, True, torch.float16, bb.F32),
    (12, 2048, 8193, 128, "f32", 0, False, torch.float16, bb.F32),
    (16, 2080, 5003, 32, "bf16", 0, True, torch.float16, bb.BF16),
    (13, 8192, 8192, 64, "f32", 0, True, torch.bfloat16, bb.F32),
    # activations' groups of 64 over weights' groups of 32
    (6, 256, 70, 32, "int8", 64, True, torch.float16, bb.F32),
    (17, 256, 70, 32, "int8", 64, True, torch.float16, bb.F32),
    (90, 192, 257, 32, "int8", 64, False, torch.float16, bb.F32),
    # few tiles of many inputs: 8, 6, 4, 3 and 2 CTAs share a tile's
    (24, 4096, 128, 128, "f32", 0, True, torch.float16, bb.F32),
    (40, 1664, 700, 32, "int8", 64, True, torch.float16, bb.F32),
    (128, 2048, 2500, 64, "f32", 0, True, torch.float16, bb.BF16),
    (70, 512, 4300, 128, "bf16", 0, False, torch.float16, bb.F32),
    (256, 1056, 2048, 32, "bf16", 0, True, torch.bfloat16, bb.F32),
    (20, 384, 300, 128, "int8", 0, True, torch.float16, bb.F32),
]
IDS = ["-".join(str(v).replace("torch.", "") for v in c) for c in CASES]


@pytest.mark.parametrize("case", CASES, ids=IDS)
def test_exact_in_whole_numbers(case):
    check(case, True)


@pytest.mark.parametrize("case", CASES, ids=IDS)
def test_normal_activations(case):
    check(case, False)


def test_many_rows_stream():
    """A vocabulary-sized matrix: every persistent CTA takes several tiles."""
    check((5, 2048, 60001, 128, "int8", 256, False, torch.float16, bb.F32), False)
    check((1, 1024, 70000, 64, "bf16", 0, True, torch.float16, bb.F32), True)


def test_host_buffers_and_numpy_weights():
    codes, sc, z = weights(300, 512, 64, 5)
    x, _ = activations(6, 512, "f32", 0, 1)
    xi, xs = activations(6, 512, "int8", 128, 1)
    wd = bb.W4Weights(codes, sc, z, group=64)
    wh = bb.W4Weights(codes.cpu().numpy(), sc.cpu().numpy(), z.cpu().numpy(), group=64)
    wc = bb.W4Weights(codes.cpu(), sc.cpu(), z.cpu(), group=64)
    want = wd.matmul(x).cpu().numpy()
    for w in (wh, wc):
        np.testing.assert_array_equal(w.matmul(x).cpu().numpy(), want)
        np.testing.assert_array_equal(w.matmul(x.cpu().numpy()), want)
        np.testing.assert_array_equal(w.matmul(xi.cpu().numpy(), xs.cpu().numpy()), wd.matmul(xi, xs).cpu().numpy())
    np.testing.assert_array_equal(wh.matmul(x[0].cpu().numpy()), want[0])
    assert torch.equal(wd.matmul(x[2]), wd.matmul(x[2:3])[0])


@pytest.mark.parametrize("t", [1, 6, 40, 150])
@pytest.mark.parametrize("kind", ["f32", "bf16", "int8"])
def test_strided_and_unaligned_rows(kind, t):
    codes, sc, z = weights(260, 416, 32, 9)
    w = bb.W4Weights(codes, sc, z, group=32)
    big, xs = activations(t, 433, kind, 0, 3)
    for off in (0, 1, 5, 16):
        view = big[:, off:off + 416]
        assert torch.equal(w.matmul(view, xs), w.matmul(view.contiguous(), xs)), off
    wide, _ = activations(t, 480, kind, 0, 3)  # aligned rows with a gap
    assert torch.equal(w.matmul(wide[:, :416], xs), w.matmul(wide[:, :416].contiguous(), xs))


@pytest.mark.parametrize("t", [1, 7, 13, 40])
@pytest.mark.parametrize("unit", [-147, -130, -100, 90])
def test_the_smallest_and_large_activations(t, unit):
    """Whole multiples of 2^unit with scales 1 and 1/2, zero points: every sum is a whole multiple of 2^(unit - 1)
    below 2^24 of them, so outputs are exact down to f32's last denormal step, 2^-149."""
    codes, sc, z = weights(300, 256, 64, 9, exact=True)
    sc = sc.clamp(min=0.5)
    x, _ = activations(t, 256, "f32", 0, 4, exact=True)
    x = torch.ldexp(x, torch.tensor(unit, device="cuda")) if unit > -127 else torch.ldexp(torch.ldexp(x, torch.tensor(unit + 64, device="cuda")), torch.tensor(-64, device="cuda"))
    w = bb.W4Weights(codes, sc, z, group=64)
    assert torch.equal(w.matmul(x).double(), x.double() @ dense(codes, sc, z, 64).t())


@pytest.mark.parametrize("t", [3, 70])
def test_infinities_and_nan_stay_in_their_token(t):
    codes, sc, z = weights(64, 256, 64, 2)
    w = bb.W4Weights(codes, sc, z, group=64)
    for kind in ("f32", "bf16"):
        x, _ = activations(t, 256, kind, 0, 8)
        clean = w.matmul(x, out_dtype=bb.F32)
        x[1, 5] = float("inf")
        x[2, 7] = float("nan")
        y = w.matmul(x, out_dtype=bb.F32)
        assert not torch.isfinite(y[1]).any() and torch.isnan(y[2]).all()
        assert torch.equal(y[0], clean[0]) and torch.equal(y[3:], clean[3:])


def test_the_largest_sums():
    """A group's sum is formed in f32 before its scale: finite up to the documented limit, where the
    sum of |code - zero| |x| reaches the largest float. (The split of an activation does not overflow.)"""
    codes, sc, z = weights(64, 256, 64, 2)
    w = bb.W4Weights(codes, sc, z, group=64)
    for t in (1, 50):
        x = torch.zeros((t, 256), device="cuda")
        x[:, 0] = 2.2e37  # 15 times that is below 3.4e38
        want = x.double() @ dense(codes, sc, z, 64).t()
        y = w.matmul(x).double()
        assert ((y - want).abs() <= 2.0 ** -20 * want.abs()).all()


def test_no_tokens_and_output_neighbours():
    codes, sc, z = weights(100, 256, 128, 6)
    w = bb.W4Weights(codes, sc, z, group=128)
    assert w.matmul(torch.empty(0, 256, device="cuda")).shape == (0, 100)
    for t in (1, 9, 40, 129):
        buf = torch.full((t + 2, 100), 5.0, device="cuda")
        x, _ = activations(t, 256, "f32", 0, 1)
        w.matmul(x, out=buf[1:t + 1])
        assert (buf[0] == 5).all() and (buf[t + 1] == 5).all()
        assert torch.equal(buf[1:t + 1], w.matmul(x))


@pytest.mark.parametrize("t", [1, 8, 48, 200])
@pytest.mark.parametrize("kind", ["f32", "bf16", "int8"])
def test_two_streams_and_a_graph(kind, t):
    """Products of one handle on two streams at once, and replayed from a graph with new activations."""
    codes, sc, z = weights(512, 1024, 128, 3)
    w = bb.W4Weights(codes, sc, z, group=128)
    a, xs = activations(t, 1024, kind, 128 if kind == "int8" else 0, 1)
    b, _ = activations(t, 1024, kind, 128 if kind == "int8" else 0, 2)
    wa, wb = w.matmul(a, xs), w.matmul(b, xs)
    s1, s2 = torch.cuda.Stream(), torch.cuda.Stream()
    torch.cuda.synchronize()
    got = []
    for _ in range(10):
        got += [(w.matmul(a, xs, stream=s1), wa), (w.matmul(b, xs, stream=s2), wb)]
    torch.cuda.synchronize()
    assert all(torch.equal(p, q) for p, q in got)
    static, out = a.clone(), torch.empty_like(wa)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        w.matmul(static, xs, out=out)
    static.copy_(b)
    graph.replay()
    assert torch.equal(out, wb)


@pytest.mark.parametrize("t,n_in,n_out", [(40, 1024, 300), (24, 256, 200 * 128), (200, 2048, 2048)])
def test_a_wait_that_gives_up_is_reported(t, n_in, n_out):
    """A bounded wait of the many-token kernel runs out (forced: the first CTA waits, with a short limit, on a barrier nothing
    completes; no fault). Its tile stays unwritten, check() reports it once, the next product is right; a host-memory
    call reports it itself; every replay of a graph that was captured with it is reported."""
    L = bb.load_library()
    codes, sc, z = weights(n_out, n_in, 64, 3)
    w = bb.W4Weights(codes, sc, z, group=64)
    x, _ = activations(t, n_in, "f32", 0, 4)
    want = w.matmul(x)
    w.check()
    try:
        out = torch.full_like(want, 7)
        assert L.bebelm_debug_expire_next_wait(1) == bb.OK
        w.matmul(x, out=out)
        with pytest.raises(bb.BebelmError) as e:
            w.check()
        assert e.value.code == bb.ERR_TIMEOUT
        tile = 32 if t <= 32 else 64 if t <= 64 else 128  # tokens
        assert (out[:tile, :128] == 7).all()  # the first CTA's tile of 128 rows (its first)
        wrong = (out != want).view(-1).nonzero().numel()
        assert wrong <= t * n_out // 2
        w.check()  # once
        assert torch.equal(w.matmul(x), want)

        xh = x.cpu().numpy()
        assert L.bebelm_debug_expire_next_wait(1) == bb.OK
        with pytest.raises(bb.BebelmError) as e:
            w.matmul(xh)
        assert e.value.code == bb.ERR_TIMEOUT
        np.testing.assert_array_equal(w.matmul(xh), want.cpu().numpy())
        w.check()

        graph = torch.cuda.CUDAGraph()
        assert L.bebelm_debug_expire_next_wait(1) == bb.OK
        with torch.cuda.graph(graph):
            w.matmul(x, out=out)
        for _ in range(2):
            graph.replay()
            with pytest.raises(bb.BebelmError):
                w.check()
        # without a check the handle's next product reports it, before its own work
        graph.replay()
        torch.cuda.synchronize()
        with pytest.raises(bb.BebelmError):
            w.matmul(x)
        assert torch.equal(w.matmul(x), want)
    finally:
        assert L.bebelm_debug_expire_next_wait(0) == bb.OK
    w.check()


def dead_inputs(n_in):
    """Two inputs of every 128 whose codes are their zero points in all rows, so that nothing there may reach an output."""
    return [c + i for c in range(0, n_in, 128) for i in (5, 17)]


def weights_with_dead_inputs(n_out, n_in, group, seed, zeros=True, exact=True, scales=torch.float16):
    codes, sc, z = weights(n_out, n_in, group, seed, zeros, scales, exact)
    full = torch.stack((codes & 15, codes >> 4), -1).view(n_out, n_in)
    for k in dead_inputs(n_in):
        full[:, k] = 8 if z is None else z[:, k // group]
    return full[:, 0::2] | full[:, 1::2] << 4, sc, z


@pytest.mark.parametrize("kind", ["f32", "bf16"])
@pytest.mark.parametrize("t", [1, 2, 7, 8, 9, 13, 16, 17, 70])
@pytest.mark.parametrize("n_in,group", [(416, 32), (448, 64), (512, 128), (768, 256)])
def test_every_digit_of_every_input(n_in, group, t, kind):
    """One activation of 19 bits (bf16: 8) at a time, at every input, alone and beside one 2^15 or 2^18 times as large that the weights
    do not see: products with the 5 bits of a code less its zero point have 24 bits, so outputs are exact. A digit or a term that is lost,
    misplaced or added under a wrong zero point shows at its input."""
    n_out = 70
    codes, sc, z = weights_with_dead_inputs(n_out, n_in, group, 5 + group)
    w, wd = bb.W4Weights(codes, sc, z, group=group), dense(codes, sc, z, group)
    dead = set(dead_inputs(n_in))
    live = [k for k in range(n_in) if k not in dead]
    g = torch.Generator(device="cuda").manual_seed(t * 1000 + n_in)
    for far in (None, 15, 18):
        for at in range(0, len(live), t):
            k = torch.tensor([live[(at + i) % len(live)] for i in range(t)], device="cuda")
            bits = 19 if kind == "f32" else 8
            x = torch.zeros(t, n_in, device="cuda", dtype=torch.float64)
            v = torch.randint(1 << (bits - 1), 1 << bits, (t,), device="cuda", generator=g) * (1 - 2 * torch.randint(0, 2, (t,), device="cuda", generator=g))
            rows = torch.arange(t, device="cuda")
            x[rows, k] = v.double()
            if far:
                x[rows, k // 128 * 128 + 5] = 2.0 ** (bits + far)
            x = x.to(KINDS[kind])
            y = w.matmul(x, out_dtype=bb.F32).double()
            want = x.double() @ wd.t()
            assert torch.equal(y, want), (far, at, float((y - want).abs().max()))


@pytest.mark.parametrize("case", [(1, 2048, 300, 128, "f32"), (1, 8192, 300, 128, "bf16"), (4, 2080, 515, 32, "f32"), (7, 1024, 100, 64, "bf16"),
                                  (8, 2048, 333, 128, "f32"), (8, 8192, 48, 64, "f32"), (12, 1024, 700, 32, "f32"), (16, 640, 400, 640, "bf16"),
                                  (16, 2048, 8192, 128, "f32"), (24, 2080, 300, 32, "f32"), (130, 512, 260, 128, "f32")],
                         ids=lambda c: "-".join(map(str, c)))
@pytest.mark.parametrize("outlier", [10.0, 1e2, 1e3, 1e4, 1e5])
def test_activations_beside_far_larger_ones(case, outlier):
    """A residual stream's: one of 128 activations is far larger than the rest, and the weights (at their zero points there) do not
    see it, so the rest must come out as precisely as without it. Bound, A = Σ|w||x| over the rest: as digits each activation is kept to
    2^-23 of the largest M of 128 where M is at most 8 times their mean magnitude, else to 2^-38 M (half steps: the largest is 2^21.99 steps or
    2^37.99 at least, hence 2^-22.99 and 2^-37.99); in more than 16 tokens f32 to 2^-24 of itself and 2^-39 of its token's largest. A sum's roundings: 3 a
    scaled sum (one a group, 128 or 32 inputs) and one for each that it is added to; more than 16 tokens 17 per 16 inputs of a group and term."""
    t, n_in, n_out, group, kind = case
    codes, sc, z = weights_with_dead_inputs(n_out, n_in, group, 3, exact=False)
    w, wd = bb.W4Weights(codes, sc, z, group=group), dense(codes, sc, z, group)
    x, _ = activations(t, n_in, kind, 0, 11)
    x[:, 5::128] = outlier * (1 + torch.rand_like(x[:, 5::128].float())).to(x.dtype)
    x[0] = activations(1, n_in, kind, 0, 12)[0]  # a token without them, beside the others
    x[0, 5::128] = 0
    y = w.matmul(x, out_dtype=bb.F32).double()
    xd = x.double()
    want, a = xd @ wd.t(), xd.abs().clone()
    a[:, 5::128] = 0
    wa = wd.abs()
    flushes = n_in / min(group, 128)
    steps = 3 * 17 * max(1, group // 16) * 2 if t > 16 else 0
    tol = (flushes + 8 + steps) * 2.0 ** -24 * (a @ wa.t())
    if t > 16:
        err = 2.0 ** -39 * xd.abs().amax(-1, keepdim=True) + 2.0 ** -24 * a if kind == "f32" else torch.zeros_like(a)
    else:
        pad = torch.nn.functional.pad(xd.abs(), (0, -n_in % 128)).view(t, -1, 128)
        counts = torch.full((pad.shape[1],), 128.0, device="cuda", dtype=torch.float64)
        if n_in % 128:
            counts[-1] = n_in % 128
        big = pad.amax(-1)
        # (next to the border either may hold)
        err = torch.where(big <= 8.001 * pad.sum(-1) / counts, 2.0 ** -22.99 * big, 2.0 ** -37.99 * big).repeat_interleave(128, 1)[:, :n_in]
    tol = tol + (err * (a > 0)) @ wa.t()
    bad = (y - want).abs() > tol
    assert not bad.any(), (int(bad.sum()), float(((y - want).abs() / tol.clamp(min=1e-300)).max()))
    # a token's results do not depend on the tokens beside it
    if t > 1 and t <= 8:
        assert torch.equal(w.matmul(x[:1], out_dtype=bb.F32).double()[0], y[0])
        assert torch.equal(w.matmul(x[1:2], out_dtype=bb.F32).double()[0], y[1])


@pytest.mark.parametrize("t", [1, 8, 9, 16, 17, 40, 130])
@pytest.mark.parametrize("n_in,group", [(32, 32), (64, 64), (64, 32), (128, 128)])
def test_the_smallest_layers(n_in, group, t):
    """Fewer inputs than a tile's 64 or 128, one row and three."""
    for n_out in (1, 3):
        for kind, xg in (("f32", 0), ("bf16", 0), ("int8", 0), ("int8", 32)):
            check((t, n_in, n_out, group, kind, xg, True, torch.float16, bb.F32), True)


def test_calls_of_one_handle_from_threads():
    """Products of one handle at once: device memory on a stream a thread, and host memory."""
    import threading
    codes, sc, z = weights(300, 512, 64, 3)
    w = bb.W4Weights(codes, sc, z, group=64)
    xs = [activations(t, 512, "f32", 0, t)[0] for t in (1, 5, 20, 40)]
    want = [w.matmul(x) for x in xs]
    host = [(x.cpu().numpy(), y.cpu().numpy()) for x, y in zip(xs, want)]
    torch.cuda.synchronize()
    bad = []

    def work(i):
        stream = torch.cuda.Stream()
        for _ in range(20):
            if i % 2:
                y = w.matmul(xs[i], stream=stream)
                stream.synchronize()
                if not torch.equal(y, want[i]):
                    bad.append(i)
            elif not np.array_equal(w.matmul(host[i][0]), host[i][1]):
                bad.append(i)

    threads = [threading.Thread(target=work, args=(i,)) for i in range(4)]
    for th in threads:
        th.start()
    for th in threads:
        th.join()
    assert not bad
    w.check()
