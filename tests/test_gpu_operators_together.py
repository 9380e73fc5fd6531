"""The operators around the attention as they are used: one decode step over drafted tokens, from the
residual stream to the verified tokens, and the calls around it (graphs, long strides, workspaces).

Every part of the step is compared with its definition in 64 bits (the attention with the oracle) on the
inputs that it was given, so that no tolerance has to cover a code of the 8-bit norm next to a border.
Products: the bound of test_gpu_w4 plus, for the few tokens of a step, the activations' own rounding,
2^-23 of the largest of 128 neighbours times the sum of |w|.
"""
import ctypes as C

import numpy as np
import pytest
import torch

import bebelm_b200 as bb
import oracle
import test_gpu_addnorm as N
import test_gpu_verify as V
import test_gpu_w4 as W

pytestmark = pytest.mark.gpu

HIDDEN, HEADS, KV, VOCAB, HISTORY = 512, 8, 2, 1003, 37
KVD = KV * 64


def product_close(y, x, w, group, terms=1):
    """y against x w^T, all float64: x [t, n_in], w [n_out, n_in]."""
    want, a = x @ w.t(), x.abs() @ w.abs().t()
    steps = max(1, group // 16) * terms
    big = torch.nn.functional.pad(x.abs(), (0, -x.shape[1] % 128)).reshape(x.shape[0], -1, 128).amax(-1)
    big = big.repeat_interleave(128, 1)[:, :x.shape[1]]
    tol = (17 * steps * 2.0 ** -23 + (x.shape[1] / group + 2) * 2.0 ** -24) * a + 2.0 ** -23 * (big @ w.abs().t())
    assert ((y.double() - want).abs() <= tol).all()


class Step:
    """The weights of one attention layer and a head, and a step of 1 + d tokens over them."""

    def __init__(self, d):
        self.t = d + 1
        self.parts = {}
        for i, (name, n_out, n_in, group, zeros) in enumerate((("qkv", HIDDEN + 2 * KVD, HIDDEN, 32, True), ("out", HIDDEN, HIDDEN, 64, False),
                                                               ("head", VOCAB, HIDDEN, 128, True))):
            codes, sc, z = W.weights(n_out, n_in, group, 10 + i, zeros)
            self.parts[name] = (bb.W4Weights(codes, sc, z, group=group), W.dense(codes, sc, z, group), group)
        g = torch.Generator(device="cuda").manual_seed(5)
        self.gains = [1 + 0.1 * torch.randn(HIDDEN, device="cuda", generator=g) for _ in range(2)]
        self.qg, self.kg = [(1 + 0.1 * torch.randn(64, device="cuda", generator=g)) for _ in range(2)]

    def before(self, x, res, h, codes, scales, qkv):
        bb.add_rmsnorm(x, self.gains[0], res, out_dtype=bb.INT8, group=128, sum_out=h, out=codes, scales=scales)
        self.parts["qkv"][0].matmul(codes, scales, out=qkv)

    def attention(self, cache, qkv):
        q, k, v = (p.contiguous() for p in qkv.split([HIDDEN, KVD, KVD], 1))
        return cache.attn_prefill(0, q, k, v, self.qg, self.kg, HISTORY, theta=1e6, n_heads=HEADS)

    def after(self, att, h, draft, tokens, u, us, out, accepted):
        o = self.parts["out"][0].matmul(att)
        y, h2 = bb.add_rmsnorm(o, self.gains[1], h)
        logits = self.parts["head"][0].matmul(y)
        bb.verify_drafts(logits.unsqueeze(0), tokens, u, us, draft=draft, temperature=0.8, out=out, accepted=accepted)
        return o, y, h2, logits


@pytest.mark.parametrize("d", [0, 4, 23])  # one token, a step of drafts, a draft long enough for the many-token products
def test_a_decode_step_over_drafts(d):
    s = Step(d)
    g = torch.Generator(device="cuda").manual_seed(d)
    new = lambda *n: torch.randn(*n, device="cuda", generator=g)
    cache = bb.Cache(n_layers=1, n_kv_heads=KV, max_context=128)
    cache.attn_prefill(0, new(HISTORY, HIDDEN), new(HISTORY, KVD), new(HISTORY, KVD), s.qg, s.kg, 0, theta=1e6, n_heads=HEADS)
    old_k, old_v = cache.read(0)
    x, res = new(s.t, HIDDEN), 2 * new(s.t, HIDDEN)
    h, codes = torch.empty_like(x), torch.empty(s.t, HIDDEN, dtype=torch.int8, device="cuda")
    scales, qkv = torch.empty(s.t, HIDDEN // 128, device="cuda"), torch.empty(s.t, HIDDEN + 2 * KVD, device="cuda")
    s.before(x, res, h, codes, scales, qkv)
    assert torch.equal(h, x + res)
    want_q, want_s = N.codes_of(N.steps(h.cpu().numpy(), s.gains[0].cpu().numpy()), 128)
    np.testing.assert_array_equal(codes.cpu().numpy(), want_q)
    np.testing.assert_array_equal(scales.cpu().numpy(), want_s)
    product_close(qkv, W.floats(codes, scales), *s.parts["qkv"][1:])
    other = cache.clone()
    att = s.attention(cache, qkv)
    q, k, v = (p.cpu().numpy() for p in qkv.split([HIDDEN, KVD, KVD], 1))
    want = oracle.attn_batch(q, k, v, HISTORY, s.qg.cpu().numpy(), s.kg.cpu().numpy(), 1e6, 1e-5, HEADS, KV, 64, old_k, old_v)[0]
    assert np.abs(att.cpu().numpy() - want).max() <= 1e-5 * max(1.0, np.abs(v).max())

    # the drafts: what a small model close to the target would have proposed
    rng = np.random.default_rng(d)
    out, accepted = torch.empty(1, s.t, dtype=torch.int32, device="cuda"), torch.empty(1, dtype=torch.int32, device="cuda")
    tokens = torch.zeros(1, d, dtype=torch.int32, device="cuda")
    u = torch.from_numpy(rng.random((1, d)).astype(np.float32)).cuda()
    us = torch.from_numpy(rng.random(1).astype(np.float32)).cuda()
    draft = torch.zeros(1, d, VOCAB, device="cuda")
    _, _, _, logits = s.after(att, h, draft, tokens, u, us, out, accepted)
    draft.copy_(logits[:d].unsqueeze(0) + 0.1 * new(1, d, VOCAB))
    p = torch.softmax(draft.double() / 0.8, -1)
    if d:
        tokens.copy_(torch.multinomial(p[0], 1, generator=g).t().int())
    o, y, h2, logits = s.after(att, h, draft, tokens, u, us, out, accepted)
    product_close(o, att.double(), *s.parts["out"][1:], terms=3)
    assert torch.equal(h2, o + h)
    np.testing.assert_array_equal(y.cpu().numpy(), N.steps(h2.cpu().numpy(), s.gains[1].cpu().numpy()))
    product_close(logits, y.double(), *s.parts["head"][1:], terms=3)
    V.same((out.cpu().numpy(), accepted.cpu().numpy()),
           V.reference(logits.unsqueeze(0).cpu().numpy(), tokens.cpu().numpy(), u.cpu().numpy(), us.cpu().numpy(), draft.cpu().numpy(),
                       temperature=0.8))

    # the same step from two graphs (the attention between them keeps host state), with the inputs changed after capture
    ins = [t.clone() for t in (x, res, h, att, draft, tokens, u, us)]
    gx, gres, gh, gatt, gdraft, gtok, gu, gus = ins
    g1, g2 = torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph()
    gcodes, gscales, gqkv, gout, gacc = (torch.empty_like(t) for t in (codes, scales, qkv, out, accepted))
    with torch.cuda.graph(g1):
        s.before(gx, gres, gh, gcodes, gscales, gqkv)
    with torch.cuda.graph(g2):
        s.after(gatt, gh, gdraft, gtok, gu, gus, gout, gacc)
    for t in (gx, gres, gatt, gout):
        t.zero_()
    gx.copy_(x), gres.copy_(res)
    g1.replay()
    assert torch.equal(gqkv, qkv) and torch.equal(gh, h)
    gatt.copy_(s.attention(other, gqkv))
    assert torch.equal(gatt, att)
    g2.replay()
    assert torch.equal(gout, out) and torch.equal(gacc, accepted)


def test_two_graphs_at_once():
    """Graphs of the calls that use a workspace, replayed side by side: each has its own."""
    codes, sc, z = W.weights(700, 1024, 128, 3)
    w = bb.W4Weights(codes, sc, z, group=128)
    runs = []
    for i in range(2):
        x, _ = W.activations(40, 1024, "f32", 0, i)
        target, tokens, u, us, draft = (torch.from_numpy(a).cuda() for a in V.inputs(3, 4, 9000, 1.0, i))
        y, tok, acc = w.matmul(x), *bb.verify_drafts(target, tokens, u, us, draft=draft)
        gy, gt, ga = torch.empty_like(y), torch.empty_like(tok), torch.empty_like(acc)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            w.matmul(x, out=gy)
            bb.verify_drafts(target, tokens, u, us, draft=draft, out=gt, accepted=ga)
        runs.append((graph, (y, tok, acc), (gy, gt, ga), torch.cuda.Stream(), (x, target, tokens, u, us, draft)))
    torch.cuda.synchronize()
    for _ in range(20):
        for graph, _, _, stream, _ in runs:
            with torch.cuda.stream(stream):
                graph.replay()
    torch.cuda.synchronize()
    for _, want, got, _, _ in runs:
        assert all(torch.equal(a, b) for a, b in zip(want, got))


def test_strides_beyond_32_bits():
    """Rows 2^28 and 2^31 elements apart: the same results as packed rows."""
    buf = torch.empty(19 * 2 ** 28 + 2048, device="cuda")
    codes, sc, z = W.weights(300, 512, 64, 3)
    w = bb.W4Weights(codes, sc, z, group=64)
    for dtype in (torch.float32, torch.bfloat16):
        b = buf.view(dtype)
        rows = b.as_strided((3, 2048), (2 ** 31, 1))
        x, _, gain = N.inputs(3, 2048, dtype, 1, residual=False)
        rows.copy_(x)
        assert torch.equal(bb.add_rmsnorm(rows, gain)[0], bb.add_rmsnorm(x, gain)[0])
        assert torch.equal(bb.add_rmsnorm(x, gain, x, sum_out=rows)[0], bb.add_rmsnorm(x, gain, x)[0])
        assert torch.equal(rows, x + x)
        far = b.as_strided((20, 512), (2 ** 28, 1))
        x = torch.randn(20, 512, device="cuda").to(dtype)
        far.copy_(x)
        for t in (3, 20):
            assert torch.equal(w.matmul(far[:t]), w.matmul(x[:t]))
    far = buf.view(torch.int8).as_strided((20, 512), (2 ** 28, 1))
    x, xs = W.activations(20, 512, "int8", 128, 1)
    far.copy_(x)
    for t in (3, 20):
        assert torch.equal(w.matmul(far[:t], xs[:t]), w.matmul(x[:t], xs[:t]))
    target, tokens, u, us, _ = (None if a is None else torch.from_numpy(a).cuda() for a in V.inputs(1, 2, 5000, 1.0, 1, draft_rows=False))
    far = buf.as_strided((1, 3, 5000), (2 ** 31, 2 ** 31, 1))
    far.copy_(target)
    for temp in (1.0, 0.0):
        a, b = bb.verify_drafts(far, tokens, u, us, temperature=temp), bb.verify_drafts(target, tokens, u, us, temperature=temp)
        assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])
    del buf, b, rows, far
    torch.cuda.empty_cache()


@pytest.mark.parametrize("t", [2, 20])
def test_codes_beyond_4_gb(t):
    n_in, n_out, group = 32768, 270000, 128
    codes, sc, _ = W.weights(n_out, n_in, group, 7, zeros=False)
    w = bb.W4Weights(codes, sc, None, group=group)
    x, xs = W.activations(t, n_in, "int8", 256, 3)
    y = w.matmul(x, xs)
    at = torch.tensor([0, 1, 127, 131071, 131072, 262143, 262144, 262145, 269983, 269999], device="cuda")
    product_close(y[:, at], W.floats(x, xs), W.dense(codes[at], sc[at], None, group), group)
    w.close()
    del codes, sc, w
    torch.cuda.empty_cache()


def test_workspaces_are_checked():
    """A workspace that is missing, too small or not aligned is refused before any launch."""
    L = bb.load_library()
    codes, sc, z = W.weights(64, 256, 64, 3)
    w = bb.W4Weights(codes, sc, z, group=64)
    x, y, n = torch.randn(40, 256, device="cuda"), torch.zeros(40, 64, device="cuda"), C.c_size_t()
    ws = torch.empty(1 << 20, dtype=torch.uint8, device="cuda")
    assert L.bebelm_w4_workspace(w._h, x.data_ptr(), bb.F32, 256, 0, 40, C.byref(n)) == bb.OK and 0 < n.value < ws.numel() - 256
    product = lambda p, b: L.bebelm_w4_matmul(w._h, x.data_ptr(), bb.F32, 256, None, 0, 40, y.data_ptr(), bb.F32, p, b, bb.MEM_DEVICE, None)
    for p, b in ((None, n.value), (ws.data_ptr(), n.value - 1), (ws.data_ptr() + 8, n.value)):
        assert product(p, b) == bb.ERR_INVALID and "workspace" in bb.last_error()
    target, tok = torch.randn(1, 3, 500, device="cuda"), torch.zeros(1, 2, dtype=torch.int32, device="cuda")
    u, out = torch.rand(1, 2, device="cuda"), torch.zeros(1, 3, dtype=torch.int32, device="cuda")
    assert L.bebelm_verify_workspace(1, 2, 500, 0, 0, 1.0, C.byref(n)) == bb.OK and 0 < n.value < ws.numel() - 256
    verify = lambda p, b: L.bebelm_verify_drafts(target.data_ptr(), 500, None, 500, 1, 2, 500, 0, 1.0, tok.data_ptr(), None, u.data_ptr(),
                                                 u.data_ptr(), out.data_ptr(), out.data_ptr(), p, b, bb.MEM_DEVICE, None)
    for p, b in ((None, n.value), (ws.data_ptr(), n.value - 1), (ws.data_ptr() + 8, n.value)):
        assert verify(p, b) == bb.ERR_INVALID and "workspace" in bb.last_error()
    torch.cuda.synchronize()
    assert not y.any() and not out.any()
    assert product(ws.data_ptr(), 1 << 19) == bb.OK
    torch.cuda.synchronize()
    assert torch.equal(y, w.matmul(x))


def later(stream, ms=60):
    """Keeps a stream busy for a while (about 2 million cycles a millisecond)."""
    with torch.cuda.stream(stream):
        torch.cuda._sleep(2_000_000 * ms)


def calls_on(stream):
    """Each operator on ``stream`` with results of its own: name -> function that gives them."""
    n = 2 ** 21
    x, gain = torch.randn(64, n // 64, device="cuda"), torch.ones(n // 64, device="cuda")
    codes, sc, z = W.weights(n // 64, 256, 64, 3)
    w, a = bb.W4Weights(codes, sc, z, group=64), torch.randn(64, 256, device="cuda")
    target, tokens = torch.randn(4096, 1, 64, device="cuda"), torch.zeros(4096, 0, dtype=torch.int32, device="cuda")
    return {"add_rmsnorm": lambda: bb.add_rmsnorm(x, gain, x, stream=stream),
            "codes": lambda: bb.add_rmsnorm(x, gain, x, out_dtype=bb.INT8, group=32, stream=stream),
            "matmul": lambda: (w.matmul(a, stream=stream),),
            "verify_drafts": lambda: bb.verify_drafts(target, tokens, None, None, temperature=0.0, stream=stream)}


def results_belong_to(side, call):
    """Blocks of the allocator's and the streams they are in use on. (1) Blocks that the current stream still works with,
    freed before the call: a result on another stream gets none of them. (2) Results dropped while their stream still works with
    them: an allocation of the current stream gets none of them. (3) Results dropped while the current stream still reads them: the
    next call on the other stream gets none of them."""
    current = torch.cuda.current_stream()
    torch.cuda.synchronize()
    got = call()
    side.synchronize()
    want = [t.clone() for t in got]
    del got
    torch.cuda.synchronize()
    spans = lambda ts: [(t.data_ptr(), t.data_ptr() + t.numel() * t.element_size()) for t in ts]
    apart = lambda places, ts: all(p1 <= q0 or q1 <= p0 for p0, p1 in places for q0, q1 in spans(ts))

    held = [torch.full_like(t, 5) for t in want for _ in range(4)]
    later(current)
    copies = [t.clone() for t in held]  # queued behind the wait
    places = spans(held)
    del held
    got = call()
    assert apart(places, got)
    torch.cuda.synchronize()
    assert all((c == 5).all() for c in copies) and all(torch.equal(a, b) for a, b in zip(got, want))
    del got, copies

    later(side)
    got = call()
    places = spans(got)
    del got
    fresh = [torch.empty_like(t) for t in want for _ in range(4)]
    assert apart(places, fresh)
    torch.cuda.synchronize()
    del fresh

    got = call()
    current.wait_stream(side)
    later(current)
    read = [t.clone() for t in got]
    places = spans(got)
    del got
    other = call()
    assert apart(places, other) or current.query()  # (once the stream is done they may be used again)
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(read, want)) and all(torch.equal(a, b) for a, b in zip(other, want))


@pytest.mark.parametrize("raw", [False, True])
@pytest.mark.parametrize("name", ["add_rmsnorm", "codes", "matmul", "verify_drafts"])
def test_results_of_a_call_on_another_stream(name, raw):
    side = torch.cuda.Stream()
    results_belong_to(side, calls_on(side.cuda_stream if raw else side)[name])


def five_caches():
    """Empty ones of one pool, which share its scratch (clearing a cache, and a pool's first call, wait for the device)."""
    pool = bb.Pool(n_layers=1, n_kv_heads=KV, n_pages=64)
    return iter([bb.Cache(pool=pool, max_context=512) for _ in range(5)])


@pytest.mark.parametrize("name", ["attn_prefill", "matmul", "logits", "sample_greedy", "attn_layer_batch"])
def test_results_of_the_other_calls_on_another_stream(name):
    """The same for the attention, the K-quant products, the head and the sampler."""
    side = torch.cuda.Stream()
    t, n_out = 300, 4096
    rng = np.random.default_rng(3)
    packed = lambda rows, n: (0.05 * rng.standard_normal((rows, n))).astype(np.float16).reshape(-1).view(np.uint8)
    ones = torch.ones(64, device="cuda")
    if name == "attn_prefill":
        q, k, v = (torch.randn(t, n, device="cuda") for n in (HIDDEN, KVD, KVD))
        caches, kept = five_caches(), []

        def call():
            kept.append(next(caches))
            return (kept[-1].attn_prefill(0, q, k, v, ones, ones, 0, n_heads=HEADS, stream=side),)
    elif name == "matmul":
        w, x = torch.from_numpy(packed(n_out, HIDDEN)).cuda(), torch.randn(t, HIDDEN, device="cuda")
        call = lambda: (bb.matmul(bb.GGML_F16, w, HIDDEN, n_out, x, t, stream=side),)
    elif name == "logits":
        head, h = bb.Head(bb.GGML_F16, packed(60000, HIDDEN), HIDDEN, 60000, np.ones(HIDDEN, np.float32)), torch.randn(HIDDEN, device="cuda")
        call = lambda: head.logits(h, stream=side)
    elif name == "sample_greedy":
        logits, history = torch.randn(60000, device="cuda"), torch.tensor([5, 7], dtype=torch.int32, device="cuda")
        call = lambda: (bb.sample_greedy(logits, history, 1.0, stream=side),)
    else:
        gain = np.ones(64, np.float32)
        weights = bb.AttnWeights((bb.GGML_F16, packed(HIDDEN, HIDDEN)), (bb.GGML_F16, packed(KVD, HIDDEN)), (bb.GGML_F16, packed(KVD, HIDDEN)),
                                 (bb.GGML_F16, packed(HIDDEN, HIDDEN)), gain, gain, n_heads=HEADS, n_kv_heads=KV, hidden=HIDDEN)
        x, kept = torch.randn(t, HIDDEN, device="cuda"), []
        caches = five_caches()

        def call():
            kept.append(next(caches))
            return (bb.attn_layer_batch(kept[-1], 0, weights, x, 0, stream=side),)
    results_belong_to(side, call)


def test_host_calls_beside_queued_device_products():
    """Host-memory products and verifications while K-quant products, which quantize into the library's scratch, are queued on
    another stream: neither disturbs the other."""
    import test_gpu_quant as Q
    n_in, n_out, t = 2048, 2048, 64
    w = torch.from_numpy(Q.random_q4k(n_out, n_in, 3)).cuda()
    x = torch.randn(t, n_in, device="cuda")
    want = bb.matmul(bb.GGML_Q4_K, w, n_in, n_out, x, t)
    codes, sc, z = W.weights(300, 512, 64, 3)
    w4 = bb.W4Weights(codes, sc, z, group=64)
    xh = W.activations(40, 512, "f32", 0, 1)[0].cpu().numpy()
    wanth = w4.matmul(xh)
    args = V.inputs(3, 4, 9000, 1.0, 2)
    wantv = bb.verify_drafts(*args[:4], draft=args[4])
    side = torch.cuda.Stream()
    torch.cuda.synchronize()
    for _ in range(10):
        outs = [bb.matmul(bb.GGML_Q4_K, w, n_in, n_out, x, t, stream=side) for _ in range(30)]
        for _ in range(4):
            np.testing.assert_array_equal(w4.matmul(xh), wanth)
            V.same(bb.verify_drafts(*args[:4], draft=args[4]), wantv)
        side.synchronize()
        assert all(torch.equal(o, want) for o in outs)
