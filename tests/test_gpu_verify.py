"""Drafted tokens against the target's rows: verify_drafts and its definition in 64 bits, row by row.

Outputs are whole numbers and must be equal. A border case (a random number within rounding of a
border between two tokens) would need a coincidence of 1e-10 in these seeded inputs for the
drawn token, and of 1e-6 for an acceptance.
"""
import ctypes as C

import numpy as np
import pytest
import torch

import bebelm_b200 as bb

pytestmark = pytest.mark.gpu


def softmax64(row, temp):
    row = np.where(np.isnan(row), -np.inf, row.astype(np.float64))
    m = row.max()
    if m == -np.inf:
        return np.zeros_like(row)
    e = np.exp((row - m) / temp)
    return e / e.sum()


def pick(w, u):
    total = np.cumsum(w)[-1]
    if not total > 0:
        return 0
    over = np.nonzero((np.cumsum(w) > float(u) * total) & (w > 0))[0]
    return int(over[0]) if over.size else int(np.nonzero(w > 0)[0][-1])


def first_max(row):
    best, at = -np.inf, 0
    for i, v in enumerate(row):
        if v > best:
            best, at = v, i
    return at


def reference(target, tokens, u, us, draft=None, n_drafts=None, temperature=1.0, probs=False):
    b, d1, v = target.shape
    d = d1 - 1
    out, acc = np.full((b, d1), -1, np.int32), np.zeros(b, np.int32)
    for s in range(b):
        n = d if n_drafts is None else int(n_drafts[s])
        prob = (lambda r: np.where(r > 0, r, 0).astype(np.float64)) if probs else (lambda r: softmax64(r, temperature))
        a = 0
        while a < n:
            x = int(tokens[s, a])
            if temperature == 0:
                if first_max(target[s, a]) != x:
                    break
            else:
                q = 1.0 if draft is None else prob(draft[s, a])[x] if 0 <= x < v else 1.0
                p = prob(target[s, a])[x] if 0 <= x < v else 0.0
                if not float(u[s, a]) * q < p:
                    break
            a += 1
        if temperature == 0:
            nxt = first_max(target[s, a])
        else:
            p = prob(target[s, a])
            w = p
            if a < n:
                if draft is None:
                    w = p.copy()
                    if 0 <= tokens[s, a] < v:
                        w[tokens[s, a]] = 0
                else:
                    w = np.maximum(p - prob(draft[s, a]), 0)
                if not w.sum() > 0:
                    w = p
            nxt = pick(w, us[s])
        out[s, :a] = tokens[s, :a]
        out[s, a] = nxt
        acc[s] = a
    return out, acc


def inputs(b, d, v, temp, seed, near=0.5, probs=False, draft_rows=True):
    rng = np.random.default_rng(seed)
    target = (2.5 * rng.standard_normal((b, d + 1, v))).astype(np.float32)
    draft = (target[:, :d] + near * rng.standard_normal((b, d, v))).astype(np.float32)
    tokens = np.zeros((b, d), np.int32)
    for s in range(b):
        for i in range(d):
            tokens[s, i] = draft[s, i].argmax() if temp == 0 else rng.choice(v, p=softmax64(draft[s, i], temp))
    if probs:
        target = np.stack([[softmax64(r, temp) for r in s] for s in target]).astype(np.float32).reshape(b, d + 1, v)
        draft = np.array([[softmax64(r, temp) for r in s] for s in draft], np.float32).reshape(b, d, v)
    u, us = rng.random((b, d)).astype(np.float32), rng.random(b).astype(np.float32)
    return target, tokens, u, us, draft if draft_rows else None


def run(target, tokens, u, us, draft=None, n_drafts=None, **kw):
    dev = [None if a is None else torch.from_numpy(np.ascontiguousarray(a)).cuda() for a in (target, tokens, u, us, draft, n_drafts)]
    o, a = bb.verify_drafts(dev[0], dev[1], dev[2], dev[3], draft=dev[4], n_drafts=dev[5], **kw)
    return o.cpu().numpy(), a.cpu().numpy()


def same(got, want):
    np.testing.assert_array_equal(got[1], want[1])
    np.testing.assert_array_equal(got[0], want[0])


@pytest.mark.parametrize("temp", [1.0, 0.7, 0.0])
@pytest.mark.parametrize("draft_rows", [True, False])
@pytest.mark.parametrize("b,d,v", [(1, 1, 1), (1, 0, 40), (2, 3, 2), (5, 4, 33), (3, 2, 1000), (4, 8, 4097), (2, 3, 20000), (1, 2, 65537)])
def test_logits(b, d, v, draft_rows, temp):
    for seed in range(3):
        t, tok, u, us, dr = inputs(b, d, v, temp, 100 * seed + v + b, draft_rows=draft_rows)
        same(run(t, tok, u, us, dr, temperature=temp), reference(t, tok, u, us, dr, temperature=temp))


@pytest.mark.parametrize("draft_rows", [True, False])
@pytest.mark.parametrize("b,d,v", [(1, 1, 1), (3, 4, 50), (6, 5, 3201), (2, 7, 32003)])
def test_probabilities(b, d, v, draft_rows):
    for seed in range(3):
        t, tok, u, us, dr = inputs(b, d, v, 1.0, 17 * seed + v, probs=True, draft_rows=draft_rows)
        same(run(t, tok, u, us, dr, probs=True), reference(t, tok, u, us, dr, probs=True))


def test_one_full_vocabulary_and_ragged_drafts():
    t, tok, u, us, dr = inputs(6, 4, 128000, 0.75, 1)
    n = np.array([4, 0, 3, 1, 4, 2], np.int32)
    same(run(t, tok, u, us, dr, n, temperature=0.75), reference(t, tok, u, us, dr, n, temperature=0.75))
    same(run(t, tok, u, us, None, n, temperature=0.75), reference(t, tok, u, us, None, n, temperature=0.75))
    same(run(t, tok, u, us, dr, n, temperature=0.0), reference(t, tok, u, us, dr, n, temperature=0.0))


def test_many_sequences():
    t, tok, u, us, dr = inputs(300, 3, 257, 1.0, 5)
    same(run(t, tok, u, us, dr), reference(t, tok, u, us, dr))
    t, tok, u, us, dr = inputs(3, 70, 100, 1.0, 6, near=0.05)  # more drafts than one group of decisions
    same(run(t, tok, u, us, dr), reference(t, tok, u, us, dr))


def test_same_rows_accept_everything():
    """p = q: each draft is accepted with certainty, and the next token comes from the last row."""
    t, tok, u, us, dr = inputs(4, 6, 500, 1.0, 9, near=0.0)
    o, a = run(t, tok, u, us, dr)
    assert (a == 6).all()
    same((o, a), reference(t, tok, u, us, dr))


@pytest.mark.parametrize("draft_rows", [True, False])
def test_masked_rows_nan_and_borders(draft_rows):
    """Logits masked with -inf and with the lowest float, NaN entries, a row with nothing left, random
    numbers at the ends of [0, 1)."""
    t, tok, u, us, dr = inputs(6, 3, 700, 1.0, 21, draft_rows=draft_rows)
    low = np.finfo(np.float32).min
    t[0, :, 5:] = -np.inf
    t[1, :, ::2] = low
    t[2, :, 7] = np.nan
    t[3, 0] = -np.inf          # refused at once, nothing to draw from: token 0
    t[4, :, :] = -np.inf
    t[4, :, 699] = 1.0         # one choice
    if draft_rows:
        dr[1, :, ::2] = low
        dr[2, 0, 9] = np.nan
        dr[5, 0] = -np.inf     # a draft row without weight: q = 0
    us[:3] = [0.0, np.nextafter(np.float32(1), np.float32(0)), 0.5]
    u[5] = 0.0
    with np.errstate(invalid="ignore"):
        want = reference(t, tok, u, us, dr)
    same(run(t, tok, u, us, dr), want)
    assert want[0][3, 0] == 0 and want[1][3] == 0


def test_greedy_ties_and_nan():
    rng = np.random.default_rng(3)
    t = rng.integers(0, 4, (40, 4, 301)).astype(np.float32)  # ties everywhere
    t[1, 0] = np.nan
    t[2, 0] = -np.inf
    t[3, :, 3] = np.inf
    tok = np.stack([[first_max(r) for r in s[:3]] for s in t]).astype(np.int32)
    tok[::3, 1] = (tok[::3, 1] + 1) % 301
    want = reference(t, tok, None, None, temperature=0.0)
    dev = [torch.from_numpy(a).cuda() for a in (t, tok)]
    o, a = bb.verify_drafts(dev[0], dev[1], None, None, temperature=0.0)
    same((o.cpu().numpy(), a.cpu().numpy()), want)


def test_tokens_outside_the_vocabulary_are_refused():
    t, tok, u, us, dr = inputs(4, 2, 300, 1.0, 2)
    tok[0, 0], tok[1, 1], tok[2, 0] = -1, 300, 2 ** 31 - 1
    u[:] = 0.0
    same(run(t, tok, u, us, dr), reference(t, tok, u, us, dr))
    same(run(t, tok, u, us, None), reference(t, tok, u, us, None))
    # a sequence claims more drafts than there are, or fewer than none
    n = np.array([5, -3, 2, 2], np.int32)
    same(run(t, tok, u, us, dr, n), reference(t, tok, u, us, dr, np.clip(n, 0, 2)))


def test_padded_rows_and_unaligned_buffers():
    t, tok, u, us, dr = inputs(3, 4, 1001, 1.0, 4)
    want = reference(t, tok, u, us, dr)
    dev = [torch.from_numpy(a).cuda() for a in (tok, u, us)]
    for width, off in ((1001, 0), (1004, 0), (1010, 1), (1024, 4)):
        tb = torch.full((3, 5, width), 50.0, device="cuda")  # whatever lies beside the rows is large
        db = torch.full((3, 4, width), 50.0, device="cuda")
        tb[:, :, off:off + 1001] = torch.from_numpy(t).cuda()
        db[:, :, off:off + 1001] = torch.from_numpy(dr).cuda()
        o, a = bb.verify_drafts(tb[:, :, off:off + 1001], *dev, draft=db[:, :, off:off + 1001])
        same((o.cpu().numpy(), a.cpu().numpy()), want)


def test_host_buffers_streams_and_a_graph():
    t, tok, u, us, dr = inputs(4, 3, 20000, 0.8, 12)
    want = reference(t, tok, u, us, dr, temperature=0.8)
    same(bb.verify_drafts(t, tok, u, us, draft=dr, temperature=0.8), want)
    same(bb.verify_drafts(t, tok, None, None, temperature=0.0), reference(t, tok, u, us, temperature=0.0))
    dev = [torch.from_numpy(a).cuda() for a in (t, tok, u, us, dr)]
    t2, tok2, u2, us2, dr2 = inputs(4, 3, 20000, 0.8, 13)
    s1, s2 = torch.cuda.Stream(), torch.cuda.Stream()
    dev2 = [torch.from_numpy(a).cuda() for a in (t2, tok2, u2, us2, dr2)]
    torch.cuda.synchronize()
    got = []
    for _ in range(5):
        got.append((bb.verify_drafts(*dev[:4], draft=dev[4], temperature=0.8, stream=s1), want))
        got.append((bb.verify_drafts(*dev2[:4], draft=dev2[4], temperature=0.8, stream=s2),
                    reference(t2, tok2, u2, us2, dr2, temperature=0.8)))
    torch.cuda.synchronize()
    for (o, a), w in got:
        same((o.cpu().numpy(), a.cpu().numpy()), w)
    out, acc = torch.empty(4, 4, dtype=torch.int32, device="cuda"), torch.empty(4, dtype=torch.int32, device="cuda")
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        bb.verify_drafts(*dev[:4], draft=dev[4], temperature=0.8, out=out, accepted=acc)
    for a, b in zip(dev, dev2):
        a.copy_(b)
    graph.replay()
    same((out.cpu().numpy(), acc.cpu().numpy()), reference(t2, tok2, u2, us2, dr2, temperature=0.8))


def test_samples_follow_the_target():
    """Whatever the drafts, the first emitted token is distributed as the target: 20000 sequences over 6
    tokens; each frequency within 5 standard deviations."""
    rng = np.random.default_rng(0)
    n, v = 20000, 6
    tl, dl = rng.standard_normal(v).astype(np.float32), rng.standard_normal(v).astype(np.float32)
    p, q = softmax64(tl, 1.0), softmax64(dl, 1.0)
    t = np.broadcast_to(tl, (n, 2, v)).copy()
    dr = np.broadcast_to(dl, (n, 1, v)).copy()
    tok = rng.choice(v, (n, 1), p=q).astype(np.int32)
    o, _ = run(t, tok, rng.random((n, 1)).astype(np.float32), rng.random(n).astype(np.float32), dr)
    freq = np.bincount(o[:, 0], minlength=v) / n
    assert (np.abs(freq - p) <= 5 * np.sqrt(p * (1 - p) / n)).all()


@pytest.mark.parametrize("draft_rows", [True, False])
@pytest.mark.parametrize("base,step,temp", [(1000.0, 1e-3, 1e-6), (20.0, 1e-5, 1e-6), (1e12, 65536.0, 1.0), (-3e38, 1e32, 1.0), (3e38, 2e31, 1e6),
                                            (0.0, 1e5, 300.0)])
def test_logits_whose_neighbours_are_far_apart(base, step, temp, draft_rows):
    """Rows where a step of f32 at the largest logit is not small against the temperature: what counts
    still reaches down to the smallest weights, and the largest always counts."""
    b, d, v = 12, 3, 9001
    rng = np.random.default_rng(7)
    target = (base + step * rng.integers(-30, 1, (b, d + 1, v))).astype(np.float32)
    draft = (base + step * rng.integers(-30, 1, (b, d, v))).astype(np.float32)
    tokens = np.array([[rng.choice(np.nonzero(draft[s, i] == draft[s, i].max())[0]) for i in range(d)] for s in range(b)], np.int32)
    u, us = rng.random((b, d)).astype(np.float32), rng.random(b).astype(np.float32)
    args = (target, tokens, u, us, draft if draft_rows else None)
    same(run(*args, temperature=temp), reference(*args, temperature=temp))


@pytest.mark.parametrize("temp", [0.0, 1.0])
@pytest.mark.parametrize("draft_rows", [0, 1])
def test_the_queried_workspace_is_enough(draft_rows, temp):
    """C callers: a call with exactly the bytes that bebelm_verify_workspace gives for the same arguments, draft rows at
    temperature 0 (where they are not read) and without drafts included. All shapes share buffers of the largest one."""
    L = bb.load_library()
    vocab, n = 8192, C.c_size_t()
    rows = torch.randn(128 * 13, vocab, device="cuda")
    ints, floats = torch.zeros(128 * 13, dtype=torch.int32, device="cuda"), torch.rand(128 * 13, device="cuda")
    out, acc = torch.empty(128 * 13, dtype=torch.int32, device="cuda"), torch.empty(128, dtype=torch.int32, device="cuda")
    ws = torch.empty(8 << 20, dtype=torch.uint8, device="cuda")
    bad = []
    for b in list(range(1, 60)) + [64, 70, 99, 128]:
        for d in (0, 1, 4, 9, 12):
            assert L.bebelm_verify_workspace(b, d, vocab, draft_rows, 0, temp, C.byref(n)) == bb.OK and n.value <= ws.numel()
            rc = L.bebelm_verify_drafts(rows.data_ptr(), vocab, rows.data_ptr() if draft_rows else None, vocab, b, d, vocab, 0, temp,
                                        ints.data_ptr(), None, floats.data_ptr(), floats.data_ptr(), out.data_ptr(), acc.data_ptr(),
                                        ws.data_ptr() if n.value else None, n.value, bb.MEM_DEVICE, None)
            if rc != bb.OK:
                bad.append((b, d, bb.last_error()))
    torch.cuda.synchronize()
    assert not bad, (len(bad), bad[:3])


@pytest.mark.parametrize("temp", [1.0, 0.625, 2.5])
@pytest.mark.parametrize("draft_rows", [True, False])
@pytest.mark.parametrize("b,d,v", [(3, 4, 50), (2, 40, 1000), (5, 6, 4099), (40, 3, 9000), (2, 5, 32003), (3, 4, 128000)])
def test_random_numbers_next_to_the_border(b, d, v, draft_rows, temp):
    """u is the f32 next below, at or next above p / q of its draft, so u q and p differ by less than two f32 steps (2^-23 of p), and by
    more than 1e-10 of p (which the inputs' p / q, not themselves f32, are checked for): the decision is that of 64-bit sums."""
    t, tok, u, us, dr = inputs(b, d, v, temp, v + d, draft_rows=draft_rows)
    rng = np.random.default_rng(d)
    for s in range(b):
        for i in range(d):
            x = tok[s, i]
            p, q = softmax64(t[s, i], temp)[x], softmax64(dr[s, i], temp)[x] if draft_rows else 1.0
            # most drafts on the accepted side, so that later ones are reached
            at = np.float32(min(p / q, 0.999))
            side = rng.choice((-2, -1, -1, -1, -1, 0, 1), p=(.2, .2, .2, .15, .15, .05, .05))
            for _ in range(abs(side)):
                at = np.nextafter(at, np.float32(0 if side < 0 else 1))
            u[s, i] = at
            assert abs(float(at) * q / p - 1) > 1e-10
    same(run(t, tok, u, us, dr, temperature=temp), reference(t, tok, u, us, dr, temperature=temp))


@pytest.mark.parametrize("shift", [0.0, 13.7])
@pytest.mark.parametrize("near", [1e-2, 1e-3, 1e-4, 1e-5])
@pytest.mark.parametrize("b,d,v", [(4, 2, 1000), (6, 2, 9000), (40, 1, 20000), (3, 2, 70001), (2, 1, 128000)])
def test_drafts_from_rows_almost_the_targets(b, d, v, near, shift):
    """Draft logits within `near` of the target's, or of those and a constant: p - q is `near` of p, on either side, and its sums have to hold the token's place among v
    all the same. u next to 1 refuses a draft whose p is below q (its smallest p / q is 1 - near or so)."""
    t, tok, u, us, dr = inputs(b, d, v, 1.0, 7 * v + b, near=near)
    dr += np.float32(shift)
    u[:] = np.nextafter(np.float32(1), np.float32(0))
    for s in range(b):
        for i in range(d):  # drafts that are refused, except a few
            tok[s, i] = int((softmax64(t[s, i], 1.0) / softmax64(dr[s, i], 1.0)).argmin()) if (s + i) % 4 else tok[s, i]
    same(run(t, tok, u, us, dr), reference(t, tok, u, us, dr))
