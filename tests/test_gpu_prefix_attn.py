"""Attention over a shared prefix and each sequence's own tail (prefix_attn,
Retriever.window_attn) against a float64 softmax of the stored values.

Tolerance, per output row, from the roundings the operator states (scores f32,
probabilities and quantised values f16, sums f32):
  dS   the error of a scaled score: 2e-6 of scale * sum |q_i k_i| for f32 sums
       of f16 products (the bound the GEMM tests use), 2^-22 of the score for
       forming the exponent; K in quant blocks is rounded to f16 (half a step,
       2^-11 of scale * sum |q_i k_i|);
  out  2 dS (numerator and denominator) + 2^-11 (the probability) + 1e-5 (f32
       sums and joins), all of sum p |v| / sum p; 2^-11 of it more for V in
       quant blocks; 2^-25 |v| a key for probabilities below f16's normal
       range (the largest one is at least 1 before the division); the output's
       own rounding 2^-11 |out| + 2^-25.
  lse  dS + 2e-6 * (1 + |lse|).
Unused cells hold NaN.
"""
import math

import numpy as np
import pytest
import torch

import kvmret
from kvm_helpers import append_history, config_for
from kvmret import synth

pytestmark = pytest.mark.gpu

F16, Q4, Q8 = kvmret.TYPE_F16, kvmret.TYPE_Q4_0, kvmret.TYPE_Q8_0
SIZE = {Q8: 34, Q4: 18}


def values(raw, kind):
    """float64 values of a page buffer [pages][page][hkv * d]."""
    if kind == F16:
        return raw.astype(np.float64).reshape(*raw.shape[:2], -1)
    scale = np.ascontiguousarray(raw[..., :2]).view(np.float16).astype(np.float64)
    body = raw[..., 2:]
    x = (body.view(np.int8).astype(np.float64) if kind == Q8 else
         np.concatenate([body & 15, body >> 4], -1).astype(np.float64) - 8)
    return (scale * x).reshape(*raw.shape[:2], -1)


class Pool:
    """Pages of one kind; every cell unused (NaN) until it is filled."""

    def __init__(self, rng, n, page, hkv, d, kt, vt):
        self.page, self.hkv, self.d, self.kinds = page, hkv, d, (kt, vt)
        self.bufs = []
        for kind in self.kinds:
            if kind == F16:
                b = np.full((n, page, hkv, d), np.nan, np.float16)
            else:
                b = rng.integers(0, 256, (n, page, hkv * d // 32, SIZE[kind])).astype(np.uint8)
                b[..., :2] = np.full(1, np.nan, np.float16).view(np.uint8)
            self.bufs.append(b)
        self.rng = rng

    def fill(self, pages, length, ntok=None):
        """Random values for the tokens of a page list; (k, v) float64
        [tokens][hkv][d]."""
        got = []
        for b, kind in zip(self.bufs, self.kinds):
            rows = []
            for i, p in enumerate(pages):
                n = min(self.page, max(0, length - i * self.page))
                n = n if ntok is None else min(n, ntok[i])
                if n == 0:
                    continue
                if kind == F16:
                    b[p, :n] = self.rng.standard_normal((n, self.hkv, self.d)).astype(np.float16)
                else:
                    top = 127 if kind == Q8 else 8
                    s = ((self.rng.random(b[p, :n].shape[:-1]) + 0.5) * 2 / top).astype(np.float16)
                    b[p, :n, :, :2] = s[..., None].view(np.uint8)
                rows.append(values(b[p:p + 1, :n], kind)[0])
            got.append(np.concatenate(rows).reshape(-1, self.hkv, self.d) if rows else
                       np.zeros((0, self.hkv, self.d)))
        return got

    def device(self):
        k, v = (torch.from_numpy(b).cuda() for b in self.bufs)
        return kvmret.Pages(k, v, self.page, self.hkv, self.d, *self.kinds)


def softmax64(q, k, v, scale, quant_k, quant_v):
    """One row of one head: out, lse and their tolerances."""
    d = q.shape[-1]
    if k.shape[0] == 0:
        return np.zeros(d), -np.inf, np.zeros(d), 0.0
    s = k @ q * scale
    mag = (np.abs(k) @ np.abs(q)) * abs(scale)
    top = s.max()
    p = np.exp(s - top)
    l = p.sum()
    ds = ((2e-6 + (2.0 ** -11 if quant_k else 0)) * mag + 2.0 ** -22 * np.abs(s)).max()
    w = p @ np.abs(v) / l
    out = p @ v / l
    tol = (2 * ds + 2.0 ** -11 + 1e-5 + (2.0 ** -11 if quant_v else 0)) * w + \
        2.0 ** -25 * np.abs(v).sum(0) / l + 2.0 ** -11 * np.abs(out) + 2.0 ** -25
    return out, top + math.log(l), tol, ds + 2e-6 * (1 + abs(top + math.log(l)))


def reference(q, hkv, scale, pre, tails, start, kinds):
    """q: float64 [n][h][d]; pre, tails[s]: (k, v); the rows of every sequence."""
    n, h, d = q.shape
    g = h // hkv
    out, lse = np.zeros((n, h, d)), np.full((n, h), -np.inf)
    tol, ltol = np.zeros((n, h, d)), np.zeros((n, h))
    real = np.zeros(n, bool)
    spans = [(0, n, None)] if tails is None else \
        [(start[s], start[s + 1], t) for s, t in enumerate(tails)]
    for a, b, t in spans:
        for r in range(a, b):
            real[r] = True
            for x in range(h):
                k, v = (pre[i][:, x // g] for i in (0, 1))
                if t is not None:
                    m = max(0, t[0].shape[0] - (b - 1 - r))
                    k = np.concatenate([k, t[0][:m, x // g]])
                    v = np.concatenate([v, t[1][:m, x // g]])
                out[r, x], lse[r, x], tol[r, x], ltol[r, x] = softmax64(
                    q[r, x], k, v, scale, kinds[0] != F16, kinds[1] != F16)
    return out, lse, tol, ltol, real


def check(got, lse, want):
    out, wl, tol, ltol, real = want
    got, lse = got.double().cpu().numpy()[real], lse.double().cpu().numpy()[real]
    err = np.abs(got - out[real])
    assert np.all(err <= tol[real]), (err - tol[real]).max()
    empty = np.isneginf(wl[real])
    assert np.array_equal(np.isneginf(lse), empty)
    assert np.all(np.abs(lse - wl[real])[~empty] <= ltol[real][~empty])


CASES = [
    # new tokens, tail lengths, prefix, hq, hkv, d, prefix page, tail page, kt, vt
    ([1], [1], 1, 1, 1, 64, 16, 16, F16, F16),
    ([1], [5], 0, 8, 2, 128, 128, 16, F16, F16),            # no prefix
    ([1, 1, 1], [1, 40, 129], 130, 8, 2, 128, 128, 32, F16, F16),
    ([1] * 5, [0, 3, 16, 17, 200], 255, 20, 4, 128, 64, 64, F16, F16),  # an empty tail
    ([3, 0, 5, 1], [3, 9, 4, 30], 100, 16, 2, 128, 32, 16, F16, F16),   # a row before its tail
    ([2, 1], [2, 0], 0, 4, 4, 64, 16, 16, F16, F16),        # a row that sees nothing
    ([40], [70], 300, 8, 2, 128, 128, 128, F16, F16),       # rows past one tile
    ([130], [130], 513, 8, 1, 128, 128, 64, F16, F16),
    ([300], [411], 140, 2, 2, 64, 48, 48, F16, F16),        # pages of 48 end inside tiles
    ([7, 6], [144, 20], 700, 16, 4, 256, 144, 16, F16, F16),
    ([20, 3], [33, 66], 257, 16, 2, 256, 128, 128, F16, F16),
    ([1] * 17, list(range(1, 18)), 1000, 8, 8, 64, 16, 32, F16, F16),
    ([1, 4, 2], [1, 100, 64], 333, 8, 2, 128, 128, 32, Q8, Q4),
    ([1, 1], [64, 31], 200, 16, 4, 64, 32, 32, Q8, Q8),
    ([5], [90], 129, 5, 1, 256, 64, 64, Q4, Q4),
    ([2, 2, 2], [2, 200, 70], 150, 8, 2, 128, 48, 16, Q4, F16),
    ([33], [50], 260, 16, 2, 128, 128, 128, F16, Q8),
    ([1] * 40, [9] * 40, 2000, 8, 2, 128, 128, 16, F16, F16),
]


def build(case, seed=0):
    new, tl, prefix, hq, hkv, d, page, tpage, kt, vt = case
    rng = np.random.default_rng(seed + prefix + d + len(new))
    n_pre, width = -(-prefix // page) if prefix else 0, max(1, -(-max(tl) // tpage))
    pool = Pool(rng, n_pre + 2, page, hkv, d, kt, vt)
    tpool = Pool(rng, width * len(new) + 1, tpage, hkv, d, kt, vt)
    table = rng.permutation(n_pre + 2)[:n_pre].astype(np.int32)
    own = rng.permutation(width * len(new) + 1)[:width * len(new)].reshape(len(new), width).astype(
        np.int32)
    pre = pool.fill(table, prefix)
    tails = [tpool.fill(own[s], t) for s, t in enumerate(tl)]
    start = np.concatenate([[0], np.cumsum(new)]).astype(np.int32)
    q = (rng.standard_normal((int(start[-1]), hq, d)) * 1.5).astype(np.float16)
    return pool, tpool, table, own, pre, tails, start, q, np.array(tl, np.int32)


def dev(a):
    return torch.from_numpy(np.ascontiguousarray(a)).cuda()


@pytest.mark.parametrize("case", CASES)
def test_matches_float64(case):
    prefix, hkv, d, kinds = case[2], case[4], case[5], case[8:]
    pool, tpool, table, own, pre, tails, start, q, tl = build(case)
    # rows of no sequence in front of and behind the batch's, strided
    n = q.shape[0]
    rows = torch.full((n + 5, q.shape[1] + 1, d), float("nan"), dtype=torch.float16, device="cuda")
    rows[2:n + 2, :-1] = dev(q)
    out = torch.full((n + 5, q.shape[1], d), 7.0, dtype=torch.float16, device="cuda")
    got, lse = kvmret.prefix_attn(
        rows[:, :-1], pool.device() if prefix else None, dev(np.array([prefix], np.int32)), tpool.device(),
        dev(own), dev(tl), dev(start + 2), prefix_table=dev(table) if prefix else None, lse=True, out=out)
    assert got is out and torch.all(out[:2] == 7) and torch.all(out[n + 2:] == 7)
    want = reference(q.astype(np.float64), hkv, d ** -0.5, pre, tails, start, kinds)
    check(out[2:n + 2], lse[2:n + 2], want)


@pytest.mark.parametrize("n,prefix,hq,hkv,d,page,kt,vt", [
    (1, 1, 1, 1, 128, 16, F16, F16), (3, 127, 8, 2, 64, 128, F16, F16),
    (200, 640, 4, 2, 128, 128, F16, F16), (9, 500, 10, 2, 128, 16, Q8, Q4),
])
def test_prefix_alone(n, prefix, hq, hkv, d, page, kt, vt):
    """No sequences: every row sees the prefix; pages in their own order, the
    length on the host. A length of zero gives zeros."""
    rng = np.random.default_rng(n)
    pool = Pool(rng, -(-prefix // page) + 1, page, hkv, d, kt, vt)
    pre = pool.fill(np.arange(-(-prefix // page)), prefix)
    q = rng.standard_normal((n, hq, d)).astype(np.float16)
    pages = pool.device()
    got, lse = kvmret.prefix_attn(dev(q), pages, None, max_prefix=prefix, lse=True, scale=0.3)
    want = reference(q.astype(np.float64), hkv, 0.3, pre, None, None, (kt, vt))
    check(got, lse, want)
    none, lse = kvmret.prefix_attn(dev(q), pages, torch.zeros(1, dtype=torch.int32, device="cuda"),
                                   max_prefix=prefix, lse=True)
    assert torch.all(none == 0) and torch.all(torch.isneginf(lse))


def test_partly_filled_and_absent_pages():
    """prefix_ntok: pages that hold fewer tokens, in the middle too; page ids
    outside the pool and tail pages of -1 count as pages without tokens;
    lengths past the tables are cut, negative ones are none."""
    rng = np.random.default_rng(5)
    hq, hkv, d, page = 8, 2, 128, 32
    pool, tpool = (Pool(rng, 9, page, hkv, d, F16, F16) for _ in range(2))
    table = np.array([4, 1, 7, 0, 99, 3, -1, 8], np.int32)
    ntok = np.array([32, 5, 0, 31, 32, 32, 32, 7], np.int32)
    held = np.where((table >= 0) & (table < 9), ntok, 0)
    pre = pool.fill(np.where(held > 0, table, 0), 8 * page, held)
    own = np.array([[2, -1, 5], [6, 0, 1], [-1, -1, -1], [4, 7, 8]], np.int32)
    lens = np.array([96, 1000, 3, -4], np.int32)
    tails = []
    for s, (keep, n) in enumerate((([32, 0, 32], 96), ([32] * 3, 96), ([0] * 3, 3), ([0] * 3, 0))):
        k, v = tpool.fill(np.maximum(own[s], 0), n, keep)
        tails.append((k, v))
    start = np.array([0, 1, 2, 3, 4], np.int32)
    q = rng.standard_normal((4, hq, d)).astype(np.float16)
    got, lse = kvmret.prefix_attn(dev(q), pool.device(), None, tpool.device(), dev(own), dev(lens),
                                  dev(start), prefix_table=dev(table), prefix_ntok=dev(ntok), lse=True)
    check(got, lse, reference(q.astype(np.float64), hkv, d ** -0.5, pre, tails, start, (F16, F16)))


@pytest.mark.parametrize("scale", [0.0, -0.7, 40.0])
def test_scores_of_any_size(scale):
    """Equal scores, negative scales, scores in the thousands whose largest
    comes late or early: no overflow, no loss of the sum."""
    rng = np.random.default_rng(8)
    hq, hkv, d, page, n = 4, 1, 128, 64, 900
    pool = Pool(rng, 15, page, hkv, d, F16, F16)
    pre = pool.fill(np.arange(15), n)
    q = rng.standard_normal((6, hq, d)).astype(np.float16)
    got, lse = kvmret.prefix_attn(dev(q), pool.device(), None, max_prefix=n, lse=True, scale=scale)
    check(got, lse, reference(q.astype(np.float64), hkv, scale, pre, None, None, (F16, F16)))


def test_rising_scores():
    """Every tile's scores above the last one's: the running maximum moves all
    the way, in small steps (under a factor of 2^8 a tile) and in large ones."""
    hq, hkv, d, page, n = 8, 2, 128, 128, 2048
    rng = np.random.default_rng(9)
    for step in (0.002, 0.2):
        pool = Pool(rng, 16, page, hkv, d, F16, F16)
        pool.fill(np.arange(16), n)
        ramp = np.arange(n).reshape(16, page)
        pool.bufs[0][..., :] = (0.05 * pool.bufs[0].astype(np.float32)).astype(np.float16)
        pool.bufs[0][..., 0] = (ramp * step)[..., None].astype(np.float16)
        pre = [values(b, F16).reshape(n, hkv, d) for b in pool.bufs]
        q = rng.standard_normal((3, hq, d)).astype(np.float16)
        q[..., 0] = 3.0
        got, lse = kvmret.prefix_attn(dev(q), pool.device(), None, scale=1.0, lse=True)
        check(got, lse, reference(q.astype(np.float64), hkv, 1.0, pre, None, None, (F16, F16)))


def test_far_pages():
    """Pages whose byte offset passes 32 bits, by the list and in order."""
    hq, hkv, d, page, n_pages = 8, 8, 128, 128, 17000  # 256 KiB a page
    k = torch.zeros(n_pages, page, hkv, d, dtype=torch.float16, device="cuda")
    v = torch.zeros(n_pages, page, hkv, d, dtype=torch.float16, device="cuda")
    g = torch.Generator(device="cuda").manual_seed(1)
    at = torch.tensor([16999, 3], device="cuda", dtype=torch.int32)
    k[at.long()] = torch.randn(2, page, hkv, d, device="cuda", generator=g).half()
    v[at.long()] = torch.randn(2, page, hkv, d, device="cuda", generator=g).half()
    q = torch.randn(2, hq, d, device="cuda", generator=g).half()
    big = kvmret.Pages(k, v, page, hkv, d)
    small = kvmret.Pages(k[at.long()], v[at.long()], page, hkv, d)
    args = (torch.tensor([[0], [1]], device="cuda", dtype=torch.int32),
            torch.tensor([100, 128], device="cuda", dtype=torch.int32),
            torch.tensor([0, 1, 2], device="cuda", dtype=torch.int32))
    want = kvmret.prefix_attn(q, small, None, small, *args)
    got = kvmret.prefix_attn(q, big, None, big, at[:, None].contiguous(), *args[1:], prefix_table=at)
    assert torch.equal(got, want)


def test_repeats_bit_for_bit_and_across_streams():
    case = ([1] * 9 + [30], [50] * 9 + [300], 3000, 16, 4, 128, 128, 32, F16, F16)
    pool, tpool, table, own, _, _, start, q, tl = build(case)
    args = (dev(q), pool.device(), dev(np.array([3000], np.int32)), tpool.device(), dev(own), dev(tl),
            dev(start))
    first = kvmret.prefix_attn(*args, prefix_table=dev(table))
    t = dev(table)
    side = [torch.cuda.Stream() for _ in range(3)]
    torch.cuda.synchronize()
    got = []
    for s in side:  # calls under way at once, each with its workspace
        with torch.cuda.stream(s):
            got += [kvmret.prefix_attn(*args, prefix_table=t) for _ in range(3)]
    torch.cuda.synchronize()
    assert all(torch.equal(x, first) for x in got)


def test_captured_call_follows_lengths_and_tables():
    case = ([1, 1, 2], [9, 40, 77], 600, 8, 2, 128, 64, 32, F16, F16)
    pool, tpool, table, own, pre, tails, start, q, tl = build(case)
    pages, tpages = pool.device(), tpool.device()
    qd, length, own_d, tl_d, start_d, table_d = (dev(q), dev(np.array([600], np.int32)), dev(own),
                                                 dev(tl), dev(start), dev(table))
    call = lambda: kvmret.prefix_attn(qd, pages, length, tpages, own_d, tl_d, start_d,  # noqa: E731
                                      prefix_table=table_d, lse=True)
    call()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got, lse = call()
    for cut, lens, at in ((600, [9, 40, 77], start), (33, [1, 40, 12], start), (0, [9, 5, 77], [0, 2, 3, 4])):
        length.fill_(cut)
        tl_d.copy_(torch.tensor(lens, dtype=torch.int32))
        start_d.copy_(torch.tensor(list(at), dtype=torch.int32))
        qd.copy_(torch.randn_like(qd))
        graph.replay()
        torch.cuda.synchronize()
        want = reference(qd.double().cpu().numpy(), 2, 128 ** -0.5, [x[:cut] for x in pre],
                         [(k[:n], v[:n]) for (k, v), n in zip(tails, lens)], list(at), (F16, F16))
        check(got, lse, want)


@pytest.mark.parametrize("quant", [False, True])
def test_step_around_a_window(quant):
    """A step as a user runs it, on one layer's tensors: norms and rotations,
    the retrieval's own append and query, the window, the new tokens of three
    branches filed into their pages, attention over the window and the tails.
    The window's and the pages' bytes give the float64 answer."""
    w = synth.Workload("step", n_layer=2, n_head=8, n_head_kv=2, d_head=128, block_tokens=64,
                       n_blocks=24, budget_blocks=6, sink_blocks=1, reserve_blocks=2, n_planted=3,
                       seed=77)
    kt, vt = (Q8, Q4) if quant else (F16, F16)
    hist = synth.NumpyHistory(w)
    r = kvmret.Retriever(config_for(w, k_type=kt, v_type=vt))
    n0 = w.n_tokens - 41  # a partial newest block
    fn = {}
    if quant:
        def rows(kind):
            return lambda x: kvmret.quantize_f16(dev(x.reshape(-1, w.E)), kind).cpu().numpy().reshape(
                x.shape[0], x.shape[1], -1)
        fn = dict(k_rows_fn=rows(Q8), v_rows_fn=rows(Q4))
    append_history(r, hist, cuts=[], stop=n0, **fn)
    g = torch.Generator(device="cuda").manual_seed(11)
    hq, hkv, d, T = 8, 2, 128, 64
    proj = torch.randn(3, hq + 2 * hkv, d, device="cuda", generator=g).half()
    wq = 1 + 0.1 * torch.randn(d, device="cuda", generator=g)
    fw = d if quant else 0
    # the unrotated queries steer the retrieval
    zero = torch.zeros(3, dtype=torch.int32, device="cuda")
    _, _, q_raw, k_raw = kvmret.qk_norm_rope(proj[:, :hq], proj[:, hq:hq + hkv], zero, wq, wq,
                                             q_rot=False, k_rot=False, q_raw=True, k_raw=True)
    r.query_reset()
    r.query_add(q_raw.reshape(1, 3, -1).expand(w.n_layer, 3, hq * d).contiguous())
    r.score()
    r.select_apply_async()
    # the newest block's tokens beyond what the window's plan saw: gen mode
    # binds it (or a new slot) and writes them in
    ids, st = r.step_collect()
    base = st["total_window_tokens"]
    tails = kvmret.Pages(*(torch.zeros(7, 16 * kvmret.row_bytes(t, hkv * d), dtype=torch.uint8,
                                       device="cuda") for t in (kt, vt)), 16, hkv, d, kt, vt)
    own = torch.tensor([[2, 5], [0, 3], [6, 1]], dtype=torch.int32, device="cuda")
    start = torch.arange(4, dtype=torch.int32, device="cuda")
    lens = torch.zeros(3, dtype=torch.int32, device="cuda")
    for step in range(18):  # past the first page
        pos = base + lens
        cells = own.gather(1, (lens // 16).long()[:, None])[:, 0] * 16 + lens % 16
        proj = torch.randn(3, hq + 2 * hkv, d, device="cuda", generator=g).half()
        q_rot, _, _, k_raw = kvmret.qk_norm_rope(proj[:, :hq], proj[:, hq:hq + hkv], pos, wq, wq,
                                                 fwht_n=fw, k_rot=False, k_raw=True)
        kvmret.paged_append(tails, k_raw, proj[:, hq + hkv:], cells, pos, fwht_n=fw)
        lens += 1
        got, lse = r.window_attn(1, q_rot, tails, own, lens, start, lse=True)
    lay, bases = r.window_layout()
    n_tok = [min(T, n0 - int(b) * T) for b in lay]
    assert sum(n_tok) == base

    def stored(buf, kind):
        return values(buf.view(np.float16) if kind == F16 else buf, kind)

    pre = []
    for is_v, kind in ((False, kt), (True, vt)):
        b = r.window_read(1, is_v, 0, len(lay))
        b = b.view(np.float16).reshape(len(lay), T, -1) if kind == F16 else b.reshape(
            len(lay), T, -1, SIZE[kind])
        x = values(b, kind)
        pre.append(np.concatenate([x[i, :n] for i, n in enumerate(n_tok)]).reshape(-1, hkv, d))
    own_h, tail_vals = own.cpu().numpy(), []
    for s in range(3):
        kv = []
        for buf, kind in ((tails.k, kt), (tails.v, vt)):
            b = buf.cpu().numpy()[own_h[s]]
            b = b.view(np.float16).reshape(2, 16, -1) if kind == F16 else b.reshape(2, 16, -1, SIZE[kind])
            kv.append(values(b, kind).reshape(-1, hkv, d)[:18])
        tail_vals.append(kv)
    want = reference(q_rot.double().cpu().numpy(), hkv, d ** -0.5, pre, tail_vals, [0, 1, 2, 3], (kt, vt))
    check(got, lse, want)
    # a cleared working set: the tails alone
    r.clear_working_set()
    got, lse = r.window_attn(0, q_rot, tails, own, lens, start, lse=True)
    none = [np.zeros((0, hkv, d))] * 2
    check(got, lse, reference(q_rot.double().cpu().numpy(), hkv, d ** -0.5, none, tail_vals, [0, 1, 2, 3],
                              (kt, vt)))
    r.close()


def test_wrapper_refusals():
    z = lambda *s, dt=torch.float16: torch.zeros(*s, dtype=dt, device="cuda")  # noqa: E731
    i = lambda *s: z(*s, dt=torch.int32)  # noqa: E731
    p = kvmret.Pages(z(4, 16, 2, 128), z(4, 16, 2, 128), 16, 2, 128)
    odd = kvmret.Pages(z(4, 12, 2, 128), z(4, 12, 2, 128), 12, 2, 128)
    other = kvmret.Pages(z(4, 16, 4, 64), z(4, 16, 4, 64), 16, 4, 64)
    q = z(3, 4, 128)
    for call in (
            lambda: kvmret.prefix_attn(q.float(), p, None), lambda: kvmret.prefix_attn(z(3, 4, 64), p, None),
            lambda: kvmret.prefix_attn(z(3, 3, 128), p, None), lambda: kvmret.prefix_attn(q, odd, None),
            lambda: kvmret.prefix_attn(q, p, None, max_prefix=65), lambda: kvmret.prefix_attn(q, None, None),
            lambda: kvmret.prefix_attn(q, p, None, p), lambda: kvmret.prefix_attn(q, p, i(2)),
            lambda: kvmret.prefix_attn(q, p, None, p, i(2, 2), i(3), i(3)),
            lambda: kvmret.prefix_attn(q, p, None, other, i(2, 2), i(2), i(3)),
            lambda: kvmret.prefix_attn(q, p, None, out=z(3, 4, 64)),
            lambda: kvmret.prefix_attn(q, p, None, scale=float("nan"))):
        with pytest.raises(kvmret.KvmretError):
            call()
    assert kvmret.prefix_attn(z(0, 4, 128), p, None).shape == (0, 4, 128)


def test_on_a_stream_given_by_its_handle():
    """The stream argument: results as on the current stream, the workspace
    and the outputs kept from other work until that stream has passed."""
    case = ([1] * 6, [30] * 6, 900, 8, 2, 128, 64, 32, F16, F16)
    pool, tpool, table, own, _, _, start, q, tl = build(case)
    args = (dev(q), pool.device(), dev(np.array([900], np.int32)), tpool.device(), dev(own), dev(tl),
            dev(start))
    t = dev(table)
    want = kvmret.prefix_attn(*args, prefix_table=t)
    side = torch.cuda.Stream()
    torch.cuda.synchronize()
    got = []
    for _ in range(8):
        got.append(kvmret.prefix_attn(*args, prefix_table=t, stream=side.cuda_stream))
        torch.full((1 << 22,), float("nan"), device="cuda")  # would take over a freed workspace
    torch.cuda.synchronize()
    assert all(torch.equal(x, want) for x in got)
    pos = torch.arange(6, device="cuda", dtype=torch.int32)
    a = kvmret.qk_norm_rope(args[0], args[0][:, :2], pos, stream=side.cuda_stream)
    torch.cuda.synchronize()
    b = kvmret.qk_norm_rope(args[0], args[0][:, :2], pos)
    assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])


@pytest.mark.parametrize("d,hkv,g,page,kt,vt,rows", [
    (128, 8, 8, 128, F16, F16, 1), (128, 8, 8, 128, F16, F16, 40), (64, 8, 8, 64, F16, F16, 3),
    (256, 4, 8, 128, F16, F16, 9), (128, 8, 8, 128, Q8, Q4, 1), (128, 4, 8, 32, Q8, Q8, 33),
    (64, 8, 8, 128, Q4, Q8, 2), (256, 8, 4, 64, Q8, Q4, 2), (256, 8, 1, 128, Q8, Q8, 5),
    (128, 8, 4, 128, Q8, F16, 3), (64, 8, 8, 64, F16, Q4, 3), (256, 8, 4, 128, F16, Q8, 40),
])
def test_long_prefixes(d, hkv, g, page, kt, vt, rows):
    """Many tiles to a CTA, so that every ring goes round often: 20,000 shared
    tokens, `rows` new tokens of each of three sequences with tails of 1700,
    `rows` and 300 + rows."""
    n_pre, tl = 20000, [1700, rows, 300 + rows]
    rng = np.random.default_rng(d + rows)
    pool = Pool(rng, -(-n_pre // page), page, hkv, d, kt, vt)
    width = -(-max(tl) // page)
    tpool = Pool(rng, 3 * width, page, hkv, d, kt, vt)
    table = rng.permutation(-(-n_pre // page)).astype(np.int32)
    own = rng.permutation(3 * width).reshape(3, width).astype(np.int32)
    pre = pool.fill(table, n_pre)
    tails = [tpool.fill(own[s], t) for s, t in enumerate(tl)]
    q = (rng.standard_normal((3 * rows, hkv * g, d)) * 1.5).astype(np.float16)
    start = np.arange(4, dtype=np.int32) * rows
    got, lse = kvmret.prefix_attn(dev(q), pool.device(), dev(np.array([n_pre], np.int32)), tpool.device(),
                                  dev(own), dev(np.array(tl, np.int32)), dev(start),
                                  prefix_table=dev(table), lse=True)
    qd, scale = dev(q).double(), d ** -0.5
    for s in range(3):
        k, v = (torch.cat([dev(pre[i]), dev(tails[s][i])]) for i in (0, 1))  # [keys][hkv][d]
        total = k.shape[0]
        seen = total - rows + 1 + torch.arange(rows, device="cuda")
        hide = torch.arange(total, device="cuda") >= seen[:, None]
        for h in range(hkv):
            x = qd[s * rows:(s + 1) * rows, h * g:(h + 1) * g]  # [rows][g][d]
            w = (x @ k[:, h].T * scale).masked_fill(hide[:, None], -math.inf)
            mag = (x.abs() @ k[:, h].abs().T * scale).masked_fill(hide[:, None], 0)
            ds = ((2e-6 + (2.0 ** -11 if kt != F16 else 0)) * mag + 2.0 ** -22 *
                  w.masked_fill(hide[:, None], 0).abs()).amax(-1)
            wl = torch.logsumexp(w, -1)
            p = torch.exp(w - wl[..., None])
            want, mass = p @ v[:, h], p @ v[:, h].abs()
            # a probability below f16's normal range, of a largest one of at least 1
            small = 2.0 ** -25 * v[:, h].abs().sum(0) * torch.exp(w.amax(-1) - wl)[..., None]
            tol = (2 * ds[..., None] + 2.0 ** -11 + 1e-5 + (2.0 ** -11 if vt != F16 else 0)) * mass + \
                small + 2.0 ** -11 * want.abs() + 2.0 ** -25
            err = (got[s * rows:(s + 1) * rows, h * g:(h + 1) * g].double() - want).abs()
            assert bool((err <= tol).all()), (s, h, float((err - tol).max()))
            el = (lse[s * rows:(s + 1) * rows, h * g:(h + 1) * g].double() - wl).abs()
            assert bool((el <= ds + 2e-6 * (1 + wl.abs())).all()), (s, h)


@pytest.mark.parametrize("d,kind", [(64, F16), (128, F16), (256, F16), (128, Q8)])
def test_rows_that_are_not_finite_stay_alone(d, kind):
    """An infinite or NaN query row changes no other row."""
    case = ([1, 4, 30], [20, 9, 400], 900, 8, 2, d, 64, 32, kind, kind)
    pool, tpool, table, own, _, _, start, q, tl = build(case)
    bad = np.array([2, 7, 34])
    args = [pool.device(), dev(np.array([900], np.int32)), tpool.device(), dev(own), dev(tl), dev(start)]
    want, lse = kvmret.prefix_attn(dev(q), *args, prefix_table=dev(table), lse=True)
    q[bad[0], :, 5] = np.nan
    q[bad[1], :, 0] = np.inf
    q[bad[2], :, d - 1] = -np.inf
    got, lse2 = kvmret.prefix_attn(dev(q), *args, prefix_table=dev(table), lse=True)
    good = np.setdiff1d(np.arange(q.shape[0]), bad)
    assert torch.equal(got[good], want[good]) and torch.equal(lse2[good], lse[good])
    assert not torch.isfinite(got[bad].float()).any()


def test_descending_starts_leave_nan():
    """Row starts that descend cannot be walked: the rows from the first start to
    the last are NaN, the others as they were, and the next call is right."""
    case = ([2, 2, 2], [9, 40, 77], 600, 8, 2, 128, 64, 32, F16, F16)
    pool, tpool, table, own, pre, tails, start, q, tl = build(case)
    rows = torch.zeros((8, 8, 128), dtype=torch.float16, device="cuda")
    rows[1:7] = dev(q)
    out = torch.full_like(rows, 7.0)
    args = [pool.device(), dev(np.array([600], np.int32)), tpool.device(), dev(own), dev(tl)]
    kw = dict(prefix_table=dev(table), lse=True)
    _, lse = kvmret.prefix_attn(rows, *args, dev(np.array([1, 5, 3, 7], np.int32)), out=out, **kw)
    assert torch.isnan(out[1:7]).all() and torch.isnan(lse[1:7]).all()
    assert torch.all(out[0] == 7) and torch.all(out[7] == 7)
    _, lse = kvmret.prefix_attn(rows, *args, dev(start + 1), out=out, **kw)
    check(out[1:7], lse[1:7], reference(q.astype(np.float64), 2, 128 ** -0.5, pre, tails, start, (F16, F16)))


@pytest.mark.parametrize("kind", [F16, Q8])
def test_pages_named_more_than_once(kind):
    """The same page twice in the prefix and in the tails of several sequences."""
    rng = np.random.default_rng(3)
    pool = Pool(rng, 3, 32, 2, 128, kind, kind)
    pool.fill(np.arange(3), 96)
    k, v = (values(b, kind).reshape(3, 32, 2, 128) for b in pool.bufs)
    table, own = np.array([1, 1, 0, 1], np.int32), np.array([[2, 2], [2, 0]], np.int32)
    tl, start = np.array([40, 50], np.int32), np.array([0, 3, 5], np.int32)
    q = rng.standard_normal((5, 8, 128)).astype(np.float16)
    pages = pool.device()
    got, lse = kvmret.prefix_attn(dev(q), pages, dev(np.array([120], np.int32)), pages, dev(own), dev(tl),
                                  dev(start), prefix_table=dev(table), lse=True)
    pre = [x[table].reshape(-1, 2, 128)[:120] for x in (k, v)]
    tails = [[x[own[s]].reshape(-1, 2, 128)[:tl[s]] for x in (k, v)] for s in range(2)]
    check(got, lse, reference(q.astype(np.float64), 2, 128 ** -0.5, pre, tails, start, (kind, kind)))


def test_two_graphs_at_once():
    """Two captured calls over one cache, replayed at the same time again and
    again, each on a stream of its own."""
    case = ([1] * 6, [50] * 6, 5000, 16, 4, 128, 128, 32, Q8, F16)
    pool, tpool, table, own, _, _, start, q, tl = build(case)
    args = (pool.device(), dev(np.array([5000], np.int32)), tpool.device(), dev(own), dev(tl), dev(start))
    t = dev(table)
    qs = [dev(q), dev(q[::-1].copy())]
    want = [kvmret.prefix_attn(x, *args, prefix_table=t) for x in qs]
    graphs, outs = [], []
    for x in qs:
        graphs.append(torch.cuda.CUDAGraph())
        with torch.cuda.graph(graphs[-1]):
            outs.append(kvmret.prefix_attn(x, *args, prefix_table=t))
    side = [torch.cuda.Stream() for _ in qs]
    torch.cuda.synchronize()
    for _ in range(20):
        for g, s in zip(graphs, side):
            with torch.cuda.stream(s):
                g.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(outs, want))


@pytest.mark.parametrize("d,pre_kinds,tail_kinds", [
    (128, (Q8, Q4), (F16, F16)), (128, (F16, F16), (Q4, Q8)), (64, (Q4, F16), (F16, Q8)),
    (256, (F16, Q8), (Q8, F16)), (256, (Q8, Q8), (F16, F16)),
])
def test_prefix_and_tails_of_different_types(d, pre_kinds, tail_kinds):
    """A quantised window with tails in f16 and other mixtures: tiles that are
    converted and tiles that are copied alternate in one CTA's order."""
    rng = np.random.default_rng(d)
    new, tl, n_pre, hq, hkv = [1, 4, 20], [300, 150, 40], 1300, 16, 4
    pool, tpool = Pool(rng, 12, 128, hkv, d, *pre_kinds), Pool(rng, 30, 32, hkv, d, *tail_kinds)
    table = rng.permutation(12)[:11].astype(np.int32)
    own = rng.permutation(30).reshape(3, 10).astype(np.int32)
    pre = pool.fill(table, n_pre)
    tails = [tpool.fill(own[s], t) for s, t in enumerate(tl)]
    start = np.concatenate([[0], np.cumsum(new)]).astype(np.int32)
    q = (rng.standard_normal((25, hq, d)) * 1.5).astype(np.float16)
    got, lse = kvmret.prefix_attn(dev(q), pool.device(), dev(np.array([n_pre], np.int32)), tpool.device(),
                                  dev(own), dev(np.array(tl, np.int32)), dev(start),
                                  prefix_table=dev(table), lse=True)
    check(got, lse, reference(q.astype(np.float64), hkv, d ** -0.5, pre, tails, start, (Q8, Q8)))


def test_many_sequences():
    """A thousand sequences, some without rows or without tokens, over no prefix
    and over a short one: more than the split looks at in one go."""
    rng = np.random.default_rng(8)
    n, hq, hkv, d = 1000, 4, 2, 64
    new, tl = rng.integers(0, 3, n), rng.integers(0, 40, n)
    tpool = Pool(rng, 3 * n, 16, hkv, d, F16, F16)
    own = rng.permutation(3 * n).reshape(n, 3).astype(np.int32)
    tails = [tpool.fill(own[s], int(t)) for s, t in enumerate(tl)]
    start = np.concatenate([[0], np.cumsum(new)]).astype(np.int32)
    q = rng.standard_normal((int(start[-1]), hq, d)).astype(np.float16)
    pool = Pool(rng, 5, 16, hkv, d, F16, F16)
    for n_pre in (0, 70):
        pre = pool.fill(np.arange(5), n_pre)
        got, lse = kvmret.prefix_attn(dev(q), pool.device() if n_pre else None,
                                      dev(np.array([n_pre], np.int32)) if n_pre else None, tpool.device(),
                                      dev(own), dev(tl.astype(np.int32)), dev(start), lse=True)
        check(got, lse, reference(q.astype(np.float64), hkv, d ** -0.5, pre, tails, start, (F16, F16)))


def check_rows(got, lse, q, spans, hkv, quant_k, quant_v):
    """Rows against a float64 softmax on the GPU: spans of (first row, end, k, v), the
    keys [tokens][hkv][d] that the span's last row sees, one fewer the row before."""
    scale, g = q.shape[-1] ** -0.5, q.shape[1] // hkv
    qd = q.double()
    for a, b, k, v in spans:
        hide = torch.arange(k.shape[0], device="cuda") >= \
            (k.shape[0] - (b - a) + 1 + torch.arange(b - a, device="cuda"))[:, None]
        for h in range(hkv):
            x, kh, vh = qd[a:b, h * g:(h + 1) * g].transpose(0, 1), k[:, h], v[:, h]  # [g][rows][d]
            w = (x @ kh.T * scale).masked_fill(hide, -math.inf)
            mag = (x.abs() @ kh.abs().T * scale).masked_fill(hide, 0)
            ds = ((2e-6 + (2.0 ** -11 if quant_k else 0)) * mag + 2.0 ** -22 *
                  w.masked_fill(hide, 0).abs()).amax(-1)
            wl = torch.logsumexp(w, -1)
            p = torch.exp(w - wl[..., None])
            want, mass = p @ vh, p @ vh.abs()
            small = 2.0 ** -25 * vh.abs().sum(0) * torch.exp(w.amax(-1) - wl)[..., None]
            tol = (2 * ds[..., None] + 2.0 ** -11 + 1e-5 + (2.0 ** -11 if quant_v else 0)) * mass + \
                small + 2.0 ** -11 * want.abs() + 2.0 ** -25
            err = (got[a:b, h * g:(h + 1) * g].transpose(0, 1).double() - want).abs()
            assert bool((err <= tol).all()), (a, h, float((err - tol).max()))
            el = (lse[a:b, h * g:(h + 1) * g].T.double() - wl).abs()
            assert bool((el <= ds + 2e-6 * (1 + wl.abs())).all()), (a, h)


@pytest.mark.parametrize("d,pre_kinds,tail_kinds", [
    (256, (Q8, F16), (Q8, F16)), (256, (F16, Q8), (Q4, F16)), (128, (Q8, F16), (F16, Q4)),
    (128, (F16, Q4), (F16, F16)), (64, (F16, Q8), (Q8, F16)), (64, (Q4, F16), (Q4, F16)),
])
def test_long_lists_with_one_operand_in_f16(d, pre_kinds, tail_kinds):
    """Tiles whose K or V is copied, by the dozen to a CTA, the copied operand changing
    on the way: every ring of the conversion goes round often. Again and again, with
    the same bits."""
    rng = np.random.default_rng(d + 1)
    n, hkv, g, n_pre = 40, 4, 8, 12000
    tl = rng.integers(500, 900, n)
    pool = Pool(rng, -(-n_pre // 128), 128, hkv, d, *pre_kinds)
    width = -(-int(tl.max()) // 64)
    tpool = Pool(rng, n * width, 64, hkv, d, *tail_kinds)
    table = rng.permutation(-(-n_pre // 128)).astype(np.int32)
    own = rng.permutation(n * width).reshape(n, width).astype(np.int32)
    pre = [dev(x) for x in pool.fill(table, n_pre)]
    tails = [[dev(x) for x in tpool.fill(own[s], int(t))] for s, t in enumerate(tl)]
    q = dev((rng.standard_normal((n, hkv * g, d)) * 1.5).astype(np.float16))
    args = (q, pool.device(), dev(np.array([n_pre], np.int32)), tpool.device(), dev(own),
            dev(tl.astype(np.int32)), dev(np.arange(n + 1, dtype=np.int32)))
    t = dev(table)
    got, lse = kvmret.prefix_attn(*args, prefix_table=t, lse=True)
    spans = [(s, s + 1, torch.cat([pre[0], tails[s][0]]), torch.cat([pre[1], tails[s][1]]))
             for s in range(n)]
    check_rows(got, lse, q, spans, hkv, True, True)
    for _ in range(20):
        assert torch.equal(kvmret.prefix_attn(*args, prefix_table=t), got)


def test_a_given_stream_takes_no_memory_still_in_use():
    """With a stream given by its handle, outputs and workspace come from that stream's
    memory: what was freed on the current stream may have work before it there."""
    case = ([1] * 6, [30] * 6, 900, 8, 2, 128, 64, 32, F16, F16)
    pool, tpool, table, own, _, _, start, q, tl = build(case)
    args = (dev(q), pool.device(), dev(np.array([900], np.int32)), tpool.device(), dev(own), dev(tl),
            dev(start))
    t, pos = dev(table), torch.arange(6, device="cuda", dtype=torch.int32)
    want = kvmret.prefix_attn(*args, prefix_table=t)
    want_qk = kvmret.qk_norm_rope(args[0], args[0][:, :2], pos)
    side = torch.cuda.Stream()
    sizes = (want.numel() * 2, int(kvmret.lib.kvmret_prefix_attn_ws_bytes(6, 8, 2, 128, 6)),
             want_qk[1].numel() * 2)
    torch.cuda.synchronize()
    torch.cuda.empty_cache()
    torch.cuda._sleep(200_000_000)  # the current stream is busy for a tenth of a second
    freed = [torch.full((n,), 255, dtype=torch.uint8, device="cuda") for n in sizes for _ in range(4)]
    spans = [(x.data_ptr(), x.numel()) for x in freed]
    del freed
    got = kvmret.prefix_attn(*args, prefix_table=t, stream=side.cuda_stream)
    got_qk = kvmret.qk_norm_rope(args[0], args[0][:, :2], pos, stream=side.cuda_stream)
    for x in (got, got_qk[0], got_qk[1]):
        assert all(x.data_ptr() + x.numel() * 2 <= a or x.data_ptr() >= a + n for a, n in spans)
    torch.cuda.synchronize()
    assert torch.equal(got, want)
    assert torch.equal(got_qk[0], want_qk[0]) and torch.equal(got_qk[1], want_qk[1])


@pytest.mark.parametrize("absent", [False, True])
def test_length_counts_the_tokens_of_partly_filled_pages(absent):
    """prefix_len and max_prefix with prefix_ntok: the first tokens that the pages
    hold, wherever a page ends; pages without tokens, and page ids outside the pool,
    hold none. More pages than the split looks at in one go."""
    rng = np.random.default_rng(21)
    hq, hkv, d, page, n = 4, 2, 128, 32, 45
    pool = Pool(rng, n, page, hkv, d, F16, F16)
    table = rng.permutation(n).astype(np.int32)
    ntok = rng.integers(0, page + 1, n).astype(np.uint32)
    ntok[:2], ntok[7], ntok[40] = (5, page), 0, page + 9  # (what is past a page does not count)
    there = np.minimum(ntok, page).astype(np.int32)
    pre = pool.fill(table, n * page, there)
    if absent:  # the filled values of these pages are no longer listed
        keep = np.ones(n, bool)
        keep[[3, 33]] = False
        lost = np.repeat(~keep, there)
        pre = [x[~lost] for x in pre]
        table[3], table[33], there = -1, n, there * keep
    total = int(there.sum())
    q = rng.standard_normal((3, hq, d)).astype(np.float16)
    pages, qd, t, nt = pool.device(), dev(q), dev(table), dev(ntok.view(np.int32))
    length = torch.zeros(1, dtype=torch.int32, device="cuda")
    edges = np.cumsum(there)
    for m in sorted({0, 1, 4, 5, 6, 36, 37, 38, int(edges[2]), int(edges[2]) + 1, int(edges[31]),
                     int(edges[31]) + 1, int(edges[40]) - 1, total - 1, total, total + 1, n * page}):
        want = reference(q.astype(np.float64), hkv, d ** -0.5, [x[:m] for x in pre], None, None,
                         (F16, F16))
        length.fill_(m)
        check(*kvmret.prefix_attn(qd, pages, length, prefix_table=t, prefix_ntok=nt, lse=True), want)
        if m:
            for longest in (None, torch.full_like(length, m + 3)):
                check(*kvmret.prefix_attn(qd, pages, longest, prefix_table=t, prefix_ntok=nt,
                                          max_prefix=m, lse=True), want)


@pytest.mark.parametrize("case", [
    ([1], [40], 20000, 64, 8, 128, 128, 32, F16, F16),
    ([1] * 300, [17] * 300, 0, 8, 2, 128, 128, 16, F16, F16),
    ([1, 3] * 40, [90, 5] * 40, 700, 12, 4, 64, 64, 16, F16, F16),
    ([5, 2, 60], [500, 2, 60], 900, 7, 1, 256, 64, 64, F16, F16),
    ([1] * 70, [70] * 70, 300, 16, 2, 128, 32, 32, Q8, Q4),
    ([400, 3], [600, 3], 200, 16, 2, 128, 128, 64, F16, F16),
    ([400, 3], [600, 3], 0, 16, 4, 64, 64, 64, Q8, Q8),
])
def test_workspace_is_kept_to_and_need_not_be_clean(case, monkeypatch):
    """Nothing outside the workspace is written, and what it held before does not matter."""
    pool, tpool, table, own, _, _, start, q, tl = build(case)
    prefix = case[2]
    args = (dev(q), pool.device() if prefix else None, dev(np.array([prefix], np.int32)), tpool.device(),
            dev(own), dev(tl), dev(start))
    kw = dict(prefix_table=dev(table) if prefix else None, lse=True)
    want, lse = kvmret.prefix_attn(*args, **kw)
    room, held = 16 << 20, []

    def workspace(shape, n_head_kv, n_seq, device):
        nb = int(kvmret.lib.kvmret_prefix_attn_ws_bytes(shape[0], shape[1], n_head_kv, shape[2], n_seq))
        held.append(torch.full((nb + 2 * room,), 0xa5, dtype=torch.uint8, device=device))
        held[-1][room:room + nb] = 0xff
        return held[-1][room:room + nb], nb

    monkeypatch.setattr(kvmret, "_attn_ws", workspace)
    got, lse2 = kvmret.prefix_attn(*args, **kw)
    assert torch.equal(got, want) and torch.equal(lse2, lse)
    assert bool((held[0][:room] == 0xa5).all()) and bool((held[0][-room:] == 0xa5).all())


def test_window_attention_is_counted_among_the_launches():
    w = synth.Workload("count", n_layer=1, n_head=4, n_head_kv=2, d_head=128, block_tokens=64,
                       n_blocks=8, budget_blocks=4, sink_blocks=1, reserve_blocks=1, n_planted=1, seed=5)
    r = kvmret.Retriever(config_for(w))
    append_history(r, synth.NumpyHistory(w), cuts=[])
    r.prof_enable()
    q = torch.zeros(3, 4, 128, dtype=torch.float16, device="cuda")
    tails = kvmret.Pages(*(torch.zeros(1, 16, 2, 128, dtype=torch.float16, device="cuda") for _ in "kv"),
                         16, 2, 128)
    ones = torch.zeros(1, 1, dtype=torch.int32, device="cuda")
    args = (tails, ones, torch.ones(1, dtype=torch.int32, device="cuda"))
    r.window_attn(0, q, *args, torch.tensor([0, 3], dtype=torch.int32, device="cuda"))
    r.window_attn(0, q[:0], *args, torch.zeros(2, dtype=torch.int32, device="cuda"))
    assert r.prof_read()["launches"] == 2
    r.close()


@pytest.mark.parametrize("d,g,new,n_pre,kt,vt", [
    (128, 8, [345], 0, F16, F16), (128, 8, [345], 3000, F16, F16),      # 11 units of 256 rows: groups of 6
    (64, 8, [300, 45], 1100, F16, F16), (128, 8, [345], 0, Q8, Q4),      # 22 units of 128: groups of 8
    (128, 8, [40, 305], 2100, Q8, Q4), (256, 5, [403], 1500, F16, F16),  # 16: groups of 8
    (256, 5, [403], 0, Q4, Q8), (64, 4, [1100], 700, Q8, F16),           # 35: groups of 7
])
def test_chunks_of_many_units(d, g, new, n_pre, kt, vt):
    """More than eight units of rows a KV head: groups of SMs walk the prefix side by
    side, the last group not always full, and causality cuts each unit's tail elsewhere."""
    rng = np.random.default_rng(d + g + n_pre)
    hkv, page = 4, 64
    tl = [n + 150 * s for s, n in enumerate(new)]
    pool = Pool(rng, -(-n_pre // page) + 1, page, hkv, d, kt, vt)
    width = -(-max(tl) // page)
    tpool = Pool(rng, len(new) * width, page, hkv, d, kt, vt)
    table = rng.permutation(-(-n_pre // page) + 1)[:-(-n_pre // page)].astype(np.int32)
    own = rng.permutation(len(new) * width).reshape(len(new), width).astype(np.int32)
    pre = [dev(x) for x in pool.fill(table, n_pre)]
    tails = [[dev(x) for x in tpool.fill(own[s], t)] for s, t in enumerate(tl)]
    start = np.concatenate([[0], np.cumsum(new)]).astype(np.int32)
    q = dev((rng.standard_normal((int(start[-1]), hkv * g, d)) * 1.5).astype(np.float16))
    got, lse = kvmret.prefix_attn(q, pool.device() if n_pre else None,
                                  dev(np.array([n_pre], np.int32)) if n_pre else None, tpool.device(),
                                  dev(own), dev(np.array(tl, np.int32)), dev(start),
                                  prefix_table=dev(table) if n_pre else None, lse=True)
    spans = [(int(start[s]), int(start[s + 1]), torch.cat([pre[0], tails[s][0]]),
              torch.cat([pre[1], tails[s][1]])) for s in range(len(new))]
    check_rows(got, lse, q, spans, hkv, kt != F16, vt != F16)


def test_a_thousand_heads_to_a_kv_head():
    rng = np.random.default_rng(12)
    pool, tpool = Pool(rng, 3, 64, 1, 64, F16, F16), Pool(rng, 2, 64, 1, 64, F16, F16)
    pre, tail = [dev(x) for x in pool.fill(np.arange(3), 150)], [dev(x) for x in tpool.fill([0, 1], 70)]
    q = dev((rng.standard_normal((3, 1000, 64)) * 1.5).astype(np.float16))
    got, lse = kvmret.prefix_attn(q, pool.device(), None, tpool.device(), dev(np.array([[0, 1]], np.int32)),
                                  dev(np.array([70], np.int32)), dev(np.array([0, 3], np.int32)),
                                  max_prefix=150, lse=True)
    check_rows(got, lse, q, [(0, 3, torch.cat([pre[0], tail[0]]), torch.cat([pre[1], tail[1]]))], 1,
               False, False)


def test_the_most_sequences():
    """65,535 sequences of one row: tails of 0 to 16 tokens, pages shared by many."""
    rng = np.random.default_rng(13)
    n, hq, hkv, d, n_pages = 65535, 4, 2, 64, 500
    pool = Pool(rng, n_pages, 16, hkv, d, F16, F16)
    k, v = (dev(x).view(n_pages, 16, hkv, d) for x in pool.fill(np.arange(n_pages), 16 * n_pages))
    own, tl = dev(rng.integers(0, n_pages, (n, 1)).astype(np.int32)), dev(rng.integers(0, 17, n).astype(np.int32))
    q = torch.randn(n, hq, d, device="cuda").half()
    got, lse = kvmret.prefix_attn(q, None, None, pool.device(), own, tl,
                                  torch.arange(n + 1, dtype=torch.int32, device="cuda"), lse=True)
    hide = (torch.arange(16, device="cuda") >= tl[:, None])[:, None]  # [n][1][16]
    for h in range(hq):
        kh, vh = (x[own[:, 0].long(), :, h // 2] for x in (k, v))  # [n][16][d]
        x = q[:, h].double()
        w = torch.einsum("nd,nkd->nk", x, kh) * d ** -0.5
        mag = torch.einsum("nd,nkd->nk", x.abs(), kh.abs()) * d ** -0.5
        w = w.masked_fill(hide[:, 0], -math.inf)
        top = w.amax(-1, keepdim=True).clamp(min=-1e300)
        p = torch.exp(w - top)
        total = p.sum(-1, keepdim=True)
        ds = ((2e-6 + 2.0 ** -22) * mag).amax(-1, keepdim=True)
        seen = torch.where(total > 0, total, 1.0)
        want = torch.einsum("nk,nkd->nd", p, vh) / seen
        mass = torch.einsum("nk,nkd->nd", p, vh.abs()) / seen
        tol = (2 * ds + 2.0 ** -11 + 1e-5) * mass + 2.0 ** -25 * vh.abs().sum(1) / seen + \
            2.0 ** -11 * want.abs() + 2.0 ** -25
        assert bool(((got[:, h].double() - want).abs() <= tol).all())
        empty = tl == 0
        assert torch.equal(torch.isneginf(lse[:, h]), empty) and bool((got[empty] == 0).all())
        wl = (top + torch.log(seen))[~empty, 0]
        assert bool(((lse[~empty, h].double() - wl).abs() <= ds[~empty, 0] + 2e-6 * (1 + wl.abs())).all())


@pytest.mark.parametrize("kt,vt", [(F16, F16), (Q8, Q4), (Q8, F16)])
def test_pages_between_others(kt, vt):
    """K and V of several layers in one buffer, a page of each after another: the strides
    of the pages, for the prefix and the tails, give what dense pages give."""
    case = ([1, 3, 2], [40, 77, 9], 700, 8, 2, 128, 48, 32, kt, vt)
    pool, tpool, table, own, _, _, start, q, tl = build(case)
    args = (dev(np.array([700], np.int32)), dev(own), dev(tl), dev(start))
    dense, tdense = pool.device(), tpool.device()

    def spread(p):
        k, v = (x.flatten(1).view(torch.uint8) for x in (p.k, p.v))
        both = torch.full((p.n_pages, k.shape[1] + v.shape[1] + 96), 0xff, dtype=torch.uint8, device="cuda")
        a, b = both[:, 32:32 + k.shape[1]], both[:, -v.shape[1] - 16:-16]
        a.copy_(k)
        b.copy_(v)
        return kvmret.Pages(a, b, p.page_tokens, 2, 128, kt, vt)

    want = kvmret.prefix_attn(dev(q), dense, args[0], tdense, *args[1:], prefix_table=dev(table), lse=True)
    got = kvmret.prefix_attn(dev(q), spread(dense), args[0], spread(tdense), *args[1:],
                             prefix_table=dev(table), lse=True)
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])


@pytest.mark.parametrize("d,kt,vt", [(64, F16, F16), (128, Q8, Q4), (256, F16, Q8)])
def test_contiguous_caches_as_one_page(d, kt, vt):
    """A cache that is not paged: one page for the prefix, one for each tail."""
    case = ([3, 1, 40], [900, 17, 1040], 4000, 12, 4, d, 4112, 1040, kt, vt)
    pool, tpool, table, own, pre, tails, start, q, tl = build(case)
    got, lse = kvmret.prefix_attn(dev(q), pool.device(), dev(np.array([4000], np.int32)), tpool.device(),
                                  dev(own), dev(tl), dev(start), prefix_table=dev(table), lse=True)
    spans = [(int(start[s]), int(start[s + 1]), *(torch.cat([dev(pre[i]), dev(tails[s][i])]) for i in (0, 1)))
             for s in range(3)]
    check_rows(got, lse, dev(q), spans, 4, kt != F16, vt != F16)


def test_calls_from_threads():
    """Several host threads at once, each on a stream of its own."""
    import threading
    cases = [([1] * 5, [50] * 5, 900, 8, 2, d, 64, 32, *kinds)
             for d, kinds in ((64, (F16, F16)), (128, (Q8, Q4)), (256, (F16, F16)), (128, (F16, F16)))]
    work, got = [], {}
    for case in cases:
        pool, tpool, table, own, _, _, start, q, tl = build(case)
        work.append(((dev(q), pool.device(), dev(np.array([900], np.int32)), tpool.device(), dev(own),
                      dev(tl), dev(start)), dev(table)))
    torch.cuda.synchronize()

    def run(i):
        s = torch.cuda.Stream()
        with torch.cuda.stream(s):
            got[i] = [kvmret.prefix_attn(*work[i][0], prefix_table=work[i][1]) for _ in range(30)]
        s.synchronize()

    threads = [threading.Thread(target=run, args=(i,)) for i in range(len(cases))]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    for i, (args, table) in enumerate(work):
        want = kvmret.prefix_attn(*args, prefix_table=table)
        assert len(got[i]) == 30 and all(torch.equal(x, want) for x in got[i])


def test_captured_window_attention():
    """A call over a context's window in a graph: replays follow the window that later
    steps build, and the tails' lengths."""
    w = synth.Workload("graph", n_layer=2, n_head=8, n_head_kv=2, d_head=128, block_tokens=64,
                       n_blocks=24, budget_blocks=6, sink_blocks=1, reserve_blocks=2, n_planted=3, seed=9)
    r = kvmret.Retriever(config_for(w))
    append_history(r, synth.NumpyHistory(w), cuts=[])
    g = torch.Generator(device="cuda").manual_seed(4)
    q = torch.randn(3, 8, 128, device="cuda", generator=g).half()
    tails = kvmret.Pages(*(torch.randn(4, 16, 2, 128, device="cuda", generator=g).half() for _ in "kv"),
                         16, 2, 128)
    own = torch.tensor([[0], [2], [3]], dtype=torch.int32, device="cuda")
    lens = torch.tensor([1, 9, 16], dtype=torch.int32, device="cuda")
    start = torch.arange(4, dtype=torch.int32, device="cuda")

    def step(seed):
        rows = torch.randn(2, 1, 8 * 128, device="cuda", generator=torch.Generator(device="cuda").manual_seed(seed))
        r.query_reset()
        r.query_add(rows.half())
        r.score()
        r.select_apply_async()
        r.step_collect()

    step(1)
    r.window_attn(1, q, tails, own, lens, start)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held, lse = r.window_attn(1, q, tails, own, lens, start, lse=True)
    seen = []
    for seed in (1, 2, 3):
        step(seed)
        lens += 0 if seed == 1 else -1
        lens.clamp_(min=0)
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        want, wl = r.window_attn(1, q, tails, own, lens, start, lse=True)
        assert torch.equal(held, want) and torch.equal(lse, wl)
        seen.append(held.clone())
    assert not torch.equal(seen[0], seen[1])
    r.close()
