"""Head norms with the position rotation (qk_norm_rope) and the append to a
paged cache (paged_append).

References are in 64 bits, with the operators' own float32 angle (position *
theta_i rounded to float, as the library's other rotations define it). The
tolerances are derived, u = 2^-24 the unit of float, 2^-11 f16's half step,
2^-25 half a step of f16's subnormals:

- normed row: the sum of squares rounds at most 16 products and sums a lane
  and 4 shuffled sums, all of one sign: 21 u relative, halved by the root;
  mean, eps, root, two products: 5 u more. |err| <= 16 u |y| before the f16
  rounding.
- rotated pair: a c - b s with a, b off by 16 u, c and s by u, two products
  and a sum rounded: |err| <= 20 u (|a c| + |b s|).
- Hadamard: a sum of D such values / sqrt(D), each through 1 scaling (2 u with
  the scale's own rounding) and log2 D <= 8 sums: |err| <= 31 u sum |z| / sqrt(D).
The appended rows are compared bit for bit: every step is one defined rounding.
"""
import numpy as np
import pytest
import torch

import kvmret
import pyoracle as po

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
DT = {"f16": torch.float16, "bf16": torch.bfloat16, "f32": torch.float32}


def angle64(pos, d, base=1e6, scale=1.0):
    theta = po.rope_theta(d, base, scale)
    ang = (pos.astype(np.float32)[:, None] * theta[None].astype(np.float32)).astype(np.float32)
    return np.cos(ang.astype(np.float64)), np.sin(ang.astype(np.float64))


def rope64(x, c, s):
    h = x.shape[-1] // 2
    a, b = x[..., :h], x[..., h:]
    c, s = c[:, None], s[:, None]
    z = np.concatenate([a * c - b * s, a * s + b * c], -1)
    mag = np.concatenate([abs(a * c) + abs(b * s), abs(a * s) + abs(b * c)], -1)
    return z, mag


def hadamard64(n):
    i = np.arange(n)
    bits = np.array([[bin(a & b).count("1") & 1 for b in i] for a in i])
    return (1.0 - 2.0 * bits) / np.sqrt(n)


def close(got, want, before):
    """got (f16) within its own rounding of want, itself off by `before`; NaN
    where want is (a row scaled past f16's range holds infinities)."""
    got = got.double().cpu().numpy()
    assert np.array_equal(np.isnan(got), np.isnan(want))
    err = np.abs(got - want)
    tol = before * (1 + 2.0 ** -11) + np.abs(want) * 2.0 ** -11 + 2.0 ** -25
    fine = ~np.isnan(want)
    assert np.all(err[fine] <= tol[fine]), (err[fine] / tol[fine]).max()


@pytest.mark.parametrize("n,hq,hkv,d,dt,fwht,strided", [
    (1, 64, 8, 128, "f16", False, False), (1, 1, 1, 64, "f32", True, True),
    (3, 5, 1, 256, "bf16", True, True), (8, 32, 8, 128, "f32", True, False),
    (33, 8, 2, 64, "bf16", False, True), (130, 20, 4, 128, "f16", True, True),
    (301, 6, 3, 256, "f16", False, True), (700, 40, 8, 128, "bf16", False, True),
])
def test_qk_norm_rope(n, hq, hkv, d, dt, fwht, strided):
    g = torch.Generator(device="cuda").manual_seed(n * 7 + d)
    rows = (torch.randn(n, hq + 2 * hkv + (3 if strided else 0), d, device="cuda", generator=g) *
            torch.exp(torch.randn(n, 1, 1, device="cuda", generator=g) * 3)).to(DT[dt])
    q, k = rows[:, :hq], rows[:, hq:hq + hkv]
    if not strided:
        q, k = q.contiguous(), k.contiguous()
    rows[0, 0] = 0  # a head of zeros: eps alone under the root
    wq = 1 + 0.3 * torch.randn(d, device="cuda", generator=g)
    wk = 1 + 0.3 * torch.randn(d, device="cuda", generator=g)
    pos = torch.randint(0, 262144, (n,), device="cuda", generator=g, dtype=torch.int32)
    eps = 1e-5
    got = kvmret.qk_norm_rope(q, k, pos, wq, wk, eps=eps, fwht_n=d if fwht else 0, q_raw=True,
                              k_raw=True)
    c, s = angle64(pos.cpu().numpy(), d)
    for x, w, rot, raw in ((q, wq, got[0], got[2]), (k, wk, got[1], got[3])):
        x = x.double().cpu().numpy()
        y = x / np.sqrt((x * x).mean(-1, keepdims=True) + np.float32(eps)) * w.double().cpu().numpy()
        close(raw, y, 16 * U * np.abs(y))
        z, mag = rope64(y, c, s)
        if fwht:
            h = hadamard64(d)
            close(rot, z @ h, 31 * U * mag.sum(-1, keepdims=True) / np.sqrt(d))
        else:
            close(rot, z, 20 * U * mag)


def test_qk_outputs_are_chosen_and_the_same():
    """Each output alone has the bits it has beside the others; no weights
    are weights of one; negative positions rotate back."""
    g = torch.Generator(device="cuda").manual_seed(3)
    q = torch.randn(21, 8, 128, device="cuda", generator=g).half()
    k = torch.randn(21, 2, 128, device="cuda", generator=g).half()
    pos = torch.arange(-5, 16, device="cuda", dtype=torch.int32)
    every = kvmret.qk_norm_rope(q, k, pos, q_raw=True, k_raw=True)
    one = torch.ones(128, device="cuda")
    names = ("q_rot", "k_rot", "q_raw", "k_raw")
    for i, name in enumerate(names):
        flags = {m: m == name for m in names}
        got = kvmret.qk_norm_rope(q, k, pos, one, one, **flags)
        assert all((x is None) == (j != i) for j, x in enumerate(got))
        assert torch.equal(got[i].view(torch.int16), every[i].view(torch.int16))
    c, s = angle64(pos.cpu().numpy(), 128)
    y = every[2].double().cpu().numpy()
    z, _ = rope64(y, c, s)
    # two f16 roundings: of the unrotated row and of the rotated one
    assert np.abs(every[0].double().cpu().numpy() - z).max() <= 3 * 2.0 ** -11 * np.abs(y).max()


def test_qk_infinite_and_nan_rows_stay_in_their_rows():
    g = torch.Generator(device="cuda").manual_seed(4)
    q = torch.randn(9, 8, 128, device="cuda", generator=g)
    k = torch.randn(9, 2, 128, device="cuda", generator=g)
    pos = torch.arange(9, device="cuda", dtype=torch.int32)
    clean = kvmret.qk_norm_rope(q, k, pos)
    q[4, 3, 17], k[2, 1, 0] = float("inf"), float("nan")
    got = kvmret.qk_norm_rope(q, k, pos)
    for x, y, at in ((got[0], clean[0], (4, 3)), (got[1], clean[1], (2, 1))):
        keep = torch.ones(x.shape[:2], dtype=torch.bool, device="cuda")
        keep[at] = False
        assert torch.equal(x[keep], y[keep]) and torch.isnan(x[at]).any()


def quantise(x, kind):
    """f32 rows -> the bytes of kind (the oracle's quantisers)."""
    x = np.ascontiguousarray(x, np.float32)
    if kind == kvmret.TYPE_F16:
        return x.astype(np.float16).view(np.uint8).reshape(x.shape[0], -1)
    return (po.quant_q8_0 if kind == kvmret.TYPE_Q8_0 else po.quant_q4_0)(x).reshape(x.shape[0], -1)


def rotated32(k, pos, fwht, base, scale):
    """The float32 rotation and transform, rounding by rounding."""
    n, h, d = k.shape
    c, s = (x.astype(np.float32)[:, None] for x in angle64(pos, d, base, scale))
    x = k.astype(np.float32)
    a, b = x[..., :d // 2], x[..., d // 2:]
    y = np.concatenate([a * c - b * s, a * s + b * c], -1)
    return po.fwht(y.reshape(-1, d), d).reshape(n, h, d) if fwht else y


F16, Q4, Q8 = kvmret.TYPE_F16, kvmret.TYPE_Q4_0, kvmret.TYPE_Q8_0


@pytest.mark.parametrize("n,hkv,d,page,kt,vt,fwht,rot", [
    (1, 8, 128, 128, F16, F16, False, True), (1, 8, 128, 128, Q8, Q4, True, True),
    (37, 1, 64, 16, F16, F16, False, True), (5, 3, 256, 7, F16, F16, False, False),
    (70, 4, 64, 32, Q8, Q8, True, True), (70, 12, 64, 32, Q4, Q8, True, True),
    (129, 8, 128, 64, Q8, Q4, False, True), (129, 2, 128, 48, Q4, F16, True, False),
    (260, 5, 256, 128, Q8, Q4, True, True), (300, 8, 128, 128, F16, Q8, False, True),
])
def test_paged_append(n, hkv, d, page, kt, vt, fwht, rot):
    """Bytes of every cell: the tokens' rows in theirs, everything else as it
    was. Some tokens have no cell (-1) or one past the last page."""
    rng = np.random.default_rng(n + d)
    pages = -(-n // page) + 3
    k = rng.standard_normal((n, hkv, d)).astype(np.float16)
    v = rng.standard_normal((n, hkv, d)).astype(np.float16)
    k[0, 0, :32] = 0  # a quant block of zeros when not rotated
    v[0, 0, :32] = 0
    if n > 2:
        v[1, 0, :32], v[1, 0, 3], v[1, 0, 9] = 0.25, -2.0, 2.0  # a tie of magnitudes
    cells = rng.permutation(pages * page)[:n].astype(np.int32)
    if n > 4:
        cells[2], cells[4], cells[3] = -1, pages * page, -2 ** 31
    pos = rng.integers(0, 262144, n).astype(np.int32)
    base, scale = 5e5, 0.25
    x = rotated32(k, pos, False, base, scale) if rot else k.astype(np.float32)
    if fwht:
        x = po.fwht(x.reshape(-1, d).copy(), d).reshape(n, hkv, d)
    want = {"k": quantise(x.reshape(n, -1), kt), "v": quantise(v.astype(np.float32).reshape(n, -1), vt)}
    bufs, before = {}, {}
    for name in "kv":
        row = want[name].shape[1]
        # pages with a gap between them
        whole = torch.from_numpy(rng.integers(0, 256, (pages, page * row + 64)).astype(np.uint8)).cuda()
        bufs[name], before[name] = whole, whole.clone()
    p = kvmret.Pages(bufs["k"][:, :-64], bufs["v"][:, :-64], page, hkv, d, kt, vt)
    # tokens strided, as in a projection's rows
    rows = torch.zeros(n, 2 * hkv + 1, d, dtype=torch.float16, device="cuda")
    rows[:, :hkv], rows[:, hkv:2 * hkv] = torch.from_numpy(k).cuda(), torch.from_numpy(v).cuda()
    dev = lambda a: torch.from_numpy(a).cuda()  # noqa: E731
    kvmret.paged_append(p, rows[:, :hkv], rows[:, hkv:2 * hkv], dev(cells), dev(pos) if rot else None,
                        freq_base=base, freq_scale=scale, fwht_n=d if fwht else 0)
    for name in "kv":
        w = before[name].cpu().numpy()
        row = want[name].shape[1]
        for t, c in enumerate(cells):
            if 0 <= c < pages * page:
                at = int(c) % page * row
                w[int(c) // page, at:at + row] = want[name][t]
        assert np.array_equal(bufs[name].cpu().numpy(), w), name


def test_append_equals_rope_f16_rows():
    """An appended f16 key has the bits that kvmret_rope_f16 gives the row."""
    n, hkv, d = 77, 4, 128
    k = torch.randn(n, hkv, d, device="cuda").half()
    v = torch.randn(n, hkv, d, device="cuda").half()
    kc, vc = (torch.zeros(3, 32, hkv, d, dtype=torch.float16, device="cuda") for _ in range(2))
    pos = torch.arange(1000, 1000 + n, device="cuda", dtype=torch.int32)
    kvmret.paged_append(kvmret.Pages(kc, vc, 32, hkv, d), k, v, pos - 1000, pos)
    want = torch.empty_like(k)
    kvmret.rope_f16(k, want, 1000, hkv, d)
    assert torch.equal(kc.flatten(0, 1)[:n], want) and torch.equal(vc.flatten(0, 1)[:n], v)


def test_far_pages():
    """A cell whose byte offset passes 32 bits."""
    hkv, d, page = 8, 256, 128
    n_pages = 4300  # 1 MiB a page
    kc = torch.zeros(n_pages, page, hkv, d, dtype=torch.float16, device="cuda")
    vc = torch.zeros(n_pages, page, hkv, d, dtype=torch.float16, device="cuda")
    k = torch.randn(2, hkv, d, device="cuda").half()
    v = torch.randn(2, hkv, d, device="cuda").half()
    cells = torch.tensor([n_pages * page - 1, 5], device="cuda", dtype=torch.int32)
    kvmret.paged_append(kvmret.Pages(kc, vc, page, hkv, d), k, v, cells)
    assert torch.equal(kc[-1, -1], k[0]) and torch.equal(vc[-1, -1], v[0])
    assert torch.equal(kc[0, 5], k[1]) and int(kc.count_nonzero()) == int(k.count_nonzero())


def test_captured_and_on_another_stream():
    """Both calls in one graph, replayed with new inputs in the same buffers,
    and on a side stream: the bits of the plain calls."""
    n, hq, hkv, d = 6, 8, 2, 128
    q, k, v = (torch.randn(n, h, d, device="cuda").half() for h in (hq, hkv, hkv))
    pos = torch.arange(n, device="cuda", dtype=torch.int32)
    kc, vc = (torch.zeros(2, 16, hkv, d, dtype=torch.float16, device="cuda") for _ in range(2))
    p = kvmret.Pages(kc, vc, 16, hkv, d)

    def step():
        got = kvmret.qk_norm_rope(q, k, pos, k_raw=True)
        kvmret.paged_append(p, got[3], v, pos, pos)
        return got

    def filed(k_raw, pos0):  # the f16 row, rotated
        out = torch.empty_like(k_raw)
        kvmret.rope_f16(k_raw, out, pos0, hkv, d)
        return out

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        first = step()
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    assert torch.equal(kc.flatten(0, 1)[:n], filed(first[3], 0))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = step()
    q.copy_(torch.randn_like(q))
    k.copy_(torch.randn_like(k))
    pos += 9
    kc.zero_()
    graph.replay()
    want = kvmret.qk_norm_rope(q, k, pos, k_raw=True)
    assert torch.equal(held[0], want[0]) and torch.equal(held[1], want[1])
    assert torch.equal(kc.flatten(0, 1)[9:9 + n], filed(want[3], 9))


def test_wrapper_refusals():
    q = torch.zeros(4, 8, 128, dtype=torch.float16, device="cuda")
    k = torch.zeros(4, 2, 128, dtype=torch.float16, device="cuda")
    pos = torch.zeros(4, dtype=torch.int32, device="cuda")
    bad = [lambda: kvmret.qk_norm_rope(q, k.float(), pos), lambda: kvmret.qk_norm_rope(q, k, pos[:3]),
           lambda: kvmret.qk_norm_rope(q, k, pos.long()), lambda: kvmret.qk_norm_rope(q, k[:3], pos),
           lambda: kvmret.qk_norm_rope(q[..., ::2], k[..., ::2], pos),
           lambda: kvmret.qk_norm_rope(q[:1].expand(4, 8, 128), k, pos),
           lambda: kvmret.qk_norm_rope(q, k, pos, q_weight=torch.ones(64, device="cuda"))]
    kc = torch.zeros(2, 16, 2, 128, dtype=torch.float16, device="cuda")
    p = kvmret.Pages(kc, kc.clone(), 16, 2, 128)
    bad += [lambda: kvmret.Pages(kc, kc[:1], 16, 2, 128), lambda: kvmret.Pages(kc, kc, 8, 2, 128),
            lambda: kvmret.paged_append(p, k, k[:, :1], pos, pos),
            lambda: kvmret.paged_append(p, k[:1].expand(4, 2, 128), k, pos, pos),
            lambda: kvmret.paged_append(p, k, k, pos.cpu(), pos)]
    for call in bad:
        with pytest.raises(kvmret.KvmretError):
            call()


def test_pages_of_an_expanded_axis_are_refused():
    """One page repeated by a stride of zero is no paged cache: the stride would
    be taken for dense pages."""
    one = torch.zeros(1, 16, 2, 128, dtype=torch.float16, device="cuda")
    full = torch.zeros(3, 16, 2, 128, dtype=torch.float16, device="cuda")
    for k, v in ((one.expand(3, 16, 2, 128), full), (full, one.expand(3, 16, 2, 128))):
        with pytest.raises(kvmret.KvmretError):
            kvmret.Pages(k, v, 16, 2, 128)
    assert kvmret.Pages(one, one.clone(), 16, 2, 128).n_pages == 1


def test_numbers_out_of_range_are_refused():
    q = torch.zeros(4, 8, 128, dtype=torch.float16, device="cuda")
    k, pos = q[:, :2], torch.zeros(4, dtype=torch.int32, device="cuda")
    for kw in (dict(fwht_n=-1), dict(eps=1e300), dict(freq_base=1e39), dict(freq_scale=-1e39)):
        with pytest.raises(kvmret.KvmretError):
            kvmret.qk_norm_rope(q, k, pos, **kw)
    p = kvmret.Pages(*(torch.zeros(1, 16, 2, 128, dtype=torch.float16, device="cuda") for _ in "kv"),
                     16, 2, 128)
    with pytest.raises(kvmret.KvmretError):
        kvmret.prefix_attn(q, p, None, scale=1e300)


@pytest.mark.parametrize("n,hq,hkv,d,dt,fwht", [
    (512, 32, 8, 64, "f16", False), (777, 7, 1, 64, "f32", True), (513, 32, 4, 256, "bf16", True),
    (1030, 3, 1, 256, "f16", False), (2049, 1, 1, 128, "f32", True),
])
def test_qk_norm_rope_of_chunks(n, hq, hkv, d, dt, fwht):
    """Many tokens (a CTA takes all heads of a few): every head size, row counts that
    leave a CTA's last pass part empty."""
    test_qk_norm_rope(n, hq, hkv, d, dt, fwht, True)
