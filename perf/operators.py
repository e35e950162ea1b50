"""The attention step beside a retrieval window, as a decode or prefill step of
a model runs it per layer: norms of the query and key heads with the position
rotation (`qk`), the new tokens' keys and values appended to a paged cache with
the rotation on the way (`append`), and the attention of a batch of sequences
that share one long prefix (the retrieved window) and own their tails (`attn`).

Sizes: 64 query heads, 8 KV heads, head size 128, pages of 128 tokens, a window
of 256 pages (32,768 tokens) and chunks of 2048 tokens are the benchmark's
configurations 2 to 4; 32 query heads are configuration 1; 8 sequences are the
session lanes of configuration 5; head sizes 64 and 256 and pages of 32 and 64
tokens are the tests'. q8_0 K with the Hadamard rotation and q4_0 V are
configuration 3's cache.

Angles: the position rotation's angle is, by definition here as in the
library's other rotations, the float32 product position * theta_i of the
float32 frequency theta_i; its cosine and sine are taken in 64 bits.
"""
import math
import sys

import numpy as np
import torch

own = False

F16, Q4_0, Q8_0 = 1, 2, 8  # the cache formats' ids
BASE = 1e6                 # rope frequency base of the configurations
EPS = 1e-6


def listed():
    return [
        # one decode token of one conversation: the latency of a single call
        {"name": "qk one token", "op": "qk", "n": 1, "hq": 64, "hkv": 8, "d": 128, "dtype": "f16",
         "fwht": False, "raw": True, "far": 262000},
        # a step of 33 sequences with float32 activations and a quantised
        # window, whose keys are Hadamard-rotated: the query is too
        {"name": "qk batch f32 fwht", "op": "qk", "n": 33, "hq": 64, "hkv": 8, "d": 128,
         "dtype": "f32", "fwht": True, "raw": False, "far": 49000},
        # a prefill chunk: rotated queries for the attention, unrotated queries
        # and keys for the retrieval's accumulator and its block summaries
        {"name": "qk chunk", "op": "qk", "n": 2048, "hq": 64, "hkv": 8, "d": 128, "dtype": "bf16",
         "fwht": False, "raw": True, "far": 49000},
        # small heads, an odd number of tokens
        {"name": "qk d64 odd", "op": "qk", "n": 1777, "hq": 32, "hkv": 8, "d": 64, "dtype": "f16",
         "fwht": False, "raw": False, "far": 49000},
        # one token of each of eight lanes
        {"name": "append lanes", "op": "append", "n": 8, "hkv": 8, "d": 128, "page": 128,
         "kt": F16, "vt": F16, "fwht": False, "gaps": 0},
        # a prefill chunk into f16 pages; some of its tokens have no cell
        {"name": "append chunk", "op": "append", "n": 2048, "hkv": 8, "d": 128, "page": 128,
         "kt": F16, "vt": F16, "fwht": False, "gaps": 5},
        # a prefill chunk into configuration 3's formats
        {"name": "append chunk q8 q4", "op": "append", "n": 2048, "hkv": 8, "d": 128, "page": 128,
         "kt": Q8_0, "vt": Q4_0, "fwht": True, "gaps": 0},
        # a short conversation, four sequences: the latency of a small step
        {"name": "attn short", "op": "attn", "seqs": 4, "new": 1, "ragged": False, "prefix": 1000,
         "tail": 70, "hq": 32, "hkv": 8, "d": 128, "page": 64, "kt": F16, "vt": F16},
        # a decode step of 16 sequences over one full window
        {"name": "attn decode", "op": "attn", "seqs": 16, "new": 1, "ragged": True, "prefix": 32768,
         "tail": 700, "hq": 64, "hkv": 8, "d": 128, "page": 128, "kt": F16, "vt": F16},
        # the same over configuration 3's formats
        {"name": "attn decode q8 q4", "op": "attn", "seqs": 16, "new": 1, "ragged": True,
         "prefix": 32701, "tail": 700, "hq": 64, "hkv": 8, "d": 128, "page": 128, "kt": Q8_0,
         "vt": Q4_0},
        # 32 sequences checking up to five drafted tokens each
        {"name": "attn drafts", "op": "attn", "seqs": 32, "new": 5, "ragged": True, "prefix": 32768,
         "tail": 900, "hq": 64, "hkv": 8, "d": 128, "page": 128, "kt": F16, "vt": F16},
        # a prefill chunk of one conversation over its window, causal in itself
        {"name": "attn chunk", "op": "attn", "seqs": 1, "new": 2048, "ragged": False,
         "prefix": 32768, "tail": 2048, "hq": 64, "hkv": 8, "d": 128, "page": 128, "kt": F16,
         "vt": F16},
    ]


def draw(rng):
    def spread(lo, hi):  # whole numbers over their logarithm
        return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))

    op = rng.choice(["qk", "append", "attn", "attn"])
    if op == "qk":
        d, hkv = rng.choice([64, 128, 128, 256]), rng.choice([1, 2, 4, 8])
        return {"op": op, "n": spread(1, 2048), "hq": hkv * rng.choice([1, 4, 5, 8]), "hkv": hkv,
                "d": d, "dtype": rng.choice(["f16", "bf16", "f32"]), "fwht": rng.random() < 0.4,
                "raw": rng.random() < 0.5, "far": spread(2100, 262000)}
    formats = [(F16, F16), (F16, F16), (Q8_0, Q4_0), (Q8_0, Q8_0), (Q4_0, Q4_0), (Q8_0, F16)]
    if op == "append":
        d, (kt, vt) = rng.choice([64, 128, 128, 256]), rng.choice(formats)
        return {"op": op, "n": spread(1, 2048), "hkv": rng.choice([4, 8]), "d": d,
                "page": rng.choice([16, 32, 64, 128]), "kt": kt, "vt": vt,
                "fwht": kt != F16 and rng.random() < 0.7, "gaps": rng.choice([0, 0, 3, 11])}
    d, (kt, vt) = rng.choice([64, 128, 128, 256]), rng.choice(formats)
    hkv, chunk = rng.choice([4, 8]), rng.random() < 0.25
    seqs = 1 if chunk else spread(1, 32)
    new = spread(16, 1024) if chunk else rng.choice([1, 1, 2, 5])
    return {"op": op, "seqs": seqs, "new": new, "ragged": not chunk and rng.random() < 0.7,
            "prefix": spread(1, 32768), "tail": max(new, spread(1, 2048)),
            "hq": hkv * rng.choice([1, 4, 5, 8]), "hkv": hkv, "d": d,
            "page": rng.choice([16, 32, 64, 128]), "kt": kt, "vt": vt}


def _generator(seed):
    return torch.Generator(device="cuda").manual_seed(int(seed))


def _normal(gen, *shape):
    return torch.randn(*shape, device="cuda", generator=gen)


def _row_bytes(kind, n):
    return {F16: 2 * n, Q8_0: n // 32 * 34, Q4_0: n // 32 * 18}[kind]


def _cache(gen, kind, pages, page, hkv, d):
    """A page buffer with plausible contents: f16 values with a scale for each
    channel, or quant blocks of f16 scale and whole numbers."""
    if kind == F16:
        scale = torch.exp(0.5 * _normal(gen, hkv, d))
        return (_normal(gen, pages, page, hkv, d) * scale).half()
    size = 34 if kind == Q8_0 else 18
    raw = torch.randint(0, 256, (pages, page, hkv * d // 32, size), device="cuda", generator=gen,
                        dtype=torch.uint8)
    top = 127.0 if kind == Q8_0 else 8.0
    scale = (torch.rand(raw.shape[:-1], device="cuda", generator=gen) + 0.5) * 2.5 / top
    raw[..., :2] = scale.half()[..., None].view(torch.uint8)
    return raw


def _lengths(case):
    """New tokens and tail lengths of every sequence, on the host: the case's,
    whatever the seed, so that every seed does the same work."""
    n, new, tail = case["seqs"], case["new"], case["tail"]
    rng = np.random.default_rng([n, new, tail, case["prefix"]])
    if not case["ragged"]:
        return [new] * n, [tail] * n
    q = [int(x) for x in rng.integers(1, new + 1, n)]
    q[0] = new
    t = [max(a, int(x)) for a, x in zip(q, rng.integers(1, tail + 1, n))]
    t[0] = tail
    return q, t


def prepare(case, seed):
    g, op = _generator(seed), case["op"]
    d, hkv = case["d"], case["hkv"]
    state = dict(case)
    if op == "qk":
        kind = {"f16": torch.float16, "bf16": torch.bfloat16, "f32": torch.float32}[case["dtype"]]
        n, hq = case["n"], case["hq"]
        # the projection's rows: queries, keys and values of a token together
        rows = (3.0 * _normal(g, n, hq + 2 * hkv, d)).to(kind)
        state.update(q=rows[:, :hq], k=rows[:, hq:hq + hkv],
                     wq=1.0 + 0.2 * _normal(g, d), wk=1.0 + 0.2 * _normal(g, d),
                     pos=torch.randint(0, case["far"], (n,), device="cuda", generator=g,
                                       dtype=torch.int32))
        return state
    page = case["page"]
    if op == "append":
        n = case["n"]
        pages = -(-n // page) + 2
        cells = torch.randperm(pages, device="cuda", generator=g)[:, None] * page + torch.arange(
            page, device="cuda")
        first = int(seed) % page  # the run of tokens starts inside a page
        cells = cells.reshape(-1)[first:first + n].to(torch.int32)
        if case["gaps"]:
            cells[::case["gaps"]] = -1
        state.update(kc=_cache(g, case["kt"], pages, page, hkv, d),
                     vc=_cache(g, case["vt"], pages, page, hkv, d),
                     k=_normal(g, n, hkv, d).half(), v=_normal(g, n, hkv, d).half(), cells=cells,
                     pos=torch.arange(n, device="cuda", dtype=torch.int32) + 32768)
    else:
        new, tails = _lengths(case)
        width = -(-max(tails) // page)
        pp, tp = -(-case["prefix"] // page), width * case["seqs"]
        pool, spare = pp + 3, tp + 3
        start = np.concatenate([[0], np.cumsum(new)])
        q = _normal(g, int(start[-1]), case["hq"], d)
        own_table = torch.randperm(spare, device="cuda", generator=g)[:tp].to(torch.int32).view(
            case["seqs"], width)
        held = torch.tensor([-(-t // page) for t in tails], device="cuda")
        own_table[torch.arange(width, device="cuda") >= held[:, None]] = -1  # no page there
        state.update(
            q=(1.2 * q).half(), new=new, tails=tails, rows=int(start[-1]),
            start=torch.tensor(start, device="cuda", dtype=torch.int32),
            kc=_cache(g, case["kt"], pool, page, hkv, d), vc=_cache(g, case["vt"], pool, page, hkv, d),
            tk=_cache(g, case["kt"], spare, page, hkv, d), tv=_cache(g, case["vt"], spare, page, hkv, d),
            table=torch.randperm(pool, device="cuda", generator=g)[:pp].to(torch.int32),
            own_table=own_table,
            length=torch.tensor([case["prefix"]], device="cuda", dtype=torch.int32),
            own_length=torch.tensor(tails, device="cuda", dtype=torch.int32))
    if own:
        kvmret = _library()
        state["pages"] = kvmret.Pages(state["kc"], state["vc"], page, hkv, d, case["kt"], case["vt"])
        if op == "attn":
            state["own_pages"] = kvmret.Pages(state["tk"], state["tv"], page, hkv, d, case["kt"],
                                              case["vt"])
    return state


def _library():
    if "kvmret" not in sys.modules:
        sys.path.insert(0, "kvmem-llama.cpp_b200")  # the package's folder is no module name
    import kvmret
    return kvmret


def _cos_sin(pos, d):
    """float32 cosines and sines [n][d / 2] of the float32 angles."""
    i = torch.arange(d // 2, device=pos.device, dtype=torch.float64)
    theta = (float(np.float32(BASE)) ** (-2.0 * i / d)).float()
    angle = (pos.float()[:, None] * theta).double()
    return torch.cos(angle).float(), torch.sin(angle).float()


def _rotate(x, cos, sin):
    lo, hi = x.chunk(2, -1)
    c, s = cos[:, None], sin[:, None]
    return torch.cat([lo * c - hi * s, lo * s + hi * c], -1)


def _hadamard_stage(x, h):
    a, b = x.unflatten(-1, (-1, 2, h)).unbind(-2)
    return torch.stack([a + b, a - b], -2).flatten(-3)


def _hadamard(x, h=1):
    """The orthonormal Hadamard transform of the last axis: scaled on the way
    in, then butterflies of strides 1, 2, 4, ..."""
    n = x.shape[-1]
    x = x * float(np.float32(1.0) / np.sqrt(np.float32(n))) if h == 1 else x
    return x if h == n else _hadamard(_hadamard_stage(x, h), 2 * h)


def _quantise(x, kind):
    """The blocks of 32 values as (f16 scale, whole numbers 0..255 in bytes)."""
    b = x.unflatten(-1, (-1, 32))
    big = b.abs().amax(-1, keepdim=True)
    if kind == Q8_0:
        scale = big / 127.0
        inv = torch.where(scale != 0, 1.0 / scale, 0.0)
        y = b * inv
        whole = (torch.sign(y) * torch.floor(y.abs() + 0.5)).to(torch.int8).view(torch.uint8)
    else:
        # the first value of the largest magnitude, with its sign
        at = (b.abs() == big).to(torch.uint8).argmax(-1, keepdim=True)
        scale = b.gather(-1, at) / -8.0
        inv = torch.where(scale != 0, 1.0 / scale, 0.0)
        whole = (b * inv + 8.5).to(torch.int32).clamp(max=15).to(torch.uint8)
        whole = whole[..., :16] | (whole[..., 16:] << 4)
    return torch.cat([scale.half().view(torch.uint8), whole], -1)


def _stored(cache, kind, dtype):
    """The values that a page buffer holds, [pages][page][...]."""
    if kind == F16:
        return cache if dtype is torch.float16 else cache.to(dtype)
    scale, body = cache[..., :2].view(torch.float16).to(dtype), cache[..., 2:]
    if kind == Q8_0:
        return scale * body.view(torch.int8)
    return scale * (torch.cat([body & 15, body >> 4], -1).to(torch.int8) - 8)


def _norm(x, weight):
    x = x.float()
    return x * torch.rsqrt(x.square().mean(-1, keepdim=True) + EPS) * weight


def _plain_qk(s):
    cos, sin = _cos_sin(s["pos"], s["d"])
    q, k = _norm(s["q"], s["wq"]), _norm(s["k"], s["wk"])
    qr, kr = _rotate(q, cos, sin), _rotate(k, cos, sin)
    if s["fwht"]:
        qr, kr = _hadamard(qr), _hadamard(kr)
    raw = {"q_raw": q.half(), "k_raw": k.half()} if s["raw"] else {}
    return {"q_rot": qr.half(), "k_rot": kr.half(), **raw}


def _store(cache, kind, cells, x):
    at = cells.long()
    keep = at >= 0
    rows = x.half() if kind == F16 else _quantise(x.flatten(1), kind)
    cache.flatten(0, 1)[at[keep]] = rows[keep]


def _append_outputs(s):
    return {"k": _stored(s["kc"], s["kt"], torch.float16), "v": _stored(s["vc"], s["vt"], torch.float16)}


def _plain_append(s):
    cos, sin = _cos_sin(s["pos"], s["d"])
    k = _rotate(s["k"].float(), cos, sin)
    _store(s["kc"], s["kt"], s["cells"], _hadamard(k) if s["fwht"] else k)
    _store(s["vc"], s["vt"], s["cells"], s["v"].float())
    return _append_outputs(s)


def _paged(cache, kind, table, length, hkv, d, dtype):
    """The first `length` rows of a page list, [hkv][length][d]; `table` may
    have a batch axis in front."""
    x = _stored(cache[table.long()], kind, dtype).flatten(table.dim())
    x = x.view(*table.shape[:-1], -1, hkv, d)[..., :length, :, :]
    return x.transpose(-3, -2)


def _plain_attn(s):
    f32, hkv, d, g = torch.float32, s["hkv"], s["d"], s["hq"] // s["hkv"]
    new, n = max(s["new"]), len(s["new"])
    start, own_length = s["start"].long(), s["own_length"].long()
    kp = _paged(s["kc"], s["kt"], s["table"], s["prefix"], hkv, d, f32)
    vp = _paged(s["vc"], s["vt"], s["table"], s["prefix"], hkv, d, f32)
    kt = _paged(s["tk"], s["kt"], s["own_table"], max(s["tails"]), hkv, d, f32)
    vt = _paged(s["tv"], s["vt"], s["own_table"], max(s["tails"]), hkv, d, f32)
    # queries padded to [sequence][new token]
    step = torch.arange(new, device="cuda")
    count = start[1:] - start[:-1]
    real = step < count[:, None]
    row = (start[:-1, None] + step).clamp(max=s["rows"] - 1)
    q = s["q"].float()[row].view(n, new, hkv, g, d) / math.sqrt(d)
    sp = torch.einsum("bihgd,hkd->bhgik", q, kp)
    st = torch.einsum("bihgd,bhkd->bhgik", q, kt)
    last = own_length[:, None] - count[:, None] + step  # the tail position of each new token
    seen = torch.arange(st.shape[-1], device="cuda") <= last[..., None]
    st = st.masked_fill(~seen[:, None, None], -math.inf)
    top = torch.maximum(sp.amax(-1), st.amax(-1))[..., None]
    sp, st = torch.exp(sp - top), torch.exp(st - top)
    total = sp.sum(-1) + st.sum(-1)
    out = torch.einsum("bhgik,hkd->bihgd", sp, vp) + torch.einsum("bhgik,bhkd->bihgd", st, vt)
    out = out / total.permute(0, 3, 1, 2)[..., None]
    return out.reshape(n, new, s["hq"], d)[real].half()


def run(state):
    op = state["op"]
    if not own:
        return {"qk": _plain_qk, "append": _plain_append, "attn": _plain_attn}[op](state)
    kvmret = _library()
    if op == "qk":
        raw = state["raw"]
        got = kvmret.qk_norm_rope(state["q"], state["k"], state["pos"], state["wq"], state["wk"],
                                  eps=EPS, freq_base=BASE, fwht_n=state["d"] if state["fwht"] else 0,
                                  q_raw=raw, k_raw=raw)
        return {name: x for name, x in zip(("q_rot", "k_rot", "q_raw", "k_raw"), got) if x is not None}
    if op == "append":
        kvmret.paged_append(state["pages"], state["k"], state["v"], state["cells"], state["pos"],
                            freq_base=BASE, fwht_n=state["d"] if state["fwht"] else 0)
        return _append_outputs(state)
    return kvmret.prefix_attn(state["q"], state["pages"], state["length"], state["own_pages"],
                              state["own_table"], state["own_length"], state["start"],
                              prefix_table=state["table"], max_prefix=state["prefix"])


def work(case):
    op, d, hkv = case["op"], case["d"], case["hkv"]
    if op == "qk":
        n, heads = case["n"], case["hq"] + hkv
        size = 4 if case["dtype"] == "f32" else 2
        outs = 4 if case["raw"] else 2  # bytes of f16, each wanted form
        per = 3 + 4 + 3 + (math.log2(d) + 1 if case["fwht"] else 0)
        return {"bytes": n * heads * d * (size + outs) + 4 * n + 8 * d, "flops": n * heads * d * per}
    e = hkv * d
    row = _row_bytes(case["kt"], e) + _row_bytes(case["vt"], e)
    if op == "append":
        n = case["n"]
        n -= -(-n // case["gaps"]) if case["gaps"] else 0
        return {"bytes": n * (4 * e + row) + 8 * case["n"], "flops": n * e * 4}
    new, tails = _lengths(case)
    q = case["hq"] * d * sum(new)
    pairs = sum(a * case["prefix"] + a * t - a * (a - 1) // 2 for a, t in zip(new, tails))
    return {"bytes": (case["prefix"] + sum(tails)) * row + 4 * q, "flops": 4 * pairs * case["hq"] * d}


# ---- the operators' definitions in 64 bits, on numbers taken apart anew ----


def _exact_turn(pos, d):
    f = np.float32(BASE) ** (np.arange(d // 2, dtype=np.float64) * (-2.0 / d))
    a = pos.cpu().numpy().astype(np.float32)[:, None] * f.astype(np.float32)
    a = torch.from_numpy(a.astype(np.float64)).cuda()
    return torch.polar(torch.ones_like(a), a)[:, None]


def _exact_rope(x, turn):
    half = x.shape[-1] // 2
    z = torch.complex(x[..., :half], x[..., half:]) * turn
    return torch.cat([z.real, z.imag], -1)


def _exact_matrix(n):
    i = np.arange(n)
    bits = np.array([[bin(a & b).count("1") for b in i] for a in i])
    return torch.from_numpy(((-1.0) ** bits) / math.sqrt(n)).cuda()


def _exact_values(raw, kind):
    if kind == F16:
        return raw.double()
    r = raw.cpu().numpy()
    scale = np.ascontiguousarray(r[..., :2]).view(np.float16).astype(np.float64)
    if kind == Q8_0:
        v = np.ascontiguousarray(r[..., 2:]).view(np.int8).astype(np.float64)
    else:
        v = np.concatenate([r[..., 2:] % 16, r[..., 2:] // 16], -1).astype(np.float64) - 8
    return torch.from_numpy(scale * v).cuda()


def _exact_blocks(x, kind):
    """The values that the blocks of 32 of x stand for once quantised (the
    scale held in f16, the whole numbers found with the scale before that)."""
    b = x.reshape(x.shape[0], -1, 32)
    if kind == Q8_0:
        scale = b.abs().max(-1, keepdim=True).values / 127
        y = torch.where(scale > 0, b / scale, 0)
        return torch.trunc(y + torch.copysign(torch.full_like(y, 0.5), y)) * scale.half().double()
    first = b.abs().max(-1, keepdim=True).indices
    scale = b.gather(-1, first) / -8
    y = torch.where(scale != 0, torch.floor(b / scale + 8.5), torch.full_like(b, 8.0))
    return (y.clamp(max=15) - 8) * scale.half().double()


def _exact_append(s):
    turn = _exact_turn(s["pos"], s["d"])
    k = _exact_rope(s["k"].double(), turn)
    if s["fwht"]:
        k = k @ _exact_matrix(s["d"])
    found = {}
    for name, cache, kind, x in (("k", s["kc"], s["kt"], k), ("v", s["vc"], s["vt"], s["v"].double())):
        full = _exact_values(cache, kind)
        flat = full.view(-1, *full.shape[2:])
        x = x if kind == F16 else _exact_blocks(x, kind)
        for i, c in enumerate(s["cells"].tolist()):
            if c >= 0:
                flat[c] = x[i]
        found[name] = full
    return found


def _exact_attn(s):
    d, hkv, g = s["d"], s["hkv"], s["hq"] // s["hkv"]

    def values(raw, kind, table, length):
        return _exact_values(raw[table.long()], kind).reshape(-1, hkv, d)[:length]

    kp, vp = (values(s[c], s[t], s["table"], s["prefix"]) for c, t in (("kc", "kt"), ("vc", "vt")))
    out = torch.empty(s["rows"], s["hq"], d, dtype=torch.float64, device="cuda")
    at = 0
    for b, (new, tail) in enumerate(zip(s["new"], s["tails"])):
        k = torch.cat([kp, values(s["tk"], s["kt"], s["own_table"][b], tail)])
        v = torch.cat([vp, values(s["tv"], s["vt"], s["own_table"][b], tail)])
        total = k.shape[0]
        limit = total - new + torch.arange(new, device="cuda")
        for h in range(s["hq"]):
            w = s["q"][at:at + new, h].double() @ k[:, h // g].T * d ** -0.5
            w = w.masked_fill(torch.arange(total, device="cuda") > limit[:, None], -math.inf)
            out[at:at + new, h] = torch.softmax(w, -1) @ v[:, h // g]
        at += new
    return out


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "append":
        return _exact_append(s)
    if case["op"] == "attn":
        return _exact_attn(s)
    turn, found = _exact_turn(s["pos"], s["d"]), {}
    for name, w in (("q", "wq"), ("k", "wk")):
        x = s[name].double()
        x = x / (x.pow(2).sum(-1, keepdim=True) / s["d"] + EPS).sqrt() * s[w].double()
        y = _exact_rope(x, turn)
        found[name + "_rot"] = y @ _exact_matrix(s["d"]) if s["fwht"] else y
        if s["raw"]:
            found[name + "_raw"] = x
    return found
