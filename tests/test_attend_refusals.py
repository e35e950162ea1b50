"""Argument checks of the attention-step entry points: every refusal comes from
the host before any CUDA call, so the addresses here are never used."""
import ctypes

import pytest

import kvmret

lib = kvmret.lib
A = 4096  # an aligned address that nothing reads


def qk_args(**kw):
    a = dict(q_dev=A, k_dev=A, q_stride=1024, k_stride=256, q_weight_dev=None, k_weight_dev=None,
             pos_dev=A, q_rot_dev=A, k_rot_dev=A, q_raw_dev=None, k_raw_dev=None, n_tok=2,
             n_head=8, n_head_kv=2, d_head=128, n_rot=128, fwht_n=0, type=kvmret.TYPE_F16,
             eps=1e-6, freq_base=1e6, freq_scale=1.0)
    a.update(kw)
    return kvmret.QkArgs(**a)


@pytest.mark.parametrize("kw,word", [
    (dict(d_head=96, n_rot=96), b"d_head"), (dict(n_rot=64), b"n_rot"), (dict(fwht_n=64), b"fwht_n"),
    (dict(type=8), b"type"), (dict(eps=-1.0), b"eps"), (dict(eps=float("nan")), b"eps"),
    (dict(freq_base=0.0), b"freq_base"), (dict(freq_scale=float("inf")), b"freq_base"),
    (dict(pos_dev=None), b"positions"), (dict(q_dev=None), b"without its rows"),
    (dict(n_head=0), b"heads"), (dict(q_stride=1016), b"overlap"), (dict(k_stride=0), b"overlap"),
    (dict(q_dev=A + 2), b"aligned"), (dict(q_stride=1028), b"aligned"),
    (dict(k_rot_dev=A + 8), b"aligned"), (dict(type=kvmret.TYPE_F32, q_stride=1026), b"aligned"),
])
def test_qk_norm_rope_refuses(kw, word):
    assert lib.kvmret_qk_norm_rope(ctypes.byref(qk_args(**kw)), None) == -1
    assert word in lib.kvmret_last_error()


def test_qk_norm_rope_nothing_to_do():
    assert lib.kvmret_qk_norm_rope(None, None) == -1
    assert lib.kvmret_qk_norm_rope(ctypes.byref(qk_args(n_tok=0, pos_dev=None)), None) == 0
    assert lib.kvmret_qk_norm_rope(ctypes.byref(qk_args(q_rot_dev=None, k_rot_dev=None)), None) == 0


def pages_desc(**kw):
    a = dict(k_dev=A, v_dev=A, k_page_bytes=0, v_page_bytes=0, n_pages=4, page_tokens=32,
             n_head_kv=2, d_head=128, k_type=kvmret.TYPE_F16, v_type=kvmret.TYPE_F16)
    a.update(kw)
    return kvmret.PagesDesc(**a)


BAD_PAGES = [
    (dict(k_dev=None), b"null"), (dict(d_head=80), b"d_head"), (dict(n_head_kv=0), b"n_head_kv"),
    (dict(n_pages=0), b"pages"), (dict(page_tokens=0), b"pages"),
    (dict(n_pages=1 << 20, page_tokens=1 << 12), b"pages"), (dict(k_type=3), b"type"),
    (dict(v_type=0), b"type"), (dict(k_type=kvmret.TYPE_Q8_0, n_head_kv=1), b"row bytes"),
    (dict(k_dev=A + 8), b"aligned"), (dict(v_page_bytes=32 * 512 + 8), b"aligned"),
    (dict(k_page_bytes=31 * 512), b"shorter"),
]


@pytest.mark.parametrize("kw,word", BAD_PAGES)
def test_paged_append_refuses_pages(kw, word):
    rc = lib.kvmret_paged_append(ctypes.byref(pages_desc(**kw)), A, 0, A, 0, A, A, 3, 1e6, 1.0, 0,
                                 None)
    assert rc == -1 and word in lib.kvmret_last_error()


@pytest.mark.parametrize("args,word", [
    ((None, 0, A, 0, A, A, 3, 1e6, 1.0, 0), b"null"), ((A, 0, A, 0, None, A, 3, 1e6, 1.0, 0), b"null"),
    ((A, 0, A, 0, A, A, 3, 1e6, 1.0, 64), b"fwht_n"), ((A, 0, A, 0, A, A, 3, 0.0, 1.0, 0), b"freq"),
    ((A + 2, 0, A, 0, A, A, 3, 1e6, 1.0, 0), b"aligned"),
    ((A, 260, A, 0, A, A, 3, 1e6, 1.0, 0), b"aligned"),
    ((A, 0, A, 248, A, A, 3, 1e6, 1.0, 0), b"overlap"),
])
def test_paged_append_refuses(args, word):
    rc = lib.kvmret_paged_append(ctypes.byref(pages_desc()), *args, None)
    assert rc == -1 and word in lib.kvmret_last_error()


def test_paged_append_of_no_tokens():
    assert lib.kvmret_paged_append(ctypes.byref(pages_desc()), None, 0, None, 0, None, None, 0, 1e6,
                                   1.0, 0, None) == 0


def attn_args(**kw):
    a = dict(q_dev=A, q_stride=0, out_dev=A, lse_dev=None, n_q=3, n_head=4, scale=0.1, max_prefix=100,
             prefix_len_dev=None, prefix_table_dev=None, prefix_ntok_dev=None, n_seq=2, tail_pages=3,
             q_start_dev=A, tail_table_dev=A, tail_len_dev=A)
    a.update(kw)
    return kvmret.AttnArgs(**a)


def attn(prefix=None, tail=None, ws=A, ws_bytes=1 << 40, **kw):
    ref = lambda x: None if x is None else ctypes.byref(x)  # noqa: E731
    return lib.kvmret_prefix_attn(ref(prefix), ref(tail), ctypes.byref(attn_args(**kw)), ws, ws_bytes, None)


@pytest.mark.parametrize("kw,word", BAD_PAGES)
def test_prefix_attn_refuses_pages(kw, word):
    for pages in ((pages_desc(**kw), pages_desc()), (pages_desc(), pages_desc(**kw))):
        assert attn(*pages) == -1 and word in lib.kvmret_last_error()


@pytest.mark.parametrize("kw,word", [
    (dict(n_head=5), b"n_head"), (dict(n_head=0), b"n_head"), (dict(scale=float("inf")), b"scale"),
    (dict(n_q=65536), b"65535"), (dict(n_seq=70000), b"65535"), (dict(q_dev=None), b"null"),
    (dict(out_dev=None), b"null"), (dict(q_dev=A + 4), b"aligned"), (dict(q_stride=516), b"aligned"),
    (dict(q_stride=504), b"overlap"), (dict(q_start_dev=None), b"tails"),
    (dict(tail_len_dev=None), b"tails"), (dict(tail_table_dev=None), b"tails"),
    (dict(tail_pages=0), b"tails"), (dict(tail_pages=1 << 27), b"2^31"),
    (dict(max_prefix=1 << 31), b"max_prefix"), (dict(max_prefix=129), b"max_prefix"),
    (dict(max_prefix=0, n_seq=0), b"without"),
])
def test_prefix_attn_refuses(kw, word):
    assert attn(pages_desc(), pages_desc(), **kw) == -1 and word in lib.kvmret_last_error()


def test_prefix_attn_refuses_mixed_geometry_and_odd_pages():
    assert attn(pages_desc(), pages_desc(n_head_kv=4)) == -1 and b"prefix of" in lib.kvmret_last_error()
    assert attn(pages_desc(page_tokens=24), pages_desc(), max_prefix=90) == -1 and b"16 tokens" in lib.kvmret_last_error()
    assert attn(pages_desc(), pages_desc(page_tokens=8)) == -1 and b"16 tokens" in lib.kvmret_last_error()
    assert attn(None, pages_desc()) == -1 and attn(pages_desc(), None) == -1
    assert attn(pages_desc(), pages_desc(), n_q=0, q_dev=None) == 0


def test_window_attn_refuses_no_context():
    assert lib.kvmret_window_attn(None, 0, None, ctypes.byref(attn_args()), None, 0) == -1


def test_ws_bytes_of_bad_shapes():
    for shape in ((1, 3, 2, 128, 1), (1, 4, 0, 128, 1), (1, 4, 2, 96, 1), (70000, 4, 2, 128, 1)):
        assert lib.kvmret_prefix_attn_ws_bytes(*shape) == 0


class _Rows:
    """What Pages asks of a tensor, on the CPU: a CUDA tensor of zeros would do."""

    def __init__(self, x):
        self.x, self.is_cuda, self.device, self.dtype = x, True, "cuda:0", x.dtype
        self.shape, self.stride, self.element_size = x.shape, x.stride, x.element_size
        self.data_ptr, self.get_device = x.data_ptr, lambda: 0

    def __getitem__(self, i):
        return self.x[i]


@pytest.mark.parametrize("dtype,kind,good", [
    ("float16", kvmret.TYPE_F16, True), ("uint8", kvmret.TYPE_F16, True), ("int8", kvmret.TYPE_Q8_0, True),
    ("uint8", kvmret.TYPE_Q4_0, True), ("bfloat16", kvmret.TYPE_F16, False),
    ("int16", kvmret.TYPE_F16, False), ("float32", kvmret.TYPE_F16, False),
    ("float16", kvmret.TYPE_Q8_0, False), ("int16", kvmret.TYPE_Q4_0, False),
])
def test_pages_refuse_other_element_types(dtype, kind, good):
    """A cache of another type with as many bytes would be read as this one's."""
    import torch
    dt = getattr(torch, dtype)
    bytes_ = 16 * kvmret.row_bytes(kind, 256)
    x = _Rows(torch.zeros(2, bytes_ // dt.itemsize, dtype=dt))
    f = _Rows(torch.zeros(2, 16, 2, 128, dtype=torch.float16))
    for k, v, types in ((x, f, (kind, kvmret.TYPE_F16)), (f, x, (kvmret.TYPE_F16, kind))):
        if good:
            assert kvmret.Pages(k, v, 16, 2, 128, *types).n_pages == 2
        else:
            with pytest.raises(kvmret.KvmretError, match="float16"):
                kvmret.Pages(k, v, 16, 2, 128, *types)


def test_workspace_follows_the_rows():
    """Partial outputs are kept for rows, not for whole tiles of each sequence: about
    2.2 rows for each of the batch's, and what lists that several SMs share take."""
    size = lib.kvmret_prefix_attn_ws_bytes
    for n, h, hkv, d in ((1, 64, 8, 128), (16, 64, 8, 128), (1024, 64, 8, 128), (65535, 8, 8, 64),
                         (65535, 64, 8, 128), (300, 5, 1, 256)):
        for seqs in (0, 1, n):
            mine = -(-n * h // hkv // 8) * 8  # of a KV head, by eights
            rows = 2.2 * n * h + (2 * 160 + 2 * hkv) * min(256, mine) + 8
            assert 0 < size(n, h, hkv, d, seqs) <= rows * (4 * d + 8) + 32 * n * h + 4096
    assert size(1, 64, 8, 128, 1) < 4 << 20 and size(1024, 64, 8, 128, 1024) < 128 << 20


def test_prefix_attn_refuses_rows_that_no_workspace_counts():
    assert attn(pages_desc(), pages_desc(), n_q=65535, n_head=32764) == -1
    assert b"workspace" in lib.kvmret_last_error() and b"too many" in lib.kvmret_last_error()


class _OnCpu:
    """A CPU tensor that passes for one of the wrappers' device."""
    is_cuda = True

    def __init__(self, x):
        self.x = x

    def __getattr__(self, name):
        return getattr(self.x, name)

    def __getitem__(self, i):
        return self.x[i]


def test_numbers_that_no_field_holds_are_refused():
    """A negative count or a number past float32 is the library's error, before any launch."""
    import torch
    q, k = (_OnCpu(torch.zeros(4, h, 128, dtype=torch.float16)) for h in (8, 2))
    pos = torch.zeros(4, dtype=torch.int32)
    for kw in (dict(fwht_n=-1), dict(eps=1e300), dict(freq_base=1e39), dict(freq_scale=-1e39)):
        with pytest.raises(kvmret.KvmretError, match="range"):
            kvmret.qk_norm_rope(q, k, pos, **kw)
    p = kvmret.Pages(*(_OnCpu(torch.zeros(1, 16, 2, 128, dtype=torch.float16)) for _ in "kv"), 16, 2, 128)
    with pytest.raises(kvmret.KvmretError, match="range"):
        kvmret.prefix_attn(q, p, None, scale=1e300)
