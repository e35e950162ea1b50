// C ABI of the attention step beside the window: per-head norms with the
// position rotation, the append to a paged cache and the attention over a
// shared prefix. Every argument is checked
// on the host before the launch; no C++ exception leaves this file.
#include "attend.hpp"

#include <cmath>
#include <cstdarg>
#include <cstdio>

namespace {

int fail(int code, const char *fmt, ...) {
    char buf[512];
    va_list ap;
    va_start(ap, fmt);
    vsnprintf(buf, sizeof(buf), fmt, ap);
    va_end(ap);
    try {
        return kvmret::set_error(code, buf);
    } catch (...) {  // no memory for the message
        return code;
    }
}

int launched(cudaError_t e) {
    return e == cudaSuccess ? KVMRET_OK
                            : fail(KVMRET_ERR_CUDA, "launch: %s", cudaGetErrorString(e));
}

bool aligned16(const void *p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }

// Frequencies as the library's other rotations compute them
// (kvmem/src/host/rope.cpp:20-24).
kvmret::Theta make_theta(uint32_t n_rot, float base, float scale) {
    kvmret::Theta t{};
    for (uint32_t i = 0; i < n_rot / 2 && i < 128; ++i) {
        t.v[i] = std::pow(base, -2.0f * static_cast<float>(i) / static_cast<float>(n_rot));
        t.v[i] *= scale;
    }
    return t;
}

bool rope_ok(float base, float scale) {
    return base > 0.0f && std::isfinite(base) && std::isfinite(scale);
}

bool head_ok(uint32_t d) { return d == 64 || d == 128 || d == 256; }

}  // namespace

namespace kvmret {

int resolve_pages(const kvmret_pages *p, const char *what, PageView *out) {
    if (!p || !p->k_dev || !p->v_dev) return fail(KVMRET_ERR_ARG, "%s: null buffer", what);
    if (!head_ok(p->d_head))
        return fail(KVMRET_ERR_ARG, "%s: d_head %u not in {64, 128, 256}", what, p->d_head);
    if (p->n_head_kv == 0 || p->n_head_kv > 1024)
        return fail(KVMRET_ERR_ARG, "%s: n_head_kv %u not in 1..1024", what, p->n_head_kv);
    if (p->n_pages == 0 || p->page_tokens == 0 ||
        static_cast<uint64_t>(p->n_pages) * p->page_tokens > 0x7fffffffull)
        return fail(KVMRET_ERR_ARG, "%s: %u pages of %u tokens", what, p->n_pages, p->page_tokens);
    for (int32_t t : {p->k_type, p->v_type})
        if (t != KVMRET_TYPE_F16 && t != KVMRET_TYPE_Q8_0 && t != KVMRET_TYPE_Q4_0)
            return fail(KVMRET_ERR_ARG, "%s: type %d unsupported (f16, q8_0 or q4_0)", what, t);
    PageView v{};
    v.k = static_cast<uint8_t *>(p->k_dev);
    v.v = static_cast<uint8_t *>(p->v_dev);
    v.k_row = kvmret_row_bytes(p->k_type, p->n_head_kv * p->d_head);
    v.v_row = kvmret_row_bytes(p->v_type, p->n_head_kv * p->d_head);
    v.k_page = p->k_page_bytes ? p->k_page_bytes : v.k_row * p->page_tokens;
    v.v_page = p->v_page_bytes ? p->v_page_bytes : v.v_row * p->page_tokens;
    v.n_pages = p->n_pages;
    v.page_tokens = p->page_tokens;
    v.n_head_kv = p->n_head_kv;
    v.d_head = p->d_head;
    v.k_type = p->k_type;
    v.v_type = p->v_type;
    if (v.k_row % 16 || v.v_row % 16)
        return fail(KVMRET_ERR_ARG, "%s: row bytes %llu / %llu not multiples of 16", what,
                    static_cast<unsigned long long>(v.k_row),
                    static_cast<unsigned long long>(v.v_row));
    if (!aligned16(v.k) || !aligned16(v.v) || v.k_page % 16 || v.v_page % 16)
        return fail(KVMRET_ERR_ARG, "%s: bases and page strides must be 16-byte aligned", what);
    if (v.k_page < v.k_row * v.page_tokens || v.v_page < v.v_row * v.page_tokens)
        return fail(KVMRET_ERR_ARG, "%s: page strides %llu / %llu shorter than a page", what,
                    static_cast<unsigned long long>(v.k_page),
                    static_cast<unsigned long long>(v.v_page));
    *out = v;
    return KVMRET_OK;
}

int prefix_attn_call(const KeyList &prefix, const kvmret_pages *tail, const kvmret_attn *a,
                     void *ws, size_t ws_bytes, cudaStream_t st) {
    if (!a) return fail(KVMRET_ERR_ARG, "null arguments");
    PrefixAttn r{};
    r.prefix = prefix;
    if (a->n_seq) {
        if (const int rc = resolve_pages(tail, "tail", &r.tail.pages); rc != KVMRET_OK) return rc;
        if (r.prefix.max_len && (r.prefix.pages.n_head_kv != r.tail.pages.n_head_kv ||
                                 r.prefix.pages.d_head != r.tail.pages.d_head))
            return fail(KVMRET_ERR_ARG, "prefix of %u heads of %u, tail of %u heads of %u",
                        r.prefix.pages.n_head_kv, r.prefix.pages.d_head, r.tail.pages.n_head_kv,
                        r.tail.pages.d_head);
    } else if (!r.prefix.max_len) {
        return fail(KVMRET_ERR_ARG, "attention without a prefix or tails");
    }
    const PageView &pv = r.prefix.max_len ? r.prefix.pages : r.tail.pages;
    if ((r.prefix.max_len && r.prefix.pages.page_tokens % 16) ||
        (a->n_seq && r.tail.pages.page_tokens % 16))
        return fail(KVMRET_ERR_ARG, "attention needs pages of a multiple of 16 tokens");
    if (a->n_head == 0 || a->n_head % pv.n_head_kv || a->n_head > 65535)
        return fail(KVMRET_ERR_ARG, "n_head %u over %u KV heads", a->n_head, pv.n_head_kv);
    if (!std::isfinite(a->scale)) return fail(KVMRET_ERR_ARG, "scale must be finite");
    if (a->n_q > 65535 || a->n_seq > 65535)
        return fail(KVMRET_ERR_ARG, "n_q %u / n_seq %u above 65535", a->n_q, a->n_seq);
    if (a->n_q == 0) return KVMRET_OK;
    if (!a->q_dev || !a->out_dev) return fail(KVMRET_ERR_ARG, "null query or output");
    const uint64_t row = static_cast<uint64_t>(a->n_head) * pv.d_head;
    r.q_stride = a->q_stride ? a->q_stride : row;
    if (!aligned16(a->q_dev) || !aligned16(a->out_dev) || r.q_stride % 8)
        return fail(KVMRET_ERR_ARG, "query rows and output must be 16-byte aligned");
    if (a->n_q > 1 && r.q_stride < row)
        return fail(KVMRET_ERR_ARG, "query rows of %llu elements overlap",
                    static_cast<unsigned long long>(row));
    if (a->n_seq) {
        if (!a->q_start_dev || !a->tail_len_dev || !a->tail_table_dev || a->tail_pages == 0)
            return fail(KVMRET_ERR_ARG, "tails without their rows, lengths or pages");
        const uint64_t most = static_cast<uint64_t>(a->tail_pages) * r.tail.pages.page_tokens;
        if (most > 0x7fffffffull)
            return fail(KVMRET_ERR_ARG, "tails of %u pages pass 2^31 tokens", a->tail_pages);
        r.tail.table = a->tail_table_dev;
        r.tail.len = a->tail_len_dev;
        r.tail.n_list = a->tail_pages;
        r.tail.max_len = static_cast<uint32_t>(most);
    }
    // 32-bit rows and tile counts (at least 16 tokens a tile)
    const uint64_t units = static_cast<uint64_t>(a->n_q) * (a->n_head / pv.n_head_kv) / 128 + a->n_seq + 1;
    const uint64_t reach = r.prefix.max_len / 16ull + r.tail.max_len / 16ull + 4;
    if (static_cast<uint64_t>(a->n_q) * a->n_head > 0x7fffffffull ||
        reach > 0xffffffffull / pv.n_head_kv / units)
        return fail(KVMRET_ERR_ARG, "%u rows of %u heads over %u + %u tokens are too many for one call",
                    a->n_q, a->n_head, r.prefix.max_len, r.tail.max_len);
    r.q = a->q_dev;
    r.out = a->out_dev;
    r.lse = a->lse_dev;
    r.n_q = a->n_q;
    r.n_head = a->n_head;
    r.n_head_kv = pv.n_head_kv;
    r.d_head = pv.d_head;
    r.scale = a->scale;
    r.n_seq = a->n_seq;
    r.q_start = a->q_start_dev;
    const size_t need = prefix_attn_ws_bytes(a->n_q, a->n_head, pv.n_head_kv, pv.d_head, a->n_seq);
    if (need / (4ull * pv.d_head) > 0xffffffffull)  // its rows are counted in 32 bits
        return fail(KVMRET_ERR_ARG, "%u rows of %u heads are too many for one workspace", a->n_q, a->n_head);
    if (need && (!ws || ws_bytes < need || (reinterpret_cast<uintptr_t>(ws) & 255)))
        return fail(KVMRET_ERR_ARG, "workspace of %zu bytes at 256-byte alignment, %zu needed",
                    ws_bytes, need);
    return launched(launch_prefix_attn(r, ws, st));
}

}  // namespace kvmret

extern "C" {

int kvmret_qk_norm_rope(const kvmret_qk *a, void *stream) {
    if (!a) return fail(KVMRET_ERR_ARG, "null arguments");
    if (!head_ok(a->d_head) || a->n_rot != a->d_head)
        return fail(KVMRET_ERR_ARG, "qk_norm_rope needs d_head in {64,128,256} and n_rot == d_head");
    if (a->fwht_n != 0 && a->fwht_n != a->d_head)
        return fail(KVMRET_ERR_ARG, "fwht_n must be 0 or d_head");
    uint32_t size = 2;
    if (a->type == KVMRET_TYPE_F32)
        size = 4;
    else if (a->type != KVMRET_TYPE_F16 && a->type != KVMRET_TYPE_BF16)
        return fail(KVMRET_ERR_ARG, "type %d unsupported (f16, bf16 or f32)", a->type);
    if (!(a->eps >= 0.0f) || !std::isfinite(a->eps))
        return fail(KVMRET_ERR_ARG, "eps must be finite and >= 0");
    if (!rope_ok(a->freq_base, a->freq_scale))
        return fail(KVMRET_ERR_ARG, "freq_base must be > 0, freq_scale finite");
    if (a->n_tok == 0) return KVMRET_OK;
    if (!a->pos_dev) return fail(KVMRET_ERR_ARG, "null positions");
    kvmret::QkNormRope r{};
    struct Side {
        const void *in;
        uint64_t stride;
        uint16_t *rot, *raw;
        uint32_t heads;
        const char *name;
    } side[2] = {{a->q_dev, a->q_stride, a->q_rot_dev, a->q_raw_dev, a->n_head, "q"},
                 {a->k_dev, a->k_stride, a->k_rot_dev, a->k_raw_dev, a->n_head_kv, "k"}};
    for (Side &s : side) {
        if (!s.rot && !s.raw) {  // nothing wanted of this side
            s.heads = 0;
            continue;
        }
        if (!s.in) return fail(KVMRET_ERR_ARG, "outputs of %s without its rows", s.name);
        if (s.heads == 0 || s.heads > 65535)
            return fail(KVMRET_ERR_ARG, "%u heads of %s not in 1..65535", s.heads, s.name);
        if (s.stride < static_cast<uint64_t>(s.heads) * a->d_head && a->n_tok > 1)
            return fail(KVMRET_ERR_ARG, "%s rows of %u heads overlap at a stride of %llu elements",
                        s.name, s.heads, static_cast<unsigned long long>(s.stride));
        if (!aligned16(s.in) || s.stride * size % 16 || !aligned16(s.rot) || !aligned16(s.raw))
            return fail(KVMRET_ERR_ARG, "%s rows and outputs must be 16-byte aligned", s.name);
    }
    r.q = a->q_dev;
    r.k = a->k_dev;
    r.q_stride = a->q_stride;
    r.k_stride = a->k_stride;
    r.q_weight = a->q_weight_dev;
    r.k_weight = a->k_weight_dev;
    r.pos = a->pos_dev;
    r.q_rot = a->q_rot_dev;
    r.k_rot = a->k_rot_dev;
    r.q_raw = a->q_raw_dev;
    r.k_raw = a->k_raw_dev;
    r.n_tok = a->n_tok;
    r.n_head = side[0].heads;
    r.n_head_kv = side[1].heads;
    r.d_head = a->d_head;
    r.type = a->type;
    r.eps = a->eps;
    r.fwht_n = a->fwht_n;
    r.theta = make_theta(a->n_rot, a->freq_base, a->freq_scale);
    if (r.n_head + r.n_head_kv == 0) return KVMRET_OK;
    return launched(kvmret::launch_qk_norm_rope(r, static_cast<cudaStream_t>(stream)));
}

int kvmret_paged_append(const kvmret_pages *pages, const uint16_t *k, uint64_t k_stride,
                        const uint16_t *v, uint64_t v_stride, const int32_t *cells,
                        const int32_t *pos, uint32_t n_tok, float freq_base, float freq_scale,
                        uint32_t fwht_n, void *stream) {
    kvmret::PagedAppend a{};
    if (const int rc = kvmret::resolve_pages(pages, "paged_append", &a.pages); rc != KVMRET_OK)
        return rc;
    if (fwht_n != 0 && fwht_n != a.pages.d_head)
        return fail(KVMRET_ERR_ARG, "fwht_n must be 0 or d_head");
    if (pos && !rope_ok(freq_base, freq_scale))
        return fail(KVMRET_ERR_ARG, "freq_base must be > 0, freq_scale finite");
    if (n_tok == 0) return KVMRET_OK;
    if (!k || !v || !cells) return fail(KVMRET_ERR_ARG, "null buffer");
    const uint64_t e = static_cast<uint64_t>(a.pages.n_head_kv) * a.pages.d_head;
    a.k_stride = k_stride ? k_stride : e;
    a.v_stride = v_stride ? v_stride : e;
    if (!aligned16(k) || !aligned16(v) || a.k_stride % 8 || a.v_stride % 8)
        return fail(KVMRET_ERR_ARG, "k and v rows must be 16-byte aligned");
    if (n_tok > 1 && (a.k_stride < e || a.v_stride < e))
        return fail(KVMRET_ERR_ARG, "k or v rows of %llu elements overlap",
                    static_cast<unsigned long long>(e));
    a.k = k;
    a.v = v;
    a.cells = cells;
    a.pos = pos;
    a.n_tok = n_tok;
    a.fwht_n = fwht_n;
    if (pos) a.theta = make_theta(a.pages.d_head, freq_base, freq_scale);
    return launched(kvmret::launch_paged_append(a, static_cast<cudaStream_t>(stream)));
}

size_t kvmret_prefix_attn_ws_bytes(uint32_t n_q, uint32_t n_head, uint32_t n_head_kv,
                                   uint32_t d_head, uint32_t n_seq) {
    if (n_head_kv == 0 || n_head % n_head_kv || !head_ok(d_head) || n_q > 65535 || n_seq > 65535)
        return 0;
    return kvmret::prefix_attn_ws_bytes(n_q, n_head, n_head_kv, d_head, n_seq);
}

int kvmret_prefix_attn(const kvmret_pages *prefix, const kvmret_pages *tail, const kvmret_attn *a,
                       void *ws, size_t ws_bytes, void *stream) {
    if (!a) return fail(KVMRET_ERR_ARG, "null arguments");
    kvmret::KeyList p{};
    if (a->max_prefix) {
        if (a->max_prefix > 0x7fffffffu)
            return fail(KVMRET_ERR_ARG, "max_prefix %u passes 2^31 - 1", a->max_prefix);
        if (const int rc = kvmret::resolve_pages(prefix, "prefix", &p.pages); rc != KVMRET_OK)
            return rc;
        p.table = a->prefix_table_dev;
        p.ntok = a->prefix_ntok_dev;
        p.len = a->prefix_len_dev;
        p.max_len = a->max_prefix;
        p.n_list = (a->max_prefix - 1) / p.pages.page_tokens + 1;
        if (!p.table && p.n_list > p.pages.n_pages)
            return fail(KVMRET_ERR_ARG, "max_prefix %u passes the %u pages", a->max_prefix,
                        p.pages.n_pages);
    }
    return kvmret::prefix_attn_call(p, tail, a, ws, ws_bytes, static_cast<cudaStream_t>(stream));
}

}  // extern "C"
